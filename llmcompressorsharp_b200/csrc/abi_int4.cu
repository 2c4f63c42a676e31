// extern "C" entry points of the packed 4-bit products and of the embedding (llmc_b200.h).
#include "ops.h"

namespace llmc {
namespace {

// Makes `device` current and gives the calling thread its own back.  The device is set even where it is current
// already: a thread that has made no CUDA call yet (autograd's) has no context that cuTensorMapEncodeTiled could use.
struct DeviceScope {
    int prev = -1;
    llmc_status enter(int device) {
        int cur = -1;
        LLMC_CUDA_TRY(cudaGetDevice(&cur));
        LLMC_CUDA_TRY(cudaSetDevice(device));
        if (cur != device) prev = cur;
        return LLMC_OK;
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

constexpr int64_t MAX_DIM = (int64_t)1 << 30;     // rows, columns, tokens
// Products that go to the few-row kernel, which reads the codes anew for each 16 tokens: few tokens, and more while the
// tensor-core kernel, which takes as long for 17 tokens as for 128, does not pass it.  us here and there, 16-bit: 4096 -> 14336,
// 32 tokens 33 and 33, 48: 47 and 33; 4096 -> 4096, 32: 12.5 and 16.5, 64: 18.1 and 17.1; 576 -> 1536, 256: 11.5 and 14.
// fp32 costs six products there and three here: 4096 -> 14336, 256: 373 and 489; 4096 -> 4096, 256: 114 and 127; with
// few columns (not eight tiles) there is less to overlap: 576 -> 49152, 64: 117 and 118, 96: 172 and 122.  The borders lie
// between these shapes; others near them may be up to a third slower on the side that they are given.
bool few_rows(bool f32, int64_t tokens, int64_t rows, int64_t cols) {
    if (tokens <= (f32 ? 64 : 32)) return true;
    if (tokens > 256) return false;
    return (f32 && cols >= 8 * w4::TILE) || (tokens + 15) / 16 * rows * cols <= (int64_t)1 << (f32 ? 27 : 25);
}

llmc_status check_sizes(int64_t rows, int64_t cols, int64_t gs) {
    if (rows <= 0 || cols <= 0) return fail(LLMC_ERR_SHAPE, "a packed weight needs positive sizes (got %lld x %lld)", (long long)rows, (long long)cols);
    if (rows > MAX_DIM || cols > MAX_DIM) return fail(LLMC_ERR_OUT_OF_RANGE, "a packed weight has at most 2^30 rows and columns");
    if (gs < 16 && gs < cols)
        return fail(LLMC_ERR_UNSUPPORTED, "group_size must be at least 16, or at least the columns (got %lld)", (long long)gs);
    // the kernels count the layout's columns, up to twice the weight's (groups of 16 take 32 each), in 32 bits
    if (gs < cols && (cols + gs - 1) / gs * w4::up(gs, 32) > MAX_DIM)
        return fail(LLMC_ERR_OUT_OF_RANGE, "%lld columns in groups of %lld take more than 2^30 of the layout", (long long)cols, (long long)gs);
    return LLMC_OK;
}

llmc_status view_of(const llmc_int4_weight* w, w4::View& v) {
    if (!w) return fail(LLMC_ERR_INVALID_ARG, "weight must not be null");
    if (!w->packed || !w->exps) return fail(LLMC_ERR_INVALID_ARG, "the weight's arrays must not be null");
    if ((uintptr_t)w->packed % 16 != 0) return fail(LLMC_ERR_INVALID_ARG, "packed must be 16-byte aligned");
    LLMC_TRY(check_sizes(w->rows, w->cols, w->group_size));
    v.packed = w->packed;
    v.exps = w->exps;
    w4::set_sizes(v, w->rows, w->cols, w->group_size);
    return LLMC_OK;
}

cudaStream_t stream_of(llmc_ctx* ctx, void* s) { return s ? (cudaStream_t)s : ctx->stream; }

llmc_status check_matrix(const char* name, const void* p, int32_t dtype, int64_t rows, int64_t cols, int64_t ld) {
    if (!dtype_ok(dtype)) return fail(LLMC_ERR_INVALID_ARG, "unsupported dtype %d", dtype);
    if (rows < 0 || rows > MAX_DIM) return fail(LLMC_ERR_SHAPE, "%s: bad number of rows (%lld)", name, (long long)rows);
    if (ld < cols) return fail(LLMC_ERR_SHAPE, "%s: last dim (ld=%lld) must be at least %lld", name, (long long)ld, (long long)cols);
    if (rows > 0 && !p) return fail(LLMC_ERR_INVALID_ARG, "%s must not be null", name);
    if ((uintptr_t)p % dtype_size(dtype) != 0) return fail(LLMC_ERR_INVALID_ARG, "%s is not aligned to its type", name);
    return LLMC_OK;
}

llmc_status check_ws(const void* ws, int64_t have, size_t need) {
    if (need == 0) return LLMC_OK;
    if (!ws || have < (int64_t)need)
        return fail(LLMC_ERR_INVALID_ARG, "the workspace needs %zu bytes (got %lld)", need, (long long)(ws ? have : 0));
    if ((uintptr_t)ws % 256 != 0) return fail(LLMC_ERR_INVALID_ARG, "the workspace must be 256-byte aligned");
    return LLMC_OK;
}

llmc_status check_ids(const void* ids, int32_t ids64, int64_t tokens) {
    if (tokens < 0 || tokens > MAX_DIM) return fail(LLMC_ERR_SHAPE, "bad number of ids (%lld)", (long long)tokens);
    if (tokens > 0 && !ids) return fail(LLMC_ERR_INVALID_ARG, "ids must not be null");
    if ((uintptr_t)ids % (ids64 ? 8 : 4) != 0) return fail(LLMC_ERR_INVALID_ARG, "ids are not aligned to their type");
    return LLMC_OK;
}

// How one product runs: the few-row kernel or the tensor-core one, on x itself or on a staged copy, in
// how many splits of the contraction.
struct LinearPlan {
    bool few, stage;
    int64_t pitch;
    int pieces, splits;
    size_t part_at, bytes;
};

LinearPlan plan_linear(const llmc_ctx* ctx, const w4::View& v, int dir, const void* a, int dtype, int64_t tokens, int64_t ld) {
    LinearPlan p{};
    const bool f32 = dtype == LLMC_DTYPE_F32;
    p.few = dir == 0 && few_rows(f32, tokens, v.rows, v.cols);
    // 16-byte rows are what both kernels load; the few-row one reads whole vectors of eight columns, TMA
    // fills what is past the last column.  fp32 is read in bf16 pieces, other groups in the layout's columns.
    p.stage = f32 || (uintptr_t)a % 16 != 0 || (ld % 8 != 0) || (dir == 0 && !v.identity) || (p.few && v.cols % 8 != 0);
    p.pitch = dir == 0 ? v.kp : v.mp;
    p.pieces = !f32 ? 1 : p.few ? 3 : 4;
    size_t off = p.stage ? align_up((size_t)p.pieces * tokens * p.pitch * 2, 256) : 0;
    p.splits = 1;
    p.part_at = off;
    if (!p.few) {
        p.splits = int4_gemm_splits(ctx, dtype, tokens, dir == 0 ? v.rows : v.kp, p.pitch);
        if (p.splits > 1) off += align_up((size_t)p.splits * tokens * (dir == 0 ? v.rows : v.cols) * sizeof(float), 256);
    }
    p.bytes = off;
    return p;
}

llmc_status run_linear(llmc_ctx* ctx, void* stream, const llmc_int4_weight* w, int dir, const void* a, int32_t dtype, int64_t tokens,
                       int64_t ld, const void* bias, void* out, int64_t ldo, void* ws, int64_t ws_bytes) {
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    w4::View v;
    LLMC_TRY(view_of(w, v));
    const int64_t in = dir == 0 ? v.cols : v.rows, on = dir == 0 ? v.rows : v.cols;
    LLMC_TRY(check_matrix(dir == 0 ? "x" : "dy", a, dtype, tokens, in, ld));
    LLMC_TRY(check_matrix(dir == 0 ? "y" : "dx", out, dtype, tokens, on, ldo));
    if ((uintptr_t)bias % dtype_size(dtype) != 0) return fail(LLMC_ERR_INVALID_ARG, "bias is not aligned to its type");
    const LinearPlan p = plan_linear(ctx, v, dir, a, dtype, tokens, ld);
    LLMC_TRY(check_ws(ws, ws_bytes, p.bytes));
    if (tokens == 0) return LLMC_OK;
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    cudaStream_t st = stream_of(ctx, stream);
    int64_t acols = in, lda = ld;
    if (p.stage) {
        LLMC_TRY(int4_stage(ctx, st, a, dtype, tokens, in, ld, p.pitch, dir == 0 ? &v : nullptr, p.pieces, (uint16_t*)ws));
        a = ws;
        acols = lda = p.pitch;
    }
    if (p.few) return int4_few(ctx, st, v, a, dtype, tokens, lda, acols, bias, out, ldo);
    float* part = (float*)((char*)ws + p.part_at);
    LLMC_TRY(int4_gemm(ctx, st, v, dir, dtype, a, acols, lda, tokens, bias, out, ldo, p.splits, part));
    if (p.splits > 1) LLMC_TRY(int4_join(ctx, st, part, p.splits, tokens, on, bias, out, dtype, ldo));
    return LLMC_OK;
}

llmc_status linear_bytes(llmc_ctx* ctx, const llmc_int4_weight* w, int dir, const void* a, int32_t dtype, int64_t tokens, int64_t ld,
                         int64_t* bytes) {
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    if (!bytes) return fail(LLMC_ERR_INVALID_ARG, "bytes must not be null");
    w4::View v;
    LLMC_TRY(view_of(w, v));
    if (!dtype_ok(dtype)) return fail(LLMC_ERR_INVALID_ARG, "unsupported dtype %d", dtype);
    if (tokens < 0 || tokens > MAX_DIM) return fail(LLMC_ERR_SHAPE, "bad number of rows (%lld)", (long long)tokens);
    *bytes = (int64_t)plan_linear(ctx, v, dir, a, dtype, tokens, ld).bytes;
    return LLMC_OK;
}

// Parts of a column sum's rows: enough to occupy the device, 256 rows each at least (a part less is a launch less at
// one: 96 rows of 1,536 columns take 2 us in one part).
int col_sum_splits(const llmc_ctx* ctx, int64_t rows, int64_t cols) {
    const int64_t blocks = (cols + 31) / 32;
    int64_t s = (8 * (int64_t)ctx->sm_count + blocks - 1) / blocks;
    if (s > (rows + 255) / 256) s = (rows + 255) / 256;
    return (int)(s < 1 ? 1 : (s > 1024 ? 1024 : s));
}

}  // namespace
}  // namespace llmc

using namespace llmc;

extern "C" {

llmc_status llmc_int4_layout_sizes(int64_t rows, int64_t cols, int64_t group_size, int64_t* packed_bytes, int64_t* exps) {
    LLMC_ENTRY();
    if (!packed_bytes || !exps) return fail(LLMC_ERR_INVALID_ARG, "the sizes must not be null");
    LLMC_TRY(check_sizes(rows, cols, group_size));
    w4::View v{};
    w4::set_sizes(v, rows, cols, group_size);
    *packed_bytes = v.mp / w4::ROWS * (v.kp / w4::TILE) * v.rec;
    *exps = v.mp + v.kp / w4::TILE * v.ng;
    return LLMC_OK;
}

llmc_status llmc_int4_layout(llmc_ctx* ctx, void* stream, const uint8_t* codes, int64_t crow, const float* scales, const int32_t* zps,
                             int32_t strategy, int32_t symmetric, const llmc_int4_weight* w) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    w4::View v;
    LLMC_TRY(view_of(w, v));
    if (!codes) return fail(LLMC_ERR_INVALID_ARG, "codes must not be null");
    if (!scales) return fail(LLMC_ERR_INVALID_ARG, "scales must not be null");
    if (!symmetric && !zps) return fail(LLMC_ERR_INVALID_ARG, "an asymmetric grid needs zero-points");
    if (crow < (v.cols + 1) / 2) return fail(LLMC_ERR_SHAPE, "crow (%lld) is less than a row's bytes", (long long)crow);
    int64_t srow;
    if (strategy == LLMC_STRATEGY_GROUP) srow = v.groups;
    else if (strategy == LLMC_STRATEGY_CHANNEL) srow = 1;
    else if (strategy == LLMC_STRATEGY_TENSOR) srow = 0;
    else return fail(LLMC_ERR_UNSUPPORTED, "Quantization strategy %d is not supported.", strategy);
    if (strategy != LLMC_STRATEGY_GROUP && v.groups != 1)
        return fail(LLMC_ERR_SHAPE, "a tensor or channel scale needs group_size >= cols");
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    return int4_layout(ctx, stream_of(ctx, stream), codes, crow, scales, zps, srow, symmetric ? 1 : 0, v, const_cast<uint8_t*>(w->packed),
                       const_cast<int32_t*>(w->exps));
}

llmc_status llmc_int4_dequantize(llmc_ctx* ctx, void* stream, const llmc_int4_weight* w, int32_t dtype, void* out, int64_t ldo) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    w4::View v;
    LLMC_TRY(view_of(w, v));
    LLMC_TRY(check_matrix("out", out, dtype, v.rows, v.cols, ldo));
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    return int4_rows(ctx, stream_of(ctx, stream), v, nullptr, 0, v.rows, 1.f, out, dtype, ldo);
}

llmc_status llmc_int4_linear_workspace(llmc_ctx* ctx, const llmc_int4_weight* w, const void* x, int32_t dtype, int64_t tokens, int64_t ldx,
                                       int64_t* bytes) {
    LLMC_ENTRY();
    return linear_bytes(ctx, w, 0, x, dtype, tokens, ldx, bytes);
}

llmc_status llmc_int4_linear(llmc_ctx* ctx, void* stream, const llmc_int4_weight* w, const void* x, int32_t dtype, int64_t tokens, int64_t ldx,
                             const void* bias, void* y, int64_t ldy, void* ws, int64_t ws_bytes) {
    LLMC_ENTRY();
    return run_linear(ctx, stream, w, 0, x, dtype, tokens, ldx, bias, y, ldy, ws, ws_bytes);
}

llmc_status llmc_int4_linear_grad_workspace(llmc_ctx* ctx, const llmc_int4_weight* w, const void* dy, int32_t dtype, int64_t tokens,
                                            int64_t lddy, int64_t* bytes) {
    LLMC_ENTRY();
    return linear_bytes(ctx, w, 1, dy, dtype, tokens, lddy, bytes);
}

llmc_status llmc_int4_linear_grad(llmc_ctx* ctx, void* stream, const llmc_int4_weight* w, const void* dy, int32_t dtype, int64_t tokens,
                                  int64_t lddy, void* dx, int64_t lddx, void* ws, int64_t ws_bytes) {
    LLMC_ENTRY();
    return run_linear(ctx, stream, w, 1, dy, dtype, tokens, lddy, nullptr, dx, lddx, ws, ws_bytes);
}

llmc_status llmc_col_sum_workspace(llmc_ctx* ctx, int64_t rows, int64_t cols, int64_t* bytes) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    if (!bytes) return fail(LLMC_ERR_INVALID_ARG, "bytes must not be null");
    if (rows < 0 || rows > MAX_DIM || cols <= 0 || cols > MAX_DIM) return fail(LLMC_ERR_SHAPE, "bad shape");
    *bytes = (int64_t)align_up((size_t)col_sum_splits(ctx, rows, cols) * cols * sizeof(float), 256);
    return LLMC_OK;
}

llmc_status llmc_col_sum(llmc_ctx* ctx, void* stream, const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld, void* out,
                         void* ws, int64_t ws_bytes) {
    LLMC_ENTRY();
    int64_t need = 0;
    LLMC_TRY(llmc_col_sum_workspace(ctx, rows, cols, &need));
    LLMC_TRY(check_matrix("x", x, dtype, rows, cols, ld));
    LLMC_TRY(check_matrix("out", out, dtype, 1, cols, cols));
    LLMC_TRY(check_ws(ws, ws_bytes, (size_t)need));
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    cudaStream_t st = stream_of(ctx, stream);
    const int splits = col_sum_splits(ctx, rows, cols);
    return col_sum(ctx, st, x, dtype, rows, cols, ld, splits, (float*)ws, out);
}

llmc_status llmc_embedding(llmc_ctx* ctx, void* stream, const void* ids, int32_t ids64, int64_t tokens, const void* table, int32_t dtype,
                           int64_t vocab, int64_t hidden, int64_t ldt, float scale, void* out, int64_t ldo) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    LLMC_TRY(check_ids(ids, ids64, tokens));
    if (vocab <= 0 || hidden <= 0 || hidden > MAX_DIM) return fail(LLMC_ERR_SHAPE, "a table needs positive sizes (got %lld x %lld)", (long long)vocab, (long long)hidden);
    LLMC_TRY(check_matrix("table", table, dtype, vocab, hidden, ldt));
    LLMC_TRY(check_matrix("out", out, dtype, tokens, hidden, ldo));
    if (tokens == 0) return LLMC_OK;
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    return embedding_lookup(ctx, stream_of(ctx, stream), ids, ids64, tokens, table, dtype, vocab, hidden, ldt, scale, out, ldo);
}

llmc_status llmc_int4_embedding(llmc_ctx* ctx, void* stream, const void* ids, int32_t ids64, int64_t tokens, const llmc_int4_weight* w,
                                int32_t dtype, float scale, void* out, int64_t ldo) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    LLMC_TRY(check_ids(ids, ids64, tokens));
    w4::View v;
    LLMC_TRY(view_of(w, v));
    LLMC_TRY(check_matrix("out", out, dtype, tokens, v.cols, ldo));
    if (tokens == 0) return LLMC_OK;
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    return int4_rows(ctx, stream_of(ctx, stream), v, ids, ids64, tokens, scale, out, dtype, ldo);
}

llmc_status llmc_embedding_grad_workspace(llmc_ctx* ctx, int64_t tokens, int64_t vocab, int64_t hidden, int64_t* bytes) {
    LLMC_ENTRY();
    if (!ctx) return fail(LLMC_ERR_INVALID_ARG, "context must not be null");
    if (!bytes) return fail(LLMC_ERR_INVALID_ARG, "bytes must not be null");
    if (tokens < 0 || tokens > MAX_DIM) return fail(LLMC_ERR_SHAPE, "bad number of ids (%lld)", (long long)tokens);
    if (vocab <= 0 || vocab > MAX_DIM || hidden <= 0 || hidden > MAX_DIM) return fail(LLMC_ERR_SHAPE, "a table needs positive sizes (got %lld x %lld)", (long long)vocab, (long long)hidden);
    *bytes = (int64_t)embedding_grad_bytes(tokens, vocab, hidden);
    return LLMC_OK;
}

llmc_status llmc_embedding_grad(llmc_ctx* ctx, void* stream, const void* ids, int32_t ids64, int64_t tokens, const void* dy, int32_t dtype,
                                int64_t lddy, int64_t vocab, int64_t hidden, float scale, int64_t padding_idx, void* dtable, void* ws,
                                int64_t ws_bytes) {
    LLMC_ENTRY();
    int64_t need = 0;
    LLMC_TRY(llmc_embedding_grad_workspace(ctx, tokens, vocab, hidden, &need));
    LLMC_TRY(check_ids(ids, ids64, tokens));
    if (padding_idx < -1 || padding_idx >= vocab) return fail(LLMC_ERR_OUT_OF_RANGE, "padding_idx %lld is outside the table", (long long)padding_idx);
    LLMC_TRY(check_matrix("dy", dy, dtype, tokens, hidden, lddy));
    LLMC_TRY(check_matrix("dtable", dtable, dtype, vocab, hidden, hidden));
    LLMC_TRY(check_ws(ws, ws_bytes, (size_t)need));
    DeviceScope scope;
    LLMC_TRY(scope.enter(ctx->device));
    cudaStream_t st = stream_of(ctx, stream);
    if (tokens == 0) {
        LLMC_CUDA_TRY(cudaMemsetAsync(dtable, 0, (size_t)vocab * hidden * dtype_size(dtype), st));
        return LLMC_OK;
    }
    return embedding_grad(ctx, st, ids, ids64, tokens, dy, dtype, lddy, vocab, hidden, scale, padding_idx, dtable, ws);
}

}  // extern "C"
