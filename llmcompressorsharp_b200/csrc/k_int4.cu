// Packed 4-bit weights: laying them out, reading them back, and products with few rows.
//
// The reference quantises (RtnModifier.cs:44-122, GPTQModifier.cs:108-137) and dequantises
// (Int4PackedTensor.cs:152-161); it multiplies only dense weights.  These kernels take the codes as
// they are: y[t][n] = sum_k x[t][k] (u - z) s + b[n].
#include "int4.cuh"
#include "ops.h"

namespace llmc {
namespace {

using namespace w4;

// ---- layout ---------------------------------------------------------------------------------------
struct LayoutArgs {
    const uint8_t* codes;
    int64_t crow;
    const float* scales;
    const int32_t* zps;
    int64_t srow;      // scale entries per row (0: one entry for the tensor)
    int sym;
    View v;
    uint32_t* packed;
    float* sout;
    uint8_t* zout;
};

__device__ __forceinline__ uint32_t zero_of(const LayoutArgs& a, int64_t r, int g) {
    if (a.sym || r >= a.v.rows) return 8u;
    return (uint32_t)a.zps[a.srow ? r * a.srow + g : 0] & 0xFu;
}

// One thread per word of eight codes; one read of the codes and one write, bound by memory.
__global__ void __launch_bounds__(256) layout_kernel(const LayoutArgs a) {
    const int64_t words = a.v.mp * (a.v.kp / 8);
    const int64_t ktiles = a.v.kp / TILE;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int64_t tile = i / TILE_WORDS;
        const int in = (int)(i % TILE_WORDS), t = (in % 16) / 4, c = in % 4;
        const int64_t r = tile / ktiles * TILE + in / 16;
        const int kv0 = (int)(tile % ktiles) * TILE + 32 * c + 8 * t;
        const int g = group_of(kv0, a.v.gsv, a.v.groups);
        const uint32_t z = zero_of(a, r, g);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t u = z;
            const int64_t k = r < a.v.rows ? column_of(kv0 + j, a.v.gs, a.v.gsv, a.v.groups, a.v.cols) : -1;
            if (k >= 0) {
                const uint32_t b = a.codes[r * a.crow + (k >> 1)];
                const uint32_t nib = (k & 1) ? (b & 0xFu) : (b >> 4);
                // the code is (q - zp) mod 16; u = q (asymmetric) or q + 8 (symmetric, zp = 0)
                u = (nib + z) & 0xFu;
            }
            w |= u << ((j & 1) * 16 + (j >> 1) * 4);
        }
        a.packed[i] = w;
    }
    const int64_t entries = a.v.mp * a.v.groups;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
        const int64_t g = i / a.v.mp, r = i % a.v.mp;
        a.sout[i] = r < a.v.rows ? a.scales[a.srow ? r * a.srow + g : 0] : 0.f;
        a.zout[i] = (uint8_t)zero_of(a, r, (int)g);
    }
}

// Exponents that bring the scales near one before they meet fp16's range: for each row, and for each
// group, e with 2^(e-1) <= max |s| < 2^e, within +-120 (0 where the maximum is 0 or not finite).  A product
// kernel in fp16 uses s 2^-e and gives 2^e back in fp32, both exact.
__global__ void __launch_bounds__(256) exps_kernel(const float* scales, int64_t mp, int groups, int32_t* exps) {
    const int64_t row_blocks = mp / TILE;
    float m = 0.f;
    __shared__ float sm[256];
    const bool rows = blockIdx.x < row_blocks;
    if (rows) {
        const int64_t r = (int64_t)blockIdx.x * TILE + threadIdx.x % TILE;
        for (int g = threadIdx.x / TILE; g < groups; g += 2) m = fmax_nan(m, fabsf(scales[(int64_t)g * mp + r]));
    } else {
        const int64_t g = blockIdx.x - row_blocks;
        for (int64_t r = threadIdx.x; r < mp; r += 256) m = fmax_nan(m, fabsf(scales[g * mp + r]));
    }
    sm[threadIdx.x] = m;
    for (int step = 128; step >= (rows ? TILE : 1); step >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < step) sm[threadIdx.x] = fmax_nan(sm[threadIdx.x], sm[threadIdx.x + step]);
    }
    __syncthreads();
    m = sm[threadIdx.x];
    int e = 0;
    if (m > 0.f && isfinite(m)) frexpf(m, &e);
    e = min(120, max(-120, e));
    if (rows) {
        if (threadIdx.x < TILE) exps[(int64_t)blockIdx.x * TILE + threadIdx.x] = e;
    } else if (threadIdx.x == 0) {
        exps[mp + blockIdx.x - row_blocks] = e;
    }
}

// ---- reading back, and looking rows up ------------------------------------------------------------
template <typename T> __device__ __forceinline__ void store8(T* dst, const float (&v)[8], bool wide, int n) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            union { T h[8]; uint4 u; } o;
#pragma unroll
            for (int j = 0; j < 8; j++) o.h[j] = from_f<T>(v[j]);
            *reinterpret_cast<uint4*>(dst) = o.u;
        }
    } else {
        for (int j = 0; j < n; j++) dst[j] = from_f<T>(v[j]);
    }
}

// out[t] = scale * W[ids ? ids[t] : t], rounded once to T.  One thread per word: eight columns of one
// row, sixteen lanes per 64 bytes of a tile's row.  Bound by the writes.  An id outside [0, rows)
// writes zeros and raises the context's flag.
template <typename T, typename I>
__global__ void __launch_bounds__(256) rows_kernel(const View v, const I* ids, int64_t tokens, float scale, T* out,
                                                  int64_t ldo, int wide, int* flag) {
    const int64_t wpr = v.kp / 8;
    const int64_t total = tokens * wpr;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / wpr;
        const int b = (int)(i % wpr), kt = b / 16, kb = b % 16;  // word of the row: columns 8 b ..
        int64_t r = t;
        bool ok = true;
        if (ids) {
            r = (int64_t)ids[t];
            ok = r >= 0 && r < v.rows;
            if (!ok) atomicOr(flag, 1);
        }
        const int kv0 = b * 8;
        const int g = group_of(kv0, v.gsv, v.groups);
        float val[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ok) {
            const uint32_t w = v.packed[((r / TILE) * (v.kp / TILE) + kt) * TILE_WORDS + (r % TILE) * 16 + (kb % 4) * 4 + kb / 4];
            const float s = v.scales[g * v.mp + r];
            const int z = v.zeros[g * v.mp + r];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int u = (int)(w >> ((j & 1) * 16 + (j >> 1) * 4)) & 0xF;
                val[j] = __fmul_rn(__fmul_rn((float)(u - z), s), scale);
            }
        }
        T* dst = out + t * ldo;
        if (v.identity) {
            const int n = (int)min((int64_t)8, v.cols - kv0);
            if (n > 0) store8<T>(dst + kv0, val, wide && n == 8, n);
        } else {
            for (int j = 0; j < 8; j++) {
                const int64_t k = column_of(kv0 + j, v.gs, v.gsv, v.groups, v.cols);
                if (k >= 0) dst[k] = from_f<T>(val[j]);
            }
        }
    }
}

// ---- x in the layout's columns ------------------------------------------------------------------
// out[p][t][kv], p < pieces: x[t][k(kv)] in its own 16-bit type, zeros where no column is; or, for fp32,
// three bf16 pieces whose sum is x exactly: each takes the eight leading bits that are left (truncated, so
// nothing overflows).  An infinity or a NaN is all in the first piece; a fourth (pieces = 4) is the first with
// zeros in their place, for products with the smaller pieces of a weight, where an infinity times zero or
// times the other sign would make a NaN that the whole product does not have.
template <typename T>
__global__ void __launch_bounds__(256) stage_kernel(const T* x, int64_t tokens, int64_t n, int64_t ldx, int64_t pitch,
                                                   int gs, int gsv, int groups, int pieces, uint16_t* out) {
    const int64_t per = pitch / 8, total = tokens * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per;
        const int kv0 = (int)(i % per) * 8;
        union { uint16_t h[8]; uint4 u; } p[4];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int64_t k = gs ? column_of(kv0 + j, gs, gsv, groups, n) : (kv0 + j < n ? kv0 + j : -1);
            T v = k >= 0 ? x[t * ldx + k] : from_f<T>(0.f);
            if constexpr (sizeof(T) == 4) {
                const float f = v;
                const uint32_t b = __float_as_uint(f);
                const bool fin = isfinite(f);
                const float hi = __uint_as_float(b & 0xFFFF0000u);
                const float r1 = fin ? __fsub_rn(f, hi) : 0.f;
                const float mid = __uint_as_float(__float_as_uint(r1) & 0xFFFF0000u);
                const float lo = __fsub_rn(r1, mid);
                p[0].h[j] = f != f ? (uint16_t)0x7FC0 : (uint16_t)(b >> 16);
                p[1].h[j] = (uint16_t)(__float_as_uint(mid) >> 16);
                p[2].h[j] = (uint16_t)(__float_as_uint(lo) >> 16);
                p[3].h[j] = fin ? p[0].h[j] : (uint16_t)0;
            } else {
                p[0].h[j] = *reinterpret_cast<uint16_t*>(&v);
            }
        }
#pragma unroll
        for (int q = 0; q < (sizeof(T) == 4 ? 4 : 1); q++)
            if (q < pieces) *reinterpret_cast<uint4*>(out + ((int64_t)q * tokens + t) * pitch + kv0) = p[q].u;
    }
}

// ---- products with few rows ---------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct FewArgs {
    View v;
    const void* x;      // [PIECES][tokens][ldx], 16-byte aligned rows, columns of the layout
    int64_t ldx, xcols; // xcols: columns to read (a multiple of 8)
    int tokens;
    const void* bias;
    void* y;
    int64_t ldy;
};

// The codes are the A operand of m16n8k16 (16 weight rows x 16 columns), x the B operand (8 tokens), so one
// dequantised fragment serves eight tokens and a single token costs no more than the codes.  Codes enter as
// the exact integers u - z; the fp32 sum of a group is multiplied by its scale (FL granules of 32 columns
// per group sum), so x and W are never rounded.
// A CTA holds 16 rows; its warps take the 128-column tiles in turn and add their sums in shared memory, in
// warp order.
template <typename T, typename O, int NT, int PIECES, int FL>
__global__ void __launch_bounds__(256) few_kernel(const FewArgs a) {
    extern __shared__ float red[];  // [warps][16][8 NT]
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const int g = lane >> 2, t = lane & 3;
    const int64_t row0 = (int64_t)blockIdx.x * 16;
    const int ktiles = (int)(a.v.kp / TILE);
    const uint4* wp = reinterpret_cast<const uint4*>(a.v.packed) + (row0 / TILE) * ktiles * (TILE_WORDS / 4) +
                      (row0 % TILE + g) * 4 + t;
    const T* x = reinterpret_cast<const T*>(a.x);
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[n][j] = 0.f;

    uint4 wa, wb;
    if (warp < ktiles) {
        wa = __ldcs(wp + (int64_t)warp * (TILE_WORDS / 4));
        wb = __ldcs(wp + (int64_t)warp * (TILE_WORDS / 4) + 8 * 4);
    }
    for (int kt = warp; kt < ktiles; kt += warps) {
        const uint4 ca = wa, cb = wb;
        if (kt + warps < ktiles) {
            wa = __ldcs(wp + (int64_t)(kt + warps) * (TILE_WORDS / 4));
            wb = __ldcs(wp + (int64_t)(kt + warps) * (TILE_WORDS / 4) + 8 * 4);
        }
        const uint32_t w0[4] = {ca.x, ca.y, ca.z, ca.w}, w1[4] = {cb.x, cb.y, cb.z, cb.w};
        float d[NT][4];
        uint32_t z0 = 0, z1 = 0;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int kv = kt * TILE + 32 * c;
            if (c % FL == 0) {
                const int64_t o = (int64_t)group_of(kv, a.v.gsv, a.v.groups) * a.v.mp + row0 + g;
                s0 = a.v.scales[o];
                s1 = a.v.scales[o + 8];
                z0 = zero_pair<T>(a.v.zeros[o]);
                z1 = zero_pair<T>(a.v.zeros[o + 8]);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) d[n][j] = 0.f;
            }
            const uint32_t f0[4] = {int_pair<T>(w0[c], 0, z0), int_pair<T>(w1[c], 0, z1), int_pair<T>(w0[c], 1, z0),
                                    int_pair<T>(w1[c], 1, z1)};
            const uint32_t f1[4] = {int_pair<T>(w0[c], 2, z0), int_pair<T>(w1[c], 2, z1), int_pair<T>(w0[c], 3, z0),
                                    int_pair<T>(w1[c], 3, z1)};
            const int k = kv + 8 * t;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int tok = n * 8 + g;
#pragma unroll
                for (int p = PIECES - 1; p >= 0; p--) {
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (tok < a.tokens && k < a.xcols)
                        b = __ldg(reinterpret_cast<const uint4*>(x + ((int64_t)p * a.tokens + tok) * a.ldx + k));
                    mma16816(d[n], f0, b.x, b.y, T());
                    mma16816(d[n], f1, b.z, b.w, T());
                }
            }
            if (c % FL == FL - 1) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    acc[n][0] = fmaf(s0, d[n][0], acc[n][0]);
                    acc[n][1] = fmaf(s0, d[n][1], acc[n][1]);
                    acc[n][2] = fmaf(s1, d[n][2], acc[n][2]);
                    acc[n][3] = fmaf(s1, d[n][3], acc[n][3]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float* r = red + (warp * 8 * NT + n * 8 + 2 * t) * 16 + g;  // [warp][token][row]
        r[0] = acc[n][0];
        r[16] = acc[n][1];
        r[8] = acc[n][2];
        r[24] = acc[n][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += blockDim.x) {
        const int64_t row = row0 + i % 16;
        const int tok = i / 16;
        if (row >= a.v.rows || tok >= a.tokens) continue;
        float s = 0.f;
        for (int w = 0; w < warps; w++) s += red[w * 8 * NT * 16 + i];
        if (a.bias) s += to_f<O>(reinterpret_cast<const O*>(a.bias)[row]);
        reinterpret_cast<O*>(a.y)[tok * a.ldy + row] = from_f<O>(s);
    }
}

// ---- joining partial sums, column sums ------------------------------------------------------------
// out[r][c] = sum over s of part[s][r][c] (in order) + bias[c], rounded once.
template <typename O>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int64_t rows, int64_t cols, const O* bias,
                                                  O* out, int64_t ldo) {
    const int64_t total = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < splits; p++) s += part[p * total + i];
        const int64_t c = i % cols;
        if (bias) s += to_f<O>(bias[c]);
        out[i / cols * ldo + c] = from_f<O>(s);
    }
}

// part[split][c] = sum of rows split * per .. of x[:, c]; a block holds 32 columns x 8 row lanes.
template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const T* x, int64_t rows, int64_t cols, int64_t ld, int64_t per, float* part) {
    __shared__ float sm[8][33];
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    const int64_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    float s = 0.f;
    if (c < cols)
        for (int64_t r = r0 + w; r < r1; r += 8) s += to_f<T>(x[r * ld + c]);
    sm[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; i++) s += sm[i][lane];
        part[blockIdx.y * cols + c] = s;
    }
}

int grid_n(const llmc_ctx* ctx, int64_t items) {
    const int64_t b = (items + 255) / 256, cap = (int64_t)ctx->sm_count * 16;
    return (int)(b < 1 ? 1 : (b > cap ? cap : b));
}

template <typename T, typename O, int NT, int PIECES>
void launch_few(const FewArgs& a, int warps, cudaStream_t st) {
    const unsigned grid = (unsigned)((a.v.rows + 15) / 16);
    const size_t sm = (size_t)warps * 16 * 8 * NT * sizeof(float);
    // granules per group sum: the largest of 4, 2, 1 that divides the group
    if (a.v.gsv % 128 == 0) few_kernel<T, O, NT, PIECES, 4><<<grid, warps * 32, sm, st>>>(a);
    else if (a.v.gsv % 64 == 0) few_kernel<T, O, NT, PIECES, 2><<<grid, warps * 32, sm, st>>>(a);
    else few_kernel<T, O, NT, PIECES, 1><<<grid, warps * 32, sm, st>>>(a);
}

}  // namespace

llmc_status int4_layout(llmc_ctx* ctx, cudaStream_t st, const uint8_t* codes, int64_t crow, const float* scales,
                        const int32_t* zps, int64_t srow, int sym, const w4::View& v, uint32_t* packed, float* sout,
                        uint8_t* zout, int32_t* exps) {
    LayoutArgs a{codes, crow, scales, zps, srow, sym, v, packed, sout, zout};
    layout_kernel<<<grid_n(ctx, v.mp * (v.kp / 8)), 256, 0, st>>>(a);
    LLMC_TRY(check_launch(ctx, "int4_layout"));
    exps_kernel<<<(unsigned)(v.mp / TILE + v.groups), 256, 0, st>>>(sout, v.mp, v.groups, exps);
    return check_launch(ctx, "int4_exps");
}

llmc_status int4_rows(llmc_ctx* ctx, cudaStream_t st, const w4::View& v, const void* ids, int ids64, int64_t tokens,
                      float scale, void* out, int dtype, int64_t ldo) {
    const int es = dtype_size(dtype);
    const int wide = (uintptr_t)out % 16 == 0 && (ldo * es) % 16 == 0;
    const int grid = grid_n(ctx, tokens * (v.kp / 8));
    int* flag = ctx->dflags + 4;
#define ROWS(T)                                                                                                      \
    do {                                                                                                             \
        if (ids64) rows_kernel<T, int64_t><<<grid, 256, 0, st>>>(v, (const int64_t*)ids, tokens, scale, (T*)out, ldo, wide, flag); \
        else rows_kernel<T, int32_t><<<grid, 256, 0, st>>>(v, (const int32_t*)ids, tokens, scale, (T*)out, ldo, wide, flag); \
    } while (0)
    if (dtype == LLMC_DTYPE_F32) ROWS(float);
    else if (dtype == LLMC_DTYPE_BF16) ROWS(__nv_bfloat16);
    else ROWS(__half);
#undef ROWS
    return check_launch(ctx, "int4_rows");
}

llmc_status int4_stage(llmc_ctx* ctx, cudaStream_t st, const void* x, int dtype, int64_t tokens, int64_t n, int64_t ldx,
                       int64_t pitch, const w4::View* v, int pieces, uint16_t* out) {
    const int gs = v ? v->gs : 0, gsv = v ? v->gsv : 0, groups = v ? v->groups : 0;
    const int grid = grid_n(ctx, tokens * (pitch / 8));
    if (dtype == LLMC_DTYPE_F32)
        stage_kernel<float><<<grid, 256, 0, st>>>((const float*)x, tokens, n, ldx, pitch, gs, gsv, groups, pieces, out);
    else if (dtype == LLMC_DTYPE_BF16)
        stage_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, tokens, n, ldx, pitch, gs, gsv, groups, pieces, out);
    else
        stage_kernel<__half><<<grid, 256, 0, st>>>((const __half*)x, tokens, n, ldx, pitch, gs, gsv, groups, pieces, out);
    return check_launch(ctx, "int4_stage");
}

llmc_status int4_few(llmc_ctx* ctx, cudaStream_t st, const w4::View& v, const void* x, int dtype, int64_t tokens, int64_t ldx,
                     int64_t xcols, const void* bias, void* y, int64_t ldy) {
    FewArgs a{v, x, ldx, xcols, (int)tokens, bias, y, ldy};
    const int ktiles = (int)(v.kp / TILE);
    const int warps = ktiles < 8 ? ktiles : 8;
    const bool two = tokens > 8;
    if (dtype == LLMC_DTYPE_F32) {
        if (two) launch_few<__nv_bfloat16, float, 2, 3>(a, warps, st);
        else launch_few<__nv_bfloat16, float, 1, 3>(a, warps, st);
    } else if (dtype == LLMC_DTYPE_BF16) {
        if (two) launch_few<__nv_bfloat16, __nv_bfloat16, 2, 1>(a, warps, st);
        else launch_few<__nv_bfloat16, __nv_bfloat16, 1, 1>(a, warps, st);
    } else {
        if (two) launch_few<__half, __half, 2, 1>(a, warps, st);
        else launch_few<__half, __half, 1, 1>(a, warps, st);
    }
    return check_launch(ctx, "int4_few");
}

llmc_status int4_join(llmc_ctx* ctx, cudaStream_t st, const float* part, int splits, int64_t rows, int64_t cols, const void* bias,
                      void* out, int dtype, int64_t ldo) {
    const int grid = grid_n(ctx, rows * cols);
    if (dtype == LLMC_DTYPE_F32)
        join_kernel<float><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const float*)bias, (float*)out, ldo);
    else if (dtype == LLMC_DTYPE_BF16)
        join_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const __nv_bfloat16*)bias, (__nv_bfloat16*)out, ldo);
    else
        join_kernel<__half><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const __half*)bias, (__half*)out, ldo);
    return check_launch(ctx, "int4_join");
}

llmc_status col_sum_parts(llmc_ctx* ctx, cudaStream_t st, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld,
                          int splits, float* part) {
    const dim3 grid((unsigned)((cols + 31) / 32), (unsigned)splits);
    const int64_t per = (rows + splits - 1) / splits;
    if (dtype == LLMC_DTYPE_F32) colsum_kernel<float><<<grid, 256, 0, st>>>((const float*)x, rows, cols, ld, per, part);
    else if (dtype == LLMC_DTYPE_BF16) colsum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, rows, cols, ld, per, part);
    else colsum_kernel<__half><<<grid, 256, 0, st>>>((const __half*)x, rows, cols, ld, per, part);
    return check_launch(ctx, "col_sum");
}

}  // namespace llmc
