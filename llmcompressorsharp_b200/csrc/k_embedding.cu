// Embedding lookup with a scale, and the gradient of the table.
//
//   y[t] = scale * table[ids[t]]            dtable[v] = scale * sum over t with ids[t] = v of dy[t]
//
// The reference's hooks start behind the embedding (GPTQModifier.cs:98-104 leaves the model's forward to the
// caller); the lookup is the first step of that forward, and its gradient completes the straight-through
// backward of FakeQuantize (FakeQuantizeFunction.cs:56-68) for a quantised table.
//
// The gradient adds each row's tokens in a fixed order, whatever ran when: the ids are sorted (stable), every
// row sums its own run in token order in fp32, and runs of more than RUN tokens are cut into pieces whose sums are
// added in order, or of more than 64 pieces every sixteenth in order and then those sixteen.
// No float atomics, so two calls give the same bits.
#include "ops.h"
#include "tc_common.cuh"

#include <atomic>

namespace llmc {
namespace {

using tc::cluster_ctarank;
using tc::cluster_sync;
using tc::mapa_shared;

// ---- 16 bytes of a row as floats -----------------------------------------------------------------
template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

template <typename T> __device__ __forceinline__ void unpack(uint4 u, float (&f)[Vec<T>::N]) {
    union { uint4 u; T h[Vec<T>::N]; } x;
    x.u = u;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) f[i] = to_f<T>(x.h[i]);
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&f)[Vec<T>::N], float scale) {
    union { uint4 u; T h[Vec<T>::N]; } x;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) x.h[i] = from_f<T>(__fmul_rn(f[i], scale));
    return x.u;
}

// ---- lookup ------------------------------------------------------------------------------------------
// L lanes per row, R rows at a time per lane group so that R loads are in flight; bound by memory.
template <typename T, typename I, int R>
__global__ void __launch_bounds__(256) lookup_kernel(const T* table, int64_t ldt, const I* ids, int64_t tokens, int64_t vocab,
                                                    int64_t hidden, int L, float scale, T* out, int64_t ldo, int wide, int* flag) {
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x % L;
    const int64_t group = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t t0 = group * R;
    int64_t row[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        row[r] = -1;
        if (t0 + r < tokens) {
            const int64_t id = (int64_t)ids[t0 + r];
            if (id >= 0 && id < vocab) row[r] = id;
            else if (lane == 0) atomicOr(flag, 1);
        }
    }
    if (wide) {
        const int nv = (int)(hidden / N);
        for (int j = lane; j < nv; j += L) {
            uint4 u[R];
#pragma unroll
            for (int r = 0; r < R; r++)
                u[r] = row[r] >= 0 ? __ldg(reinterpret_cast<const uint4*>(table + row[r] * ldt) + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (t0 + r >= tokens) continue;
                if (scale != 1.f) {  // a scale of one copies the bits
                    float f[N];
                    unpack<T>(u[r], f);
                    u[r] = pack<T>(f, scale);
                }
                __stcs(reinterpret_cast<uint4*>(out + (t0 + r) * ldo) + j, u[r]);
            }
        }
    } else {
        for (int64_t j = lane; j < hidden; j += L)
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (t0 + r >= tokens) continue;
                T v = row[r] >= 0 ? table[row[r] * ldt + j] : from_f<T>(0.f);
                if (scale != 1.f) v = from_f<T>(__fmul_rn(to_f<T>(v), scale));
                out[(t0 + r) * ldo + j] = v;
            }
    }
}

// ---- sorting the tokens -----------------------------------------------------------------------------
constexpr int SORT_WARPS = 32, SORT_NT = SORT_WARPS * 32;
constexpr int DIGIT = 9, BINS = 1 << DIGIT, BATCH = 8, MAX_CTAS = 16;
// Tokens that one row sums by itself; a longer run is cut into pieces of this many.  A piece costs a
// partial row in fp32 (an eighth of what its 32 bf16 rows cost to read, written and read again), a long
// run costs its serial sum.
constexpr int RUN = 32;

struct Plan {           // the workspace of one gradient call
    uint2 *pairs0, *pairs1;  // (token, id), sorted by id; the passes go from one to the other
    __host__ __device__ uint2* pairs(int i) const { return i & 1 ? pairs1 : pairs0; }
    int2* span;         // [vocab] first and one past the last sorted position, (0, 0) for an absent row
    int* counts;        // pieces, cut rows
    int2* pieces;       // first position, tokens
    int4* cut;          // row, first piece, pieces
    float* partial;     // [pieces][hidden]
};

int64_t max_pieces(int64_t tokens) { return 2 * (tokens / RUN) + 2; }

// One cluster sorts: stable passes of up to nine bits, each warp counting and placing its own stretch of
// tokens, the counts of a pass added up over the warps in shared memory and over the CTAs through it
// (hardware cluster barriers, no spinning).  One launch in place of three per pass.  Bound by the scattered stores,
// of which an SM does about one a clock, so token and id go out as one store of eight bytes and the cluster is as
// large as it may be.  Padding tokens and ids outside the table sort last, as `vocab`.
template <typename I>
__global__ void __launch_bounds__(SORT_NT) sort_kernel(const I* ids, uint32_t tokens, int64_t vocab, int64_t padding, int passes,
                                                      int bits, Plan p, int* flag) {
    extern __shared__ uint32_t hist[];                 // [SORT_WARPS][BINS]
    __shared__ uint32_t total[BINS], base[BINS], wsum[SORT_WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank(), ctas = gridDim.x;
    const uint32_t stretch = (tokens + ctas * SORT_WARPS * 32 - 1) / (ctas * SORT_WARPS * 32) * 32;
    const uint64_t w0 = (uint64_t)(rank * SORT_WARPS + warp) * stretch;
    const uint32_t first = (uint32_t)min((uint64_t)tokens, w0), last = (uint32_t)min((uint64_t)tokens, w0 + stretch);
    uint32_t* mine = hist + warp * BINS;
    const int bins = 1 << bits;

    for (int64_t v = rank * SORT_NT + threadIdx.x; v < vocab; v += ctas * SORT_NT) p.span[v] = make_int2(0, 0);
    if (rank == 0 && threadIdx.x < 2) p.counts[threadIdx.x] = 0;

    // Each warp takes its stretch in batches of BATCH x 32 tokens, whose keys it loads at once: one latency a batch
    // instead of one for each 32 tokens.  65,536 tokens take 22 us (60 with single loads, a cluster of eight and matches).
    uint2 pair[BATCH];  // token, id
    bool bad = false;
    auto load = [&](int pass, uint32_t i0) {
#pragma unroll
        for (int q = 0; q < BATCH; q++) {
            const uint32_t i = i0 + q * 32 + lane;
            pair[q] = make_uint2(i, 0);
            if (i >= last) continue;
            if (pass) {
                pair[q] = __ldcg(p.pairs(pass + 1) + i);
            } else {
                const int64_t id = (int64_t)ids[i];
                const bool out = id < 0 || id >= vocab;
                bad |= out;
                pair[q].y = out || id == padding ? (uint32_t)vocab : (uint32_t)id;
            }
        }
    };

    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * bits;
        for (int b = threadIdx.x; b < SORT_WARPS * BINS; b += SORT_NT) hist[b] = 0;
        __syncthreads();
        for (uint32_t i = first; i < last; i += 32 * BATCH) {
            load(pass, i);
#pragma unroll
            for (int q = 0; q < BATCH; q++) {
                if (i + q * 32 + lane < last) atomicAdd(&mine[(pair[q].y >> shift) & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        if ((int)threadIdx.x < bins) {  // exclusive over the warps
            uint32_t s = 0;
#pragma unroll
            for (int w0 = 0; w0 < SORT_WARPS; w0 += 8) {
                uint32_t c[8];
#pragma unroll
                for (int w = 0; w < 8; w++) c[w] = hist[(w0 + w) * BINS + threadIdx.x];
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    hist[(w0 + w) * BINS + threadIdx.x] = s;
                    s += c[w];
                }
            }
            total[threadIdx.x] = s;
        }
        cluster_sync();
        uint32_t before = 0, all = 0;
        if ((int)threadIdx.x < bins) {
            uint32_t n[MAX_CTAS];  // all under way before the first is used
#pragma unroll
            for (uint32_t c = 0; c < MAX_CTAS; c++) {
                n[c] = 0;
                if (c < ctas) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n[c]) : "r"(mapa_shared(tc::smem_u32(&total[threadIdx.x]), c)));
            }
#pragma unroll
            for (uint32_t c = 0; c < MAX_CTAS; c++) {
                if (c < rank) before += n[c];
                all += n[c];
            }
        }
        uint32_t inc = all;  // inclusive over the bins, by warp and then over the warps
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += n;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        if ((int)threadIdx.x < bins) {
            uint32_t s = inc - all + before;
            for (int w = 0; w < warp; w++) s += wsum[w];
            base[threadIdx.x] = s;
        }
        __syncthreads();
        for (uint32_t i = first; i < last; i += 32 * BATCH) {
            if (last - first > 32 * BATCH) load(pass, i);  // else the batch counted is the one to place
#pragma unroll
            for (int q = 0; q < BATCH; q++) {
                if (i + q * 32 >= last) break;
                // the lanes of the same digit, a vote to a bit (a match instruction took 40 clocks of the SM each)
                const bool in = i + q * 32 + lane < last;
                const uint32_t d = (pair[q].y >> shift) & (bins - 1);
                unsigned peers = __ballot_sync(0xffffffffu, in);
                for (int b = 0; b < bits; b++) {
                    const unsigned ones = __ballot_sync(0xffffffffu, d >> b & 1u);
                    peers &= d >> b & 1u ? ones : ~ones;
                }
                if (in) {
                    const uint32_t pos = base[d] + mine[d] + __popc(peers & ((1u << lane) - 1));
                    __stcg(p.pairs(pass) + pos, pair[q]);
                }
                __syncwarp();
                if (in && (peers & ((1u << lane) - 1)) == 0) mine[d] += __popc(peers);
                __syncwarp();
            }
        }
        __threadfence();
        cluster_sync();  // the other CTAs read what this one placed, and its totals are read no more
    }
    if (bad) atomicOr(flag, 1);
    const uint2* sorted = p.pairs(passes + 1);
    const auto key_at = [&](uint32_t i) { return __ldcg(&sorted[i].y); };
    const uint32_t hop = ctas * SORT_NT;
    for (uint32_t i0 = rank * SORT_NT + threadIdx.x; i0 < tokens; i0 += hop * BATCH) {
        uint32_t key[BATCH], prev[BATCH], next[BATCH], far[BATCH];
#pragma unroll
        for (int q = 0; q < BATCH; q++) {
            const uint32_t i = i0 + q * hop;
            key[q] = i < tokens ? key_at(i) : (uint32_t)vocab;
            prev[q] = i < tokens && i > 0 ? key_at(i - 1) : ~0u;
            next[q] = i + 1 < tokens ? key_at(i + 1) : ~0u;
            far[q] = i + RUN < tokens ? key_at(i + RUN) : ~0u;
        }
#pragma unroll
        for (int q = 0; q < BATCH; q++) {
            const uint32_t i = i0 + q * hop;
            if (key[q] >= (uint64_t)vocab) continue;
            if (next[q] != key[q]) __stcg(&p.span[key[q]].y, (int)i + 1);
            if (prev[q] == key[q]) continue;
            __stcg(&p.span[key[q]].x, (int)i);
            if (far[q] != key[q]) continue;
            // A run that is cut: its length by doubling and halving steps over the sorted keys.
            uint32_t lo = i + RUN, step = RUN;
            while (lo + step < tokens && key_at(lo + step) == key[q]) {
                lo += step;
                step *= 2;
            }
            for (; step > 0; step /= 2)
                if (lo + step < tokens && key_at(lo + step) == key[q]) lo += step;
            // Which slots a row gets is a race, but its pieces stand in order and are joined in order.
            const int n = (int)(lo + 1 - i), np = (n + RUN - 1) / RUN;
            const int at = atomicAdd(p.counts, np);
            for (int j = 0; j < np; j++) p.pieces[at + j] = make_int2((int)i + j * RUN, min(RUN, n - j * RUN));
            p.cut[atomicAdd(p.counts + 1, 1)] = make_int4((int)key[q], at, np, 0);
        }
    }
}

// ---- summing --------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void sum_run(const T* dy, int64_t ld, const uint2* idx, int n, int j, float (&acc)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    int i = 0;
    for (; i + 4 <= n; i += 4) {  // four rows in flight, added in token order
        uint4 u[4];
#pragma unroll
        for (int q = 0; q < 4; q++) u[q] = __ldcs(reinterpret_cast<const uint4*>(dy + (int64_t)idx[i + q].x * ld) + j);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float f[N];
            unpack<T>(u[q], f);
#pragma unroll
            for (int k = 0; k < N; k++) acc[k] = __fadd_rn(acc[k], f[k]);
        }
    }
    for (; i < n; i++) {
        float f[N];
        unpack<T>(__ldcs(reinterpret_cast<const uint4*>(dy + (int64_t)idx[i].x * ld) + j), f);
#pragma unroll
        for (int k = 0; k < N; k++) acc[k] = __fadd_rn(acc[k], f[k]);
    }
}

// The first `pblocks` blocks sum pieces, the others rows (L lanes per row): every row of the table is
// written once, zeros where no token looked it up.  Bound by memory: dy read once, the table written once.
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const T* dy, int64_t ld, const uint2* idx, Plan p, int64_t vocab,
                                                 int64_t hidden, int L, int pblocks, float scale, T* out, int wide) {
    constexpr int N = Vec<T>::N;
    if ((int)blockIdx.x < pblocks) {
        const int n = p.counts[0];
        for (int i = blockIdx.x; i < n; i += pblocks) {
            const int2 s = p.pieces[i];
            float* part = p.partial + (int64_t)i * hidden;
            if (wide) {
                for (int j = threadIdx.x; j < (int)(hidden / N); j += 256) {
                    float acc[N] = {};
                    sum_run<T>(dy, ld, idx + s.x, s.y, j, acc);
#pragma unroll
                    for (int k = 0; k < N; k += 4)
                        reinterpret_cast<float4*>(part + j * N)[k / 4] = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
                }
            } else {
                for (int64_t j = threadIdx.x; j < hidden; j += 256) {
                    float acc = 0.f;
                    for (int k = 0; k < s.y; k++) acc = __fadd_rn(acc, to_f<T>(dy[(int64_t)idx[s.x + k].x * ld + j]));
                    part[j] = acc;
                }
            }
        }
        return;
    }
    const int lane = threadIdx.x % L;
    const int64_t groups = (int64_t)(gridDim.x - pblocks) * (256 / L);
    for (int64_t v = (int64_t)(blockIdx.x - pblocks) * (256 / L) + threadIdx.x / L; v < vocab; v += groups) {
        const int2 s = p.span[v];
        const int n = s.y - s.x;
        if (n > RUN) continue;
        if (wide) {
            for (int j = lane; j < (int)(hidden / N); j += L) {
                float acc[N] = {};
                sum_run<T>(dy, ld, idx + s.x, n, j, acc);
                __stcs(reinterpret_cast<uint4*>(out + v * hidden) + j, pack<T>(acc, scale));
            }
        } else {
            for (int64_t j = lane; j < hidden; j += L) {
                float acc = 0.f;
                for (int k = 0; k < n; k++) acc = __fadd_rn(acc, to_f<T>(dy[(int64_t)idx[s.x + k].x * ld + j]));
                out[v * hidden + j] = from_f<T>(__fmul_rn(acc, scale));
            }
        }
    }
}

// Rows that were cut, 512 columns to an item.  A thread adds a column's pieces in order, or, where they are many,
// sixteen warps add every sixteenth piece of 32 columns at a time and then their sums.
template <typename T>
__global__ void __launch_bounds__(512) join_cut_kernel(Plan p, int64_t hidden, float scale, T* out) {
    __shared__ float sm[16][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t slabs = (hidden + 511) / 512, items = (int64_t)p.counts[1] * slabs;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int4 c = p.cut[i / slabs];
        const int64_t col0 = i % slabs * 512;
        const float* part = p.partial + (int64_t)c.y * hidden;
        T* row = out + (int64_t)c.x * hidden;
        if (c.z <= 64) {
            const int64_t col = col0 + threadIdx.x;
            float s = 0.f;
            if (col < hidden) {
#pragma unroll 8
                for (int k = 0; k < c.z; k++) s = __fadd_rn(s, part[k * hidden + col]);
                row[col] = from_f<T>(__fmul_rn(s, scale));
            }
            continue;
        }
        for (int64_t col = col0 + lane; col - lane < min(hidden, col0 + 512); col += 32) {
            float s = 0.f;
            if (col < hidden)
#pragma unroll 8
                for (int k = warp; k < c.z; k += 16) s = __fadd_rn(s, part[k * hidden + col]);
            sm[warp][lane] = s;
            __syncthreads();
            if (warp == 0 && col < hidden) {
#pragma unroll
                for (int w = 1; w < 16; w++) s = __fadd_rn(s, sm[w][lane]);
                row[col] = from_f<T>(__fmul_rn(s, scale));
            }
            __syncthreads();
        }
    }
}

// Lanes per row: of the powers of two from 8 to 256 the largest that leaves an eighth of its lanes' turns idle at most,
// or the one that leaves the fewest (144 vectors: 32 lanes in 5 turns, not 256 in one).
int lanes_for(int64_t vectors) {
    int best = 8;
    int64_t least = -1;
    for (int L = 256; L >= 8; L /= 2) {
        const int64_t turns = (vectors + L - 1) / L * L;
        if (8 * (turns - vectors) <= vectors) return L;
        if (least < 0 || turns < least) {
            least = turns;
            best = L;
        }
    }
    return best;
}

template <typename T, typename I>
llmc_status lookup(llmc_ctx* ctx, cudaStream_t st, const void* table, int64_t ldt, const void* ids, int64_t tokens, int64_t vocab,
                   int64_t hidden, float scale, void* out, int64_t ldo) {
    constexpr int N = Vec<T>::N;
    const int wide = hidden % N == 0 && ldt % N == 0 && ldo % N == 0 && ((uintptr_t)table | (uintptr_t)out) % 16 == 0;
    const int L = lanes_for(wide ? hidden / N : hidden);
    const int per = 256 / L;
    int* flag = ctx->dflags + 4;
    // four rows per lane group once that still leaves every SM a few blocks
    if (tokens / (4 * per) >= 4 * (int64_t)ctx->sm_count) {
        const unsigned grid = (unsigned)((tokens + 4 * per - 1) / (4 * per));
        lookup_kernel<T, I, 4><<<grid, 256, 0, st>>>((const T*)table, ldt, (const I*)ids, tokens, vocab, hidden, L, scale, (T*)out, ldo, wide, flag);
    } else {
        const unsigned grid = (unsigned)((tokens + per - 1) / per);
        lookup_kernel<T, I, 1><<<grid, 256, 0, st>>>((const T*)table, ldt, (const I*)ids, tokens, vocab, hidden, L, scale, (T*)out, ldo, wide, flag);
    }
    return check_launch(ctx, "embedding");
}

// Readies the sort on a device, once, and gives its largest cluster: sixteen where the device places such a cluster, else
// the portable eight.
llmc_status ready_sort(int device, int ids64, const void* fn, size_t sm, int& n) {
    static std::atomic<int> known[2][64];
    const bool keep = device >= 0 && device < 64;
    n = keep ? known[ids64 ? 1 : 0][device].load(std::memory_order_relaxed) : 0;
    if (n) return LLMC_OK;
    LLMC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    LLMC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(SORT_NT);
    cfg.dynamicSmemBytes = sm;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 16;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int clusters = 0;
    const bool ok = cudaOccupancyMaxActiveClusters(&clusters, fn, &cfg) == cudaSuccess && clusters > 0;
    if (!ok) cudaGetLastError();
    n = ok ? 16 : 8;
    if (keep) known[ids64 ? 1 : 0][device].store(n, std::memory_order_relaxed);
    return LLMC_OK;
}

size_t carve(Plan& p, void* ws, int64_t tokens, int64_t vocab, int64_t hidden) {
    Carver c{(char*)ws};
    p.pairs0 = c.take<uint2>(tokens);
    p.pairs1 = c.take<uint2>(tokens);
    p.span = c.take<int2>(vocab);
    p.counts = c.take<int>(2);
    p.pieces = c.take<int2>(max_pieces(tokens));
    p.cut = c.take<int4>(max_pieces(tokens));
    p.partial = c.take<float>(max_pieces(tokens) * hidden);
    return c.off;
}

template <typename T>
llmc_status sums(llmc_ctx* ctx, cudaStream_t st, const void* dy, int64_t ld, int passes, const Plan& p, int64_t tokens,
                 int64_t vocab, int64_t hidden, float scale, void* out) {
    constexpr int N = Vec<T>::N;
    const int wide = hidden % N == 0 && ld % N == 0 && ((uintptr_t)dy | (uintptr_t)out) % 16 == 0;
    const int L = lanes_for(wide ? hidden / N : hidden);
    const int64_t per = 256 / L;
    const int64_t cap = (int64_t)ctx->sm_count * 8;
    const int64_t rows = (vocab + per - 1) / per;
    const int64_t most = max_pieces(tokens);
    const int pblocks = tokens > RUN ? (int)(most < cap ? most : cap) : 0;
    const uint2* idx = p.pairs(passes + 1);
    sum_kernel<T><<<(unsigned)(pblocks + (rows < 4 * cap ? rows : 4 * cap)), 256, 0, st>>>((const T*)dy, ld, idx, p, vocab, hidden, L, pblocks,
                                                                                  scale, (T*)out, wide);
    LLMC_TRY(check_launch(ctx, "embedding_grad_sum"));
    if (!pblocks) return LLMC_OK;
    join_cut_kernel<T><<<2 * ctx->sm_count, 512, 0, st>>>(p, hidden, scale, (T*)out);
    return check_launch(ctx, "embedding_grad_join");
}

}  // namespace

llmc_status embedding_lookup(llmc_ctx* ctx, cudaStream_t st, const void* ids, int ids64, int64_t tokens, const void* table, int dtype,
                             int64_t vocab, int64_t hidden, int64_t ldt, float scale, void* out, int64_t ldo) {
#define LOOKUP(T)                                                                                                            \
    return ids64 ? lookup<T, int64_t>(ctx, st, table, ldt, ids, tokens, vocab, hidden, scale, out, ldo)                     \
                 : lookup<T, int32_t>(ctx, st, table, ldt, ids, tokens, vocab, hidden, scale, out, ldo)
    if (dtype == LLMC_DTYPE_F32) LOOKUP(float);
    if (dtype == LLMC_DTYPE_BF16) LOOKUP(__nv_bfloat16);
    LOOKUP(__half);
#undef LOOKUP
}

size_t embedding_grad_bytes(int64_t tokens, int64_t vocab, int64_t hidden) {
    Plan p;
    return carve(p, nullptr, tokens, vocab, hidden);
}

llmc_status embedding_grad(llmc_ctx* ctx, cudaStream_t st, const void* ids, int ids64, int64_t tokens, const void* dy, int dtype,
                           int64_t lddy, int64_t vocab, int64_t hidden, float scale, int64_t padding, void* out, void* ws) {
    Plan p;
    carve(p, ws, tokens, vocab, hidden);
    int width = 1;
    while ((1ll << width) <= vocab) width++;
    const int passes = (width + DIGIT - 1) / DIGIT, bits = (width + passes - 1) / passes;
    const size_t sm = (size_t)SORT_WARPS * BINS * sizeof(uint32_t);
    const void* fn = ids64 ? (const void*)sort_kernel<int64_t> : (const void*)sort_kernel<int32_t>;
    int most = 0;
    LLMC_TRY(ready_sort(ctx->device, ids64, fn, sm, most));
    int ctas = 1;  // about 2,048 tokens to a CTA
    while (ctas < most && (int64_t)ctas * 2048 < tokens) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(SORT_NT);
    cfg.dynamicSmemBytes = sm;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (ids64)
        LLMC_CUDA_TRY(cudaLaunchKernelEx(&cfg, sort_kernel<int64_t>, (const int64_t*)ids, (uint32_t)tokens, vocab, padding, passes, bits, p,
                                         ctx->dflags + 4));
    else
        LLMC_CUDA_TRY(cudaLaunchKernelEx(&cfg, sort_kernel<int32_t>, (const int32_t*)ids, (uint32_t)tokens, vocab, padding, passes, bits, p,
                                         ctx->dflags + 4));
    LLMC_TRY(check_launch(ctx, "embedding_grad_sort"));
    if (dtype == LLMC_DTYPE_F32) return sums<float>(ctx, st, dy, lddy, passes, p, tokens, vocab, hidden, scale, out);
    if (dtype == LLMC_DTYPE_BF16) return sums<__nv_bfloat16>(ctx, st, dy, lddy, passes, p, tokens, vocab, hidden, scale, out);
    return sums<__half>(ctx, st, dy, lddy, passes, p, tokens, vocab, hidden, scale, out);
}

}  // namespace llmc
