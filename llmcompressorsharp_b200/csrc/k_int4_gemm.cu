// Products of many rows with a packed 4-bit weight on the 5th-generation tensor cores:
//
//   forward   y[t][n]  = sum_k x[t][k] W[n][k] + b[n]
//   gradient  dx[t][k] = sum_n dy[t][n] W[n][k]
//
// The activations (A, K-major) come by TMA; the weight (B) is dequantised by eight warps straight into the
// shared memory the MMA reads: K-major for the forward product (rows n, 128 columns k to a stage), MN-major for
// the gradient (rows n are the contraction, 128 columns k to a CTA), so one copy of the codes serves both and
// no 16-bit weight is ever written to memory.
//
// W in 16 bits.  (u - z) s is rounded once to the activations' type (2^-8 relative at most in bf16, 2^-11 in fp16): the
// scale goes in as a sum of two 16-bit numbers, fma(v, s_hi, v s_lo), v an exact integer.  That is the weight
// that the quantisers themselves hand back in a model of that type (FakeQuantizeFunction.cs:39-44 rounds its
// last product to the tensor's type), and it lets a product run over any group size without leaving TMEM.  In
// fp16 the scales are first brought near one by a power of two per row (forward) or per group over all rows (gradient)
// that the epilogue takes back in fp32, so scales of any size keep their bits, and ratios do as far as fp16 goes: beside
// the largest scale s of its row (its group's column) a scale counts to 2^-24 s, so that its weights have 2^-11 down to
// about 2^-13 s and lose a bit for each power of two below.
//
// fp32 activations come as three bf16 pieces that add up to them exactly (rounded to nearest, so the second and third
// are 2^-8 and 2^-17 of the leading power at most); W is split after its product in fp32 by truncation (2^-7, 2^-15).  Six
// piece products are added, small ones first; the three left out are x1 w2 and x2 w1, 2^-23 and 2^-24, and less, so a
// term is off by 2^-22.4 of itself at most, with either sign (of 4 million, 2^-22.6; 2^-21.2 and always towards zero with x
// truncated, too).  Tensor-core fp32
// accumulation truncates, so TMEM then holds 256 terms of the contraction at most before the epilogue adds them
// to fp32 registers.
//
// A persistent grid of CTA pairs (256 tokens x 256 columns, cta_group::2) or, for products that a round of them holds and
// for fp32, single CTAs (128 x 128).  Per CTA: a TMA warp for the activations and one for the codes (a tile of 128 x 128
// weights in one bulk copy), an MMA warp, epilogue warps, eight dequantising warps, a ring of
// STAGES x (32 KB activations + 32 KB weights) and one of CODE_STAGES tiles of codes, two accumulators in TMEM.
// A stage is a whole tile, 128 of the contraction: the MMA warp's two waits and its commit take some hundreds of
// clocks, which the MMAs of 64 (512 clocks) did not cover.
//
// 4096 -> 14336, 8,192 tokens, bf16: 735 to 775 us in short runs (1.25 to 1.3 PFLOP/s; the library's product of a 16-bit weight 648),
// 860 back to back at the power limit (731); 813 in short runs with one thread issuing the MMAs inside a branch and
// building its descriptors each time.  2,048 tokens of 4096 -> 4096: 68 us back to back (53), its gradient 66.  At 33 to 128
// tokens the eight warps that dequantise bound it: 29 us for 4096 -> 14336, where the codes alone are read in 5.  Numbers
// made before the wait for a free stage instead of behind it: no faster.  fp32, 2,048 tokens of 4096 -> 4096: 937 us, its
// gradient 905 (0.31 of the rate of six bf16 products).
// Every wait is bounded.
//
// What orders the rings, each turn of a slot by one phase of its barriers:
//   activations  afull: the copies' bytes complete the phase that the MMA warp waits for; empty: the MMAs that read the
//                stage complete before the commit's arrival, which the copying thread waits for.
//   weights      bfull: each dequantising lane fences its stores for the async proxy, the warp syncs, one lane arrives;
//                a pair's arrival at the leader's barrier stands for shared memory that the arriving SM's half of the
//                MMA reads.  empty: as above, waited for before the stores.
//   codes        cfull: the copy's bytes; cempty: all eight warps arrive, the two groups alike, those that read after the
//                stores made of what they read.  A slot has no new phase before all have seen the last one.
//   accumulators tfull: the commit after a fold's last MMA; tempty: each epilogue warp's loads are waited for in the
//                statement that makes them, and fenced, before its arrival.
#include "int4.cuh"
#include "ops.h"
#include "tc_common.cuh"

#include <cuda.h>

#include <mutex>

namespace llmc {
namespace {

using namespace tc;
using namespace w4;

constexpr int BOX = 64;                       // columns of a TMA box: 128 bytes, the swizzle's width
constexpr int BOX_BYTES = 128 * BOX * 2;
constexpr int STAGES = 2, A_BYTES = 2 * BOX_BYTES, B_BYTES = 2 * BOX_BYTES, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int CODE_STAGES = 4, CODE_BYTES = (TILE / ROWS) * (1024 + 80 * MAX_NG);  // tiles of codes
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + CODE_STAGES * CODE_BYTES + 1024 + 256;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a CTA");
constexpr int DQ_WARPS = 8;
constexpr int FOLD = 2;  // tiles of the contraction between folds (fp32)

struct GemmInt4 {
    View v;
    int64_t tokens;
    int64_t ocols;           // columns of the output
    int tiles_m, tiles_n, splits, kt_total, kt_per, group_m;  // kt: tiles of 128 of the contraction, one stage each
    int64_t piece_rows;      // rows between the pieces of the activations' map
    const void* bias;
    void* out;
    int64_t ldo;
    float* part;             // [splits][tokens][ocols] when splits > 1
    int wide;
    int* err;
    uint32_t wait_limit;
    uint32_t idesc;
};

struct Unit {
    int64_t m0, n0;  // first token and column of the tile
    int kt0, kt1, split;
};

template <int CG> __device__ __forceinline__ Unit unit_at(const GemmInt4& a, int u) {
    const int tiles = a.tiles_m * a.tiles_n;
    const int t = u % tiles;
    Unit r;
    r.split = u / tiles;
    // group_m token tiles wide strips, so that the tiles in flight share both operands through L2
    const int per = a.group_m * a.tiles_n, g = t / per, first = g * a.group_m, gm = min(a.group_m, a.tiles_m - first), l = t - g * per;
    r.m0 = (int64_t)(first + l % gm) * (128 * CG);
    r.n0 = (int64_t)(l / gm) * (128 * CG);
    r.kt0 = r.split * a.kt_per;
    r.kt1 = min(a.kt_total, r.kt0 + a.kt_per);
    return r;
}

// The six products of pieces, small ones first: x piece (3: the first without infinities and NaN), w piece.
constexpr int COMBOS = 6;
__device__ __forceinline__ void combo(int c, int& xp, int& wp) {
    xp = c == 0 ? 2 : (c == 2 || c == 3) ? 1 : c == 5 ? 0 : 3;
    wp = c == 1 ? 2 : (c == 2 || c == 4) ? 1 : 0;
}

// Two groups of four dequantising warps take the tiles in turn, so that one converts while the other waits, fences or
// signals; a warp has two records of a tile, four rows' chunks (sixteen words) to a thread.
// Lanes 4 i .. 4 i + 3 hold the chunks of one row, in the order of rows below: an 8-lane phase then meets
// rows of different parity, so that its 16-byte loads (rows 64 bytes apart) touch every bank once, and of
// different bit 2, so that its stores into the 128-byte swizzle do.
__device__ __forceinline__ int row_of(int lane) { return (0x36271450 >> (lane / 4 * 4)) & 7; }

// Reads of a tile of codes, which a bulk copy fills again once it is let go of.  Volatile: an ordinary load may be done
// later, or again, instead of keeping its value, and the fp32 kernels are short of registers.  With ordinary loads and the
// tile let go of right after them, fp32 gradients on two streams at once (32 of 80) had codes of a later tile in them; with
// these and the same order none of 48,000 products of any type did.
__device__ __forceinline__ uint4 read_codes(uint32_t addr) {
    uint4 v;
    asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float read_scale(uint32_t addr) {
    float v;
    asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t read_zero(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.volatile.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// A scale and zero ready for eight weights at a time.
template <typename T, int PIECES> struct Scale {
    typename Num<T>::T2 hi, lo;  // PIECES == 1
    float s;
    uint32_t zz;
    __device__ __forceinline__ void set(float scale, uint32_t z) {
        zz = zero_pair<T>(z);
        s = scale;
        if constexpr (PIECES == 1) {
            hi.x = hi.y = from_f<T>(scale);
            lo.x = lo.y = from_f<T>(__fsub_rn(scale, to_f<T>(hi.x)));
        }
    }
};

// Eight weights of a word in T: rounded once, or piece wp of their fp32 value (truncated, eight bits each, so the three
// add up to it).
template <typename T, int PIECES>
__device__ __forceinline__ uint4 dequant(uint32_t word, const Scale<T, PIECES>& sc, Bits bits, int wp) {
    uint32_t o[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const uint32_t v = int_pair<T>(word, p, sc.zz, bits);
        if constexpr (PIECES == 1) {
            o[p] = bits2(__hfma2(as2<T>(v), sc.hi, __hmul2(as2<T>(v), sc.lo)));
        } else {
            float w0 = __fmul_rn(__uint_as_float(v << 16), sc.s), w1 = __fmul_rn(__uint_as_float(v & 0xFFFF0000u), sc.s);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                if (q >= wp) continue;
                w0 = __fsub_rn(w0, __uint_as_float(__float_as_uint(w0) & 0xFFFF0000u));
                w1 = __fsub_rn(w1, __uint_as_float(__float_as_uint(w1) & 0xFFFF0000u));
            }
            o[p] = __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x7632);
        }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// T: operand type; O: output (and bias) type; DIR 0 forward, 1 gradient; CG CTAs per tile; PIECES 1, or 3 for fp32; ONE
// group to a tile's columns (whose scales a thread then keeps once), or up to four.
template <typename T, typename O, int DIR, int CG, int PIECES, bool ONE>
__global__ void __launch_bounds__(32 * (3 + (PIECES == 3 ? 8 : 4) + DQ_WARPS), 1)
    gemm_int4_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ GemmInt4 a) {
    constexpr bool FOLDS = PIECES == 3;
    constexpr int EW = FOLDS ? 8 : 4;          // epilogue warps
    constexpr int BN = 128 * CG;              // columns of a tile
    constexpr int TMEM_COLS = 2 * BN;
    constexpr int EC = BN * 4 / EW;           // columns per epilogue warp
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* codes = smem + STAGES * STAGE_BYTES;
    uint64_t* afull = reinterpret_cast<uint64_t*>(codes + CODE_STAGES * CODE_BYTES);
    uint64_t* bfull = afull + STAGES;
    uint64_t* empty = bfull + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* cfull = tempty + 2;
    uint64_t* cempty = cfull + CODE_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cempty + CODE_STAGES);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint2* slot = reinterpret_cast<uint2*>(tmem_slot + 2);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&afull[s], 1);
            mbar_init(&bfull[s], DQ_WARPS / 2 * CG);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], EW * CG);
        }
        for (int s = 0; s < CODE_STAGES; s++) {
            mbar_init(&cfull[s], 1);
            mbar_init(&cempty[s], DQ_WARPS);
        }
        *abort_flag = 0;
        put_bits<T>(slot);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int units = a.tiles_m * a.tiles_n * a.splits;
    uint32_t it = 0, ct = 0, cc = 0;  // stages, tiles of codes and accumulators used so far, counted alike by every role
    int commit_par[2] = {-1, -1};

    // Calls body(kt, xp, wp, first, last) for each tile of a unit's contraction in ring order (one stage each): first /
    // last mark the tiles that open and close an accumulator.  body returns false to stop.
    auto tiles = [&](const Unit& u, auto&& body) -> bool {
        if constexpr (!FOLDS) {
            for (int kt = u.kt0; kt < u.kt1; kt++)
                if (!body(kt, 0, 0, kt == u.kt0, kt == u.kt1 - 1)) return false;
        } else {
            for (int c0 = u.kt0; c0 < u.kt1; c0 += FOLD) {
                const int c1 = min(u.kt1, c0 + FOLD);
                for (int c = 0; c < COMBOS; c++) {
                    int xp, wp;
                    combo(c, xp, wp);
                    for (int kt = c0; kt < c1; kt++)
                        if (!body(kt, xp, wp, c == 0 && kt == c0, c == COMBOS - 1 && kt == c1 - 1)) return false;
                }
            }
        }
        return true;
    };

    if (warp == 0) {
        if (lane == 0) {
            // ---- TMA: this CTA's 128 tokens
            for (int un = worker; un < units && !*abort_flag; un += workers) {
                const Unit u = unit_at<CG>(a, un);
                const int row = (int)(u.m0 + rank * 128);
                const bool ok = tiles(u, [&](int kt, int xp, int, bool, bool) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&empty[s], ((it / STAGES) & 1u) ^ 1u, abort_flag, a.err, a.wait_limit)) return false;
                    unsigned char* dst = smem + s * STAGE_BYTES;
                    const int x = kt * TILE, y = row + (int)(xp * a.piece_rows);
                    if constexpr (CG == 2) {
                        if (rank == 0) mbar_expect_tx(&afull[s], 2 * A_BYTES);
                        const uint32_t bar = mapa_shared(smem_u32(&afull[s]), 0);
                        tma_load_2d_pair(dst, &amap, x, y, bar);
                        tma_load_2d_pair(dst + BOX_BYTES, &amap, x + BOX, y, bar);
                    } else {
                        mbar_expect_tx(&afull[s], A_BYTES);
                        tma_load_2d(dst, &amap, x, y, &afull[s]);
                        tma_load_2d(dst + BOX_BYTES, &amap, x + BOX, y, &afull[s]);
                    }
                    it++;
                    return true;
                });
                if (!ok) break;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- MMA, issued by one lane of the converged warp; what is computed between two is time between two, so the
            // descriptors are built once: a stage's and a step's differ from them in the address's low word only.
            const uint32_t base = smem_u32(smem);
            const uint64_t desc_a = smem_desc_k_sw128(base);
            const uint64_t desc_b = DIR == 0 ? smem_desc_k_sw128(base + A_BYTES) : smem_desc_mn_sw128(base + A_BYTES, BOX_BYTES);
            const auto desc_at = [](uint64_t d, uint32_t off) { return (d & 0xFFFFFFFF00000000ull) | ((uint32_t)d + off); };
            const auto ready = [&](uint64_t* bar, uint32_t parity) {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.err, a.wait_limit)) != 0;
            };
            for (int un = worker; un < units; un += workers) {
                const Unit u = unit_at<CG>(a, un);
                bool open = false;
                const bool ok = tiles(u, [&](int, int, int, bool first, bool last) {
                    const int b = (int)(cc & 1u);
                    if (first) {
                        if (!ready(&tempty[b], ((cc >> 1) & 1u) ^ 1u)) return false;
                        tc_fence_after();
                        open = true;
                    }
                    const int s = it % STAGES;
                    const uint32_t ph = (it / STAGES) & 1u;
                    if (!ready(&afull[s], ph) || !ready(&bfull[s], ph)) return false;
                    tc_fence_after();
                    const uint32_t dst = tmem + (uint32_t)(b * BN);
                    const uint32_t at = (uint32_t)(s * (STAGE_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < TILE / 16; kk++) {
                        const uint32_t k = (kk / 4 * BOX_BYTES + kk % 4 * 32) >> 4;  // K-major: 16 columns are 32 bytes of a box
                        const uint64_t da = desc_at(desc_a, at + k), db = desc_at(desc_b, at + (DIR == 0 ? k : kk * (2048 >> 4)));
                        umma_f16_warp<CG>(dst, da, db, a.idesc, first && kk == 0 ? 0u : 1u);
                    }
                    umma_commit_warp<CG>(&empty[s]);
                    it++;
                    if (last) {
                        umma_commit_warp<CG>(&tfull[b]);
                        commit_par[b] = (int)((cc >> 1) & 1u);
                        open = false;
                        cc++;
                    }
                    return true;
                });
                if (!ok) {
                    if (open) {  // so that the tail can wait for what was issued
                        umma_commit_warp<CG>(&tfull[cc & 1u]);
                        commit_par[cc & 1u] = (int)((cc >> 1) & 1u);
                    }
                    break;
                }
            }
        }
        __syncwarp();
    } else if (warp < 2 + EW) {
        // ---- epilogue: TMEM lane quadrant q, columns h EC ..
        const int q = warp % 4, h = (warp - 2) / 4;
        float acc[FOLDS ? EC : 1];
        for (int un = worker; un < units && !*abort_flag; un += workers) {
            const Unit u = unit_at<CG>(a, un);
            const int64_t tok = u.m0 + rank * 128 + q * 32 + lane;
            // Columns n0 + c0 .. + 31 of this warp's 32 tokens, one token to a thread.
            auto emit = [&](float (&v)[32], int c0) {
                constexpr bool HALF = Num<T>::MAGIC == Num<__half>::MAGIC;
                const int64_t col0 = u.n0 + c0;
                const bool part = a.splits > 1, mapped = DIR == 1 && !a.v.identity;
                if (!HALF && !mapped && !a.bias && (part ? a.ocols % 4 == 0 : a.wide) && col0 + 32 <= a.ocols) {
                    // 16 bytes at a time along the thread's own row
                    if (tok >= a.tokens) return;
                    if (part) {
                        float* row = a.part + ((int64_t)u.split * a.tokens + tok) * a.ocols + col0;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(row + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    } else {
                        constexpr int N = 16 / (int)sizeof(O);
                        O* row = reinterpret_cast<O*>(a.out) + tok * a.ldo + col0;
#pragma unroll
                        for (int i = 0; i < 32; i += N) {
                            union { O h[N]; uint4 u4; } x;
#pragma unroll
                            for (int j = 0; j < N; j++) x.h[j] = from_f<O>(v[i + j]);
                            *reinterpret_cast<uint4*>(row + i) = x.u4;
                        }
                    }
                    return;
                }
                // Otherwise the block is transposed in registers, so that a thread has one column (its bias, its exponent,
                // where it goes) and a store is 32 neighbours of a row; element by element along rows, a product with
                // an odd number of columns spent 27 us of 36 in its stores.
#pragma unroll
                for (int s = 16; s > 0; s >>= 1)
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        if (i & s) continue;
                        const bool hi = lane & s;
                        const float y = __shfl_xor_sync(0xffffffffu, hi ? v[i] : v[i | s], s);
                        if (hi) v[i] = y;
                        else v[i | s] = y;
                    }
                int64_t col = col0 + lane;
                float f = 1.f;
                if (HALF) {
                    if (DIR == 0) f = col < a.v.rows ? pow2(__ldg(a.v.exps + col)) : 1.f;
                    else f = col < a.v.kp ? pow2(__ldg(a.v.exps + a.v.mp + col / TILE * a.v.ng + slot_of((int)(col % TILE) / 32, a.v.ng))) : 1.f;
                }
                if (mapped) col = col < a.v.kp ? column_of((int)col, a.v.gs, a.v.gsv, a.v.groups, a.v.cols) : -1;
                if (col < 0 || col >= a.ocols) return;
                const float bias = a.bias ? to_f<O>(reinterpret_cast<const O*>(a.bias)[col]) : 0.f;
                const int64_t tok0 = tok - lane;
                const int n = (int)min((int64_t)32, a.tokens - tok0);
                float* pcol = a.part + ((int64_t)u.split * a.tokens + tok0) * a.ocols + col;
                O* ocol = reinterpret_cast<O*>(a.out) + tok0 * a.ldo + col;
#pragma unroll
                for (int r = 0; r < 32; r++) {
                    if (r >= n) break;
                    if (part) pcol[r * a.ocols] = v[r] * f;
                    else ocol[r * a.ldo] = from_f<O>(fmaf(v[r], f, bias));
                }
            };
            const int chunks = FOLDS ? (u.kt1 - u.kt0 + FOLD - 1) / FOLD : 1;
            if constexpr (FOLDS) {
#pragma unroll
                for (int i = 0; i < EC; i++) acc[i] = 0.f;
            }
            bool ok = true;
            for (int c = 0; c < chunks; c++, cc++) {
                const int b = (int)(cc & 1u);
                const bool have = mbar_wait(&tfull[b], (cc >> 1) & 1u, abort_flag, a.err, a.wait_limit);
                if (!__all_sync(0xffffffffu, have ? 1 : 0)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN + h * EC);
#pragma unroll
                for (int p = 0; p < EC / 32; p++) {
                    uint32_t r[32];
                    tmem_ld32(taddr + p * 32, r);
                    if constexpr (FOLDS) {
#pragma unroll
                        for (int i = 0; i < 32; i++) acc[p * 32 + i] = __fadd_rn(acc[p * 32 + i], __uint_as_float(r[i]));
                    } else {
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
                        emit(v, h * EC + p * 32);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) mbar_arrive_cluster_cta(mapa_shared(smem_u32(&tempty[b]), 0));
                    else mbar_arrive(&tempty[b]);
                }
            }
            if (!ok) break;
            if constexpr (FOLDS) {
#pragma unroll
                for (int p = 0; p < EC / 32; p++) {
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = acc[p * 32 + i];
                    emit(v, h * EC + p * 32);
                }
            }
        }
    } else if (warp < 2 + EW + DQ_WARPS) {
        // ---- dequantising
        const int grp = (warp - 2 - EW) / 4, w = (warp - 2 - EW) % 4, ng = ONE ? 1 : a.v.ng, t = lane & 3, r8 = row_of(lane);
        const int64_t lim = (DIR == 0 ? a.v.mp : a.v.kp) - 128;
        constexpr int GROUPS = ONE ? 1 : 4;
        const Bits bits = get_bits(slot);
        for (int un = worker; un < units && !*abort_flag; un += workers) {
            const Unit u = unit_at<CG>(a, un);
            // the last tile of a pair may reach past the padded weight: its columns are never stored
            const int64_t nl = min(u.n0 + (int64_t)rank * 128, lim);
            float e[4] = {1.f, 1.f, 1.f, 1.f};  // fp16: 2^-exponent of this thread's rows, or of the groups
            if constexpr (Num<T>::MAGIC == Num<__half>::MAGIC) {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    e[c] = pow2(-(DIR == 0 ? a.v.exps[nl + 32 * w + 8 * c + r8] : a.v.exps[a.v.mp + nl / TILE * ng + slot_of(c, ng)]));
            }
            const bool ok = tiles(u, [&](int, int, int wp, bool, bool) {
                const int cs = ct % CODE_STAGES;
                // The other group's tiles are waited for as well: copies may land out of order, and a stage of this ring
                // changes hands every turn, so that a group that skipped one could take its old phase for the new one; and
                // both let go of each, so that none is filled again before both have seen it full.
                if (!mbar_wait(&cfull[cs], (ct / CODE_STAGES) & 1u, abort_flag, a.err, a.wait_limit)) return false;
                ct++;
                const int sg = it % STAGES;
                const uint32_t ph = (it / STAGES) & 1u;
                if ((it++ & 1u) != (uint32_t)grp) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&cempty[cs]);
                    return true;
                }
                const uint32_t tile = smem_u32(codes) + cs * CODE_BYTES;
                uint4 q[4];
                Scale<T, PIECES> sc[4][GROUPS];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t rec = tile + (2 * w + i / 2) * a.v.rec;
                    const int in = 8 * (i & 1) + r8;
                    q[i] = read_codes(rec + in * 64 + t * 16);
                    const uint32_t scales = rec + 1024 + 4 * in * ng, zeros = rec + 1024 + 64 * ng + in * ng;
#pragma unroll
                    for (int c = 0; c < GROUPS; c++)
                        sc[i][c].set(read_scale(scales + 4 * slot_of(c, ng)) * e[DIR == 0 ? i : c], read_zero(zeros + slot_of(c, ng)));
                }
                if (!mbar_wait(&empty[sg], ph ^ 1u, abort_flag, a.err, a.wait_limit)) return false;
                unsigned char* b = smem + sg * STAGE_BYTES + A_BYTES;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t word[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        // K-major and MN-major alike: a box holds 64 layout columns of 128 rows, rows of 128 bytes
                        const int off = c / 2 * BOX_BYTES + (32 * w + 8 * i + r8) * 128 + (((4 * (c & 1) + t) ^ r8) << 4);
                        *reinterpret_cast<uint4*>(b + off) = dequant<T, PIECES>(word[c], sc[i][ONE ? 0 : c], bits, wp);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                // To the leader's barrier without a cluster-wide fence (with one the product took 1.6 times as long):
                // what the arrival stands for is in this SM's own shared memory, complete for the async proxy by the
                // fence above, and it is this SM's half of the MMA that reads it.
                if (lane == 0) {
                    if constexpr (CG == 2) mbar_arrive_cluster_cta(mapa_shared(smem_u32(&bfull[sg]), 0));
                    else mbar_arrive(&bfull[sg]);
                    // The tile of codes is let go of when what was read of it has gone into the stores above, so that its
                    // reads come first by their data, too (no slower than right after them).
                    mbar_arrive(&cempty[cs]);
                }
                return true;
            });
            if (!ok) break;
        }
    } else if (lane == 0) {
        // ---- TMA: tiles of codes
        const int64_t lim = (DIR == 0 ? a.v.mp : a.v.kp) - 128;
        const uint32_t bytes = (uint32_t)(TILE / ROWS * a.v.rec);
        for (int un = worker; un < units && !*abort_flag; un += workers) {
            const Unit u = unit_at<CG>(a, un);
            const int64_t nl = min(u.n0 + (int64_t)rank * 128, lim);
            const bool ok = tiles(u, [&](int kt, int, int, bool, bool) {
                const int cs = ct % CODE_STAGES;
                if (!mbar_wait(&cempty[cs], ((ct / CODE_STAGES) & 1u) ^ 1u, abort_flag, a.err, a.wait_limit)) return false;
                const int64_t at = DIR == 0 ? record_at(a.v, nl, kt) : record_at(a.v, (int64_t)kt * TILE, nl / TILE);
                mbar_expect_tx(&cfull[cs], bytes);
                bulk_load(codes + cs * CODE_BYTES, a.v.packed + at, bytes, &cfull[cs]);
                ct++;
                return true;
            });
            if (!ok) break;
        }
    }

    // Tail: no commit may still be on its way to a barrier of this CTA, nor, after an abort, a load to its memory.
    __syncwarp();
    if (warp == 0 && lane == 0)
        for (uint32_t k = it > STAGES ? it - STAGES : 0; k < it; k++) {
            if (!*abort_flag) mbar_wait_drain(&empty[k % STAGES], (k / STAGES) & 1u);
            else if (rank == 0) mbar_wait_drain(&afull[k % STAGES], (k / STAGES) & 1u);
        }
    if (*abort_flag && warp == 2 + EW + DQ_WARPS && lane == 0)
        for (uint32_t k = ct > CODE_STAGES ? ct - CODE_STAGES : 0; k < ct; k++) mbar_wait_drain(&cfull[k % CODE_STAGES], (k / CODE_STAGES) & 1u);
    if (*abort_flag && warp == 1 && lane == 0 && rank == 0)
        for (int b = 0; b < 2; b++)
            if (commit_par[b] >= 0) mbar_wait_drain(&tfull[b], (uint32_t)commit_par[b]);
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// Workers (CTAs, or pairs) of a kernel that fit the device at once; asked once per kernel and device.
template <auto kernel> int max_workers(llmc_ctx* ctx, int cg, int threads) {
    static std::mutex mu;
    static int cache[64];
    static bool known[64];
    const int dev = ctx->device;
    if (dev < 0 || dev >= 64) return 0;
    std::lock_guard<std::mutex> lock(mu);
    if (!known[dev]) {
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        if (cg == 1) {
            n = ctx->sm_count;
        } else {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(2 * (unsigned)ctx->sm_count);
            cfg.blockDim = dim3((unsigned)threads);
            cfg.dynamicSmemBytes = SMEM_BYTES;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 2;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, (const void*)kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
        }
        cache[dev] = n;
        known[dev] = true;
    }
    return cache[dev];
}

template <typename T, typename O, int DIR, int CG, int PIECES, bool ONE>
llmc_status launch_as(llmc_ctx* ctx, cudaStream_t st, const CUtensorMap& map, GemmInt4& g) {
    constexpr auto kernel = gemm_int4_kernel<T, O, DIR, CG, PIECES, ONE>;
    constexpr int threads = 32 * (3 + (PIECES == 3 ? 8 : 4) + DQ_WARPS);
    int cap = max_workers<kernel>(ctx, CG, threads);
    if (cap < 1) return fail(LLMC_ERR_CUDA, "the packed product's kernel does not fit this device");
    const int allowed = persistent_sms(ctx) >= CG ? persistent_sms(ctx) / CG : 1;  // one pair at least
    if (cap > allowed) cap = allowed;
    const int64_t units = (int64_t)g.tiles_m * g.tiles_n * g.splits;
    const int workers = units < cap ? (int)units : cap;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(workers * CG));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    LLMC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map, g));
    return check_launch(ctx, "int4_gemm");
}

template <typename T, typename O, int DIR, int CG, int PIECES>
llmc_status launch(llmc_ctx* ctx, cudaStream_t st, const CUtensorMap& map, GemmInt4& g) {
    return g.v.ng == 1 ? launch_as<T, O, DIR, CG, PIECES, true>(ctx, st, map, g) : launch_as<T, O, DIR, CG, PIECES, false>(ctx, st, map, g);
}

}  // namespace

// CTAs per tile: pairs (256 x 256) share what they dequantise and load, single CTAs (128 x 128) fill more SMs, so they are
// taken while one round of them holds the product and the contraction is not so long that sharing counts for more.  us, fp16,
// single and pairs: 4096 -> 4096, 512 tokens (128 tiles) 33 and 38, 768 (192) 54 and 41; 2048 -> 2048, 1,024 (128) 21 and 32,
// 2,048 (256) 34 and 29; 576 -> 1536, 1,024 (96) 12 and 25; 14336 -> 4096, 160 tokens 52 and 42, 512 86 and 76.  Contractions
// between 4,096 and 14,336 were not measured: the border is their geometric middle, rounded.
int int4_gemm_cg(const llmc_ctx* ctx, int dtype, int64_t tokens, int64_t cols, int64_t contraction) {
    if (dtype == LLMC_DTYPE_F32 || tokens <= 128 || cols <= 128) return 1;
    const bool round = (tokens + 127) / 128 * ((cols + 127) / 128) <= ctx->sm_count;
    return round && contraction <= 64 * TILE ? 1 : 2;
}

// Splits of the contraction: enough to give every worker a tile, two tiles of 128 to a split at least (one in fp32,
// where a tile is six products).
int int4_gemm_splits(const llmc_ctx* ctx, int dtype, int64_t tokens, int64_t cols, int64_t contraction) {
    const int cg = int4_gemm_cg(ctx, dtype, tokens, cols, contraction);
    const int64_t tile = 128 * cg, tiles = ((tokens + tile - 1) / tile) * ((cols + tile - 1) / tile);
    // by the device's SMs, not llmc_set_sm_limit's: a workspace that was asked for stays large enough
    const int64_t kt = contraction / TILE, workers = ctx->sm_count / cg;
    int64_t s = workers / tiles;
    const int64_t most = dtype == LLMC_DTYPE_F32 ? kt : kt / 2;
    if (s > most) s = most;
    if (s > 32) s = 32;
    if (s < 1) s = 1;
    const int64_t per = (kt + s - 1) / s;
    return (int)((kt + per - 1) / per);
}

// A [pieces][tokens][lda] 16-bit, K-major (see int4_stage for the pieces of fp32); out [tokens][ldo].
llmc_status int4_gemm(llmc_ctx* ctx, cudaStream_t st, const w4::View& v, int dir, int dtype, const void* A, int64_t acols, int64_t lda,
                      int64_t tokens, const void* bias, void* out, int64_t ldo, int splits, float* part) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(LLMC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int pieces = dtype == LLMC_DTYPE_F32 ? 4 : 1;
    const int64_t cols = dir == 0 ? v.rows : v.kp, contraction = dir == 0 ? v.kp : v.mp;
    const int cg = int4_gemm_cg(ctx, dtype, tokens, cols, contraction);
    GemmInt4 g{};
    g.v = v;
    g.tokens = tokens;
    g.ocols = dir == 0 ? v.rows : v.cols;
    const int64_t tile = 128 * cg;
    g.tiles_m = (int)((tokens + tile - 1) / tile);
    g.tiles_n = (int)((cols + tile - 1) / tile);
    g.splits = splits;
    g.kt_total = (int)(contraction / TILE);
    g.kt_per = (g.kt_total + splits - 1) / splits;
    g.group_m = 8;
    g.piece_rows = tokens;
    g.bias = splits > 1 ? nullptr : bias;
    g.out = out;
    g.ldo = ldo;
    g.part = part;
    const int es = dtype_size(dtype);
    g.wide = (uintptr_t)out % 16 == 0 && (ldo * es) % 16 == 0;
    g.err = ctx->dflags + 2;
    g.wait_limit = ctx->wait_limit;
    const uint32_t fmt = dtype == LLMC_DTYPE_F16 ? 0u : 1u;
    g.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)dir << 16) | ((uint32_t)(tile >> 3) << 17) | ((uint32_t)(tile >> 4) << 24);

    CUtensorMap map;
    const cuuint64_t dim[2] = {(cuuint64_t)acols, (cuuint64_t)(tokens * pieces)};
    const cuuint64_t stride[1] = {(cuuint64_t)lda * 2};
    const cuuint32_t box[2] = {BOX, 128}, es1[2] = {1, 1};
    const CUresult cr = enc(&map, fmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(A), dim, stride,
                            box, es1, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) return fail(LLMC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    using B = __nv_bfloat16;
    if (dtype == LLMC_DTYPE_F32) return dir ? launch<B, float, 1, 1, 3>(ctx, st, map, g) : launch<B, float, 0, 1, 3>(ctx, st, map, g);
    if (dtype == LLMC_DTYPE_BF16) {
        if (cg == 2) return dir ? launch<B, B, 1, 2, 1>(ctx, st, map, g) : launch<B, B, 0, 2, 1>(ctx, st, map, g);
        return dir ? launch<B, B, 1, 1, 1>(ctx, st, map, g) : launch<B, B, 0, 1, 1>(ctx, st, map, g);
    }
    if (cg == 2) return dir ? launch<__half, __half, 1, 2, 1>(ctx, st, map, g) : launch<__half, __half, 0, 2, 1>(ctx, st, map, g);
    return dir ? launch<__half, __half, 1, 1, 1>(ctx, st, map, g) : launch<__half, __half, 0, 1, 1>(ctx, st, map, g);
}

}  // namespace llmc
