// Packed 4-bit weights: laying them out, reading them back, and products with few rows.
//
// The reference quantises (RtnModifier.cs:44-122, GPTQModifier.cs:108-137) and dequantises
// (Int4PackedTensor.cs:152-161); it multiplies only dense weights.  These kernels take the codes as
// they are: y[t][n] = sum_k x[t][k] (u - z) s + b[n].
#include "int4.cuh"
#include "ops.h"
#include "tc_common.cuh"

#include <atomic>

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
    uint8_t* packed;
};

__device__ __forceinline__ uint32_t zero_of(const LayoutArgs& a, int64_t r, int g) {
    if (a.sym || r >= a.v.rows) return 8u;
    return (uint32_t)a.zps[a.srow ? r * a.srow + g : 0] & 0xFu;
}

// One thread per word of eight codes, and per scale; one read of the codes and one write, bound by memory.
__global__ void __launch_bounds__(256) layout_kernel(const LayoutArgs a) {
    const int64_t ktiles = a.v.kp / TILE;
    const int64_t words = a.v.mp * (a.v.kp / 8);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int64_t rec = i / (ROWS * 16);
        const int in = (int)(i % (ROWS * 16)), t = in % 16 / 4, c = in % 4;
        const int64_t tile = rec / (TILE / ROWS);
        const int64_t r = tile / ktiles * TILE + rec % (TILE / ROWS) * ROWS + in / 16;
        const int kv0 = (int)(tile % ktiles) * TILE + 32 * c + 8 * t;
        const uint32_t z = zero_of(a, r, group_of(kv0, a.v.gsv, a.v.groups));
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
        *reinterpret_cast<uint32_t*>(a.packed + rec * a.v.rec + in * 4) = w;
    }
    const int64_t entries = a.v.mp * ktiles * a.v.ng;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
        const int per = ROWS * a.v.ng;
        const int64_t rec = i / per, tile = rec / (TILE / ROWS);
        const int in = (int)(i % per), j = in % a.v.ng;
        const int64_t r = tile / ktiles * TILE + rec % (TILE / ROWS) * ROWS + in / a.v.ng;
        const int g = group_of((int)(tile % ktiles) * TILE + j * (TILE / a.v.ng), a.v.gsv, a.v.groups);
        uint8_t* p = a.packed + rec * a.v.rec + 1024;
        reinterpret_cast<float*>(p)[in] = r < a.v.rows ? a.scales[a.srow ? r * a.srow + g : 0] : 0.f;
        p[64 * a.v.ng + in] = (uint8_t)zero_of(a, r, g);
    }
}

// Exponents that bring the scales near one before they meet fp16's range: for each row, and for each group of
// each tile, e with 2^(e-1) <= max |s| < 2^e, within +-120 (0 where the maximum is 0 or not finite).  A product
// kernel in fp16 uses s 2^-e and gives 2^e back in fp32, both exact.
__global__ void __launch_bounds__(256) exps_kernel(const View v, int32_t* exps) {
    const int64_t row_blocks = v.mp / TILE;
    const int slots = (int)(v.kp / TILE) * v.ng;
    const auto scale = [&](int64_t r, int s) {
        return fabsf(reinterpret_cast<const float*>(v.packed + record_at(v, r, s / v.ng) + 1024)[r % ROWS * v.ng + s % v.ng]);
    };
    float m = 0.f;
    __shared__ float sm[256];
    const bool rows = blockIdx.x < row_blocks;
    if (rows) {
        for (int s = threadIdx.x / TILE; s < slots; s += 2) m = fmax_nan(m, scale((int64_t)blockIdx.x * TILE + threadIdx.x % TILE, s));
    } else {
        for (int64_t r = threadIdx.x; r < v.mp; r += 256) m = fmax_nan(m, scale(r, (int)(blockIdx.x - row_blocks)));
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
        exps[v.mp + blockIdx.x - row_blocks] = e;
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
        float val[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ok) {
            const uint8_t* rec = v.packed + record_at(v, r, kt);
            const int in = (int)(r % ROWS), slot = in * v.ng + slot_of(kb / 4, v.ng);
            const uint32_t w = reinterpret_cast<const uint32_t*>(rec)[in * 16 + (kb % 4) * 4 + kb / 4];
            const float s = reinterpret_cast<const float*>(rec + 1024)[slot];
            const int z = rec[1024 + 64 * v.ng + slot];
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
// three bf16 pieces whose sum is x exactly: each takes the eight leading bits that are left, rounded to nearest so
// that what the products of pieces leave out (k_int4_gemm.cu) is small and of either sign (truncated where the
// first would round to an infinity).  An infinity or a NaN is all in the first piece; a fourth (pieces = 4) is the
// first with zeros in their place, for products with the smaller pieces of a weight, where an infinity times zero or
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
                float hi = to_f<__nv_bfloat16>(__float2bfloat16_rn(f));
                if (!isfinite(hi)) hi = __uint_as_float(b & 0xFFFF0000u);
                const float r1 = fin ? __fsub_rn(f, hi) : 0.f;
                const float mid = to_f<__nv_bfloat16>(__float2bfloat16_rn(r1));
                const float lo = __fsub_rn(r1, mid);
                p[0].h[j] = f != f ? (uint16_t)0x7FC0 : (uint16_t)(__float_as_uint(hi) >> 16);
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
// d = a b + c, with c = 0 where `fresh`.
template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool fresh) {
    const float c0 = fresh ? 0.f : d[0], c1 = fresh ? 0.f : d[1], c2 = fresh ? 0.f : d[2], c3 = fresh ? 0.f : d[3];
    if constexpr (Num<T>::MAGIC == Num<__half>::MAGIC)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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

// Warps to a CTA at most, and its shared memory: half an SM's, with fewer warps where it has to be (one CTA to an SM with
// eight warps took 21.4 us for 4096 -> 14336 and 16 tokens, two with six 18.4; 14 or 16 warps for one token, no less than 8).
constexpr int FEW_WARPS = 8, FEW_SMEM = 112 * 1024;
// Tiles of the columns to a step and steps to a ring.
__host__ __device__ constexpr int few_tiles(int nt, int rb) { return nt == 1 && rb == 1 ? 2 : 1; }
__host__ __device__ constexpr int few_stages(int nt, int rb) { return nt == 1 && rb < 4 ? 3 : 2; }

__device__ __forceinline__ void copy16(void* dst, const void* src, int bytes) {  // bytes < 16: zeros for the rest
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// The codes are the A operand of m16n8k16 (16 weight rows x 16 columns), x the B operand (8 tokens), so one
// dequantised fragment serves eight tokens and a single token costs no more than the codes.  Codes enter as
// the exact integers u - z; the fp32 sum of a group is multiplied by its scale (4 / NG granules of 32 columns per
// group sum), so x and W are never rounded.  Columns of the MMA that stand for no token repeat the last one's x.
// A CTA holds RB records' rows (16 RB) and 8 NT tokens; its warps take steps of FEW_TILES 128-column tiles in turn and
// add their sums in shared memory, in warp order.  Each warp keeps a ring of STAGES steps, the records and the 256 bytes
// a tile of each token's x (XS), by 16-byte asynchronous copies that it waits for by itself.  The three pieces of fp32
// x would take most of the ring and are read through L1, which row blocks of few columns share.
// What bounds it is latency and balance.  A record's instructions (88 to turn its codes into numbers, 26 of other
// arithmetic, about 70 of loops, copies and waits) are 1.06 times the issue slots that an SM has for it at the HBM's rate,
// and one token of 14336 -> 4096 takes 2.4 times that: a scheduler's three or four warps, each one chain of load, mask,
// subtract, multiply, scale, leave 48 % of its slots empty, and an SM is active 0.66 of the time (256 CTAs on 148 SMs, start
// and end).  One token, bf16: 14336 -> 4096 11.5 us (2.8 TB/s), 576 -> 576 2.3, 4096 -> 14336 12.4.  16 tokens 18 (2.3 warps
// to a scheduler, 64 % of the slots empty).
template <typename T, typename O, int NT, int PIECES, int NG, int RB>
__global__ void __launch_bounds__(32 * FEW_WARPS) few_kernel(const FewArgs a) {
    constexpr int REC = 1024 + 80 * NG, FL = 4 / NG, SUMS = 8 * NT * ROWS * RB, STAGES = few_stages(NT, RB), FEW_TILES = few_tiles(NT, RB);
    constexpr bool XS = PIECES == 1;
    extern __shared__ __align__(128) uint8_t smem[];  // int_pair's operands, rings; afterwards [warps][8 NT][16 RB] of sums
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const int g = lane >> 2, t = lane & 3;
    const int tok0 = blockIdx.y * 8 * NT, toks = min(8 * NT, a.tokens - tok0);
    const int64_t row0 = (int64_t)blockIdx.x * (ROWS * RB);
    const int ktiles = (int)(a.v.kp / TILE);
    const int xrow = FEW_TILES * 256, xat0 = FEW_TILES * RB * REC, room = xat0 + (XS ? toks * xrow : 0);
    uint8_t* ring = smem + 16 + warp * STAGES * room;
    if (threadIdx.x == 0) put_bits<T>(reinterpret_cast<uint2*>(smem));
    __syncthreads();
    const Bits bits = get_bits(reinterpret_cast<const uint2*>(smem));

    constexpr int64_t TILE_BYTES = TILE / ROWS * REC;
    const int hop = warps * FEW_TILES;  // tiles from one of this warp's steps to its next
    int fkt = warp * FEW_TILES;         // the step to fetch next
    const uint8_t* src = a.v.packed + record_at(a.v, row0, fkt) + lane * 16;
    const T* xsrc = reinterpret_cast<const T*>(a.x) + (int64_t)(tok0 + lane / (16 * FEW_TILES)) * a.ldx + fkt * TILE + lane % (16 * FEW_TILES) * 8;
    auto fetch = [&](uint8_t* stage) {
        if (fkt < ktiles) {
            uint8_t* dst = stage + lane * 16;
#pragma unroll
            for (int k = 0; k < FEW_TILES; k++) {
                if (k > 0 && fkt + k >= ktiles) break;
#pragma unroll
                for (int i = 0; i < RB * REC / 512; i++) copy16(dst + k * RB * REC + i * 512, src + k * TILE_BYTES + i * 512, 16);
                if (lane < RB * REC % 512 / 16)
                    copy16(dst + k * RB * REC + RB * REC / 512 * 512, src + k * TILE_BYTES + RB * REC / 512 * 512, 16);
            }
            if (XS) {  // zeros past the last column
                constexpr int EACH = 2 / FEW_TILES;  // tokens to a copy: a token's x of a step is 16 lanes' or 32
                const bool in = fkt * TILE + lane % (16 * FEW_TILES) * 8 < a.xcols;
                const T* xr = in ? xsrc : reinterpret_cast<const T*>(a.x);
                const int64_t next = in ? EACH * a.ldx : 0;
                for (int r = lane / (16 * FEW_TILES); r < toks; r += EACH, xr += next)
                    copy16(stage + xat0 + r * xrow + lane % (16 * FEW_TILES) * 16, xr, in ? 16 : 0);
            }
            fkt += hop;
            src += hop * TILE_BYTES;
            xsrc += hop * TILE;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) fetch(ring + s * room);

    int xat[NT];  // this lane's token of each eight: its x in a stage, or its number
#pragma unroll
    for (int n = 0; n < NT; n++) xat[n] = XS ? xat0 + min(n * 8 + g, toks - 1) * xrow + t * 16 : min(n * 8 + g, toks - 1);
    auto load_x = [&](const uint8_t* stage, int kt, int c, int n, int p) {
        if (XS) return *reinterpret_cast<const uint4*>(stage + xat[n] + c * 64);
        const int k = kt * TILE + 32 * c + 8 * t;
        if (k >= a.xcols) return make_uint4(0, 0, 0, 0);
        return __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x) + ((int64_t)p * a.tokens + tok0 + xat[n]) * a.ldx + k));
    };
    float acc[RB][NT][4];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[r][n][j] = 0.f;
    int at = 0, free = (STAGES - 1) * room;  // the stages to multiply and to fill
    for (int kt0 = warp * FEW_TILES; kt0 < ktiles; kt0 += hop) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        fetch(ring + free);
        free = at;
        const uint8_t *rec = ring + at, *xstage = rec;
        at = at == (STAGES - 1) * room ? 0 : at + room;
#pragma unroll 1
        for (int kt = kt0; kt < min(ktiles, kt0 + FEW_TILES); kt++, rec += RB * REC, xstage += 256) {
            uint32_t w[RB][2][4], zz[RB][2][NG];
            float sc[RB][2][NG];
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint8_t* q = rec + r * REC;
                    const int row = g + 8 * h;
                    const uint4 u = *reinterpret_cast<const uint4*>(q + row * 64 + t * 16);
                    w[r][h][0] = u.x;
                    w[r][h][1] = u.y;
                    w[r][h][2] = u.z;
                    w[r][h][3] = u.w;
#pragma unroll
                    for (int j = 0; j < NG; j++) {
                        sc[r][h][j] = reinterpret_cast<const float*>(q + 1024)[row * NG + j];
                        zz[r][h][j] = q[1024 + 64 * NG + row * NG + j] * 0x10001u + bits.magic;
                    }
                }
            float d[RB][NT][4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int j = c / FL;
                uint4 b[NT][PIECES];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int p = 0; p < PIECES; p++) b[n][p] = load_x(xstage, kt, c, n, p);
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int k = 0; k < 4; k++) f[h][k] = int_pair<T>(w[r][k & 1][c], 2 * h + k / 2, zz[r][k & 1][j], bits);
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int p = PIECES - 1; p >= 0; p--) {
                            mma16816<T>(d[r][n], f[0], b[n][p].x, b[n][p].y, c % FL == 0 && p == PIECES - 1);
                            mma16816<T>(d[r][n], f[1], b[n][p].z, b[n][p].w, false);
                        }
                    if (c % FL == FL - 1)
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int k = 0; k < 4; k++) acc[r][n][k] = fmaf(sc[r][k / 2][j], d[r][n][k], acc[r][n][k]);
                }
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the rings are done with
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)  // [warp][token][row]
                red[warp * SUMS + (n * 8 + 2 * t + (i & 1)) * (ROWS * RB) + r * ROWS + g + 8 * (i / 2)] = acc[r][n][i];
    __syncthreads();
    for (int i = threadIdx.x; i < toks * (ROWS * RB); i += blockDim.x) {
        const int64_t row = row0 + i % (ROWS * RB);
        if (row >= a.v.rows) continue;
        float s = 0.f;
        for (int w = 0; w < warps; w++) s += red[w * SUMS + i];
        if (a.bias) s += to_f<O>(reinterpret_cast<const O*>(a.bias)[row]);
        reinterpret_cast<O*>(a.y)[(tok0 + i / (ROWS * RB)) * a.ldy + row] = from_f<O>(s);
    }
}

// ---- joining partial sums, column sums ------------------------------------------------------------
// out[r][c] = sum over s of part[s][r][c] (in order) + bias[c], rounded once.
template <typename O>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int64_t rows, int64_t cols, const O* bias,
                                                  O* out, int64_t ldo) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    const float b = bias ? to_f<O>(bias[c]) : 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        float s = 0.f;
        const float* p = part + r * cols + c;
#pragma unroll 4
        for (int k = 0; k < splits; k++) s += p[k * rows * cols];
        out[r * ldo + c] = from_f<O>(s + b);
    }
}

// part[split][c] = sum of rows split * per .. of x[:, c], or (one split) out[c] rounded; a block holds 32 columns x
// 8 row lanes.
template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const T* x, int64_t rows, int64_t cols, int64_t ld, int64_t per, float* part, T* out) {
    __shared__ float sm[8][33];
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    const int64_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    float s = 0.f;
    if (c < cols)
#pragma unroll 4
        for (int64_t r = r0 + w; r < r1; r += 8) s += to_f<T>(x[r * ld + c]);
    sm[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; i++) s += sm[i][lane];
        if (out) out[c] = from_f<T>(s);
        else part[blockIdx.y * cols + c] = s;
    }
}

int grid_n(const llmc_ctx* ctx, int64_t items) {
    const int64_t b = (items + 255) / 256, cap = (int64_t)ctx->sm_count * 16;
    return (int)(b < 1 ? 1 : (b > cap ? cap : b));
}

template <typename T, typename O, int NT, int PIECES, int NG, int RB>
llmc_status launch_few(llmc_ctx* ctx, const FewArgs& a, cudaStream_t st) {
    constexpr auto kernel = few_kernel<T, O, NT, PIECES, NG, RB>;
    constexpr int REC = 1024 + 80 * NG, STAGES = few_stages(NT, RB), FEW_TILES = few_tiles(NT, RB);
    static std::atomic<bool> ready[64];
    const int64_t blocks = (a.v.rows + ROWS * RB - 1) / (ROWS * RB);
    const int ktiles = (int)(a.v.kp / TILE), tiles = (a.tokens + 8 * NT - 1) / (8 * NT);
    const int steps = (ktiles + FEW_TILES - 1) / FEW_TILES, toks = a.tokens < 8 * NT ? a.tokens : 8 * NT;
    const int each = STAGES * FEW_TILES * (RB * REC + (PIECES == 1 ? toks * 256 : 0));
    int warps = FEW_WARPS;
    if (warps > (FEW_SMEM - 16) / each) warps = (FEW_SMEM - 16) / each;
    const int rounds = (steps + warps - 1) / warps;
    warps = (steps + rounds - 1) / rounds;  // no more than finish as early
    size_t sm = 16 + (size_t)warps * each, sums = (size_t)warps * 8 * NT * ROWS * RB * sizeof(float);
    if (sm < sums) sm = sums;
    static_assert(16 + 2 * STAGES * FEW_TILES * (RB * REC + (PIECES == 1 ? 8 * NT * 256 : 0)) <= FEW_SMEM, "room for two warps");
    if (ctx->device < 0 || ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_relaxed)) {
        LLMC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
        if (ctx->device >= 0 && ctx->device < 64) ready[ctx->device].store(true, std::memory_order_relaxed);
    }
    kernel<<<dim3((unsigned)blocks, (unsigned)tiles), warps * 32, sm, st>>>(a);
    return check_launch(ctx, "int4_few");
}

template <typename T, typename O, int NT, int PIECES, int RB> llmc_status few_by_group(llmc_ctx* ctx, const FewArgs& a, cudaStream_t st) {
    if (a.v.ng == 1) return launch_few<T, O, NT, PIECES, 1, RB>(ctx, a, st);
    if (a.v.ng == 2) return launch_few<T, O, NT, PIECES, 2, RB>(ctx, a, st);
    return launch_few<T, O, NT, PIECES, 4, RB>(ctx, a, st);
}

// Record rows to a CTA.  Several share x, from memory and out of shared memory, at the cost of fewer CTAs: worth it where
// the SMs have some to spare, and (with x in two fragments or three pieces, whose rings leave few warps) where the
// contraction gives each warp a tile.  us for 1, 2, 4 rows, 16-bit: 4096 -> 14336, 8 tokens 22.2, 16.9, 13.7, 16 tokens 29.0,
// 23.7, 18.4; 4096 -> 4096, 8 tokens 8.4, 6.2, 8.3; 576 -> 49152, 1 token 15.9, 10.5, 9.0, 16 tokens 15.4, 17.1, 17.3.  fp32: 4096 -> 14336,
// 8 tokens 27.6, 22.1, 20.7, 16 tokens 40.6, 37.6, 31.7; 4096 -> 4096, 8 tokens 7.7, 9.3, 10.9, 16 tokens 15.3, 10.1, 16.3;
// 576 -> 49152, 5 tokens 12.5, 11.4, 12.8, 16 tokens 23.1, 34.2, 32.6; 576 -> 1536, 16 tokens 5.2, 4.1, 6.4.
template <int NT, int PIECES> int few_record_rows(const llmc_ctx* ctx, const FewArgs& a) {
    const int64_t blocks = (a.v.rows + ROWS - 1) / ROWS * ((a.tokens + 8 * NT - 1) / (8 * NT)), sms = ctx->sm_count;
    const bool deep = a.v.kp >= 8 * TILE;
    if (PIECES == 1) {
        if (NT == 2 && !deep) return 1;
        // one token: 14336 rows 12.4, 12.7, 12.8
        return blocks >= (a.tokens > 1 ? 4 : 8) * sms ? 4 : a.tokens > 1 && 2 * blocks >= 3 * sms ? 2 : 1;
    }
    if (NT == 1) return blocks < 4 * sms ? 1 : deep ? 4 : 2;
    if (!deep) return blocks < 3 * sms ? 2 : 1;
    return blocks < 6 * sms ? 2 : 4;
}

template <typename T, typename O, int NT, int PIECES> llmc_status few_by_rows(llmc_ctx* ctx, const FewArgs& a, cudaStream_t st) {
    const int rb = few_record_rows<NT, PIECES>(ctx, a);
    if (rb == 4) return few_by_group<T, O, NT, PIECES, 4>(ctx, a, st);
    if (rb == 2) return few_by_group<T, O, NT, PIECES, 2>(ctx, a, st);
    return few_by_group<T, O, NT, PIECES, 1>(ctx, a, st);
}

template <typename T, typename O, int PIECES> llmc_status few_by_size(llmc_ctx* ctx, const FewArgs& a, cudaStream_t st) {
    return a.tokens > 8 ? few_by_rows<T, O, 2, PIECES>(ctx, a, st) : few_by_rows<T, O, 1, PIECES>(ctx, a, st);
}

}  // namespace

llmc_status int4_layout(llmc_ctx* ctx, cudaStream_t st, const uint8_t* codes, int64_t crow, const float* scales,
                        const int32_t* zps, int64_t srow, int sym, const w4::View& v, uint8_t* packed, int32_t* exps) {
    LayoutArgs a{codes, crow, scales, zps, srow, sym, v, packed};
    layout_kernel<<<grid_n(ctx, v.mp * (v.kp / 8)), 256, 0, st>>>(a);
    LLMC_TRY(check_launch(ctx, "int4_layout"));
    exps_kernel<<<(unsigned)(v.mp / TILE + v.kp / TILE * v.ng), 256, 0, st>>>(v, exps);
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
    if (dtype == LLMC_DTYPE_F32) return few_by_size<__nv_bfloat16, float, 3>(ctx, a, st);
    if (dtype == LLMC_DTYPE_BF16) return few_by_size<__nv_bfloat16, __nv_bfloat16, 1>(ctx, a, st);
    return few_by_size<__half, __half, 1>(ctx, a, st);
}

llmc_status int4_join(llmc_ctx* ctx, cudaStream_t st, const float* part, int splits, int64_t rows, int64_t cols, const void* bias,
                      void* out, int dtype, int64_t ldo) {
    const int64_t wide = (cols + 255) / 256, most = 16 * (int64_t)ctx->sm_count / wide + 1;
    const dim3 grid((unsigned)wide, (unsigned)(rows < most ? rows : most));
    if (dtype == LLMC_DTYPE_F32)
        join_kernel<float><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const float*)bias, (float*)out, ldo);
    else if (dtype == LLMC_DTYPE_BF16)
        join_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const __nv_bfloat16*)bias, (__nv_bfloat16*)out, ldo);
    else
        join_kernel<__half><<<grid, 256, 0, st>>>(part, splits, rows, cols, (const __half*)bias, (__half*)out, ldo);
    return check_launch(ctx, "int4_join");
}

llmc_status col_sum(llmc_ctx* ctx, cudaStream_t st, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int splits,
                    float* part, void* out) {
    const dim3 grid((unsigned)((cols + 31) / 32), (unsigned)splits);
    const int64_t per = (rows + splits - 1) / splits;
    void* direct = splits == 1 ? out : nullptr;
    if (dtype == LLMC_DTYPE_F32) colsum_kernel<float><<<grid, 256, 0, st>>>((const float*)x, rows, cols, ld, per, part, (float*)direct);
    else if (dtype == LLMC_DTYPE_BF16)
        colsum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, rows, cols, ld, per, part, (__nv_bfloat16*)direct);
    else colsum_kernel<__half><<<grid, 256, 0, st>>>((const __half*)x, rows, cols, ld, per, part, (__half*)direct);
    LLMC_TRY(check_launch(ctx, "col_sum"));
    return splits == 1 ? LLMC_OK : int4_join(ctx, st, part, splits, 1, cols, nullptr, out, dtype, cols);
}

}  // namespace llmc
