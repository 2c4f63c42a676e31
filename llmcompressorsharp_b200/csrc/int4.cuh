// The packed 4-bit weight as the kernels see it (see llmc_int4_weight in llmc_b200.h).
//
// W[n][k] = (u - z) * s, u the 4-bit code moved to [0, 15] and z the byte that stands for zero: the
// zero-point of an asymmetric grid, 8 for a symmetric one, so that both grids are one form.
//
// Columns.  A group of gs columns takes gsv = gs rounded up to 32 columns of the layout, so that 32
// consecutive layout columns ("a granule") share one scale; gs a multiple of 32, or one group per
// row, leaves the columns where they were.  kp is their number rounded up to 128.  Rows are rounded
// up to 128 (mp).  Codes that stand for no weight hold u = z, and rows past the last have s = 0.
//
// Tiles of 128 rows x 128 columns stand one row block after the other; a tile is eight records of 16 rows:
//
//   codes   16 rows x 64 bytes.  A row's 64 bytes are four 16-byte chunks t of four words c; word c of chunk t
//           holds columns 32 c + 8 t .. + 7, column 2 p in bits 4 p .. 4 p + 3 and column 2 p + 1 sixteen bits
//           above, so that (word >> 4 p) & 0x000F000F is a pair of neighbours.  A thread's 16-byte load then is,
//           for an m16n8k16 fragment, lane t's part of all four granules, and the pairs meet x unpermuted.
//   scales  16 rows x ng floats, ng = 1, 2 or 4 groups to a tile's 128 columns (the fewest that fit the group
//           size; a group of 256 columns or more has its scale in each tile)
//   zeros   16 rows x ng bytes
//
// So whatever a product needs of a tile is one stretch of 8,832 bytes (ng = 1), which one bulk copy brings in, and
// nothing comes from a second place with a latency of its own.
#pragma once
#include "common.cuh"

namespace llmc {
namespace w4 {

constexpr int TILE = 128;  // rows and columns of a tile
constexpr int ROWS = 16;   // rows of a record
constexpr int MAX_NG = 4;

struct View {
    const uint8_t* packed;
    const int32_t* exps;     // [mp] of the rows, then [kp / 128 * ng] of the groups: see exps_kernel
    int64_t rows, cols;
    int64_t mp, kp;
    int32_t gs, gsv, groups;
    int32_t ng, rec;         // groups per tile, bytes of a record
    int32_t identity;        // layout columns are the weight's own
};

inline int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// Fills the derived sizes from rows, cols and gs (columns per group; >= cols: one group).
inline void set_sizes(View& v, int64_t rows, int64_t cols, int64_t gs) {
    v.rows = rows;
    v.cols = cols;
    v.mp = up(rows, TILE);
    if (gs >= cols) {
        v.groups = 1;
        v.gs = (int32_t)cols;
        v.gsv = (int32_t)up(cols, TILE);
        v.kp = v.gsv;
        v.identity = 1;
    } else {
        v.gs = (int32_t)gs;
        v.gsv = (int32_t)up(gs, 32);
        v.groups = (int32_t)((cols + gs - 1) / gs);
        v.kp = up((int64_t)(v.groups - 1) * v.gsv + (cols - (int64_t)(v.groups - 1) * gs), TILE);
        v.identity = gs % 32 == 0;
    }
    v.ng = v.gsv % 128 == 0 ? 1 : v.gsv % 64 == 0 ? 2 : 4;
    v.rec = 1024 + 80 * v.ng;
}

// Group of the granule that holds layout column kv (columns past the last group: the last).
__host__ __device__ __forceinline__ int group_of(int kv, int gsv, int groups) {
    const int g = kv / gsv;
    return g < groups ? g : groups - 1;
}

// Byte at which the record of row r's 16 rows and columns 128 kt .. stands.
__host__ __device__ __forceinline__ int64_t record_at(const View& v, int64_t r, int64_t kt) {
    return ((r / TILE * (v.kp / TILE) + kt) * (TILE / ROWS) + r % TILE / ROWS) * v.rec;
}

// Group, of a tile's ng, that granule c belongs to.
__host__ __device__ __forceinline__ int slot_of(int c, int ng) { return c * ng / 4; }

// The weight's column of layout column kv, -1 where none is.
__host__ __device__ __forceinline__ int64_t column_of(int kv, int gs, int gsv, int groups, int64_t cols) {
    const int g = group_of(kv, gsv, groups);
    const int j = kv - g * gsv;
    const int64_t k = (int64_t)g * gs + j;
    return (j < gs && k < cols) ? k : -1;
}

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// ---- codes to numbers -------------------------------------------------------------------------
// 0x4300 | u is bf16 128 + u and 0x6400 | u is fp16 1024 + u, both exact; taking 128 + z (1024 + z)
// away leaves the integer u - z, exact as well.
template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
    using T2 = __nv_bfloat162;
    static constexpr uint32_t MAGIC = 0x43004300u;
};
template <> struct Num<__half> {
    using T2 = __half2;
    static constexpr uint32_t MAGIC = 0x64006400u;
};

template <typename T> __device__ __forceinline__ typename Num<T>::T2 as2(uint32_t u) {
    typename Num<T>::T2 r;
    *reinterpret_cast<uint32_t*>(&r) = u;
    return r;
}
template <typename T2> __device__ __forceinline__ uint32_t bits2(T2 v) { return *reinterpret_cast<uint32_t*>(&v); }

template <typename T> __device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
    return Num<T>::MAGIC | z | (z << 16);
}

// The operands of int_pair's logic operation, in registers: as literals the compiler, which can put one into an
// instruction, fetches the other anew for each pair, a fourth instruction on the three that a pair takes.  They come
// through shared memory (`slot`, written by one thread before a barrier) to hide their values from it.
struct Bits {
    uint32_t mask, magic;
};
template <typename T> __device__ __forceinline__ void put_bits(uint2* slot) { *slot = make_uint2(0x000F000Fu, Num<T>::MAGIC); }
__device__ __forceinline__ Bits get_bits(const uint2* slot) {
    Bits b;
    asm volatile("ld.volatile.shared.v2.u32 {%0, %1}, [%2];"
                 : "=r"(b.mask), "=r"(b.magic)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot))));
    return b;
}

// Pair p (columns 2 p, 2 p + 1) of a word as the two integers u - z in T.
template <typename T> __device__ __forceinline__ uint32_t int_pair(uint32_t word, int p, uint32_t zz, Bits k) {
    uint32_t m;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(word >> (4 * p)), "r"(k.mask), "r"(k.magic));
    return bits2(__hsub2(as2<T>(m), as2<T>(zz)));
}

}  // namespace w4
}  // namespace llmc
