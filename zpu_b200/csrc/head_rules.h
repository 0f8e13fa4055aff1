// Sizes that the language-model head's kernels go by, free of CUDA so that a
// host program can walk through them.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define ZC_RULE __host__ __device__ inline
#else
#define ZC_RULE inline
#endif

namespace zc {

// ---- the 8-bit product of one or two tokens (int8.cu)
constexpr int GV_WARPS = 16, GV_SLOTS = 2, GV_SLOT = 4096, GV_ROWS = 8, GV_CHANNELS = 512;
constexpr int GV_RING = GV_WARPS * GV_SLOTS * GV_SLOT, GV_X = 64 * 1024;  // shared memory: weights, tokens

struct VecUnits {
    int per;        // channels of a block's round
    int seg, segs;  // bytes of a piece, pieces of a row
    int rows;       // rows of a unit (1 where a row has several pieces)
};
// Bytes of a token's row in shared memory.
ZC_RULE int vec_pitch(int k) { return (k + 511) / 512 * 512; }
inline size_t vec_smem(int m, int k) { return GV_RING + (size_t)m * vec_pitch(k); }
inline VecUnits vec_units(int64_t n, int k, int sms) {
    VecUnits U;
    U.seg = k >= GV_SLOT ? GV_SLOT : (k + 15) / 16 * 16;
    U.segs = (k + U.seg - 1) / U.seg;
    U.rows = U.segs > 1 ? 1 : GV_SLOT / U.seg < GV_ROWS ? GV_SLOT / U.seg : GV_ROWS;
    const int64_t per = (n + sms - 1) / sms;
    U.per = (int)(per > GV_CHANNELS ? GV_CHANNELS : per);
    // fewer rows a unit while a block has fewer units than warps
    while (U.rows > 1 && (U.per + U.rows - 1) / U.rows < GV_WARPS) U.rows--;
    return U;
}
// Rows are worked on four at a time; where a unit of `rows` has no such row, its last one is read again.
ZC_RULE int vec_row(int row, int rows) { return row < rows ? row : rows - 1; }

// ---- a block (cluster) a row (distill.cu)
// Rows along y and z of a grid, each at most 65535, with less than z places too many (1 <= rows < 2^31).
struct RowGrid {
    unsigned y, z;
};
inline RowGrid row_grid(int64_t rows) {
    const int64_t z = (rows + 65534) / 65535;
    return {(unsigned)((rows + z - 1) / z), (unsigned)z};
}

// ---- rows on their way to shared memory (head.cuh)
// Whether the 16 aligned bytes in which a row begins begin before its matrix: the row starts `skew` elements into them, and
// `before` elements of the matrix (row * pitch) lie before it.  With short rows that is so for more than the first.
ZC_RULE bool begins_outside(int64_t before, int skew) { return before < skew; }

// ---- the next token (sample.cu)
// floor(2^40 e) from the bits of e, 0 <= e <= 1: the significand shifted into place.  Below 2^-40 nothing is left of it; how far
// it would be shifted there passes 64 bits, which C++ does not define.
ZC_RULE uint64_t weigh_bits(uint32_t u) {
    const uint32_t down = 127u - (u >> 23);
    return ((uint64_t)((u & 0x7fffffu) | 0x800000u) << 17) >> (down < 63u ? down : 63u);
}

}  // namespace zc
