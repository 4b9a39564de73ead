// Microscaled 4-bit floating point (gfx950): what the kernels for it share.
//
// A block is 32 consecutive values of a row: 4-bit codes (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign in bit 3) and one scale, a byte
// b for 2^(b - 127), 255 for no number.  Rows are padded to whole chunks of 256 values, so a chunk is 128 bytes of codes, a cache line, and
// 8 bytes of scales, both aligned, and no kernel has a tail along a row: codes and scales behind the end are zeros, which add nothing.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace vtlhip {
namespace mx {

constexpr int kBlock = 32, kChunk = 256;
constexpr int kChunkCodes = kChunk / 2, kChunkScales = kChunk / kBlock;   // bytes
constexpr int kMostCols = 1 << 24;                                       // a tile's rows stay within 32 bits of bytes

inline int chunks_of(int cols) { return (cols + kChunk - 1) / kChunk; }

// Rows of codes and scales.
struct Rows {
    const uint8_t *codes, *scales;
};

// Codes are read in vectors of 16 bytes, scales of 8.
inline bool rows_aligned(const void *codes, const void *scales)
{
    return !(reinterpret_cast<uintptr_t>(codes) & 15) && !(reinterpret_cast<uintptr_t>(scales) & 7);
}

int launch_quantize(const float *x, int64_t x_stride, int64_t rows, int cols, uint8_t *codes, uint8_t *scales, hipStream_t st);

#ifdef __HIPCC__
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has these bits: 2^(floor(log2 max) - 2), so that the largest code's binade is the
// block's.  A block with an infinity or NaN is no number as a whole.
__device__ __forceinline__ unsigned scale_byte(unsigned max_bits)
{
    return max_bits >= 0x7f800000u ? 255u : (unsigned)max((int)(max_bits >> 23) - 2, 0);
}

// What the conversion instructions take for a scale: an f32 whose exponent field is the byte (0 there is 2^-127 too, 255 no number).
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// The 16x16x128 product of 4-bit operands, each lane's own block and scale (the low byte of sa and sb).  Block sums are exact in the
// matrix unit (at most 32 products of at most 8 bits and a half), and are added to the f32 accumulator with one rounding.
__device__ __forceinline__ v4f mfma_16(v4i a, v4i b, v4f c, int sa, int sb)
{
    const v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, sa, 0, sb);
}
#endif

}  // namespace mx
}  // namespace vtlhip
