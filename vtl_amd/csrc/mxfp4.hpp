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

inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
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

// Between the last product and anything else that reads or writes results: a 16x16x128 product with an 8-bit operand and a 32x32x64 product of 4-bit ones take 12
// wait states until then, a 16x16x128 product of 4-bit ones 8.  The compiler puts them in where it sees a way from one to the other, but of two ways around conditional code
// between them it once looked at the longer only: a lane's first register was read too early there.  Without an operand, and with nothing moved
// past it: of results in accumulation registers the copy into a vector register is the read, and would come in front of a wait that names the copy.
__device__ __forceinline__ void settle()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int N>
__device__ __forceinline__ void wait_vmcnt()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Weights that a wave reads once, for the products of few rows: FRAGS times 16 rows, a unit of 512 values at a time, straight into shared memory
// of its own, from where they are read as the 16x16x128 product takes them.  By way of shared memory because of how memory is read: a load that gives
// the matrix unit its operand directly has 64 bytes of each of 16 rows, this one 256 bytes of each of 4.
constexpr int kUnit = 2 * kChunk, kUnitSteps = kUnit / 128;
// PAST: past the caches, for weights that none of them holds until the next call (reading 218 MB that way 33.2 us, 6.6 TB/s, else 37.2; but 31 MB that are read over and
// over 8.5 for 7.9).
template <int FRAGS, bool PAST = false>
struct Stream {
    static constexpr int kCodes = 16 * kUnit / 2, kFrag = kCodes + 16 * (kUnit / kBlock), kSlot = FRAGS * kFrag;
    static constexpr int kLoads = 5 * FRAGS;        // of a unit

    // Row `row` of a fragment lies at rows of 256 bytes; 16-byte piece i of it at place i ^ row, so that a read of 16 rows meets all banks.
    const uint8_t *codes[FRAGS], *scales[FRAGS];    // the fragment's first row
    unsigned code_at[FRAGS][4], scale_at[FRAGS];    // the lane's rows
    unsigned pitch, spitch;

    // Fragment f has rows first[f] .. first[f] + 15 of w; rows from `most` of them on are not read (the last one is, instead).
    __device__ __forceinline__ void rows(int f, const Rows &w, size_t first, int most, int chunks)
    {
        const int lane = threadIdx.x % kWave;
        pitch = (unsigned)chunks * kChunkCodes;
        spitch = (unsigned)chunks * kChunkScales;
        codes[f] = w.codes + first * pitch;
        scales[f] = w.scales + first * spitch;
#pragma unroll
        for (int j = 0; j < 4; j++)
            code_at[f][j] = (unsigned)min(4 * j + lane / 16, most - 1) * pitch;
        scale_at[f] = (unsigned)min(lane / 4, most - 1) * spitch;
    }
    // The loads of a unit.  Where a row has only the first half of it, the rest is the row's end once more.  (Buffer loads: behind global ones into
    // shared memory the compiler takes loads into registers to arrive in any order, and waits for all that there are.)
    __device__ __forceinline__ void issue(int unit, char *slot) const
    {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int f = 0; f < FRAGS; f++) {
            const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(codes[f]), 0, (int)(16u * pitch), 0x00027000);
            const __amdgpu_buffer_rsrc_t scales_from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(scales[f]), 0, (int)(16u * spitch), 0x00027000);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned in_row = min((unsigned)unit * (kUnit / 2) + (unsigned)((lane % 16) ^ (4 * j + lane / 16)) * 16u, pitch - 16u);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(from, VTL_LPTR(slot + f * kFrag + j * 1024), 16, (int)(code_at[f][j] + in_row), 0, 0, PAST ? 2 : 0);
            }
            const unsigned in_row = min((unsigned)unit * (kUnit / kBlock) + (unsigned)(lane % 4) * 4u, spitch - 4u);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(scales_from, VTL_LPTR(slot + f * kFrag + kCodes), 4, (int)(scale_at[f] + in_row), 0, 0, 0);
        }
    }
    __device__ __forceinline__ static v4i operand(const char *slot, int f, int step)
    {
        const int lane = threadIdx.x % kWave, r = lane % 16, q = lane / 16;
        return *reinterpret_cast<const v4i *>(slot + f * kFrag + r * (kUnit / 2) + (((4 * step + q) ^ r) << 4));
    }
    // The scale bytes of all steps: byte 0 of each.
    __device__ __forceinline__ static v4i all_scales(const char *slot, int f)
    {
        const int lane = threadIdx.x % kWave, r = lane % 16, q = lane / 16;
        v4i v = *reinterpret_cast<const v4i *>(slot + f * kFrag + kCodes + r * 16);
#pragma unroll
        for (int s = 0; s < 4; s++)
            v[s] = (int)((unsigned)v[s] >> (8 * q));
        return v;
    }
    // What is read of a slot is in registers before the slot is filled again.
    __device__ __forceinline__ static void done_reading() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
};
#endif

}  // namespace mx
}  // namespace vtlhip
