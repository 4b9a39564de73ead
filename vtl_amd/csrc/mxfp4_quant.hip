// f32 rows into microscaled 4-bit codes and back (gfx950).
#include "mxfp4.hpp"

using namespace vtlhip;
using namespace vtlhip::mx;

namespace {

// Both kernels are bound by memory: 4 bytes a value on one side, 17 / 32 on the other.  A wave has a chunk at a time, a lane four
// consecutive values, so that a wave's access to f32 rows is 1 KiB in one piece and to codes 128 bytes; eight lanes are a block.
constexpr int kThreads = 256, kWaves = kThreads / kWave;

struct Args {
    const float *x;
    float *out;
    uint8_t *codes, *scales;
    int64_t stride;             // of x or out
    unsigned chunks, per_row;   // of all rows, of one
    int cols;
    unsigned waves;
};

template <bool VEC>
__device__ __forceinline__ v4f load_four(const float *row, int col, int cols)
{
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (VEC) {
        if (col < cols)
            v = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(row + col));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (col + i < cols)
                v[i] = row[col + i];
    }
    return v;
}

// The largest over the eight lanes of a block: over quads, then with the other quad of the half row.
__device__ __forceinline__ unsigned block_max_bits(v4f v)
{
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));    // quad_perm [1,0,3,2]
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));    // quad_perm [2,3,0,1]
    return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));  // row_half_mirror
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_mxfp4_kernel(const Args a)
{
    const unsigned lane = threadIdx.x % kWave;
    for (unsigned c = blockIdx.x * kWaves + threadIdx.x / kWave; c < a.chunks; c += a.waves) {
        const unsigned row = c / a.per_row, col = (c % a.per_row) * kChunk + 4 * lane;
        v4f v = load_four<VEC>(a.x + (int64_t)row * a.stride, (int)col, a.cols);
        const unsigned byte = scale_byte(block_max_bits(v));
        float s = scale_of(byte);
        if (byte == 255) {
            v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            s = 1.0f;
        }
        // to the nearest code, to the even one of two, 6 at most
        unsigned q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
        reinterpret_cast<uint16_t *>(a.codes + (size_t)c * kChunkCodes)[lane] = (uint16_t)q;
        if (lane % 8 == 0)
            a.scales[(size_t)c * kChunkScales + lane / 8] = (uint8_t)byte;
    }
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void dequantize_mxfp4_kernel(const Args a)
{
    const unsigned lane = threadIdx.x % kWave;
    for (unsigned c = blockIdx.x * kWaves + threadIdx.x / kWave; c < a.chunks; c += a.waves) {
        const unsigned row = c / a.per_row;
        const int col = (int)((c % a.per_row) * kChunk + 4 * lane);
        const unsigned q = reinterpret_cast<const uint16_t *>(a.codes + (size_t)c * kChunkCodes)[lane];
        const float s = scale_of(a.scales[(size_t)c * kChunkScales + lane / 8]);
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1);
        const v4f v = {lo[0], lo[1], hi[0], hi[1]};
        float *const out = a.out + (int64_t)row * a.stride + col;
        if constexpr (VEC) {
            if (col < a.cols)
                __builtin_nontemporal_store(v, reinterpret_cast<v4f *>(out));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (col + i < a.cols)
                    out[i] = v[i];
        }
    }
}

bool in_vectors(const void *p, int64_t stride, int cols) { return cols % 4 == 0 && stride % 4 == 0 && !(reinterpret_cast<uintptr_t>(p) & 15); }

// Sizes that both ways share.  Chunks are counted in 32 bits: more would be terabytes of f32.
int sizes(int64_t rows, int64_t cols, int64_t stride, Args &a)
{
    if (rows < 0 || cols < 0 || stride < cols)
        return VTL_HIP_ERR_INVALID_ARG;
    if (cols > kMostCols || rows > INT32_MAX || rows * (int64_t)chunks_of((int)cols) > INT32_MAX)
        return VTL_HIP_ERR_UNSUPPORTED;
    a.stride = stride;
    a.cols = (int)cols;
    a.per_row = (unsigned)chunks_of((int)cols);
    a.chunks = (unsigned)rows * a.per_row;
    return VTL_HIP_OK;
}

unsigned grid_of(Args &a)
{
    const unsigned blocks = std::min((a.chunks + kWaves - 1) / kWaves, 1u << 20);
    a.waves = blocks * kWaves;
    return blocks;
}

int quantize(Args a, hipStream_t st)
{
    const unsigned blocks = grid_of(a);
    hipLaunchKernelGGL(in_vectors(a.x, a.stride, a.cols) ? quantize_mxfp4_kernel<true> : quantize_mxfp4_kernel<false>, dim3(blocks), dim3(kThreads), 0, st, a);
    return check_launch("quantize_mxfp4_kernel");
}

}  // namespace

namespace vtlhip {
namespace mx {

int launch_quantize(const float *x, int64_t x_stride, int64_t rows, int cols, uint8_t *codes, uint8_t *scales, hipStream_t st)
{
    Args a{};
    const int rc = sizes(rows, cols, x_stride, a);
    if (rc != VTL_HIP_OK || a.chunks == 0)
        return rc;
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    return quantize(a, st);
}

}  // namespace mx
}  // namespace vtlhip

extern "C" {

int vtl_hip_mxfp4_padded_row(int cols) { return cols <= 0 || cols > kMostCols ? 0 : chunks_of(cols) * kChunk; }

int vtl_hip_quantize_f32_mxfp4(const float *x, int64_t x_stride, int64_t rows, int64_t cols, uint8_t *codes, uint8_t *scales)
{
    Args a{};
    const int rc = sizes(rows, cols, x_stride, a);
    if (rc != VTL_HIP_OK || a.chunks == 0)
        return rc;
    if (!x || !codes || !scales || !rows_aligned(codes, scales))
        return VTL_HIP_ERR_INVALID_ARG;
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    return quantize(a, current_stream());
}

int vtl_hip_dequantize_mxfp4_f32(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, float *x, int64_t x_stride)
{
    Args a{};
    const int rc = sizes(rows, cols, x_stride, a);
    if (rc != VTL_HIP_OK || a.chunks == 0)
        return rc;
    if (!x || !codes || !scales || !rows_aligned(codes, scales))
        return VTL_HIP_ERR_INVALID_ARG;
    a.out = x;
    a.codes = const_cast<uint8_t *>(codes);
    a.scales = const_cast<uint8_t *>(scales);
    const unsigned blocks = grid_of(a);
    hipLaunchKernelGGL(in_vectors(x, x_stride, a.cols) ? dequantize_mxfp4_kernel<true> : dequantize_mxfp4_kernel<false>, dim3(blocks), dim3(kThreads), 0,
                       current_stream(), a);
    return check_launch("dequantize_mxfp4_kernel");
}

}  // extern "C"
