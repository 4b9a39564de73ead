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

// U chunks of a wave at once, one behind the other: as many loads are on their way.
template <bool VEC, int U>
__global__ __launch_bounds__(kThreads) void quantize_mxfp4_kernel(const Args a)
{
    const unsigned lane = threadIdx.x % kWave;
    for (unsigned first = U * (blockIdx.x * kWaves + threadIdx.x / kWave); first < a.chunks; first += U * a.waves) {
        v4f v[U];
        unsigned row = first / a.per_row, in_row = first % a.per_row;
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (first + u < a.chunks)
                v[u] = load_four<VEC>(a.x + (int64_t)row * a.stride, (int)(in_row * kChunk + 4 * lane), a.cols);
            if (++in_row == a.per_row) {
                in_row = 0;
                row++;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t c = first + u;
            if (c >= a.chunks)
                break;
            const unsigned byte = scale_byte(block_max_bits(v[u]));
            float s = scale_of(byte);
            if (byte == 255) {
                v[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                s = 1.0f;
            }
            // to the nearest code, to the even one of two, 6 at most
            unsigned q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[u][0], v[u][1], s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[u][2], v[u][3], s, 1);
            reinterpret_cast<uint16_t *>(a.codes + c * kChunkCodes)[lane] = (uint16_t)q;
            if (lane % 8 == 0)
                a.scales[c * kChunkScales + lane / 8] = (uint8_t)byte;
        }
    }
}

template <bool VEC, int U>
__global__ __launch_bounds__(kThreads) void dequantize_mxfp4_kernel(const Args a)
{
    const unsigned lane = threadIdx.x % kWave;
    for (unsigned first = U * (blockIdx.x * kWaves + threadIdx.x / kWave); first < a.chunks; first += U * a.waves) {
        unsigned q[U], byte[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t c = min(first + u, a.chunks - 1);
            q[u] = reinterpret_cast<const uint16_t *>(a.codes + c * kChunkCodes)[lane];
            byte[u] = a.scales[c * kChunkScales + lane / 8];
        }
        unsigned row = first / a.per_row, in_row = first % a.per_row;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (first + u >= a.chunks)
                break;
            const float s = scale_of(byte[u]);
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], s, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[u], s, 1);
            const v4f v = {lo[0], lo[1], hi[0], hi[1]};
            const int col = (int)(in_row * kChunk + 4 * lane);
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
            if (++in_row == a.per_row) {
                in_row = 0;
                row++;
            }
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

// Whether one side's memory is the other's: waves read and write chunks in no order.
bool shared(const Args &a, const float *x, const uint8_t *codes, const uint8_t *scales)
{
    const size_t rows = a.chunks / a.per_row, bytes = ((rows - 1) * (size_t)a.stride + (size_t)a.cols) * sizeof(float);
    return meet(x, bytes, codes, (size_t)a.chunks * kChunkCodes) || meet(x, bytes, scales, (size_t)a.chunks * kChunkScales);
}

// Chunks of a wave at once, one where there are not enough of them for all compute units' waves.  (14336 x 4096 f32 into codes with 1 / 2 / 4 / 8
// at once: 51.7 / 45.6 / 43.7 / 43.0 us, 6.1 TB/s; back 37.3 / 37.7 / 38.8 / 41.8; 16384 x 16384 213 / 196 / 195 / 195 and 223 / 200 / 203 / 217.)
constexpr int kQuantizeAtOnce = 4, kDequantizeAtOnce = 2;
constexpr unsigned kSeveral = 8192;     // waves

template <int U>
unsigned grid_of(Args &a, bool &several)
{
    several = a.chunks >= U * kSeveral;
    const unsigned units = several ? (a.chunks + U - 1) / U : a.chunks, blocks = std::min((units + kWaves - 1) / kWaves, 1u << 20);
    a.waves = blocks * kWaves;
    return blocks;
}

int quantize(Args a, hipStream_t st)
{
    constexpr int kAtOnce = kQuantizeAtOnce;
    bool several;
    const unsigned blocks = grid_of<kAtOnce>(a, several);
    const auto one = in_vectors(a.x, a.stride, a.cols) ? quantize_mxfp4_kernel<true, 1> : quantize_mxfp4_kernel<false, 1>;
    const auto more = in_vectors(a.x, a.stride, a.cols) ? quantize_mxfp4_kernel<true, kAtOnce> : quantize_mxfp4_kernel<false, kAtOnce>;
    hipLaunchKernelGGL(several ? more : one, dim3(blocks), dim3(kThreads), 0, st, a);
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
    if (shared(a, x, codes, scales))
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
    if (shared(a, x, codes, scales))
        return VTL_HIP_ERR_INVALID_ARG;
    a.out = x;
    a.codes = const_cast<uint8_t *>(codes);
    a.scales = const_cast<uint8_t *>(scales);
    constexpr int kAtOnce = kDequantizeAtOnce;
    bool several;
    const unsigned blocks = grid_of<kAtOnce>(a, several);
    const auto one = in_vectors(x, x_stride, a.cols) ? dequantize_mxfp4_kernel<true, 1> : dequantize_mxfp4_kernel<false, 1>;
    const auto more = in_vectors(x, x_stride, a.cols) ? dequantize_mxfp4_kernel<true, kAtOnce> : dequantize_mxfp4_kernel<false, kAtOnce>;
    hipLaunchKernelGGL(several ? more : one, dim3(blocks), dim3(kThreads), 0, current_stream(), a);
    return check_launch("dequantize_mxfp4_kernel");
}

}  // extern "C"
