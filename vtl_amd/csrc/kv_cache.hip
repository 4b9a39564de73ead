// The int8 key/value cache for gfx950: rows of new tokens quantized into their pages, and rows back as f32.
// The arithmetic is that of the row quantizer and of the dequantizer (quant.hip), one row for each token and head.
#include "kv_cache.hpp"
#include "quant_device.hpp"

using namespace vtlhip;
using namespace vtlhip::qdev;

namespace {

// A wave for each row, head and half (keys, values).
__global__ __launch_bounds__(256) void kv_write_kernel(Kv kv, const float *__restrict__ k, int64_t k_stride, const float *__restrict__ v,
                                                       int64_t v_stride, unsigned units)
{
    const unsigned unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (unit >= units)
        return;
    const int lane = threadIdx.x & 63;
    const bool values = unit & 1;
    const int head = (unit >> 1) % (unsigned)kv.kv_heads, row = (unit >> 1) / (unsigned)kv.kv_heads;
    int b, position;
    if (!kv_row(kv, row, b, position) || position < 0)
        return;
    unsigned at;
    char *const page = kv_group(kv, b, (unsigned)position / kKvGroup, head, at);
    if (!page)
        return;
    const float *x = values ? v + row * v_stride : k + row * k_stride;
    x += head * kv.head_dim;
    float most = 0.0f, mine[kKvMostDim / 64];
#pragma unroll
    for (int i = 0; i < kKvMostDim / 64; i++) {
        const int d = lane + 64 * i;
        mine[i] = d < kv.head_dim ? x[d] : 0.0f;
        most = fmaxf(most, fabsf(mine[i]));
    }
    most = wave_max(most);
    const QuantScale p = make_quant_scale(most / 127.0f);
    const unsigned slot = at * kKvGroup + (unsigned)position % kKvGroup;
#pragma unroll
    for (int i = 0; i < kKvMostDim / 64; i++) {
        const int d = lane + 64 * i;
        if (d < kv.padded)
            page[values ? kv_value_at(kv, at, d) + position % kKvGroup : kv_key_at(kv, d / 16, slot) + d % 16] = (char)quant_code(mine[i], p);
    }
    if (lane == 0)
        reinterpret_cast<float *>(page + kv_scales_at(kv))[slot + (values ? kv.page_size : 0)] = p.scale;
}

__global__ __launch_bounds__(256) void kv_read_kernel(Kv kv, float *__restrict__ k, int64_t k_stride, float *__restrict__ v, int64_t v_stride,
                                                      unsigned units)
{
    const unsigned unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (unit >= units)
        return;
    const int lane = threadIdx.x & 63;
    const bool values = unit & 1;
    const int head = (unit >> 1) % (unsigned)kv.kv_heads, row = (unit >> 1) / (unsigned)kv.kv_heads;
    int b, position;
    if (!(values ? v : k) || !kv_row(kv, row, b, position))
        return;
    unsigned at = 0;
    const char *const page = position < 0 ? nullptr : kv_group(kv, b, (unsigned)position / kKvGroup, head, at);
    float *x = values ? v + row * v_stride : k + row * k_stride;
    x += head * kv.head_dim;
    const unsigned slot = at * kKvGroup + (unsigned)position % kKvGroup;
    const float scale = page ? reinterpret_cast<const float *>(page + kv_scales_at(kv))[slot + (values ? kv.page_size : 0)] : 0.0f;
    for (int d = lane; d < kv.head_dim; d += 64) {
        float y = 0.0f;
        if (page)
            y = (float)(int8_t)page[values ? kv_value_at(kv, at, d) + position % kKvGroup : kv_key_at(kv, d / 16, slot) + d % 16] * scale;
        x[d] = y;
    }
}

}  // namespace

extern "C" {

size_t vtl_hip_kv_cache_bytes(int num_pages, int page_size, int kv_heads, int head_dim)
{
    if (num_pages < 1 || page_size < kKvGroup || page_size > kKvMostPage || page_size % kKvGroup || kv_heads < 1 || head_dim < 1 ||
        head_dim > kKvMostDim)
        return 0;
    const size_t page = (size_t)page_size * (2u * ((head_dim + 15) & ~15) + 8u) * (size_t)kv_heads;
    if (page >> 32)
        return 0;
    return page * (size_t)num_pages;
}

int vtl_hip_kv_write_f32(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, const float *k, int64_t k_stride, const float *v,
                         int64_t v_stride)
{
    Kv kv;
    const int st = kv_sizes(cache, batch, kv);
    if (st != VTL_HIP_OK)
        return st;
    if (!kv_stride_ok(kv, kv.kv_heads, k_stride) || !kv_stride_ok(kv, kv.kv_heads, v_stride))
        return VTL_HIP_ERR_INVALID_ARG;
    if (kv.rows == 0 || kv.batch == 0)
        return VTL_HIP_OK;
    if (!k || !v)
        return VTL_HIP_ERR_INVALID_ARG;
    const int64_t units = (int64_t)kv.rows * kv.kv_heads * 2;
    if (units > 0x7fffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kv_write_kernel, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, current_stream(), kv, k, k_stride, v, v_stride,
                       (unsigned)units);
    return check_launch("kv_write_kernel");
}

int vtl_hip_kv_read_f32(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, float *k, int64_t k_stride, float *v, int64_t v_stride)
{
    Kv kv;
    const int st = kv_sizes(cache, batch, kv);
    if (st != VTL_HIP_OK)
        return st;
    if ((k && !kv_stride_ok(kv, kv.kv_heads, k_stride)) || (v && !kv_stride_ok(kv, kv.kv_heads, v_stride)))
        return VTL_HIP_ERR_INVALID_ARG;
    if (kv.rows == 0 || kv.batch == 0 || (!k && !v))
        return VTL_HIP_OK;
    const int64_t units = (int64_t)kv.rows * kv.kv_heads * 2;
    if (units > 0x7fffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, current_stream(), kv, k, k_stride, v, v_stride,
                       (unsigned)units);
    return check_launch("kv_read_kernel");
}

}  // extern "C"
