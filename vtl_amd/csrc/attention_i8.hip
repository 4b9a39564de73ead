// Attention over the int8 key/value cache for gfx950.
//
//   s_j = scale * sum_d q_d K_jd sk_j,   w = softmax over the tokens that the row sees,   o_d = sum_j w_j sv_j V_jd
#include "kv_cache.hpp"
#include "quant_device.hpp"

using namespace vtlhip;
using namespace vtlhip::qdev;

namespace {

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int i = 32; i; i >>= 1)
        v += __shfl_xor(v, i);
    return v;
}

// A wave for each row and head: 64 tokens at a time, a token a lane for the scores and a dimension a lane for the values, with
// the running maximum and sum.
__global__ __launch_bounds__(256) void attention_rows_kernel(Kv kv, const float *__restrict__ q, int64_t q_stride, int heads, float scale,
                                                             int causal, float *__restrict__ out, int64_t out_stride, unsigned units)
{
    __shared__ float q_of[4][kKvMostDim], p_of[4][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + w);
    if (unit >= units)
        return;
    const int head = unit % (unsigned)heads, row = unit / (unsigned)heads, kv_head = head / (heads / kv.kv_heads);
    int b, position;
    if (!kv_row(kv, row, b, position))
        return;
    const int length = kv_length(kv, b), seen = causal ? min(position + 1, length) : length;
    const float *x = q + row * q_stride + head * kv.head_dim;
    for (int d = lane; d < kv.padded; d += 64)
        q_of[w][d] = d < kv.head_dim ? x[d] * scale : 0.0f;
    float top = -INFINITY, sum = 0.0f, o[kKvMostDim / 64] = {};
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int j = j0 + lane;
        unsigned at;
        const char *page = j < seen ? kv_group(kv, b, (unsigned)j / 16, kv_head, at) : nullptr;
        float s = -INFINITY, sv = 0.0f;
        if (page) {
            const unsigned slot = at * 16 + j % 16;
            float dot = 0.0f;
            for (int c = 0; c < kv.padded / 16; c++) {
                const int4_t codes = *reinterpret_cast<const int4_t *>(page + kv_key_at(kv, c, slot));
                for (int i = 0; i < 16; i++)
                    dot = __builtin_fmaf((float)(int8_t)(codes[i / 4] >> (8 * (i % 4))), q_of[w][16 * c + i], dot);
            }
            const float *scales = reinterpret_cast<const float *>(page + kv_scales_at(kv));
            s = dot * scales[slot];
            sv = scales[slot + kv.page_size];
        }
        float most = s;
        for (int i = 32; i; i >>= 1)
            most = fmaxf(most, __shfl_xor(most, i));
        const float now = fmaxf(top, most), keep = top == now ? 1.0f : expf(top - now);
        const float p = page ? expf(s - now) : 0.0f;
        top = now;
        sum = sum * keep + wave_sum(p);
        p_of[w][lane] = page ? p * sv : 0.0f;
        for (int i = 0; i < kKvMostDim / 64; i++)
            o[i] *= keep;
        for (int g = 0; g < 4 && j0 + 16 * g < seen; g++) {
            unsigned place;
            const char *from = kv_group(kv, b, (unsigned)j0 / 16 + g, kv_head, place);
            if (!from)
                continue;
            for (int i = 0; i < kKvMostDim / 64; i++) {
                const int d = lane + 64 * i;
                if (d < kv.head_dim) {
                    const int4_t codes = *reinterpret_cast<const int4_t *>(from + kv_value_at(kv, place, d));
                    for (int t = 0; t < 16; t++)
                        o[i] = __builtin_fmaf((float)(int8_t)(codes[t / 4] >> (8 * (t % 4))), p_of[w][16 * g + t], o[i]);
                }
            }
        }
    }
    float *y = out + row * out_stride + head * kv.head_dim;
    for (int i = 0; i < kKvMostDim / 64; i++) {
        const int d = lane + 64 * i;
        if (d < kv.head_dim)
            y[d] = sum == 0.0f ? 0.0f : o[i] / sum;
    }
}

}  // namespace

extern "C" {

size_t vtl_hip_attention_i8_workspace(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, int heads)
{
    (void)cache, (void)batch, (void)heads;
    return 0;
}

int vtl_hip_attention_i8_f32(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, const float *q, int64_t q_stride, int heads,
                             float scale, int causal, float *out, int64_t out_stride, void *workspace, size_t workspace_bytes)
{
    (void)workspace, (void)workspace_bytes;
    Kv kv;
    const int st = kv_sizes(cache, batch, kv);
    if (st != VTL_HIP_OK)
        return st;
    if (heads < 1 || heads % kv.kv_heads || !kv_stride_ok(kv, heads, q_stride) || !kv_stride_ok(kv, heads, out_stride))
        return VTL_HIP_ERR_INVALID_ARG;
    if (kv.rows == 0 || kv.batch == 0)
        return VTL_HIP_OK;
    if (!q || !out || meet(q, kv_span(kv, heads, q_stride), out, kv_span(kv, heads, out_stride)))
        return VTL_HIP_ERR_INVALID_ARG;
    const int64_t units = (int64_t)kv.rows * heads;
    if (units > 0x7fffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(attention_rows_kernel, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, current_stream(), kv, q, q_stride, heads, scale,
                       causal, out, out_stride, (unsigned)units);
    return check_launch("attention_rows_kernel");
}

}  // extern "C"
