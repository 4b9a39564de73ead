// The int8 key/value cache for gfx950: rows of new tokens quantized into their pages, and rows back as f32.
// The arithmetic is that of the row quantizer and of the dequantizer (quant.hip), one row for each token and head.
#include "kv_cache.hpp"
#include "quant_device.hpp"

using namespace vtlhip;
using namespace vtlhip::qdev;

namespace {

// Both kernels are bound by memory: 4 D bytes of f32 and D + 4 of codes and scale for each token, head and half (keys, values).
//
// The unit is the 16 tokens of a group of one sequence that lie together in its page, or those of them that are the call's; SEG lanes (16, 32 or 64,
// four dimensions each) have an item: four of the tokens (all 16 where they are all written), of one head, of one half.  So f32 rows move in vectors of
// 16 bytes, SEG of them side by side, and codes of values, whose tokens lie together, are put in order in registers.  As many workgroups share a group as
// its items fill once: several rounds in one workgroup were slower (6 ragged sequences of up to 5001 tokens, 8 heads of 128, read in 1 / 2 / 4 / 8 rounds:
// 54 / 55 / 60 / 68 us).  Results are written past the caches (there 54 -> 36 us, 6.3 TB/s).  2 x 8192 tokens: written in 40 us (4.2 TB/s), read back in 27;
// 64 tokens of as many sequences: 4.8 and 4.1 us, which is what a launch with three memory latencies behind each other takes.
struct Rows {
    const float *k, *v;       // read
    float *k_out, *v_out;     // or written
    int64_t k_stride, v_stride;
    int vectors;              // whether rows of both may be moved in vectors of 16 bytes
    int groups;               // of 16 tokens that a sequence of the call touches at most, as far as the host knows
    int parts;                // workgroups that share a group's items
};

// The tokens of a group that are the call's, and where their rows are.
struct Group {
    int b, first_row;         // the row of token 0 of the group, were it one of the call's
    int low, high;            // tokens low .. high - 1 of the group
    unsigned at;
    char *page0;              // head 0 of its page; nullptr: there is no such page
};

// Group number `i` of those that the call has in sequence b; false: there are no more.
__device__ __forceinline__ bool group_of(const Kv &kv, int b, int i, Group &g)
{
    int length, first, count;
    kv_sequence(kv, b, length, first, count);
    const int start = length - count;                       // below 0: rows in front of the first token
    const int base = (start >> 4) * kKvGroup + i * kKvGroup;
    if (base >= length)
        return false;
    g.b = b;
    g.low = max(start - base, 0);
    g.high = min(length - base, kKvGroup);
    g.first_row = first + base - start;
    g.page0 = base < 0 ? nullptr : kv_group(kv, b, (unsigned)base / kKvGroup, 0, g.at);
    return true;
}

// Four dimensions of a row from d on; zeros behind the last.
__device__ __forceinline__ float4_t load_four(const float *x, int d, int dims, int vectors)
{
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (vectors) {
        if (d < dims)
            v = __builtin_nontemporal_load(reinterpret_cast<const float4_t *>(x + d));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (d + i < dims)
                v[i] = x[d + i];
    }
    return v;
}
__device__ __forceinline__ void store_four(float *x, int d, int dims, int vectors, float4_t v)
{
    if (vectors) {
        if (d < dims)
            __builtin_nontemporal_store(v, reinterpret_cast<float4_t *>(x + d));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (d + i < dims)
                x[d + i] = v[i];
    }
}

// Byte j of word i becomes byte i of word j.
__device__ __forceinline__ void transpose_bytes(unsigned (&w)[4])
{
    const unsigned a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
    const unsigned c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302);
}

// Lane i of four gets word i of each: word j of lane i becomes word i of lane j.
__device__ __forceinline__ void transpose_words(unsigned (&w)[4])
{
    const int lane = threadIdx.x;
    unsigned x[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {      // with the neighbour
        const unsigned give = lane & 1 ? w[i] : w[i + 1];
        const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)give, 0xB1, 0xF, 0xF, false);
        x[i] = lane & 1 ? got : w[i];
        x[i + 1] = lane & 1 ? w[i + 1] : got;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {         // and with the one behind it
        const unsigned give = lane & 2 ? x[i] : x[i + 2];
        const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)give, 0x4E, 0xF, 0xF, false);
        w[i] = lane & 2 ? got : x[i];
        w[i + 2] = lane & 2 ? x[i + 2] : got;
    }
}

// Groups whose 16 tokens are all new, as a prompt's: an item is all of them, so that the values' codes are written in the 16 bytes that 16 tokens of a
// dimension take; four lanes exchange theirs to write 16 bytes of keys of one token each.
template <int SEG>
__device__ __forceinline__ void write_whole_group(const Kv &kv, const Rows &rows, const Group &g, int item)
{
    const int d = 4 * (threadIdx.x % SEG), head = item >> 1;
    const bool values = item & 1;
    const int64_t stride = values ? rows.v_stride : rows.k_stride;
    const float *x = (values ? rows.v : rows.k) + (int64_t)g.first_row * stride + head * kv.head_dim;
    float4_t four[kKvGroup];
#pragma unroll
    for (int t = 0; t < kKvGroup; t++)
        four[t] = load_four(x + t * stride, d, kv.head_dim, rows.vectors);
    char *const page = g.page0 + (uint64_t)head * kv.head_bytes;
    float *const to = reinterpret_cast<float *>(page + kv_scales_at(kv)) + (values ? kv.page_size : 0) + g.at * kKvGroup;
    unsigned of_values[4][4];      // dimension, four tokens
#pragma unroll
    for (int quad = 0; quad < 4; quad++) {
        unsigned codes[4];
        float4_t scales;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const QuantScale p = make_quant_scale(segment_max<SEG>(absmax4(0.0f, four[4 * quad + t])) / 127.0f);
            codes[t] = quant4(four[4 * quad + t], p);
            scales[t] = p.scale;
        }
        if (d == 0)
            *reinterpret_cast<float4_t *>(to + 4 * quad) = scales;
        if (values) {
            transpose_bytes(codes);
#pragma unroll
            for (int k = 0; k < 4; k++)
                of_values[k][quad] = codes[k];
        } else {
            transpose_words(codes);
            if (d < kv.padded)
                *reinterpret_cast<uint4 *>(page + kv_key_at(kv, d / 16, g.at * kKvGroup + 4 * quad + threadIdx.x % 4)) =
                    make_uint4(codes[0], codes[1], codes[2], codes[3]);
        }
    }
    if (values && d < kv.padded)
#pragma unroll
        for (int k = 0; k < 4; k++)
            *reinterpret_cast<uint4 *>(page + kv_value_at(kv, g.at, d + k)) =
                make_uint4(of_values[k][0], of_values[k][1], of_values[k][2], of_values[k][3]);
}

// Others: an item is up to four tokens.
template <int SEG>
__device__ __forceinline__ void write_quad(const Kv &kv, const Rows &rows, const Group &g, int quad, int head, bool values)
{
    const int d = 4 * (threadIdx.x % SEG), low = g.low - 4 * quad, high = g.high - 4 * quad;
    const int64_t stride = values ? rows.v_stride : rows.k_stride;
    const float *x = (values ? rows.v : rows.k) + (int64_t)(g.first_row + 4 * quad) * stride + head * kv.head_dim;
    float4_t four[4];
#pragma unroll
    for (int t = 0; t < 4; t++)
        four[t] = t >= low && t < high ? load_four(x + t * stride, d, kv.head_dim, rows.vectors) : float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    char *const page = g.page0 + (uint64_t)head * kv.head_bytes;
    float *const to = reinterpret_cast<float *>(page + kv_scales_at(kv)) + (values ? kv.page_size : 0) + g.at * kKvGroup + 4 * quad;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        if (t < low || t >= high)
            continue;
        const QuantScale p = make_quant_scale(segment_max<SEG>(absmax4(0.0f, four[t])) / 127.0f);
        const unsigned codes = quant4(four[t], p);
        if (d == 0)
            to[t] = p.scale;
        if (d < kv.padded) {
            if (!values)
                *reinterpret_cast<unsigned *>(page + kv_key_at(kv, d / 16, g.at * kKvGroup + 4 * quad + t) + d % 16) = codes;
            else
#pragma unroll
                for (int k = 0; k < 4; k++)
                    page[kv_value_at(kv, g.at, d + k) + 4 * quad + t] = (char)(codes >> (8 * k));
        }
    }
}

template <int SEG>
__global__ __launch_bounds__(256, 4) void kv_write_kernel(Kv kv, Rows rows)
{
    const int part = blockIdx.x % (unsigned)rows.parts, unit = blockIdx.x / (unsigned)rows.parts, b = unit / rows.groups;
    Group g;
    for (int i = unit % rows.groups; group_of(kv, b, i, g); i += rows.groups) {
        if (!g.page0)
            continue;
        const bool all = g.low == 0 && g.high == kKvGroup;
        const int quad0 = g.low / 4, quads = all ? 1 : (g.high + 3) / 4 - quad0, items = 2 * quads * kv.kv_heads;
        for (int item = part * (256 / SEG) + threadIdx.x / SEG; item < items; item += rows.parts * (256 / SEG)) {
            if (all)
                write_whole_group<SEG>(kv, rows, g, item);
            else
                write_quad<SEG>(kv, rows, g, quad0 + (item >> 1) % quads, (item >> 1) / quads, item & 1);
        }
    }
}

template <int SEG>
__global__ __launch_bounds__(256) void kv_read_kernel(Kv kv, Rows rows)
{
    const int part = blockIdx.x % (unsigned)rows.parts, unit = blockIdx.x / (unsigned)rows.parts, b = unit / rows.groups;
    Group g;
    for (int i = unit % rows.groups; group_of(kv, b, i, g); i += rows.groups) {
        const int quad0 = g.low / 4, quads = (g.high + 3) / 4 - quad0, items = 2 * quads * kv.kv_heads;
        const int d = 4 * (threadIdx.x % SEG);
        for (int item = part * (256 / SEG) + threadIdx.x / SEG; item < items; item += rows.parts * (256 / SEG)) {
            const bool values = item & 1;
            float *x = values ? rows.v_out : rows.k_out;
            if (!x || d >= kv.head_dim)
                continue;
            const int quad = quad0 + (item >> 1) % quads, head = (item >> 1) / quads;
            const int64_t stride = values ? rows.v_stride : rows.k_stride;
            x += (int64_t)(g.first_row + 4 * quad) * stride + head * kv.head_dim;
            unsigned codes[4] = {0, 0, 0, 0};
            float4_t scales = {0.0f, 0.0f, 0.0f, 0.0f};
            if (g.page0) {
                const char *const page = g.page0 + (uint64_t)head * kv.head_bytes;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    codes[k] = *reinterpret_cast<const unsigned *>(values ? page + kv_value_at(kv, g.at, d + k) + 4 * quad
                                                                          : page + kv_key_at(kv, d / 16, g.at * kKvGroup + 4 * quad + k) + d % 16);
                scales = *reinterpret_cast<const float4_t *>(page + kv_scales_at(kv) +
                                                            4 * ((values ? kv.page_size : 0) + g.at * kKvGroup + 4 * quad));
                if (values)
                    transpose_bytes(codes);
            }
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (4 * quad + t >= g.low && 4 * quad + t < g.high) {
                    float4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (g.page0)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            y[k] = (float)(int8_t)(codes[t] >> (8 * k)) * scales[t];
                    store_four(x + t * stride, d, kv.head_dim, rows.vectors, y);
                }
        }
    }
}

bool in_vectors(const Kv &kv, const void *p, int64_t stride)
{
    return !p || (kv.head_dim % 4 == 0 && stride % 4 == 0 && !(reinterpret_cast<uintptr_t>(p) & 15));
}

// Groups that a sequence of the call touches at most, and the launch of as many workgroups for each sequence.
int grid_of(const Kv &kv, const vtl_hip_kv_batch &b, int items, Rows &rows, unsigned &blocks)
{
    const int64_t most = !kv.starts ? 1 : b.most_rows ? std::min(b.most_rows, kv.rows) : kv.rows;
    rows.groups = kv.starts ? (int)((most + 2 * kKvGroup - 2) / kKvGroup) : 1;
    const int seg = kv.padded <= 64 ? 16 : kv.padded <= 128 ? 32 : 64, at_once = 256 / seg;
    rows.parts = (items + at_once - 1) / at_once;
    const int64_t a_group_each = (int64_t)kv.batch * rows.parts;
    if (a_group_each > 0xffffff)      // workgroups of 256 that a grid may have
        return VTL_HIP_ERR_UNSUPPORTED;
    rows.groups = (int)std::min<int64_t>(rows.groups, std::max<int64_t>(1, kKvMostBlocks / a_group_each));
    const int64_t all = rows.groups * a_group_each;
    blocks = (unsigned)all;
    return VTL_HIP_OK;
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
    Rows rows{k, v, nullptr, nullptr, k_stride, v_stride, in_vectors(kv, k, k_stride) && in_vectors(kv, v, v_stride), 0, 0};
    unsigned blocks;
    const int grid = grid_of(kv, *batch, 2 * kv.kv_heads, rows, blocks);
    if (grid != VTL_HIP_OK)
        return grid;
    hipLaunchKernelGGL(kv.padded <= 64 ? kv_write_kernel<16> : kv.padded <= 128 ? kv_write_kernel<32> : kv_write_kernel<64>, dim3(blocks), dim3(256), 0,
                       current_stream(), kv, rows);
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
    Rows rows{nullptr, nullptr, k, v, k_stride, v_stride, in_vectors(kv, k, k_stride) && in_vectors(kv, v, v_stride), 0, 0};
    unsigned blocks;
    const int grid = grid_of(kv, *batch, 8 * kv.kv_heads, rows, blocks);
    if (grid != VTL_HIP_OK)
        return grid;
    hipLaunchKernelGGL(kv.padded <= 64 ? kv_read_kernel<16> : kv.padded <= 128 ? kv_read_kernel<32> : kv_read_kernel<64>, dim3(blocks), dim3(256), 0,
                       current_stream(), kv, rows);
    return check_launch("kv_read_kernel");
}

}  // extern "C"
