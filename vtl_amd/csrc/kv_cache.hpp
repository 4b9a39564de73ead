// The int8 key/value cache as kernels see it, and the host's checks of a call's arguments (gfx950 only).
#pragma once

#include <algorithm>

#include "common.hpp"

namespace vtlhip {

constexpr int kKvGroup = 16;                  // tokens that lie together for a dimension of the values
constexpr int kKvMostPage = 4096;
constexpr int kKvMostDim = 256;
constexpr int64_t kKvMostTokens = 1 << 28;    // of a sequence
constexpr int kKvMostRows = 1 << 30;          // of a call, and sequences: what is counted past the last one fits 32 bits
constexpr int kKvMostBlocks = 1 << 22;        // of a launch, or one for each sequence and head where those are more; what is behind is theirs too

// A cache and the sequences of a call, by value.
struct Kv {
    char *pages;
    int num_pages, page_size, kv_heads, head_dim;
    int padded;                   // head_dim rounded up to whole groups of 16
    unsigned page_groups;         // groups of 16 tokens in a page
    unsigned magic, one;          // what divides by that (kv_page_of)
    unsigned head_bytes, page_bytes;
    const int32_t *table, *lengths, *starts;
    int batch, max_pages, rows;
    int most_tokens;              // max_pages * page_size, at most kKvMostTokens
};

// VTL_HIP_OK and the sizes, or why they are none.
inline int kv_sizes(const vtl_hip_kv_cache *c, const vtl_hip_kv_batch *b, Kv &kv)
{
    if (!c || !b || !c->pages || (reinterpret_cast<uintptr_t>(c->pages) & 15))
        return VTL_HIP_ERR_INVALID_ARG;
    if (!vtl_hip_kv_cache_bytes(c->num_pages, c->page_size, c->kv_heads, c->head_dim))
        return VTL_HIP_ERR_INVALID_ARG;
    if (b->batch < 0 || b->rows < 0 || b->max_pages < 1 || b->most_rows < 0 || b->most_length < 0)
        return VTL_HIP_ERR_INVALID_ARG;
    if (b->batch > 0 && (!b->page_table || !b->lengths || (!b->starts && b->rows != b->batch)))
        return VTL_HIP_ERR_INVALID_ARG;
    if (b->batch > kKvMostRows || b->rows > kKvMostRows)
        return VTL_HIP_ERR_UNSUPPORTED;
    kv.pages = static_cast<char *>(c->pages);
    kv.num_pages = c->num_pages;
    kv.page_size = c->page_size;
    kv.kv_heads = c->kv_heads;
    kv.head_dim = c->head_dim;
    kv.padded = (c->head_dim + 15) & ~15;
    kv.page_groups = (unsigned)c->page_size / kKvGroup;
    kv.magic = kv.page_groups == 1 ? 0 : (unsigned)((((uint64_t)1 << 32) + kv.page_groups - 1) / kv.page_groups);
    kv.one = kv.page_groups == 1 ? ~0u : 0;
    kv.head_bytes = (unsigned)c->page_size * (2u * (unsigned)kv.padded + 8u);
    kv.page_bytes = kv.head_bytes * (unsigned)c->kv_heads;
    kv.table = b->page_table;
    kv.lengths = b->lengths;
    kv.starts = b->starts;
    kv.batch = b->batch;
    kv.max_pages = b->max_pages;
    kv.rows = b->rows;
    kv.most_tokens = (int)std::min<int64_t>((int64_t)b->max_pages * c->page_size, kKvMostTokens);
    return VTL_HIP_OK;
}

// Rows of f32 that the call reads or writes: whether `stride` holds one.
inline bool kv_stride_ok(const Kv &kv, int heads, int64_t stride) { return stride >= (int64_t)heads * kv.head_dim; }

// How many bytes of memory they span.
inline size_t kv_span(const Kv &kv, int heads, int64_t stride)
{
    return kv.rows ? ((size_t)(kv.rows - 1) * (size_t)stride + (size_t)heads * kv.head_dim) * sizeof(float) : 0;
}

#ifdef __HIPCC__
// Group `g` of 16 tokens is in page g / page_groups of its sequence.  Exact for g < 2^24, and so for every token below 2^28: the
// product is off by less than g * page_groups / 2^32 <= 1 / page_groups.
__device__ __forceinline__ unsigned kv_page_of(const Kv &kv, unsigned g) { return __umulhi(g, kv.magic) + (g & kv.one); }

__device__ __forceinline__ int kv_length(const Kv &kv, int b) { return min(max(kv.lengths[b], 0), kv.most_tokens); }

// Rows first .. first + count - 1 of the call are sequence b's.
__device__ __forceinline__ void kv_rows_of(const Kv &kv, int b, int &first, int &count)
{
    if (!kv.starts) {
        first = b;
        count = 1;
        return;
    }
    first = min(max(kv.starts[b], 0), kv.rows);
    count = max(min(max(kv.starts[b + 1], 0), kv.rows) - first, 0);
}

// The same for a sequence that the whole wave works on.
__device__ __forceinline__ void kv_sequence(const Kv &kv, int b, int &length, int &first, int &count)
{
    kv_rows_of(kv, b, first, count);
    length = __builtin_amdgcn_readfirstlane(kv_length(kv, b));
    first = __builtin_amdgcn_readfirstlane(first);
    count = __builtin_amdgcn_readfirstlane(count);
}

// One head of the page that group g of sequence b is in, and the group's place there; nullptr: there is no such page.
__device__ __forceinline__ char *kv_group(const Kv &kv, int b, unsigned g, int head, unsigned &at)
{
    const unsigned p = kv_page_of(kv, g);
    at = g - p * kv.page_groups;
    if (p >= (unsigned)kv.max_pages)
        return nullptr;
    const int page = kv.table[(int64_t)b * kv.max_pages + p];
    if ((unsigned)page >= (unsigned)kv.num_pages)
        return nullptr;
    return kv.pages + (uint64_t)(unsigned)page * kv.page_bytes + (uint64_t)head * kv.head_bytes;
}

// The same without a way around the loads: one head (first_page: that of page 0) of page `page`, or of page 0 where there is no such page.
__device__ __forceinline__ const char *kv_page_or_any(const Kv &kv, int page, const char *first_page, bool &there)
{
    there = (unsigned)page < (unsigned)kv.num_pages;
    return first_page + (uint64_t)(there ? (unsigned)page : 0u) * kv.page_bytes;
}

// Where things are in one head of a page.
__device__ __forceinline__ unsigned kv_key_at(const Kv &kv, unsigned dim16, unsigned slot) { return (dim16 * kv.page_size + slot) * 16u; }
__device__ __forceinline__ unsigned kv_value_at(const Kv &kv, unsigned group, unsigned dim)
{
    return (unsigned)kv.padded * kv.page_size + (group * kv.padded + dim) * 16u;
}
__device__ __forceinline__ unsigned kv_scales_at(const Kv &kv) { return 2u * kv.padded * kv.page_size; }
#endif

}  // namespace vtlhip
