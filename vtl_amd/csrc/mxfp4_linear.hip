// Linear layers on microscaled 4-bit rows (gfx950): y = x . W^T + bias with W as stored, [out_features, in_features], and x either codes
// too or f32 rows that become codes on the way.
#include <type_traits>

#include "mxfp4.hpp"

using namespace vtlhip;
using namespace vtlhip::mx;

namespace {

struct Args {
    Rows a, w;            // [M, K], [N, K]
    const float *bias;
    float *y;
    float *partials;      // [splits, M, N] sums of ranges of K, where there is more than one
    int M, N, K;
    int chunks;           // of a row
    int splits;
    int relu;
};

__device__ __forceinline__ float finish(float v, float bias, bool has_bias, bool relu)
{
    if (has_bias)
        v = v + bias;
    return relu && v < 0.0f ? 0.0f : v;
}

// ---- few rows ------------------------------------------------------------------------------

// A workgroup has 32 rows of weights and all of x; its waves deal the chunks of K out among them.  Weights go from memory straight into the
// registers that the matrix unit takes them from (a lane has a block of 16 bytes of one row, four lanes 64 bytes side by side, two loads a chunk).
constexpr int kFewRows = 32, kFewWaves = 8;

template <int MT>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_mxfp4_kernel(const Args g)
{
    __shared__ __attribute__((aligned(16))) float part[kFewWaves][16 * MT][kFewRows + 4];
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane % 16, q = lane / 16;
    const int n0 = blockIdx.x * kFewRows;
    const size_t pitch = (size_t)g.chunks * kChunkCodes, spitch = (size_t)g.chunks * kChunkScales;
    const uint8_t *wc[2], *ws[2], *xc[MT], *xs[MT];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const size_t row = (size_t)min(n0 + 16 * i + r, g.N - 1);
        wc[i] = g.w.codes + row * pitch + q * 16;
        ws[i] = g.w.scales + row * spitch;
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const size_t row = (size_t)min(16 * i + r, g.M - 1);
        xc[i] = g.a.codes + row * pitch + q * 16;
        xs[i] = g.a.scales + row * spitch;
    }
    v4f acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < MT; j++)
            acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int begin = (int)((int64_t)g.chunks * w / kFewWaves), end = (int)((int64_t)g.chunks * (w + 1) / kFewWaves);
    for (int c = begin; c < end; c++) {
        v4i wf[2][2], xq[MT][2];
        int wb[2][2], xb[MT][2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int s = 0; s < 2; s++)
                wf[i][s] = *reinterpret_cast<const v4i *>(wc[i] + (size_t)c * kChunkCodes + 64 * s);
            const v2u scales = *reinterpret_cast<const v2u *>(ws[i] + (size_t)c * kChunkScales);
#pragma unroll
            for (int s = 0; s < 2; s++)
                wb[i][s] = (int)(scales[s] >> (8 * q));
        }
#pragma unroll
        for (int j = 0; j < MT; j++) {
#pragma unroll
            for (int s = 0; s < 2; s++)
                xq[j][s] = *reinterpret_cast<const v4i *>(xc[j] + (size_t)c * kChunkCodes + 64 * s);
            const v2u scales = *reinterpret_cast<const v2u *>(xs[j] + (size_t)c * kChunkScales);
#pragma unroll
            for (int s = 0; s < 2; s++)
                xb[j][s] = (int)(scales[s] >> (8 * q));
        }
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < MT; j++)
                    acc[i][j] = mfma_16(wf[i][s], xq[j][s], acc[i][j], wb[i][s], xb[j][s]);
    }
    // a lane has rows 4 q .. 4 q + 3 of the weights and column r
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) {
            settle(acc[i][j]);
            *reinterpret_cast<v4f *>(&part[w][16 * j + r][16 * i + 4 * q]) = acc[i][j];
        }
    __syncthreads();
    for (int item = threadIdx.x; item < 16 * MT * kFewRows; item += 64 * kFewWaves) {
        const int m = item / kFewRows, nl = item % kFewRows, n = n0 + nl;
        if (m >= g.M || n >= g.N)
            continue;
        float v = part[0][m][nl];
#pragma unroll
        for (int i = 1; i < kFewWaves; i++)
            v += part[i][m][nl];
        g.y[(int64_t)m * g.N + n] = finish(v, g.bias ? g.bias[n] : 0.0f, g.bias != nullptr, g.relu);
    }
}

// ---- many rows -----------------------------------------------------------------------------

// Workgroups are dealt round robin to the 8 XCDs; renumber them so that each XCD, which has an L2 of its own, works on a compact patch
// of the tile grid, and walk the grid in groups of 8 tile rows.
__device__ __forceinline__ void tile_of_block(int tiles_m, int tiles_n, int block, int &tile_m, int &tile_n)
{
    const int total = tiles_m * tiles_n;
    const int xcd = block & 7, rest = total & 7;
    const int pid = xcd * (total >> 3) + min(xcd, rest) + (block >> 3);
    constexpr int kGroup = 8;
    const int group_size = kGroup * tiles_n;
    const int first_m = (pid / group_size) * kGroup;
    const int gm = min(tiles_m - first_m, kGroup);
    tile_m = first_m + (pid % group_size) % gm;
    tile_n = (pid % group_size) / gm;
}

// 16-byte pieces of a tile's rows of 128 bytes are put where a wave's read of 32 rows meets every bank as often.
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// A workgroup has a tile of BM x BN outputs, WR x WC waves a part of it each.  A chunk of K of both operands, 128 bytes of codes and 8 of
// scales a row, goes from memory straight into shared memory, STAGES chunks on their way; a lane of the 32x32x64 product takes a block
// of 16 bytes and its scale byte.
template <int BM, int BN, int WR, int WC, int STAGES>
struct Tile {
    static constexpr int kWaves = WR * WC, kThreads = 64 * kWaves;
    static constexpr int WM = BM / WR, WN = BN / WC, TM = WM / 32, TN = WN / 32;
    static constexpr int kALoads = BM / 8 / kWaves, kBLoads = BN / 8 / kWaves;        // a wave's load: 8 rows of codes
    static constexpr int kSLoads = (BM + BN) / 32 / kWaves;                           // or the scales of 32 rows
    static constexpr int kLoads = kALoads + kBLoads + kSLoads;
    static constexpr int kCodes = (BM + BN) * kChunkCodes, kStage = kCodes + (BM + BN) * kChunkScales;
    static constexpr int kLds = STAGES * kStage;
    static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && (BM + BN) % (32 * kWaves) == 0, "loads are dealt out evenly");
    static_assert(STAGES >= 2 && STAGES * kLoads <= 63, "the counter of loads has 6 bits");
};

template <int BM, int BN, int WR, int WC, int STAGES, bool EDGE>
__global__ __launch_bounds__(64 * WR * WC) void linear_tile_mxfp4_kernel(const Args g)
{
    using T = Tile<BM, BN, WR, WC, STAGES>;
    constexpr int TM = T::TM, TN = T::TN, NW = T::kWaves;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int split = (int)(blockIdx.x % (unsigned)g.splits);
    int tile_m, tile_n;
    tile_of_block((g.M + BM - 1) / BM, (g.N + BN - 1) / BN, (int)(blockIdx.x / (unsigned)g.splits), tile_m, tile_n);
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wr = w / WC, wc = w % WC;
    const int begin = (int)((int64_t)g.chunks * split / g.splits), end = (int)((int64_t)g.chunks * (split + 1) / g.splits);
    const int count = end - begin;
    const size_t pitch = (size_t)g.chunks * kChunkCodes, spitch = (size_t)g.chunks * kChunkScales;

    const int lrow = lane / 8;                            // of the 8 rows of a load
    auto issue = [&](int chunk, int stage) {
        char *const base = smem + stage * T::kStage;
#pragma unroll
        for (int j = 0; j < T::kALoads; j++) {
            const int at = 8 * (w + NW * j), row = at + lrow;
            const size_t from = (size_t)(EDGE ? min(m0 + row, g.M - 1) : m0 + row) * pitch + (size_t)(begin + chunk) * kChunkCodes +
                                (unsigned)(((lane % 8) ^ swizzle(row)) * 16);
            __builtin_amdgcn_global_load_lds(VTL_GPTR(g.a.codes + from), VTL_LPTR(base + at * kChunkCodes), 16, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < T::kBLoads; j++) {
            const int at = 8 * (w + NW * j), row = at + lrow;
            const size_t from = (size_t)(EDGE ? min(n0 + row, g.N - 1) : n0 + row) * pitch + (size_t)(begin + chunk) * kChunkCodes +
                                (unsigned)(((lane % 8) ^ swizzle(row)) * 16);
            __builtin_amdgcn_global_load_lds(VTL_GPTR(g.w.codes + from), VTL_LPTR(base + (BM + at) * kChunkCodes), 16, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < T::kSLoads; j++) {
            const int at = 32 * (w + NW * j), row = at + lane / 2;
            const bool of_a = at < BM;
            const int in = of_a ? (EDGE ? min(m0 + row, g.M - 1) : m0 + row) : (EDGE ? min(n0 + row - BM, g.N - 1) : n0 + row - BM);
            const size_t from = (size_t)in * spitch + (size_t)(begin + chunk) * kChunkScales + (unsigned)(lane % 2 * 4);
            __builtin_amdgcn_global_load_lds(VTL_GPTR((of_a ? g.a.scales : g.w.scales) + from), VTL_LPTR(base + T::kCodes + at * kChunkScales), 4, 0, 0);
        }
    };

    v16f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int k = 0; k < 16; k++)
                acc[i][j][k] = 0.0f;

    const int r = lane % 32, half = lane / 32;
    const unsigned pick = half ? 0x07050301 : 0x06040200;   // of a row's 8 scale bytes, the four of this half's blocks
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
        if (s < count)
            issue(s, s);
    int stage = 0;
    for (int c = 0; c < count; c++) {
        if (c + STAGES - 1 < count) {
            issue(c + STAGES - 1, (c + STAGES - 1) % STAGES);
            wait_vmcnt<(STAGES - 1) * T::kLoads>();
        } else {
            wait_vmcnt<0>();
        }
        __syncthreads();
        const char *const base = smem + stage * T::kStage;
        unsigned sa[TM], sb[TN];
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const v2u v = *reinterpret_cast<const v2u *>(base + T::kCodes + (wr * T::WM + 32 * i + r) * kChunkScales);
            sa[i] = __builtin_amdgcn_perm(v[1], v[0], pick);
        }
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const v2u v = *reinterpret_cast<const v2u *>(base + T::kCodes + (BM + wc * T::WN + 32 * j + r) * kChunkScales);
            sb[j] = __builtin_amdgcn_perm(v[1], v[0], pick);
        }
        auto step = [&](auto s_t) {
            constexpr int s = decltype(s_t)::value;
            v8i fa[TM], fb[TN];
            const unsigned off = (unsigned)(r * kChunkCodes + (((2 * s + half) ^ swizzle(r)) << 4));
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const v4i v = *reinterpret_cast<const v4i *>(base + (wr * T::WM + 32 * i) * kChunkCodes + off);
                fa[i] = v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const v4i v = *reinterpret_cast<const v4i *>(base + (BM + wc * T::WN + 32 * j) * kChunkCodes + off);
                fb[j] = v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], 4, 4, s, (int)sa[i], s, (int)sb[j]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
        __syncthreads();
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }

    // register k of a lane is row 8 (k / 4) + 4 half + k % 4 of a 32 x 32 tile, column r
    float *const out = g.splits > 1 ? g.partials + (size_t)split * g.M * g.N : g.y;
    const bool last = g.splits == 1, has_bias = g.bias != nullptr;
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int n = n0 + wc * T::WN + 32 * j + r;
        if (EDGE && n >= g.N)
            continue;
        const float bias = last && has_bias ? g.bias[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const int m = m0 + wr * T::WM + 32 * i + 8 * (k / 4) + 4 * half + k % 4;
                if (EDGE && m >= g.M)
                    continue;
                const float v = acc[i][j][k];
                __builtin_nontemporal_store(last ? finish(v, bias, has_bias, g.relu) : v, out + (size_t)m * g.N + n);
            }
    }
}

// Adds the ranges of K up, in order.
__global__ __launch_bounds__(256) void linear_join_mxfp4_kernel(const Args g)
{
    const size_t all = (size_t)g.M * g.N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        float v = g.partials[i];
        for (int s = 1; s < g.splits; s++)
            v += g.partials[s * all + i];
        g.y[i] = finish(v, g.bias ? g.bias[i % (size_t)g.N] : 0.0f, g.bias != nullptr, g.relu);
    }
}

// ---- host ----------------------------------------------------------------------------------

template <int BM, int BN, int WR, int WC, int STAGES>
int launch_tile(const Args &g, hipStream_t st)
{
    using T = Tile<BM, BN, WR, WC, STAGES>;
    static PerDevice<DoneFlag> done_flags[2];
    const bool edge = g.M % BM || g.N % BN;
    const auto kernel = edge ? linear_tile_mxfp4_kernel<BM, BN, WR, WC, STAGES, true> : linear_tile_mxfp4_kernel<BM, BN, WR, WC, STAGES, false>;
    DoneFlag &done = done_flags[edge].get();
    if (!done.load(std::memory_order_acquire)) {
        VTL_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds));
        done.store(true, std::memory_order_release);
    }
    const int64_t blocks = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.splits;
    if (blocks > 0xffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(T::kThreads), T::kLds, st, g);
    return check_launch("linear_tile_mxfp4_kernel");
}

// How a product is made: by the kernel for few rows, or by tiles, with K in so many ranges.
struct Plan {
    bool few;
    int splits;
    size_t partials;   // bytes
};

Plan plan_of(int M, int N, int K)
{
    Plan p{M <= 32, 1, 0};
    return p;
}

int product(Args g, const Plan &p, hipStream_t st)
{
    if (p.few) {
        const unsigned blocks = (unsigned)((g.N + kFewRows - 1) / kFewRows);
        const auto kernel = g.M <= 16 ? linear_few_mxfp4_kernel<1> : linear_few_mxfp4_kernel<2>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kFewWaves), 0, st, g);
        return check_launch("linear_few_mxfp4_kernel");
    }
    g.splits = p.splits;
    if (g.M > 128 && g.N > 128 && (int64_t)g.M * g.N >= (int64_t)256 * 256 * 128)
        return launch_tile<256, 256, 2, 2, 2>(g, st);
    return launch_tile<128, 128, 2, 2, 2>(g, st);
}

int check(const Args &g)
{
    if (g.M < 0 || g.N < 0 || g.K < 0)
        return VTL_HIP_ERR_INVALID_ARG;
    if (g.K > kMostCols || (int64_t)g.M * g.N > ((int64_t)1 << 40))
        return VTL_HIP_ERR_UNSUPPORTED;
    return VTL_HIP_OK;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t codes_workspace(int M, int K) { return up256((size_t)M * chunks_of(K) * kChunkCodes) + up256((size_t)M * chunks_of(K) * kChunkScales); }

}  // namespace

extern "C" {

size_t vtl_hip_linear_mxfp4_workspace(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || K > kMostCols)
        return 0;
    return up256(plan_of(M, N, K).partials);
}

size_t vtl_hip_linear_f32_mxfp4_workspace(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || K > kMostCols)
        return 0;
    const Plan p = plan_of(M, N, K);
    return codes_workspace(M, K) + up256(p.partials);
}

int vtl_hip_linear_mxfp4_f32(const uint8_t *x, const uint8_t *x_scales, const uint8_t *w, const uint8_t *w_scales, const float *bias, float *Y, int M,
                             int N, int K, int relu, void *workspace, size_t workspace_bytes)
{
    Args g{{x, x_scales}, {w, w_scales}, bias, Y, nullptr, M, N, K, 0, 1, relu};
    const int rc = check(g);
    if (rc != VTL_HIP_OK || M == 0 || N == 0)
        return rc;
    if (!Y || (K > 0 && (!x || !x_scales || !w || !w_scales)) || !rows_aligned(x, x_scales) || !rows_aligned(w, w_scales))
        return VTL_HIP_ERR_INVALID_ARG;
    g.chunks = chunks_of(K);
    return product(g, plan_of(M, N, K), current_stream());
}

int vtl_hip_linear_f32_mxfp4(const float *X, const uint8_t *w, const uint8_t *w_scales, const float *bias, float *Y, int M, int N, int K, int relu,
                             void *workspace, size_t workspace_bytes)
{
    Args g{{nullptr, nullptr}, {w, w_scales}, bias, Y, nullptr, M, N, K, 0, 1, relu};
    const int rc = check(g);
    if (rc != VTL_HIP_OK || M == 0 || N == 0)
        return rc;
    if (!Y || (K > 0 && (!X || !w || !w_scales)) || !rows_aligned(w, w_scales))
        return VTL_HIP_ERR_INVALID_ARG;
    g.chunks = chunks_of(K);
    const Plan p = plan_of(M, N, K);
    const hipStream_t st = current_stream();
    const size_t need = vtl_hip_linear_f32_mxfp4_workspace(M, N, K);
    char *ws = static_cast<char *>(workspace);
    if (!ws) {
        if (workspace_bytes)
            return VTL_HIP_ERR_INVALID_ARG;
        ws = static_cast<char *>(library_workspace(need, 1));
        if (!ws && need)
            return workspace_status();
    } else if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15)) {
        return VTL_HIP_ERR_INVALID_ARG;
    }
    uint8_t *const codes = reinterpret_cast<uint8_t *>(ws), *const scales = codes + up256((size_t)M * g.chunks * kChunkCodes);
    const int q = launch_quantize(X, K, M, K, codes, scales, st);
    if (q != VTL_HIP_OK)
        return q;
    g.a = {codes, scales};
    return product(g, p, st);
}

}  // extern "C"
