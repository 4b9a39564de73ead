// A layer of experts for a few tokens (gfx950), with the experts' weights as microscaled 4-bit rows.
//
// For each token: scores of all experts, the `top` largest of them, and the sum of these experts' outputs
// (SiLU(x . Wg^T + bg) * (x . Wu^T + bu)) . Wd^T + bd, each times its weight.  A step of a few tokens is bound by the weights of the experts that
// somebody chose, which are read once; activations cost next to nothing and are not rounded to 4 bits.  The matrix unit takes 4-bit weights
// beside 8-bit operands, so an f32 value x goes in as five digits of base 32, d0 + d1 / 32 + ... in units of its block's largest binade over
// 8, each an integer from -16 to 16 and therefore an e4m3 number: 25 bits, to 2^-24 of that binade.  The digits are columns of the product (three
// tokens of five columns), each with a scale of its own, and their sums are added at the end.  A block's products are multiples of a
// half up to 96, so its sum is exact in the unit; only sums of blocks are rounded, to f32.
#include <type_traits>

#include "mxfp4.hpp"

using namespace vtlhip;
using namespace vtlhip::mx;

namespace {

constexpr int kMostTokens = VTL_HIP_MOE_MOST_TOKENS, kMostExperts = VTL_HIP_MOE_MOST_EXPERTS, kMostTop = VTL_HIP_MOE_MOST_TOP;
constexpr int kDigits = 5, kTokensATile = 3;   // 15 of a tile's 16 columns

// Which experts have tokens, in order, and which tokens: written by moe_plan_kernel.
struct Plan {
    int count;                              // experts that somebody chose
    int expert[kMostExperts];
    int offset[kMostExperts + 1];           // their first (expert, token) pair
    int token[kMostTokens * kMostTop];      // of a pair
    float weight[kMostTokens * kMostTop];
};

struct Args {
    const float *x, *router, *router_bias, *gate_up_bias, *down_bias;
    Rows gate_up, down;
    float *y;
    int tokens, experts, top, dim, hidden, renormalize;
    int dim_chunks, hidden_chunks;
    // workspace
    float *scores;                          // [tokens, experts]
    Plan *plan;
    uint8_t *x_digits, *x_scales;           // [tokens, 5, dim padded], [tokens, dim padded / 32]
    uint8_t *h_digits, *h_scales;           // the same of each pair's hidden values
};

__device__ __forceinline__ v4f mfma_digits(v4i w, v8i d, v4f c, int sw, int sd)
{
    const v8i w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, d, c, 4, 0, 0, sw, 0, sd);
}

// Digits of four values a lane, eight lanes a block; the byte is that of the first digit (the next ones' are 5 less each).  Blocks below
// 2^-103 are cut off at 2^-128.
__device__ __forceinline__ unsigned digits_of(v4f v, unsigned (&d)[kDigits])
{
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
    const unsigned field = max(m >> 23, 23u);
    const bool bad = field == 255;
    const float to_unit = __uint_as_float((bad ? 127u : 257u - field) << 23);
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = bad ? 0.0f : v[i] * to_unit;
#pragma unroll
    for (int j = 0; j < kDigits; j++) {
        float n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            n[i] = rintf(v[i]);
            v[i] = (v[i] - n[i]) * 32.0f;   // exact
        }
        int q = __builtin_amdgcn_cvt_pk_fp8_f32(n[0], n[1], 0, false);
        q = __builtin_amdgcn_cvt_pk_fp8_f32(n[2], n[3], q, true);
        d[j] = (unsigned)q;
    }
    return bad ? 255u : field - 3u;
}

__device__ __forceinline__ void store_digits(uint8_t *digits, uint8_t *scales, int cols_padded, int col, v4f v)
{
    unsigned d[kDigits];
    const unsigned byte = digits_of(v, d);
#pragma unroll
    for (int j = 0; j < kDigits; j++)
        *reinterpret_cast<unsigned *>(digits + (size_t)j * cols_padded + col) = d[j];
    if (col % kBlock == 0)
        scales[col / kBlock] = (uint8_t)byte;
}

// ---- scores ---------------------------------------------------------------------------------

// A workgroup has one expert's scores for up to eight tokens, sums in f64 (scores next to each other decide on experts), or, behind those, four
// chunks of the tokens' digits.
constexpr int kScoreTokens = 8;

__global__ __launch_bounds__(256) void moe_scores_kernel(const Args g)
{
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const int groups = (g.tokens + kScoreTokens - 1) / kScoreTokens;
    int b = (int)blockIdx.x;
    if (b >= g.experts * groups) {
        const int c = 4 * (b - g.experts * groups) + w;
        if (c >= g.tokens * g.dim_chunks)
            return;
        const int t = c / g.dim_chunks, col = c % g.dim_chunks * kChunk + 4 * lane;
        const float *const row = g.x + (size_t)t * g.dim;
        v4f v;
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = col + i < g.dim ? row[col + i] : 0.0f;
        const int padded = g.dim_chunks * kChunk;
        store_digits(g.x_digits + (size_t)t * kDigits * padded, g.x_scales + (size_t)t * (padded / kBlock), padded, col, v);
        return;
    }
    const int e = b % g.experts, t0 = b / g.experts * kScoreTokens, n = min(kScoreTokens, g.tokens - t0);
    double sum[kScoreTokens];
#pragma unroll
    for (int t = 0; t < kScoreTokens; t++)
        sum[t] = 0.0;
    const float *const router = g.router + (size_t)e * g.dim;
    for (int k = (int)threadIdx.x; k < g.dim; k += 256) {
        const double r = router[k];
#pragma unroll
        for (int t = 0; t < kScoreTokens; t++)
            if (t < n)
                sum[t] = fma((double)g.x[(size_t)(t0 + t) * g.dim + k], r, sum[t]);
    }
    __shared__ double part[4][kScoreTokens];
#pragma unroll
    for (int t = 0; t < kScoreTokens; t++)
        if (t < n) {
#pragma unroll
            for (int step = 32; step; step >>= 1)
                sum[t] += __shfl_xor(sum[t], step);
            if (lane == 0)
                part[w][t] = sum[t];
        }
    __syncthreads();
    if ((int)threadIdx.x < n) {
        float s = (float)(((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x]);
        if (g.router_bias)
            s = s + g.router_bias[e];
        g.scores[(size_t)(t0 + threadIdx.x) * g.experts + e] = s;
    }
}

// ---- the plan -------------------------------------------------------------------------------

__device__ __forceinline__ unsigned wave_max_u32(unsigned v)
{
#pragma unroll
    for (int step = 32; step; step >>= 1)
        v = max(v, (unsigned)__shfl_xor((int)v, step));
    return v;
}
__device__ __forceinline__ float wave_sum_f32(float v)
{
#pragma unroll
    for (int step = 32; step; step >>= 1)
        v += __shfl_xor(v, step);
    return v;
}

// Numbers in their order, from 2 on; 1: NaN, behind all of them.
__device__ __forceinline__ unsigned order_of(float v)
{
    const unsigned b = __float_as_uint(v);
    if (v != v)
        return 1u;
    return max(b & 0x80000000u ? ~b : b | 0x80000000u, 2u);
}

// One workgroup: a wave has a token's scores, finds its `top` largest (the lower index of two that are equal) and notes the token with these experts;
// then the experts that were noted are put in order.
__global__ __launch_bounds__(1024) void moe_plan_kernel(const Args g)
{
    __shared__ unsigned long long chosen_by[kMostExperts];
    __shared__ int place[kMostExperts], pairs[kMostExperts];
    __shared__ float most[kMostTokens], total[kMostTokens];
    constexpr int kEach = kMostExperts / kWave;
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    for (int e = (int)threadIdx.x; e < kMostExperts; e += 1024)
        chosen_by[e] = 0;
    __syncthreads();
    for (int t = w; t < g.tokens; t += 16) {
        float v[kEach];
        unsigned key[kEach];
        float high = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int e = lane + i * kWave;
            v[i] = e < g.experts ? g.scores[(size_t)t * g.experts + e] : -__builtin_inff();
            key[i] = e < g.experts ? order_of(v[i]) : 0u;
            high = fmaxf(high, v[i]);
        }
#pragma unroll
        for (int step = 32; step; step >>= 1)
            high = fmaxf(high, __shfl_xor(high, step));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (lane + i * kWave < g.experts)
                sum += expf(v[i] - high);
        sum = wave_sum_f32(sum);
        float taken = 0.0f;
        for (int k = 0; k < g.top; k++) {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < kEach; i++)
                m = max(m, key[i]);
            m = wave_max_u32(m);
            bool found = false;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const unsigned long long here = __ballot(key[i] == m);
                if (!found && here) {
                    found = true;
                    const int at = __ffsll(here) - 1;
                    taken += __shfl(expf(v[i] - high), at);
                    if (lane == at) {
                        key[i] = 0;
                        atomicOr(&chosen_by[lane + i * kWave], 1ull << t);
                    }
                }
            }
        }
        if (lane == 0) {
            most[t] = high;
            total[t] = g.renormalize && sum == sum ? taken : sum;
        }
    }
    __syncthreads();
    if (w == 0) {
        int count = 0, at = 0;
        for (int i = 0; i < g.experts; i += kWave) {
            const int e = i + lane;
            const unsigned long long who = e < g.experts ? chosen_by[e] : 0;
            const unsigned long long some = __ballot(who != 0);
            const int before = __popcll(some & ((1ull << lane) - 1));
            int n = __popcll(who), first = n;
#pragma unroll
            for (int step = 1; step < kWave; step <<= 1) {
                const int from = __shfl_up(first, step);
                if (lane >= step)
                    first += from;
            }
            const int all = __shfl(first, kWave - 1);
            if (who) {
                place[count + before] = e;
                pairs[count + before] = at + first - n;
            }
            count += __popcll(some);
            at += all;
        }
        if (lane == 0) {
            g.plan->count = count;
            g.plan->offset[count] = at;
        }
        for (int a = lane; a < count; a += kWave) {
            g.plan->expert[a] = place[a];
            g.plan->offset[a] = pairs[a];
        }
        __threadfence_block();
        for (int a = lane; a < count; a += kWave) {
            const int e = place[a];
            unsigned long long who = chosen_by[e];
            for (int i = pairs[a]; who; who &= who - 1, i++) {
                const int t = __ffsll(who) - 1;
                g.plan->token[i] = t;
                g.plan->weight[i] = expf(g.scores[(size_t)t * g.experts + e] - most[t]) / total[t];
            }
        }
    }
}

// ---- products -------------------------------------------------------------------------------

// The digits of up to 3 TILES pairs of one expert as the matrix unit takes them: column 5 i + j of tile `tile` is digit j of pair 3 tile + i.  A lane of
// the 16x16x128 product has bytes 16 q .. and 64 + 16 q .. of a step of 128, and the scale of block q.
template <int TILES>
struct Columns {
    const uint8_t *digits[TILES], *scales[TILES];
    int down;                       // what this digit's scale byte is less by
    __device__ __forceinline__ void at(const uint8_t *d, const uint8_t *s, int padded, const int *rows, int first, int count)
    {
        const int r = min((int)(threadIdx.x % 16), 14), q = (int)(threadIdx.x % kWave) / 16;
        down = r % kDigits * 5;
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const int pair = first + min(i * kTokensATile + r / kDigits, count - 1);
            const size_t row = rows ? (size_t)rows[pair] : (size_t)pair;
            digits[i] = d + (row * kDigits + r % kDigits) * (size_t)padded + 16 * q;
            scales[i] = s + row * (size_t)(padded / kBlock);
        }
    }
    __device__ __forceinline__ v8i load(int tile, int chunk, int step) const
    {
        const uint8_t *const p = digits[tile] + (size_t)chunk * kChunk + 128 * step;
        const v4i lo = *reinterpret_cast<const v4i *>(p), hi = *reinterpret_cast<const v4i *>(p + 64);
        return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
    __device__ __forceinline__ v2u load_scales(int tile, int chunk) const
    {
        return *reinterpret_cast<const v2u *>(scales[tile] + (size_t)chunk * kChunkScales);
    }
    __device__ __forceinline__ int scale(v2u both, int step) const
    {
        const int byte = (int)(both[step] >> ((int)(threadIdx.x % kWave) / 16 * 8)) & 255;
        return byte == 255 ? 255 : byte - down;
    }
};

// The sum of a pair's five columns, in the lanes of the first; the smallest digits first.
__device__ __forceinline__ float sum_digits(float v)
{
    auto right = [&](auto n) {
        constexpr int kControl = 0x100 + decltype(n)::value;   // row_shl
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, 0xF, 0xF, true));
    };
    float s = right(std::integral_constant<int, 4>{}) + right(std::integral_constant<int, 3>{});
    s += right(std::integral_constant<int, 2>{});
    s += right(std::integral_constant<int, 1>{});
    return s + v;
}

constexpr int kProductWaves = 8;

// 32 hidden values of an expert's tokens: 32 rows of its gate and as many of its up, K dealt out among the waves.  They go out as digits, already
// times their weights, so that the next product adds experts up as it adds up K.
template <int TILES>
__global__ __launch_bounds__(64 * kProductWaves) void moe_gate_up_kernel(const Args g)
{
    __shared__ __attribute__((aligned(16))) float part[kProductWaves][TILES * kTokensATile][68];
    const int tiles = g.hidden_chunks * (kChunk / 32), a = (int)blockIdx.x / tiles, row0 = (int)blockIdx.x % tiles * 32;
    if (a >= g.plan->count)
        return;
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int e = g.plan->expert[a], offset = g.plan->offset[a], n = g.plan->offset[a + 1] - offset;
    const size_t pitch = (size_t)g.dim_chunks * kChunkCodes, spitch = (size_t)g.dim_chunks * kChunkScales;
    const uint8_t *wc[4], *ws[4];
#pragma unroll
    for (int f = 0; f < 4; f++) {
        const size_t row = (size_t)e * 2 * g.hidden + (f / 2) * (size_t)g.hidden + (size_t)min(row0 + f % 2 * 16 + r, g.hidden - 1);
        wc[f] = g.gate_up.codes + row * pitch + q * 16;
        ws[f] = g.gate_up.scales + row * spitch;
    }
    const int begin = g.dim_chunks * w / kProductWaves, end = g.dim_chunks * (w + 1) / kProductWaves;
    for (int first = 0; first < n; first += TILES * kTokensATile) {
        const int now = min(n - first, TILES * kTokensATile);
        if (row0 < g.hidden) {
            Columns<TILES> x;
            x.at(g.x_digits, g.x_scales, g.dim_chunks * kChunk, g.plan->token, offset + first, now);
            v4f acc[4][TILES];
#pragma unroll
            for (int f = 0; f < 4; f++)
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    acc[f][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = begin; c < end; c++) {
                v4i codes[4][2];
                v2u scales[4];
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    codes[f][0] = *reinterpret_cast<const v4i *>(wc[f] + (size_t)c * kChunkCodes);
                    codes[f][1] = *reinterpret_cast<const v4i *>(wc[f] + (size_t)c * kChunkCodes + 64);
                    scales[f] = *reinterpret_cast<const v2u *>(ws[f] + (size_t)c * kChunkScales);
                }
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    if (i * kTokensATile < now) {
                        const v2u xs = x.load_scales(i, c);
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            const v8i d = x.load(i, c, s);
                            const int xb = x.scale(xs, s);
#pragma unroll
                            for (int f = 0; f < 4; f++)
                                acc[f][i] = mfma_digits(codes[f][s], d, acc[f][i], (int)(scales[f][s] >> (8 * q)), xb);
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    v4f v;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        v[k] = sum_digits(acc[f][i][k]);
                    if (r % kDigits == 0 && r < 15)
                        *reinterpret_cast<v4f *>(&part[w][i * kTokensATile + r / kDigits][16 * f + 4 * q]) = v;
                }
        }
        __syncthreads();
        for (int item = (int)threadIdx.x; item < now * 8; item += 64 * kProductWaves) {   // eight lanes: a pair's block of 32
            const int i = item / 8, row = item % 8 * 4, pair = offset + first + i;
            v4f h = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row0 < g.hidden) {
                v4f gate = *reinterpret_cast<const v4f *>(&part[0][i][row]), up = *reinterpret_cast<const v4f *>(&part[0][i][32 + row]);
#pragma unroll
                for (int j = 1; j < kProductWaves; j++) {
                    gate += *reinterpret_cast<const v4f *>(&part[j][i][row]);
                    up += *reinterpret_cast<const v4f *>(&part[j][i][32 + row]);
                }
                const float weight = g.plan->weight[pair];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (row0 + row + k >= g.hidden)
                        continue;
                    if (g.gate_up_bias) {
                        const float *const bias = g.gate_up_bias + (size_t)e * 2 * g.hidden + row0 + row + k;
                        gate[k] += bias[0];
                        up[k] += bias[g.hidden];
                    }
                    h[k] = gate[k] / (1.0f + expf(-gate[k])) * up[k] * weight;
                }
            }
            const int padded = g.hidden_chunks * kChunk;
            store_digits(g.h_digits + (size_t)pair * kDigits * padded, g.h_scales + (size_t)pair * (padded / kBlock), padded, row0 + row, h);
        }
        __syncthreads();
    }
}

// 16 output values of all tokens: the chunks of all chosen experts, one expert's behind the other's, are dealt out among the waves.  A wave adds
// what an expert gives to its own sums of the tokens, and the waves' sums meet in order.
template <int TILES>
__global__ __launch_bounds__(64 * kProductWaves) void moe_down_kernel(const Args g)
{
    extern __shared__ __attribute__((aligned(16))) float sums[];   // [waves, tokens, 16]
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int row0 = (int)blockIdx.x * 16;
    for (int i = (int)threadIdx.x; i < kProductWaves * g.tokens * 16; i += 64 * kProductWaves)
        sums[i] = 0.0f;
    __syncthreads();
    const size_t pitch = (size_t)g.hidden_chunks * kChunkCodes, spitch = (size_t)g.hidden_chunks * kChunkScales;
    const int count = g.plan->count, all = count * g.hidden_chunks;
    const int end = (int)((int64_t)all * (w + 1) / kProductWaves);
    float *const mine = sums + (size_t)w * g.tokens * 16;
    for (int u = (int)((int64_t)all * w / kProductWaves); u < end;) {
        const int a = u / g.hidden_chunks, c0 = u - a * g.hidden_chunks, c1 = min(end - a * g.hidden_chunks, g.hidden_chunks);
        const int e = g.plan->expert[a], offset = g.plan->offset[a], n = g.plan->offset[a + 1] - offset;
        const size_t row = (size_t)e * g.dim + (size_t)min(row0 + r, g.dim - 1);
        const uint8_t *const wc = g.down.codes + row * pitch + q * 16, *const ws = g.down.scales + row * spitch;
        for (int first = 0; first < n; first += TILES * kTokensATile) {
            const int now = min(n - first, TILES * kTokensATile);
            Columns<TILES> h;
            h.at(g.h_digits, g.h_scales, g.hidden_chunks * kChunk, nullptr, offset + first, now);
            v4f acc[TILES];
#pragma unroll
            for (int i = 0; i < TILES; i++)
                acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = c0; c < c1; c++) {
                v4i codes[2];
                codes[0] = *reinterpret_cast<const v4i *>(wc + (size_t)c * kChunkCodes);
                codes[1] = *reinterpret_cast<const v4i *>(wc + (size_t)c * kChunkCodes + 64);
                const v2u scales = *reinterpret_cast<const v2u *>(ws + (size_t)c * kChunkScales);
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    if (i * kTokensATile < now) {
                        const v2u hs = h.load_scales(i, c);
#pragma unroll
                        for (int s = 0; s < 2; s++)
                            acc[i] = mfma_digits(codes[s], h.load(i, c, s), acc[i], (int)(scales[s] >> (8 * q)), h.scale(hs, s));
                    }
            }
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                v4f v;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    v[k] = sum_digits(acc[i][k]);
                const int pair = i * kTokensATile + r / kDigits;
                if (r % kDigits == 0 && r < 15 && pair < now) {
                    v4f *const to = reinterpret_cast<v4f *>(mine + (size_t)g.plan->token[offset + first + pair] * 16 + 4 * q);
                    *to = *to + v;
                }
            }
        }
        u = a * g.hidden_chunks + c1;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < g.tokens * 16; i += 64 * kProductWaves) {
        const int t = i / 16, row = row0 + i % 16;
        if (row >= g.dim)
            continue;
        float v = sums[i];
#pragma unroll
        for (int j = 1; j < kProductWaves; j++)
            v += sums[(size_t)j * g.tokens * 16 + i];
        if (g.down_bias) {
            float b = 0.0f;
            for (int p = 0, a = 0; a < count; a++)
                for (; p < g.plan->offset[a + 1]; p++)
                    if (g.plan->token[p] == t)
                        b += g.plan->weight[p] * g.down_bias[(size_t)g.plan->expert[a] * g.dim + row];
            v += b;
        }
        g.y[(size_t)t * g.dim + row] = v;
    }
}

// ---- host -----------------------------------------------------------------------------------

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

int check(const vtl_hip_moe *m, int tokens)
{
    if (!m || tokens < 0 || m->experts < 1 || m->top_k < 1 || m->top_k > m->experts || m->dim < 1 || m->hidden < 1)
        return VTL_HIP_ERR_INVALID_ARG;
    if (tokens > kMostTokens || m->experts > kMostExperts || m->top_k > kMostTop || m->dim > VTL_HIP_MOE_MOST_DIM || m->hidden > VTL_HIP_MOE_MOST_DIM)
        return VTL_HIP_ERR_UNSUPPORTED;
    return VTL_HIP_OK;
}

// Lays the workspace out from `at` on; the bytes it takes.
size_t lay_out(Args &g, char *at)
{
    const size_t pairs = (size_t)g.tokens * g.top, d = (size_t)g.dim_chunks * kChunk, h = (size_t)g.hidden_chunks * kChunk;
    size_t used = 0;
    auto take = [&](size_t bytes) {
        char *const p = at + used;
        used += up256(bytes);
        return p;
    };
    g.scores = reinterpret_cast<float *>(take((size_t)g.tokens * g.experts * sizeof(float)));
    g.plan = reinterpret_cast<Plan *>(take(sizeof(Plan)));
    g.x_digits = reinterpret_cast<uint8_t *>(take(g.tokens * kDigits * d));
    g.x_scales = reinterpret_cast<uint8_t *>(take(g.tokens * d / kBlock));
    g.h_digits = reinterpret_cast<uint8_t *>(take(pairs * kDigits * h));
    g.h_scales = reinterpret_cast<uint8_t *>(take(pairs * h / kBlock));
    return used;
}

Args args_of(const vtl_hip_moe *m, int tokens)
{
    Args g{};
    g.router = m->router;
    g.router_bias = m->router_bias;
    g.gate_up_bias = m->gate_up_bias;
    g.down_bias = m->down_bias;
    g.gate_up = {m->gate_up, m->gate_up_scales};
    g.down = {m->down, m->down_scales};
    g.tokens = tokens;
    g.experts = m->experts;
    g.top = m->top_k;
    g.dim = m->dim;
    g.hidden = m->hidden;
    g.renormalize = m->renormalize != 0;
    g.dim_chunks = chunks_of(m->dim);
    g.hidden_chunks = chunks_of(m->hidden);
    return g;
}

}  // namespace

extern "C" {

size_t vtl_hip_moe_mxfp4_workspace(const vtl_hip_moe *layer, int tokens)
{
    if (check(layer, tokens) != VTL_HIP_OK || tokens == 0)
        return 0;
    Args g = args_of(layer, tokens);
    return lay_out(g, nullptr);
}

int vtl_hip_moe_mxfp4_f32(const vtl_hip_moe *layer, const float *X, float *Y, int tokens, void *workspace, size_t workspace_bytes)
{
    const int rc = check(layer, tokens);
    if (rc != VTL_HIP_OK || tokens == 0)
        return rc;
    if (!X || !Y || !layer->router || !layer->gate_up || !layer->gate_up_scales || !layer->down || !layer->down_scales ||
        !rows_aligned(layer->gate_up, layer->gate_up_scales) || !rows_aligned(layer->down, layer->down_scales))
        return VTL_HIP_ERR_INVALID_ARG;
    Args g = args_of(layer, tokens);
    g.x = X;
    g.y = Y;
    const size_t need = vtl_hip_moe_mxfp4_workspace(layer, tokens);
    char *ws = static_cast<char *>(workspace);
    if (!ws) {
        if (workspace_bytes)
            return VTL_HIP_ERR_INVALID_ARG;
        ws = static_cast<char *>(library_workspace(need));
        if (!ws)
            return workspace_status();
    } else if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15)) {
        return VTL_HIP_ERR_INVALID_ARG;
    }
    lay_out(g, ws);
    const hipStream_t st = current_stream();
    const unsigned scores = (unsigned)(g.experts * ((tokens + kScoreTokens - 1) / kScoreTokens) + (tokens * g.dim_chunks + 3) / 4);
    hipLaunchKernelGGL(moe_scores_kernel, dim3(scores), dim3(256), 0, st, g);
    int status = check_launch("moe_scores_kernel");
    if (status != VTL_HIP_OK)
        return status;
    hipLaunchKernelGGL(moe_plan_kernel, dim3(1), dim3(1024), 0, st, g);
    if ((status = check_launch("moe_plan_kernel")) != VTL_HIP_OK)
        return status;
    const unsigned blocks = (unsigned)std::min(g.experts, tokens * g.top) * (unsigned)(g.hidden_chunks * (kChunk / 32));
    hipLaunchKernelGGL(tokens <= 3 ? moe_gate_up_kernel<1> : moe_gate_up_kernel<2>, dim3(blocks), dim3(64 * kProductWaves), 0, st, g);
    if ((status = check_launch("moe_gate_up_kernel")) != VTL_HIP_OK)
        return status;
    const unsigned lds = (unsigned)(kProductWaves * tokens * 16 * sizeof(float));
    hipLaunchKernelGGL(tokens <= 3 ? moe_down_kernel<1> : moe_down_kernel<2>, dim3((unsigned)(g.dim + 15) / 16), dim3(64 * kProductWaves), lds, st, g);
    return check_launch("moe_down_kernel");
}

}  // extern "C"
