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

// Which experts have tokens, in order, and which tokens: pairs of an expert and a token.
struct Entry {
    int expert, offset, pairs, unused;      // the expert's first pair, and how many it has
};
struct Plan {
    int count, unused[3];                   // experts that somebody chose
    Entry entry[kMostExperts];
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
    float *parts;                           // [splits, tokens, dim] where several workgroups share rows of the output
    int splits;
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

// Added up over the lanes of a wave within the vector unit; the last lane has the sum.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_from(double v)
{
    const long long bits = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)bits, CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(bits >> 32), CTRL, ROWS, 0xF, false);
    return v + __builtin_bit_cast(double, (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo));
}
__device__ __forceinline__ double wave_sum_f64(double v)
{
    v = add_from<0xB1, 0xF>(v);     // quad_perm [1,0,3,2]
    v = add_from<0x4E, 0xF>(v);     // quad_perm [2,3,0,1]
    v = add_from<0x141, 0xF>(v);    // row_half_mirror
    v = add_from<0x140, 0xF>(v);    // row_mirror
    v = add_from<0x142, 0xA>(v);    // lane 15 of a row into the next row
    return add_from<0x143, 0xC>(v); // lane 31 into the upper half
}

// A workgroup has one expert's scores for NT tokens, sums in f64 (scores next to each other decide on experts), or, behind those, four
// chunks of the tokens' digits.
template <int NT, bool VEC>
__global__ __launch_bounds__(256) void moe_scores_kernel(const Args g)
{
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const int groups = (g.tokens + NT - 1) / NT;
    const int b = (int)blockIdx.x;
    auto four = [&](const float *row, int k) {
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (VEC) {
            if (k < g.dim)
                v = *reinterpret_cast<const v4f *>(row + k);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (k + i < g.dim)
                    v[i] = row[k + i];
        }
        return v;
    };
    if (b >= g.experts * groups) {
        const int c = 4 * (b - g.experts * groups) + w;
        if (c >= g.tokens * g.dim_chunks)
            return;
        const int t = c / g.dim_chunks, col = c % g.dim_chunks * kChunk + 4 * lane, padded = g.dim_chunks * kChunk;
        const v4f v = four(g.x + (size_t)t * g.dim, col);
        store_digits(g.x_digits + (size_t)t * kDigits * padded, g.x_scales + (size_t)t * (padded / kBlock), padded, col, v);
        return;
    }
    const int e = b % g.experts, t0 = b / g.experts * NT;
    double sum[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
        sum[t] = 0.0;
    const float *const router = g.router + (size_t)e * g.dim;
#pragma unroll 4
    for (int k = 4 * (int)threadIdx.x; k < g.dim; k += 1024) {
        const v4f r = four(router, k);
        v4f x[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
            x[t] = four(g.x + (size_t)min(t0 + t, g.tokens - 1) * g.dim, k);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                sum[t] = fma((double)x[t][i], (double)r[i], sum[t]);
    }
    __shared__ double part[4][NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        sum[t] = wave_sum_f64(sum[t]);
        if (lane == kWave - 1)
            part[w][t] = sum[t];
    }
    __syncthreads();
    if (threadIdx.x < NT && t0 + (int)threadIdx.x < g.tokens) {
        float s = (float)(((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x]);
        if (g.router_bias)
            s = s + g.router_bias[e];
        g.scores[(size_t)(t0 + threadIdx.x) * g.experts + e] = s;
    }
}

// ---- the plan -------------------------------------------------------------------------------

template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned max_from(unsigned v)
{
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ unsigned wave_max_u32(unsigned v)
{
    v = max_from<0xB1, 0xF>(v);
    v = max_from<0x4E, 0xF>(v);
    v = max_from<0x141, 0xF>(v);
    v = max_from<0x140, 0xF>(v);
    v = max_from<0x142, 0xA>(v);
    v = max_from<0x143, 0xC>(v);
    return (unsigned)__builtin_amdgcn_readlane((int)v, kWave - 1);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float sum_from(float v)
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float wave_sum_f32(float v)
{
    v = sum_from<0xB1, 0xF>(v);
    v = sum_from<0x4E, 0xF>(v);
    v = sum_from<0x141, 0xF>(v);
    v = sum_from<0x140, 0xF>(v);
    v = sum_from<0x142, 0xA>(v);
    v = sum_from<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}

// Numbers in their order, from 2 on; 1: NaN, behind all of them.
__device__ __forceinline__ unsigned order_of(float v)
{
    const unsigned b = __float_as_uint(v);
    if (v != v)
        return 1u;
    return max(b & 0x80000000u ? ~b : b | 0x80000000u, 2u);
}

struct Choice {
    Plan plan;
    unsigned long long by[kMostExperts];    // the tokens that chose an expert, a bit each
    float most[kMostTokens], total[kMostTokens];
};

// The plan, made in shared memory by the NW waves of a workgroup: a wave has a token's scores, EACH a lane, finds its `top` largest (the lower
// index of two that are equal) and notes the token with these experts; then the experts that were noted are put in order.
template <int EACH, int NW>
__device__ __forceinline__ void make_plan(const Args &g, Choice &c)
{
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    for (int e = (int)threadIdx.x; e < EACH * kWave; e += NW * kWave)
        c.by[e] = 0;
    __syncthreads();
    for (int t = w; t < g.tokens; t += NW) {
        float v[EACH];
        unsigned key[EACH], top = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int e = lane + i * kWave;
            v[i] = e < g.experts ? g.scores[(size_t)t * g.experts + e] : -__builtin_inff();
        }
        float high = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            key[i] = lane + i * kWave < g.experts ? order_of(v[i]) : 0u;
            top = max(top, key[i]);
        }
        top = wave_max_u32(top);
        // the largest score: NaN where there is nothing else, and then so is all that follows
        high = top == 1u ? __builtin_nanf("") : __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
        float sum = 0.0f, taken = 0.0f;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            v[i] = lane + i * kWave < g.experts ? expf(v[i] - high) : 0.0f;
            sum += v[i];
        }
        sum = wave_sum_f32(sum);
        for (int k = 0; k < g.top; k++) {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < EACH; i++)
                m = max(m, key[i]);
            m = wave_max_u32(m);
            bool found = false;
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const unsigned long long here = __ballot(key[i] == m);
                if (!found && here) {
                    found = true;
                    const int at = __ffsll(here) - 1;
                    taken += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[i]), at));
                    if (lane == at) {
                        key[i] = 0;
                        atomicOr(&c.by[lane + i * kWave], 1ull << t);
                    }
                }
            }
        }
        if (lane == 0) {
            c.most[t] = high;
            c.total[t] = g.renormalize && sum == sum ? taken : sum;
        }
    }
    __syncthreads();
    if (w == 0) {
        int count = 0, at = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int e = i * kWave + lane;
            const unsigned long long who = c.by[e], some = __ballot(who != 0);
            const int n = __popcll(who);
            int first = n;
#pragma unroll
            for (int step = 1; step < kWave; step <<= 1) {
                const int from = __shfl_up(first, step);
                if (lane >= step)
                    first += from;
            }
            if (who)
                c.plan.entry[count + __popcll(some & ((1ull << lane) - 1))] = Entry{e, at + first - n, n, 0};
            count += __popcll(some);
            at += __shfl(first, kWave - 1);
        }
        if (lane == 0)
            c.plan.count = count;
    }
    __syncthreads();
    for (int a = (int)threadIdx.x; a < c.plan.count; a += NW * kWave) {
        const Entry entry = c.plan.entry[a];
        unsigned long long who = c.by[entry.expert];
        for (int i = entry.offset; who; who &= who - 1, i++) {
            const int t = __ffsll(who) - 1;
            c.plan.token[i] = t;
            c.plan.weight[i] = expf(g.scores[(size_t)t * g.experts + entry.expert] - c.most[t]) / c.total[t];
        }
    }
    __syncthreads();
}

// For the launches behind.
template <int NW>
__device__ __forceinline__ void publish(const Args &g, const Choice &c)
{
    const int pairs = g.tokens * g.top;
    for (int i = (int)threadIdx.x; i < max(c.plan.count, pairs); i += NW * kWave) {
        if (i < c.plan.count)
            g.plan->entry[i] = c.plan.entry[i];
        if (i < pairs) {
            g.plan->token[i] = c.plan.token[i];
            g.plan->weight[i] = c.plan.weight[i];
        }
    }
    if (threadIdx.x == 0)
        g.plan->count = c.plan.count;
}

template <int EACH>
__global__ __launch_bounds__(1024) void moe_plan_kernel(const Args g)
{
    __shared__ Choice c;
    make_plan<EACH, 16>(g, c);
    publish<16>(g, c);
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

constexpr int kProductWaves = 8, kKWaves = 4;

// Two 16-byte pieces of a row's chunk, and its scales.
struct Weights {
    v4i codes[2];
    v2u scales;
    __device__ __forceinline__ void load(const uint8_t *c, const uint8_t *s, int chunk)
    {
        codes[0] = *reinterpret_cast<const v4i *>(c + (size_t)chunk * kChunkCodes);
        codes[1] = *reinterpret_cast<const v4i *>(c + (size_t)chunk * kChunkCodes + 64);
        scales = *reinterpret_cast<const v2u *>(s + (size_t)chunk * kChunkScales);
    }
    __device__ __forceinline__ int scale(int step) const { return (int)(scales[step] >> ((int)(threadIdx.x % kWave) / 16 * 8)); }
};

// 32 hidden values of an expert's tokens: two times 16 rows of its gate and as many of its up, four waves each, which deal K out among them.
// They go out as digits, already times their weights, so that the next product adds experts up as it adds up K.
// EACH: every workgroup makes the plan for itself (a few tokens: less than a launch takes); 0: it is there.
template <int TILES, int EACH>
__global__ __launch_bounds__(64 * kProductWaves) void moe_gate_up_kernel(const Args g)
{
    __shared__ __attribute__((aligned(16))) float part[kProductWaves][TILES * kTokensATile][36];
    const int tiles = g.hidden_chunks * (kChunk / 32), a = (int)blockIdx.x / tiles, row0 = (int)blockIdx.x % tiles * 32;
    const Plan *plan = g.plan;
    if constexpr (EACH != 0) {
        __shared__ Choice c;
        make_plan<EACH, kProductWaves>(g, c);
        if (blockIdx.x == 0)
            publish<kProductWaves>(g, c);
        plan = &c.plan;
    }
    if (a >= plan->count)
        return;
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int e = __builtin_amdgcn_readfirstlane(plan->entry[a].expert), offset = __builtin_amdgcn_readfirstlane(plan->entry[a].offset),
              n = __builtin_amdgcn_readfirstlane(plan->entry[a].pairs);
    const size_t pitch = (size_t)g.dim_chunks * kChunkCodes, spitch = (size_t)g.dim_chunks * kChunkScales;
    const uint8_t *wc[2], *ws[2];
#pragma unroll
    for (int f = 0; f < 2; f++) {
        const size_t row = ((size_t)e * 2 + f) * g.hidden + (size_t)min(row0 + w / kKWaves * 16 + r, g.hidden - 1);
        wc[f] = g.gate_up.codes + row * pitch + q * 16;
        ws[f] = g.gate_up.scales + row * spitch;
    }
    const int begin = g.dim_chunks * (w % kKWaves) / kKWaves, end = g.dim_chunks * (w % kKWaves + 1) / kKWaves;
    for (int first = 0; first < n; first += TILES * kTokensATile) {
        const int now = min(n - first, TILES * kTokensATile);
        if (row0 < g.hidden) {
            Columns<TILES> x;
            x.at(g.x_digits, g.x_scales, g.dim_chunks * kChunk, plan->token, offset + first, now);
            v4f acc[2][TILES];
#pragma unroll
            for (int f = 0; f < 2; f++)
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    acc[f][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = begin; c < end; c += 2) {
                const bool two = c + 1 < end;
                Weights weights[2][2];
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (h == 0 || two)
#pragma unroll
                        for (int f = 0; f < 2; f++)
                            weights[h][f].load(wc[f], ws[f], c + h);
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (h == 0 || two)
#pragma unroll
                        for (int i = 0; i < TILES; i++)
                            if (i * kTokensATile < now) {
                                const v2u xs = x.load_scales(i, c + h);
#pragma unroll
                                for (int s = 0; s < 2; s++) {
                                    const v8i d = x.load(i, c + h, s);
                                    const int xb = x.scale(xs, s);
#pragma unroll
                                    for (int f = 0; f < 2; f++)
                                        acc[f][i] = mfma_digits(weights[h][f].codes[s], d, acc[f][i], weights[h][f].scale(s), xb);
                                }
                            }
            }
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int f = 0; f < 2; f++) {
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
                const float(*const mine)[TILES * kTokensATile][36] = &part[row / 16 * kKWaves];
                v4f gate = *reinterpret_cast<const v4f *>(&mine[0][i][row % 16]), up = *reinterpret_cast<const v4f *>(&mine[0][i][16 + row % 16]);
#pragma unroll
                for (int j = 1; j < kKWaves; j++) {
                    gate += *reinterpret_cast<const v4f *>(&mine[j][i][row % 16]);
                    up += *reinterpret_cast<const v4f *>(&mine[j][i][16 + row % 16]);
                }
                const float weight = plan->weight[pair];
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

// 16 output values of all tokens: the chunks of all chosen experts, one expert's behind the other's, are dealt out among the waves of `splits`
// workgroups.  A wave adds what an expert gives to its own sums of the tokens, and the waves' sums meet in order.
constexpr int kAhead = 4;    // chunks whose weights a wave has on their way

__device__ __forceinline__ float down_bias(const Args &g, int t, int row)
{
    float b = 0.0f;
    for (int a = 0; a < g.plan->count; a++) {
        const Entry entry = g.plan->entry[a];
        for (int p = entry.offset; p < entry.offset + entry.pairs; p++)
            if (g.plan->token[p] == t)
                b += g.plan->weight[p] * g.down_bias[(size_t)entry.expert * g.dim + row];
    }
    return b;
}

template <int TILES>
__global__ __launch_bounds__(64 * kProductWaves) void moe_down_kernel(const Args g)
{
    extern __shared__ __attribute__((aligned(16))) float sums[];   // [waves, tokens, 16]
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int split = (int)blockIdx.x % g.splits, row0 = (int)blockIdx.x / g.splits * 16;
    const int count = g.plan->count, all = count * g.hidden_chunks;
    for (int i = (int)threadIdx.x; i < kProductWaves * g.tokens * 16; i += 64 * kProductWaves)
        sums[i] = 0.0f;
    __syncthreads();
    const size_t pitch = (size_t)g.hidden_chunks * kChunkCodes, spitch = (size_t)g.hidden_chunks * kChunkScales;
    const int share = split * kProductWaves + w, shares = g.splits * kProductWaves;
    const int end = (int)((int64_t)all * (share + 1) / shares);
    float *const mine = sums + (size_t)w * g.tokens * 16;
    for (int u = (int)((int64_t)all * share / shares); u < end;) {
        const int a = u / g.hidden_chunks, c0 = u - a * g.hidden_chunks, c1 = min(min(end - a * g.hidden_chunks, g.hidden_chunks), c0 + kAhead);
        const Entry entry = g.plan->entry[a];
        const size_t row = (size_t)entry.expert * g.dim + (size_t)min(row0 + r, g.dim - 1);
        const uint8_t *const wc = g.down.codes + row * pitch + q * 16, *const ws = g.down.scales + row * spitch;
        Weights weights[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (c0 + j < c1)
                weights[j].load(wc, ws, c0 + j);
        for (int first = 0; first < entry.pairs; first += TILES * kTokensATile) {
            const int now = min(entry.pairs - first, TILES * kTokensATile);
            Columns<TILES> h;
            h.at(g.h_digits, g.h_scales, g.hidden_chunks * kChunk, nullptr, entry.offset + first, now);
            v4f acc[TILES];
#pragma unroll
            for (int i = 0; i < TILES; i++)
                acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kAhead; j++)
                if (c0 + j < c1)
#pragma unroll
                    for (int i = 0; i < TILES; i++)
                        if (i * kTokensATile < now) {
                            const v2u hs = h.load_scales(i, c0 + j);
#pragma unroll
                            for (int s = 0; s < 2; s++)
                                acc[i] = mfma_digits(weights[j].codes[s], h.load(i, c0 + j, s), acc[i], weights[j].scale(s), h.scale(hs, s));
                        }
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                v4f v;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    v[k] = sum_digits(acc[i][k]);
                const int pair = i * kTokensATile + r / kDigits;
                if (r % kDigits == 0 && r < 15 && pair < now) {
                    v4f *const to = reinterpret_cast<v4f *>(mine + (size_t)g.plan->token[entry.offset + first + pair] * 16 + 4 * q);
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
        if (g.splits > 1) {
            g.parts[((size_t)split * g.tokens + t) * g.dim + row] = v;
            continue;
        }
        if (g.down_bias)
            v += down_bias(g, t, row);
        g.y[(size_t)t * g.dim + row] = v;
    }
}

// The parts of an output that several workgroups have made, in order.
__global__ __launch_bounds__(256) void moe_join_kernel(const Args g)
{
    const int all = g.tokens * g.dim, i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= all)
        return;
    float v = g.parts[i];
    for (int s = 1; s < g.splits; s++)
        v += g.parts[(size_t)s * all + i];
    if (g.down_bias)
        v += down_bias(g, i / g.dim, i % g.dim);
    g.y[i] = v;
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
    g.parts = reinterpret_cast<float *>(take(g.splits > 1 ? (size_t)g.splits * g.tokens * g.dim * sizeof(float) : 0));
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
    // 512 workgroups for the down product, as long as a wave has four chunks
    const int rows = (m->dim + 15) / 16, chunks = std::min(m->experts, tokens * m->top_k) * g.hidden_chunks;
    g.splits = std::max(1, std::min(512 / rows, chunks / (4 * kProductWaves)));
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
    // no more tokens a workgroup than there are: their loads would be made all the same
    const int at_once = tokens == 1 ? 1 : tokens <= 4 ? 4 : 8;
    const bool vec = g.dim % 4 == 0 && !((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(g.router)) & 15);
    const unsigned scores = (unsigned)(g.experts * ((tokens + at_once - 1) / at_once) + (tokens * g.dim_chunks + 3) / 4);
    const auto scores_vec = at_once == 1 ? moe_scores_kernel<1, true> : at_once == 4 ? moe_scores_kernel<4, true> : moe_scores_kernel<8, true>;
    const auto scores_any = at_once == 1 ? moe_scores_kernel<1, false> : at_once == 4 ? moe_scores_kernel<4, false> : moe_scores_kernel<8, false>;
    hipLaunchKernelGGL(vec ? scores_vec : scores_any, dim3(scores), dim3(256), 0, st, g);
    int status = check_launch("moe_scores_kernel");
    if (status != VTL_HIP_OK)
        return status;
    const bool own_plan = tokens <= kProductWaves, narrow = g.experts <= 2 * kWave;
    if (!own_plan) {
        hipLaunchKernelGGL(narrow ? moe_plan_kernel<2> : moe_plan_kernel<kMostExperts / kWave>, dim3(1), dim3(1024), 0, st, g);
        if ((status = check_launch("moe_plan_kernel")) != VTL_HIP_OK)
            return status;
    }
    const unsigned blocks = (unsigned)std::min(g.experts, tokens * g.top) * (unsigned)(g.hidden_chunks * (kChunk / 32));
    const auto planned = tokens <= kTokensATile ? (narrow ? moe_gate_up_kernel<1, 2> : moe_gate_up_kernel<1, kMostExperts / kWave>)
                                                : (narrow ? moe_gate_up_kernel<2, 2> : moe_gate_up_kernel<2, kMostExperts / kWave>);
    hipLaunchKernelGGL((own_plan ? planned : moe_gate_up_kernel<2, 0>), dim3(blocks), dim3(64 * kProductWaves), 0, st, g);
    if ((status = check_launch("moe_gate_up_kernel")) != VTL_HIP_OK)
        return status;
    const unsigned lds = (unsigned)(kProductWaves * tokens * 16 * sizeof(float)), rows = (unsigned)(g.dim + 15) / 16;
    hipLaunchKernelGGL(tokens <= kTokensATile ? moe_down_kernel<1> : moe_down_kernel<2>, dim3(rows * (unsigned)g.splits), dim3(64 * kProductWaves), lds, st, g);
    if ((status = check_launch("moe_down_kernel")) != VTL_HIP_OK || g.splits == 1)
        return status;
    hipLaunchKernelGGL(moe_join_kernel, dim3((unsigned)(tokens * g.dim + 255) / 256), dim3(256), 0, st, g);
    return check_launch("moe_join_kernel");
}

}  // extern "C"
