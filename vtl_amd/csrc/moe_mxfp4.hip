// A layer of experts for a few tokens (gfx950), with the experts' weights as microscaled 4-bit rows.
//
// For each token: scores of all experts, the `top` largest of them, and the sum of these experts' outputs
// (SiLU(x . Wg^T + bg) * (x . Wu^T + bu)) . Wd^T + bd, each times its weight.  A step of a few tokens is bound by the weights of the experts that
// somebody chose, which are read once; activations cost next to nothing and are not rounded to 4 bits.  The matrix unit takes 4-bit weights
// beside 8-bit operands, so an f32 value x goes in as five digits of base 32, d0 + d1 / 32 + ... in units of its block's largest binade, each an
// e4m3 number of four bits: 25 bits of x, to 2^-30 of that binade.  The digits are columns of the product (three tokens of five columns), each with a
// scale of its own, and their sums are added at the end.  The products of a block are multiples of 2^-10 up to 12, and their sum is exact in the
// unit; only sums of blocks are rounded, to f32.
#include <cmath>

#include "mxfp4.hpp"

using namespace vtlhip;
using namespace vtlhip::mx;

namespace {

constexpr int kMostTokens = VTL_HIP_MOE_MOST_TOKENS, kMostExperts = VTL_HIP_MOE_MOST_EXPERTS, kMostTop = VTL_HIP_MOE_MOST_TOP;
constexpr int kDigits = 5, kTokensATile = 3;   // 15 of a tile's 16 columns
constexpr int kOwnPlan = 8;                    // tokens up to which every workgroup makes the plan for itself

// Which experts have tokens, in order, and which tokens: pairs of an expert and a token.
struct Entry {
    int expert, offset, pairs, unused;      // the expert's first pair, and how many it has
};
template <int ENTRIES, int PAIRS>
struct PlanOf {
    int count, unused[3];                   // experts that somebody chose
    Entry entry[ENTRIES];
    int token[PAIRS];                       // of a pair
    float weight[PAIRS];
};
using Plan = PlanOf<kMostExperts, kMostTokens * kMostTop>;

struct Args {
    const float *x, *router, *router_bias, *gate_up_bias, *down_bias;
    Rows gate_up, down;
    float *y;
    int tokens, experts, top, dim, hidden, renormalize;
    int dim_chunks, hidden_chunks;          // of a row of weights
    int dim_units, hidden_units;            // of a row of digits, which is padded to whole units
    // workspace
    float *scores;                          // [tokens, experts]
    Plan *plan;
    uint8_t *x_digits, *x_scales;           // [tokens, 5 dim padded], [tokens, dim padded / 32]
    uint8_t *h_digits, *h_scales;           // the same of each pair's hidden values
    float *parts;                           // [splits, tokens, dim] where several workgroups share rows of the output
    int splits;
    int many, dense, large;                 // how the products are launched
    int passes;                             // workgroups of gate and up among which an expert's pairs are dealt out
};

__device__ __forceinline__ v4f mfma_digits(v4i w, v8i d, v4f c, int sw, int sd)
{
    const v8i w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, d, c, 4, 0, 0, sw, 0, sd);
}

__device__ __forceinline__ unsigned max_bits(v4f v)
{
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// Of a block whose largest magnitude has the bits `top`: the scale byte of the first digits (the next ones' are 5 less each; 255: no number), and the
// digits of four of its values.  A digit is the nearest e4m3 number, of four bits, to what the digits before it have left, 32 times that: at most half
// a step, 2^-5 of a value's binade, so that the fifth leaves nothing of 24 bits.  The largest value's first digit is 1 to 2, and the least digit
// 2^-9: values from 2^-6 of the largest on are whole, and of smaller ones at most 2^-30 of the largest is lost.  Blocks below 2^-107 are cut off at 2^-137.
// (The unit adds the products of eight values side by side up in 14 bits, from the largest one's down: 12 is 2^3 and 2^-10 is within.  With the
// largest digit at 2^8, where values from 2^-14 of the largest on are whole, sums were off by 2^-15.)
__device__ __forceinline__ unsigned digit_byte(unsigned top) { return top >= 0x7f800000u ? 255u : min(max(top >> 23, 20u), 253u); }
__device__ __forceinline__ void digits_of(v4f v, unsigned top, unsigned (&d)[kDigits])
{
    const unsigned byte = digit_byte(top);
    const float to_unit = byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = byte == 255u ? 0.0f : v[i] * to_unit;
#pragma unroll
    for (int j = 0; j < kDigits; j++) {
        int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        q = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
        d[j] = (unsigned)q;
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(q, true);
        const float n[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = (v[i] - n[i]) * 32.0f;   // exact
    }
}

// Where the digits of value k of a row lie, and how far from one digit to the next: the 16 bytes of all five that lanes side by side take lie together, for
// a lane of the 16x16x128 product has bytes 16 q .. and 64 + 16 q .. of a step of 128 (and the scale of the q-th block).
constexpr int kDigitStep = 16, kBlockQ = kDigits * kDigitStep, kHalfStep = 4 * kBlockQ, kStep = 2 * kHalfStep;
__device__ __forceinline__ size_t digit_at(int k)
{
    return (size_t)(k / 128) * kStep + (unsigned)(k / 64 % 2 * kHalfStep + k / 16 % 4 * kBlockQ + k % 16);
}

// Those of four values a lane, eight lanes a block.
__device__ __forceinline__ void store_digits(uint8_t *digits, uint8_t *scales, int col, v4f v)
{
    unsigned top = max_bits(v), d[kDigits];
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xF, 0xF, false));
    digits_of(v, top, d);
#pragma unroll
    for (int j = 0; j < kDigits; j++)
        *reinterpret_cast<unsigned *>(digits + digit_at(col) + j * kDigitStep) = d[j];
    if (col % kBlock == 0)
        scales[col / kBlock] = (uint8_t)digit_byte(top);
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
// chunks of the tokens' digits.  Bound by its launch and one way through memory: one token and 64 experts of 4096 2.6 us, 24 and 128 of 2048 4.9.
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
        const int chunks = 2 * g.dim_units, padded = g.dim_units * kUnit;
        if (c >= g.tokens * chunks)
            return;
        const int t = c / chunks, col = c % chunks * kChunk + 4 * lane;
        const v4f v = four(g.x + (size_t)t * g.dim, col);
        store_digits(g.x_digits + (size_t)t * kDigits * padded, g.x_scales + (size_t)t * (padded / kBlock), col, v);
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

// Numbers in their order, from 2 on, the two zeros as one (a sum too small for f32 is -0 where it is negative); 1: NaN, behind all of them.
__device__ __forceinline__ unsigned order_of(float v)
{
    const unsigned b = __float_as_uint(v + 0.0f);
    if (v != v)
        return 1u;
    return max(b & 0x80000000u ? ~b : b | 0x80000000u, 2u);
}

// Added up over a wave's lanes up to each.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned plus_from(unsigned v)
{
    return v + (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ unsigned wave_scan_u32(unsigned v)
{
    v = plus_from<0x111, 0xF>(v);   // row_shr
    v = plus_from<0x112, 0xF>(v);
    v = plus_from<0x114, 0xF>(v);
    v = plus_from<0x118, 0xF>(v);
    v = plus_from<0x142, 0xA>(v);   // lane 15 of a row into the next row
    return plus_from<0x143, 0xC>(v);  // lane 31 into the upper half
}

template <int TOKENS, int EACH>
struct Choice {
    static constexpr int kPairs = TOKENS * kMostTop;
    PlanOf<(kPairs < EACH * kWave ? kPairs : EACH * kWave), kPairs> plan;
    unsigned long long by[EACH * kWave];    // the tokens that chose an expert, a bit each
    int offset[EACH * kWave];               // its first pair
    int expert[kPairs];                     // a token's choices, and what the exponentials of their scores are
    float part[kPairs];
    float total[TOKENS];
};

// The plan, made in shared memory by the NW waves of a workgroup: a wave has a token's scores, EACH a lane, finds its `top` largest (the lower
// index of two that are equal) and notes the token with these experts; then the experts that were noted are put in order.
// Bound by latencies: the scores' way through memory, then `top` maxima over a wave behind each other.  As a launch 6.0 us for 24 tokens of 128 experts, for 64 tokens 11.4, of 256
// experts 14.4 (with EACH 8 21), of 512 21.5; in the workgroups of the next launch 3.8 for one token of 64 (with launch and end), 5.5 for five of 20.  Two tokens of a
// wave beside each other: 1 us less for 64 tokens, 1 us more for one.
template <int NW, int TOKENS, int EACH>
__device__ __forceinline__ void make_plan(const Args &g, Choice<TOKENS, EACH> &c)
{
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    for (int e = (int)threadIdx.x; e < EACH * kWave; e += NW * kWave)
        c.by[e] = 0;
    __syncthreads();
    for (int t = w; t < g.tokens; t += NW) {
        float v[EACH];
        unsigned key[EACH], first = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int e = lane + i * kWave;
            v[i] = e < g.experts ? g.scores[(size_t)t * g.experts + e] : -__builtin_inff();
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            key[i] = lane + i * kWave < g.experts ? order_of(v[i]) : 0u;
            first = max(first, key[i]);
        }
        first = wave_max_u32(first);
        // the largest score: NaN where there is nothing else, and then so is all that follows
        const float high = first == 1u ? __builtin_nanf("") : __uint_as_float(first & 0x80000000u ? first & 0x7fffffffu : ~first);
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
                        c.expert[t * kMostTop + k] = lane + i * kWave;
                        c.part[t * kMostTop + k] = v[i];
                    }
                }
            }
        }
        if (lane == 0)
            c.total[t] = g.renormalize && sum == sum ? taken : sum;
    }
    __syncthreads();
    if (w == 0) {
        unsigned before = 0;     // experts with tokens, and 65536 times their pairs
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int e = i * kWave + lane, n = __popcll(c.by[e]);
            const unsigned mine = (unsigned)n << 16 | (n ? 1u : 0u), up_to = before + wave_scan_u32(mine), at = up_to - mine;
            c.offset[e] = (int)(at >> 16);
            if (n)
                c.plan.entry[at & 0xffff] = Entry{e, (int)(at >> 16), n, 0};
            before = (unsigned)__builtin_amdgcn_readlane((int)up_to, kWave - 1);
        }
        if (lane == 0)
            c.plan.count = (int)(before & 0xffff);
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < g.tokens * g.top; i += NW * kWave) {
        const int t = i / g.top, from = t * kMostTop + i % g.top, e = c.expert[from];
        const int pair = c.offset[e] + __popcll(c.by[e] & ((1ull << t) - 1));
        c.plan.token[pair] = t;
        c.plan.weight[pair] = c.part[from] / c.total[t];
    }
    __syncthreads();
}

// For the launches behind.
template <int NW, typename C>
__device__ __forceinline__ void publish(const Args &g, const C &c)
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
    __shared__ Choice<kMostTokens, EACH> c;
    make_plan<16>(g, c);
    publish<16>(g, c);
}

// ---- products -------------------------------------------------------------------------------

// The digits of up to 3 TILES pairs of one expert as the matrix unit takes them: column 5 i + j of tile `tile` is digit j of pair 3 tile + i.
// Columns of no pair hold anything, which stays in their column.
template <int TILES>
struct Columns {
    const uint8_t *digits[TILES], *scales[TILES];
    bool present[TILES];
    int down;                       // what this digit's scale byte is less by
    v8i d[TILES][kUnitSteps];       // a unit
    v4i s[TILES];
    __device__ __forceinline__ void at(const uint8_t *first_digits, const uint8_t *first_scales, int units, const int *rows, int first, int count)
    {
        const int r = (int)(threadIdx.x % 16), q = (int)(threadIdx.x % kWave) / 16;
        down = r % kDigits * 5;
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const int pair = i * kTokensATile + r / kDigits;
            present[i] = r < kTokensATile * kDigits && pair < count;
            const int at = first + min(pair, count - 1);
            const size_t row = rows ? (size_t)rows[at] : (size_t)at;
            digits[i] = first_digits + row * (size_t)(kDigits * kUnit) * units + (q * kBlockQ + r % kDigits * kDigitStep);
            scales[i] = first_scales + row * (size_t)(kUnit / kBlock) * units;
        }
    }
    // They are asked for in front of the weights of the units behind: loads arrive in order, so that waiting for them would be waiting for those.
    __device__ __forceinline__ void load(int unit)
    {
#pragma unroll
        for (int i = 0; i < TILES; i++)
            if (present[i]) {
                s[i] = *reinterpret_cast<const v4i *>(scales[i] + (size_t)unit * (kUnit / kBlock));
                const uint8_t *const p = digits[i] + (size_t)unit * (kUnitSteps * kStep);
#pragma unroll
                for (int k = 0; k < kUnitSteps; k++) {
                    const v4i lo = *reinterpret_cast<const v4i *>(p + k * kStep), hi = *reinterpret_cast<const v4i *>(p + k * kStep + kHalfStep);
                    d[i][k] = v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                }
            }
    }
    __device__ __forceinline__ int scale(int tile, int step) const
    {
        const int byte = (int)((unsigned)s[tile][step] >> ((int)(threadIdx.x % kWave) / 16 * 8)) & 255;
        return byte == 255 ? 255 : byte - down;
    }
};

// The sum of a pair's five columns, in the lanes of the first.
template <int N>
__device__ __forceinline__ float plus_right(float v, float of)
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(of), 0x100 + N, 0xF, 0xF, true));   // row_shl
}
__device__ __forceinline__ float sum_digits(float v)
{
    const float two = plus_right<1>(v, v), four = plus_right<2>(two, two);
    return plus_right<4>(four, v);
}

// SiLU(gate) * up * weight, as gate * up / (1 + e) where gate is positive and gate * up * e / (1 + e) where it is not, e = exp(-|gate|): e and its sum with 1 are
// numbers for any gate.  Of e the fourth root is made, and goes into factor after factor: e itself is below f32's least number from 104 on, where gate * up * e
// need not be (up to 185, where the root is 2^-67).  The exponential is the vector unit's, corrected by what its argument lost to rounding (|gate| half steps of the value);
// the reciprocal is its own, corrected once.  (By the library's functions, a wave's 32 values of a token took longer than their weights.)
__device__ __forceinline__ float hidden_value(float gate, float up, float weight)
{
    const float m = fabsf(gate), t = m * -0.36067376f;
    float root = __builtin_amdgcn_exp2f(t);
    root = fmaf(root, fmaf(m, -4.81491e-09f, fmaf(m, -0.36067376f, -t)) * 0.6931472f, root);    // (times 2 to what t has lost)
    const float part = gate < 0.0f ? root : 1.0f, half = root * root;
    const float d = fmaf(half, half, 1.0f);
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(r, fmaf(-d, r, 1.0f), r);
    return (gate * part) * (up * part) * part * part * r * weight;
}

// A workgroup's copy of the plan.  All entries that there may be, so that nothing waits for their number.
struct Held {
    Plan plan;
    __device__ __forceinline__ void copy(const Args &g)
    {
        const int pairs = g.tokens * g.top, most = min(g.experts, pairs), threads = (int)blockDim.x;
        if (threadIdx.x == 0)
            plan.count = g.plan->count;
        for (int i = (int)threadIdx.x; i < pairs; i += threads) {
            plan.token[i] = g.plan->token[i];
            plan.weight[i] = g.plan->weight[i];
            if (i < most)
                plan.entry[i] = g.plan->entry[i];
        }
        __syncthreads();
    }
};

// 16 RW FH hidden values of an expert's tokens: RW times 16 FH rows of its gate and as many of its up, KW waves each, which deal K out among them.
// The values go out as digits, already times their weights, so that the next product adds experts up as it adds up K.
// Bound by the weights; from some pairs of an expert on by the digits, which every wave asks for by itself: five bytes of a pair for half a byte of each row.
// One wave along K where that gives 640 workgroups or more, else two (whole calls, us, with one / two / four waves: 1 token, 6 of 64 experts of 4096 x 1024 20.3 / 19.4 / 19.5;
// 1 token, 2 of 8 of 4096 x 7168 25.7 / 25.7 / 29.4; 8 tokens, 2 of 8 of 2048 x 3584, 806 workgroups, 32.9 / 34.5 / 39.7; 4 tokens, 8 of 256 of 4096 x 1024 56 / 57 / 62, and
// 67 to 74 with the plan made in every workgroup).  For 24 tokens of 128 experts of 2048 x 1024, us (their weights alone take 41):
//   waves along K (32 values a workgroup)       1: 45.4     2: 51.4     4: 72.8
//   64 values, 128                              46.1, 54.4; two waves along K and 64 values 58.1
//   one tile (three tokens a pass)              48.0 with one wave along K, 51.9 with two
// Also measured: a workgroup for each compute unit that goes through a run of (expert, 32 values) with the next one's weights on their way 51.8, waves that
// do so by themselves 60.
// FH 2 and four tiles where an expert has four pairs or more by chance (whole calls of 8 experts of 4096 x 7168, 2 a token, us: 16 tokens 105 for 114, 32 125 for 160,
// 64 221 for 254; 64 tokens and 6 of 64 of 2048 x 1408 110 for 125; but 24 tokens and 8 of 128 95 for 86).  Digits by way of shared memory for four
// waves with all pairs' sums in registers were no faster but for 36 pairs of an expert: one wave a SIMD, which waits for its own reads.
// EACH: every workgroup makes the plan for itself (a few tokens: less than a launch takes); 0: it is there.
template <int TILES, int RW, int KW, int EACH, int FH = 1, bool PAST = false>
__global__ __launch_bounds__(64 * RW * KW) void moe_gate_up_kernel(const Args g)
{
    constexpr int NW = RW * KW, kRows = 16 * RW * FH, kPairs = TILES * kTokensATile;
    using S = Stream<2 * FH, PAST>;
    static_assert(RW * FH % 2 == 0, "whole blocks of hidden values");
    static_assert(64 * NW % (kRows / 4) == 0, "a thread's values are the same of every pair");
    extern __shared__ __attribute__((aligned(16))) char smem[];   // two slots a wave
    __shared__ __attribute__((aligned(16))) float part[NW * FH][kPairs][36];
    const int tiles = g.hidden_units * (kUnit / kRows), a = (int)blockIdx.x / tiles / g.passes, pass = (int)blockIdx.x / tiles % g.passes, row0 = (int)blockIdx.x % tiles * kRows;
    const Entry *entries = g.plan->entry;
    const int *tokens = g.plan->token, *count = &g.plan->count;
    const float *weights = g.plan->weight;
    if constexpr (EACH != 0) {
        __shared__ Choice<kOwnPlan, EACH> c;
        make_plan<NW>(g, c);
        if (blockIdx.x == 0)
            publish<NW>(g, c);
        entries = c.plan.entry;
        tokens = c.plan.token;
        count = &c.plan.count;
        weights = c.plan.weight;
    }
    // (an entry behind the last holds anything; it is read beside the number, not behind it)
    const Entry entry = entries[a];
    if (a >= *count)
        return;
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int e = __builtin_amdgcn_readfirstlane(entry.expert), offset = __builtin_amdgcn_readfirstlane(entry.offset), n = __builtin_amdgcn_readfirstlane(entry.pairs);
    char *const ring = smem + w * (2 * S::kSlot);
    const int begin = g.dim_units * (w % KW) / KW, end = g.dim_units * (w % KW + 1) / KW;
    const int my_row = row0 + w / KW * 16 * FH;
    S stream;
    if (my_row < g.hidden) {
#pragma unroll
        for (int f = 0; f < 2 * FH; f++) {
            const int row_f = min(my_row + f / 2 * 16, g.hidden - 1);
            stream.rows(f, g.gate_up, ((size_t)e * 2 + f % 2) * g.hidden + row_f, min(16, g.hidden - row_f), g.dim_chunks);
        }
    }
    // A thread's four of the hidden values below, whatever the pair: their biases are asked for in front of the weights.
    const int row = (int)threadIdx.x % (kRows / 4) * 4;
    v4f gate_bias = {0.0f, 0.0f, 0.0f, 0.0f}, up_bias = gate_bias;
    if (g.gate_up_bias) {
        const float *const bias = g.gate_up_bias + (size_t)e * 2 * g.hidden + row0 + row;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (row0 + row + k < g.hidden) {
                gate_bias[k] = bias[k];
                up_bias[k] = bias[g.hidden + k];
            }
    }
    for (int first = pass * kPairs; first < n; first += g.passes * kPairs) {
        const int now = min(n - first, kPairs);
        if (my_row < g.hidden) {
            if (begin < end)
                stream.issue(begin, ring);
            Columns<TILES> x;
            x.at(g.x_digits, g.x_scales, g.dim_units, tokens, offset + first, now);
            v4f acc[2 * FH][TILES];
#pragma unroll
            for (int f = 0; f < 2 * FH; f++)
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    acc[f][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            const auto work = [&](const char *slot) {
                v4i scales[2 * FH];
#pragma unroll
                for (int f = 0; f < 2 * FH; f++)
                    scales[f] = S::all_scales(slot, f);
#pragma unroll
                for (int k = 0; k < kUnitSteps; k++) {
                    v4i codes[2 * FH];
#pragma unroll
                    for (int f = 0; f < 2 * FH; f++)
                        codes[f] = S::operand(slot, f, k);
#pragma unroll
                    for (int i = 0; i < TILES; i++)
                        if (i * kTokensATile < now) {
                            const int xb = x.scale(i, k);
#pragma unroll
                            for (int f = 0; f < 2 * FH; f++)
                                acc[f][i] = mfma_digits(codes[f], x.d[i][k], acc[f][i], scales[f][k], xb);
                        }
                }
                S::done_reading();
            };
            // (the last unit by itself: the compiler waits for digits as for the way with the fewest loads behind them)
            for (int u = begin; u < end - 1; u++) {
                x.load(u);
                stream.issue(u + 1, ring + (u + 1 - begin) % 2 * S::kSlot);
                wait_vmcnt<S::kLoads>();
                work(ring + (u - begin) % 2 * S::kSlot);
            }
            if (begin < end) {
                x.load(end - 1);
                wait_vmcnt<0>();
                work(ring + (end - 1 - begin) % 2 * S::kSlot);
            }
            settle();
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int f = 0; f < 2 * FH; f++) {
                    v4f v;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        v[k] = sum_digits(acc[f][i][k]);
                    if (r % kDigits == 0 && r < 15)
                        *reinterpret_cast<v4f *>(&part[w + f / 2 * NW][i * kTokensATile + r / kDigits][16 * (f % 2) + 4 * q]) = v;
                }
        }
        __syncthreads();
        for (int item = (int)threadIdx.x; item < now * (kRows / 4); item += 64 * NW) {   // eight lanes: a pair's block of 32
            const int i = item / (kRows / 4), pair = offset + first + i;
            v4f h = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row0 + row < g.hidden) {
                const float(*const mine)[kPairs][36] = &part[row / (16 * FH) * KW + row / 16 % FH * NW];
                v4f gate = *reinterpret_cast<const v4f *>(&mine[0][i][row % 16]), up = *reinterpret_cast<const v4f *>(&mine[0][i][16 + row % 16]);
#pragma unroll
                for (int j = 1; j < KW; j++) {
                    gate += *reinterpret_cast<const v4f *>(&mine[j][i][row % 16]);
                    up += *reinterpret_cast<const v4f *>(&mine[j][i][16 + row % 16]);
                }
                const float weight = weights[pair];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (row0 + row + k < g.hidden)
                        h[k] = hidden_value(gate[k] + gate_bias[k], up[k] + up_bias[k], weight);
                }
            }
            const int padded = g.hidden_units * kUnit;
            store_digits(g.h_digits + (size_t)pair * kDigits * padded, g.h_scales + (size_t)pair * (padded / kBlock), row0 + row, h);
        }
        __syncthreads();
    }
}

// 16 F output values of all tokens: the units of all chosen experts, one expert's behind the other's, are dealt out among the waves of `splits`
// workgroups.  A wave adds what an expert gives to its own sums of the tokens, and the waves' sums meet in order.
// Bound by the weights, and by the hidden values' digits as above: 24 tokens of 128 experts of 2048 x 1024 27.5 us, 4.1 TB/s
// (24.8 without the digits; four waves a workgroup and twice as many workgroups 27.9, sixteen waves a compute unit 32.6); one token, 6 of 4096 x 1024 6.4.
template <int TILES, int F, int NW, bool PAST = false>
__global__ __launch_bounds__(64 * NW) void moe_down_kernel(const Args g)
{
    using S = Stream<F, PAST>;
    constexpr int kSlots = 3, kPairs = TILES * kTokensATile, kRows = 16 * F;
    extern __shared__ __attribute__((aligned(16))) char smem[];    // three slots a wave
    float *const sums = reinterpret_cast<float *>(smem + NW * kSlots * S::kSlot);   // [waves, tokens, kRows]
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    __shared__ Held held;
    held.copy(g);
    const Plan &plan = held.plan;
    const int split = (int)blockIdx.x % g.splits, row0 = (int)blockIdx.x / g.splits * kRows;
    const int units = g.hidden_units, all = __builtin_amdgcn_readfirstlane(plan.count) * units;
    const int share = split * NW + w, shares = g.splits * NW;
    const int begin = (int)((int64_t)all * share / shares), end = (int)((int64_t)all * (share + 1) / shares);
    char *const ring = smem + w * (kSlots * S::kSlot);
    float *const mine = sums + (size_t)w * g.tokens * kRows;
    S stream;
    int streamed = -1;      // whose rows it has
    const auto issue = [&](int u) {
        const int a = u / units;
        if (a != streamed) {
            const size_t expert = (size_t)__builtin_amdgcn_readfirstlane(plan.entry[a].expert) * g.dim;
#pragma unroll
            for (int f = 0; f < F; f++) {
                const int row = min(row0 + 16 * f, g.dim - 1);
                stream.rows(f, g.down, expert + row, min(16, g.dim - row), g.hidden_chunks);
            }
            streamed = a;
        }
        stream.issue(u - a * units, ring + (u - begin) % kSlots * S::kSlot);
    };
    // two units on their way
    if (begin < end)
        issue(begin);
    if (begin + 1 < end)
        issue(begin + 1);
    for (int i = lane; i < g.tokens * kRows; i += kWave)
        mine[i] = 0.0f;
    for (int u = begin; u < end;) {
        const int a = u / units, stop = min(end, (a + 1) * units);
        const Entry entry = plan.entry[a];
        const int offset = __builtin_amdgcn_readfirstlane(entry.offset), pairs = __builtin_amdgcn_readfirstlane(entry.pairs);
        // The wave that has an expert's first unit adds its bias, in the lanes that have a pair's sums.
        v4f bias[F];
#pragma unroll
        for (int f = 0; f < F; f++) {
            bias[f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (g.down_bias && u == a * units)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (row0 + 16 * f + 4 * q + k < g.dim)
                        bias[f][k] = g.down_bias[(size_t)entry.expert * g.dim + row0 + 16 * f + 4 * q + k];
        }
        Columns<TILES> h;
        v4f acc[F][TILES];
        const auto multiply = [&](const char *slot, const v4i (&scales)[F], int now) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < kUnitSteps; k++) {
                v4i codes[F];
#pragma unroll
                for (int f = 0; f < F; f++)
                    codes[f] = S::operand(slot, f, k);
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    if (i * kTokensATile < now) {
                        const int hb = h.scale(i, k);
#pragma unroll
                        for (int f = 0; f < F; f++)
                            acc[f][i] = mfma_digits(codes[f], h.d[i][k], acc[f][i], scales[f][k], hb);
                    }
            }
        };
        const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < F; f++)
#pragma unroll
                for (int i = 0; i < TILES; i++)
                    acc[f][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        };
        const auto add = [&](int first, int now) __attribute__((always_inline)) {
            settle();
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int f = 0; f < F; f++) {
                    v4f v;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        v[k] = sum_digits(acc[f][i][k]);
                    const int pair = i * kTokensATile + r / kDigits;
                    if (r % kDigits == 0 && r < 15 && pair < now) {
                        const float weight = plan.weight[offset + first + pair];
                        v4f *const to = reinterpret_cast<v4f *>(mine + (size_t)plan.token[offset + first + pair] * kRows + 16 * f + 4 * q), sum = *to;
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            (*to)[k] = sum[k] + fmaf(weight, bias[f][k], v[k]);
                    }
                }
            clear();
        };
        clear();
        h.at(g.h_digits, g.h_scales, units, nullptr, offset, min(pairs, kPairs));
        const auto work = [&](const char *slot, int in_row) {
            v4i scales[F];
#pragma unroll
            for (int f = 0; f < F; f++)
                scales[f] = S::all_scales(slot, f);
            multiply(slot, scales, min(pairs, kPairs));
            if (pairs > kPairs) {       // more than fit: unit by unit
                add(0, kPairs);
                for (int first = kPairs; first < pairs; first += kPairs) {
                    h.at(g.h_digits, g.h_scales, units, nullptr, offset + first, min(pairs - first, kPairs));
                    h.load(in_row);
                    multiply(slot, scales, min(pairs - first, kPairs));
                    add(first, min(pairs - first, kPairs));
                }
                h.at(g.h_digits, g.h_scales, units, nullptr, offset, kPairs);
#pragma unroll
                for (int f = 0; f < F; f++)
                    bias[f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
            S::done_reading();
        };
        // (the last two units by themselves: the compiler waits for digits as for the way with the fewest loads behind them)
        for (; u < min(stop, end - 2); u++) {
            h.load(u - a * units);
            issue(u + 2);
            wait_vmcnt<2 * S::kLoads>();
            work(ring + (u - begin) % kSlots * S::kSlot, u - a * units);
        }
        for (; u < stop; u++) {
            h.load(u - a * units);
            wait_vmcnt<0>();
            work(ring + (u - begin) % kSlots * S::kSlot, u - a * units);
        }
        if (pairs <= kPairs)
            add(0, pairs);
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < g.tokens * kRows; i += 64 * NW) {
        const int t = i / kRows, row = row0 + i % kRows;
        if (row >= g.dim)
            continue;
        float v = sums[i];
#pragma unroll
        for (int j = 1; j < NW; j++)
            v += sums[(size_t)j * g.tokens * kRows + i];
        if (g.splits > 1) {
            g.parts[((size_t)split * g.tokens + t) * g.dim + row] = v;
            continue;
        }
        g.y[(size_t)t * g.dim + row] = v;
    }
}

// The parts of an output that several workgroups have made, in order.  (24 x 2048 of two parts: 4.7 us, most of it the launch and one way through memory.)
__global__ __launch_bounds__(256) void moe_join_kernel(const Args g)
{
    const int all = g.tokens * g.dim, i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= all)
        return;
    float v = g.parts[i];
    for (int s = 1; s < g.splits; s++)
        v += g.parts[(size_t)s * all + i];
    g.y[i] = v;
}

// ---- host -----------------------------------------------------------------------------------

// Workgroups of 32 hidden values from which on they are enough with one wave along K each.  Fewer of them deal out an expert's passes over its pairs too, up to twice as many
// workgroups as that (whole calls, us: 32 tokens, 2 of 4 experts of 4096 x 256 29.6, else 43.9; 64 tokens, 2 of 8 of 256 x 128 25.7 and 30.0; 16 tokens, 2 of 8 of 1024 x 512
// 18.6 and 20.5).
constexpr double kManyFrom = 640;

// Pairs of an expert, if tokens choose by chance, from which on waves have twice the weights, so that digits are asked for half as often, where workgroups are enough
// (with fewer: 32 tokens, 2 of 8 of 1024 x 1024 34.5 for 28.1).
constexpr double kDenseFrom = 4.0;

// Bytes of the chosen experts' weights from which on they are read past the caches: half the last-level one.  (24 tokens, 8 of 128 experts of 2048 x 1024, 337 MB, gate and up
// 43.4 us for 45.1; whole calls of 4 tokens, 8 of 256 of 4096 x 1024, 204 MB, 53.8 for 57.0; 8 tokens, 2 of 8 of 4096 x 7168, 336 MB, 87.8 for 92.7; but one token, 2 of 8, 94 MB, 27.7
// for 25.8, and 64 tokens, whose pairs take two passes, 226 for 220.)
constexpr double kLargeFrom = 128e6;

// The kernels with more shared memory than a launch has unasked.
template <void (*KERNEL)(const Args), int MOST>
int launch_with_lds(unsigned blocks, int threads, int lds, hipStream_t st, const Args &g)
{
    static PerDevice<DoneFlag> flags;
    DoneFlag &done = flags.get();
    if (!done.load(std::memory_order_acquire)) {
        VTL_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, MOST));
        done.store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(KERNEL, dim3(blocks), dim3((unsigned)threads), (unsigned)lds, st, g);
    return check_launch("moe_mxfp4 product");
}

template <int TILES, int KW, int EACH, int RW = 2, int FH = 1, bool PAST = false>
int launch_gate_up(const Args &g, unsigned most, hipStream_t st)
{
    constexpr int kLds = RW * KW * 2 * Stream<2 * FH>::kSlot;
    return launch_with_lds<moe_gate_up_kernel<TILES, RW, KW, EACH, FH, PAST>, kLds>(most * (unsigned)(g.passes * g.hidden_units * (kUnit / (16 * RW * FH))), RW * KW * kWave, kLds, st, g);
}

// With the plan made in every workgroup, of so many scores a lane.
template <int TILES>
int launch_few(const Args &g, int each, unsigned most, hipStream_t st)
{
    return each == 2   ? launch_gate_up<TILES, 2, 2>(g, most, st)
           : each == 4 ? launch_gate_up<TILES, 2, 4>(g, most, st)
                       : launch_gate_up<TILES, 2, kMostExperts / kWave>(g, most, st);
}

// Waves of a workgroup of down's.
constexpr int kDownWaves = 8, kDenseWaves = 4;
template <int TILES, int F, int NW, bool PAST = false>
int launch_down(const Args &g, hipStream_t st)
{
    constexpr int kLds = NW * 3 * Stream<F>::kSlot, kToken = NW * 16 * F * (int)sizeof(float);
    const unsigned blocks = (unsigned)(g.dim + 16 * F - 1) / (16 * F) * (unsigned)g.splits;
    return launch_with_lds<moe_down_kernel<TILES, F, NW, PAST>, kLds + kMostTokens * kToken>(blocks, 64 * NW, kLds + g.tokens * kToken, st, g);
}

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
    const size_t pairs = (size_t)g.tokens * g.top, d = (size_t)g.dim_units * kUnit, h = (size_t)g.hidden_units * kUnit;
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
    g.dim_units = (g.dim_chunks + 1) / 2;
    g.hidden_units = (g.hidden_chunks + 1) / 2;
    // if the tokens choose experts as they would by chance: workgroups of 32 hidden values, and pairs of an expert
    const double chosen = g.experts * (1.0 - std::pow(1.0 - (double)g.top / g.experts, tokens)), workgroups = chosen * ((g.hidden + 31) / 32);
    g.many = workgroups >= kManyFrom;
    g.dense = g.many && tokens * g.top >= kDenseFrom * chosen;
    g.large = g.many && !g.dense && chosen * g.hidden * g.dim * (3 * 17.0 / 32.0) >= kLargeFrom;
    // where they are few, an expert's passes over its pairs in workgroups of their own
    g.passes = g.many || tokens <= kOwnPlan ? 1 : std::min((tokens + 2 * kTokensATile - 1) / (2 * kTokensATile), (int)std::ceil(2 * kManyFrom / workgroups));
    // a workgroup for each compute unit for the down product, as long as a wave has two units
    const int rows = g.dense ? (m->dim + 31) / 32 : (m->dim + 15) / 16, units = std::min(m->experts, tokens * m->top_k) * g.hidden_units;
    g.splits = std::max(1, std::min(256 / rows, units / (2 * (g.dense ? kDenseWaves : kDownWaves))));
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
    const size_t results = (size_t)tokens * g.dim * sizeof(float), experts = (size_t)g.experts, into = experts * 2 * g.hidden, out = experts * g.dim;
    const size_t need = vtl_hip_moe_mxfp4_workspace(layer, tokens);
    const auto shared = [&](const void *p, size_t bytes) { return meet(Y, results, p, bytes) || meet(workspace, need, p, bytes); };
    if (meet(Y, results, workspace, need) || shared(X, results) || shared(layer->router, experts * g.dim * sizeof(float)) || shared(layer->router_bias, experts * sizeof(float)) ||
        shared(layer->gate_up, into * g.dim_chunks * kChunkCodes) || shared(layer->gate_up_scales, into * g.dim_chunks * kChunkScales) ||
        shared(layer->gate_up_bias, into * sizeof(float)) || shared(layer->down, out * g.hidden_chunks * kChunkCodes) ||
        shared(layer->down_scales, out * g.hidden_chunks * kChunkScales) || shared(layer->down_bias, out * sizeof(float)))
        return VTL_HIP_ERR_INVALID_ARG;
    g.x = X;
    g.y = Y;
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
    const unsigned scores = (unsigned)(g.experts * ((tokens + at_once - 1) / at_once) + (tokens * 2 * g.dim_units + 3) / 4);
    const auto scores_vec = at_once == 1 ? moe_scores_kernel<1, true> : at_once == 4 ? moe_scores_kernel<4, true> : moe_scores_kernel<8, true>;
    const auto scores_any = at_once == 1 ? moe_scores_kernel<1, false> : at_once == 4 ? moe_scores_kernel<4, false> : moe_scores_kernel<8, false>;
    hipLaunchKernelGGL(vec ? scores_vec : scores_any, dim3(scores), dim3(256), 0, st, g);
    int status = check_launch("moe_scores_kernel");
    if (status != VTL_HIP_OK)
        return status;
    const bool own_plan = tokens <= kOwnPlan && !g.many;
    const int each = g.experts <= 2 * kWave ? 2 : g.experts <= 4 * kWave ? 4 : kMostExperts / kWave;     // scores of a token a lane
    if (!own_plan) {
        hipLaunchKernelGGL(each == 2 ? moe_plan_kernel<2> : each == 4 ? moe_plan_kernel<4> : moe_plan_kernel<kMostExperts / kWave>, dim3(1), dim3(1024), 0, st, g);
        if ((status = check_launch("moe_plan_kernel")) != VTL_HIP_OK)
            return status;
    }
    const unsigned most = (unsigned)std::min(g.experts, tokens * g.top);
    if (g.dense)
        status = launch_gate_up<4, 1, 0, 1, 2>(g, most, st);
    else if (!own_plan)
        status = g.large  ? launch_gate_up<2, 1, 0, 2, 1, true>(g, most, st)
                 : g.many ? launch_gate_up<2, 1, 0>(g, most, st)
                          : launch_gate_up<2, 2, 0>(g, most, st);
    else if (tokens <= kTokensATile)
        status = launch_few<1>(g, each, most, st);
    else
        status = launch_few<2>(g, each, most, st);
    if (status != VTL_HIP_OK)
        return status;
    status = g.dense                  ? launch_down<4, 2, kDenseWaves>(g, st)
             : g.large                ? launch_down<2, 1, kDownWaves, true>(g, st)
             : tokens <= kTokensATile ? launch_down<1, 1, kDownWaves>(g, st)
                                      : launch_down<2, 1, kDownWaves>(g, st);
    if (status != VTL_HIP_OK || g.splits == 1)
        return status;
    hipLaunchKernelGGL(moe_join_kernel, dim3((unsigned)(tokens * g.dim + 255) / 256), dim3(256), 0, st, g);
    return check_launch("moe_join_kernel");
}

}  // extern "C"
