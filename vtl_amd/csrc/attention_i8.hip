// Attention over the int8 key/value cache for gfx950.
//
//   s_j = scale * sum_d q_d K_jd sk_j,   w = softmax over the tokens that the row sees,   o_d = sum_j w_j sv_j V_jd
//
// The codes K and V are whole numbers below 128, which fp16 holds exactly, so both products run on the fp16 matrix units with f32 sums.  What
// meets them is no whole number: q (with scale and log2 e) and w_j sv_j, two halves of 11 bits each, hi = f16(x), lo = f16(x - hi), one product
// for each.  So 22 bits of the operands enter, where one half alone would leave an error of 2^-11, and a third would cost half as much again.
// q is scaled by a power of two to a largest value between 2^14 and 2^15 (the rows of a workgroup that shares tiles by one, but for those more than
// 2^kNear below, and else each row by its own): lo keeps its bits down to 2^-16 of the largest, and is off by 2^-39 of it below that.  The products
// w_j sv_j are kept between 2^13 and 2^14 likewise, by the largest that the row itself has had: a token that a row gives no weight takes nothing from
// it, however large its values.  (Few rows take the largest of each tile; many rows take the values' scales for it and look at the products only where
// those are far apart, `kNear`.)
//
// One pass over the tokens, with the running maximum and sum of the softmax, in powers of two.  Products are transposed, tokens as the
// rows of S^T = K Q^T and dimensions as those of O^T = V^T W^T: a lane then holds what belongs to one row of q, maximum and sum are taken within the
// lane but for two exchanges, and the weights lie as the second product's operand wants them (which token a row of the first product is
// is chosen so).  Nothing of the scores or weights goes through memory.
#include "kv_cache.hpp"
#include "quant_device.hpp"

using namespace vtlhip;
using namespace vtlhip::qdev;

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 0x1.715476p+0f;

// Eight codes as fp16: the byte b + 128 below 0x64 is the number 1024 + b + 128.
__device__ __forceinline__ half8_t codes_to_half(int a, int b)
{
    union {
        unsigned u[4];
        half8_t h;
    } r;
    const unsigned x = (unsigned)a ^ 0x80808080u, y = (unsigned)b ^ 0x80808080u;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u);
    return r.h - (_Float16)1152.0f;
}

// The two halves of two numbers, as elements 2 i and 2 i + 1 of each: one product with each half is one with 22 bits.
__device__ __forceinline__ void split_two(float x, float y, half8_t &hi, half8_t &lo, int i)
{
    unsigned minus = 0xbc00;      // -1, unknown to the compiler (see split)
    asm("" : "+s"(minus));
    const float one = (float)__builtin_bit_cast(half2_t, minus)[0];
    const half2_t a = __builtin_convertvector((float2_t{x, y}), half2_t);
    const half2_t b = __builtin_convertvector((float2_t{__builtin_fmaf((float)a[0], one, x), __builtin_fmaf((float)a[1], one, y)}), half2_t);
    hi[2 * i] = a[0];
    hi[2 * i + 1] = a[1];
    lo[2 * i] = b[0];
    lo[2 * i + 1] = b[1];
}

// The two halves of eight numbers.
__device__ __forceinline__ void split(const float *x, half8_t &hi, half8_t &lo)
{
    union {
        half2_t p[4];
        half8_t h;
    } a, b;
    // x - f32(hi) in one instruction, which multiplies a half and adds an f32; a -1 that the compiler sees it would make two of
    unsigned minus = 0xbc00;
    asm("" : "+s"(minus));
    const float one = (float)__builtin_bit_cast(half2_t, minus)[0];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a.p[i] = __builtin_convertvector((float2_t{x[2 * i], x[2 * i + 1]}), half2_t);
        b.p[i] = __builtin_convertvector((float2_t{__builtin_fmaf((float)a.p[i][0], one, x[2 * i]), __builtin_fmaf((float)a.p[i][1], one, x[2 * i + 1])}),
                                         half2_t);
    }
    hi = a.h;
    lo = b.h;
}

__device__ __forceinline__ float max_across_16(float v)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_across_16(float v)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float sum_across_32(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float max_across_32(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ int exponent_of(float v) { return (int)((__float_as_uint(v) >> 23) & 255) - 127; }

// Rows of a tile are tokens of `size` heads each: which token and which of its heads a row is, given those of the tile's first row and how far behind it
// (less than 256) the row is.
struct Group {
    int size;
    float part;
    explicit Group(int n) : size(n), part(1.0f / (float)n) {}
    __device__ __forceinline__ void row(int token0, int head0, int behind, int &token, int &head) const
    {
        const unsigned n = (unsigned)head0 + (unsigned)behind;
        int more = (int)((float)n * part);      // at most 256: no further off than by one
        head = (int)(n - (unsigned)more * (unsigned)size);
        more += head < 0 ? -1 : head >= size ? 1 : 0;
        head += head < 0 ? size : head >= size ? -size : 0;
        token = token0 + more;
    }
};

// The launch as the host has planned it.
struct Parts {
    int tiles;      // of rows, in the sequence with the most
    int splits;     // of the tokens
    int chunk;      // tokens of a split; more where a sequence is longer than the host knew
    float *sums;    // [unit][split][row][padded head_dim]
    float (*tops)[2];   // [unit][split][row]: maximum, sum of weights
};

// Tokens of a split of a sequence of which `seen` are of use.
__device__ __forceinline__ int chunk_of(const Parts &parts, int seen)
{
    return max(parts.chunk, (int)((((unsigned)seen + parts.splits - 1) / (unsigned)parts.splits + 63) & ~63u));
}

// Parts of a row are made on one XCD and read on another: past the L2 caches, which are not coherent with each other.
__device__ __forceinline__ void store_far(float *p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Over each 16 lanes.
__device__ __forceinline__ float row_max_16(float v)
{
#pragma unroll
    for (int i = 1; i < 16; i *= 2)
        v = fmaxf(v, __shfl_xor(v, i));
    return v;
}
__device__ __forceinline__ float row_sum_16(float v)
{
#pragma unroll
    for (int i = 1; i < 16; i *= 2)
        v += __shfl_xor(v, i);
    return v;
}

// Two of a part's numbers.  THERE: an earlier launch wrote them, so the caches have nothing older.
template <bool THERE>
__device__ __forceinline__ float2_t load_two(const float *p)
{
    if (THERE)
        return *reinterpret_cast<const float2_t *>(p);
    return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Parts of a row put together: numbers begin .. begin + AT_ONCE - 1, then `step` further on, as long as there are any of n.  A lane has four values of the row;
// they and the maxima and sums of AT_ONCE parts are on their way at once, so that what bounds this is a trip to memory for so many.
struct Joined {
    float top = -INFINITY, sum = 0.0f;
    float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};

    template <int AT_ONCE, bool THERE, typename SLOT>
    __device__ __forceinline__ void add(int begin, int n, int step, const float *sums, int pitch, const float (*tops)[2], SLOT slot)
    {
        for (int i0 = begin; i0 < n; i0 += step) {
            float2_t t[AT_ONCE], v[AT_ONCE][2];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const int64_t at = slot(min(i0 + k, n - 1));
                t[k] = load_two<THERE>(tops[at]);
                v[k][0] = load_two<THERE>(sums + at * pitch);
                v[k][1] = load_two<THERE>(sums + at * pitch + 2);
            }
            float now = top;
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++)
                now = fmaxf(now, t[k][0]);
            const float off = now == -INFINITY ? 0.0f : now, keep = __builtin_amdgcn_exp2f(top - off);
            top = now;
            sum *= keep;
            o *= keep;
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const float more = i0 + k < n ? t[k][1] : 0.0f, weight = more == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(t[k][0] - off);
                sum = more == 0.0f ? sum : __builtin_fmaf(more, weight, sum);      // also where the weight is 0: a sum that is no number stays none
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[j] = weight == 0.0f ? o[j] : __builtin_fmaf(v[k][j / 2][j % 2], weight, o[j]);
            }
        }
    }
    // The row's values d .. d + 3, of which there are `dims` at all.
    __device__ __forceinline__ void store(float *y, int d, int dims, bool vectors) const
    {
        const float4_t v = sum == 0.0f ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : o / sum;
        if (vectors)
            *reinterpret_cast<float4_t *>(y + d) = v;
        else
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (d + j < dims)
                    y[d + j] = v[j];
    }
};

// ---- few rows: a tile's rows are 16 or 32, all of a sequence's that read one key/value head ------------
//
// Bound by the way of the cache's bytes into registers (2 D + 8 a token and head; 2 sequences of 65000 tokens, 8 heads of 128: 275 MB in 60.7 us, 4.5 TB/s,
// where a stream that is only read has 7.3; 48 of up to 6000: 63.8 us) and, where those are few, by the latencies behind each other and the code read for the
// first time (one of 300: 8.4 us; 8 of 3001 with 5 rows each, 16 heads of 64: 17.9 us, 1.9 TB/s).  So every wave takes tiles of 64 tokens for itself, straight from memory into the registers in
// the order in which the matrix units take them; keys of the next tile are on their way while the weights of one are made, its values while the next
// one's scores are, and the pages of both are looked up a tile before.
//
// A unit is a tile of rows and a key/value head; its tokens are cut into rounds, in which every wave of a workgroup has a tile of 64.  All
// rounds of all units, behind each other, are dealt out evenly, as many workgroups as the chip takes at once: so ragged lengths cost nothing, and a
// workgroup has parts of at most two units, its first and its last.  The workgroups that share a unit meet in the launch where
// they have a counter: each writes its part through to memory and counts itself, and the last one adds the parts up and
// leaves the counter at zero.  Else a launch of their own adds them up.
constexpr int kMostShares = 512;
__device__ unsigned g_arrived[kStreamSlots][2 * kMostShares];

struct Shares {
    int count;          // workgroups
    int counters;       // which set of counters; -1: parts are added up by a launch of their own
    float *sums;        // [2 count][rows of a tile][padded head_dim]: parts of the first unit and of the last of each workgroup
    float (*tops)[2];   // [2 count][rows of a tile]
    int vectors;        // whether a row of the result is written in vectors of 16 bytes
};

// What a workgroup has, and where others' begins: q or q + 1 rounds each.
struct Deal {
    int each, more;
    __device__ __forceinline__ Deal(int total, int shares) : each((int)((unsigned)total / (unsigned)shares)), more(total - each * shares) {}
    __device__ __forceinline__ int start(int share) const { return share * each + min(share, more); }
    __device__ __forceinline__ int of(int round) const
    {
        const int mark = more * (each + 1);
        return round < mark ? (int)((unsigned)round / (unsigned)(each + 1)) : more + (int)((unsigned)(round - mark) / (unsigned)max(each, 1));
    }
};

// Over the lanes up to each.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int scan_step(int v)
{
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ int scan_add(int v)
{
    v = scan_step<0x111, 0xF>(v);      // row_shr:1, 2, 4, 8
    v = scan_step<0x112, 0xF>(v);
    v = scan_step<0x114, 0xF>(v);
    v = scan_step<0x118, 0xF>(v);
    v = scan_step<0x142, 0xA>(v);      // row_bcast:15 into rows 1 and 3
    return scan_step<0x143, 0xC>(v);   // row_bcast:31 into rows 2 and 3
}

// 64 sequences from `base` on, one a lane, and the rounds of all units of each: how many, and how many there are up to and with it.
template <int ROWS, int STEP>
struct Sequences {
    int base, length, first, count, rounds, upto;
    __device__ __forceinline__ Sequences(const Kv &kv, int group, int base_) : base(base_), length(0), first(0), count(0), rounds(0)
    {
        const int b = base + (int)(threadIdx.x & 63);
        if (b < kv.batch) {
            kv_rows_of(kv, b, first, count);
            length = kv_length(kv, b);
            rounds = (count * group + ROWS - 1) / ROWS * max((length + STEP - 1) / STEP, 1) * kv.kv_heads;
        }
        upto = scan_add(rounds);
    }
    __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(upto, 63); }
};

// The rounds of all sequences.  The host has seen to it that they are kMostRounds at most as long as `starts` ascends; where it does not, and they are
// more than 32 bits count, there is nothing to do.
constexpr int kMostRounds = 1 << 30;
template <int ROWS, int STEP>
__device__ __forceinline__ int all_rounds(const Kv &kv, int group, const Sequences<ROWS, STEP> &begin)
{
    int all = begin.all();
    float size = (float)begin.rounds;
    for (int base = 64; base < kv.batch; base += 64) {
        const Sequences<ROWS, STEP> s(kv, group, base);
        all += s.all();
        size += (float)s.rounds;
    }
    const unsigned long long lots = __ballot(size > 1.5f * kMostRounds / 64.0f);      // of one lane's
    if (!lots)
        return all;
    size = sum_across_32(sum_across_16(row_sum_16(size)));
    return __builtin_amdgcn_readfirstlane(size > 1.5f * kMostRounds) ? 0 : all;
}

// Finds the sequences whose rounds a workgroup has, one behind the other.
template <int ROWS, int STEP>
struct Finder {
    Sequences<ROWS, STEP> in;
    int before;      // the rounds of all before in.base
    __device__ __forceinline__ Finder(const Sequences<ROWS, STEP> &begin) : in(begin), before(0) {}
    // The lane that has the sequence of `round`.
    __device__ __forceinline__ int lane_of(const Kv &kv, int group, int round)
    {
        for (;;) {
            const unsigned long long past = __ballot(before + in.upto > round);
            if (past)
                return __builtin_ctzll(past);
            if (in.base + 64 >= kv.batch)
                return 63;      // not reached: the rounds of all sequences are more
            before += in.all();
            in = Sequences<ROWS, STEP>(kv, group, in.base + 64);
        }
    }
};

// The part of a unit that a workgroup has: rounds begin .. end - 1 of its `rounds`, which are first_round .. of all.
struct Part {
    int b, length, first, count;      // the sequence and its rows of the call
    int head, row0, here;             // key/value head; rows of the tile
    int begin, end, rounds, first_round;
};
template <int ROWS, int STEP>
__device__ __forceinline__ Part part_of(const Kv &kv, int group, Finder<ROWS, STEP> &find, int round, int stop)
{
    Part u;
    const int at = find.lane_of(kv, group, round);
    u.b = find.in.base + at;
    u.length = __builtin_amdgcn_readlane(find.in.length, at);
    u.first = __builtin_amdgcn_readlane(find.in.first, at);
    u.count = __builtin_amdgcn_readlane(find.in.count, at);
    const int before = find.before + __builtin_amdgcn_readlane(find.in.upto - find.in.rounds, at);
    u.rounds = max((u.length + STEP - 1) / STEP, 1);
    // none is negative: a division of signs costs twice the code
    const unsigned unit = (unsigned)(round - before) / (unsigned)u.rounds, tile = unit / (unsigned)kv.kv_heads;
    u.head = (int)(unit - tile * (unsigned)kv.kv_heads);
    u.row0 = (int)tile * ROWS;
    u.here = min(ROWS, u.count * group - u.row0);
    u.first_round = before + (int)unit * u.rounds;
    u.begin = round - u.first_round;
    u.end = min(u.rounds, stop - u.first_round);
    return u;
}

// Where a workgroup leaves its part of a unit that begins with `first_round`.
__device__ __forceinline__ int part_slot(const Deal &deal, int share, int first_round) { return 2 * share + (first_round > deal.start(share) ? 1 : 0); }

// Adds up a unit's parts: the first workgroup's may be its second, the others' are their first.
template <int DT, int ROWS, bool THERE>
__device__ __forceinline__ void join_unit(const Kv &kv, const Shares &shares, const Deal &deal, const Part &u, int share0, int share1, const Group &of, float *out,
                                          int64_t out_stride, int wave, int waves)
{
    constexpr int kLanes = DT / 4, kTogether = 64 / kLanes;
    const int64_t slot0 = part_slot(deal, share0, u.first_round);
    const int lane = threadIdx.x & 63, d = lane % kLanes * 4;
    const int token0 = (int)((unsigned)u.row0 / (unsigned)of.size), head0 = u.row0 - token0 * of.size;
    for (int r0 = wave * kTogether; r0 < u.here; r0 += waves * kTogether) {
        const int r = min(r0 + lane / kLanes, u.here - 1);
        const bool mine = r0 + lane / kLanes < u.here && d < kv.head_dim;
        Joined row;
        row.add<(DT > 128 ? 8 : 16), THERE>(0, share1 - share0 + 1, DT > 128 ? 8 : 16, shares.sums + (mine ? d : 0), kv.padded, shares.tops,
                                           [&](int i) { return (i ? 2 * (share0 + i) : slot0) * ROWS + r; });
        int token, of_token;
        of.row(token0, head0, r, token, of_token);
        if (mine)
            row.store(out + (int64_t)(u.first + token) * out_stride + (u.head * of.size + of_token) * kv.head_dim, d, kv.head_dim, shares.vectors);
    }
}

template <int DT, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DT * NB > 128 ? 1 : 2) void attention_few_kernel(Kv kv, const float *__restrict__ q, int64_t q_stride, Group of,
                                                                                         float scale, int causal, float *__restrict__ out,
                                                                                         int64_t out_stride, Shares shares)
{
    constexpr int kRows = 16 * NB, kPitch = DT + 4, kStep = 64 * WAVES;
    __shared__ __align__(16) _Float16 q_half[DT / 8][2][kRows][8];
    __shared__ float q_unit[kRows];
    __shared__ __align__(16) float o_part[WAVES][kRows][kPitch];
    __shared__ float top_part[WAVES][kRows], sum_part[WAVES][kRows];
    __shared__ float level_part[WAVES][kRows];
    __shared__ int is_last;

    const int share = blockIdx.x;
    const Sequences<kRows, kStep> begin(kv, of.size, 0);
    const Deal deal(all_rounds(kv, of.size, begin), shares.count);
    const int stop = deal.start(share + 1);
    Finder<kRows, kStep> find(begin);
    // Opaque: what follows from it is worked out in each turn of the loop, of which there hardly are two, and not kept in registers that there are none of.
    auto opaque = [](int v) {
        asm volatile("" : "+s"(v));
        return v;
    };
    for (int round = deal.start(share); round < stop;) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int col = lane & 15, g = lane >> 4;
        const int group = opaque(of.size);
        const Part u = part_of(kv, group, find, round, stop);
        const int b = u.b, length = u.length, first = u.first, count = u.count, head = u.head, row0 = u.row0, here = u.here, rows = count * group;
        const int token0 = (int)((unsigned)row0 / (unsigned)group), head0 = row0 - token0 * group;      // of the tile's first row
        int token, of_token;
        of.row(token0, head0, here - 1, token, of_token);
        const int seen = causal ? max(length - count + token + 1, 0) : length;      // by its last
        const int from = u.begin * kStep, to = min(seen, u.end * kStep);
        const int32_t *const table = kv.table + (int64_t)b * kv.max_pages;
        const char *const first_page = kv.pages + (uint64_t)head * kv.head_bytes;

        // Pages of the 16 tokens whose keys, and of those whose scales and values, this lane takes.
        int key_page, value_page;
        auto look_up = [&](int j0) {
            key_page = table[kv_page_of(kv, (unsigned)min(j0 + 16 * (col >> 2), to - 1) / 16)];
            value_page = table[kv_page_of(kv, (unsigned)min(j0 + 16 * g, to - 1) / 16)];
        };
        int j0 = from + 64 * w;
        if (j0 < to)
            look_up(j0);
        // the wave's rows of q
        constexpr int kMine = kRows / WAVES;
        float q_row[kMine][DT / 64];
#pragma unroll
        for (int r = 0; r < kMine; r++) {
            const int row = row0 + w + r * WAVES;
            of.row(token0, head0, w + r * WAVES, token, of_token);
            const float *from_q = q + (int64_t)(first + token) * q_stride + (head * group + of_token) * kv.head_dim;
#pragma unroll
            for (int i = 0; i < DT / 64; i++)
                q_row[r][i] = row < rows && lane + 64 * i < kv.head_dim ? from_q[lane + 64 * i] : 0.0f;
        }

        int4_t keys[4][DT / 64], values[DT / 16];
        float4_t ks[4], vs[4];
        bool there;
        auto load_keys = [&](int j0) {
            const int padded = opaque(kv.padded);
            const unsigned group16 = (unsigned)min(j0 + 16 * (col >> 2), to - 1) / 16;
            bool any;      // where there is no token, or no dimension, any codes do: q or the weight is 0 there
            const char *page = kv_page_or_any(kv, key_page, first_page, any);
            const unsigned slot = (group16 - kv_page_of(kv, group16) * kv.page_groups) * 16 + (col & 3);
#pragma unroll
            for (int u = 0; u < DT / 64; u++) {
                const unsigned c = 16 * (4 * u + g) < padded ? 4 * u + g : 0;
                const char *p = page + kv_key_at(kv, c, slot);
#pragma unroll
                for (int t = 0; t < 4; t++)
                    keys[t][u] = *reinterpret_cast<const int4_t *>(p + 64 * t);
            }
        };
        auto load_values = [&](int j0) {
            const unsigned group16 = (unsigned)min(j0 + 16 * g, to - 1) / 16;
            const char *page = kv_page_or_any(kv, value_page, first_page, there);
            there = there && j0 + 16 * g < to;
            const unsigned place = group16 - kv_page_of(kv, group16) * kv.page_groups;
            const float *scales = reinterpret_cast<const float *>(page + kv_scales_at(kv)) + place * 16;
            const char *p = page + kv_value_at(kv, place, 0);
            const int padded = opaque(kv.padded);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                ks[t] = reinterpret_cast<const float4_t *>(scales)[t];
                vs[t] = reinterpret_cast<const float4_t *>(scales + kv.page_size)[t];
            }
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                values[i] = *reinterpret_cast<const int4_t *>(p + ((16 * i < padded ? 16 * i : 0) + col) * 16);
        };
        if (j0 < to) {
            load_keys(j0);
            load_values(j0);
            if (j0 + kStep < to)
                look_up(j0 + kStep);
        }

        // ---- rows of q as halves
#pragma unroll
        for (int r = 0; r < kMine; r++) {
            if (w + r * WAVES >= here)
                break;      // what lies there gives sums that no row has
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < DT / 64; i++) {
                q_row[r][i] = q_row[r][i] * scale * kLog2e;
                most = fmaxf(most, fabsf(q_row[r][i]));
            }
            const int e = exponent_of(wave_max(most)), at = w + r * WAVES;
#pragma unroll
            for (int i = 0; i < DT / 64; i++) {
                const int d = lane + 64 * i;
                const float v = __builtin_ldexpf(q_row[r][i], 14 - e);
                const _Float16 hi = (_Float16)v;
                q_half[d / 8][0][at][d % 8] = hi;
                q_half[d / 8][1][at][d % 8] = (_Float16)(v - (float)hi);
            }
            if (lane == 0)
                q_unit[at] = __builtin_ldexpf(1.0f, e - 14);
        }
        __syncthreads();

        float unit_of[NB], top[NB], sum[NB];
        int limit[NB], level[NB];      // sums of values are in units of 2^(level - 13)
        float4_t o[NB][DT / 16];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            unit_of[n] = q_unit[16 * n + col];
            of.row(token0, head0, min(16 * n + col, here - 1), token, of_token);
            limit[n] = causal ? min(length - count + token + 1, to) : to;
            top[n] = -INFINITY;
            sum[n] = 0.0f;
            level[n] = -127;
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                o[n][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }

        for (; j0 < to; j0 += kStep) {
            asm volatile("" ::: "memory");      // q's halves are read again for every tile, not kept in registers
            // S^T: row r of product t is token j0 + 16 (r / 4) + 4 t + r % 4, so that this lane's are 16 g .. 16 g + 15
            float4_t s[NB][4];
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    s[n][t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < DT / 64; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    half8_t k[4];
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        k[t] = codes_to_half(keys[t][u][2 * h], keys[t][u][2 * h + 1]);
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int part = 0; part < 2; part++) {
                            const half8_t x = *reinterpret_cast<const half8_t *>(&q_half[8 * u + 2 * g + h][part][16 * n + col][0]);
#pragma unroll
                            for (int t = 0; t < 4; t++)
                                s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], x, s[n][t], 0, 0, 0);
                        }
                }
            if (j0 + kStep < to)
                load_keys(j0 + kStep);

            // scales of tokens that are none count for nothing
            const int mine = there ? j0 + 16 * g : 0x7fffffff;
            float4_t zeros = ks[0] * 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    zeros[i] = __builtin_fmaf(vs[t][i], 0.0f, t ? __builtin_fmaf(ks[t][i], 0.0f, zeros[i]) : zeros[i]);
            if (__any(!(zeros[0] + zeros[1] + zeros[2] + zeros[3] == 0.0f)))
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // a token with such a scale is no number for the rows that see it, and out of the way of the others
                        const bool finite = fabsf(vs[t][i]) < INFINITY && fabsf(ks[t][i]) < INFINITY;
                        ks[t][i] = finite ? ks[t][i] : NAN;
                        vs[t][i] = finite ? vs[t][i] : 0.0f;
                    }

            half8_t p[NB][2][2];
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int until = limit[n];
                float best = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // the unit goes to the key's scale first: either may be far from 1 where their product is not
                        const float v = s[n][t][i] * (ks[t][i] * unit_of[n]);
                        s[n][t][i] = mine < until - (4 * t + i) ? v : -INFINITY;
                        best = fmaxf(best, s[n][t][i]);
                    }
                best = max_across_32(max_across_16(best));
                const float now = fmaxf(top[n], best);
                const float off = now == -INFINITY ? 0.0f : now;
                const float keep = __builtin_amdgcn_exp2f(top[n] - off);
                top[n] = now;
                float x[16], add = 0.0f, most = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float e = __builtin_amdgcn_exp2f(s[n][t][i] - off);
                        add += e;
                        x[4 * t + i] = e * vs[t][i];
                        most = fmaxf(most, fabsf(x[4 * t + i]));
                    }
                sum[n] = __builtin_fmaf(sum[n], keep, add);
                // the row's level is the largest power of two that a weight times its value's scale has had, brought to the present maximum
                most = max_across_32(max_across_16(most));
                const int before = level[n];
                level[n] = max(before + exponent_of(keep), exponent_of(most));
#pragma unroll
                for (int i = 0; i < 16; i++)
                    x[i] = __builtin_ldexpf(x[i], 13 - level[n]);
                split(x, p[n][0][0], p[n][0][1]);
                split(x + 8, p[n][1][0], p[n][1][1]);
                const float by = __builtin_ldexpf(keep, before - level[n]);
#pragma unroll
                for (int i = 0; i < DT / 16; i++)
                    o[n][i] *= by;
            }
            // O^T: 64 tokens in two steps of 32, lane group g has 16 g + 8 step ..
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8_t v = codes_to_half(values[i][2 * h], values[i][2 * h + 1]);
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int part = 0; part < 2; part++)
                            o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[n][h][part], o[n][i], 0, 0, 0);
                }
            if (j0 + kStep < to)
                load_values(j0 + kStep);
            if (j0 + 2 * kStep < to)
                look_up(j0 + 2 * kStep);
        }

        // ---- the waves meet: what each has of the rows that there are, in its own units
#pragma unroll
        for (int n = 0; n < NB; n++) {
            sum[n] = sum_across_32(sum_across_16(sum[n]));
            if (g == 0) {
                level_part[w][16 * n + col] = (float)level[n];
                top_part[w][16 * n + col] = top[n];
                sum_part[w][16 * n + col] = sum[n];
            }
            if (16 * n + col < here)
#pragma unroll
                for (int i = 0; i < DT / 16; i++)
                    *reinterpret_cast<float4_t *>(&o_part[w][16 * n + col][16 * i + 4 * g]) = o[n][i];
        }
        __syncthreads();
        const bool alone = u.begin == 0 && u.end == u.rounds;
        const int64_t slot0 = (int64_t)part_slot(deal, share, u.first_round) * kRows;
        const int part = min(lane & 15, WAVES - 1);      // lane i of 16 has what wave i knows of a row
        for (int r = w; r < here; r += WAVES) {
            const float level_mine = level_part[part][r], top_mine = top_part[part][r], sum_mine = (lane & 15) < WAVES ? sum_part[part][r] : 0.0f;
            const float t = row_max_16(top_mine), off = t == -INFINITY ? 0.0f : t, e = __builtin_amdgcn_exp2f(top_mine - off);
            const float total = row_sum_16(sum_mine == 0.0f ? 0.0f : sum_mine * e);
            const float over = total == 0.0f ? 0.0f : alone ? 1.0f / total : 1.0f;
            // nothing: of a wave that had no tokens, or of a row that sees none
            const bool none = sum_mine == 0.0f || e == 0.0f;
            const int high = (int)row_max_16(none ? -1000.0f : level_mine + (float)exponent_of(e));
            const float by = none ? 0.0f : __builtin_ldexpf(e, (int)level_mine - high);
            of.row(token0, head0, r, token, of_token);
            float *to_o = alone ? out + (int64_t)(first + token) * out_stride + (head * group + of_token) * kv.head_dim
                                : shares.sums + (slot0 + r) * kv.padded;
            float v[DT / 64] = {};
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                const float by_wave = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), k));
#pragma unroll
                for (int i = 0; i < DT / 64; i++)
                    v[i] = __builtin_fmaf(o_part[k][r][lane + 64 * i], by_wave, v[i]);
            }
#pragma unroll
            for (int i = 0; i < DT / 64; i++) {
                const int d = lane + 64 * i;
                v[i] = total == 0.0f ? 0.0f : __builtin_ldexpf(v[i] * over, high - 13);
                if (d < kv.head_dim) {
                    if (alone)
                        to_o[d] = v[i];
                    else
                        store_far(to_o + d, v[i]);
                }
            }
            if (!alone && lane < 2)
                store_far(&shares.tops[slot0 + r][lane], lane ? total : t);
        }
        if (shares.counters >= 0 && !alone) {
            // the parts are complete in memory before the workgroup counts itself
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const int share0 = deal.of(u.first_round), share1 = deal.of(u.first_round + u.rounds - 1);
            unsigned *const counter = &g_arrived[shares.counters][part_slot(deal, share0, u.first_round)];
            if (threadIdx.x == 0)
                is_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (unsigned)(share1 - share0 + 1);
            __syncthreads();
            if (is_last) {
                if (threadIdx.x == 0)
                    __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                join_unit<DT, kRows, false>(kv, shares, deal, u, share0, share1, of, out, out_stride, w, WAVES);
            }
        }
        round = u.first_round + u.end;
    }
}

// The parts of the units that several workgroups have: a workgroup for each that may have the first part of one.
template <int DT, int NB, int WAVES>
__global__ __launch_bounds__(256) void attention_few_join_kernel(Kv kv, Group of, float *__restrict__ out, int64_t out_stride, Shares shares)
{
    constexpr int kRows = 16 * NB, kStep = 64 * WAVES;
    const int group = of.size, share = blockIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Sequences<kRows, kStep> begin(kv, group, 0);
    const Deal deal(all_rounds(kv, group, begin), shares.count);
    const int stop = deal.start(share + 1);
    if (deal.start(share) >= stop)
        return;
    Finder<kRows, kStep> find(begin);
    const Part u = part_of(kv, group, find, stop - 1, stop);
    if (u.end == u.rounds || deal.of(u.first_round) != share)
        return;
    join_unit<DT, kRows, true>(kv, shares, deal, u, share, deal.of(u.first_round + u.rounds - 1), of, out, out_stride, w, 4);
}

// ---- many rows: every wave has 32 of them, and the waves of a workgroup share the tokens -------------------
//
// Bound by the matrix units, and by the power that they take: 2048 rows behind 14336 tokens, 32 heads of 128 on 8, take 888 to 950 us from card to card, 1.09
// to 1.16 PFLOP/s of fp16 products (two halves for each), where the library's product of 8192 x 8192 x 8192 makes 1.16 to 1.22; the clock is down to 1.6 GHz
// then, and nothing but those products, on such operands, takes 605 to 647 us.  A prompt of 4096: 258 to 276 us.  Vector work is nearly as much (ten
// operations a score, four of them the exponential) and goes on beside the products.  A tile of 64 tokens (32 above 128 dimensions, where registers are short) is made fp16 once for all
// waves, on its way into LDS; a tile is worked on while the next is written to the other half of LDS and the one behind it is on its way from
// memory.  Pieces of 8 dimensions (keys) and of 8 tokens (values) lie together there, [piece][token or dimension][8], so that a wave's operand is 512
// consecutive bytes for each half wave.  Where there are few tiles a workgroup's start and end are what counts (code read for the first time, q's way
// in, the results' out): 4 x 77 rows over 1500 tokens, 12 heads of 64, take 18.1 us, 3 x 201 rows over up to 1777, 20 heads of 80, 36.
//
// The sums are brought to a new maximum only where a row's has risen by more than 2^kSlack: until then its weights are up to 2^kSlack, for
// which the values' scales leave room (2^(kSlack + 10) is below fp16's largest number).
constexpr int kManyRows = 32;     // of a wave
constexpr float kSlack = 5.0f;
constexpr int kManyLevel = 9;     // the largest scale so far is brought to 2^9 .. 2^10
// Scales further below the largest than 2^kNear, zeros among them, or a largest one that has risen by more than 2^kRise, leave fp16 few bits for the rows
// that have no weight where the large ones are.  In such a tile each row is brought to where the largest product of a weight and a scale that it sees there is 2^14, as far as its
// sums stay within f32, for which 2^kMost leaves room.
constexpr int kNear = 10, kRise = 2, kMost = 110;

typedef float float16_t __attribute__((ext_vector_type(16)));

// What the waves of a workgroup share of a tile.
template <int DT, int TOKENS>
struct alignas(16) ManyTile {
    _Float16 keys[DT / 8][TOKENS][8];
    _Float16 values[TOKENS / 8][DT][8];
    float key_scale[TOKENS], value_scale[TOKENS];
    float minus[TOKENS];              // added to a token's scores: -infinity where there is none, NaN where a scale of it is no finite number
    int marked;                   // whether there is any such, 1; whether the values' scales are far apart, 2
    int level;                    // the values' scales are in units of 2^(level - kManyLevel)
};

// What __builtin_amdgcn_sched_group_barrier calls them.
constexpr int kSchedVector = 0x2, kSchedProduct = 0x8, kSchedRead = 0x100;

// SPLIT: whether tokens are split (a variant of its own: without, two prompts of 2500 with 16 heads of 256 take 317 us and not 327, the chunk 900 and not 905).
template <int DT, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, DT > 128 ? 1 : 2) void attention_many_kernel(Kv kv, const float *__restrict__ q, int64_t q_stride, Group of, float scale,
                                                                                     int causal, float *__restrict__ out, int64_t out_stride, Parts parts,
                                                                                     int aligned)
{
    constexpr int T = 64 * WAVES;
    constexpr int TOKENS = DT > 128 ? 32 : 64;             // of a tile: what the registers have room for
    constexpr int kPieces = DT / 16 * TOKENS;              // of 16 bytes: as many of keys as of values
    constexpr int kUnits = (kPieces + T - 1) / T;          // that a thread brings
    constexpr bool kWhole = kPieces % T == 0;
    constexpr int kBlocks = TOKENS / 32, kSteps = TOKENS / 16;
    // Two tiles.  Before them each wave's rows of q, and behind them its results: rows of DT + 4 floats.
    typedef ManyTile<DT, TOKENS> Tile;
    constexpr int kRows = kManyRows * WAVES;
    constexpr int kPitch = DT + 4;
    constexpr size_t kWaveBytes = kManyRows * kPitch * sizeof(float);
    constexpr size_t kBytes = 2 * sizeof(Tile) > WAVES * kWaveBytes ? 2 * sizeof(Tile) : WAVES * kWaveBytes;
    __shared__ __align__(16) char lds[kBytes];
    __shared__ float q_most[WAVES];
    __shared__ int q_below[kRows];      // how many powers of two a row's unit is below the workgroup's
    Tile *const tiles = reinterpret_cast<Tile *>(lds);

    const int group = of.size;
    // heads vary fastest: workgroups of one head meet in one L2 where their number is a multiple of eight; of a sequence's rows the last, which see most, go first
    const unsigned bh = blockIdx.x;
    const int split_at = SPLIT ? blockIdx.y : 0, b = (int)(bh / (unsigned)kv.kv_heads), head = (int)(bh - (unsigned)b * (unsigned)kv.kv_heads);
    int tile = parts.tiles - 1 - (int)blockIdx.z;
    int length, first, count;
    kv_sequence(kv, b, length, first, count);
    const int rows = count * group, tiles_here = (int)(((unsigned)rows + kRows - 1) / kRows);

    for (; tile < tiles_here; tile += parts.tiles) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));      // what follows from it is not kept in registers from one tile of rows to the next, of which there hardly is one
        const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int col = lane & 31, h = lane >> 5;
        const int row0 = tile * kRows + w * kManyRows;
        const int tile_token = (int)((unsigned)(tile * kRows) / (unsigned)group), tile_head = tile * kRows - tile_token * group;      // of the first row
        int token0, head0, last_token, of_last;      // of the wave's first row (where it has none, of the tile's last), and of the tile's last
        of.row(tile_token, tile_head, min(w * kManyRows, rows - tile * kRows - 1), token0, head0);
        of.row(tile_token, tile_head, min(kRows, rows - tile * kRows) - 1, last_token, of_last);
        const int keeper = rows - tile * kRows <= kRows - kManyRows ? WAVES - 1 : 0;      // makes the scales: the wave that has no rows, if there is one
        const int behind = max(min(kManyRows, rows - row0) - 1, 0);      // how far behind its first the wave's last row is
        const bool whole = !SPLIT || tile >= parts.tiles;
        if (whole && split_at)
            break;
        const int seen = causal ? max(length - count + last_token + 1, 0) : length;
        const int chunk = whole ? 0x7fffffc0 : chunk_of(parts, length);
        const int from = whole ? 0 : split_at * chunk;
        if (from >= seen && split_at)
            break;
        const int to = min(seen, whole ? seen : from + chunk);

        // ---- a tile on its way: which page, what piece
        int4_t keys[kUnits], values[kUnits];
        float key_scale, value_scale;
        bool is, first_tile = true;
        int level = -100, base = 127;      // the values' level, and what it was when all rows were last brought to it
        int unit_at;      // q is in units of 2^unit_at, which the keys' scales make up for
        // Where there is no token, or no dimension, any codes do: q or the weight is 0 there.
        const int32_t *const table = kv.table + (int64_t)b * kv.max_pages;
        const char *const first_page = kv.pages + (uint64_t)head * kv.head_bytes;
        int key_page, value_page[kUnits];      // looked up a tile before they are needed
        auto key_token = [&](int j0) { return (unsigned)min(j0 + lane % TOKENS, to - 1); };
        auto value_group = [&](int j0, int i) { return (unsigned)min(j0 + 16 * ((tid + T * i) / DT), to - 1) / 16; };
        auto look_up = [&](int j0) {
            key_page = table[kv_page_of(kv, key_token(j0) / 16)];
#pragma unroll
            for (int i = 0; i < kUnits; i++)
                if (kWhole || tid + T * i < kPieces)
                    value_page[i] = table[kv_page_of(kv, value_group(j0, i))];
        };
        auto fetch = [&](int j0) {
            const unsigned token = key_token(j0), slot = token - kv_page_of(kv, token / 16) * kv.page_size;
            const char *p = kv_page_or_any(kv, key_page, first_page, is);
#pragma unroll
            for (int i = 0; i < kUnits; i++)
                if (kWhole || tid + T * i < kPieces) {
                    const int c = (tid + T * i) / TOKENS;
                    keys[i] = *reinterpret_cast<const int4_t *>(p + kv_key_at(kv, 16 * c < kv.padded ? c : 0, slot));
                }
            const float *scales = reinterpret_cast<const float *>(p + kv_scales_at(kv)) + slot;
            is = is && j0 + lane % TOKENS < to;
            key_scale = scales[0];
            value_scale = scales[kv.page_size];
#pragma unroll
            for (int i = 0; i < kUnits; i++)
                if (kWhole || tid + T * i < kPieces) {
                    const int d = (tid + T * i) % DT;
                    const unsigned g = value_group(j0, i), place = g - kv_page_of(kv, g) * kv.page_groups;
                    bool any;
                    p = kv_page_or_any(kv, value_page[i], first_page, any);
                    values[i] = *reinterpret_cast<const int4_t *>(p + kv_value_at(kv, place, d < kv.padded ? d : 0));
                }
        };
        // half `part` of the codes of a thread's piece i, of keys or values
        auto store_part = [&](Tile &t, int i, int of_values, int part) {
            if (kWhole || tid + T * i < kPieces) {
                const int4_t &codes = of_values ? values[i] : keys[i];
                const half8_t eight = codes_to_half(codes[2 * part], codes[2 * part + 1]);
                if (of_values) {
                    const int g = (tid + T * i) / DT, d = (tid + T * i) % DT;
                    *reinterpret_cast<half8_t *>(&t.values[2 * g + part][d][0]) = eight;
                } else {
                    const int c = (tid + T * i) / TOKENS, token = lane % TOKENS;
                    *reinterpret_cast<half8_t *>(&t.keys[2 * c + part][token][0]) = eight;
                }
            }
        };
        auto store = [&](Tile &t) {
#pragma unroll
            for (int i = 0; i < 4 * kUnits; i++)
                store_part(t, i / 4, i / 2 % 2, i % 2);
        };
        auto store_scales = [&](Tile &t) {
            // a scale that is no finite number makes its token's score no number for the rows that see it, and is out of the way of the others
            const bool finite = fabsf(value_scale) < INFINITY && fabsf(key_scale) < INFINITY;
            t.key_scale[lane % TOKENS] = is ? __builtin_ldexpf(key_scale, unit_at) : 0.0f;
            value_scale = is && finite ? value_scale : 0.0f;
            t.minus[lane % TOKENS] = !is ? -INFINITY : finite ? 0.0f : NAN;
            const float size = fabsf(value_scale);
            level = max(level, exponent_of(wave_max(size)));
            t.value_scale[lane % TOKENS] = __builtin_ldexpf(value_scale, kManyLevel - level);
            base = first_tile ? level : base;
            first_tile = false;
            const bool apart = __any(is && exponent_of(size) < level - kNear) || level > base + kRise;
            base = apart ? level : base;
            const int marked = (__any(!is || !finite) ? 1 : 0) | (apart ? 2 : 0);
            if (lane == 0) {
                t.marked = marked;
                t.level = level;
            }
        };
        if (from < to) {
            look_up(from);
            fetch(from);
            look_up(from + TOKENS);
        }

        // ---- rows of q as halves, all in one unit but for small ones: rows into LDS as they are, and from there to the lanes, of which lane `col` gets 8 dimensions of
        // every 16 of a row
        float(*const own)[kPitch] = reinterpret_cast<float(*)[kPitch]>(lds + w * kWaveBytes);
        float most = 0.0f, least = INFINITY;      // of four values of a row that are not all 0, the largest
        {
            // as many lanes side by side as have a row in vectors of 16 bytes
            constexpr int kLanes = DT / 4, kTogether = 64 / kLanes, kLoads = kManyRows / (kTogether ? kTogether : 1);
            static_assert(DT / 4 <= 64, "a row in one instruction");
            const int lane_row = lane / kLanes, d = lane % kLanes * 4;
            if (aligned & 1) {
                float4_t v[kLoads];
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    const int r = i * kTogether + lane_row;
                    int token, of_token;      // of the last row, or of the first dimensions, where there is none
                    of.row(token0, head0, min(r, behind), token, of_token);
                    v[i] = *reinterpret_cast<const float4_t *>(q + (int64_t)(first + token) * q_stride + (head * group + of_token) * kv.head_dim +
                                                               (d < kv.head_dim ? d : 0));
                }
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    if (row0 + i * kTogether + lane_row >= rows || d >= kv.head_dim)
                        v[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
                    float size = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        size = fmaxf(size, fabsf(v[i][j]) < INFINITY ? fabsf(v[i][j]) : 0.0f);      // a row that is no number spoils no other
                    most = fmaxf(most, size);
                    least = size == 0.0f ? least : fminf(least, size);
                    if (lane_row < kTogether)
                        *reinterpret_cast<float4_t *>(&own[i * kTogether + lane_row][d]) = v[i];
                }
            } else {
                least = 0.0f;
#pragma unroll 1
                for (int r = 0; r < kManyRows; r++) {
                    int token, of_token;
                    of.row(token0, head0, min(r, behind), token, of_token);
                    const float *from_q = q + (int64_t)(first + token) * q_stride + (head * group + of_token) * kv.head_dim;
#pragma unroll 1
                    for (int at = lane; at < DT; at += 64) {
                        const float one = row0 + r < rows && at < kv.head_dim ? from_q[at] : 0.0f;
                        own[r][at] = one;
                        most = fmaxf(most, fabsf(one) < INFINITY ? fabsf(one) : 0.0f);
                    }
                }
            }
        }
        float to_exponents = scale;
        asm volatile("" : "+s"(to_exponents));      // nor this
        to_exponents *= kLog2e;
        most = wave_max(most);
        if (lane == 0)
            q_most[w] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++)
            most = fmaxf(most, q_most[i]);
        auto unit_for = [&](float size) { return exponent_of(fminf(size * fabsf(to_exponents), 0x1.fffffep127f)) - 14; };
        unit_at = __builtin_amdgcn_readfirstlane(unit_for(most));
        int below = 0;
        bool rows_apart = false;
        if (__builtin_expect(__any(exponent_of(least) < exponent_of(most) - kNear), 0)) {
            float size = 0.0f;
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const float4_t four = *reinterpret_cast<const float4_t *>(&own[col][16 * i + 8 * h + k]);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        size = fmaxf(size, fabsf(four[j]));
                }
            size = max_across_32(size);
            below = size == 0.0f ? 0 : unit_at - unit_for(size);
            below = below > kNear ? below : 0;
            rows_apart = __any(below);
            q_below[w * kManyRows + col] = below;
        }
        half8_t x[DT / 16][2];
#pragma unroll
        for (int i = 0; i < DT / 16; i++) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const float4_t four = *reinterpret_cast<const float4_t *>(&own[col][16 * i + 8 * h + k]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[k + j] = __builtin_ldexpf(four[j] * to_exponents, below - unit_at);
            }
            split(v, x[i][0], x[i][1]);
        }
        __syncthreads();

        int token, of_token, limit = to, all_see = to, any_sees = row0 >= rows ? 0 : to;      // tokens that a row, all rows of the wave, and any see
        if (causal) {
            of.row(token0, head0, min(col, behind), token, of_token);
            limit = min(length - count + token + 1, to);
            all_see = min(length - count + token0 + 1, to);
            of.row(token0, head0, behind, token, of_token);
            any_sees = row0 >= rows ? 0 : min(length - count + token + 1, to);
        }

        // `off` is what a row's scores are more than by kSlack at most; kNone before the row has seen a token
        constexpr float kNone = -INFINITY;
        float off = kNone, sum = 0.0f;
        float16_t o[DT / 32];
#pragma unroll
        for (int i = 0; i < DT / 32; i++)
#pragma unroll
            for (int k = 0; k < 16; k++)
                o[i][k] = 0.0f;
        int level_at = 0;

        if (from < to) {
            store(tiles[0]);
            if (w == keeper)
                store_scales(tiles[0]);
            fetch(from + TOKENS);
            look_up(from + 2 * TOKENS);
        }
        int which = 0;
        for (int j0 = from; j0 < to; j0 += TOKENS, which ^= 1) {
            const Tile &t = tiles[which];
            Tile &next = tiles[which ^ 1];
            __syncthreads();
            if (w == keeper)
                store_scales(next);
            if (j0 >= any_sees) {
                store(next);
                fetch(j0 + 2 * TOKENS);
                look_up(j0 + 3 * TOKENS);
                continue;
            }
            const int marked = __builtin_amdgcn_readfirstlane(t.marked), level_here = __builtin_amdgcn_readfirstlane(t.level);
            // S^T.  Row r of a product is the token with bits 2 and 3 of r exchanged: a lane then has 8 consecutive tokens for a step of the second
            // product.  Value k of block i is token 32 i + 16 (k / 8) + 8 h + k % 8.
            float16_t s[kBlocks];
            const int of_row = (col & 19) | ((col & 4) << 1) | ((col & 8) >> 1);
            // With the next tile's way into LDS beside them; operands are a step ahead of the products.
            {
                half8_t k[2][kBlocks];
                auto operand = [&](int d) {
#pragma unroll
                    for (int i = 0; i < kBlocks; i++)
                        k[d % 2][i] = *reinterpret_cast<const half8_t *>(&t.keys[2 * d + h][32 * i + of_row][0]);
                };
                operand(0);
#pragma unroll
                for (int d = 0; d < DT / 16; d++) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (d + 1 < DT / 16)
                        operand(d + 1);
#pragma unroll
                    for (int part = 0; part < 2; part++)
#pragma unroll
                        for (int i = 0; i < kBlocks; i++)
                            s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[d % 2][i], x[d][part], d || part ? s[i] : float16_t{}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4 * kUnits; i++)
                        if (i * (DT / 16) / (4 * kUnits) == d)
                            store_part(next, i / 4, i / 2 % 2, i % 2);
                    __builtin_amdgcn_sched_group_barrier(kSchedRead, kBlocks, 0);
#pragma unroll
                    for (int i = 0; i < 2 * kBlocks; i++) {
                        __builtin_amdgcn_sched_group_barrier(kSchedProduct, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(kSchedVector, 3, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (__builtin_expect(rows_apart, 0)) {
                // the lane counted anew, for want of registers
                const int below = q_below[w * kManyRows + __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)) % kManyRows];
#pragma unroll
                for (int i = 0; i < kBlocks; i++)
#pragma unroll
                    for (int k = 0; k < 16; k++)
                        s[i][k] = __builtin_ldexpf(s[i][k], -below);
            }
            // scores less `off`, and the largest of this lane's; a row's first scores are taken as they are
            const float less = off == kNone ? 0.0f : off;
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float4_t ks = *reinterpret_cast<const float4_t *>(&t.key_scale[32 * i + 16 * (k / 8) + 8 * h + k % 8]);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s[i][k + j] = __builtin_fmaf(s[i][k + j], ks[j], -less);
                }
            if (j0 + TOKENS > all_see || marked & 1) {
                const int until = limit - j0 - 8 * h;
#pragma unroll
                for (int i = 0; i < kBlocks; i++)
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        const int at = 32 * i + 16 * (k / 8) + k % 8;
                        const float4_t minus = *reinterpret_cast<const float4_t *>(&t.minus[at + 8 * h]);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            s[i][k + j] = at + j < until ? s[i][k + j] + minus[j] : -INFINITY;
                    }
            }
            float best = -INFINITY;
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int k = 0; k < 16; k++)
                    best = fmaxf(best, s[i][k]);
            const bool apart = marked & 2;
            if (__any(best > (off == kNone ? -INFINITY : kSlack)) || level_here != level_at || apart) {
                // A new maximum.  The scores are rounded once where they are brought to it by a difference, by 2^-24 of how far it has risen at most.
                const float top = max_across_32(best);
                float rise = off == kNone || top > kSlack ? top : 0.0f;
                if (__builtin_expect(apart, 0)) {
                    // what its scores are taken less is what a row's products want, not its weights: below the maximum where its values are small
                    float most = -INFINITY, size = 0.0f;
#pragma unroll
                    for (int i = 0; i < kBlocks; i++)
#pragma unroll
                        for (int k = 0; k < 16; k += 4) {
                            const float4_t vs = *reinterpret_cast<const float4_t *>(&t.value_scale[32 * i + 16 * (k / 8) + 8 * h + k % 8]);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                most = fmaxf(most, s[i][k + j] + __builtin_amdgcn_logf(fabsf(vs[j])));
                        }
#pragma unroll
                    for (int i = 0; i < DT / 32; i++)
#pragma unroll
                        for (int k = 0; k < 16; k++)
                            size = fmaxf(size, fabsf(o[i][k]));
                    const int up = level_here - level_at;
                    most = max_across_32(most);
                    most = most == -INFINITY ? (rise == 0.0f ? (float)-up : rise) : most - (float)min(14, kMost - level_here);
                    const int least = max(exponent_of(max_across_32(sum)) - kMost,
                                          exponent_of(max_across_32(size)) - up - min(kMost, kMost + 17 - level_here));
                    rise = fmaxf(fmaxf(most, top - kMost), off == kNone ? -INFINITY : (float)least);
                }
                // a row that has not seen a token has sums of 0 and scores of -infinity, and keeps them
                const float now = off == kNone && top == -INFINITY ? off : less + rise, keep = off == kNone ? 1.0f : __builtin_amdgcn_exp2f(off - now);
                // as much as `off` moves, but of scores with steps of more than 1 as much as the largest is above
                const float moves = now - less, further = now == kNone ? 0.0f : fabsf(moves - rise) < 1.0f ? moves : rise;
                off = now;
                sum *= keep;
                const float by = __builtin_ldexpf(keep, level_at - level_here);
                level_at = level_here;
#pragma unroll
                for (int i = 0; i < DT / 32; i++)
                    o[i] *= by;
#pragma unroll
                for (int i = 0; i < kBlocks; i++)
#pragma unroll
                    for (int k = 0; k < 16; k++)
                        s[i][k] -= further;
            }
            // O^T, 16 tokens a step.  Beside each product, in this order, a part of the next step's weights, and beside the last step's the loads
            // of a later tile: a product holds the vector units' issue for half of its time, which leaves room for four operations.
            constexpr int kSlots = DT / 16;      // products of a step
            half8_t p[2][2], v[2][DT / 32];
            float e[8], vs[8], of_tile = 0.0f;      // the tile's sum by itself: a long sequence's is rounded once a tile
            auto operand = [&](int step) {
#pragma unroll
                for (int c = 0; c < DT / 32; c++)
                    v[step % 2][c] = *reinterpret_cast<const half8_t *>(&t.values[2 * step + h][32 * c + col][0]);
            };
            auto scales_of = [&](int step) {
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const float4_t four = *reinterpret_cast<const float4_t *>(&t.value_scale[16 * step + 8 * h + k]);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        vs[k + j] = four[j];
                }
            };
            // weight k of a step: first its exponential, and one slot later (its result takes a while) the rest
            auto raise = [&](int step, int k) { e[k] = __builtin_amdgcn_exp2f(s[step / 2][8 * (step % 2) + k]); };
            auto weigh = [&](int step, int k) {
                of_tile += e[k];
                e[k] *= vs[k];
                if (k % 2)
                    split_two(e[k - 1], e[k], p[step % 2][0], p[step % 2][1], k / 2);
            };
            operand(0);
            scales_of(0);
#pragma unroll
            for (int k = 0; k < 8; k++)
                raise(0, k);
#pragma unroll
            for (int k = 0; k < 8; k++)
                weigh(0, k);
#pragma unroll
            for (int step = 0; step < kSteps; step++) {
                const bool last = step + 1 == kSteps;
                __builtin_amdgcn_sched_barrier(0);
                if (!last) {
                    operand(step + 1);
                    scales_of(step + 1);
                }
#pragma unroll
                for (int slot = 0; slot < kSlots; slot++) {
                    const int part = slot / (DT / 32), c = slot % (DT / 32);
                    o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[step % 2][c], p[step % 2][part], o[c], 0, 0, 0);
                    if (!last) {
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            if (k * kSlots / 8 == slot)
                                raise(step + 1, k);
                            if (k * kSlots / 8 + 1 == slot)
                                weigh(step + 1, k);
                        }
                        if (slot + 1 == kSlots)
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                if (k * kSlots / 8 + 1 == kSlots)
                                    weigh(step + 1, k);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (last) {
                    int from_here = __builtin_amdgcn_readfirstlane(j0);
                    asm volatile("" : "+s"(from_here));      // addresses are not made any earlier
                    fetch(from_here + 2 * TOKENS);
                    look_up(from_here + 3 * TOKENS);
#pragma unroll
                    for (int i = 0; i < kSlots; i++) {
                        __builtin_amdgcn_sched_group_barrier(kSchedProduct, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(kSchedVector, 5, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            sum += of_tile;
        }
        __syncthreads();      // the next tile of rows writes where this one reads

        sum = sum_across_32(sum);
        const bool alone = whole || chunk >= length;
        // results by way of LDS, so that rows are written whole, in vectors where they are aligned (parts always are)
        const float by = sum == 0.0f ? 0.0f : __builtin_ldexpf(alone ? 1.0f / sum : 1.0f, level_at - kManyLevel);
#pragma unroll
        for (int i = 0; i < DT / 32; i++)
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                float4_t v;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[j] = o[i][k + j] * by;
                *reinterpret_cast<float4_t *>(&own[col][32 * i + 2 * k + 4 * h]) = v;
            }
        const int64_t slot0 = (((int64_t)bh * parts.tiles + tile) * parts.splits + split_at) * kRows + w * kManyRows;
        if (!alone && h == 0 && row0 + col < rows) {
            parts.tops[slot0 + col][0] = off;
            parts.tops[slot0 + col][1] = sum;
        }
        __syncthreads();
        if (!alone || aligned & 2) {
            constexpr int kLanes = DT / 4, kTogether = 64 / kLanes;
            const int lane_row = lane / kLanes, d = lane % kLanes * 4;
            if (lane_row < kTogether && d < kv.head_dim)
#pragma unroll 4
                for (int r = lane_row; r < kManyRows; r += kTogether) {
                    if (row0 + r >= rows)
                        break;
                    of.row(token0, head0, r, token, of_token);
                    float *to_o = alone ? out + (int64_t)(first + token) * out_stride + (head * group + of_token) * kv.head_dim
                                        : parts.sums + (slot0 + r) * kv.padded;
                    *reinterpret_cast<float4_t *>(to_o + d) = *reinterpret_cast<const float4_t *>(&own[r][d]);
                }
        } else {
#pragma unroll 1
            for (int r = 0; r < min(kManyRows, rows - row0); r++) {
                of.row(token0, head0, r, token, of_token);
                float *to_o = out + (int64_t)(first + token) * out_stride + (head * group + of_token) * kv.head_dim;
#pragma unroll 1
                for (int at = lane; at < kv.head_dim; at += 64)
                    to_o[at] = own[r][at];
            }
        }
        __syncthreads();
    }
}

// Where the tokens of a tile of rows are split: what bounds it is two trips to memory, one for the sequence and one for the parts.  SHARE waves have
// the same rows and take turns with the parts where there are many.
template <int DT, int WAVES, int SHARE>
__global__ __launch_bounds__(256) void attention_many_join_kernel(Kv kv, Group of, int causal, float *__restrict__ out, int64_t out_stride, Parts parts,
                                                                  int aligned)
{
    constexpr int kRows = kManyRows * WAVES, kLanes = DT / 4, kTogether = 64 / kLanes, kAtOnce = 8;
    const unsigned bh = blockIdx.x;
    const int b = (int)(bh / (unsigned)kv.kv_heads), head = (int)(bh - (unsigned)b * (unsigned)kv.kv_heads), tile = blockIdx.z;
    int length, first, count;
    kv_sequence(kv, b, length, first, count);
    const int group = of.size, rows = count * group, chunk = chunk_of(parts, length);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane_row = lane / kLanes, d = lane % kLanes * 4;
    const int r = ((int)blockIdx.y * (4 / SHARE) + (SHARE == 1 ? w : 0)) * kTogether + lane_row, behind = min(kRows, rows - tile * kRows) - 1;
    if (chunk >= length || tile * kRows >= rows || r - lane_row > behind)
        return;      // there already, or no rows
    const int tile_token = (int)((unsigned)(tile * kRows) / (unsigned)group), tile_head = tile * kRows - tile_token * group;
    int token, of_token;
    of.row(tile_token, tile_head, behind, token, of_token);
    const int seen = causal ? max(length - count + token + 1, 0) : length;
    const int n = max((int)((unsigned)(seen + chunk - 1) / (unsigned)chunk), 1);
    const bool mine = lane_row < kTogether && r <= behind && d < kv.head_dim;
    const int64_t slot = ((int64_t)bh * parts.tiles + tile) * parts.splits * kRows + min(r, behind);
    Joined joined;
    joined.add<kAtOnce, true>(SHARE == 1 ? 0 : w * kAtOnce, n, kAtOnce * SHARE, parts.sums + (mine ? d : 0), kv.padded, parts.tops,
                              [&](int i) { return slot + (int64_t)i * kRows; });
    if (SHARE > 1) {
        __shared__ float4_t o_part[SHARE][64];
        __shared__ float top_part[SHARE][64], sum_part[SHARE][64];
        o_part[w][lane] = joined.o;
        top_part[w][lane] = joined.top;
        sum_part[w][lane] = joined.sum;
        __syncthreads();
        if (w)
            return;
        float top = -INFINITY;
        for (int i = 0; i < SHARE; i++)
            top = fmaxf(top, top_part[i][lane]);
        const float off = top == -INFINITY ? 0.0f : top;
        joined = Joined();
        for (int i = 0; i < SHARE; i++) {
            const float more = sum_part[i][lane], weight = more == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top_part[i][lane] - off);
            joined.sum = more == 0.0f ? joined.sum : __builtin_fmaf(more, weight, joined.sum);
            if (weight != 0.0f)
                joined.o += o_part[i][lane] * weight;
        }
    }
    of.row(tile_token, tile_head, min(r, behind), token, of_token);
    if (mine)
        joined.store(out + (int64_t)(first + token) * out_stride + (head * group + of_token) * kv.head_dim, d, kv.head_dim, aligned & 2);
}

// How a call is cut.
struct Plan {
    bool many;
    int tile_rows, tiles;
    int splits, chunk;      // many rows: of the tokens of a tile
    int waves;              // of a workgroup
    int shares;             // few rows
    size_t sums_bytes, tops_bytes;
    size_t bytes() const { return sums_bytes + tops_bytes; }
};

// VTL_HIP_OK and how, or why not.
int plan_of(const Kv &kv, const vtl_hip_kv_batch &b, int heads, Plan &p)
{
    p = Plan{};
    const int64_t most_rows = kv.starts ? (b.most_rows ? std::min(b.most_rows, kv.rows) : kv.rows) : 1;
    const int64_t most_length = std::max(b.most_length ? std::min(b.most_length, kv.most_tokens) : kv.most_tokens, 1);
    const int64_t group = heads / kv.kv_heads, rows = most_rows * group;
    if ((int64_t)kv.rows * heads > 0x7fffffc0 || (int64_t)heads * kv.head_dim > 0x7fffffc0)
        return VTL_HIP_ERR_UNSUPPORTED;
    // Up to 32 rows are few (16 above 128 dimensions, as many as the registers hold): 8 sequences of 3001 tokens with 16 heads of 64 values take 27.4 us with
    // 32 rows each, where the other kernel takes 47.6 with any number up to 128; of 128 values 50.4 and 65.5.  But 17 and more are many where there
    // is little to read for a compute unit, 256 tokens or, above 64 dimensions, where half as many waves have room, 1024: 20 sequences of 333, 24 rows each, 8 heads
    // of 128, take 21.8 us and 24.0, 20 of 1000 31.2 and 41.1, 45 of 1000 50.5 and 55.0; of 64 values 20 of 1000 22.3 and 17.8.
    p.many = rows > (kv.padded > 128 ? 16 : 32) ||
             (rows > 16 && (double)kv.batch * kv.kv_heads * (double)most_length <= 256.0 * (kv.padded > 64 ? 1024 : 256));
    // Many rows: eight waves share the codes that are made fp16 and brought to LDS once, and have a compute unit for themselves, where there is enough to do, four
    // tiles of tokens for each of them (a row sees half of its sequence's new tokens), and their rows do not lie idle.  2048 rows behind 14336 tokens, 32 heads of
    // 128 on 8: 905 us and 945 with four waves on the same card, a prompt of 4096 266 and 287, 512 rows behind 29500 442 and 519; but a prompt of
    // 1000 49.0 and 44.3, 40 rows over 3000 23.1 and 20.7, 4 x 70 over 3000 with 8 x 4 heads of 64 (three halves of tiles) 38.9 and 36.8.
    const int64_t halves = (rows + kManyRows * 4 - 1) / (kManyRows * 4);      // tiles of four waves' rows
    const double work = (double)kv.batch * kv.kv_heads * (double)((halves + 1) / 2) * (double)(most_length - std::min(most_rows, most_length) / 2);
    // a grid has less than 2^32 threads in a row
    const bool fits = (int64_t)kv.batch * kv.kv_heads * 64 * 8 <= 0xffffffff;
    p.waves = p.many && kv.padded <= 128 && fits && work >= 256 * 256 && (halves % 2 == 0 || halves > 8) ? 8 : 4;
    p.tile_rows = p.many ? kManyRows * p.waves : rows <= 16 ? 16 : 32;
    p.tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    int64_t units = (int64_t)kv.batch * kv.kv_heads * p.tiles;
    int64_t parts = 0;      // of rows that meet
    if (p.many) {
        // what a grid may have, and no more than a launch's worth where most_rows is not known; a workgroup goes on to the tiles behind
        const int64_t both = (int64_t)kv.batch * kv.kv_heads;
        if (both > 0xffffff)
            return VTL_HIP_ERR_UNSUPPORTED;
        p.tiles = (int)std::min<int64_t>(p.tiles, std::min<int64_t>(0xffff, std::max<int64_t>(1, kKvMostBlocks / both)));
        units = both * p.tiles;
        // Whatever has least to do one after the other.  Four waves: a workgroup for each compute unit or two, which take turns with its matrix units
        // (48 tiles of rows over 1500 tokens: 5 splits take 18.5 us, 8 take 19.2 and 12 take 24.2; 96 over 1777: 2 take 45.1 and 5 take 38.8).  Where a compute
        // unit has one, as many splits as fill them once or, of few, whose rounds leave fewer idle; a round's start and end count as 512 tokens
        // (1826 rows behind 11564 tokens, 20 heads of 64 on 4, 144 tiles: 417 us without splits, 311 with 5).  Not from 256
        // tiles on: as many short ones as long ones fill the last round where a prompt is causal.
        const bool alone = p.waves == 8 || kv.padded > 128;
        int64_t least = 0;
        auto consider = [&](int64_t n, int64_t turns, int64_t more) {
            const int64_t chunk = ((most_length + n - 1) / n + 63) / 64 * 64, cost = turns * (chunk + more);
            if (!least || cost < least) {
                least = cost;
                p.chunk = (int)chunk;
            }
        };
        if (alone && units > 32 && units < 256)
            for (int64_t n = 1; n <= 8; n++)
                consider(n, (units * n + 255) / 256, 512);
        else
            for (int each = 1; each <= (alone ? 1 : 2); each++)
                consider(std::max<int64_t>(1, 256 * each / units), each, 0);
        p.splits = (int)((most_length + p.chunk - 1) / p.chunk);
        parts = p.splits > 1 ? units * p.splits : 0;
    } else {
        // Eight waves, of which a unit has one workgroup, where they save the meeting of several (up to 512 tokens: 20 sequences with 8 heads of 128 values
        // and 500 tokens take 10.4 us, with four waves 13.7), where the parts to meet are many (a sequence of 20000: 22.1 and 23.5) or a tile has
        // half the bytes (8 sequences of 3001, 16 heads of 64 values: 17.7 and 18.8).  Else four, of which a compute unit has two workgroups that are not
        // in step (48 sequences of 6000: 64.7 and 69.6; 2 of 3000: 11.4 and 12.8).
        const bool eight = kv.padded <= 128 && (p.tile_rows == 16 || kv.padded <= 64);
        const bool better = most_length <= 512 || kv.padded <= 64 ? units <= 256 : units <= 32 && most_length > 15 * 256;
        p.waves = eight && better ? 8 : 4;
        const int64_t step = 64 * p.waves;
        // what the device counts in 32 bits
        if (((int64_t)kv.rows * group / p.tile_rows + kv.batch) * kv.kv_heads > kMostRounds / (kv.most_tokens / step + 1))
            return VTL_HIP_ERR_UNSUPPORTED;
        const int64_t at_once = p.waves == 8 || kv.padded > 128 || (kv.padded > 64 && p.tile_rows == 32) ? 256 : kMostShares;
        p.shares = (int)std::min(at_once, units * ((most_length + step - 1) / step));
        parts = p.shares > 1 ? 2 * p.shares : 0;
    }
    p.sums_bytes = ((size_t)parts * p.tile_rows * kv.padded * sizeof(float) + 255) & ~(size_t)255;
    p.tops_bytes = (size_t)parts * p.tile_rows * 2 * sizeof(float);
    return VTL_HIP_OK;
}

// The arguments that the kernels share.
struct Call {
    Kv kv;
    const float *q;
    int64_t q_stride;
    int heads;
    float scale;
    int causal;
    float *out;
    int64_t out_stride;
    Plan plan;
    float *sums;
    float (*tops)[2];
    // Whether rows can be read and written in vectors of 16 bytes.
    bool vectors(const float *p, int64_t stride) const { return kv.head_dim % 4 == 0 && stride % 4 == 0 && !(reinterpret_cast<uintptr_t>(p) & 15); }
};

template <int DT, int NB, int WAVES>
int launch_few(const Call &c)
{
    const Shares shares{c.plan.shares, c.sums ? stream_slot(current_stream()) : -1, c.sums, c.tops, c.vectors(c.out, c.out_stride)};
    const dim3 blocks((unsigned)c.plan.shares);
    hipLaunchKernelGGL((attention_few_kernel<DT, NB, WAVES>), blocks, dim3(64 * WAVES), 0, current_stream(), c.kv, c.q, c.q_stride,
                       Group(c.heads / c.kv.kv_heads), c.scale, c.causal, c.out, c.out_stride, shares);
    const int st = check_launch("attention_few_kernel");
    if (st != VTL_HIP_OK || !c.sums || shares.counters >= 0)
        return st;
    hipLaunchKernelGGL((attention_few_join_kernel<DT, NB, WAVES>), blocks, dim3(256), 0, current_stream(), c.kv,
                       Group(c.heads / c.kv.kv_heads), c.out, c.out_stride, shares);
    return check_launch("attention_few_join_kernel");
}

template <int DT, int WAVES>
int launch_many(const Call &c)
{
    const Parts parts{c.plan.tiles, c.plan.splits, c.plan.chunk, c.sums, c.tops};
    const Group of(c.heads / c.kv.kv_heads);
    const dim3 blocks((unsigned)(c.kv.batch * c.kv.kv_heads), (unsigned)c.plan.splits, (unsigned)c.plan.tiles);
    // rows that vectors of 16 bytes read, 1, and write, 2
    const int aligned = (c.vectors(c.q, c.q_stride) ? 1 : 0) | (c.vectors(c.out, c.out_stride) ? 2 : 0);
    hipLaunchKernelGGL((c.sums ? attention_many_kernel<DT, WAVES, true> : attention_many_kernel<DT, WAVES, false>), blocks, dim3(64 * WAVES), 0,
                       current_stream(), c.kv, c.q, c.q_stride, of, c.scale, c.causal, c.out, c.out_stride, parts, aligned);
    const int st = check_launch("attention_many_kernel");
    if (st != VTL_HIP_OK || !c.sums)
        return st;
    constexpr int kTogether = 256 / DT;      // rows of a wave
    auto join = [&](auto kernel, int at_once) {
        hipLaunchKernelGGL(kernel, dim3(blocks.x, (unsigned)(kManyRows * WAVES / at_once), blocks.z), dim3(256), 0, current_stream(), c.kv, of, c.causal,
                           c.out, c.out_stride, parts, aligned);
    };
    // many parts: 128 rows over 8000 tokens with one head of 64 are done after 16.2 us, with a wave for a row's parts after 25.9
    if (c.plan.splits > 16)
        join(attention_many_join_kernel<DT, WAVES, 4>, kTogether);
    else
        join(attention_many_join_kernel<DT, WAVES, 1>, 4 * kTogether);
    return check_launch("attention_many_join_kernel");
}

int launch_attention(const Call &c)
{
    const int padded = c.kv.padded;
    if (c.plan.many && c.plan.waves == 8)
        return padded <= 64 ? launch_many<64, 8>(c) : padded <= 96 ? launch_many<96, 8>(c) : launch_many<128, 8>(c);
    if (c.plan.many)
        return padded <= 64 ? launch_many<64, 4>(c) : padded <= 96 ? launch_many<96, 4>(c) : padded <= 128 ? launch_many<128, 4>(c) : launch_many<256, 4>(c);
    if (c.plan.tile_rows == 16) {
        if (c.plan.waves == 8)
            return padded <= 64 ? launch_few<64, 1, 8>(c) : launch_few<128, 1, 8>(c);
        return padded <= 64 ? launch_few<64, 1, 4>(c) : padded <= 128 ? launch_few<128, 1, 4>(c) : launch_few<256, 1, 4>(c);
    }
    if (c.plan.waves == 8)
        return launch_few<64, 2, 8>(c);
    return padded <= 64 ? launch_few<64, 2, 4>(c) : launch_few<128, 2, 4>(c);
}

bool attention_sizes_ok(const Kv &kv, int heads) { return heads >= 1 && heads % kv.kv_heads == 0; }

}  // namespace

extern "C" {

size_t vtl_hip_attention_i8_workspace(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, int heads)
{
    Kv kv;
    if (kv_sizes(cache, batch, kv) != VTL_HIP_OK || !attention_sizes_ok(kv, heads) || kv.rows == 0 || kv.batch == 0)
        return 0;
    Plan plan;
    return plan_of(kv, *batch, heads, plan) == VTL_HIP_OK ? plan.bytes() : 0;
}

int vtl_hip_attention_i8_f32(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, const float *q, int64_t q_stride, int heads,
                             float scale, int causal, float *out, int64_t out_stride, void *workspace, size_t workspace_bytes)
{
    Kv kv;
    const int st = kv_sizes(cache, batch, kv);
    if (st != VTL_HIP_OK)
        return st;
    if (!attention_sizes_ok(kv, heads) || !kv_stride_ok(kv, heads, q_stride) || !kv_stride_ok(kv, heads, out_stride))
        return VTL_HIP_ERR_INVALID_ARG;
    if (kv.rows == 0 || kv.batch == 0)
        return VTL_HIP_OK;
    if (!q || !out || meet(q, kv_span(kv, heads, q_stride), out, kv_span(kv, heads, out_stride)))
        return VTL_HIP_ERR_INVALID_ARG;
    Call call{kv, q, q_stride, heads, scale, causal, out, out_stride, {}, nullptr, nullptr};
    const int planned = plan_of(kv, *batch, heads, call.plan);
    if (planned != VTL_HIP_OK)
        return planned;
    const size_t need = call.plan.bytes();
    if (workspace && ((reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return VTL_HIP_ERR_INVALID_ARG;
    if (need) {
        if (!workspace)
            workspace = library_workspace(need);
        if (!workspace)
            return workspace_status();
        call.sums = static_cast<float *>(workspace);
        call.tops = reinterpret_cast<float(*)[2]>(static_cast<char *>(workspace) + call.plan.sums_bytes);
    }
    return launch_attention(call);
}

}  // extern "C"
