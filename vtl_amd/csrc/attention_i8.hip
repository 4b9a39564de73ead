// Attention over the int8 key/value cache for gfx950.
//
//   s_j = scale * sum_d q_d K_jd sk_j,   w = softmax over the tokens that the row sees,   o_d = sum_j w_j sv_j V_jd
//
// The codes K and V are whole numbers below 128, which fp16 holds exactly, so both products run on the fp16 matrix units with f32 sums.  What
// meets them is no whole number: q (with scale and log2 e) and w_j sv_j, two halves of 11 bits each, hi = f16(x), lo = f16(x - hi), one product
// for each.  So 22 bits of the operands enter, where one half alone would leave an error of 2^-11, and a third would cost half as much again.
// Rows of q are scaled by a power of two to a largest value between 2^14 and 2^15; the values' scales of a tile likewise (`Level`): lo keeps
// its bits down to 2^-16 of the largest, and is off by 2^-39 of it below that.
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

// The two halves of eight numbers.
__device__ __forceinline__ void split(const float *x, half8_t &hi, half8_t &lo)
{
    union {
        half2_t p[4];
        half8_t h;
    } a, b;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a.p[i] = __builtin_convertvector((float2_t{x[2 * i], x[2 * i + 1]}), half2_t);
        b.p[i] = __builtin_convertvector((float2_t{__builtin_fmaf((float)a.p[i][0], -1.0f, x[2 * i]), __builtin_fmaf((float)a.p[i][1], -1.0f, x[2 * i + 1])}),
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
__device__ __forceinline__ float max_across_32(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ int exponent_of(float v) { return (int)((__float_as_uint(v) >> 23) & 255) - 127; }

// The power of two that the values' scales are divided by, uniform in a wave: that of the largest of the tile's at hand.  It stays while the tile's
// is at most 2^6 below it (a change costs a pass over the sums), and rises no further than the sums, which grow when it falls, have room for.
struct Level {
    int at = -100;
    int room = 0;      // powers of two that the sums may have grown by

    // The new level for a tile whose largest scale is `most`; what the sums are multiplied by is 2^(old - new).
    __device__ __forceinline__ int next(float most, bool first)
    {
        const int tile = max(exponent_of(most), -100);
        if (first) {
            at = tile;
            return 0;
        }
        int by = tile > at ? tile - at : tile < at - 6 ? max(tile - at, room - 60) : 0;
        at += by;
        room = max(room - by, 0);
        return -by;
    }
};

// The launch as the host has planned it.
struct Parts {
    int tiles;      // of rows, in the sequence with the most
    int splits;     // of the tokens
    int chunk;      // tokens of a split; more where a sequence is longer than the host knew
    float *sums;    // [unit][split][row][head_dim]
    float2_t *tops; // [unit][split][row]: maximum, sum of weights
};

// Tokens of a split of a sequence of which `seen` are of use.
__device__ __forceinline__ int chunk_of(const Parts &parts, int seen)
{
    return max(parts.chunk, ((seen + parts.splits - 1) / parts.splits + 63) & ~63);
}

// ---- few rows: a tile's rows are 16 or 32, all of a sequence's that read one key/value head ------------
//
// Bound by the cache's bytes (2 D + 8 a token and head): so every wave takes tiles of 64 tokens for itself, straight from memory into the registers in
// the order in which the matrix units take them, a tile of keys on its way while the one before is worked on and its values behind it.
// Waves of a workgroup meet once, at the end.

template <int DT, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attention_few_kernel(Kv kv, const float *__restrict__ q, int64_t q_stride, int heads, float scale,
                                                                     int causal, float *__restrict__ out, int64_t out_stride, Parts parts)
{
    constexpr int kRows = 16 * NB;
    constexpr int kPitch = DT + 4;
    __shared__ __align__(16) _Float16 q_half[DT / 8][2][kRows][8];
    __shared__ float q_unit[kRows];
    __shared__ __align__(16) float o_part[WAVES / 2][kRows][kPitch];
    __shared__ float top_part[WAVES][kRows], sum_part[WAVES][kRows];
    __shared__ int level_part[WAVES];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int group = heads / kv.kv_heads;
    unsigned unit = blockIdx.x;
    const int split_at = unit % (unsigned)parts.splits;
    unit /= (unsigned)parts.splits;
    int tile = unit % (unsigned)parts.tiles;
    const int head = (unit / (unsigned)parts.tiles) % (unsigned)kv.kv_heads;
    const int b = unit / (unsigned)parts.tiles / (unsigned)kv.kv_heads;
    const int length = kv_length(kv, b);
    int first, count;
    kv_rows_of(kv, b, first, count);
    const int rows = count * group;      // the host has checked that all rows of all heads are below 2^31

    for (; tile * kRows < rows; tile += parts.tiles) {
        const int row0 = tile * kRows;
        const bool whole = tile >= parts.tiles;      // beyond what the host knew: in one piece
        if (whole && split_at)
            break;
        // the last token that the tile's last row sees
        const int last_row = min(row0 + kRows, rows) - 1;
        const int seen = causal ? max(length - count + last_row / group + 1, 0) : length;
        const int chunk = whole ? 0x7fffffc0 : chunk_of(parts, length);
        const int from = whole ? 0 : split_at * chunk;
        if (from >= seen && split_at)
            break;                                   // later tiles of the sequence see more, but they are beyond parts.tiles
        const int to = min(seen, whole ? seen : from + chunk);

        // ---- rows of q as halves
        for (int r = w; r < kRows; r += WAVES) {
            const int row = row0 + r;
            float x[DT / 64], most = 0.0f;
            const float *from_q = q + (int64_t)(first + row / group) * q_stride + (head * group + row % group) * kv.head_dim;
#pragma unroll
            for (int i = 0; i < DT / 64; i++) {
                const int d = lane + 64 * i;
                x[i] = row < rows && d < kv.head_dim ? from_q[d] * scale * kLog2e : 0.0f;
                most = fmaxf(most, fabsf(x[i]));
            }
            const int e = exponent_of(wave_max(most));
#pragma unroll
            for (int i = 0; i < DT / 64; i++) {
                const int d = lane + 64 * i;
                const float v = __builtin_ldexpf(x[i], 14 - e);
                const _Float16 hi = (_Float16)v;
                q_half[d / 8][0][r][d % 8] = hi;
                q_half[d / 8][1][r][d % 8] = (_Float16)(v - (float)hi);
            }
            if (lane == 0)
                q_unit[r] = __builtin_ldexpf(1.0f, e - 14);
        }
        __syncthreads();

        float unit_of[NB], top[NB], sum[NB];
        int limit[NB];
        float4_t o[NB][DT / 16];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const int row = min(row0 + 16 * n + col, rows - 1);
            unit_of[n] = q_unit[16 * n + col];
            limit[n] = causal ? min(length - count + row / group + 1, to) : to;
            top[n] = -INFINITY;
            sum[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                o[n][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        Level level;
        bool fresh = true;

        // Loads of a tile: pages of the 16 tokens whose keys, and whose scales and values, this lane takes.
        int4_t keys[4][DT / 64], values[DT / 16];
        const char *value_page;
        unsigned value_place;
        bool there;
        auto page_for = [&](int token, unsigned &place, bool &ok) -> const char * {
            const char *p = nullptr;
            place = 0;
            if (token < to)
                p = kv_group(kv, b, (unsigned)token / 16, head, place);
            ok = p != nullptr;
            if (!ok)
                place = 0;
            return ok ? p : kv.pages;
        };
        auto load_keys = [&](int j0) {
            unsigned place;
            bool ok;
            const char *page = page_for(j0 + 16 * (col >> 2), place, ok);
            const unsigned slot = place * 16 + (col & 3);
#pragma unroll
            for (int u = 0; u < DT / 64; u++) {
                const unsigned c = 16 * (4 * u + g) < kv.padded ? 4 * u + g : 0;     // behind the dimensions: any codes, q is 0 there
                const char *p = page + kv_key_at(kv, c, slot);
#pragma unroll
                for (int t = 0; t < 4; t++)
                    keys[t][u] = *reinterpret_cast<const int4_t *>(p + 64 * t);
            }
        };
        auto load_values = [&] {
            const char *p = value_page + kv_value_at(kv, value_place, 0);
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                if (16 * i < kv.padded)
                    values[i] = *reinterpret_cast<const int4_t *>(p + (16 * i + col) * 16);
        };

        const int step = 64 * WAVES;
        int j0 = from + 64 * w;
        if (j0 < to)
            load_keys(j0);
        for (; j0 < to; j0 += step) {
            asm volatile("" ::: "memory");      // q's halves are read again for every tile, not kept in registers
            value_page = page_for(j0 + 16 * g, value_place, there);
            load_values();
            const float *scales = reinterpret_cast<const float *>(value_page + kv_scales_at(kv)) + value_place * 16;
            float4_t ks[4], vs[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                ks[t] = reinterpret_cast<const float4_t *>(scales)[t];
                vs[t] = reinterpret_cast<const float4_t *>(scales + kv.page_size)[t];
            }

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
            if (j0 + step < to)
                load_keys(j0 + step);

            // scales of tokens that are none count for nothing
            const int mine = there ? j0 + 16 * g : 0x7fffffff;
            float most = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool is = mine < to - (4 * t + i);
                    vs[t][i] = is ? vs[t][i] : 0.0f;
                    most = fmaxf(most, fabsf(vs[t][i]) < INFINITY ? fabsf(vs[t][i]) : 0.0f);
                }
            most = max_across_32(max_across_16(most));      // the same in every lane of a column, and the columns hold the same
            const int moved = level.next(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(most))), fresh);
            fresh = false;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    vs[t][i] = __builtin_ldexpf(vs[t][i], 13 - level.at);

            half8_t p[NB][2][2];
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int until = limit[n];
                float best = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float v = s[n][t][i] * ks[t][i];
                        s[n][t][i] = mine < until - (4 * t + i) ? v : -INFINITY;
                        best = fmaxf(best, s[n][t][i]);
                    }
                best = max_across_32(max_across_16(best)) * unit_of[n];
                const float now = fmaxf(top[n], best);
                const float off = now == -INFINITY ? 0.0f : now;
                const float keep = __builtin_amdgcn_exp2f(top[n] - off);
                top[n] = now;
                float x[16], add = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][t][i], unit_of[n], -off));
                        add += e;
                        x[4 * t + i] = s[n][t][i] == -INFINITY ? 0.0f : e * vs[t][i];
                    }
                sum[n] = __builtin_fmaf(sum[n], keep, add);
                split(x, p[n][0][0], p[n][0][1]);
                split(x + 8, p[n][1][0], p[n][1][1]);
                const float by = __builtin_ldexpf(keep, moved);
#pragma unroll
                for (int i = 0; i < DT / 16; i++)
                    o[n][i] *= by;
            }
            // O^T: 64 tokens in two steps of 32, lane group g has 16 g + 8 step ..
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                if (16 * i < kv.padded)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const half8_t v = codes_to_half(values[i][2 * h], values[i][2 * h + 1]);
#pragma unroll
                        for (int n = 0; n < NB; n++)
#pragma unroll
                            for (int part = 0; part < 2; part++)
                                o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[n][h][part], o[n][i], 0, 0, 0);
                    }
        }

        // ---- the waves meet
        if (lane == 0)
            level_part[w] = fresh ? -1000 : level.at;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            sum[n] += __shfl_xor(sum[n], 16);
            sum[n] += __shfl_xor(sum[n], 32);
            if (g == 0) {
                top_part[w][16 * n + col] = top[n];
                sum_part[w][16 * n + col] = sum[n];
            }
        }
        __syncthreads();
        int high = -1000;
#pragma unroll
        for (int i = 0; i < WAVES; i++)
            high = max(high, level_part[i]);
        float all_top[NB], all_sum[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            all_top[n] = -INFINITY;
            all_sum[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; i++)
                all_top[n] = fmaxf(all_top[n], top_part[i][16 * n + col]);
            const float off = all_top[n] == -INFINITY ? 0.0f : all_top[n];
#pragma unroll
            for (int i = 0; i < WAVES; i++) {
                const float t = top_part[i][16 * n + col], v = sum_part[i][16 * n + col];
                all_sum[n] += v == 0.0f ? 0.0f : v * __builtin_amdgcn_exp2f(t - off);
            }
            const float by = fresh ? 0.0f : __builtin_ldexpf(__builtin_amdgcn_exp2f(top[n] - off), level.at - high);
#pragma unroll
            for (int i = 0; i < DT / 16; i++)
                o[n][i] = fresh ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : o[n][i] * by;
        }
        // half of them hand over to the other half, and so on
#pragma unroll
        for (int half = WAVES / 2; half; half /= 2) {
            if (w >= half && w < 2 * half)
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int i = 0; i < DT / 16; i++)
                        *reinterpret_cast<float4_t *>(&o_part[w - half][16 * n + col][16 * i + 4 * g]) = o[n][i];
            __syncthreads();
            if (w < half)
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int i = 0; i < DT / 16; i++)
                        o[n][i] += *reinterpret_cast<const float4_t *>(&o_part[w][16 * n + col][16 * i + 4 * g]);
            __syncthreads();
        }
        // one part, and it is the result; or the part of a split
        const bool alone = whole || chunk >= length;
        if (w == 0) {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int row = row0 + 16 * n + col;
                if (row >= rows)
                    continue;
                float *to_o;
                float by;
                if (alone) {
                    to_o = out + (int64_t)(first + row / group) * out_stride + (head * group + row % group) * kv.head_dim;
                    by = all_sum[n] == 0.0f ? 0.0f : 1.0f / all_sum[n];
                } else {
                    const int64_t slot = ((int64_t)unit * parts.splits + split_at) * kRows + 16 * n + col;
                    to_o = parts.sums + slot * kv.head_dim;
                    by = 1.0f;
                    if (g == 0)
                        parts.tops[slot] = float2_t{all_top[n], all_sum[n]};
                }
#pragma unroll
                for (int i = 0; i < DT / 16; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int d = 16 * i + 4 * g + k;
                        if (d < kv.head_dim)
                            to_o[d] = all_sum[n] == 0.0f ? 0.0f : __builtin_ldexpf(o[n][i][k] * by, high - 13);
                    }
            }
        }
        __syncthreads();
    }
}

// The parts of the rows whose tokens are split: a wave for each row and head.
__global__ __launch_bounds__(256) void attention_join_kernel(Kv kv, int heads, int causal, float *__restrict__ out, int64_t out_stride, Parts parts,
                                                             int tile_rows, unsigned units)
{
    const unsigned unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (unit >= units)
        return;
    const int lane = threadIdx.x & 63;
    const int h = unit % (unsigned)heads, row = unit / (unsigned)heads;
    int b, position;
    if (!kv_row(kv, row, b, position))
        return;
    int first, count;
    kv_rows_of(kv, b, first, count);
    const int group = heads / kv.kv_heads, length = kv_length(kv, b);
    const int mine = (row - first) * group + h % group, tile = mine / tile_rows;
    const int chunk = chunk_of(parts, length);
    if (tile >= parts.tiles || chunk >= length)
        return;                                         // there already
    const int last_row = min((tile + 1) * tile_rows, count * group) - 1;
    const int seen = causal ? max(length - count + last_row / group + 1, 0) : length;
    const int n = max((seen + chunk - 1) / chunk, 1);
    const int64_t slot = (((int64_t)b * kv.kv_heads + h / group) * parts.tiles + tile) * parts.splits * tile_rows + mine % tile_rows;
    float top = -INFINITY;
    for (int i = 0; i < n; i++)
        top = fmaxf(top, parts.tops[slot + (int64_t)i * tile_rows][0]);
    const float off = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, o[kKvMostDim / 64] = {};
    for (int i = 0; i < n; i++) {
        const int64_t at = slot + (int64_t)i * tile_rows;
        const float2_t t = parts.tops[at];
        const float by = __builtin_amdgcn_exp2f(t[0] - off);
        if (t[1] == 0.0f)
            continue;
        sum = __builtin_fmaf(t[1], by, sum);
#pragma unroll
        for (int k = 0; k < kKvMostDim / 64; k++)
            if (lane + 64 * k < kv.head_dim)
                o[k] = __builtin_fmaf(parts.sums[at * kv.head_dim + lane + 64 * k], by, o[k]);
    }
    float *y = out + (int64_t)row * out_stride + h * kv.head_dim;
#pragma unroll
    for (int k = 0; k < kKvMostDim / 64; k++)
        if (lane + 64 * k < kv.head_dim)
            y[lane + 64 * k] = sum == 0.0f ? 0.0f : o[k] / sum;
}

// How a call is cut: rows in tiles, tokens in splits.
struct Plan {
    int tile_rows, tiles, splits, chunk;
    int64_t units;      // (sequence, key/value head, tile)
    size_t sums_bytes, tops_bytes;
    size_t bytes() const { return sums_bytes + tops_bytes; }
};

Plan plan_of(const Kv &kv, const vtl_hip_kv_batch &b, int heads)
{
    Plan p{};
    const int64_t most_rows = kv.starts ? (b.most_rows ? std::min(b.most_rows, kv.rows) : kv.rows) : 1;
    const int64_t most_length = b.most_length ? std::min(b.most_length, kv.most_tokens) : kv.most_tokens;
    const int64_t rows = most_rows * (heads / kv.kv_heads);
    p.tile_rows = rows <= 16 || kv.padded > 128 ? 16 : 32;
    p.tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    p.units = (int64_t)kv.batch * kv.kv_heads * p.tiles;
    const int64_t wanted = std::max<int64_t>(1, 1024 / p.units);
    p.splits = (int)std::min(wanted, (most_length + 511) / 512);
    p.splits = std::max(p.splits, 1);
    p.chunk = (int)((((most_length + p.splits - 1) / p.splits) + 511) / 512 * 512);
    p.splits = (int)std::max<int64_t>(1, (most_length + p.chunk - 1) / p.chunk);
    if (p.splits > 1) {
        const size_t rows_in = (size_t)p.units * p.splits * p.tile_rows;
        p.sums_bytes = (rows_in * kv.head_dim * sizeof(float) + 255) & ~(size_t)255;
        p.tops_bytes = rows_in * sizeof(float2_t);
    }
    return p;
}

template <int DT, int NB, int WAVES>
void launch_few(const Kv &kv, const float *q, int64_t q_stride, int heads, float scale, int causal, float *out, int64_t out_stride,
                const Parts &parts, unsigned blocks)
{
    hipLaunchKernelGGL((attention_few_kernel<DT, NB, WAVES>), dim3(blocks), dim3(64 * WAVES), 0, current_stream(), kv, q, q_stride, heads, scale, causal,
                       out, out_stride, parts);
}

bool attention_sizes_ok(const Kv &kv, int heads) { return heads >= 1 && heads % kv.kv_heads == 0; }

}  // namespace

extern "C" {

size_t vtl_hip_attention_i8_workspace(const vtl_hip_kv_cache *cache, const vtl_hip_kv_batch *batch, int heads)
{
    Kv kv;
    if (kv_sizes(cache, batch, kv) != VTL_HIP_OK || !attention_sizes_ok(kv, heads) || kv.rows == 0 || kv.batch == 0)
        return 0;
    return plan_of(kv, *batch, heads).bytes();
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
    const int64_t row_heads = (int64_t)kv.rows * heads;
    const Plan plan = plan_of(kv, *batch, heads);
    if (row_heads > 0x7fffffc0 || plan.units * plan.splits > 0x7fffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    if (workspace && ((reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes()))
        return VTL_HIP_ERR_INVALID_ARG;
    Parts parts{plan.tiles, plan.splits, plan.chunk, nullptr, nullptr};
    if (plan.splits > 1) {
        if (!workspace)
            workspace = library_workspace(plan.bytes());
        if (!workspace)
            return workspace_status();
        parts.sums = static_cast<float *>(workspace);
        parts.tops = reinterpret_cast<float2_t *>(static_cast<char *>(workspace) + plan.sums_bytes);
    }
    const unsigned blocks = (unsigned)(plan.units * plan.splits);
    if (kv.padded <= 64) {
        if (plan.tile_rows == 16)
            launch_few<64, 1, 8>(kv, q, q_stride, heads, scale, causal, out, out_stride, parts, blocks);
        else
            launch_few<64, 2, 8>(kv, q, q_stride, heads, scale, causal, out, out_stride, parts, blocks);
    } else if (kv.padded <= 128) {
        if (plan.tile_rows == 16)
            launch_few<128, 1, 8>(kv, q, q_stride, heads, scale, causal, out, out_stride, parts, blocks);
        else
            launch_few<128, 2, 4>(kv, q, q_stride, heads, scale, causal, out, out_stride, parts, blocks);
    } else {
        launch_few<256, 1, 4>(kv, q, q_stride, heads, scale, causal, out, out_stride, parts, blocks);
    }
    const int launched = check_launch("attention_few_kernel");
    if (launched != VTL_HIP_OK || plan.splits == 1)
        return launched;
    hipLaunchKernelGGL(attention_join_kernel, dim3((unsigned)((row_heads + 3) / 4)), dim3(256), 0, current_stream(), kv, heads, causal, out, out_stride,
                       parts, plan.tile_rows, (unsigned)row_heads);
    return check_launch("attention_join_kernel");
}

}  // extern "C"
