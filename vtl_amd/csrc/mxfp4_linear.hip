// Linear layers on microscaled 4-bit rows (gfx950): y = x . W^T + bias with W as stored, [out_features, in_features], and x either codes
// too or f32 rows that become codes on the way.
#include <type_traits>
#include <utility>

#include "mxfp4.hpp"

using namespace vtlhip;
using namespace vtlhip::mx;

namespace {

struct Args {
    Rows a, w;            // [M, K], [N, K]
    const float *x;       // instead of a: f32 rows
    const float *bias;
    float *y;
    float *partials;      // [splits, M, N] sums of ranges of K, where there is more than one
    int M, N, K;
    int chunks;           // of a row
    int splits;
    int relu;
    int cached;           // results by way of the caches
    int slots;            // of a wave's shared memory
};

// Bias (0: none) and ReLU: what is below `floor` becomes 0 (NaN is not).
__device__ __forceinline__ float finish(float v, float bias, float floor)
{
    v = v + bias;
    return v < floor ? 0.0f : v;
}
__device__ __forceinline__ float floor_of(int relu) { return relu ? 0.0f : -__builtin_inff(); }

// ---- few rows ------------------------------------------------------------------------------

// A workgroup has 16 FR rows of weights and 4 MX rows of x; its waves deal the units of K out among them, each with two slots of shared memory
// that its own loads fill, and their sums meet in order.  The product's first operand is the weights, so a lane has four results of one row of x side by side.
// XF32: x is f32, and each wave makes the codes of its units itself.
// Bound by the weights' way from memory: one row and 28672 x 8192 weights 19.0 us, 6.6 TB/s with the last-level cache's part in it (eight waves a workgroup, and with them one workgroup a compute unit, 24.3);
// 14336 x 4096 7.0, 4.5 TB/s: it begins and ends.  From 17 rows on bound by x's way into shared memory too, four or eight times that of the weights: 32 rows and
// 4096 x 4096 4.2 us (one row 3.1), 4096 x 14336 9.4 (7.1).
constexpr int kFewMost = 16;     // rows up to which there is no other way

template <int FR, int MX, bool XF32>
struct Few {
    using W = Stream<FR>;
    static constexpr int kTiles = (MX + 3) / 4;                                     // of 16 columns
    static constexpr int kXBytes = 4 * MX * (kUnit / 2) + 256 * kTiles;             // rows of codes, then scales of whole tiles
    static constexpr int kSlot = W::kSlot + kXBytes, kLoads = W::kLoads + (XF32 ? 0 : MX + kTiles);
    static constexpr int kPart = 16 * FR + 4;                                       // floats of a row of sums
    static_assert(MX <= 4 || MX % 4 == 0, "whole tiles");
};

// Row m of x in a slot: codes like a row of weights (piece i at place i ^ m % 16), scales behind all of them.
template <int MX>
struct XRows {
    static constexpr int kScalesAt = 4 * MX * (kUnit / 2), kTiles = (MX + 3) / 4;
    v4f v[4 * MX][2];       // a lane's eight values of f32 rows; four lanes are a block

    __device__ __forceinline__ static void issue(const Args &g, int unit, char *x, unsigned pitch, unsigned spitch)
    {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int j = 0; j < MX; j++) {
            const int row = 4 * j + lane / 16;
            const unsigned in_row = min((unsigned)unit * (kUnit / 2) + (unsigned)((lane % 16) ^ (row % 16)) * 16u, pitch - 16u);
            __builtin_amdgcn_global_load_lds(VTL_GPTR(g.a.codes + ((size_t)min(row, g.M - 1) * pitch + in_row)), VTL_LPTR(x + j * 1024), 16, 0, 0);
        }
        const unsigned in_row = min((unsigned)unit * (kUnit / kBlock) + (unsigned)(lane % 4) * 4u, spitch - 4u);
#pragma unroll
        for (int j = 0; j < kTiles; j++)
            __builtin_amdgcn_global_load_lds(VTL_GPTR(g.a.scales + ((size_t)min(16 * j + lane / 4, g.M - 1) * spitch + in_row)), VTL_LPTR(x + kScalesAt + 256 * j), 4, 0, 0);
    }
    template <bool VEC>
    __device__ __forceinline__ void load(const Args &g, int unit)
    {
        const int col = unit * kUnit + 8 * (int)(threadIdx.x % kWave);
#pragma unroll
        for (int m = 0; m < 4 * MX; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                v[m][h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                const float *const row = g.x + (size_t)min(m, g.M - 1) * g.K;
                if constexpr (VEC) {
                    if (col + 4 * h < g.K)
                        v[m][h] = *reinterpret_cast<const v4f *>(row + col + 4 * h);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (col + 4 * h + i < g.K)
                            v[m][h][i] = row[col + 4 * h + i];
                }
            }
    }
    __device__ __forceinline__ void make_codes(char *x) const
    {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int m = 0; m < 4 * MX; m++) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 8; i++)
                top = max(top, __float_as_uint(v[m][i / 4][i % 4]) & 0x7fffffffu);
            top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
            top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
            const unsigned byte = scale_byte(top);
            const float s = byte == 255 ? 1.0f : scale_of(byte);
            unsigned q = 0;
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[m][0][0], v[m][0][1], s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[m][0][2], v[m][0][3], s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[m][1][0], v[m][1][1], s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[m][1][2], v[m][1][3], s, 3);
            *reinterpret_cast<unsigned *>(x + m * (kUnit / 2) + (((lane / 4) ^ m) << 4) + lane % 4 * 4) = byte == 255 ? 0u : q;
            if (lane % 4 == 0)
                x[kScalesAt + m * 16 + lane / 4] = (char)byte;
        }
    }
};

template <int FR, int MX, bool XF32, bool VEC, int NW>
__global__ __launch_bounds__(64 * NW) void linear_few_mxfp4_kernel(Args g)
{
    using F = Few<FR, MX, XF32>;
    using W = typename F::W;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane % 16, q = lane / 16;
    const int blocks = (g.N + 16 * FR - 1) / (16 * FR), n0 = (int)blockIdx.x % blocks * 16 * FR;
    if constexpr (MX == 8) {        // more rows than these: blocks of them
        const int m0 = (int)blockIdx.x / blocks * 4 * MX;
        g.a.codes += (size_t)m0 * g.chunks * kChunkCodes;
        g.a.scales += (size_t)m0 * g.chunks * kChunkScales;
        g.y += (size_t)m0 * g.N;
        g.M = min(g.M - m0, 4 * MX);
    }
    const int units = (g.chunks + 1) / 2, begin = (int)((int64_t)units * w / NW), end = (int)((int64_t)units * (w + 1) / NW);
    char *const ring = smem + w * g.slots * F::kSlot;
    W weights;
#pragma unroll
    for (int f = 0; f < FR; f++)
        weights.rows(f, g.w, (size_t)min(n0 + 16 * f, g.N - 1), min(16, max(1, g.N - n0 - 16 * f)), g.chunks);
    XRows<MX> rows;
    // (f32 rows in front of the weights: what arrives first is worked on first)
    auto issue = [&](int u) {
        char *const slot = ring + (u - begin) % 2 * F::kSlot;
        if constexpr (XF32)
            rows.template load<VEC>(g, u);
        weights.issue(u, slot);
        if constexpr (!XF32)
            rows.issue(g, u, slot + W::kSlot, weights.pitch, weights.spitch);
    };
    v4f acc[FR][F::kTiles];
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int j = 0; j < F::kTiles; j++)
            acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (begin < end)
        issue(begin);
    const int m = r % (4 * MX);      // (columns of no row repeat others)
    for (int u = begin; u < end; u++) {
        char *const slot = ring + (u - begin) % 2 * F::kSlot, *const x = slot + W::kSlot;
        if constexpr (XF32)
            rows.make_codes(x);
        if (u + 1 < end) {
            issue(u + 1);
            wait_vmcnt<F::kLoads>();
        } else {
            wait_vmcnt<0>();
        }
        const bool two = 2 * u + 1 < g.chunks;  // the second half of the last unit may be missing
        v4i sw[FR];
#pragma unroll
        for (int i = 0; i < FR; i++)
            sw[i] = W::all_scales(slot, i);
        v4i sx[F::kTiles];
#pragma unroll
        for (int j = 0; j < F::kTiles; j++)
            sx[j] = *reinterpret_cast<const v4i *>(x + XRows<MX>::kScalesAt + (16 * j + m) * 16);
#pragma unroll
        for (int s = 0; s < kUnitSteps; s++)
            if (s < 2 || two) {
                v4i cw[FR];
#pragma unroll
                for (int i = 0; i < FR; i++)
                    cw[i] = W::operand(slot, i, s);
#pragma unroll
                for (int j = 0; j < F::kTiles; j++) {
                    const v4i cx = *reinterpret_cast<const v4i *>(x + (16 * j + m) * (kUnit / 2) + (((4 * s + q) ^ m) << 4));
#pragma unroll
                    for (int i = 0; i < FR; i++)
                        acc[i][j] = mfma_16(cw[i], cx, acc[i][j], sw[i][s], (int)((unsigned)sx[j][s] >> (8 * q)));
                }
            }
        W::done_reading();
    }
    settle();
    __syncthreads();        // every wave is done with its slots
    float *const part = reinterpret_cast<float *>(smem);     // [waves][4 MX][kPart]
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int j = 0; j < F::kTiles; j++)
            if (r < 4 * MX)
                *reinterpret_cast<v4f *>(part + (w * 4 * MX + 16 * j + r) * F::kPart + 16 * i + 4 * q) = acc[i][j];
    __syncthreads();
    for (int item = (int)threadIdx.x; item < 4 * MX * 16 * FR; item += 64 * NW) {
        const int row = item / (16 * FR), nl = item % (16 * FR), n = n0 + nl;
        if (row >= g.M || n >= g.N)
            continue;
        float v = part[row * F::kPart + nl];
#pragma unroll
        for (int i = 1; i < NW; i++)
            v += part[(i * 4 * MX + row) * F::kPart + nl];
        g.y[(int64_t)row * g.N + n] = finish(v, g.bias ? g.bias[n] : 0.0f, floor_of(g.relu));
    }
}

// Value c of lane i of four becomes value i of lane c.
__device__ __forceinline__ void exchange(v4f &v)
{
    const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
    auto from = [](float x, auto control) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(control)::value, 0xF, 0xF, false)); };
    float x[4];
#pragma unroll
    for (int c = 0; c < 4; c += 2) {       // with the neighbour
        const float got = from(odd ? v[c] : v[c + 1], std::integral_constant<int, 0xB1>{});
        x[c] = odd ? got : v[c];
        x[c + 1] = odd ? v[c + 1] : got;
    }
#pragma unroll
    for (int c = 0; c < 2; c++) {          // and with the one behind it
        const float got = from(upper ? x[c] : x[c + 2], std::integral_constant<int, 0x4E>{});
        v[c] = upper ? got : x[c];
        v[c + 2] = upper ? x[c + 2] : got;
    }
}

// f(0), f(1) and so on with the numbers as constants: what the compiler leaves as a loop where it finds the body too large would keep the
// accumulators in memory.
template <typename F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}

// ---- many rows -----------------------------------------------------------------------------

// 16-byte pieces of a tile's rows of 128 bytes are put where a wave's read of 32 rows meets every bank as often.
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// A workgroup has a tile of BM x BN outputs, WR x WC waves a part of it each.  A chunk of K of both operands, 128 bytes of codes and 8 of
// scales a row, goes from memory straight into shared memory, STAGES chunks on their way; a lane of the 32x32x64 product takes a block
// of 16 bytes and its scale byte.  Operands are read one of the chunk's four steps ahead.  The barrier between two chunks comes in front of a chunk's last step, so that
// its latency, the first reads of the next chunk and the loads into the stage that became free hide behind that step's products: a read and its
// share of the loads behind each of them, in this order, because loads in one burst wait for each other in front of the unit that makes their addresses.
// Tiles of 256 x 256 are bound by power: 8192 x 8192 x 8192 265 to 286 us from card to card, 3.8 to 4.15 PFLOP/s; 1.68 us a chunk, of which the products alone take 1.34 on random codes (reads left out
// 1.49, loads left out 1.43).  Smaller ones by their operands' way from the L2 into shared memory, with these loads some 22 bytes a cycle of a compute unit whatever
// the tile: 201 x 11008 x 4096 15.6 us.
template <int BM, int BN, int WR, int WC, int STAGES, int SPREAD, bool EDGE>
struct Tile {
    static constexpr int kWaves = WR * WC, kThreads = 64 * kWaves;
    static constexpr int WM = BM / WR, WN = BN / WC, TM = WM / 32, TN = WN / 32;
    static constexpr int kALoads = BM / 8 / kWaves, kBLoads = BN / 8 / kWaves;        // a wave's load: 8 rows of codes
    // or the scales of 32 rows (8 where rows of scales may end in the middle of a load)
    static constexpr bool kWide = !EDGE && (BM + BN) / 4 % (32 * kWaves) == 0;
    static constexpr int kSRows = kWide ? 32 : 8, kSAll = (BM + BN) / 4 / kSRows, kSLoads = (kSAll + kWaves - 1) / kWaves;
    static constexpr int kLoads = kALoads + kBLoads + kSLoads;
    static constexpr int kStage = (BM + BN) * kChunkCodes;
    // Scales come for kGroup chunks at once, 32 bytes of a row (of each 8 bytes a request would be one for a line of its own, as many as
    // for the codes: 37.8 million requests to the L2 caches for 8192 x 8192 x 8192, so 25.7), a quarter of the rows with the codes of each chunk; the last quarter of a group with those of its first chunk.
    static constexpr int kGroup = 4, kGroupRow = kGroup * kChunkScales, kScales = (BM + BN) * kGroupRow;
    static constexpr int kBuffers = STAGES >= 3 ? 3 : 2;   // of scales: the next group is being loaded up to STAGES + 3 chunks ahead
    static constexpr int kLds = STAGES * kStage + kBuffers * kScales;
    static constexpr int kSteps = kChunk / 64;
    static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && (BM + BN) % (4 * kSRows) == 0, "loads are dealt out evenly");
    static_assert(STAGES >= 2 && STAGES <= 5 && (STAGES - 1) * kLoads <= 63, "the counter of loads has 6 bits");
};

template <int BM, int BN, int WR, int WC, int STAGES, int SPREAD, bool EDGE>
__global__ __launch_bounds__(64 * WR * WC) void linear_tile_mxfp4_kernel(const Args g)
{
    using T = Tile<BM, BN, WR, WC, STAGES, SPREAD, EDGE>;
    constexpr int TM = T::TM, TN = T::TN, NW = T::kWaves, kSteps = T::kSteps, kLoads = T::kLoads;
    constexpr bool kWide = T::kWide;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int split = (int)(blockIdx.x % (unsigned)g.splits);
    int tile_m, tile_n;
    tile_of_block((g.M + BM - 1) / BM, (g.N + BN - 1) / BN, (int)(blockIdx.x / (unsigned)g.splits), tile_m, tile_n);
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int lane = threadIdx.x % kWave, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wr = w / WC, wc = w % WC;
    const int begin = (int)((int64_t)g.chunks * split / g.splits), end = (int)((int64_t)g.chunks * (split + 1) / g.splits);
    const int count = end - begin;
    const unsigned pitch = (unsigned)g.chunks * kChunkCodes, spitch = (unsigned)g.chunks * kChunkScales;

    // A load's address: a uniform base (operand, the tile's first row, the chunk and, without EDGE, the load's rows) and the lane's offset from it,
    // at most 255 rows.  With EDGE rows past the last are that one, and offsets differ from load to load.
    const int lrow = 8 * w + lane / 8;                    // of the first load's rows: + 8 NW from one to the next, which keeps the swizzle
    const unsigned lpiece = (unsigned)((lane % 8) ^ swizzle(lrow)) * 16u;
    static_assert(8 * NW % 16 == 0, "rows 16 apart share the swizzle");
    const uint8_t *const a0 = g.a.codes + (size_t)m0 * pitch + (size_t)begin * kChunkCodes;
    const uint8_t *const b0 = g.w.codes + (size_t)n0 * pitch + (size_t)begin * kChunkCodes;
    unsigned oa[EDGE ? T::kALoads : 1], ob[EDGE ? T::kBLoads : 1];
    if constexpr (EDGE) {
#pragma unroll
        for (int j = 0; j < T::kALoads; j++)
            oa[j] = (unsigned)min(lrow + 8 * NW * j, g.M - 1 - m0) * pitch + lpiece;
#pragma unroll
        for (int j = 0; j < T::kBLoads; j++)
            ob[j] = (unsigned)min(lrow + 8 * NW * j, g.N - 1 - n0) * pitch + lpiece;
    } else {
        oa[0] = ob[0] = (unsigned)lrow * pitch + lpiece;
    }
    char *const scales_at = smem + STAGES * T::kStage;
    // Of 8 rows of the tile (32 where kWide) from `row` on (first those of x, then those of the weights), the scales of a group.
    auto load_scales = [&](int group, int row) {
        const bool of_a = row < BM;
        const int first = of_a ? m0 + row : n0 + row - BM;
        // (the group behind the last one is asked for too: it is the last one once more)
        const int at = kWide ? min(group, g.chunks / T::kGroup - 1) * T::kGroup : begin + group * T::kGroup;
        const uint8_t *const base = (of_a ? g.a.scales : g.w.scales) + (int64_t)first * spitch + at * kChunkScales;
        char *const to = scales_at + group % T::kBuffers * T::kScales + row * T::kGroupRow;
        if constexpr (kWide) {
            __builtin_amdgcn_global_load_lds(VTL_GPTR(base + ((unsigned)(lane / 2) * spitch + (unsigned)(lane % 2 * 16))), VTL_LPTR(to), 16, 0, 0);
        } else {
            const int up = min(lane / 8, (of_a ? g.M : g.N) - 1 - first);       // (below 0 where all of them are past the last)
            const int in_row = min(lane % 8 * 4, (int)spitch - 4 - at * kChunkScales);
            __builtin_amdgcn_global_load_lds(VTL_GPTR(base + ((int64_t)up * spitch + in_row)), VTL_LPTR(to), 4, 0, 0);
        }
    };
    auto load = [&](int d, int chunk, int stage) {
        char *const base = smem + stage * T::kStage;
        if (d < T::kALoads) {
            const uint8_t *const p = a0 + (size_t)chunk * kChunkCodes + (EDGE ? 0 : (size_t)(8 * NW * d) * pitch) + oa[EDGE ? d : 0];
            __builtin_amdgcn_global_load_lds(VTL_GPTR(p), VTL_LPTR(base + 8 * (w + NW * d) * kChunkCodes), 16, 0, 0);
        } else if (d < T::kALoads + T::kBLoads) {
            const int j = d - T::kALoads;
            const uint8_t *const p = b0 + (size_t)chunk * kChunkCodes + (EDGE ? 0 : (size_t)(8 * NW * j) * pitch) + ob[EDGE ? j : 0];
            __builtin_amdgcn_global_load_lds(VTL_GPTR(p), VTL_LPTR(base + (BM + 8 * (w + NW * j)) * kChunkCodes), 16, 0, 0);
        } else {
            const int from = chunk + T::kGroup - 1, group = from / T::kGroup;
            load_scales(group, from % T::kGroup * ((BM + BN) / T::kGroup) + T::kSRows * min(w + NW * (d - T::kALoads - T::kBLoads), T::kSAll - 1));
        }
    };
    auto issue = [&](int chunk, int stage) {
#pragma unroll
        for (int d = 0; d < kLoads; d++)
            load(d, chunk, stage);
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
    unsigned at[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++)
        at[s] = (unsigned)(r * kChunkCodes + (((2 * s + half) ^ swizzle(r)) << 4));
    v4i fa[2][TM], fb[2][TN];
    v2u raw[TM + TN];               // a chunk's scales as they lie in shared memory, and as the products take them: byte s for step s
    unsigned scale[TM + TN];
    // Read i of a step: the columns' operands first, then the rows', which the products below take in this order; then, for a chunk's first step,
    // the scales.
    constexpr int kReads = TM + TN;
    auto read = [&](int i, int chunk, int stage, int s, int buffer) {
        const char *const base = smem + stage * T::kStage;
        const char *const scales = scales_at + chunk / T::kGroup % T::kBuffers * T::kScales + chunk % T::kGroup * kChunkScales;
        if (i < TN)
            fb[buffer][i] = *reinterpret_cast<const v4i *>(base + (BM + wc * T::WN + 32 * i) * kChunkCodes + at[s]);
        else if (i < kReads)
            fa[buffer][i - TN] = *reinterpret_cast<const v4i *>(base + (wr * T::WM + 32 * (i - TN)) * kChunkCodes + at[s]);
        else if (i < kReads + TN)
            raw[TM + i - kReads] = *reinterpret_cast<const v2u *>(scales + (BM + wc * T::WN + 32 * (i - kReads) + r) * T::kGroupRow);
        else
            raw[i - kReads - TN] = *reinterpret_cast<const v2u *>(scales + (wr * T::WM + 32 * (i - kReads - TN) + r) * T::kGroupRow);
    };
    // Step s of a chunk, with the reads of the step behind it and loads d0 .. d1 - 1 of chunk `chunk` between its products.
    auto step = [&](auto s_t, auto d0_t, auto d1_t, auto last_t, int read_chunk, int read_stage, int chunk, int stage) {
        constexpr bool kLast = decltype(last_t)::value;    // no step behind it
        constexpr int s = decltype(s_t)::value, next = (s + 1) % kSteps, buffer = s & 1, d0 = decltype(d0_t)::value, d1 = decltype(d1_t)::value;
        constexpr int kProducts = TM * TN, kAll = next == 0 ? 2 * kReads : kReads, kEach = (kAll + kProducts - 1) / kProducts;
        constexpr int kShare = (d1 - d0 + kProducts - 1) / kProducts;
        if constexpr (s == 0) {
#pragma unroll
            for (int i = 0; i < TM + TN; i++)
                scale[i] = __builtin_amdgcn_perm(raw[i][1], raw[i][0], pick);
        }
        __builtin_amdgcn_sched_barrier(0);
        each([&](auto p_t) {
            constexpr int p = decltype(p_t)::value;
            const v4i a = fa[buffer][p / TN], b = fb[buffer][p % TN];
            acc[p / TN][p % TN] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}, v8i{b[0], b[1], b[2], b[3], 0, 0, 0, 0},
                                                                                 acc[p / TN][p % TN], 4, 4, s, (int)scale[p / TN], s, (int)scale[TM + p % TN]);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!kLast) {
#pragma unroll
                for (int i = 0; i < kEach; i++)
                    if (p * kEach + i < kAll)
                        read(p * kEach + i, read_chunk, read_stage, next, buffer ^ 1);
            }
#pragma unroll
            for (int i = 0; i < kShare; i++)
                if (d0 + p * kShare + i < d1)
                    load(d0 + p * kShare + i, chunk, stage);
            __builtin_amdgcn_sched_barrier(0);
        }, std::make_integer_sequence<int, kProducts>{});
    };

    if (count > 0) {
#pragma unroll
        for (int i = 0; i < (T::kGroup - 1) * T::kSLoads; i++)     // the other quarters of the first group
            load_scales(0, i / T::kSLoads * ((BM + BN) / T::kGroup) + T::kSRows * min(w + NW * (i % T::kSLoads), T::kSAll - 1));
    }
#pragma unroll
    for (int s = 0; s < STAGES; s++)
        if (s < count)
            issue(s, s);
    if (count >= STAGES)
        wait_vmcnt<(STAGES - 1) * kLoads>();
    else
        wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    if (count > 0) {
#pragma unroll
        for (int i = 0; i < 2 * kReads; i++)
            read(i, 0, 0, 0, 0);
    }
    int stage = 0;
    using Yes = std::true_type;
    using No = std::false_type;
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    // A chunk but the last.  The stage that it leaves takes chunk c + STAGES: the first share of its loads in this chunk's last step (MORE), the
    // others in the first steps of the next chunk (REST).
    auto chunk_steps = [&](auto rest_t, auto more_t, int c) {
        constexpr bool kRest = decltype(rest_t)::value && SPREAD > 1, kMore = decltype(more_t)::value;
        const int before = stage == 0 ? STAGES - 1 : stage - 1;
        using First = std::integral_constant<int, kLoads / SPREAD>;
        using Second = std::integral_constant<int, kRest ? 2 * kLoads / SPREAD : kLoads / SPREAD>;
        using All = std::integral_constant<int, kRest ? kLoads : kLoads / SPREAD>;
        step(I0{}, First{}, Second{}, No{}, c, stage, c - 1 + STAGES, before);
        step(I1{}, Second{}, All{}, No{}, c, stage, c - 1 + STAGES, before);
        step(I2{}, I0{}, I0{}, No{}, c, stage, 0, 0);
        // every read of this chunk has been asked for: wait for them, see that the next one has arrived, and hand this one's stage over
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        if (kMore || c + STAGES - 1 < count)
            wait_vmcnt<(STAGES - 2) * kLoads>();
        else
            wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        step(I3{}, I0{}, std::integral_constant<int, kMore ? kLoads / SPREAD : 0>{}, No{}, c + 1, next, c + STAGES, stage);
        stage = next;
    };
    int c = 0;
    if (STAGES < count) {
        chunk_steps(No{}, Yes{}, 0);
        for (c = 1; c + STAGES < count; c++)
            chunk_steps(Yes{}, Yes{}, c);
        chunk_steps(Yes{}, No{}, c);
        c++;
    }
    for (; c < count - 1; c++)
        chunk_steps(No{}, No{}, c);
    if (count > 0) {
        step(I0{}, I0{}, I0{}, No{}, c, stage, 0, 0);
        step(I1{}, I0{}, I0{}, No{}, c, stage, 0, 0);
        step(I2{}, I0{}, I0{}, No{}, c, stage, 0, 0);
        step(I3{}, I0{}, I0{}, Yes{}, 0, 0, 0, 0);
        settle();
    }

    // Register k of a lane is row 8 (k / 4) + 4 half + k % 4 of a 32 x 32 tile, column r.  Four lanes exchange theirs (lane i gets row i of four
    // columns), so that a store is 16 bytes a lane and 8 whole lines.  An address is a uniform row and the lane's offset from it.  Results are not
    // read again here.  Where all tiles are at work at once and store at the end, by way of the caches (4096 x 4096 x 4096: 41.3 us, else 43.6).  Else past them, and rows of 1024
    // bytes at a time where a tile has them: what memory takes of a matrix that no cache holds depends on that (8192 x 8192 f32 in tiles of 256 x 256, nothing
    // but stores: 8 rows of 128 bytes 76 us, 2 of 512 70, one of 1024 50; 4096 x 4096 11 each).  So 8192 x 8192 x 8192 takes 286 us for 295, 8192 x 28672 x 2048 368 for 396.
    const bool cached = g.cached;
    const bool whole = g.splits == 1;
    float *const out = (whole ? g.y : g.partials + (size_t)split * g.M * g.N) + (size_t)(m0 + wr * T::WM) * g.N + (n0 + wc * T::WN);
    const float floor = floor_of(whole && g.relu);
    const int n = n0 + wc * T::WN + r;
    float bias[TN];
#pragma unroll
    for (int j = 0; j < TN; j++)
        bias[j] = whole && g.bias && (!EDGE || n + 32 * j < g.N) ? g.bias[n + 32 * j] : 0.0f;
    const bool vectors = !EDGE || (g.N % 4 == 0 && !(reinterpret_cast<uintptr_t>(out) & 15));
    if constexpr (BN == 256 && !EDGE) {
        if (!cached) {
            // Rows of the tile by way of shared memory, 32 of each wave at a time: 16-byte piece i of row m lies at place i ^ 4 (m % 4), so that neither writes
            // of four rows nor reads of a whole one meet a bank twice.
            constexpr int kRows = 32 * WR, kEach = kRows / NW;
            static_assert(2 * kRows * BN * 4 <= T::kLds && kRows % NW == 0, "two turns' rows");
            float *const rows = reinterpret_cast<float *>(smem);
            const int turn = (r % 4) << 2;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TM; i++) {
                float *const at_i = rows + i % 2 * kRows * BN;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float *const to = at_i + (32 * wr + 8 * k + 4 * half + r % 4) * BN;
#pragma unroll
                    for (int j = 0; j < TN; j++) {
                        v4f v;
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            v[c] = finish(acc[i][j][4 * k + c], bias[j], floor);
                        exchange(v);
                        *reinterpret_cast<v4f *>(to + (((wc * T::WN + 32 * j) / 4 + r / 4) ^ turn) * 4) = v;
                    }
                    asm volatile("" ::: "memory");   // all results at once would be more registers than there are
                }
                __syncthreads();
                const int n4 = n0 + 4 * lane;
#pragma unroll 4
                for (int k = 0; k < kEach; k++) {
                    const int row = w * kEach + k, m = m0 + row / 32 * T::WM + 32 * i + row % 32;
                    const v4f v = *reinterpret_cast<const v4f *>(at_i + row * BN + (lane ^ ((row % 4) << 2)) * 4);
                    __builtin_nontemporal_store(v, reinterpret_cast<v4f *>(g.y + (size_t)m * g.N + n4));
                }
            }
            return;
        }
    }
    if (vectors) {
        const unsigned mine = (unsigned)(4 * half + r % 4) * (unsigned)g.N + (unsigned)(r & ~3);
        const int n4 = n0 + wc * T::WN + (r & ~3);
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int row = 32 * i + 8 * k;
                float *const to = out + (size_t)row * g.N + mine;
                const bool in = !EDGE || m0 + wr * T::WM + row + 4 * half + r % 4 < g.M;
#pragma unroll
                for (int j = 0; j < TN; j++) {
                    v4f v;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        v[c] = finish(acc[i][j][4 * k + c], bias[j], floor);
                    exchange(v);
                    if (in && (!EDGE || n4 + 32 * j < g.N)) {
                        if (cached)
                            *reinterpret_cast<v4f *>(to + 32 * j) = v;
                        else
                            __builtin_nontemporal_store(v, reinterpret_cast<v4f *>(to + 32 * j));
                    }
                }
                asm volatile("" ::: "memory");   // all results at once would be more registers than there are
            }
    } else {
        const unsigned mine = (unsigned)(4 * half) * (unsigned)g.N + (unsigned)r;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const int row = 32 * i + 8 * (k / 4) + k % 4;
                float *const to = out + (size_t)row * g.N + mine;
                if (m0 + wr * T::WM + row + 4 * half < g.M)
#pragma unroll
                    for (int j = 0; j < TN; j++)
                        if (n + 32 * j < g.N)
                            to[32 * j] = finish(acc[i][j][k], bias[j], floor);
                asm volatile("" ::: "memory");
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
        g.y[i] = finish(v, g.bias ? g.bias[i % (size_t)g.N] : 0.0f, floor_of(g.relu));
    }
}

// ---- host ----------------------------------------------------------------------------------

template <int BM, int BN, int WR, int WC, int STAGES, int SPREAD>
int launch_tile(Args g, hipStream_t st)
{
    using T = Tile<BM, BN, WR, WC, STAGES, SPREAD, true>;
    static_assert(T::kLds <= 160 << 10, "shared memory of a compute unit");
    static PerDevice<DoneFlag> done_flags[2];
    const bool edge = g.M % BM || g.N % BN || g.chunks % T::kGroup || g.splits > 1 || (reinterpret_cast<uintptr_t>(g.y) & 15) ||
                      ((reinterpret_cast<uintptr_t>(g.a.scales) | reinterpret_cast<uintptr_t>(g.w.scales)) & 15);
    const auto kernel = edge ? linear_tile_mxfp4_kernel<BM, BN, WR, WC, STAGES, SPREAD, true> : linear_tile_mxfp4_kernel<BM, BN, WR, WC, STAGES, SPREAD, false>;
    DoneFlag &done = done_flags[edge].get();
    if (!done.load(std::memory_order_acquire)) {
        VTL_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds));
        done.store(true, std::memory_order_release);
    }
    const int64_t blocks = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.splits;
    if (blocks > 0xffffff)
        return VTL_HIP_ERR_UNSUPPORTED;
    g.cached = blocks <= 256;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(T::kThreads), T::kLds, st, g);
    return check_launch("linear_tile_mxfp4_kernel");
}

template <int FR, int MX, bool XF32, bool VEC, int NW>
int launch_few(Args g, hipStream_t st)
{
    using F = Few<FR, MX, XF32>;
    constexpr int kMostLds = NW * 2 * F::kSlot;
    static_assert(kMostLds <= 160 << 10 && NW * 4 * MX * F::kPart * 4 <= kMostLds / 2, "shared memory of a compute unit, and sums fit where operands were");
    const auto kernel = linear_few_mxfp4_kernel<FR, MX, XF32, VEC, NW>;
    static PerDevice<DoneFlag> flags;
    DoneFlag &done = flags.get();
    if (!done.load(std::memory_order_acquire)) {
        VTL_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds));
        done.store(true, std::memory_order_release);
    }
    const int units = (g.chunks + 1) / 2;
    g.slots = units <= NW ? 1 : 2;
    const int64_t blocks = (int64_t)((g.N + 16 * FR - 1) / (16 * FR)) * ((g.M + 4 * MX - 1) / (4 * MX));
    if (blocks * 64 * NW > 0xffffffffll)
        return VTL_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NW), NW * g.slots * F::kSlot, st, g);
    return check_launch("linear_few_mxfp4_kernel");
}

// Four waves; eight where they make codes of f32 rows, have a unit each and are not begun again and again: one row and 14336 x 4096 weights 7.0 us, with four 7.7;
// 4096 x 14336 9.1 and 10.5; but 28672 x 8192 26.4 and 22.0, 8192 x 2048 4.1 and 3.7.
template <int FR, int MX, bool XF32, bool VEC>
int launch_few(const Args &g, hipStream_t st)
{
    if constexpr (XF32)
        if (g.chunks > 8 && g.N <= 16 * FR * 512)
            return launch_few<FR, MX, XF32, VEC, 8>(g, st);
    return launch_few<FR, MX, XF32, VEC, 4>(g, st);
}

template <int MX, bool XF32, bool VEC>
int launch_few(const Args &g, hipStream_t st)
{
    if constexpr (MX == 1)
        if (g.N > 16 * 256)
            return launch_few<2, MX, XF32, VEC>(g, st);
    return launch_few<1, MX, XF32, VEC>(g, st);
}

// How a product is made: by the kernel for few rows, which may make their codes itself, or by tiles, with K in so many ranges.
struct Plan {
    bool few, codes;
    int fragments;     // of weights in a workgroup, for more rows than kFewMost
    int tile, splits;
    size_t partials;   // bytes
};

// Tiles and what they cost, by which one is chosen: microseconds for a chunk of K where a compute unit has one workgroup (and two, where it takes two), and
// for a workgroup's beginning and end.  Fitted to all tiles and ranges of K for 48 to 1024 rows, 1024 to 14336 columns, K of 4096 and 14336, where the choice is the
// fastest or within 6 % of it, 0.2 % on average.  Some of them, us (rows x columns x K):
//    256 x  4096 x  4096   64 x 64  9.5, 128 x 128 15.4           512 x 11008 x 4096   128 x 96 23.5, 256 x 128 25.5, 128 x 128 26.2
//    201 x 11008 x  4096   128 x 96 15.6, 128 x 128 17.0, 64 x 64 19.0    1024 x 11008 x 4096   256 x 256 34.8, 128 x 128 40.9
//     64 x  4096 x 14336   64 x 64 with K in four 12.7, in two 14.7, in eight 14.3
// 128 x 96 is for what would be 129 to 192 or 257 to 384 tiles of 128 x 128; with three or four chunks on their way it takes 16.2 us in the place of 15.6.
// A tile of 32 x 64 for 17 to 32 rows gains nothing for K of 4096, and has 12.4 us for 13.4 where K is 14336: not worth a kernel.
struct TileCost {
    int rows, cols;
    float one, two, ends;
};
constexpr TileCost kTiles[] = {{64, 64, 0.34f, 0.50f, 3.0f}, {128, 96, 0.70f, 1.14f, 3.0f}, {128, 128, 0.78f, 1.40f, 3.0f}, {256, 128, 1.2f, 0.0f, 5.0f}, {256, 256, 1.7f, 0.0f, 8.0f}};
constexpr float kJoin = 3.0f, kJoinBytes = 6e-7f;     // for the launch that adds ranges up, and for a byte of their sums
constexpr int kUnits = 256;
// The same of the kernel for few rows, 32 of them and 16 or 32 columns in a workgroup, one of which fills a compute unit; and what the launch takes.  It has all of a
// K within a workgroup, and wins where there is little else to deal out, us: 17 to 32 rows x 4096 x 4096 4.2 (64 x 64 8.5), x 14336 9.4 (13.4), 28672 columns of 8192 26 (21.7);
// 64 rows x 4096 x 4096 5.5 (8.9), x 8192 columns of 4096 9.6 (9.4); 128 rows x 1024 x 4096 4.1 (8.7), x 4096 x 4096 9.5 (9.3).
constexpr TileCost kFewTiles[] = {{32, 16, 0.11f, 0.0f, 0.84f}, {32, 32, 0.18f, 0.0f, 1.0f}};
constexpr float kFewLaunch = 1.6f;

Plan plan_of(int M, int N, int K)
{
    // Every workgroup makes the codes of all rows: 8 rows and 4096 x 4096 weights 4.9 us, with a launch for the codes 6.0; 11008 x 4096 9.6 and 8.9, 28672 x 8192
    // 35 and 22; four rows are level at worst.
    const bool codes = M > 8 || (M > 4 && (int64_t)N * K > 6144 * 4096);
    Plan p{M <= kFewMost, codes, 0, 0, 1, 0};
    if (p.few)
        return p;
    const int chunks = chunks_of(K);
    float best = 0.0f;
    for (int f = 0; f < 2; f++) {
        const TileCost &c = kFewTiles[f];
        const int64_t tiles = (((int64_t)M + c.rows - 1) / c.rows) * (((int64_t)N + c.cols - 1) / c.cols);
        const float cost = kFewLaunch + (float)((tiles + kUnits - 1) / kUnits) * ((float)chunks * c.one + c.ends);
        if (f == 0 || cost < best) {
            best = cost;
            p.few = true;
            p.fragments = f + 1;
        }
    }
    for (int t = 0; t < (int)(sizeof(kTiles) / sizeof(kTiles[0])); t++) {
        const TileCost &c = kTiles[t];
        const int64_t tiles = (((int64_t)M + c.rows - 1) / c.rows) * (((int64_t)N + c.cols - 1) / c.cols);
        for (int splits = 1; splits <= 8; splits += splits < 4 ? 1 : 2) {
            if (splits > 1 && (chunks < 4 * splits || tiles * splits > 2 * kUnits))
                break;
            const int64_t all = tiles * splits, at_once = c.two > 0.0f && all > kUnits ? 2 * kUnits : kUnits;
            const float chunk = at_once > kUnits ? c.two : c.one;
            const size_t bytes = splits > 1 ? (size_t)splits * M * N * sizeof(float) : 0;
            const float cost = (float)((all + at_once - 1) / at_once) * ((float)((chunks + splits - 1) / splits) * chunk + c.ends) +
                               (splits > 1 ? kJoin + kJoinBytes * (float)bytes : 0.0f);
            if (cost < best) {
                best = cost;
                p.few = false;
                p.tile = t;
                p.splits = splits;
                p.partials = bytes;
            }
        }
    }
    return p;
}

int product(Args g, const Plan &p, hipStream_t st)
{
    if (p.few) {
        if (g.x) {
            const bool vec = g.K % 4 == 0 && !(reinterpret_cast<uintptr_t>(g.x) & 15);
            if (g.M <= 4)
                return vec ? launch_few<1, true, true>(g, st) : launch_few<1, true, false>(g, st);
            return vec ? launch_few<2, true, true>(g, st) : launch_few<2, true, false>(g, st);
        }
        return g.M <= 4    ? launch_few<1, false, true>(g, st)
               : g.M <= 8  ? launch_few<2, false, true>(g, st)
               : g.M <= kFewMost ? launch_few<4, false, true>(g, st)
               : p.fragments == 1 ? launch_few<1, 8, false, true>(g, st) : launch_few<2, 8, false, true>(g, st);
    }
    g.splits = p.splits;
    const int rc = p.tile == 0   ? launch_tile<64, 64, 2, 2, 4, 3>(g, st)
                   : p.tile == 1 ? launch_tile<128, 96, 4, 1, 2, 1>(g, st)
                   : p.tile == 2 ? launch_tile<128, 128, 2, 2, 2, 1>(g, st)
                   : p.tile == 3 ? launch_tile<256, 128, 2, 2, 2, 2>(g, st)
                                 : launch_tile<256, 256, 2, 2, 2, 2>(g, st);
    if (rc != VTL_HIP_OK || p.splits == 1)
        return rc;
    const size_t blocks = ((size_t)g.M * g.N + 255) / 256;
    hipLaunchKernelGGL(linear_join_mxfp4_kernel, dim3((unsigned)std::min<size_t>(blocks, 8192)), dim3(256), 0, st, g);
    return check_launch("linear_join_mxfp4_kernel");
}

size_t codes_workspace(int M, int K) { return up256((size_t)M * chunks_of(K) * kChunkCodes) + up256((size_t)M * chunks_of(K) * kChunkScales); }

// What a product needs beside its operands: codes of f32 rows, and sums of ranges of K.
size_t workspace_of(const Plan &p, int M, int K, bool f32) { return (f32 && p.codes ? codes_workspace(M, K) : 0) + up256(p.partials); }

// The caller's, or the library's own where there is none.
int workspace_at(void *given, size_t bytes, size_t need, char *&at)
{
    at = static_cast<char *>(given);
    if (!at && bytes)
        return VTL_HIP_ERR_INVALID_ARG;
    if (at)
        return bytes < need || (reinterpret_cast<uintptr_t>(at) & 15) ? VTL_HIP_ERR_INVALID_ARG : VTL_HIP_OK;
    if (need && !(at = static_cast<char *>(library_workspace(need))))
        return workspace_status();
    return VTL_HIP_OK;
}

int linear(Args g, const uint8_t *w, const uint8_t *w_scales, const float *bias, float *Y, int M, int N, int K, int relu, void *workspace,
           size_t workspace_bytes, bool f32 = false)
{
    if (M < 0 || N < 0 || K < 0)
        return VTL_HIP_ERR_INVALID_ARG;
    // (a lane's offset from a row of results and a grid's threads are counted in 32 bits)
    if (K > kMostCols || M >= 1 << 30 || N > (1 << 27) - 16 || (int64_t)M * chunks_of(K) > INT32_MAX || (int64_t)N * chunks_of(K) > INT32_MAX)
        return VTL_HIP_ERR_UNSUPPORTED;
    if (M == 0 || N == 0)
        return VTL_HIP_OK;
    if (!Y || (K > 0 && ((f32 ? !g.x : !g.a.codes || !g.a.scales) || !w || !w_scales)) || !rows_aligned(g.a.codes, g.a.scales) || !rows_aligned(w, w_scales))
        return VTL_HIP_ERR_INVALID_ARG;
    g.chunks = chunks_of(K);
    const size_t pitch = (size_t)g.chunks * kChunkCodes, spitch = (size_t)g.chunks * kChunkScales, results = (size_t)M * N * sizeof(float);
    const Plan p = plan_of(M, N, K);
    const size_t need = workspace_of(p, M, K, f32);
    const auto written = [&](const void *operand, size_t bytes) { return meet(Y, results, operand, bytes) || meet(workspace, need, operand, bytes); };
    if (written(g.x, (size_t)M * K * sizeof(float)) || written(g.a.codes, M * pitch) || written(g.a.scales, M * spitch) || written(w, N * pitch) ||
        written(w_scales, N * spitch) || written(bias, (size_t)N * sizeof(float)) || meet(Y, results, workspace, need))
        return VTL_HIP_ERR_INVALID_ARG;
    g.w = {w, w_scales};
    g.bias = bias;
    g.y = Y;
    g.M = M;
    g.N = N;
    g.K = K;
    g.relu = relu;
    char *at = nullptr;
    const int rc = workspace_at(workspace, workspace_bytes, need, at);
    if (rc != VTL_HIP_OK)
        return rc;
    const hipStream_t st = current_stream();
    if (f32 && p.codes) {
        uint8_t *const codes = reinterpret_cast<uint8_t *>(at), *const scales = codes + up256(M * pitch);
        at += codes_workspace(M, K);
        const int quantized = launch_quantize(g.x, K, M, K, codes, scales, st);
        if (quantized != VTL_HIP_OK)
            return quantized;
        g.a = {codes, scales};
        g.x = nullptr;
    }
    g.partials = reinterpret_cast<float *>(at);
    return product(g, p, st);
}

}  // namespace

extern "C" {

size_t vtl_hip_linear_mxfp4_workspace(int M, int N, int K)
{
    return M <= 0 || N <= 0 || K <= 0 || K > kMostCols ? 0 : workspace_of(plan_of(M, N, K), M, K, false);
}

size_t vtl_hip_linear_f32_mxfp4_workspace(int M, int N, int K)
{
    return M <= 0 || N <= 0 || K <= 0 || K > kMostCols ? 0 : workspace_of(plan_of(M, N, K), M, K, true);
}

int vtl_hip_linear_mxfp4_f32(const uint8_t *x, const uint8_t *x_scales, const uint8_t *w, const uint8_t *w_scales, const float *bias, float *Y, int M,
                             int N, int K, int relu, void *workspace, size_t workspace_bytes)
{
    Args g{};
    g.a = {x, x_scales};
    return linear(g, w, w_scales, bias, Y, M, N, K, relu, workspace, workspace_bytes);
}

int vtl_hip_linear_f32_mxfp4(const float *X, const uint8_t *w, const uint8_t *w_scales, const float *bias, float *Y, int M, int N, int K, int relu,
                             void *workspace, size_t workspace_bytes)
{
    Args g{};
    g.x = X;
    return linear(g, w, w_scales, bias, Y, M, N, K, relu, workspace, workspace_bytes, true);
}

}  // extern "C"
