// The key/value cache and attention of the C++ host mirror (vtl_amd/host/vtl_hip.hpp): its refusals, and on a device two
// sequences written in two calls, read back and attended to, against the formulas in f64.
// Exit code 0 = all checks passed.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>

#include "vtl_hip.hpp"

static int failures = 0;
#define CHECK(cond)                                                        \
    do {                                                                   \
        if (!(cond)) {                                                     \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            failures++;                                                    \
        }                                                                  \
    } while (0)

template <typename F>
static bool refused(F f)
{
    try {
        f();
    } catch (const std::invalid_argument &) {
        return true;
    }
    return false;
}

// A code and its scale as a value, of the largest magnitude among n values.
static std::vector<float> as_stored(const float *x, int n)
{
    float most = 0.f;
    for (int i = 0; i < n; i++)
        most = std::max(most, std::fabs(x[i]));
    const float scale = most / 127.f;
    std::vector<float> y(n);
    for (int i = 0; i < n; i++)
        y[i] = scale == 0.f ? 0.f : std::nearbyint(x[i] / scale) * scale;
    return y;
}

int main(int argc, char **argv)
{
    CHECK(refused([] { vtl::HipKVCache(1, 17, 1, 64); }));
    CHECK(refused([] { vtl::HipKVCache(1, 16, 1, 257); }));
    {
        vtl::HipTensor<int32_t> table, lengths, starts;
        table.shape = {2, 3};
        lengths.size = 3;
        CHECK(refused([&] { vtl::HipKVBatch(table, lengths); }));
        lengths.size = 2;
        starts.size = 2;
        CHECK(refused([&] { vtl::HipKVBatch(table, lengths, &starts, 5); }));
        vtl::HipKVBatch batch(table, lengths);
        CHECK(batch.rows == 2);
        vtl::HipTensor<float> k;
        int64_t stride;
        k.shape = {3, 8};
        k.size = 24;
        CHECK(refused([&] { vtl::kv_rows(k, batch, 8, 0, stride); }));
        k.shape = {2, 12};
        CHECK(refused([&] { vtl::kv_rows(k, batch, 8, 5, stride); }));
        vtl::kv_rows(k, batch, 8, 4, stride);
        CHECK(stride == 12);
    }
    if (argc > 1 && !std::strcmp(argv[1], "--no-device")) {
        std::printf(failures ? "kv mirror: %d failure(s)\n" : "kv mirror (no device): ok\n", failures);
        return failures ? 1 : 0;
    }

    const int kv_heads = 2, heads = 6, dim = 40, page = 16, max_pages = 3, group = heads / kv_heads;
    const std::vector<int32_t> counts{33, 7};      // a prompt each, then a token each
    std::mt19937 rng(7);
    std::normal_distribution<float> nd(0.f, 1.f);
    vtl::HipKVCache cache(2 * max_pages, page, kv_heads, dim);
    const auto table = vtl::HipTensor<int32_t>::from_host({5, 0, 3, 1, 4, 2}, {2, max_pages});
    const int columns = (heads + 2 * kv_heads) * dim;      // q, k and v of a token beside each other
    std::vector<std::vector<float>> tokens(2);
    for (int step = 0; step < 2; step++) {
        std::vector<int32_t> lengths(2), starts{0, 0, 0};
        std::vector<float> rows;
        for (int b = 0; b < 2; b++) {
            const int fresh = step ? 1 : counts[b];
            lengths[b] = counts[b] + step;
            starts[b + 1] = starts[b] + fresh;
            for (int i = 0; i < fresh * columns; i++) {
                rows.push_back(nd(rng));
                tokens[b].push_back(rows.back());
            }
        }
        const int n = starts[2];
        const auto x = vtl::HipTensor<float>::from_host(rows, {n, columns});
        const auto l = vtl::HipTensor<int32_t>::from_host(lengths, {2}), s = vtl::HipTensor<int32_t>::from_host(starts, {3});
        const vtl::HipKVBatch batch = step ? vtl::HipKVBatch(table, l) : vtl::HipKVBatch(table, l, &s, n);
        vtl::kv_write_hip(cache, batch, x, x, heads * dim, (heads + kv_heads) * dim);
        const auto back = vtl::kv_read_hip(cache, batch);
        const std::vector<float> k = back.first.cpu(), v = back.second.cpu();
        const float scale = 1.f / std::sqrt((float)dim);
        const std::vector<float> got = vtl::attention_i8_hip(cache, batch, x, heads, scale, true).cpu();
        for (int b = 0; b < 2; b++)
            for (int r = starts[b]; r < starts[b + 1]; r++) {
                const int position = lengths[b] - (starts[b + 1] - r);
                for (int h = 0; h < kv_heads; h++)
                    for (int of = 0; of < 2; of++) {
                        const std::vector<float> stored = as_stored(&tokens[b][(size_t)position * columns + (heads + of * kv_heads + h) * dim], dim);
                        CHECK(std::equal(stored.begin(), stored.end(), (of ? v : k).begin() + ((size_t)r * kv_heads + h) * dim));
                    }
                for (int h = 0; h < heads; h++) {
                    std::vector<double> weights(position + 1), o(dim);
                    double most = -INFINITY, sum = 0;
                    std::vector<std::vector<float>> values;
                    for (int j = 0; j <= position; j++) {
                        const float *token = &tokens[b][(size_t)j * columns];
                        const std::vector<float> key = as_stored(token + (heads + h / group) * dim, dim);
                        values.push_back(as_stored(token + (heads + kv_heads + h / group) * dim, dim));
                        for (int d = 0; d < dim; d++)
                            weights[j] += (double)scale * rows[(size_t)r * columns + h * dim + d] * key[d];
                        most = std::max(most, weights[j]);
                    }
                    for (double &w : weights)
                        sum += w = std::exp(w - most);
                    for (int j = 0; j <= position; j++)
                        for (int d = 0; d < dim; d++)
                            o[d] += weights[j] / sum * values[j][d];
                    // 40 products of magnitude 1 at most and 34 tokens, in f32 sums of halves with 22 bits: well below 1e-5
                    for (int d = 0; d < dim; d++)
                        CHECK(std::fabs(got[((size_t)r * heads + h) * dim + d] - o[d]) < 1e-5);
                }
            }
    }
    cache.release();
    std::printf(failures ? "kv mirror: %d failure(s)\n" : "kv mirror: ok\n", failures);
    return failures ? 1 : 0;
}
