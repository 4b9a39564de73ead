// The microscaled 4-bit part of the C++ host mirror (vtl_amd/host/vtl_hip.hpp): its refusals, and on a device a projection into a layer
// of experts with a workspace of its own, against the formulas in f64 on the values that the codes stand for.
// Exit code 0 = all checks passed.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <numeric>
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

// y = x . w^T in f64.
static std::vector<double> product(const float *x, const float *w, int rows, int cols)
{
    std::vector<double> y(rows);
    for (int n = 0; n < rows; n++)
        for (int k = 0; k < cols; k++)
            y[n] += (double)x[k] * w[(size_t)n * cols + k];
    return y;
}

int main(int argc, char **argv)
{
    const auto matrix = [](int rows, int cols) {
        vtl::HipTensor<float> t;
        t.shape = {rows, cols};
        t.size = (size_t)rows * cols;
        return t;
    };
    CHECK(refused([] { vtl::HipMxfp4(3, 0); }));
    CHECK(refused([] { vtl::HipMxfp4(3, (1 << 24) + 1); }));
    CHECK(refused([] { vtl::HipMxfp4::from_packed(std::vector<uint8_t>(128), std::vector<uint8_t>(7), 1, 200); }));
    {
        vtl::HipMxfp4 none, other;      // (no memory)
        none.cols = 64;
        other.cols = 65;
        CHECK(refused([&] { vtl::linear_mxfp4_hip(none, other); }));
        CHECK(refused([&] { vtl::linear_f32_mxfp4_hip(matrix(2, 63), none); }));
        const auto bias = matrix(1, 3);
        CHECK(refused([&] { vtl::linear_f32_mxfp4_hip(matrix(2, 64), none, &bias); }));
        CHECK(refused([&] { vtl::HipMoE(matrix(4, 64), none, none, 1); }));
    }
    if (argc > 1 && !std::strcmp(argv[1], "--no-device")) {
        std::printf(failures ? "mxfp4 mirror: %d failure(s)\n" : "mxfp4 mirror (no device): ok\n", failures);
        return failures ? 1 : 0;
    }

    const int experts = 5, top = 2, dim = 72, hidden = 40, tokens = 6;
    std::mt19937 rng(11);
    std::normal_distribution<float> nd(0.f, 1.f);
    const auto random = [&](int rows, int cols, float std) {
        std::vector<float> v((size_t)rows * cols);
        for (float &x : v)
            x = nd(rng) * std;
        return v;
    };
    const auto quantized = [&](int rows, int cols, std::vector<float> &values) {
        vtl::HipMxfp4 q = vtl::quantize_mxfp4_hip(vtl::HipTensor<float>::from_host(random(rows, cols, 1.f / std::sqrt((float)cols)), {rows, cols}));
        values = q.dequantize().cpu();
        return q;
    };
    std::vector<float> proj_v, gu_v, dn_v;
    const vtl::HipMxfp4 proj = quantized(dim, dim, proj_v), gate_up = quantized(experts * 2 * hidden, dim, gu_v), down = quantized(experts * dim, hidden, dn_v);
    const std::vector<float> router = random(experts, dim, 0.1f), bias = random(1, dim, 1.f), router_bias = random(1, experts, 0.1f);
    const auto x = vtl::HipTensor<float>::from_host(random(tokens, dim, 1.f), {tokens, dim});
    const auto db = vtl::HipTensor<float>::from_host(bias, {dim}), drb = vtl::HipTensor<float>::from_host(router_bias, {experts});
    const auto dr = vtl::HipTensor<float>::from_host(router, {experts, dim});

    const vtl::HipMxfp4 xq = vtl::quantize_mxfp4_hip(x);
    const std::vector<float> x_v = xq.dequantize().cpu();
    const vtl::HipStorage<uint8_t> ws(std::max<size_t>(16, vtl::linear_mxfp4_workspace(tokens, dim, dim)));
    const auto a = vtl::linear_f32_mxfp4_hip(x, proj, &db, true, &ws);
    const std::vector<float> a_v = a.cpu(), a2_v = vtl::linear_mxfp4_hip(xq, proj, &db, true).cpu();
    for (int t = 0; t < tokens; t++) {
        const std::vector<double> y = product(&x_v[(size_t)t * dim], proj_v.data(), dim, dim);
        // 72 products of magnitude 10 at most in sums of f32: well below 1e-4
        for (int n = 0; n < dim; n++) {
            const double want = std::max(0.0, y[n] + bias[n]);
            CHECK(std::fabs(a_v[(size_t)t * dim + n] - want) < 1e-4 && std::fabs(a2_v[(size_t)t * dim + n] - want) < 1e-4);
        }
    }

    const vtl::HipMoE layer(dr, gate_up, down, top, true, &drb);
    CHECK(refused([&] { vtl::moe_mxfp4_hip(layer, matrix(2, dim + 1)); }));
    CHECK(refused([&] { vtl::HipMoE(dr, gate_up, down, experts + 1); }));
    const vtl::HipStorage<uint8_t> moe_ws(layer.workspace(tokens)), less(layer.workspace(tokens) - 1);
    const std::vector<float> got = vtl::moe_mxfp4_hip(layer, a, &moe_ws).cpu();
    bool thrown = false;
    try {
        vtl::moe_mxfp4_hip(layer, a, &less);
    } catch (const vtl::HipError &) {
        thrown = true;
    }
    CHECK(thrown);
    for (int t = 0; t < tokens; t++) {
        const float *row = &a_v[(size_t)t * dim];
        std::vector<double> scores = product(row, router.data(), experts, dim), y(dim);
        std::vector<int> order(experts);
        std::iota(order.begin(), order.end(), 0);
        for (int e = 0; e < experts; e++)
            scores[e] += router_bias[e];
        std::sort(order.begin(), order.end(), [&](int p, int q) { return scores[p] > scores[q]; });
        double all = 0;
        for (int k = 0; k < top; k++)
            all += std::exp(scores[order[k]] - scores[order[0]]);
        for (int k = 0; k < top; k++) {
            const int e = order[k];
            const double weight = std::exp(scores[e] - scores[order[0]]) / all;
            const std::vector<double> gu = product(row, &gu_v[(size_t)e * 2 * hidden * dim], 2 * hidden, dim);
            for (int h = 0; h < hidden; h++) {
                const double value = weight * gu[h] / (1 + std::exp(-gu[h])) * gu[hidden + h];
                for (int n = 0; n < dim; n++)
                    y[n] += value * dn_v[((size_t)e * dim + n) * hidden + h];
            }
        }
        // values of magnitude 10 at most, activations of 24 bits, sums of f32: well below 1e-4
        for (int n = 0; n < dim; n++)
            CHECK(std::fabs(got[(size_t)t * dim + n] - y[n]) < 1e-4);
    }
    std::printf(failures ? "mxfp4 mirror: %d failure(s)\n" : "mxfp4 mirror: ok\n", failures);
    return failures ? 1 : 0;
}
