// A tensor used twice, once by an operator that hands back a gradient with strides and once by one that adds to it row by row: the sum is that of
// the two uses apart.  A line "name value" per check, 0 where it holds.
#include "gradc/gradc.hpp"

#include <cstdio>
#include <functional>

using namespace gradc;

static const Device gpu(DeviceType::CUDA, 0);
static gcb_ctx* ctx() { return Backend::get().ctx(gpu); }
static std::vector<float> host(Tensor<float> t) {
    t.realize();
    t = make_contiguous(t);
    std::vector<float> h((size_t)t.volume());
    gcb_check(gcb_copy_d2h(ctx(), h.data(), t.data_ptr(), sizeof(float) * h.size()), "download");
    return h;
}
static Tensor<float> leaf(const std::vector<float>& values, const std::vector<int64_t>& shape, bool wants_gradient) {
    Tensor<float> t(shape, gpu, uninitialized);
    gcb_check(gcb_copy_h2d(ctx(), t.data_ptr(), values.data(), sizeof(float) * values.size()), "upload");
    t.set_requires_grad(wants_gradient);
    t.realize();
    return t;
}
using F = std::function<Tensor<float>(Tensor<float>)>;
static std::vector<float> gradient(const std::vector<float>& x, const std::vector<int64_t>& shape, const F& f) {
    Tensor<float> t = leaf(x, shape, true), y = f(t);
    y.realize();
    y.backward();
    return host(t.grad().value());
}

int main() {
    const std::vector<int64_t> shape{2, 3, 5, 8};
    const int64_t n = shape_volume(shape);
    auto values = [&](uint32_t seed) {
        std::vector<float> v((size_t)n);
        for (float& e : v) { seed = seed * 1664525u + 1013904223u; e = (float)(seed >> 8) * 0x1p-23f - 1.0f; }
        return v;
    };
    const std::vector<float> xs = values(1), ks = values(2), vs = values(3);
    const AttentionRule rule{3, 1, {}};
    const std::vector<float> ones(8, 1.0f), zeros(8, 0.0f);
    const std::vector<std::pair<const char*, F>> flat = {
        {"dropout", [](Tensor<float> x) { DropoutCounter c{7, 0}; return dropout(x, 0.25f, c); }},
        {"gelu", [](Tensor<float> x) { return x.gelu(); }},
        {"scaled", [](Tensor<float> x) { return x * 0.7f; }},
        {"layernorm", [&](Tensor<float> x) { return layernorm(x, leaf(ones, {8}, false), leaf(zeros, {8}, false), {-1}, 1e-5f); }},
        {"swiglu", [&](Tensor<float> x) { return swiglu_fast(x, leaf(ks, shape, true)); }},
    };
    for (int others = 0; others < 3; ++others) {  // k and v need no gradient, are leaves, are results of an operation
        auto other = [&](const std::vector<float>& v) {
            Tensor<float> t = leaf(v, shape, others > 0);
            return others == 2 ? t.gelu() : t;
        };
        const std::vector<std::pair<const char*, F>> strided = {
            {"window", [&](Tensor<float> x) { return window_attention(x, other(ks), other(vs), rule); }},
            {"keys", [&](Tensor<float> x) { return window_attention(other(ks), x, other(vs), rule); }},
            {"causal", [&](Tensor<float> x) { return sdpa(x, other(ks), other(vs), true); }},
            {"permuted", [&](Tensor<float> x) { return x.permute({0, 2, 1, 3}).gelu().permute({0, 2, 1, 3}); }},
        };
        for (const auto& [a, fa] : strided)
            for (const auto& [b, fb] : flat) {
                const std::vector<float> ga = gradient(xs, shape, fa), gb = gradient(xs, shape, fb);
                for (int order = 0; order < 2; ++order) {
                    const std::vector<float> g = gradient(xs, shape, [&](Tensor<float> x) { return order ? fb(x) + fa(x) : fa(x) + fb(x); });
                    // one addition of two terms, and a product that it may be fused with: two roundings apart at most, half a step each
                    bool same = true;
                    for (size_t i = 0; i < g.size(); ++i) same = same && std::abs((double)g[i] - ((double)ga[i] + gb[i])) <= 2 * 0x1p-24 * (std::abs((double)ga[i]) + std::abs((double)gb[i]));
                    std::printf("%s_%s_%d_%d %d\n", a, b, others, order, same ? 0 : 1);
                }
            }
    }
    return 0;
}
