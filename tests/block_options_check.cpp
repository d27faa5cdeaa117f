// A model's dropout and attention rule, and the operators under them, through the C++ API: a line "name value" per check, 0 where it holds.
#include "gradc/gradc.hpp"

#include <cstdio>

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
static Tensor<float> leaf(const std::vector<int64_t>& shape) {
    Tensor<float> t = Tensor<float>::normal(shape, 0.0f, 1.0f, Device(DeviceType::CPU)).to(gpu);
    t.realize();
    t = t.detach();
    t.set_requires_grad(true);
    t.realize();
    return t;
}
static Tensor<float> copy_of(const Tensor<float>& x) {
    Tensor<float> t(x.shape(), gpu, uninitialized);
    gcb_check(gcb_copy_d2d(ctx(), t.data_ptr(), const_cast<Tensor<float>&>(x).data_ptr(), sizeof(float) * (size_t)x.volume()), "copy");
    t = t.detach();
    t.set_requires_grad(true);
    t.realize();
    return t;
}
static double off(const std::vector<float>& a, const std::vector<float>& b) {
    double d = 0.0, top = 0.0;
    for (size_t i = 0; i < a.size(); ++i) { d = std::max(d, std::abs((double)a[i] - b[i])); top = std::max(top, std::abs((double)b[i])); }
    return d / top;
}
template <class F>
static int refused(F&& f) {
    try { f(); } catch (const std::exception&) { return 0; }
    return 1;
}
struct Model : GPT<float> {
    using GPT<float>::GPT;
    Module<float>& block(size_t i) { return *m_blocks[i]; }
};

int main() {
    NormalInit<float> init(0.0f, 0.02f);
    BlockOptions opt;
    opt.window = 5; opt.sinks = 1; opt.rel_buckets = 4; opt.rel_reach = 8; opt.dropout = 0.5f;
    Model model(96, 16, 32, 4, 2, init, init, 1e-5f, opt);
    model.to(gpu);
    auto tokens = [&] { return generate_tokens_incremental(model, {1, 2, 3}, 16, 14, 1, gpu); };
    model.eval();
    const auto quiet = tokens();
    model.block(0).train();
    const bool same = tokens() == quiet;
    std::printf("modes_kept %d\n", same && !model.is_training() && model.block(0).is_training() && !model.block(1).is_training() ? 0 : 1);
    model.train();
    model.block(1).eval();
    std::printf("modes_kept_in_training %d\n", tokens() == quiet && model.is_training() && !model.block(1).is_training() ? 0 : 1);

    {  // the same tensor dropped and added to: d/dx sum (x + f x) = 1 + f, and so is (x + f x) / x
        DropoutCounter counter{7, 0};
        Tensor<float> x = leaf({33, 5});
        Tensor<float> y = dropout(x, 0.25f, counter, x);
        y.realize();
        const std::vector<float> xs = host(x), ys = host(y);
        y.backward();
        const std::vector<float> g = host(x.grad().value());
        double worst = 0.0;
        for (size_t i = 0; i < g.size(); ++i) worst = std::max(worst, std::abs((double)g[i] - ys[i] / xs[i]));
        std::printf("dropped_onto_itself %d\n", worst < 8 * 0x1p-24 * (1 + 4.0 / 3) && counter.next == (33 * 5 + 3) / 4 ? 0 : 1);
    }
    {  // one tensor as q, k and v: its gradient is the sum of the three, an addition each
        AttentionRule rule{9, 2, AttentionRule::relative_buckets(6, 12)};
        Tensor<float> x = leaf({2, 3, 40, 16}), bias = leaf({3, 6}), a = copy_of(x), b = copy_of(x), c = copy_of(x), other = copy_of(bias);
        for (Tensor<float> y : {window_attention(x, x, x, rule, bias).gelu(), window_attention(a, b, c, rule, other).gelu()}) {
            y.realize();
            y.backward();
        }
        const std::vector<float> g = host(x.grad().value()), ga = host(a.grad().value()), gb = host(b.grad().value()), gc = host(c.grad().value());
        double worst = 0.0, most = 0.0;  // two additions of up to 3 `most`, each off by half a step
        for (size_t i = 0; i < g.size(); ++i) {
            worst = std::max(worst, std::abs((double)g[i] - ((double)ga[i] + gb[i] + gc[i])));
            for (float v : {ga[i], gb[i], gc[i]}) most = std::max(most, std::abs((double)v));
        }
        std::printf("one_tensor_thrice %d\n", worst <= 2 * 0x1p-24 * 3 * most ? 0 : 1);
        std::printf("bias_gradient %d\n", off(host(bias.grad().value()), host(other.grad().value())) == 0.0 ? 0 : 1);
        std::printf("no_table %d\n", refused([&] { window_attention(x, x, x, rule); }));
        std::printf("no_buckets %d\n", refused([&] { window_attention(x, x, x, AttentionRule{4, 0, {}}, bias); }));
        std::printf("table_of_another_shape %d\n", refused([&] { window_attention(x, x, x, rule, leaf({6, 3})); }));
        std::printf("other_shapes %d\n", refused([&] { window_attention(x, x, leaf({2, 3, 41, 16}), rule, bias); }));
        std::printf("three_dimensions %d\n", refused([&] { window_attention(bias, bias, bias, rule, bias); }));
        std::printf("negative_window %d\n", refused([&] { window_attention(x, x, x, AttentionRule{-1, 0, {}}).realize(); }));
        DropoutCounter counter;
        std::printf("probability %d\n", refused([&] { dropout(x, 1.5f, counter); }));
        std::printf("residual_of_another_shape %d\n", refused([&] { dropout(x, 0.5f, counter, bias); }));
        BlockOptions wide;
        wide.window = 4;
        std::printf("wide_heads %d\n", refused([&] { GPT<float> m(96, 16, 512, 2, 1, init, init, 1e-5f, wide); }));
        BlockOptions often;
        often.dropout = -0.1f;
        std::printf("negative_probability %d\n", refused([&] { GPT<float> m(96, 16, 32, 4, 1, init, init, 1e-5f, often); }));
    }
    return 0;
}
