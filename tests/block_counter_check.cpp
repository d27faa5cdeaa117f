// Blocks with dropout that are put together without a GPT around them: a line "name value" per check, 0 where it holds.
#include "gradc/gradc.hpp"

#include <cstdio>

using namespace gradc;

template <class F>
static int refused(F&& f) {
    try { f(); } catch (const std::exception&) { return 1; }
    return 0;
}

int main() {
    NormalInit<float> init(0.0f, 0.02f);
    BlockOptions drops, none;
    drops.dropout = 0.25f;
    using Other = BlockT<float, LayerNorm<float>, GeluMLP<float>>;
    auto norm = [] { return LayerNorm<float>({32}, {-1}, OnesInit<float>(), ZerosInit<float>(), 1e-5f); };
    auto counter = std::make_shared<DropoutCounter>();
    std::printf("plain %d\n", refused([&] { TransformerBlock<float> b(32, 4, 16, init, init); }));
    std::printf("without_dropout %d\n", refused([&] { TransformerBlock<float> b(32, 4, 16, init, init, 1e-5f, none); }));
    std::printf("with_a_counter %d\n", refused([&] { TransformerBlock<float> a(32, 4, 16, init, init, 1e-5f, drops, counter), b(32, 4, 16, init, init, 1e-5f, drops, counter); }));
    std::printf("without_one %d\n", 1 - refused([&] { TransformerBlock<float> b(32, 4, 16, init, init, 1e-5f, drops); }));
    std::printf("other_with_a_counter %d\n", refused([&] { Other b(32, 4, 16, 64, init, init, norm, drops, counter); }));
    std::printf("other_without_one %d\n", 1 - refused([&] { Other b(32, 4, 16, 64, init, init, norm, drops); }));
    std::printf("models %d\n", refused([&] { GPT<float> a(96, 16, 32, 4, 2, init, init, 1e-5f, drops); LayerNormGPT<float> b(96, 16, 32, 4, 2, 64, init, init, 1e-5f, drops); }));
    return 0;
}
