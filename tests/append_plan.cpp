// Run by tests/test_append_plan.py: how 8-bit appends of many sizes are divided (vxs_append_plan.h). Chunks cover the tokens, and a launch's
// threads fit 32 bits whatever the tokens and heads.
#include <cmath>
#include <cstdio>
#include <random>

#include "../voxwerk_amd/csrc/vxs_append_plan.h"

int main() {
    std::mt19937_64 r(1);
    auto size = [&](int64_t most) { return (int64_t)(std::generate_canonical<double, 53>(r) < 0.2 ? most : std::exp2(std::generate_canonical<double, 53>(r) * std::log2((double)most))); };
    int failures = 0, limited = 0;
    for (int i = 0; i < 300000; i++) {
        const int dim = 64 << (int)(r() % 3), tokens = (int)size((1 << 24) - 1), kv = r() % 5 ? (int)size(1 << 22) : 0;
        const int q = r() % 5 || !kv ? (kv ? kv : 1) * (int)size(64) : 0;
        const vxs::Append8Grid g = vxs::plan_append8(tokens, q, kv, dim);
        const bool covers = (int64_t)g.chunks * vxs::kChunk >= tokens && (int64_t)(g.chunks - 1) * vxs::kChunk < tokens;
        const bool fits = g.parts >= 1 && g.parts <= 65535 && (uint64_t)g.chunks * g.parts * vxs::kAppend8Threads <= UINT32_MAX;
        limited += g.parts > 1 && (uint64_t)g.chunks * (g.parts + 1) * vxs::kAppend8Threads > UINT32_MAX;
        if ((!covers || !fits) && failures++ < 20)
            std::printf("%d tokens, heads %d / %d of %d: %u chunks, %u parts\n", tokens, q, kv, dim, g.chunks, g.parts);
    }
    // the sizes that the kernel's figures are of
    const vxs::Append8Grid one = vxs::plan_append8(1, 16, 8, 128), batch = vxs::plan_append8(256, 16, 8, 128), prompts = vxs::plan_append8(18000, 32, 8, 128);
    if (one.chunks != 1 || one.parts != 2 || batch.chunks != 16 || batch.parts != 20 || prompts.chunks != 1125 || prompts.parts != 6) {
        failures++;
        std::printf("%u x %u, %u x %u, %u x %u\n", one.chunks, one.parts, batch.chunks, batch.parts, prompts.chunks, prompts.parts);
    }
    if (!limited) {
        failures++;
        std::printf("no size reached the limit\n");
    }
    return failures != 0;
}
