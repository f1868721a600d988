// Run by tests/test_attention_host.py: how steps of many sizes are divided (vxs_attn_plan.h). Parts after a row's or a prefix's
// first begin at whole granules of 16 tokens (a granule lies in one page, and the kernel looks up one page for it), parts
// cover the announced lengths, and the sums of all parts fit the workspace of these sizes and of any larger ones.
#include <cstdio>
#include <initializer_list>
#include <random>

#include "../voxwerk_amd/csrc/vxs_attn_plan.h"

namespace {

int failures = 0;
void fail(const vxs::StepArgs& a, const vxs::Split& s, const char* what) {
    if (failures++ < 20)
        std::printf("%s: rows %d, heads %d / %d of %d, max_len %d, prefix %d in %d groups: own %d x %d, prefix %d x %d, solo %d\n", what, a.rows,
                    a.q_heads, a.cache.kv_heads, a.cache.head_dim, a.max_len, a.prefix.max_len, a.prefix.groups, s.own_parts, s.own_chunk,
                    s.pre_parts, s.pre_chunk, s.solo);
}

// Whether parts of `chunk` tokens each (the last takes what is left) are as the kernel takes them.
bool sound(int parts, int chunk, int64_t len) {
    return parts >= 1 && parts <= vxs::kMaxParts && chunk > 0 && (parts == 1 || (chunk % 64 == 0 && (parts - 1) * (int64_t)chunk < len));
}

void check(const vxs::StepArgs& a, int64_t larger) {
    const int64_t most = a.cache.ld_table << a.cache.page_bits, len = std::min<int64_t>(a.max_len, most), shared = std::min<int64_t>(a.prefix.max_len, most);
    for (bool work : {true, false}) {
        const vxs::Split s = vxs::plan_step(a, work);
        if (!sound(s.own_parts, s.own_chunk, len)) fail(a, s, "own parts");
        if (s.pre_parts && !sound(s.pre_parts, s.pre_chunk, shared)) fail(a, s, "prefix parts");
        const int64_t tiles = a.prefix.groups ? (int64_t)a.rows * (a.q_heads / a.cache.kv_heads) / vxs::kCols + a.prefix.groups : 0;
        if (s.pre_parts && s.pre_tiles != std::min<int64_t>(tiles, INT32_MAX)) fail(a, s, "prefix tiles");
        if (!work && (s.own_parts != 1 || s.pre_parts)) fail(a, s, "divided without a workspace");
        const bool joins = s.own_parts + s.pre_parts > 1;
        const int64_t need = joins ? vxs::record_bytes(a, (int64_t)a.rows * (s.own_parts + s.pre_parts)) : 0;
        if (work && (need > vxs::work_bytes(a) || need > larger)) fail(a, s, "the workspace is too small");
        if (joins && need < (int64_t)a.rows * a.cache.kv_heads * vxs::kBlock * 4) fail(a, s, "no place for the counts");
    }
}

}  // namespace

int main() {
    std::mt19937_64 rng(1);
    auto below = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)n); };
    auto spread = [&](int64_t lo, int64_t hi) {  // over the logarithm
        const int bits = 63 - __builtin_clzll((uint64_t)hi);
        const int64_t top = std::min<int64_t>(hi, int64_t(2) << below(bits + 1));
        return std::max(lo, std::min(hi, 1 + below(top)));
    };
    const int64_t edges[] = {0, 1, 255, 256, 257, 1023, 1024, 1025, 262143, 262144, 262145, 262208, 300000, 300100, 1 << 20, (1 << 20) + 1, INT32_MAX - 257, INT32_MAX - 256};
    for (int i = 0; i < 2000000; i++) {
        vxs::StepArgs a{};
        a.cache.kv_heads = (int)spread(1, i % 2 ? 16 : 700);
        a.q_heads = a.cache.kv_heads * (int)spread(1, i % 3 ? 16 : 100);
        a.cache.head_dim = 64 << below(3);
        a.cache.page_bits = (int)(4 + below(13));
        a.cache.ld_table = below(4) ? (INT32_MAX - 256) >> a.cache.page_bits : spread(1, (INT32_MAX - 256) >> a.cache.page_bits);
        a.rows = (int)spread(1, 1 << 14);
        a.max_len = (int)(below(3) ? spread(1, INT32_MAX - 256) : edges[below(sizeof edges / sizeof *edges)]);
        if (below(3)) {
            a.prefix.groups = (int)(i % 64 ? spread(1, 300) : INT32_MAX - below(3));
            a.prefix.flags = below(2) ? VXS_FLAG_SHARE_ALWAYS : 0;
            const int64_t near = a.max_len - below(300);  // (what is left is short: each wave a part of its own)
            a.prefix.max_len = (int)(below(2) ? std::max<int64_t>(near, 1) : spread(1, INT32_MAX - 256));
        }
        vxs::StepArgs more = a;  // a workspace asked for with larger sizes serves this step too
        more.rows = (int)std::min<int64_t>(a.rows + below(a.rows + 1), 1 << 15);
        more.max_len = (int)std::min<int64_t>((int64_t)a.max_len + below((int64_t)a.max_len + 1), INT32_MAX - 256);
        if (a.prefix.groups) more.prefix.max_len = (int)std::min<int64_t>((int64_t)a.prefix.max_len + below((int64_t)a.prefix.max_len + 1), INT32_MAX - 256);
        check(a, vxs::work_bytes(more));
    }
    for (int d : {1, 2, 3, 5, 7, 12, 28, 255, 256, 257, 65535, 65536, 1000003, INT32_MAX})
        for (int64_t n : {int64_t(0), int64_t(1), int64_t(d) - 1, int64_t(d), int64_t(d) + 1, int64_t(INT32_MAX) - 1, int64_t(INT32_MAX), below(INT32_MAX)})
            if (n <= INT32_MAX && vxs::Divisor::of(d).div((int)n) != n / d) {
                std::printf("%lld / %d\n", (long long)n, d);
                failures++;
            }
    std::printf("%d failures\n", failures);
    return failures != 0;
}
