// vxs_attn_plan.h — how the work of a step (vxs_attn_step.hip) is divided, and the workspace that its parts leave their sums in.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "vxs_attn.h"

namespace vxs {

constexpr int kCols = 32;       // query rows of a workgroup
constexpr int kMaxParts = 256;  // of a row's keys

// n / d for 0 <= n < 2^31 by one product: with s = 31 + ceil(log2 d) and m = ceil(2^s / d), m d - 2^s < d <= 2^(s - 31), so
// n (m d - 2^s) < 2^s and floor(n m / 2^s) is exact.
struct Divisor {
    uint32_t m, s;
    int d;
    static Divisor of(int d) {
        uint32_t l = 0;
        while ((int64_t(1) << l) < d) l++;
        return {(uint32_t)(((uint64_t(1) << (31 + l)) + d - 1) / d), 31 + l, d};
    }
    __device__ __forceinline__ int div(int n) const { return (int)((uint64_t)(unsigned)n * m >> s); }
};

// How a call's work is divided.
struct Split {
    int solo;        // a row's own keys: each wave takes a part of its own (else the workgroup's four waves share one)
    int head_tiles;  // of 32 query heads of a key head each
    // Parts are of whole 64s: a granule of 16 tokens lies in one page, for which the kernel looks up one table entry.
    int own_parts;   // of a row's own keys, of own_chunk each (the last takes what is left; their product may pass 32 bits)
    int own_chunk;
    int pre_tiles;   // of 32 stacked query rows of all prefix groups, at most
    int pre_parts;
    int pre_chunk;
    Divisor group, heads, tiles, parts, pre;  // query heads per key head, key heads, head_tiles, own_parts, pre_tiles
};

inline Split plan_step(const StepArgs& a, bool work) {
    const int rows = a.rows, kv_heads = a.cache.kv_heads, G = a.q_heads / kv_heads, groups = work ? a.prefix.groups : 0;
    const int64_t most = a.cache.ld_table << a.cache.page_bits;  // (below 2^31 - 256)
    const int max_len = (int)std::min<int64_t>(a.max_len, most), max_prefix = (int)std::min<int64_t>(a.prefix.max_len, most);
    Split s{};
    s.head_tiles = (G + kCols - 1) / kCols;
    const int64_t units = (int64_t)std::max(rows, 1) * kv_heads * s.head_tiles;
    // A workgroup costs about 9 us beside its keys (first loads 3, leaving and joining parts 4), so a row's keys are
    // divided only until there are two workgroups for each compute unit (own keys; us for fill 512 / 1024: 24 rows of
    // 1000 to 2000 33 / 37, 4 of 65000 82 / 89) or one (prefixes: 96 rows 37, with two 43), in parts of at least 256 keys
    // (128: one row of 8000 20 us, not 14).
    auto parts = [&](int64_t n, int len, int64_t least, int64_t fill, int& chunk) {
        n = std::max<int64_t>(1, (fill + n - 1) / n);
        n = std::max<int64_t>(1, std::min<int64_t>({n, (len + least - 1) / least, kMaxParts}));
        chunk = (int)std::max<int64_t>(least, (((int64_t)len + n - 1) / n + 63) / 64 * 64);
        return (int)std::max<int64_t>(1, ((int64_t)len + chunk - 1) / chunk);
    };
    s.own_parts = parts(units, max_len, 256, 512, s.own_chunk);
    // Reading a prefix once costs the joining of its parts and a workgroup's wait for the others. It is worth that where reading
    // it for every row takes longer: from about 200 MB of keys and values, much of which comes from the caches (us, shared / not, 8
    // key heads of 128: 16 rows of 2000 15.6 / 14.2, of 8000 20 / 28, 64 of 500 15.6 / 12.5, of 1000 16.3 / 17.3, of 4000 21 / 45,
    // 128 of 4000 24 / 85; 4 key heads: 64 of 2000 19.1 / 18.7).
    const bool shares = groups > 0 && max_prefix > 0 &&
                        ((a.prefix.flags & VXS_FLAG_SHARE_ALWAYS) || (double)rows * max_prefix * kv_heads * a.cache.head_dim * 4 >= 2e8);
    // Short rows, more than fit at once: a wave each, with nothing to join (us, one wave / four: 1024 of (row, key head) with
    // 32 keys 6.3 / 10.8, with 200 18.3 / 21.9, 300 24.6 / 25.6, 500 36.6 / 34.8; 512 with 100 keys 9.6 / 7.4).
    s.solo = units > 512 && max_len - (shares ? max_prefix : 0) <= 256;
    if (s.solo) {  // (a row that shares no prefix while the others do may be long)
        s.own_chunk = (int)std::max<int64_t>(1024, ((int64_t)max_len + 64 * kMaxParts - 1) / (64 * kMaxParts) * 64);
        s.own_parts = (int)std::max<int64_t>(1, ((int64_t)max_len + s.own_chunk - 1) / s.own_chunk);
    }
    if (!work) {
        s.own_parts = 1;
        s.own_chunk = INT32_MAX;
    }
    if (shares) {
        s.pre_tiles = (int)std::min<int64_t>(((int64_t)rows * G) / kCols + groups, INT32_MAX);  // (a launch of that many is refused)
        s.pre_parts = parts((int64_t)s.pre_tiles * kv_heads, max_prefix, 256, 256, s.pre_chunk);
    }
    s.group = Divisor::of(G);
    s.heads = Divisor::of(kv_heads);
    s.tiles = Divisor::of(s.head_tiles);
    s.parts = Divisor::of(s.own_parts);
    s.pre = Divisor::of(std::max(s.pre_tiles, 1));
    return s;
}

// The workspace: for each (row, key head), part and query head a record of D / 64 blocks of 68 words: m, l, a count, one
// unused, and 64 entries of o. The count of block i is that of the query rows that have arrived of (row, key head) i; being
// where no call of any size or type has anything else, counts that a call has set back are zero for the next. A part's sums are
// written and read at the device's common memory (agent scope: past the caches of one XCD); fences over whole caches would
// cost more than the step.
constexpr int kBlock = 68;  // words
struct Records {
    float* base;
    int parts;
};
inline int64_t record_bytes(const StepArgs& a, int64_t row_parts) { return 4 * row_parts * a.q_heads * (a.cache.head_dim / 64) * kBlock; }

// Enough for every call of up to a.rows rows, a.max_len tokens and a.prefix.max_len shared ones (whatever its groups): sums over
// rows of plan_step's parts, which are at most min(ceil(fill / units), ceil(len / 256), kMaxParts) of a row's keys.
inline int64_t work_bytes(const StepArgs& a) {
    const int64_t rows = a.rows, kv_heads = a.cache.kv_heads, G = a.q_heads / kv_heads, k = kv_heads * ((G + kCols - 1) / kCols);
    const int64_t most = a.cache.ld_table << a.cache.page_bits, len = std::min<int64_t>(a.max_len, most);
    auto parts = [](int64_t len, int64_t least) { return std::max<int64_t>(1, std::min<int64_t>((len + least - 1) / least, kMaxParts)); };
    if (a.prefix.groups == 0) {
        const int64_t split = std::min(rows, 511 / k);  // more rows than these are not divided
        return len <= 256 || split == 0 ? 0 : record_bytes(a, std::min(split * parts(len, 256), 512 / k + split));
    }
    const int64_t shared = std::min<int64_t>(a.prefix.max_len, most);
    int64_t own = std::min(rows * parts(len, 256), 512 / k + rows);
    if (rows * k > 512) own = std::max(own, rows * parts(std::min(len, shared + 256), 1024));
    return record_bytes(a, own + std::min(rows * parts(shared, 256), 256 * kCols / a.q_heads + rows));
}

}  // namespace vxs
