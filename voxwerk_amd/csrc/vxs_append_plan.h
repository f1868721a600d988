// vxs_append_plan.h — how the work of an append to an 8-bit cache (vxs_append8.hip) is divided.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace vxs {

// A workgroup's waves, and those of the others at its blockIdx.x, share the items of kChunk rows: each block of 16 tokens that
// begins among them (its rows may go on in the next chunk), a head's keys or values; and each row's queries, kSets wave loads of them.
constexpr int kAppend8Threads = 256;
constexpr int kSets = 4;
constexpr int kChunk = 16;

struct Append8Grid {
    unsigned chunks, parts;  // blockIdx.x and .y
};

// q_heads, kv_heads: 0 where the call has none of them.
inline Append8Grid plan_append8(int tokens, int q_heads, int kv_heads, int head_dim) {
    const int heads = 512 / head_dim;  // of a wave at a time
    const int64_t chunks = (tokens + kChunk - 1) / kChunk, rows = std::min(tokens, kChunk);
    // Two items a wave where rows fill their blocks; where each is alone in its own there are more of them, which get a wave each up to
    // 2048 workgroups (us, two / one: 24 prompts of 500 to 1000, 32 + 2 x 8 heads, 138 / 146; 16 of 1000 88 / 91; 1100 tokens of one or of as
    // many sequences 11 and 12, 11 and 12; a wave for each item that there might be 150; 97; 11 and 12).
    const int64_t queries = rows * ((q_heads + (int64_t)kSets * heads - 1) / (kSets * heads));
    const int64_t filled = (2 * (int64_t)kv_heads + queries) / 8, alone = (rows * 2 * ((kv_heads + (int64_t)heads - 1) / heads) + queries + 3) / 4;
    // (a launch's threads are counted in 32 bits)
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({std::max(filled, std::min(alone, 2048 / chunks)), UINT32_MAX / kAppend8Threads / chunks, 65535}));
    return {(unsigned)chunks, (unsigned)parts};
}

}  // namespace vxs
