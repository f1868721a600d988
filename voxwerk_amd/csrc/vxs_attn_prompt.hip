// vxs_attn_prompt.hip — causal attention of packed sequences' new tokens over a paged cache.
//
// Token j of a sequence's n new ones (of `len` in the cache) sees its keys s < len - n + j + 1:
//   out[t] = sum_s w_s v[s] / sum_s w_s,   w_s = exp(scale q[t] . k[s] - m)
// carried along the keys with the running maximum m.
//
// Bound by the matrix cores: 4 D operations for each query head and key that it sees. The query heads of one key head
// are stacked, row rho = j G + g for token j and head g of G, so all rows of a workgroup read the same keys: a wave
// holds 32 rows (vxs_attn_core.h), the four waves of a workgroup 128 consecutive ones, and each tile of 64 keys is loaded
// into LDS once for all four, the next one while this one is used.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_attn_core.h"
#include "vxs_attn_types.h"

namespace vxs {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // query rows of a workgroup
constexpr int kKeys = 64;           // of a tile

template <int D, typename T, typename TO>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void attn_prompt_kernel(PromptArgs a, int tiles) {
    constexpr int TB = kKeys * 2 * D, NB = kKeys / 32, GB = 16 * 2 * D;
    constexpr bool SPLIT = sizeof(TO) == 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];  // [2 buffers][keys, values][64][D]
    const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
    const int kvh = a.cache.kv_heads, G = a.q_heads / kvh;
    // later tiles of a sequence see more keys: they go first
    const int head = blockIdx.x % kvh, tile = tiles - 1 - blockIdx.x / kvh;
    // Sequence i's tiles begin at floor(off[i] G / 128) + i, so a tile's sequence is found without a scan: the last that
    // begins at or before it, 64 of them in one read.
    int seq = 0, t0 = 0, n = 0;
    auto begin = [&](int off, int i) { return (int)((int64_t)off * G / kRows) + i; };
    for (int i0 = 0; i0 < a.seqs; i0 += 64) {
        const int i = min(i0 + lane, a.seqs - 1);
        const int off = min(max(a.q_off[i], 0), a.tokens), next = min(max(a.q_off[i + 1], off), a.tokens);
        const uint64_t before = __ballot(i0 + lane < a.seqs && begin(off, i) <= tile);
        if (!before) break;
        const int at = 63 - __builtin_clzll(before);
        seq = i0 + at;
        t0 = __builtin_amdgcn_readlane(off, at);
        n = __builtin_amdgcn_readlane(next, at) - t0;
    }
    const int rho0 = (tile - begin(t0, seq)) * kRows;
    const int rows = min(n * G - rho0, kRows);
    if (rows <= 0 || rho0 < 0) return;
    const int slot = a.slots ? scalar(a.slots, seq) : seq;
    const int len = (int)cache_length(a.cache, slot, scalar(a.kv_len, seq));

    Queries<D, T, SPLIT> w;
    w.init();
    const int col = wv * 32 + (lane & 31);
    const int rho = rho0 + min(col, rows - 1);
    const int j = rho / G, qh = head * G + rho % G;
    const int seen = max(len - n + j + 1, 0);
    const int first = uniform(max(len - n + (rho0 + min(wv * 32, rows - 1)) / G + 1, 0));  // seen by the wave's first row
    const int last = uniform(max(len - n + (rho0 + min(wv * 32 + 31, rows - 1)) / G + 1, 0));
    const int end = max(len - n + (rho0 + rows - 1) / G + 1, 0);  // keys of the workgroup
    const float c = a.scale * kLog2e;

    Loader<D> loader;
    loader.init(a.cache, lane);
    const int32_t* pages = a.cache.table + (int64_t)(end ? slot : 0) * a.cache.ld_table;
    const int last_page = (int)a.cache.ld_table - 1;
    const char* const k_base = a.cache.k + (uint64_t)head * a.cache.head_stride;
    const char* const v_base = a.cache.v + (uint64_t)head * a.cache.head_stride;
    auto fetch = [&](int t, int buffer) {  // each wave 16 of the tile's 64 rows
        const uint64_t at = granule_offset(a.cache, pages, last_page, t + 16 * wv);
        const unsigned to = lds_address(lds + buffer * 2 * TB + wv * GB);
        loader.load(k_base + at, to);
        loader.load(v_base + at, to + TB);
    };
    if (end > 0) fetch(0, 0);
    w.load(col < rows ? static_cast<const T*>(a.q) + (int64_t)(t0 + j) * a.ldq + (int64_t)qh * D : nullptr, lane);
    w.loaded();
    const int all = uniform(max(len - n + rho0 / G + 1, 0));  // keys that every row of the workgroup sees
    bool odd = false;
    int buffer = 0;
    for (int t = 0; t < end; t += kKeys, buffer ^= 1) {
        wait_vm<0>();
        __syncthreads();  // the tile is there, and nobody reads the other buffer any more
        if (t + kKeys < end) fetch(t + kKeys, buffer ^ 1);
        char* const kt = lds + buffer * 2 * TB;
        if (t + kKeys > all) {  // some row does not see all of the tile: each wave looks through a quarter of the values
            odd |= scrub<D, T, GB>(kt + TB + wv * GB, t + 16 * wv, end, true, lane);
            __syncthreads();
        }
        if (t >= last) continue;
        f16v s[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) s[b] = w.scores(kt + b * 32 * 2 * D, lane);
        if (t + kKeys > first) w.hide(s, seen - t, lane);
        w.weigh(s, c);
        w.add(kt + TB, s, lane);
    }
    if (__syncthreads_or(odd)) {
        for (int t = all & ~(kKeys - 1); t < end; t++)
            w.add_odd(a.cache.v + (uint64_t)head * a.cache.head_stride + granule_offset(a.cache, pages, last_page, t & ~15) +
                          (uint64_t)(t & 15) * a.cache.token_stride,
                      t < seen, lane);
    }
    w.finish_sum();
    if (col < rows) {
        const float r = seen > 0 ? 1.0f / w.l : 0.f;
        using o4 = typename Vec<TO>::v4;
        TO* out = static_cast<TO*>(a.out) + (int64_t)(t0 + j) * a.ldo + (int64_t)qh * D + 4 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<o4*>(out + 32 * b + 8 * i) =
                    o4{(TO)(w.o[b][4 * i] * r), (TO)(w.o[b][4 * i + 1] * r), (TO)(w.o[b][4 * i + 2] * r), (TO)(w.o[b][4 * i + 3] * r)};
    }
}

template <int D, typename T, typename TO>
struct Prompt {
    static hipError_t go(const PromptArgs& a, hipStream_t stream) {
        constexpr int lds = 2 * 2 * kKeys * 2 * D;
        const int G = a.q_heads / a.cache.kv_heads;
        const int64_t tiles = (int64_t)a.tokens * G / kRows + a.seqs;
        if (tiles * a.cache.kv_heads > INT32_MAX) return hipErrorInvalidValue;
        static const hipError_t ready = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_prompt_kernel<D, T, TO>),
                                                            hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (ready != hipSuccess) return ready;
        hipLaunchKernelGGL((attn_prompt_kernel<D, T, TO>), dim3((unsigned)(tiles * a.cache.kv_heads)), dim3(kThreads), lds, stream, a,
                           (int)tiles);
        return hipGetLastError();
    }
};

}  // namespace

hipError_t launch_attn_prompt(const PromptArgs& a, int dtype, int out_dtype, hipStream_t stream) {
    return by_type<Prompt>(a, a.cache.head_dim, dtype, out_dtype, stream);
}

}  // namespace vxs
