// vxs_attn_prompt.hip — causal attention of packed sequences' new tokens over a paged cache.
//
// Token j of a sequence's n new ones (of `len` in the cache) sees its keys s < len - n + j + 1:
//   out[t] = sum_s w_s v[s] / sum_s w_s,   w_s = exp(scale q[t] . k[s] - m)
// carried along the keys with the running maximum m.
//
// Bound by the matrix cores: 4 D operations for each query head and key that it sees. The query heads of one key head
// are stacked, row rho = j G + g for token j and head g of G, so all rows of a workgroup read the same keys: a wave
// holds 32 rows (vxs_attn_core.h), QW waves 32 QW consecutive ones, and each tile of keys is loaded into LDS once for
// all of them, the next one while this one is used. Where that leaves compute units idle, KW such groups of waves take a
// workgroup's tiles in turn, and their sums are joined through LDS at the end.
//
// Measured (head_dim 128 unless said): one prompt of 8192, 32 query and 8 key heads, bf16, 533 to 564 us: 1.03 PFLOP/s, where a plain product of
// 8192^3 reaches 1.39; matrix cores busy half of the time at a clock that their load holds near 1.83 GHz, the rest waits on the
// exponentials of the same wave. 24 prompts of 500 to 1000, 16 and 8 heads: 100 us with bf16 outputs (head_dim 64: 60, 256: 271), 156 with fp32 ones, which multiply
// the values three times (fp16 caches twice, with sums apart: 144 to 150). 4 times 65 to 130 tokens after 8000, 32 and 4 heads of 64, fp16: 40 to 42 us, 440 TFLOP/s. One prompt of 93: 8 us.
//
// 8-bit entries: each wave asks for a granule of the tile after the next in registers and leaves it in LDS in 16 bits (vxs_attn_core8.h), between
// the scores of this tile and their weights; conversions at each wave's own reads were as long as the products (prompt of 8192 652 us). With the
// figures' sizes: 561 to 586 us, 24 prompts with fp32 outputs 158 to 161. Queries of fp16, whose scores take a factor for each granule and whose outputs two
// parts of each weight, need more registers than there are (8 to 324 bytes of scratch a lane, but for most instances of D = 64): the prompt of 8192
// 901; 24 prompts with 16-bit outputs, fp16 / bf16, 160 / 113, of 64 93 / 67, of 256 568 / 316.
//
// Cross attention: every token sees all of its slot's keys. 8 times 500 to 1000 tokens over 750 to 1500 8-bit states, 16 heads of 128: 89 us, 590 TFLOP/s;
// 24 times 4 over as many, 8 key heads of 64, fp16: 15.5 us, 3.6 TB/s, 192 workgroups. A workgroup reads all keys of its 64 or 128 rows: few tokens of few
// sequences over long states are faster as rows of a step with their sequences as prefix groups (4 times 4 over 4000 to 8000 of 128: 83 us here, 20
// there; 24 times 4 over 1000 to 2000 of 64: 18.5, 29).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_attn_core8.h"
#include "vxs_attn_types.h"

namespace vxs {
namespace {

template <int D, int QW, int KW, bool E8>
struct Shape {
    static constexpr int kThreads = 64 * QW * KW;
    static constexpr int kRows = 32 * QW;    // query rows of a workgroup
    static constexpr int kKeys = 16 * QW;    // of a tile: each wave loads a granule of 16
    static constexpr int kTile = kKeys * 2 * D;
    static constexpr int kTiles = KW * 4 * kTile;                             // [groups][2 buffers][keys, values]
    static constexpr int kSums = KW == 1 ? 0 : QW * KW * 32 * (D + 4 + 2) * 4;  // [waves][32][D + 4], [waves][32] m and l
    static constexpr int kFactors = KW * 2 * (kKeys / 16) * 4;  // [groups][2 buffers][granules] of 8-bit keys
    static constexpr int kLds = (kTiles > kSums ? kTiles : kSums) + (E8 ? kFactors : 0);
};

// T: the queries' type, E8: over 8-bit entries (else of T), CROSS: every token sees all of its sequence's keys.
template <int D, typename T, typename TO, int QW, int KW, bool E8, bool CROSS>
__global__ __launch_bounds__(64 * QW * KW, D == 256 || QW * KW > 8 ? 1 : 2) void attn_prompt_kernel(PromptArgs a, int tiles, CacheScales entry_scales) {
    using S = Shape<D, QW, KW, E8>;
    constexpr int TB = S::kTile, NB = S::kKeys / 32, NG = S::kKeys / 16, GB = TB / NG, kRows = S::kRows, kKeys = S::kKeys;
    constexpr int PARTS = weight_parts<T, TO, E8>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wv = wave % QW, kg = wave / QW;
    const int kvh = a.cache.kv_heads, G = a.q_heads / kvh;
    // later tiles of a sequence see more keys: they go first
    const int head = blockIdx.x % kvh, tile = tiles - 1 - blockIdx.x / kvh;
    // Sequence i's tiles begin at floor(off[i] G / kRows) + i, so a tile's sequence is found without a scan: the last that
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

    constexpr bool FACTORS = E8 && !std::is_same_v<T, __bf16>;
    std::conditional_t<FACTORS, Queries8<D, T, PARTS, true>, Queries<D, T, PARTS>> w;
    w.init();
    const int col = wv * 32 + (lane & 31);
    const int rho = rho0 + min(col, rows - 1);
    const int j = rho / G, qh = head * G + rho % G;
    auto limit = [&](int j) { return CROSS ? len : max(len - n + j + 1, 0); };  // keys that token j sees
    const int seen = limit(j);
    const int first = uniform(limit((rho0 + min(wv * 32, rows - 1)) / G));  // seen by the wave's first row
    const int last = uniform(limit((rho0 + min(wv * 32 + 31, rows - 1)) / G));
    const int all = uniform(limit(rho0 / G));               // keys that every row of the workgroup sees
    const int end = uniform(limit((rho0 + rows - 1) / G));  // that some row sees
    const float c = a.scale * kLog2e;

    std::conditional_t<E8, Stager<D, T>, Loader<D>> loader;
    loader.init(a.cache, lane);
    const int32_t* pages = a.cache.table + (int64_t)(end ? slot : 0) * a.cache.ld_table;
    const int last_page = (int)a.cache.ld_table - 1;
    const char* const k_base = a.cache.k + (uint64_t)head * a.cache.head_stride;
    const char* const v_base = a.cache.v + (uint64_t)head * a.cache.head_stride;
    char* const own = lds + kg * 4 * TB;
    float* const factors = reinterpret_cast<float*>(lds + S::kLds - S::kFactors) + kg * 2 * NG;
    Scales<1> scales;  // of the granule that was last fetched
    auto fetch = [&](int t, int buffer) {  // each wave 16 of the tile's rows
        const int page = granule_page(a.cache, pages, last_page, t + 16 * wv);
        const uint64_t at = cache_offset(a.cache, page, 0, t + 16 * wv);
        if constexpr (E8) {
            loader.load(k_base + at, v_base + at);
            scales.read(a.cache, entry_scales, 0, page, head, t + 16 * wv, end);
        } else {
            const unsigned to = lds_address(own + buffer * 2 * TB + wv * GB);
            loader.load(k_base + at, to);
            loader.load(v_base + at, to + TB);
        }
    };
    bool odd = false;
    // 8-bit entries: the tile at t, asked for before, goes to its buffer, and the next one is asked for
    auto stage = [&](int t, int buffer) {
        if constexpr (E8) {
            if (t >= end) return;
            if (t - kg * kKeys + KW * kKeys > all) odd |= loader.scrub(t + 16 * wv, end);
            loader.store(own + buffer * 2 * TB + wv * GB, TB, scales);
            if (FACTORS && lane == 0) factors[buffer * NG + wv] = score_factor(c, scales.k[0]);
            if (t + KW * kKeys < end) fetch(t + KW * kKeys, 0);
        }
    };
    if (kg * kKeys < end) fetch(kg * kKeys, 0);
    w.load(col < rows ? static_cast<const T*>(a.q) + (int64_t)(t0 + j) * a.ldq + (int64_t)qh * D : nullptr, lane);
    w.loaded();
    int buffer = 0;
    stage(kg * kKeys, 0);
    for (int base = 0; base < end; base += KW * kKeys, buffer ^= 1) {
        const int t = base + kg * kKeys;
        char* const kt = own + buffer * 2 * TB;
        const bool partly = base + KW * kKeys > all;  // some row does not see all of the tiles: each wave looks through its part of the values
        if (!E8) wait_vm<0>();
        __syncthreads();  // the tiles are there, and nobody reads the other buffers any more
        if (!E8 && t + KW * kKeys < end) fetch(t + KW * kKeys, buffer ^ 1);
        if (!E8 && partly) {
            if (t < end) odd |= scrub<D, T, GB>(kt + TB + wv * GB, t + 16 * wv, end, true, lane);
            __syncthreads();
        }
        if (t >= (E8 ? end : last)) continue;  // (8-bit entries: every wave has its part of the next tile to stage)
        f16v s[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) s[b] = w.scores(kt + b * 2 * GB, lane);
        stage(t + KW * kKeys, buffer ^ 1);
        if (t + kKeys > first) w.hide(s, seen - t, lane);
        if constexpr (FACTORS) {
            float f[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) f[g] = factors[buffer * NG + g];
            w.weigh(s, f);
        } else {
            w.weigh(s, c);
        }
        w.add(kt + TB, s, lane);
    }
    if (__syncthreads_or(odd)) {
        for (int t = all / (KW * kKeys) * (KW * kKeys); t < end; t++)  // (the tiles that were looked through)
            if (KW == 1 || t / kKeys % KW == kg)
                add_odd<E8>(w, v_base + granule_offset(a.cache, pages, last_page, t & ~15) + (uint64_t)(t & 15) * a.cache.token_stride, t < seen, lane);
    }
    w.finish_sum();
    using o4 = typename Vec<TO>::v4;
    if (KW == 1) {
        if (col < rows) {
            const float r = seen > 0 ? 1.0f / w.l : 0.f;
            TO* out = static_cast<TO*>(a.out) + (int64_t)(t0 + j) * a.ldo + (int64_t)qh * D + 4 * (lane >> 5);
#pragma unroll
            for (int b = 0; b < D / 32; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<o4*>(out + 32 * b + 8 * i) =
                        o4{(TO)(w.o[b][4 * i] * r), (TO)(w.o[b][4 * i + 1] * r), (TO)(w.o[b][4 * i + 2] * r), (TO)(w.o[b][4 * i + 3] * r)};
        }
        return;
    }
    // (the barrier above: every wave is done with its tiles)
    constexpr int OS = D + 4;
    float* const sums = reinterpret_cast<float*>(lds);
    float* const ml = sums + QW * KW * 32 * OS;
#pragma unroll
    for (int b = 0; b < D / 32; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<f4*>(sums + (wave * 32 + (lane & 31)) * OS + 32 * b + 8 * i + 4 * (lane >> 5)) =
                f4{w.o[b][4 * i], w.o[b][4 * i + 1], w.o[b][4 * i + 2], w.o[b][4 * i + 3]};
    if (lane < 32) *reinterpret_cast<float2*>(ml + (wave * 32 + lane) * 2) = make_float2(w.m, w.l);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += S::kThreads) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));  // row r is column r % 32 of waves r / 32 + QW * group
        float m = kLowest, l = 0.f;
#pragma unroll
        for (int g = 0; g < KW; g++) m = fmaxf(m, ml[(g * QW * 32 + r) * 2]);
        f4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KW; g++) {
            const float2 x = *reinterpret_cast<const float2*>(ml + (g * QW * 32 + r) * 2);
            const float f = __builtin_amdgcn_exp2f(x.x - m);
            l = __builtin_fmaf(x.y, f, l);
            o = o + *reinterpret_cast<const f4*>(sums + (g * QW * 32 + r) * OS + d) * f;
        }
        const int jr = (rho0 + r) / G, h = head * G + (rho0 + r) % G;
        const float y = limit(jr) > 0 ? 1.0f / l : 0.f;
        *reinterpret_cast<o4*>(static_cast<TO*>(a.out) + (int64_t)(t0 + jr) * a.ldo + (int64_t)h * D + d) =
            o4{(TO)(o[0] * y), (TO)(o[1] * y), (TO)(o[2] * y), (TO)(o[3] * y)};
    }
}

struct Call {
    PromptArgs a;
    CacheScales scales;
    bool cross;
};

template <int D, typename T, typename TO, bool E8>
struct Prompt {
    template <int QW, int KW>
    static hipError_t launch(const Call& c, hipStream_t stream) {
        return c.cross ? launch<QW, KW, true>(c, stream) : launch<QW, KW, false>(c, stream);
    }
    template <int QW, int KW, bool CROSS>
    static hipError_t launch(const Call& c, hipStream_t stream) {
        const PromptArgs& a = c.a;
        using S = Shape<D, QW, KW, E8>;
        const int64_t tiles = tiles_of(a, S::kRows);
        if (tiles * a.cache.kv_heads > UINT32_MAX / S::kThreads) return hipErrorInvalidValue;  // (a launch's threads are counted in 32 bits)
        static std::atomic<uint64_t> devices{0};
        if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(attn_prompt_kernel<D, T, TO, QW, KW, E8, CROSS>), S::kLds, devices); e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_prompt_kernel<D, T, TO, QW, KW, E8, CROSS>), dim3((unsigned)(tiles * a.cache.kv_heads)), dim3(S::kThreads), S::kLds, stream,
                           a, (int)tiles, c.scales);
        return hipGetLastError();
    }
    static int64_t tiles_of(const PromptArgs& a, int rows) { return (int64_t)a.tokens * (a.q_heads / a.cache.kv_heads) / rows + a.seqs; }
    static hipError_t go(const Call& c, hipStream_t stream) {
        const PromptArgs& a = c.a;
        // Four groups of two waves (two at D = 256, for the LDS) while 128 rows a workgroup leave compute units idle and a cache
        // may hold more than a few tiles (us, groups / 128 rows: one prompt of 1000 18.8 / 25.5, of 2000, 264 workgroups, 37 / 45,
        // 4 of 500 to 1000, 408 workgroups, 43 / 27; 130 tokens after 8000 91 / 162; one of 93 9.5 / 7.9).
        const int64_t keys = a.cache.ld_table << a.cache.page_bits;
        if (tiles_of(a, 128) * a.cache.kv_heads <= 288 && keys > 256) {
            // D = 64 leaves LDS for eight groups, one workgroup a compute unit: over long contexts, whose tiles arrive too
            // late for four (us, eight / four: 4 times 130 after 8000 47 / 56, after 4000 27 / 31, after 2000 18 / 19, one time 64 after
            // 1000 13.0 / 12.5; 16 times 64 after 2000, 576 workgroups, 31 / 26; whole states, which nothing hides: 24
            // times 4 over 750 to 1500 15.5 / 15.9, of 8 bits 19.3 / 21.6; over 350 to 700 10.8 / 10.3, 11.6 / 12.0; over 500 to 1000 12.6 /
            // 12.5, 14.5 / 15.7; over 1000 to 2000 18.3 / 18.8, 23.8 / 27.9; 4 times 64 over 550 to 1100 13.0 / 12.3, 16.6 / 16.8; over 100 to
            // 200 in a table of 2000 7.4 / 6.4, 8.0 / 7.1).
            if constexpr (D == 64)
                if (keys > (c.cross ? 1024 : 2048) && tiles_of(a, 64) * a.cache.kv_heads <= 256) return launch<2, 8>(c, stream);
            return launch<2, D == 256 ? 2 : 4>(c, stream);
        }
        return launch<4, 1>(c, stream);
    }
};

}  // namespace

hipError_t launch_attn_prompt(const PromptArgs& a, const CacheScales& scales, bool cross, int dtype, int out_dtype, hipStream_t stream) {
    const Call c{a, scales, cross};
    return scales.k ? by_type<Prompt, true>(c, a.cache.head_dim, dtype, out_dtype, stream) : by_type<Prompt, false>(c, a.cache.head_dim, dtype, out_dtype, stream);
}

}  // namespace vxs
