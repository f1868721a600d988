// vxs_attn_step.hip — attention of one token per sequence over a paged cache, shared prefixes read once.
//
//   out[r] = sum_s w_s v[s] / sum_s w_s,   w_s = exp(scale q[r] . k[s] - m)
// carried along the keys with the running maximum m; the sums of disjoint sets of keys join as
//   m = max(m_a, m_b),  o = o_a 2^(m_a - m) + o_b 2^(m_b - m),  l likewise      (m in units of log 2).
//
// Bound by reading the cache. A workgroup takes up to 32 query rows that read the same keys, and a range of those
// keys: the heads that share a key head, of one sequence, or for a prefix that sequences share also theirs, stacked. Its
// four waves take the range's tiles in turn, each through LDS of its own that nobody else touches: a wave waits for its
// own loads only, and has the next keys' on the way while it weighs, the next values' while it multiplies. The matrix
// cores are mostly idle columns at few heads, which costs nothing here. At the end the waves join through LDS; where a
// row's keys are in several workgroups, each leaves its sums in the workspace and the last to arrive joins them.
//
// Measured (bf16, 8 key heads of 128 unless said): 256 rows of 1500 to 3000 402 us, 2.36 GB at 5.9 TB/s (a copy: 5.2); 24 of 1000 to 2000
// 32 us, 4.6 TB/s; 4 of 32,500 to 65,000 with 32 query and 4 key heads 82 us, 4.9 TB/s; 96 rows of two prefixes of 4100 and 150 to 300
// tokens of their own 39 us, 122 MB (each row reading its prefix itself: 1.7 GB); one row of 37 tokens 5.5 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_attn_core.h"
#include "vxs_attn_plan.h"
#include "vxs_attn_types.h"

namespace vxs {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kAtOnce = 8;  // parts that are asked for at once to join them

template <int D>
constexpr int kTile = D == 64 ? 64 : 32;  // keys of a wave's tile: 8 KiB of keys, 16 at D = 256

__device__ __forceinline__ void put2(float* p, float a, float b) {
    const uint64_t x = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// (16-byte aligned; the wait for it is the caller's.) The store reads x's registers after it has been issued: they must keep it for two
// wait states more, which the compiler does not see.
__device__ __forceinline__ void put4(float* p, f4 x) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(x) : "memory");
}
__device__ __forceinline__ float2 get2(const float* p) {
    const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)x), __uint_as_float((unsigned)(x >> 32)));
}

// The last prefix group g whose begin(d_off[g], g) <= x: its rows [r0, r1) and the tokens that they read together: whole
// 32s (the rest is each row's own), none for one row alone or where the first row's slot is none. One read for 64 groups.
struct Group {
    int g, r0, r1, shared, slot;
};
template <typename F>
__device__ __forceinline__ Group find_group(const StepArgs& a, int x, int lane, F begin) {
    Group y{0, 0, 0, 0, 0};
    int len = 0;
    for (int g0 = 0; g0 < a.prefix.groups; g0 += 64) {
        const int g = min(g0 + lane, a.prefix.groups - 1);
        const int lo = min(max(a.prefix.d_off[g], 0), a.rows), hi = min(max(a.prefix.d_off[g + 1], lo), a.rows), n = a.prefix.d_len[g];
        const uint64_t before = __ballot(g0 + lane < a.prefix.groups && begin(lo, g) <= x);
        if (!before) break;
        const int at = 63 - __builtin_clzll(before);
        y.g = g0 + at;
        y.r0 = __builtin_amdgcn_readlane(lo, at);
        y.r1 = __builtin_amdgcn_readlane(hi, at);
        len = __builtin_amdgcn_readlane(n, at);
    }
    if (y.r1 - y.r0 >= 2) {
        y.slot = a.slots ? scalar(a.slots, y.r0) : y.r0;
        y.shared = (int)cache_length(a.cache, y.slot, min(len, a.prefix.max_len)) & ~31;
    }
    return y;
}

struct KernelArgs {
    StepArgs a;
    Split sp;
    Records rec;
};

// LDS of a wave: its tile of keys and its tile of values, later its sums [32][D + 4]; then of the workgroup m and l of each
// wave's query rows, and what is done after.
template <int D>
constexpr int kWaveBytes = 2 * kTile<D> * 2 * D > kCols * (D + 4) * 4 ? 2 * kTile<D> * 2 * D : kCols * (D + 4) * 4;
template <int D>
constexpr int kLdsBytes = kWaves * (kWaveBytes<D> + kCols * 8) + kCols * 4;

template <int D, typename T, typename TO>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void attn_step_kernel(KernelArgs args) {
    constexpr int KT = kTile<D>, NB = KT / 32, NG = KT / 16, NI = KT * 2 * D / 1024, TB = KT * 2 * D;
    constexpr int PARTS = sizeof(TO) == 4 ? Vec<T>::kParts : 1;
    constexpr int OS = D + 4;  // floats of a row of the wave's sums
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* wave_ml = reinterpret_cast<float*>(lds + kWaves * kWaveBytes<D>);  // [waves][32][2]
    int* complete = reinterpret_cast<int*>(wave_ml + kWaves * kCols * 2);     // [32]: parts of the rows that are complete
    const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
    const StepArgs& a = args.a;
    const Split& sp = args.sp;

    // ---- this workgroup's query rows and keys: columns c < cols are query rows rho0 + c of the stack that begins at
    // row rbase; keys [c0, c1) of the slot `slot`, whose rows have `own` keys of their own after `shared` ones
    int id = blockIdx.x, head, rbase, rho0, cols, c0, c1, slot, part, len = 0, shared = 0;
    auto range = [&](int from, int i, int chunk, int n, int end) {
        const int64_t a0 = from + (int64_t)i * chunk;
        c0 = (int)min(a0, (int64_t)end);
        c1 = i == n - 1 ? end : (int)min(a0 + chunk, (int64_t)end);
    };
    const int pre_blocks = sp.pre_tiles * sp.pre_parts * sp.heads.d;
    const bool pre = id < pre_blocks;
    if (!pre) id -= pre_blocks;
    // The threads that share this work: the workgroup's, or the wave's (solo); there are no barriers among the latter.
    const bool solo = !pre && sp.solo;
    const int tid = solo ? lane : threadIdx.x, threads = solo ? 64 : kThreads, step = solo ? kTile<D> : kWaves * kTile<D>;
    if (solo) id = id * kWaves + wv;
    auto sync = [&] {
        if (!solo) {
            __syncthreads();
        } else {  // (a wave's own LDS accesses happen in order; the compiler has to keep it for other lanes' data too)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    const int rest = sp.heads.div(id);
    head = id - rest * sp.heads.d;
    const int G = sp.group.d;
    if (pre) {
        part = sp.pre.div(rest);
        const int tile = rest - part * sp.pre_tiles;
        auto begin = [&](int lo, int g) { return (int)((int64_t)lo * G / kCols) + g; };
        const Group x = find_group(a, tile, lane, begin);
        rbase = x.r0;
        rho0 = (tile - begin(x.r0, x.g)) * kCols;
        cols = min((x.r1 - x.r0) * G - rho0, kCols);
        shared = x.shared;
        slot = x.slot;
        if (cols <= 0 || rho0 < 0) return;
        range(0, part, sp.pre_chunk, sp.pre_parts, shared);
        if (c0 >= c1) return;
    } else {
        const int unit = sp.tiles.div(rest), ht = rest - unit * sp.head_tiles;
        rbase = sp.parts.div(unit);
        if (rbase >= a.rows) return;  // (solo: past the last)
        part = unit - rbase * sp.own_parts;
        rho0 = ht * kCols;
        cols = min(G - rho0, kCols);
        slot = a.slots ? scalar(a.slots, rbase) : rbase;
        len = (int)cache_length(a.cache, slot, scalar(a.kv_len, rbase));
        if (sp.pre_parts) {
            const Group x = find_group(a, rbase, lane, [](int lo, int) { return lo; });
            if (rbase >= x.r0 && rbase < x.r1) shared = x.shared;
        }
        range(shared, part, sp.own_chunk, sp.own_parts, len);
        if (c0 >= c1) {
            if (part || shared) return;
            // no keys at all: zeros
            for (int i = tid; i < cols * D; i += threads)
                static_cast<TO*>(a.out)[rbase * a.ldo + (int64_t)(head * G + rho0 + i / D) * D + i % D] = (TO)0.f;
            return;
        }
    }
    const int32_t* pages = a.cache.table + (int64_t)slot * a.cache.ld_table;

    // ---- the wave's tiles begin to load; queries; how many tokens of the slot each sees
    Loader<D> loader;
    loader.init(a.cache, lane);
    char* const kt = lds + wv * kWaveBytes<D>;
    char* const vt = kt + TB;
    const unsigned k_lds = lds_address(kt), v_lds = lds_address(vt);
    const char* const k_base = a.cache.k + (uint64_t)head * a.cache.head_stride;
    const char* const v_base = a.cache.v + (uint64_t)head * a.cache.head_stride;
    const int last_page = (int)a.cache.ld_table - 1;
    uint64_t at[NG];
    auto find = [&](int t) {
#pragma unroll
        for (int g = 0; g < NG; g++) at[g] = granule_offset(a.cache, pages, last_page, t + 16 * g);
    };
    auto fetch = [&](const char* base, unsigned to) {
#pragma unroll
        for (int g = 0; g < NG; g++) loader.load(base + at[g], to + g * 16 * 2 * D);
    };
    int t = c0 + (solo ? 0 : wv * KT);
    if (t < c1) {
        find(t);
        fetch(k_base, k_lds);
        fetch(v_base, v_lds);
    }
    const int col = lane & 31;
    Queries<D, T, PARTS> w;
    w.init();
    const int rho = rho0 + min(col, cols - 1);
    const int over = pre ? sp.group.div(rho) : 0, row = rbase + over, qh = head * G + rho - over * G;
    w.load(col < cols ? static_cast<const T*>(a.q) + row * a.ldq + (int64_t)qh * D : nullptr, lane);
    int seen = c1;
    bool each = false;
    if (pre) {  // a row that ends within the prefix
        len = (int)cache_length(a.cache, a.slots ? a.slots[row] : row, a.kv_len[row]);
        seen = min(c1, len);
        each = __ballot(col < cols && seen < c1) != 0;
    }
    const float c = a.scale * kLog2e;
    w.loaded();
    bool odd = false;
    for (; t < c1; t += step) {
        const bool more = t + step < c1;
        if (more) find(t + step);
        wait_vm<NI>();
        f16v s[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) s[b] = w.scores(kt + b * 32 * 2 * D, lane);
        wait_lds();
        if (more) fetch(k_base, k_lds);
        const bool tail = t + KT > c1;
        if (each || tail) w.hide(s, (each ? seen : c1) - t, lane);
        w.weigh(s, c);
        if (more) wait_vm<NI>();
        else wait_vm<0>();
        if (each || tail) odd |= scrub<D, T, TB>(vt, t, c1, each, lane);
        w.add(vt, s, lane);
        wait_lds();
        if (more) fetch(v_base, v_lds);
    }
    w.finish_sum();
    const KernelArgs again = arguments_again<KernelArgs>();
    const StepArgs& b = again.a;
    if (each && __ballot(odd)) {
        for (t = c0 + wv * KT; t < c1; t += t % KT == KT - 1 ? step - KT + 1 : 1)
            w.add_odd(b.cache.v + (uint64_t)head * b.cache.head_stride +
                          granule_offset(b.cache, b.cache.table + (int64_t)slot * b.cache.ld_table, (int)b.cache.ld_table - 1, t & ~15) +
                          (uint64_t)(t & 15) * b.cache.token_stride,
                      t < seen, lane);
    }
    const Split& sq = again.sp;
    const Records& rec = again.rec;

    // ---- each wave's sums to LDS; whoever reads them joins the waves'
    float* const sums = reinterpret_cast<float*>(kt);
    if (lane < 32) *reinterpret_cast<float2*>(wave_ml + (wv * kCols + col) * 2) = make_float2(w.m, w.l);
    if (col < cols) {
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<f4*>(sums + col * OS + 32 * d + 8 * j + 4 * (lane >> 5)) =
                    f4{w.o[d][4 * j], w.o[d][4 * j + 1], w.o[d][4 * j + 2], w.o[d][4 * j + 3]};
    }
    sync();
    float m, l;
    auto joined = [&](int q, int d) {  // entries d..d + 3 of the sums of query row rho0 + q; sets m and l
        float2 x[kWaves];
        f4 y[kWaves];
        m = kLowest;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            const int from = solo ? wv : i;
            x[i] = *reinterpret_cast<const float2*>(wave_ml + (from * kCols + q) * 2);
            y[i] = *reinterpret_cast<const f4*>(lds + from * kWaveBytes<D> + (q * OS + d) * 4);
            m = fmaxf(m, x[i].x);
        }
        f4 o{0.f, 0.f, 0.f, 0.f};
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            if (solo && i) break;
            const float f = __builtin_amdgcn_exp2f(x[i].x - m);
            l = __builtin_fmaf(x[i].y, f, l);
            o = o + y[i] * f;
        }
        return o;
    };

    auto out_at = [&](int r, int h) { return static_cast<TO*>(b.out) + r * b.ldo + (int64_t)h * D; };
    using o4 = typename Vec<TO>::v4;
    auto parts_of = [](int n, int chunk, int most) { return n > 0 ? min((n - 1) / chunk + 1, most) : 0; };
    constexpr int L = D / 4;  // lanes of a query row, four entries each
    const int d4 = 4 * (tid % L);
    if (!pre && c0 == 0 && c1 == len) {  // the row's keys are all here
        for (int q = tid / L; q < cols; q += threads / L) {
            const f4 x = joined(q, d4);
            const float y = 1.0f / l;
            *reinterpret_cast<o4*>(out_at(rbase, head * G + rho0 + q) + d4) = o4{(TO)(x[0] * y), (TO)(x[1] * y), (TO)(x[2] * y), (TO)(x[3] * y)};
        }
        return;
    }

    // ---- leave the sums, count the query rows that have arrived
    auto record = [&](int r, int p, int q) {
        return rec.base + ((((int64_t)r * sq.heads.d + head) * rec.parts + p) * G + q) * (D / 64 * kBlock);
    };
    auto entries = [](int d) { return d / 64 * kBlock + 4 + d % 64; };
    for (int q = tid / L; q < cols; q += threads / L) {
        const f4 x = joined(q, d4);
        const int up = pre ? sq.group.div(rho0 + q) : 0;
        float* const to = record(rbase + up, pre ? sq.own_parts + part : part, rho0 + q - up * G);
        put4(to + entries(d4), x);
        if (d4 == 0) put2(to, m, l);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    sync();
    const int first = pre ? sq.group.div(rho0) : 0, rows = pre ? sq.group.div(rho0 + cols - 1) - first + 1 : 1;
    int mine = 0;  // parts of row `first + tid` where it is complete
    if (tid < rows) {
        const int r = rbase + first + tid;
        if (pre) len = (int)cache_length(b.cache, b.slots ? b.slots[r] : r, b.kv_len[r]);
        const int own = parts_of(len - shared, sq.own_chunk, sq.own_parts), pres = parts_of(shared, sq.pre_chunk, sq.pre_parts);
        const unsigned n = pre ? min((first + tid + 1) * G, rho0 + cols) - max((first + tid) * G, rho0) : cols;
        unsigned* const count = reinterpret_cast<unsigned*>(rec.base) + ((int64_t)r * sq.heads.d + head) * kBlock + 2;
        const unsigned before = __hip_atomic_fetch_add(count, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool done = before + n == (unsigned)((own + pres) * G);
        if (done) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        mine = done ? (len > 0 ? 1 << 30 : 0) | own << 15 | pres : 0;
        if (!solo) complete[tid] = mine;
    }
    sync();
    // L lanes take a (row, query head) whose row is complete, four entries each, two of them at a time: kAtOnce parts are asked for
    // together (each read is one of the common memory) and joined lane by lane.
    const int sub = tid % L, apart = threads / L;
    for (int pair0 = tid / L; pair0 < rows * G; pair0 += 2 * apart) {
        float2 ml[2][kAtOnce], lo[2][kAtOnce], hi[2][kAtOnce];
        int what[2], own[2], all[2], row[2], q[2];
        auto fetch_parts = [&](int u, int p0) {
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                const int p = p0 + j;
                ml[u][j] = make_float2(kLowest, 0.f);
                lo[u][j] = hi[u][j] = make_float2(0.f, 0.f);
                if (p >= all[u]) continue;
                const float* const at = record(row[u], p < own[u] ? p : sq.own_parts + p - own[u], q[u]);
                ml[u][j] = get2(at);
                lo[u][j] = get2(at + entries(4 * sub));
                hi[u][j] = get2(at + entries(4 * sub) + 2);
            }
        };
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int pair = pair0 + u * apart;
            const int i = sq.group.div(min(pair, rows * G - 1));
            q[u] = pair - i * G;
            row[u] = rbase + first + i;
            what[u] = pair < rows * G ? (solo ? uniform(mine) : complete[i]) : 0;
            own[u] = (what[u] >> 15) & 0x7fff;
            all[u] = own[u] + (what[u] & 0x7fff);
            fetch_parts(u, 0);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float top = kLowest, total = 0.f;
            f4 sum{0.f, 0.f, 0.f, 0.f};
            for (int p = 0; p < all[u]; p += kAtOnce) {
                if (p) fetch_parts(u, p);
                float next = top;
#pragma unroll
                for (int j = 0; j < kAtOnce; j++) next = fmaxf(next, ml[u][j].x);
                const float shrink = __builtin_amdgcn_exp2f(top - next);
                top = next;
                total *= shrink;
                sum = sum * shrink;
#pragma unroll
                for (int j = 0; j < kAtOnce; j++) {
                    const float g = __builtin_amdgcn_exp2f(ml[u][j].x - top);  // (a part that is not there adds zeros)
                    total = __builtin_fmaf(ml[u][j].y, g, total);
                    sum[0] = __builtin_fmaf(lo[u][j].x, g, sum[0]);
                    sum[1] = __builtin_fmaf(lo[u][j].y, g, sum[1]);
                    sum[2] = __builtin_fmaf(hi[u][j].x, g, sum[2]);
                    sum[3] = __builtin_fmaf(hi[u][j].y, g, sum[3]);
                }
            }
            const float y = what[u] >> 30 ? 1.0f / total : 0.f;  // (a row without keys in a group: all weights are zero)
            if (what[u])
                *reinterpret_cast<o4*>(out_at(row[u], head * G + q[u]) + 4 * sub) = o4{(TO)(sum[0] * y), (TO)(sum[1] * y), (TO)(sum[2] * y), (TO)(sum[3] * y)};
        }
    }
}

template <int D, typename T, typename TO>
struct Step {
    static hipError_t go(const StepArgs& a, hipStream_t stream) {
        const Split s = plan_step(a, a.work != nullptr);
        const Records r{static_cast<float*>(a.work), s.own_parts + s.pre_parts};
        const int64_t own = (int64_t)a.rows * a.cache.kv_heads * s.head_tiles * s.own_parts;
        const int64_t blocks = (int64_t)s.pre_tiles * s.pre_parts * a.cache.kv_heads + (s.solo ? (own + kWaves - 1) / kWaves : own);
        if (blocks > UINT32_MAX / kThreads || own > INT32_MAX) return hipErrorInvalidValue;  // (a launch's threads are counted in 32 bits)
        static std::atomic<uint64_t> devices{0};
        if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(attn_step_kernel<D, T, TO>), kLdsBytes<D>, devices); e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_step_kernel<D, T, TO>), dim3((unsigned)blocks), dim3(kThreads), kLdsBytes<D>, stream, KernelArgs{a, s, r});
        return hipGetLastError();
    }
};

}  // namespace

int64_t attn_step_work_bytes(const StepArgs& a) {
    return work_bytes(a);
}

hipError_t launch_attn_step(const StepArgs& a, int dtype, int out_dtype, hipStream_t stream) {
    return by_type<Step>(a, a.cache.head_dim, dtype, out_dtype, stream);
}

}  // namespace vxs
