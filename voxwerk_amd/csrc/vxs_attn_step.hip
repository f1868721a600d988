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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_attn_core.h"
#include "vxs_attn_types.h"

namespace vxs {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 32;       // query rows of a workgroup
constexpr int kMaxParts = 256;  // of a row's keys
constexpr int kJoin = 8;        // parts that a wave reads at once to join them

// How a call's work is divided; the host and the kernel compute it from the same numbers.
struct Split {
    int group;        // query heads per key head
    int head_tiles;   // of 32 query heads each
    int own_parts;    // of a row's own keys, of own_chunk each (the last takes what is left)
    int own_chunk;    // (chunk times parts may pass 32 bits)
    int pre_tiles;    // of 32 stacked query rows of all prefix groups, at most
    int pre_parts;
    int pre_chunk;
};

template <int D>
constexpr int kTile = D == 64 ? 64 : 32;  // keys of a wave's tile: 8 KiB of keys, 16 at D = 256

Split plan_step(const StepArgs& a, bool work) {
    const int rows = a.rows, kv_heads = a.cache.kv_heads, groups = work ? a.prefix.groups : 0;
    const int64_t most = a.cache.ld_table << a.cache.page_bits;  // (below 2^31 - 256)
    const int max_len = (int)std::min<int64_t>(a.max_len, most), max_prefix = (int)std::min<int64_t>(a.prefix.max_len, most);
    Split s{};
    s.group = a.q_heads / kv_heads;
    s.head_tiles = (s.group + kCols - 1) / kCols;
    auto parts = [](int64_t units, int len, int& chunk) {
        // about two workgroups for each compute unit, of at least 256 keys
        int64_t n = std::max<int64_t>(1, (512 + units - 1) / units);
        n = std::min<int64_t>({n, ((int64_t)len + 255) / 256, kMaxParts});
        n = std::max<int64_t>(n, 1);
        chunk = (int)std::max<int64_t>(256, (((int64_t)len + n - 1) / n + 255) / 256 * 256);
        return (int)std::max<int64_t>(1, ((int64_t)len + chunk - 1) / chunk);
    };
    s.own_parts = parts((int64_t)std::max(rows, 1) * kv_heads * s.head_tiles, max_len, s.own_chunk);
    if (!work) {
        s.own_parts = 1;
        s.own_chunk = INT32_MAX;
    }
    if (groups > 0 && max_prefix > 0) {
        s.pre_tiles = (int)(((int64_t)rows * s.group) / kCols + groups);
        s.pre_parts = parts((int64_t)s.pre_tiles * kv_heads, max_prefix, s.pre_chunk);
    }
    return s;
}

// The workspace: a count of arrived query rows per (row, key head), then the sums: per (row, key head), part and
// query head, D entries of o; then m and l. A part's sums are written and read at the device's common memory (agent
// scope: past the caches of one XCD), whole-cache fences would cost more than the step.
struct Records {
    unsigned* count;
    float* o;
    float* ml;
    int parts;
};
__host__ __device__ inline int64_t records_counts(int rows, int kv_heads) { return ((int64_t)rows * kv_heads + 3) / 4 * 4; }

int64_t work_bytes(const StepArgs& a, const Split& s) {
    const int parts = s.own_parts + s.pre_parts;
    if (parts <= 1) return 0;
    return 4 * (records_counts(a.rows, a.cache.kv_heads) + (int64_t)a.rows * a.q_heads * parts * (a.cache.head_dim + 2));
}

__device__ __forceinline__ void put2(float* p, float a, float b) {
    const uint64_t x = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
    const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)x), __uint_as_float((unsigned)(x >> 32)));
}

// The last i with base(i) <= x, of n > 0 ascending ones (base(0) taken as below x).
template <typename F>
__device__ __forceinline__ int last_at_or_below(int n, int x, F base) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base(mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Group g's rows [r0, r1) and the tokens that they read together: whole 32s (the rest is each row's own), none for
// one row alone or where the first row's slot is none.
struct Group {
    int r0, r1, shared;
};
__device__ __forceinline__ Group group_at(const StepArgs& a, int g) {
    Group x;
    x.r0 = min(max(a.prefix.d_off[g], 0), a.rows);
    x.r1 = min(max(a.prefix.d_off[g + 1], x.r0), a.rows);
    x.shared = 0;
    if (x.r1 - x.r0 >= 2) {
        const int slot = a.slots ? a.slots[x.r0] : x.r0;
        x.shared = (int)cache_length(a.cache, slot, min(a.prefix.d_len[g], a.prefix.max_len)) & ~31;
    }
    return x;
}
// The tokens that row r shares with its group.
__device__ __forceinline__ int shared_of(const StepArgs& a, const Split& s, int r) {
    if (!s.pre_parts) return 0;
    const int g = last_at_or_below(a.prefix.groups, r, [&](int i) { return a.prefix.d_off[i]; });
    const Group x = group_at(a, g);
    return r >= x.r0 && r < x.r1 ? x.shared : 0;
}
__device__ __forceinline__ int parts_of(int len, int chunk, int most) { return len > 0 ? min((len - 1) / chunk + 1, most) : 0; }

struct KernelArgs {
    StepArgs a;
    Split sp;
    Records rec;
};

template <int D>
constexpr int lds_bytes() {
    const int tiles = kWaves * 2 * kTile<D> * 2 * D, join = 2 * kCols * (D + 4) * 4;
    return (tiles > join ? tiles : join) + 4 * kWaves * kCols * 2 + 4 * kCols * 2;
}

template <int D, typename T, typename TO>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void attn_step_kernel(KernelArgs args) {
    const StepArgs& a = args.a;
    const Split& sp = args.sp;
    constexpr int KT = kTile<D>, NB = KT / 32, NG = KT / 16, NI = KT * 2 * D / 1024, TB = KT * 2 * D;
    constexpr bool SPLIT = sizeof(TO) == 4;
    constexpr int OS = D + 4;  // floats of a row in the join
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int kTop = kWaves * 2 * TB > 2 * kCols * OS * 4 ? kWaves * 2 * TB : 2 * kCols * OS * 4;
    float* wave_ml = reinterpret_cast<float*>(lds + kTop);  // [waves][32][2]
    float* sums = wave_ml + kWaves * kCols * 2;              // [32]: l of the workgroup; then the rows that are complete
    const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
    const int kvh = a.cache.kv_heads, G = sp.group;

    // ---- this workgroup's query rows and keys: columns c < cols are query rows rho0 + c of the stack that begins at
    // row rbase; keys [c0, c1) of the slot `slot`
    int id = blockIdx.x, head, rbase, rho0, cols, c0, c1, slot, part, last_page, own_shared = 0;
    auto range = [&](int from, int i, int chunk, int n, int end) {
        const int64_t a0 = from + (int64_t)i * chunk;
        c0 = (int)min(a0, (int64_t)end);
        c1 = i == n - 1 ? end : (int)min(a0 + chunk, (int64_t)end);
    };
    const int pre_blocks = sp.pre_tiles * sp.pre_parts * kvh;
    const bool pre = id < pre_blocks;
    if (pre) {
        head = id % kvh;
        const int tile = (id / kvh) % sp.pre_tiles;
        part = id / kvh / sp.pre_tiles;
        const int g = last_at_or_below(a.prefix.groups, tile, [&](int i) {
            return (int)((int64_t)min(max(a.prefix.d_off[i], 0), a.rows) * G / kCols) + i;
        });
        const Group x = group_at(a, g);
        rbase = x.r0;
        rho0 = (tile - ((int)((int64_t)x.r0 * G / kCols) + g)) * kCols;
        cols = min((x.r1 - x.r0) * G - rho0, kCols);
        if (cols <= 0 || rho0 < 0) return;
        range(0, part, sp.pre_chunk, sp.pre_parts, x.shared);
        if (c0 >= c1) return;
        slot = a.slots ? a.slots[x.r0] : x.r0;
        last_page = (x.shared - 1) >> a.cache.page_bits;
    } else {
        id -= pre_blocks;
        head = id % kvh;
        id /= kvh;
        const int ht = id % sp.head_tiles;
        id /= sp.head_tiles;
        part = id % sp.own_parts;
        rbase = id / sp.own_parts;
        rho0 = ht * kCols;
        cols = min(G - rho0, kCols);
        slot = a.slots ? a.slots[rbase] : rbase;
        const int len = (int)cache_length(a.cache, slot, a.kv_len[rbase]);
        const int shared = own_shared = shared_of(a, sp, rbase);
        range(shared, part, sp.own_chunk, sp.own_parts, len);
        if (c0 >= c1) {
            if (part || shared) return;
            // no keys at all: zeros
            for (int i = threadIdx.x; i < cols * D; i += kThreads)
                static_cast<TO*>(a.out)[rbase * a.ldo + (int64_t)(head * G + rho0 + i / D) * D + i % D] = (TO)0.f;
            return;
        }
        last_page = (len - 1) >> a.cache.page_bits;
    }
    const int32_t* pages = a.cache.table + (int64_t)slot * a.cache.ld_table;

    // ---- queries; how many tokens of the slot each sees
    const int col = lane & 31;
    Queries<D, T, SPLIT> w;
    w.init();
    const int rho = rho0 + min(col, cols - 1);
    const int row = rbase + (pre ? rho / G : 0), qh = head * G + (pre ? rho % G : rho);
    w.load(col < cols ? static_cast<const T*>(a.q) + row * a.ldq + (int64_t)qh * D : nullptr, lane);
    int seen = c1;
    bool each = false;
    if (pre) {  // a row that ends within the prefix
        seen = min(c1, (int)cache_length(a.cache, a.slots ? a.slots[row] : row, a.kv_len[row]));
        each = __ballot(col < cols && seen < c1) != 0;
    }
    const float c = a.scale * kLog2e;

    // ---- the wave's tiles
    Loader<D> loader;
    loader.init(a.cache, lane);
    char* kt = lds + wv * 2 * TB;
    char* vt = kt + TB;
    const unsigned k_lds = lds_address(kt), v_lds = lds_address(vt);
    const char* const k_base = a.cache.k + (uint64_t)head * a.cache.head_stride;
    const char* const v_base = a.cache.v + (uint64_t)head * a.cache.head_stride;
    uint64_t at[NG];
    auto find = [&](int t) {
#pragma unroll
        for (int g = 0; g < NG; g++) at[g] = granule_offset(a.cache, pages, last_page, t + 16 * g);
    };
    auto fetch = [&](const char* base, unsigned to) {
#pragma unroll
        for (int g = 0; g < NG; g++) loader.load(base + at[g], to + g * 16 * 2 * D);
    };
    int t = c0 + wv * KT;
    if (t < c1) {
        find(t);
        fetch(k_base, k_lds);
        fetch(v_base, v_lds);
    }
    w.loaded();
    for (; t < c1; t += kWaves * KT) {
        const bool more = t + kWaves * KT < c1;
        if (more) find(t + kWaves * KT);
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
        if (each) w.template add<NB, decltype(w)::kEach>(vt, s, seen - t, lane);
        else if (tail) w.template add<NB, decltype(w)::kTail>(vt, s, c1 - t, lane);
        else w.template add<NB, decltype(w)::kAll>(vt, s, KT, lane);
        wait_lds();
        if (more) fetch(v_base, v_lds);
    }
    w.finish_sum();
    const KernelArgs again = arguments_again<KernelArgs>();
    const StepArgs& b = again.a;
    const Split& sq = again.sp;
    const Records& rec = again.rec;

    // ---- the waves' sums become one: each at the common maximum, waves 2 and 3 to 0 and 1, then all threads add those two
    if (lane < 32) {
        wave_ml[(wv * kCols + col) * 2] = w.m;
        wave_ml[(wv * kCols + col) * 2 + 1] = w.l;
    }
    __syncthreads();  // (also: every wave is done with its tiles)
    float m = kLowest, l = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) m = fmaxf(m, wave_ml[(i * kCols + col) * 2]);
#pragma unroll
    for (int i = 0; i < kWaves; i++) l += wave_ml[(i * kCols + col) * 2 + 1] * __builtin_amdgcn_exp2f(wave_ml[(i * kCols + col) * 2] - m);
    const float f = __builtin_amdgcn_exp2f(w.m - m);
    float* joined = reinterpret_cast<float*>(lds);
    auto place = [&](int half, int b, int j) {
        return reinterpret_cast<f4*>(joined + (half * kCols + col) * OS + 32 * b + 8 * j + 4 * (lane >> 5));
    };
#pragma unroll
    for (int b = 0; b < D / 32; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) w.o[b][i] *= f;
    if (wv >= 2 && col < cols) {
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) *place(wv - 2, b, j) = f4{w.o[b][4 * j], w.o[b][4 * j + 1], w.o[b][4 * j + 2], w.o[b][4 * j + 3]};
    }
    __syncthreads();
    if (wv < 2 && col < cols) {
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                f4* p = place(wv, b, j);
                *p = *p + f4{w.o[b][4 * j], w.o[b][4 * j + 1], w.o[b][4 * j + 2], w.o[b][4 * j + 3]};
            }
        if (wv == 0 && lane < 32) {
            wave_ml[col * 2] = m;  // (wave 0 has read its part; the others' are read above, before the barrier)
            sums[col] = l;
        }
    }
    __syncthreads();

    const int first = pre ? rho0 / G : 0, rows = pre ? (rho0 + cols - 1) / G - first + 1 : 1;
    const int my_parts = pre ? 0 : parts_of((int)cache_length(b.cache, slot, b.kv_len[rbase]) - own_shared, sq.own_chunk, sq.own_parts);
    auto out_at = [&](int r, int h) { return static_cast<TO*>(b.out) + r * b.ldo + (int64_t)h * D; };
    using o4 = typename Vec<TO>::v4;
    if (!pre && my_parts == 1 && c0 == 0) {  // the row's keys are all here
        for (int i = threadIdx.x; i < cols * (D / 4); i += kThreads) {
            const int q = i / (D / 4), d = 4 * (i % (D / 4));
            const f4 x = *reinterpret_cast<const f4*>(joined + q * OS + d) + *reinterpret_cast<const f4*>(joined + (kCols + q) * OS + d);
            const float r = 1.0f / sums[q];
            *reinterpret_cast<o4*>(out_at(rbase, head * G + rho0 + q) + d) = o4{(TO)(x[0] * r), (TO)(x[1] * r), (TO)(x[2] * r), (TO)(x[3] * r)};
        }
        return;
    }

    // ---- leave the sums, count the query rows that have arrived
    const int slot_of_part = pre ? sq.own_parts + part : part;
    auto record = [&](int r, int p, int q) { return (((int64_t)r * b.cache.kv_heads + head) * rec.parts + p) * G + q; };
    for (int i = threadIdx.x; i < cols * (D / 4); i += kThreads) {
        const int q = i / (D / 4), d = 4 * (i % (D / 4));
        const f4 x = *reinterpret_cast<const f4*>(joined + q * OS + d) + *reinterpret_cast<const f4*>(joined + (kCols + q) * OS + d);
        const int at = rho0 + q;
        float* to = rec.o + record(rbase + (pre ? at / G : 0), slot_of_part, pre ? at % G : at) * D + d;
        put2(to, x[0], x[1]);
        put2(to + 2, x[2], x[3]);
    }
    if (threadIdx.x < cols) {
        const int at = rho0 + threadIdx.x;
        put2(rec.ml + record(rbase + (pre ? at / G : 0), slot_of_part, pre ? at % G : at) * 2, wave_ml[threadIdx.x * 2], sums[threadIdx.x]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* complete = reinterpret_cast<int*>(sums + kCols);  // [32]: parts of each row that is complete, or 0
    if (threadIdx.x < rows) {
        const int r = rbase + first + threadIdx.x;
        const int from = max((first + (int)threadIdx.x) * G, rho0), to = min((first + (int)threadIdx.x + 1) * G, rho0 + cols);
        const int rs = shared_of(b, sq, r);
        const int len = (int)cache_length(b.cache, b.slots ? b.slots[r] : r, b.kv_len[r]);
        const int own = parts_of(max(len - rs, 0), sq.own_chunk, sq.own_parts), all = own + (rs ? parts_of(rs, sq.pre_chunk, sq.pre_parts) : 0);
        const unsigned n = (pre ? to - from : cols);
        const unsigned before = __hip_atomic_fetch_add(rec.count + (int64_t)r * b.cache.kv_heads + head, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool done = before + n == (unsigned)(all * G);
        if (done) __hip_atomic_store(rec.count + (int64_t)r * b.cache.kv_heads + head, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        complete[threadIdx.x] = done ? own << 16 | (all - own) : 0;
    }
    __syncthreads();
    for (int i = 0; i < rows; i++) {
        const int parts = complete[i], own = parts >> 16, all = own + (parts & 0xffff);
        if (!parts) continue;
        const int r = rbase + first + i;
        const bool any = cache_length(b.cache, b.slots ? b.slots[r] : r, b.kv_len[r]) > 0;
        // A wave takes a query head at a time: a part's m and l are a lane's, then its sums are read, kJoin at once
        // (each such read comes from the common memory), lanes along D.
        for (int q = wv; q < G; q += kWaves) {
            auto at = [&](int p) { return record(r, p < own ? p : sq.own_parts + p - own, q); };
            constexpr int E = D / 128 ? D / 128 : 1;  // pairs of entries of a lane
            const bool mine = 2 * lane < D;
            float top = kLowest, total = 0.f;
            for (int p = lane; p < all; p += 64) top = fmaxf(top, get2(rec.ml + at(p) * 2).x);
            for (int x = 32; x >= 1; x /= 2) top = fmaxf(top, __shfl_xor(top, x));
            float2 sum[E];
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = make_float2(0.f, 0.f);
            for (int p0 = 0; p0 < all; p0 += 64) {
                const float2 ml = p0 + lane < all ? get2(rec.ml + at(p0 + lane) * 2) : make_float2(kLowest, 0.f);
                const float g = p0 + lane < all ? __builtin_amdgcn_exp2f(ml.x - top) : 0.f;
                total = __builtin_fmaf(ml.y, g, total);
                for (int p = p0; p < min(all, p0 + 64); p += kJoin) {
                    float2 o[kJoin][E];
#pragma unroll
                    for (int j = 0; j < kJoin; j++)
#pragma unroll
                        for (int e = 0; e < E; e++)
                            o[j][e] = mine ? get2(rec.o + at(min(p + j, all - 1)) * D + 2 * (lane + 64 * e)) : make_float2(0.f, 0.f);
#pragma unroll
                    for (int j = 0; j < kJoin; j++) {
                        const float f = __shfl(g, p - p0 + j);
                        if (p + j >= all) continue;  // (read again above)
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            sum[e].x = __builtin_fmaf(o[j][e].x, f, sum[e].x);
                            sum[e].y = __builtin_fmaf(o[j][e].y, f, sum[e].y);
                        }
                    }
                }
            }
            for (int x = 32; x >= 1; x /= 2) total += __shfl_xor(total, x);
            const float y = any ? 1.0f / total : 0.f;  // (a row without keys in a group: all weights are zero)
            using o2 = TO __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int e = 0; e < E; e++)
                if (mine) *reinterpret_cast<o2*>(out_at(r, head * G + q) + 2 * (lane + 64 * e)) = o2{(TO)(sum[e].x * y), (TO)(sum[e].y * y)};
        }
    }
}

template <int D, typename T, typename TO>
struct Step {
    static hipError_t go(const StepArgs& a, hipStream_t stream) {
        const bool work = a.work != nullptr;
        const Split s = plan_step(a, work);
        Records r{};
        r.parts = s.own_parts + s.pre_parts;
        r.count = static_cast<unsigned*>(a.work);
        r.ml = static_cast<float*>(a.work) + (work ? records_counts(a.rows, a.cache.kv_heads) : 0);
        r.o = r.ml + (int64_t)a.rows * a.q_heads * r.parts * 2;
        const int64_t blocks = (int64_t)s.pre_tiles * s.pre_parts * a.cache.kv_heads + (int64_t)a.rows * a.cache.kv_heads * s.head_tiles * s.own_parts;
        if (blocks > INT32_MAX) return hipErrorInvalidValue;
        static const hipError_t ready = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_step_kernel<D, T, TO>),
                                                            hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes<D>());
        if (ready != hipSuccess) return ready;
        hipLaunchKernelGGL((attn_step_kernel<D, T, TO>), dim3((unsigned)blocks), dim3(kThreads), lds_bytes<D>(), stream, KernelArgs{a, s, r});
        return hipGetLastError();
    }
};

}  // namespace

int64_t attn_step_work_bytes(const StepArgs& a) {
    return work_bytes(a, plan_step(a, true));
}

hipError_t launch_attn_step(const StepArgs& a, int dtype, int out_dtype, hipStream_t stream) {
    return by_type<Step>(a, a.cache.head_dim, dtype, out_dtype, stream);
}

}  // namespace vxs
