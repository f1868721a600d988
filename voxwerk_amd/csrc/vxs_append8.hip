// vxs_append8.hip — new tokens' queries, keys and values on their way to attention over an 8-bit cache.
//
// Heads are normed and rotated as for a 16-bit cache (vxs_append.hip); then, for each block of 16 tokens and key head,
//   A = max |x| over the block's finite entries,   scale = 2^e with the least e for which A <= 448 2^e,
//   entry = e4m3(x / scale)        (to nearest even; e4m3 ends at 448)
// A = 1.f * 2^E, 448 = 1.75 * 2^8: e = E - 8, or E - 7 where f is above .75, so e comes from the bits of A by one addition.
// A block that has tokens already keeps the larger of its scale and the new ones'; where it grows, what is there is divided by the
// quotient, which being a power of two leaves e4m3's bits as they are down to its subnormals: blocks that fill token by token lose
// nothing against those that come whole.
//
// Bound by memory (each input read once, queries and bytes written once), and by latency for the few rows of a step. A wave
// takes a block's rows of one head at once, all of them in registers until the block's maximum is known; consecutive rows of one block
// belong to the wave that finds the first of them. Where every row is alone in its block, as in a step, a wave takes HW heads of one.
// Rows of queries are items of their own.
//
// Measured: 18,000 tokens of 32 + 2 x 8 heads of 128, fp32 in, fp16 queries, 138 us: 627 MB at 4.5 TB/s (a copy: 5.2); 256 tokens of 16 + 2 x 8
// heads 7.3 us, one 5.4: slot and place, page, entries, what the block holds, one after the other.
#include <hip/hip_runtime.h>

#include "vxs_append.h"
#include "vxs_append_plan.h"

namespace vxs {
namespace {

constexpr int kAT = kAppend8Threads;

typedef float f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4 scaled(f4 x, int by) {
    return f4{__builtin_ldexpf(x[0], by), __builtin_ldexpf(x[1], by), __builtin_ldexpf(x[2], by), __builtin_ldexpf(x[3], by)};
}
__device__ __forceinline__ unsigned to_e4m3(f4 x) {  // (infinite and NaN: NaN)
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], low, true);
}
__device__ __forceinline__ f4 from_e4m3(unsigned x) {
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
    return f4{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ float finite_size(f4 x, float most) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float y = __builtin_fabsf(x[e]);
        most = fmaxf(most, y < __builtin_inff() ? y : 0.f);  // (false for NaN too)
    }
    return most;
}

// Row t alone to its place in head h (a wave's heads each have their lanes; those of heads that are not there do nothing).
template <int D, typename TI>
__device__ __forceinline__ void one_row(const AppendArgs& a, const HeadLane<D>& at_head, bool is_k, int h, int t, int place, int page, int lane) {
    if (h >= a.cache.kv_heads) return;
    const int ra = at_head.ra, rb = at_head.rb;
    const TI* const src = (is_k ? static_cast<const TI*>(a.k) + t * a.ldk : static_cast<const TI*>(a.v) + t * a.ldv) + (int64_t)h * D;
    uint8_t* const scale = (is_k ? a.scales.k : a.scales.v) + scale_index(a.cache, page, h, place);
    char* const to = (is_k ? a.cache.k : a.cache.v) + cache_offset(a.cache, page, h, place & ~15);
    f4 x = load4(src + ra), y = load4(src + rb);
    const bool fresh = (place & 15) == 0;
    const int old = fresh ? 1 : *scale;
    if (is_k) {
        f4 c, s;
        at_head.angles(a, t, c, s);
        if (a.prep.k_norm) at_head.norm(x, y, a.prep.k_norm, a.prep.eps);
        at_head.rotate(x, y, c, s);
    }
    float most = finite_size(x, finite_size(y, 0.f));
#pragma unroll
    for (int m = D / 16; m >= 1; m /= 2) most = fmaxf(most, __shfl_xor(most, m));
    const int byte = max(max((int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 8, old), 1);
    if (!fresh && byte > old) {
#pragma unroll 1
        for (int from = 0; from < 16; from += 8) {
            char* const at = to + (uint64_t)from * a.cache.token_stride;
            unsigned was[8][2];
#pragma unroll
            for (int p = 0; p < 8; p++) {
                was[p][0] = *reinterpret_cast<const unsigned*>(at + (uint64_t)p * a.cache.token_stride + ra);
                was[p][1] = *reinterpret_cast<const unsigned*>(at + (uint64_t)p * a.cache.token_stride + rb);
            }
#pragma unroll
            for (int p = 0; p < 8; p++) {
                if (from + p == (place & 15)) continue;
                *reinterpret_cast<unsigned*>(at + (uint64_t)p * a.cache.token_stride + ra) = to_e4m3(scaled(from_e4m3(was[p][0]), old - byte));
                *reinterpret_cast<unsigned*>(at + (uint64_t)p * a.cache.token_stride + rb) = to_e4m3(scaled(from_e4m3(was[p][1]), old - byte));
            }
        }
    }
    char* const row = to + (uint64_t)(place & 15) * a.cache.token_stride;
    *reinterpret_cast<unsigned*>(row + ra) = to_e4m3(scaled(x, 127 - byte));
    *reinterpret_cast<unsigned*>(row + rb) = to_e4m3(scaled(y, 127 - byte));
    if (lane % HeadLane<D>::kLanes == 0 && (fresh || byte != old)) *scale = (uint8_t)byte;
}

template <int D, typename TI, typename TO>
__global__ __launch_bounds__(kAT, D == 256 ? 3 : 4) void kv8_append_kernel(AppendArgs a) {
    constexpr int L = D / 8;      // lanes of a head
    constexpr int HW = 64 / L;    // rows, or heads of a row's queries, of a wave at a time
    constexpr int NI = 16 / HW;   // times that for a block
    const int lane = threadIdx.x & 63, wave = blockIdx.y * (kAT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = gridDim.y * (kAT / 64);
    const int t0 = blockIdx.x * kChunk, rows = min(kChunk, a.tokens - t0);
    const HeadLane<D> at_head(a.prep, lane);
    const int ra = at_head.ra, rb = at_head.rb;
    const int qh = a.q ? a.q_heads : 0, kh = a.k ? a.cache.kv_heads : 0;

    // ---- the blocks that begin here: lane i has row t0 - 1 + i, so that of `mine` begins at lane i where its slot and block are not
    // those of the lane before
    const int t = t0 - 1 + lane;
    int slot = -1, place = -1, page = -1;
    uint64_t first = 0;
    if (kh) {
        if (t >= 0 && t < a.tokens) {
            slot = a.slots ? a.slots[t] : t;
            place = a.index[t];
            page = place_page(a.cache, slot, place);
        }
        const bool mine = lane >= 1 && lane <= rows;
        const int before_slot = __shfl_up(slot, 1), before_place = __shfl_up(place, 1);
        first = __ballot(mine && page >= 0 && (t == 0 || before_slot != slot || (before_place >> 4) != (place >> 4)));
        if (a.status && wave == 0 && mine) a.status[t] = page >= 0 ? 0 : VXS_ERR_ID_OUT_OF_RANGE;
    } else if (a.status && wave == 0 && lane >= 1 && lane <= rows) {
        a.status[t] = 0;
    }
    // Where each of them has a single row in this call (a step's), a wave takes HW heads at a time, a head's lanes each.
    const int next_slot = __shfl_down(slot, 1), next_place = __shfl_down(place, 1);
    const bool single = (__ballot(next_slot == slot && (next_place >> 4) == (place >> 4)) & first) == 0;
    const int kv_sets = single ? (kh + HW - 1) / HW : kh;
    const int kv_items = __builtin_popcountll(first) * 2 * kv_sets, q_sets = (qh + kSets * HW - 1) / (kSets * HW), items = kv_items + rows * q_sets;

    for (int item = wave; item < items; item += waves) {
        if (item >= kv_items) {  // ---- queries of one row
            const int i = (item - kv_items) / q_sets, q = t0 + i, h0 = (item - kv_items - i * q_sets) * kSets * HW + lane / L;
            f4 x[kSets], y[kSets], c, s;
#pragma unroll
            for (int g = 0; g < kSets; g++) {
                if (h0 + g * HW >= qh) continue;  // (a whole head's lanes)
                const TI* src = static_cast<const TI*>(a.q) + q * a.ldq + (int64_t)(h0 + g * HW) * D;
                x[g] = load4(src + ra);
                y[g] = load4(src + rb);
            }
            at_head.angles(a, q, c, s);
#pragma unroll
            for (int g = 0; g < kSets; g++) {
                if (h0 + g * HW >= qh) continue;
                if (a.prep.q_norm) at_head.norm(x[g], y[g], a.prep.q_norm, a.prep.eps);
                at_head.rotate(x[g], y[g], c, s);
                TO* dst = static_cast<TO*>(a.q_out) + q * a.ldqo + (int64_t)(h0 + g * HW) * D;
                store4(dst + ra, x[g]);
                store4(dst + rb, y[g]);
            }
            continue;
        }
        // ---- a block of one head: `row` in lane p < 16 is the last of its rows whose place is p, or -1
        const int which = item / (2 * kv_sets), rest = item - which * 2 * kv_sets;
        const bool is_k = rest < kv_sets;
        const int h = is_k ? rest : rest - kv_sets;
        uint64_t left = first;
        for (int i = 0; i < which; i++) left &= left - 1;
        const int at = __builtin_ctzll(left);
        if (single) {
            one_row<D, TI>(a, at_head, is_k, h * HW + lane / L, t0 - 1 + at, __builtin_amdgcn_readlane(place, at), __builtin_amdgcn_readlane(page, at), lane);
            continue;
        }
        const int its_slot = __builtin_amdgcn_readlane(slot, at), block = __builtin_amdgcn_readlane(place, at) >> 4;
        const int its_page = __builtin_amdgcn_readlane(page, at);
        uint8_t* const scale = (is_k ? a.scales.k : a.scales.v) + scale_index(a.cache, its_page, h, block << 4);
        int old = *scale;
        int row = -1;
        // rows from the block's first on, `there` of which are known here: those of lanes `at` to 63, then 64 more as long as they go on
        auto collect = [&](int from, int start, int its, int where) {
            const uint64_t other = ~__ballot(lane < start || (its == its_slot && (where >> 4) == block));
            const int n = other ? __builtin_ctzll(other) : 64;
#pragma unroll
            for (int p = 0; p < 16; p++) {
                const uint64_t mask = __ballot(lane >= start && lane < n && (where & 15) == p);
                if (mask && lane == p) row = from + 63 - __builtin_clzll(mask);
            }
            return n == 64;
        };
        bool more = collect(t0 - 1, at, slot, place);
        for (int from = t0 + 63; more; from += 64) {
            int its = -1, where = -1;
            if (from + lane < a.tokens) {
                its = a.slots ? a.slots[from + lane] : from + lane;
                where = a.index[from + lane];
            }
            more = collect(from, 0, its, where);
        }
        const bool fresh = __ballot(row >= 0) & 1;
        if (fresh) old = 1;
        const TI* const in = (is_k ? static_cast<const TI*>(a.k) : static_cast<const TI*>(a.v)) + (int64_t)h * D;
        const int64_t ld = is_k ? a.ldk : a.ldv;
        int r[NI];
        f4 x[NI], y[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            r[i] = __shfl(row, i * HW + lane / L);
            x[i] = y[i] = f4{0.f, 0.f, 0.f, 0.f};
            if (r[i] >= 0) {
                x[i] = load4(in + r[i] * ld + ra);
                y[i] = load4(in + r[i] * ld + rb);
            }
        }
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            if (is_k && r[i] >= 0) {
                f4 c, s;
                at_head.angles(a, r[i], c, s);
                if (a.prep.k_norm) at_head.norm(x[i], y[i], a.prep.k_norm, a.prep.eps);
                at_head.rotate(x[i], y[i], c, s);
            }
            most = finite_size(x[i], finite_size(y[i], most));
        }
#pragma unroll
        for (int m = 32; m >= 1; m /= 2) most = fmaxf(most, __shfl_xor(most, m));
        const int own = (int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 8;
        const int byte = __builtin_amdgcn_readfirstlane(max(max(own, old), 1));
        char* const to = (is_k ? a.cache.k : a.cache.v) + cache_offset(a.cache, its_page, h, block << 4);
        const bool grown = !fresh && byte > old;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            char* const at_row = to + (uint64_t)(i * HW + lane / L) * a.cache.token_stride;
            unsigned* const pa = reinterpret_cast<unsigned*>(at_row + ra);
            unsigned* const pb = reinterpret_cast<unsigned*>(at_row + rb);
            if (r[i] >= 0) {
                *pa = to_e4m3(scaled(x[i], 127 - byte));
                *pb = to_e4m3(scaled(y[i], 127 - byte));
            } else if (grown) {
                *pa = to_e4m3(scaled(from_e4m3(*pa), old - byte));
                *pb = to_e4m3(scaled(from_e4m3(*pb), old - byte));
            }
        }
        if (lane == 0 && (fresh || byte != old)) *scale = (uint8_t)byte;
    }
}

template <int D, typename TI, typename TO>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
    const Append8Grid g = plan_append8(a.tokens, a.q ? a.q_heads : 0, a.k ? a.cache.kv_heads : 0, D);
    hipLaunchKernelGGL((kv8_append_kernel<D, TI, TO>), dim3(g.chunks, g.parts), dim3(kAT), 0, stream, a);
    return hipGetLastError();
}

template <int D, typename TO>
hipError_t launch_in(const AppendArgs& a, int in_dtype, hipStream_t stream) {
    if (in_dtype == VXS_F32) return launch<D, float, TO>(a, stream);
    if (in_dtype == VXS_BF16) return launch<D, __bf16, TO>(a, stream);
    return launch<D, _Float16, TO>(a, stream);
}

template <int D>
hipError_t launch_out(const AppendArgs& a, int in_dtype, int q_dtype, hipStream_t stream) {
    return q_dtype == VXS_BF16 ? launch_in<D, __bf16>(a, in_dtype, stream) : launch_in<D, _Float16>(a, in_dtype, stream);
}

}  // namespace

hipError_t launch_kv8_append(const AppendArgs& a, int in_dtype, int q_dtype, hipStream_t stream) {
    switch (a.cache.head_dim) {
        case 64: return launch_out<64>(a, in_dtype, q_dtype, stream);
        case 128: return launch_out<128>(a, in_dtype, q_dtype, stream);
        default: return launch_out<256>(a, in_dtype, q_dtype, stream);
    }
}

}  // namespace vxs
