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
// belong to the wave that finds the first of them. Rows of queries are items of their own.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_append.h"

namespace vxs {
namespace {

constexpr int kAT = 256;

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

// A workgroup's waves, and those of the others at its blockIdx.x, share the items of `chunk` rows: each block of 16 tokens that
// begins among them (its rows may go on in the next chunk), for keys and for values, `per` heads at a time; and each row's queries.
template <int D, typename TI, typename TO>
__global__ __launch_bounds__(kAT) void kv8_append_kernel(AppendArgs a, int chunk, int per) {
    constexpr int L = D / 8;      // lanes of a head
    constexpr int HW = 64 / L;    // rows, or heads of a row's queries, of a wave at a time
    constexpr int NI = 16 / HW;   // times that for a block
    const int lane = threadIdx.x & 63, wave = blockIdx.y * (kAT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = gridDim.y * (kAT / 64);
    const int t0 = blockIdx.x * chunk, rows = min(chunk, a.tokens - t0);
    const HeadLane<D> at_head(a.prep, lane);
    const int ra = at_head.ra, rb = at_head.rb;
    const int qh = a.q ? a.q_heads : 0, kh = a.k ? a.cache.kv_heads : 0;

    // ---- the blocks that begin here: lane i < rows has row t0 + i
    int slot = 0, place = 0;
    uint64_t first = 0;
    if (kh) {
        bool valid = false, begins = false;
        if (lane < rows) {
            const int t = t0 + lane;
            slot = a.slots ? a.slots[t] : t;
            place = a.index[t];
            valid = place_page(a.cache, slot, place) >= 0;
            begins = valid && (t == 0 || (a.slots ? a.slots[t - 1] : t - 1) != slot || (a.index[t - 1] >> 4) != (place >> 4));
            if (a.status && wave == 0) a.status[t] = valid ? 0 : VXS_ERR_ID_OUT_OF_RANGE;
        }
        first = __ballot(begins);
    } else if (a.status && wave == 0 && lane < rows) {
        a.status[t0 + lane] = 0;
    }
    const int blocks = __builtin_popcountll(first), head_sets = kh ? (kh + per - 1) / per : 0;
    const int kv_items = blocks * 2 * head_sets, q_sets = (qh + HW - 1) / HW, q_per = chunk > 1 ? q_sets : 1;
    const int q_items = q_sets ? rows * (q_sets / q_per) : 0;

    for (int item = wave; item < kv_items + q_items; item += waves) {
        if (item >= kv_items) {  // ---- queries of one row
            const int i = item - kv_items, t = t0 + i % rows;
            f4 c, s;
            at_head.angles(a, t, c, s);
            for (int g = i / rows * q_per; g < (i / rows + 1) * q_per; g++) {
                const int h = g * HW + lane / L;
                if (h >= qh) continue;  // (a whole head's lanes)
                const TI* src = static_cast<const TI*>(a.q) + t * a.ldq + (int64_t)h * D;
                f4 x = load4(src + ra), y = load4(src + rb);
                if (a.prep.q_norm) at_head.norm(x, y, a.prep.q_norm, a.prep.eps);
                at_head.rotate(x, y, c, s);
                TO* dst = static_cast<TO*>(a.q_out) + t * a.ldqo + (int64_t)h * D;
                store4(dst + ra, x);
                store4(dst + rb, y);
            }
            continue;
        }
        // ---- a block: `row` in lane p < 16 is the last of its rows whose place is p, or -1
        const int which = item / (2 * head_sets), rest = item - which * 2 * head_sets;
        const bool is_k = rest < head_sets;
        const int h0 = (is_k ? rest : rest - head_sets) * per;
        uint64_t left = first;
        for (int i = 0; i < which; i++) left &= left - 1;
        const int at = __builtin_ctzll(left);
        const int my_slot = __builtin_amdgcn_readlane(slot, at), block = __builtin_amdgcn_readlane(place, at) >> 4;
        int row = -1;
        for (int from = t0 + at;; from += 64) {
            const int t = from + lane;
            int its = -1, where = 0;
            if (t < a.tokens) {
                its = a.slots ? a.slots[t] : t;
                where = a.index[t];
            }
            const bool same = t < a.tokens && its == my_slot && (where >> 4) == block;
            const uint64_t other = ~__ballot(same);
            const int n = other ? __builtin_ctzll(other) : 64;
#pragma unroll
            for (int p = 0; p < 16; p++) {
                const uint64_t mask = __ballot(lane < n && (where & 15) == p);
                if (mask && lane == p) row = from + 63 - __builtin_clzll(mask);
            }
            if (n < 64) break;
        }
        const uint64_t there = __ballot(row >= 0);
        const bool fresh = there & 1;
        const int page = place_page(a.cache, my_slot, block << 4);
        int r[NI];
        f4 c[NI], s[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            r[i] = __shfl(row, i * HW + lane / L);
            if (is_k && r[i] >= 0) at_head.angles(a, r[i], c[i], s[i]);
        }
        const TI* const in = static_cast<const TI*>(is_k ? a.k : a.v);
        const int64_t ld = is_k ? a.ldk : a.ldv;
        for (int h = h0; h < min(h0 + per, kh); h++) {
            f4 x[NI], y[NI];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                x[i] = y[i] = f4{0.f, 0.f, 0.f, 0.f};
                if (r[i] >= 0) {
                    const TI* src = in + r[i] * ld + (int64_t)h * D;
                    x[i] = load4(src + ra);
                    y[i] = load4(src + rb);
                }
            }
            uint8_t* const scale = (is_k ? a.scales.k : a.scales.v) + scale_index(a.cache, page, h, block << 4);
            const int old = fresh ? 1 : *scale;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                if (is_k && r[i] >= 0) {
                    if (a.prep.k_norm) at_head.norm(x[i], y[i], a.prep.k_norm, a.prep.eps);
                    at_head.rotate(x[i], y[i], c[i], s[i]);
                }
                most = finite_size(x[i], finite_size(y[i], most));
            }
#pragma unroll
            for (int m = 32; m >= 1; m /= 2) most = fmaxf(most, __shfl_xor(most, m));
            const int own = (int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 8;
            const int byte = __builtin_amdgcn_readfirstlane(max(max(own, old), 1));
            char* const to = (is_k ? a.cache.k : a.cache.v) + cache_offset(a.cache, page, h, block << 4);
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
}

template <int D, typename TI, typename TO>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
    const int chunk = a.tokens >= 1024 ? 16 : 1, per = 1;
    const int kh = a.k ? a.cache.kv_heads : 0, qh = a.q ? a.q_heads : 0;
    const int64_t chunks = (a.tokens + chunk - 1) / chunk;
    const int64_t items = (kh ? 2 * ((kh + per - 1) / per) : 0) + (chunk > 1 ? chunk : (qh + 512 / D - 1) / (512 / D));
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({(items + 3) / 4, (1024 + chunks - 1) / chunks, 65535}));
    hipLaunchKernelGGL((kv8_append_kernel<D, TI, TO>), dim3((unsigned)chunks, (unsigned)parts), dim3(kAT), 0, stream, a, chunk, per);
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
