// vxs_append.hip — new tokens' queries, keys and values on their way to attention.
//
// Per head x of head_dim = D entries (a query's or a key's):
//   y = x / sqrt(mean(x^2) + eps) * w                    (RMS norm, when a weight is given)
//   y_a' = y_a cos - y_b sin,  y_b' = y_a sin + y_b cos  (rotation by position * inv_freq[i], i-th pair (a, b))
// in fp32, rounded once to the cache's type; values only change their type. Queries go to q_out, keys and
// values to their places in the pages: one pass over the projections' outputs, bound by memory, and by the launch
// for the few rows of a generation step.
//
// Layout: D/8 lanes hold a head, each two runs of four entries, so that both entries of every pair are in one lane:
// for pairs (i, i + rot/2) runs 4u and 4u + rot/2, past the rotated part 4u' and 4u' + (D - rot)/2 of the rest; for
// interleaved pairs two neighbouring runs. A wave takes one token and 512/D heads at a time, so the four angles of a
// lane are formed once per token. An angle is position * inv_freq / 2pi in fp64, whose fraction (exact to 2^-20 of a
// turn at any int32 position) goes to the fp32 sine and cosine, which take turns.
//
// Measured: 18,000 tokens of 32 + 2 x 8 heads of 128, fp32 to fp16, 122 us: 664 MB at 5.4 TB/s, what a copy reaches; one token of
// 16 + 2 x 8 heads 3.2 us, 256 of them 4.2 (a launch alone is 2.6).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_attn.h"

namespace vxs {
namespace {

constexpr int kAT = 256;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Four;
template <>
struct Four<float> { using type = f4; };
template <>
struct Four<__bf16> { using type = bf4; };
template <>
struct Four<_Float16> { using type = h4; };

template <typename T>
__device__ __forceinline__ f4 load4(const T* p) {
    const typename Four<T>::type x = *reinterpret_cast<const typename Four<T>::type*>(p);
    return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
template <typename T>
__device__ __forceinline__ void store4(T* p, f4 v) {  // conversions round to nearest even
    *reinterpret_cast<typename Four<T>::type*>(p) = typename Four<T>::type{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
}

template <int D, typename TI, typename TO>
__global__ __launch_bounds__(kAT) void kv_append_kernel(AppendArgs a) {
    constexpr int L = D / 8;    // lanes of a head
    constexpr int HW = 64 / L;  // heads of a wave at a time
    const int t = blockIdx.x;
    const int lane = threadIdx.x & 63, u = lane % L;
    const int rot = a.prep.rot_dim;
    const bool inter = a.prep.interleaved;
    const int qh = a.q ? a.q_heads : 0, kh = a.k ? a.cache.kv_heads : 0;
    const int heads = qh + 2 * kh;
    // this lane's two runs
    const bool turned = 8 * u < rot;
    const int ra = inter ? 8 * u : turned ? 4 * u : rot + (4 * u - rot / 2);
    const int rb = inter ? 8 * u + 4 : ra + (turned ? rot / 2 : (D - rot) / 2);
    f4 c{1.f, 1.f, 1.f, 1.f}, s{0.f, 0.f, 0.f, 0.f};
    if (turned) {
        const f4 w = *reinterpret_cast<const f4*>(a.prep.inv_freq + 4 * u);
        const double p = (double)a.pos[t];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double turns = p * ((double)w[e] * 0.15915494309189533577);
            const float part = (float)(turns - __builtin_floor(turns));
            c[e] = __builtin_amdgcn_cosf(part) * a.prep.rope_scale;
            s[e] = __builtin_amdgcn_sinf(part) * a.prep.rope_scale;
        }
    }
    // where the token's key and value go
    int64_t at = -1;
    if (kh) {
        const int slot = a.slots ? a.slots[t] : t, place = a.index[t];
        if ((unsigned)slot < (unsigned)a.cache.slots && place >= 0 && (place >> a.cache.page_bits) < a.cache.ld_table) {
            const int page = a.cache.table[(int64_t)slot * a.cache.ld_table + (place >> a.cache.page_bits)];
            if ((unsigned)page < (unsigned)a.cache.pages)
                at = (int64_t)cache_offset(a.cache, page, 0, place);
        }
    }
    if (a.status && threadIdx.x == 0 && blockIdx.y == 0) a.status[t] = kh && at < 0 ? VXS_ERR_ID_OUT_OF_RANGE : 0;
    const int step = gridDim.y * (kAT / 64) * HW;
    for (int h0 = (blockIdx.y * (kAT / 64) + (threadIdx.x >> 6)) * HW; h0 < heads; h0 += step) {
        const int h = h0 + lane / L;
        if (h >= heads) continue;  // (a whole head's lanes)
        const bool is_q = h < qh, is_k = !is_q && h < qh + kh;
        const int j = is_q ? h : is_k ? h - qh : h - qh - kh;
        const TI* src = is_q   ? static_cast<const TI*>(a.q) + t * a.ldq
                        : is_k ? static_cast<const TI*>(a.k) + t * a.ldk
                               : static_cast<const TI*>(a.v) + t * a.ldv;
        src += (int64_t)j * D;
        f4 x = load4(src + ra), y = load4(src + rb);
        const float* weight = is_q ? a.prep.q_norm : is_k ? a.prep.k_norm : nullptr;
        if (weight) {
            const f4 wa = *reinterpret_cast<const f4*>(weight + ra), wb = *reinterpret_cast<const f4*>(weight + rb);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) sum = __builtin_fmaf(x[e], x[e], __builtin_fmaf(y[e], y[e], sum));
#pragma unroll
            for (int m = L / 2; m >= 1; m /= 2) sum += __shfl_xor(sum, m);
            const float r = 1.0f / __builtin_sqrtf(sum * (1.0f / D) + a.prep.eps);
            x = x * r * wa;
            y = y * r * wb;
        }
        if (turned && !(h >= qh + kh)) {
            if (inter) {
                const f4 xx{x[0] * c[0] - x[1] * s[0], x[0] * s[0] + x[1] * c[0], x[2] * c[1] - x[3] * s[1], x[2] * s[1] + x[3] * c[1]};
                const f4 yy{y[0] * c[2] - y[1] * s[2], y[0] * s[2] + y[1] * c[2], y[2] * c[3] - y[3] * s[3], y[2] * s[3] + y[3] * c[3]};
                x = xx;
                y = yy;
            } else {
                const f4 xx = x * c - y * s;
                y = x * s + y * c;
                x = xx;
            }
        }
        TO* dst;
        if (is_q) {
            dst = static_cast<TO*>(a.q_out) + t * a.ldqo + (int64_t)j * D;
        } else {
            if (at < 0) continue;
            dst = reinterpret_cast<TO*>((is_k ? a.cache.k : a.cache.v) + at + (int64_t)j * a.cache.head_stride);
        }
        store4(dst + ra, x);
        store4(dst + rb, y);
    }
}

template <int D, typename TI, typename TO>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
    constexpr int per_group = 4 * (512 / D);  // heads of a workgroup at a time
    const int heads = (a.q ? a.q_heads : 0) + (a.k ? 2 * a.cache.kv_heads : 0);
    // A token's heads go to several workgroups until there are 1024 of them.
    const int most = (heads + per_group - 1) / per_group;
    const int parts = std::max(1, std::min({most, (1024 + a.tokens - 1) / a.tokens, 65535}));
    hipLaunchKernelGGL((kv_append_kernel<D, TI, TO>), dim3(a.tokens, parts), dim3(kAT), 0, stream, a);
    return hipGetLastError();
}

template <int D, typename TO>
hipError_t launch_in(const AppendArgs& a, int in_dtype, hipStream_t stream) {
    if (in_dtype == VXS_F32) return launch<D, float, TO>(a, stream);
    if (in_dtype == VXS_BF16) return launch<D, __bf16, TO>(a, stream);
    return launch<D, _Float16, TO>(a, stream);
}

template <int D>
hipError_t launch_out(const AppendArgs& a, int in_dtype, int dtype, hipStream_t stream) {
    return dtype == VXS_BF16 ? launch_in<D, __bf16>(a, in_dtype, stream) : launch_in<D, _Float16>(a, in_dtype, stream);
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs& a, int in_dtype, int dtype, hipStream_t stream) {
    switch (a.cache.head_dim) {
        case 64: return launch_out<64>(a, in_dtype, dtype, stream);
        case 128: return launch_out<128>(a, in_dtype, dtype, stream);
        default: return launch_out<256>(a, in_dtype, dtype, stream);
    }
}

}  // namespace vxs
