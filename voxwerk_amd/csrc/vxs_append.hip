// vxs_append.hip — new tokens' queries, keys and values on their way to attention.
//
// Per head x of head_dim = D entries (a query's or a key's):
//   y = x / sqrt(mean(x^2) + eps) * w                    (RMS norm, when a weight is given)
//   y_a' = y_a cos - y_b sin,  y_b' = y_a sin + y_b cos  (rotation by position * inv_freq[i], i-th pair (a, b))
// in fp32, rounded once to the cache's type; values only change their type. Queries go to q_out, keys and
// values to their places in the pages: one pass over the projections' outputs, bound by memory, and by the launch
// for the few rows of a generation step.
//
// Layout: vxs_append.h. A wave takes one token and 512/D heads at a time, so the four angles of a lane are formed once per token and wave.
//
// Measured: 18,000 tokens of 32 + 2 x 8 heads of 128, fp32 to fp16, 122 us: 664 MB at 5.4 TB/s, what a copy reaches; one token of
// 16 + 2 x 8 heads 3.2 us, 256 of them 4.2 (a launch alone is 2.6); 12,000 tokens of 16 + 2 x 8 bf16 heads with positions of three axes 45.4 us, 4.4 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_append.h"

namespace vxs {
namespace {

constexpr int kAT = 256;


template <int D, typename TI, typename TO>
__global__ __launch_bounds__(kAT) void kv_append_kernel(AppendArgs a, int waves) {
    constexpr int L = D / 8;    // lanes of a head
    constexpr int HW = 64 / L;  // heads of a wave at a time
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * (kAT / 64 / waves) + wave / waves, first = blockIdx.y * waves + wave % waves;  // `waves` waves of a workgroup take a token
    if (t >= a.tokens) return;
    const HeadLane<D> at_head(a.prep, lane);
    const int ra = at_head.ra, rb = at_head.rb;
    const int qh = a.q ? a.q_heads : 0, kh = a.k ? a.cache.kv_heads : 0;
    const int heads = qh + 2 * kh;
    f4 c, s;
    at_head.angles(a, t, c, s);
    // where the token's key and value go
    int64_t at = -1;
    if (kh) {
        const int place = a.index[t], page = place_page(a.cache, a.slots ? a.slots[t] : t, place);
        if (page >= 0) at = (int64_t)cache_offset(a.cache, page, 0, place);
    }
    if (a.status && lane == 0 && first == 0) a.status[t] = kh && at < 0 ? VXS_ERR_ID_OUT_OF_RANGE : 0;
    const int step = gridDim.y * waves * HW;
    for (int h0 = first * HW; h0 < heads; h0 += step) {
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
        if (weight) at_head.norm(x, y, weight, a.prep.eps);
        if (h < qh + kh) at_head.rotate(x, y, c, s);
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
    // Every wave forms the token's angles: two waves a token where its rows are short and tokens many (us, two / four: 12,000 tokens of 16 + 2 x 8 bf16
    // heads of 128, three axes, 45.4 / 50.4, of 64 21.5 / 25.3, of 256 82 / 85, 2000 8.9 / 8.8; 18,000 of 32 + 2 x 8 fp32 ones 126.7 / 123.2; one: 45.4, 19.4, 87).
    const int waves = sizeof(TI) == 2 && a.tokens >= 2048 ? 2 : kAT / 64, tokens = kAT / 64 / waves;
    hipLaunchKernelGGL((kv_append_kernel<D, TI, TO>), dim3((a.tokens + tokens - 1) / tokens, parts), dim3(kAT), 0, stream, a, waves);
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
