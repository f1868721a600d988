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
// Kernels for one position a token take no axes among their arguments and waves a token as a constant: with both at run time one token took
// 3.33 us, not 2.96, 256 of them 4.5, not 4.15.
//
// Measured: 18,000 tokens of 32 + 2 x 8 heads of 128, fp32 to fp16, 122 us: 664 MB at 5.4 TB/s, what a copy reaches; one token of
// 16 + 2 x 8 heads 3.0 us, 256 of them 4.2 (a launch alone is 2.6); 12,000 tokens of 16 + 2 x 8 bf16 heads with positions of three axes 45.4 us, 4.4 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vxs_append.h"

namespace vxs {
namespace {

constexpr int kAT = 256;

// WAVES waves of a workgroup take a token. Args: AppendOneArgs or AppendAxesArgs.
template <int D, typename TI, typename TO, int WAVES, typename Args>
__global__ __launch_bounds__(kAT) void kv_append_kernel(Args a) {
    constexpr int L = D / 8;    // lanes of a head
    constexpr int HW = 64 / L;  // heads of a wave at a time
    constexpr int kTokens = kAT / 64 / WAVES;
    const int lane = threadIdx.x & 63, wave = kTokens == 1 ? threadIdx.x >> 6 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = kTokens == 1 ? blockIdx.x : blockIdx.x * kTokens + wave / WAVES, first = blockIdx.y * WAVES + wave % WAVES;
    if (kTokens > 1 && t >= a.tokens) return;
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
    const int step = gridDim.y * WAVES * HW;
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

template <int D, typename TI, typename TO, int WAVES>
void launch(const AppendArgs& a, int parts, hipStream_t stream) {
    constexpr int kTokens = kAT / 64 / WAVES;
    const dim3 grid((a.tokens + kTokens - 1) / kTokens, parts);
    if (a.axes.axes) hipLaunchKernelGGL((kv_append_kernel<D, TI, TO, WAVES, AppendAxesArgs>), grid, dim3(kAT), 0, stream, a);
    else hipLaunchKernelGGL((kv_append_kernel<D, TI, TO, WAVES, AppendOneArgs>), grid, dim3(kAT), 0, stream, a);
}

template <int D, typename TI, typename TO>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
    constexpr int per_group = 4 * (512 / D);  // heads of a workgroup at a time
    const int heads = (a.q ? a.q_heads : 0) + (a.k ? 2 * a.cache.kv_heads : 0);
    // A token's heads go to several workgroups until there are 1024 of them.
    const int most = (heads + per_group - 1) / per_group;
    const int parts = std::max(1, std::min({most, (1024 + a.tokens - 1) / a.tokens, 65535}));
    // Every wave forms its token's angles: two waves a token, not four, where few groups of heads fill them and tokens fill the compute units
    // (us, two / four, bf16 inputs; 6000 tokens of 16 + 2 x 8 heads of 64, 4 groups, 11.6 / 12.8; of 128, 8 groups, 2048 of them 9.6 / 9.1, 3000
    // 11.2 / 11.4, 12,000 35.2 / 37.9; 64 + 2 x 8 of 64, 10 groups, 9000 of them 40.3 / 38.5; 64 + 2 x 8 of 128, 20 groups, 6000 48.5 / 44.1;
    // three axes: 12,000 of 16 + 2 x 8 of 128 39.2 / 46.6; 32 + 2 x 8, 12 groups, 2048 13.0 / 13.0, 6000 25.8 / 26.8; 20 groups 6000 49.5 / 46.6,
    // 24 groups 12,000 112.7 / 114.3, 24,000 219 / 221).
    const int groups = (heads + 512 / D - 1) / (512 / D);
    const bool few = a.axes.axes ? groups <= (a.tokens < 12000 ? 12 : 24) : groups <= 8 && a.tokens >= 400 * groups;
    if (sizeof(TI) == 2 && a.tokens >= 2048 && few) launch<D, TI, TO, 2>(a, parts, stream);
    else launch<D, TI, TO, 4>(a, parts, stream);
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
