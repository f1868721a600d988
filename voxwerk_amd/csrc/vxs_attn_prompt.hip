// vxs_attn.hip — attention of packed prompts over a paged cache.
//
//   out[r] = sum_s w_s v[s] / sum_s w_s,   w_s = exp(scale q[r] . k[s] - m)   over the keys s that row r sees,
// with the running maximum m and both sums carried along the keys (when m grows by d, the sums shrink by exp(-d)).
// Here one wave per query row and head goes over its keys one after the other, each lane holding D/64 entries.
#include <hip/hip_runtime.h>

#include "vxs_attn.h"
#include "vxs_attn_types.h"

namespace vxs {
namespace {

template <int D, typename T, typename TO>
__device__ __forceinline__ void attend_row(const PagedCache& c, const T* q, int slot, int h, int64_t n, float scale, TO* out) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    float x[E], acc[E];
    for (int e = 0; e < E; e++) {
        x[e] = (float)q[lane * E + e] * scale;
        acc[e] = 0.f;
    }
    float m = -3.0e38f, l = 0.f;
    const int32_t* pages = c.table + (int64_t)slot * c.ld_table;
    for (int t = 0; t < n; t++) {
        const uint64_t at = cache_offset(c, pages[t >> c.page_bits], h, t);
        const T* k = reinterpret_cast<const T*>(c.k + at) + lane * E;
        const T* v = reinterpret_cast<const T*>(c.v + at) + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; e++) s = __builtin_fmaf(x[e], (float)k[e], s);
        for (int b = 32; b >= 1; b /= 2) s += __shfl_xor(s, b);
        const float top = fmaxf(m, s), old = __expf(m - top), w = __expf(s - top);
        m = top;
        l = l * old + w;
        for (int e = 0; e < E; e++) acc[e] = __builtin_fmaf(w, (float)v[e], acc[e] * old);
    }
    for (int e = 0; e < E; e++) out[lane * E + e] = (TO)(n > 0 ? acc[e] / l : 0.f);
}

template <int D, typename T, typename TO>
__global__ __launch_bounds__(64) void prompt_kernel(PromptArgs a) {
    const int t = blockIdx.x, head = blockIdx.y;
    int lo = 0, hi = a.seqs;  // the last sequence that begins at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_off[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int b = a.q_off[lo], e = a.q_off[lo + 1];
    if (t < b || t >= e) return;
    const int slot = a.slots ? a.slots[lo] : lo;
    const int64_t len = cache_length(a.cache, slot, a.kv_len[lo]);
    const int64_t n = len - (e - b) + (t - b) + 1;
    attend_row<D>(a.cache, static_cast<const T*>(a.q) + t * a.ldq + (int64_t)head * D, n > 0 ? slot : 0,
                  head / (a.q_heads / a.cache.kv_heads), n, a.scale, static_cast<TO*>(a.out) + t * a.ldo + (int64_t)head * D);
}

template <int D, typename T, typename TO>
struct Prompt {
    static hipError_t go(const PromptArgs& a, hipStream_t stream) {
        hipLaunchKernelGGL((prompt_kernel<D, T, TO>), dim3(a.tokens, a.q_heads), dim3(64), 0, stream, a);
        return hipGetLastError();
    }
};
}  // namespace

hipError_t launch_attn_prompt(const PromptArgs& a, int dtype, int out_dtype, hipStream_t stream) {
    return by_type<Prompt>(a, a.cache.head_dim, dtype, out_dtype, stream);
}

}  // namespace vxs
