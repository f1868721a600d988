// vxs_attn_api.cpp — the C ABI of the paged cache's operators: argument checks and error mapping.
// No C++ exception crosses the boundary.
#include <hip/hip_runtime.h>

#include <cmath>

#include "vxs_attn.h"
#include "vxs_internal.h"

namespace {

using vxs::ctx_fail;

#define VXS_ATTN_HIP(ctx, call)                                            \
    do {                                                                   \
        hipError_t e_ = (call);                                            \
        if (e_ != hipSuccess) return vxs::ctx_hip_fail((ctx), e_, #call);  \
    } while (0)

int bytes_of(int dtype) { return dtype == VXS_F32 ? 4 : 2; }

// Cache is vxs_kv_cache or vxs_kv8_cache: the same but for the entries' bytes, the unit that strides are multiples of, and the scales.
constexpr int entry_bytes(const vxs_kv_cache*) { return 2; }
constexpr int entry_bytes(const vxs_kv8_cache*) { return 1; }
int query_type(const vxs_kv_cache* c) { return c->dtype; }
int query_type(const vxs_kv8_cache* c) { return c->q_dtype; }
int check_scales(vxs_ctx*, const vxs_kv_cache*, vxs::CacheScales&) { return VXS_OK; }
int check_scales(vxs_ctx* ctx, const vxs_kv8_cache* c, vxs::CacheScales& out) {
    if (!c->k_scale || !c->v_scale) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "cache k_scale or v_scale is NULL");
    if (((uintptr_t)c->k_scale & 3u) || ((uintptr_t)c->v_scale & 3u))
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "cache needs 4-byte aligned k_scale and v_scale");
    out = {c->k_scale, c->v_scale};
    return VXS_OK;
}

template <typename Cache>
int check_cache(vxs_ctx* ctx, const Cache* c, int q_heads, vxs::PagedCache& out, vxs::CacheScales& scales) {
    constexpr int bytes = entry_bytes(static_cast<const Cache*>(nullptr)), unit = 16 / bytes;
    if (!c) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "cache is NULL");
    if (c->slots <= 0 || c->pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0 || c->ld_table <= 0)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "cache sizes must be positive");
    if (query_type(c) != VXS_BF16 && query_type(c) != VXS_F16)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, bytes == 2 ? "cache dtype must be VXS_BF16 or VXS_F16" : "cache q_dtype must be VXS_BF16 or VXS_F16");
    if (!c->k || !c->v || !c->table) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "cache k, v or table is NULL");
    if (q_heads <= 0 || q_heads % c->kv_heads != 0)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "q_heads must be a positive multiple of kv_heads");
    if (c->token_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "cache strides below head_dim");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
    if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "page_size must be a power of two from 16 to 65536");
    if (c->token_stride % unit || c->head_stride % unit || c->page_stride % unit || ((uintptr_t)c->k & 15u) || ((uintptr_t)c->v & 15u))
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED,
                        bytes == 2 ? "cache needs strides that are multiples of 8 and 16-byte aligned k and v"
                                   : "an 8-bit cache needs strides that are multiples of 16 and 16-byte aligned k and v");
    // Token numbers are 32-bit in the kernels (tiles may run up to 256 past the end).
    if (c->ld_table > (INT32_MAX - 256) / c->page_size)
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "ld_table * page_size must stay below 2^31 - 256");
    if (c->token_stride > INT32_MAX / 64 || c->page_stride > INT32_MAX || c->head_stride > INT64_MAX / 65536)
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "token_stride must stay below 2^25, page_stride below 2^31");
    out.k = static_cast<char*>(c->k);
    out.v = static_cast<char*>(c->v);
    out.table = c->table;
    out.ld_table = c->ld_table;
    out.page_stride = (uint32_t)(bytes * c->page_stride);
    out.head_stride = bytes * c->head_stride;
    out.token_stride = (uint32_t)(bytes * c->token_stride);
    out.slots = c->slots;
    out.pages = c->pages;
    out.page_bits = __builtin_ctz((unsigned)c->page_size);
    out.kv_heads = c->kv_heads;
    out.head_dim = c->head_dim;
    return check_scales(ctx, c, scales);
}

template <typename Cache>
int check_attn(vxs_ctx* ctx, const Cache* c, int q_heads, const void* q, int64_t ldq, const void* out, int64_t ldo,
               int out_dtype, float scale) {
    const int64_t width = (int64_t)q_heads * c->head_dim;
    if (ldq < width || ldo < width) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "ldq or ldo below q_heads * head_dim");
    if (!(scale > 0.0f) || std::isinf(scale)) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "scale must be positive and finite");
    if (out_dtype != VXS_F32 && out_dtype != query_type(c))
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "out_dtype must be VXS_F32 or the cache's dtype");
    if (ldq % 8 || ldo % 8 || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u))
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "attention needs ldq and ldo multiples of 8, 16-byte aligned q and out");
    return VXS_OK;
}

template <typename Cache>
int step_args(vxs_ctx* ctx, int rows, int q_heads, const Cache* cache, int max_len, const vxs_shared_prefix* prefix,
              vxs::StepArgs& a, vxs::CacheScales& scales) {
    int rc = check_cache(ctx, cache, q_heads, a.cache, scales);
    if (rc != VXS_OK) return rc;
    if (rows < 0 || max_len < 0) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "bad rows or max_len");
    a.rows = rows;
    a.q_heads = q_heads;
    a.max_len = max_len;
    a.prefix = vxs_shared_prefix{};
    if (prefix) {
        if (prefix->flags & ~VXS_FLAG_SHARE_ALWAYS) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "unknown prefix flags");
        if (prefix->groups < 0 || prefix->max_len < 0) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "bad prefix groups or max_len");
        if (prefix->groups > 0 && (!prefix->d_off || !prefix->d_len))
            return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "prefix d_off or d_len is NULL");
        if (prefix->max_len > 0) a.prefix = *prefix;
    }
    return VXS_OK;
}

template <typename Cache>
int append(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
           int64_t ldv, int in_dtype, const vxs_kv_prep* prep, const vxs_rope_axes* axes, const int32_t* d_pos,
           const int32_t* d_slots, const int32_t* d_index, const Cache* cache, void* q_out, int64_t ldqo, int32_t* d_status) {
    if (!ctx) return VXS_ERR_INVALID_ARG;
    vxs::AppendArgs a{};
    const int rc = check_cache(ctx, cache, q_heads, a.cache, a.scales);
    if (rc != VXS_OK) return rc;
    if (tokens < 0) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "tokens < 0");
    if (in_dtype != VXS_F32 && in_dtype != VXS_BF16 && in_dtype != VXS_F16)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "in_dtype must be VXS_F32, VXS_BF16 or VXS_F16");
    const int d = cache->head_dim;
    if (prep) a.prep = *prep;
    if (a.prep.rot_dim < 0 || a.prep.rot_dim > d || a.prep.rot_dim % 2)
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "rot_dim must be even, from 0 to head_dim");
    if (a.prep.rot_dim > 0 && !a.prep.inv_freq) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "inv_freq is NULL");
    if ((a.prep.q_norm || a.prep.k_norm) && !(a.prep.eps >= 0.0f))
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "eps must not be negative");
    if (a.prep.rot_dim % 8) return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "rot_dim must be a multiple of 8");
    if (tokens >= 1 << 24) return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "tokens must stay below 2^24");
    if (tokens == 0) return vxs::ctx_ok(ctx);
    if (!k != !v) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "k and v come together");
    if (!q && !k) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "neither queries nor keys and values");
    if (q && !q_out) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "q_out is NULL");
    if (axes) {
        if (axes->axes <= 0 || !axes->d_axis) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "bad axes or d_axis");
        if (axes->ld_pos < tokens) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "ld_pos below tokens");
        if (k && !d_index) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "positions of several axes need d_index");
        if ((uintptr_t)axes->d_axis & 15u) return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "d_axis must be 16-byte aligned");
        a.axes = *axes;
    }
    if (!d_pos && (a.prep.rot_dim > 0 || (k && !d_index))) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "d_pos is NULL");
    const int64_t wq = (int64_t)q_heads * d, wk = (int64_t)cache->kv_heads * d;
    if ((q && (ldq < wq || ldqo < wq)) || (k && (ldk < wk || ldv < wk)))
        return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "a leading dimension is below its heads' entries");
    const uintptr_t unit = 4 * bytes_of(in_dtype) - 1;
    auto odd = [&](const void* p, int64_t ld) { return p && (((uintptr_t)p & unit) || ld % 4); };
    if (odd(q, ldq) || odd(k, ldk) || odd(v, ldv) || (q && (((uintptr_t)q_out & 7u) || ldqo % 4)) ||
        ((uintptr_t)a.prep.q_norm & 15u) || ((uintptr_t)a.prep.k_norm & 15u) || ((uintptr_t)a.prep.inv_freq & 15u))
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED,
                        "append needs rows of 4-entry alignment, leading dimensions multiples of 4 and 16-byte aligned prep arrays");
    VXS_ATTN_HIP(ctx, vxs::ctx_use(ctx));
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldqo = ldqo;
    a.pos = d_pos;
    a.slots = d_slots;
    a.index = d_index ? d_index : d_pos;
    a.q_out = q_out;
    a.status = d_status;
    a.tokens = tokens;
    a.q_heads = q_heads;
    const auto stream = static_cast<hipStream_t>(vxs_get_stream(ctx));
    VXS_ATTN_HIP(ctx, a.scales.k ? vxs::launch_kv8_append(a, in_dtype, query_type(cache), stream)
                                      : vxs::launch_kv_append(a, in_dtype, query_type(cache), stream));
    return vxs::ctx_ok(ctx);
}

template <typename Cache>
int packed(vxs_ctx* ctx, bool cross, int seqs, int tokens, int q_heads, const void* q, int64_t ldq, const Cache* cache,
           const int32_t* d_slots, const int32_t* d_q_off, const int32_t* d_kv_len, float scale, void* out, int64_t ldo,
           int out_dtype) {
    if (!ctx) return VXS_ERR_INVALID_ARG;
    vxs::PromptArgs a{};
    vxs::CacheScales scales{};
    int rc = check_cache(ctx, cache, q_heads, a.cache, scales);
    if (rc != VXS_OK) return rc;
    if (seqs < 0 || tokens < 0) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "bad seqs or tokens");
    if ((rc = check_attn(ctx, cache, q_heads, q, ldq, out, ldo, out_dtype, scale)) != VXS_OK) return rc;
    if (seqs == 0 || tokens == 0) return vxs::ctx_ok(ctx);
    if (!q || !out || !d_q_off || !d_kv_len) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "null pointer");
    if ((int64_t)tokens * q_heads > INT32_MAX - 1024)
        return ctx_fail(ctx, VXS_ERR_UNSUPPORTED, "tokens * q_heads must stay below 2^31 - 1024");
    VXS_ATTN_HIP(ctx, vxs::ctx_use(ctx));
    a.q = q;
    a.out = out;
    a.slots = d_slots;
    a.q_off = d_q_off;
    a.kv_len = d_kv_len;
    a.ldq = ldq;
    a.ldo = ldo;
    a.scale = scale;
    a.seqs = seqs;
    a.tokens = tokens;
    a.q_heads = q_heads;
    VXS_ATTN_HIP(ctx, vxs::launch_attn_prompt(a, scales, cross, query_type(cache), out_dtype, static_cast<hipStream_t>(vxs_get_stream(ctx))));
    return vxs::ctx_ok(ctx);
}

template <typename Cache>
int step(vxs_ctx* ctx, int rows, int q_heads, const void* q, int64_t ldq, const Cache* cache, const int32_t* d_slots,
         const int32_t* d_kv_len, int max_len, const vxs_shared_prefix* prefix, float scale, void* out, int64_t ldo,
         int out_dtype, void* work, int64_t work_bytes) {
    if (!ctx) return VXS_ERR_INVALID_ARG;
    vxs::StepArgs a{};
    vxs::CacheScales scales{};
    int rc = step_args(ctx, rows, q_heads, cache, max_len, prefix, a, scales);
    if (rc != VXS_OK) return rc;
    if ((rc = check_attn(ctx, cache, q_heads, q, ldq, out, ldo, out_dtype, scale)) != VXS_OK) return rc;
    if (rows == 0) return vxs::ctx_ok(ctx);
    if (!q || !out || !d_kv_len) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "null pointer");
    if (work) {
        if ((uintptr_t)work & 15u) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "work must be 16-byte aligned");
        if (work_bytes < vxs::attn_step_work_bytes(a)) return ctx_fail(ctx, VXS_ERR_INVALID_ARG, "work is smaller than vxs_attn_step_workspace");
    }
    VXS_ATTN_HIP(ctx, vxs::ctx_use(ctx));
    a.q = q;
    a.out = out;
    a.slots = d_slots;
    a.kv_len = d_kv_len;
    a.ldq = ldq;
    a.ldo = ldo;
    a.scale = scale;
    a.work = work;
    VXS_ATTN_HIP(ctx, vxs::launch_attn_step(a, scales, query_type(cache), out_dtype, static_cast<hipStream_t>(vxs_get_stream(ctx))));
    return vxs::ctx_ok(ctx);
}

template <typename Cache>
int64_t workspace(vxs_ctx* ctx, int rows, int q_heads, const Cache* cache, int max_len, const vxs_shared_prefix* prefix) {
    if (!ctx) return VXS_ERR_INVALID_ARG;
    vxs::StepArgs a{};
    vxs::CacheScales scales{};
    const int rc = step_args(ctx, rows, q_heads, cache, max_len, prefix, a, scales);
    return rc != VXS_OK ? rc : vxs::attn_step_work_bytes(a);
}

// f(), and no exception of it.
template <typename F>
auto guarded(F f) -> decltype(f()) {
    try {
        return f();
    } catch (...) {
        return VXS_ERR_INVALID_ARG;
    }
}

}  // namespace

extern "C" {

VXS_API int vxs_kv_append_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                 int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                 const int32_t* d_pos, const int32_t* d_slots, const int32_t* d_index,
                                 const vxs_kv_cache* cache, void* q_out, int64_t ldqo, int32_t* d_status) {
    return guarded([&] { return append(ctx, tokens, q_heads, q, ldq, k, ldk, v, ldv, in_dtype, prep, nullptr, d_pos, d_slots, d_index, cache, q_out, ldqo, d_status); });
}

VXS_API int vxs_kv_append_axes_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                      int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                      const vxs_rope_axes* axes, const int32_t* d_pos, const int32_t* d_slots,
                                      const int32_t* d_index, const vxs_kv_cache* cache, void* q_out, int64_t ldqo,
                                      int32_t* d_status) {
    return guarded([&] { return append(ctx, tokens, q_heads, q, ldq, k, ldk, v, ldv, in_dtype, prep, axes, d_pos, d_slots, d_index, cache, q_out, ldqo, d_status); });
}

VXS_API int vxs_kv8_append_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                  int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                  const vxs_rope_axes* axes, const int32_t* d_pos, const int32_t* d_slots,
                                  const int32_t* d_index, const vxs_kv8_cache* cache, void* q_out, int64_t ldqo,
                                  int32_t* d_status) {
    return guarded([&] { return append(ctx, tokens, q_heads, q, ldq, k, ldk, v, ldv, in_dtype, prep, axes, d_pos, d_slots, d_index, cache, q_out, ldqo, d_status); });
}

VXS_API int vxs_attn_prompt_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                   const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                   const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype) {
    return guarded([&] { return packed(ctx, false, seqs, tokens, q_heads, q, ldq, cache, d_slots, d_q_off, d_kv_len, scale, out, ldo, out_dtype); });
}

VXS_API int vxs_attn_cross_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                  const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                  const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype) {
    return guarded([&] { return packed(ctx, true, seqs, tokens, q_heads, q, ldq, cache, d_slots, d_q_off, d_kv_len, scale, out, ldo, out_dtype); });
}

VXS_API int vxs_attn8_prompt_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                    const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                    const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype) {
    return guarded([&] { return packed(ctx, false, seqs, tokens, q_heads, q, ldq, cache, d_slots, d_q_off, d_kv_len, scale, out, ldo, out_dtype); });
}

VXS_API int vxs_attn8_cross_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                   const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                   const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype) {
    return guarded([&] { return packed(ctx, true, seqs, tokens, q_heads, q, ldq, cache, d_slots, d_q_off, d_kv_len, scale, out, ldo, out_dtype); });
}

VXS_API int vxs_attn_step_device(vxs_ctx* ctx, int rows, int q_heads, const void* q, int64_t ldq,
                                 const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_kv_len, int max_len,
                                 const vxs_shared_prefix* prefix, float scale, void* out, int64_t ldo, int out_dtype,
                                 void* work, int64_t work_bytes) {
    return guarded([&] { return step(ctx, rows, q_heads, q, ldq, cache, d_slots, d_kv_len, max_len, prefix, scale, out, ldo, out_dtype, work, work_bytes); });
}

VXS_API int64_t vxs_attn_step_workspace(vxs_ctx* ctx, int rows, int q_heads, const vxs_kv_cache* cache, int max_len,
                                        const vxs_shared_prefix* prefix) {
    return guarded([&] { return workspace(ctx, rows, q_heads, cache, max_len, prefix); });
}

VXS_API int vxs_attn8_step_device(vxs_ctx* ctx, int rows, int q_heads, const void* q, int64_t ldq,
                                  const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_kv_len, int max_len,
                                  const vxs_shared_prefix* prefix, float scale, void* out, int64_t ldo, int out_dtype,
                                  void* work, int64_t work_bytes) {
    return guarded([&] { return step(ctx, rows, q_heads, q, ldq, cache, d_slots, d_kv_len, max_len, prefix, scale, out, ldo, out_dtype, work, work_bytes); });
}

VXS_API int64_t vxs_attn8_step_workspace(vxs_ctx* ctx, int rows, int q_heads, const vxs_kv8_cache* cache, int max_len,
                                         const vxs_shared_prefix* prefix) {
    return guarded([&] { return workspace(ctx, rows, q_heads, cache, max_len, prefix); });
}

}  // extern "C"
