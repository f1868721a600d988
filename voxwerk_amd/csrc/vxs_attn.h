// vxs_attn.h — shared declarations of the paged cache's operators: arguments of the kernels and their launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/vxs_sampler.h"

namespace vxs {

// A layer's cache as the kernels take it (vxs_kv_cache or vxs_kv8_cache, checked).
struct PagedCache {
    char* k;
    char* v;
    const int32_t* table;
    int64_t ld_table;
    int64_t head_stride;                 // bytes
    uint32_t page_stride, token_stride;  // bytes
    int slots, pages, page_bits, kv_heads, head_dim;
};

// Scales of 8-bit entries (null: entries of 16 bits).
struct CacheScales {
    uint8_t *k, *v;
};

// An append's arguments as far as each kernel needs them: longer ones take longer to launch (vxs_append.hip).
struct AppendOneArgs {  // one position a token
    PagedCache cache;
    vxs_kv_prep prep;
    const void *q, *k, *v;  // q, or k and v, may be null
    int64_t ldq, ldk, ldv, ldqo;
    const int32_t *pos, *slots, *index;
    void* q_out;
    int32_t* status;
    int tokens, q_heads;
};
struct AppendAxesArgs : AppendOneArgs {
    vxs_rope_axes axes;  // axes 0: one position a token
};
struct AppendArgs : AppendAxesArgs {
    CacheScales scales;
};
hipError_t launch_kv_append(const AppendArgs& a, int in_dtype, int dtype, hipStream_t stream);
hipError_t launch_kv8_append(const AppendArgs& a, int in_dtype, int q_dtype, hipStream_t stream);

struct PromptArgs {
    PagedCache cache;
    const void* q;
    void* out;
    const int32_t *slots, *q_off, *kv_len;
    int64_t ldq, ldo;  // elements
    float scale;
    int seqs, tokens, q_heads;
};
// dtype: the queries' type; cross: every token sees all of its sequence's keys. The scales come after the other arguments in the kernels:
// those of 16-bit caches do not move for them (a prompt of 93 tokens took 8.35 us with longer ones, 7.86 with these).
hipError_t launch_attn_prompt(const PromptArgs& a, const CacheScales& scales, bool cross, int dtype, int out_dtype, hipStream_t stream);

struct StepArgs {
    PagedCache cache;
    const void* q;
    void* out;
    const int32_t *slots, *kv_len;
    vxs_shared_prefix prefix;  // groups 0: none
    int64_t ldq, ldo;  // elements
    float scale;
    int rows, q_heads, max_len;
    void* work;
};
// The bytes of `work` that launch_attn_step asks for at sizes up to a call's (work itself is not looked at).
int64_t attn_step_work_bytes(const StepArgs& a);
hipError_t launch_attn_step(const StepArgs& a, const CacheScales& scales, int dtype, int out_dtype, hipStream_t stream);

#ifdef __HIPCC__
// Tokens that slot `slot` may read: none for a slot outside the cache, at most what its table names.
__device__ __forceinline__ int64_t cache_length(const PagedCache& c, int slot, int len) {
    if ((unsigned)slot >= (unsigned)c.slots || len <= 0) return 0;
    const int64_t most = c.ld_table << c.page_bits;
    return len < most ? len : most;
}

// Byte offset, from k or v, of token t's entries of head h, whose table entry is `page`. A page number outside the
// pool (a caller's mistake) reads some page of it.
__device__ __forceinline__ uint64_t cache_offset(const PagedCache& c, int page, int h, int t) {
    return (uint64_t)min((unsigned)page, (unsigned)c.pages - 1u) * c.page_stride + (uint64_t)h * c.head_stride +
           (uint64_t)((unsigned)t & ((1u << c.page_bits) - 1u)) * c.token_stride;
}

constexpr int kBlockTokens = 16;  // of an 8-bit cache's scale

// Index of the scale of token t's block of head h, in a page as above.
__device__ __forceinline__ uint64_t scale_index(const PagedCache& c, int page, int h, int t) {
    return (((uint64_t)min((unsigned)page, (unsigned)c.pages - 1u) * (unsigned)c.kv_heads + (unsigned)h) << (c.page_bits - 4)) +
           (((unsigned)t & ((1u << c.page_bits) - 1u)) >> 4);
}
#endif

}  // namespace vxs
