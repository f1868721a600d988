/*
 * vxs_sampler.h — C ABI of the MI355X (gfx950) token sampler.
 *
 * One call turns each row of fp32 logits into a token id with the semantics of voxwerk's
 * Sampler (src/Voxwerk/Talker/Sampler.cs:1-96) plus the talker's suppression glue
 * (src/Voxwerk/Talker/TalkerGenerator.cs:246-249, :370-373):
 *   repetition penalty -> suppression -> (greedy argmax | temperature -> top-k -> softmax
 *   -> top-p -> inverse-CDF draw from a caller-supplied uniform).
 *
 * The reference is managed C# with no native boundary; these entry points are what its
 * P/Invoke layer binds (DllImport style of src/Voxwerk/Numerics/NativeBuffer.cs:78-92).
 * Plain pointers and sizes only. No C++ exceptions cross this boundary.
 *
 * Threading: one context owns one HIP stream and may be used by one thread at a time.
 * Separate contexts may run concurrently.
 */
#ifndef VXS_SAMPLER_H
#define VXS_SAMPLER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define VXS_API __attribute__((visibility("default")))
#else
#define VXS_API
#endif

/* Return codes. A row that fails gets the code in its out_ids slot (all codes are < 0). */
#define VXS_OK 0
#define VXS_ERR_INVALID_ARG (-1)     /* bad pointer/shape/option (C#: ArgumentException family)          */
#define VXS_ERR_ID_OUT_OF_RANGE (-2) /* history id < 0 or >= vocab (C#: Span indexer at Sampler.cs:30)   */
#define VXS_ERR_NONFINITE (-3)       /* NaN or +inf logit after temperature: outside the contract        */
#define VXS_ERR_HIP (-4)             /* HIP runtime failure; text in vxs_last_error                      */
#define VXS_ERR_UNSUPPORTED (-5)     /* shape outside what the library implements; text in vxs_last_error */
#define VXS_ERR_NO_DEVICE (-6)       /* no usable gfx950 device                                          */
#define VXS_ERR_HISTORY_FULL (-7)    /* resident history slot already holds `cap` ids (vxs_sample_batch)  */

/* flags for vxs_sample / vxs_sample_device */
#define VXS_FLAG_NONE 0u
/* Kernel selection; without either flag the library chooses (one wave per row for batches of at
 * least 1024 rows with vocab <= 3072, else one workgroup per row). Results are identical. */
#define VXS_FLAG_PATH_BLOCK (1u << 8) /* one 256-thread workgroup per row                      */
#define VXS_FLAG_PATH_WAVE (1u << 9)  /* one wave per row first, 4 rows per workgroup (vocab <= 3072) */
/* vxs_sample_batch / vxs_sample_batch_device only: instead of reading `u` (which may be NULL),
 * each sampled row draws its uniform on the device from its slot's generator (vxs_history_seed):
 * the talker's new Random(Seed) or the code predictor's new Random(Seed + 1). A greedy row draws
 * nothing, as Select consumes no NextDouble when DoSample is false (Sampler.cs:37,77). */
#define VXS_FLAG_RNG_TALKER (1u << 10)
#define VXS_FLAG_RNG_SUB (1u << 11)

/*
 * Per-row sampling parameters (blittable; 36 bytes, 4-byte aligned).
 * Mirrors SamplingOptions (Sampler.cs:4-13), GenerationOptions.RepetitionPenalty
 * (TalkerGenerator.cs:11) and the talker's suppression rule (TalkerGenerator.cs:247-248).
 */
typedef struct vxs_params {
    int32_t do_sample;   /* SamplingOptions.DoSample; 0 = first-index argmax, no draw consumed      */
    int32_t top_k;       /* SamplingOptions.TopK; applied only when 0 < top_k < vocab               */
    float top_p;         /* SamplingOptions.TopP; applied only when top_p < 1                       */
    float temperature;   /* SamplingOptions.Temperature; logits are multiplied by fl32(1/T)         */
    float rep_penalty;   /* repetition penalty over the distinct history ids; 1 = off               */
    int32_t supp_begin;  /* ids in [supp_begin, supp_end) except keep_id are set to -inf            */
    int32_t supp_end;    /*   (talker: [vocab-1024, vocab) except EOS); empty range = off           */
    int32_t keep_id;     /* exempt from suppression (EOS); -1 = none                                */
    int32_t ban_id;      /* set to -inf after suppression (EOS while step < 2); -1 = none           */
} vxs_params;

typedef struct vxs_ctx vxs_ctx;

/*
 * Create a context on HIP device `device` (ordinal among visible devices). Capacities are
 * hints: buffers grow on demand and are freed by vxs_destroy.
 * Replaces: construction of Sampler (Sampler.cs:21) — the RNG stays with the caller, which
 * passes one NextDouble() per sampled row as `u`.
 */
VXS_API int vxs_create(vxs_ctx** out, int device, int max_rows, int max_vocab, int64_t max_hist);
VXS_API void vxs_destroy(vxs_ctx* ctx);

/* Text of the last error on this context ("" if none). Valid until the next call on ctx. */
VXS_API const char* vxs_last_error(const vxs_ctx* ctx);

/* Library version string, e.g. "vxs 0.1.0 gfx950". */
VXS_API const char* vxs_version(void);

/*
 * Use an external HIP stream (hipStream_t passed as void*) for all work of this context.
 * NULL restores the context's own stream. The caller keeps ownership of the stream.
 */
VXS_API int vxs_set_stream(vxs_ctx* ctx, void* hip_stream);
/* The hipStream_t (as void*) this context currently launches on. */
VXS_API void* vxs_get_stream(const vxs_ctx* ctx);

/*
 * The longest time, in units of 10 ns, that the workgroups of a row split over several of them
 * (vxs_sample_device) wait for each other before one samples it alone; 50000 (500 us) in a new
 * context, at most 10000000 (100 ms). The ids are the same. 0 gives every such wait up, for tests of that
 * path.
 */
VXS_API int vxs_set_split_wait(vxs_ctx* ctx, uint32_t ticks);

/*
 * Host-pointer sampling call; synchronous.
 * Replaces, for each row: Sampler.ApplyRepetitionPenalty (Sampler.cs:25-33), the suppression
 * loops (TalkerGenerator.cs:247-248, :371-372) and Sampler.Select (Sampler.cs:35-88) as
 * called at TalkerGenerator.cs:246-249, :268, :370-373, :419-420.
 *
 *   logits     [rows][ld] fp32, host memory; only the first `vocab` entries of a row are read
 *   hist_off   [rows+1] CSR offsets into hist_ids (hist_off[0] need not be 0); NULL = no history
 *   hist_ids   int32 generated-code history; duplicates allowed (applied once per distinct id)
 *   params     params[r * params_stride]; params_stride 0 broadcasts one struct to all rows
 *   u          [rows] uniforms in [0,1) (Random.NextDouble() per sampled row); may be NULL
 *              when no row samples
 *   out_ids    [rows] sampled ids; a failing row receives its negative error code
 *   out_logits NULL or [rows][vocab]: the row as Select leaves the caller's span (after
 *              penalty, suppression, temperature and the top-k -inf mask); may be `logits` itself
 *              when ld == vocab (in place); a row that fails keeps its contents
 *   out_probs  NULL or [rows][vocab] fp64: final probabilities the draw used (parity/debug)
 * Returns VXS_OK, or the first (lowest row) error code.
 */
VXS_API int vxs_sample(vxs_ctx* ctx, int rows, int vocab, const float* logits, int64_t ld,
                       const int32_t* hist_off, const int32_t* hist_ids,
                       const vxs_params* params, int params_stride, const double* u,
                       int32_t* out_ids, float* out_logits, double* out_probs, uint32_t flags);

/*
 * Device-pointer sampling call; asynchronous on the context stream. Every pointer is device
 * memory (params included). Per-row errors land in out_ids as negative codes; call
 * vxs_synchronize to wait. For callers whose logits are already resident on the GPU (logit
 * heads on device) and for kernel-only timing. Batches of at most 192 rows with vocab > 8192 split
 * each row over several workgroups, in a workspace of about 20 MB that the context allocates at the
 * first such call on a stream (its own, and up to four set with vxs_set_stream); where none is to be
 * had, and on a stream that is being captured, the call takes one workgroup per row. Same ids.
 */
VXS_API int vxs_sample_device(vxs_ctx* ctx, int rows, int vocab, const float* d_logits, int64_t ld,
                              const int32_t* d_hist_off, const int32_t* d_hist_ids,
                              const vxs_params* d_params, int params_stride, const double* d_u,
                              int32_t* d_out_ids, float* d_out_logits, double* d_out_probs,
                              uint32_t flags);

/*
 * vxs_sample for callers that cannot allocate (tight serving loops, harnesses that forbid hipMalloc):
 * no counterpart in the reference. Same arguments, semantics and errors as vxs_sample without the
 * write-back and probability outputs; synchronous. It allocates nothing: the inputs are copied from
 * the caller's memory into a fixed 16 MiB device scratch (one per GPU, held until the process ends),
 * the kernels read them there and write the ids there, and the ids are copied back. A call that
 * needs more than the scratch (about rows * vocab * 4 bytes plus the histories, params and
 * uniforms) fails with VXS_ERR_UNSUPPORTED. Every context on one GPU shares that GPU's scratch, so
 * the library serialises the calls on one GPU (from any threads or contexts) with a per-device lock
 * held for the whole call: concurrent calls wait for each other.
 */
VXS_API int vxs_sample_noalloc(vxs_ctx* ctx, int rows, int vocab, const float* logits, int64_t ld,
                               const int32_t* hist_off, const int32_t* hist_ids, const vxs_params* params,
                               int params_stride, const double* u, int32_t* out_ids, uint32_t flags);

/*
 * Parity/debug variant of vxs_sample_device (no counterpart in the reference): no write-back or
 * probabilities; instead, for every row sampled by the one-wave nucleus regime (sampled rows,
 * vocab <= 3072, whose top-k masks nothing and that keep more than 256 finite entries),
 *   d_stats[4r + 0] = kept fraction of the probability mass (after top-p; 1 without top-p),
 *   d_stats[4r + 1] = smallest kept probability (the top-p cut),
 *   d_stats[4r + 2] = number of kept entries (entries whose mass is 0 on the 2^-F grid excluded),
 *   d_stats[4r + 3] = 0,
 * so that the nucleus is checked beyond the id; all four are NaN for every other row (greedy,
 * exact regime, rows the one-workgroup algorithm samples). d_stats is [rows][4] fp64 device memory.
 * d_probs (optional, [rows][vocab] fp64 device memory): for the same rows, every entry's final
 * probability as the draw used it (its mass over the kept mass, 0 for removed entries); NaN for
 * every other row.
 */
VXS_API int vxs_sample_stats_device(vxs_ctx* ctx, int rows, int vocab, const float* d_logits, int64_t ld,
                                    const int32_t* d_hist_off, const int32_t* d_hist_ids,
                                    const vxs_params* d_params, int params_stride, const double* d_u,
                                    int32_t* d_out_ids, double* d_stats, double* d_probs, uint32_t flags);

/* Wait for all work queued on the context stream. */
VXS_API int vxs_synchronize(vxs_ctx* ctx);

/*
 * In-place repetition penalty on host rows (Sampler.ApplyRepetitionPenalty, Sampler.cs:25-33):
 * each distinct history id's logit s becomes s*penalty if s < 0, else s/penalty.
 * penalty == 1 is a no-op. Synchronous.
 */
VXS_API int vxs_apply_repetition_penalty(vxs_ctx* ctx, int rows, int vocab, float* logits, int64_t ld,
                                         const int32_t* hist_off, const int32_t* hist_ids,
                                         float penalty);

/* First index of the maximum of each host row (Sampler.ArgMax, Sampler.cs:90-95). Synchronous. */
VXS_API int vxs_argmax(vxs_ctx* ctx, int rows, int vocab, const float* logits, int64_t ld,
                       int32_t* out_ids);

/*
 * Resident histories for batched generation (TalkerGenerator.GenerateBatch,
 * TalkerGenerator.cs:322-455). A store holds `slots` sequence histories of at most `cap` ids each
 * in device memory of the context's device; one slot replaces one Active.History list
 * (TalkerGenerator.cs:304). The sampler reads a row's history from its slot and appends the id it
 * draws there (History.Add, TalkerGenerator.cs:374), so histories never cross PCIe per step.
 * A sequence appends one id per step and retires after MaxNewTokens steps (:375), so
 * cap = MaxNewTokens always suffices. slots * cap must not exceed 2^31 - 1. All slots start empty.
 */
typedef struct vxs_history vxs_history;
VXS_API int vxs_history_create(vxs_ctx* ctx, int slots, int cap, vxs_history** out);
/* Frees the store; no work that uses it may still be queued. */
VXS_API void vxs_history_destroy(vxs_history* h);
/* Replace slot `slot`'s history with ids[0..n) (0 <= n <= cap; n = 0 empties it, as a refilled
 * job starts with an empty History, TalkerGenerator.cs:336-349). Stream-ordered; synchronous. */
VXS_API int vxs_history_set(vxs_ctx* ctx, vxs_history* h, int slot, const int32_t* ids, int n);
/* Copy slot `slot`'s history into ids[0..max_ids) and its length into *n. Synchronous. */
VXS_API int vxs_history_get(vxs_ctx* ctx, vxs_history* h, int slot, int32_t* ids, int max_ids, int* n);
/* Seed slot `slot`'s two generators as a sequence's samplers are built (TalkerGenerator.cs:217-218,
 * :345-346): new Random(seed) for the talker, new Random(seed + 1) for the code predictor, with
 * .NET's seeded generator (Sampler.cs:21) and C#'s wrapping int arithmetic. A job without a seed
 * passes one of its own choosing. Synchronous. */
VXS_API int vxs_history_seed(vxs_ctx* ctx, vxs_history* h, int slot, int32_t seed);
/* The next n NextDouble() values (Sampler.cs:77) of slot `slot`'s talker (stream 0) or
 * code-predictor (stream 1) generator, drawn on the device into out[0..n). Synchronous. */
VXS_API int vxs_history_draw(vxs_ctx* ctx, vxs_history* h, int slot, int stream, int n, double* out);

/*
 * One batched sampling stage over host rows whose histories live in `h`: row r penalises with
 * slot slots[r]'s history, then (append != 0) its sampled id is appended to that slot.
 * Replaces the serial per-row loops of GenerateBatch: the talker stage (TalkerGenerator.cs:366-375:
 * ApplyRepetitionPenalty, suppression, a.Sampler.Select, History.Add; append = 1) and the
 * code-predictor stage (:419-420: SubSampler.Select, no penalty; pass rep_penalty 1 and append = 0).
 * Arguments as vxs_sample, with `slots` [rows] host memory: distinct slot indices in [0, slots of h).
 * A row that fails keeps its error code in out_ids and appends nothing; a full slot fails the row
 * with VXS_ERR_HISTORY_FULL. Synchronous.
 */
VXS_API int vxs_sample_batch(vxs_ctx* ctx, vxs_history* h, int rows, int vocab, const float* logits,
                             int64_t ld, const int32_t* slots, int append, const vxs_params* params,
                             int params_stride, const double* u, int32_t* out_ids, uint32_t flags);

/*
 * vxs_sample_batch with device pointers (logits, slots, params, u, out_ids); asynchronous on the
 * context stream like vxs_sample_device. A slot outside the store fails its row with
 * VXS_ERR_INVALID_ARG. Slots must be distinct within one call: the store stays in bounds if they
 * are not, but keeps only one of the ids appended to a repeated slot.
 */
VXS_API int vxs_sample_batch_device(vxs_ctx* ctx, vxs_history* h, int rows, int vocab,
                                    const float* d_logits, int64_t ld, const int32_t* d_slots,
                                    int append, const vxs_params* d_params, int params_stride,
                                    const double* d_u, int32_t* d_out_ids, uint32_t flags);

/*
 * Logit heads on the GPU, the step before the sampler: CodecHead and CodePredictorHead
 * (TalkerModel.cs:133-137, Gemm.Multiply over a bf16 PackedMatrix, WeightPrecision.BFloat16):
 *   out[r][j] = sum_k x[r][k] * W[j][k],   r < rows, j < n, k < k
 * x fp32 [rows][ldx], W bf16 [n][ldw] (the checkpoint's [out, in] layout: talker.codec_head.weight,
 * talker.code_predictor.lm_head.{g}.weight), out fp32 [rows][ldo], all device memory, so the
 * logits stay on the GPU for vxs_sample_device / vxs_sample_batch_device. fp32 products and sums
 * in an order of this library's own: each entry is within k * 2^-24 * sum_k |x w| of the exact
 * dot product, as the reference's is. Needs k <= 2048, k and ldw multiples of 8, ldx a multiple
 * of 4, 16-byte aligned x and W (else VXS_ERR_UNSUPPORTED). Asynchronous on the context stream.
 */
VXS_API int vxs_head_device(vxs_ctx* ctx, int rows, int k, int n, const float* d_x, int64_t ldx,
                            const uint16_t* d_w, int64_t ldw, float* d_out, int64_t ldo);

/*
 * The same heads with int8 weights (WeightPrecision.Int8, DecoderStack.cs:7-16; the reference packs
 * codec_head and every code_predictor.lm_head this way when asked, TalkerModel.cs:37,55):
 *   out[r][j] = scale[j] * sum_k x[r][k] * q[j][k]
 * the decode path's form (Gemm.cs:602-680: SmallM, PanelPairDotInt8 / PanelDotInt8, the scale
 * applied to the fp32 dot). q int8 [n][ldq], scale fp32 [n], as vxs_head_pack_int8_device writes
 * them. Each entry is within (k + 1) * 2^-24 * scale[j] * sum_k |x q| of the exact value, a bound
 * the reference's decode form and its batched form (Gemm.cs:95-98, which dequantizes q * scale
 * first) both satisfy. Needs k <= 2048, k and ldq multiples of 8, ldx a multiple of 4, 16-byte
 * aligned x and q (else VXS_ERR_UNSUPPORTED). Asynchronous on the context stream.
 */
VXS_API int vxs_head_int8_device(vxs_ctx* ctx, int rows, int k, int n, const float* d_x, int64_t ldx,
                                 const int8_t* d_q, int64_t ldq, const float* d_scale, float* d_out, int64_t ldo);

/*
 * int8 packing of a bf16 head weight on the GPU, PackedMatrix.FromBf16LinearInt8
 * (src/Voxwerk/Numerics/PackedMatrix.cs:124-154), bit for bit: per output row j, amax = max_k |W[j][k]|,
 * scale[j] = amax / 127 (1 when amax is 0), q[j][k] = clamp(round-half-even(W[j][k] * (1 / scale[j])),
 * -127, 127), in correctly rounded fp32, the (int) conversion saturating as in .NET 9 and later (a
 * row whose 1 / scale overflows gets +-127 and 0). W bf16 [n][ldw], q int8 [n][ldq], scale fp32 [n];
 * finite weights. Asynchronous on the context stream.
 */
VXS_API int vxs_head_pack_int8_device(vxs_ctx* ctx, int k, int n, const uint16_t* d_w, int64_t ldw, int8_t* d_q,
                                      int64_t ldq, float* d_scale);

/*
 * Embedding rows of sampled ids, the step after the sampler, so that ids need not return to the
 * host between sampling and the next forward pass. Tables are bf16 [vocab][hidden], widened to
 * fp32 exactly (Bf16.ToFloat, src/Voxwerk/Numerics/Bf16.cs:13); sums run in the reference's order,
 * so rows are bit-identical. Device pointers, asynchronous on the context stream. status[r] gets 0,
 * or VXS_ERR_ID_OUT_OF_RANGE for a row holding an id outside its table, which is then not written
 * (the reference throws ArgumentOutOfRangeException, TalkerModel.cs:102,109).
 *
 * vxs_embed_device replaces CodecEmbedding / CodePredictorEmbedding (TalkerModel.cs:100-111):
 * out[r] = table[ids[r]] (add = 0) or out[r] += table[ids[r]] (add = 1), as called at
 * TalkerGenerator.cs:258, :271, :411 and :422.
 */
VXS_API int vxs_embed_device(vxs_ctx* ctx, int rows, int hidden, const int32_t* d_ids, const uint16_t* d_table,
                             int vocab, float* d_out, int64_t ld_out, int add, int32_t* d_status);

/*
 * FrameEmbedding (TalkerModel.cs:113-117) for `rows` frames, plus the talker step's text row
 * (TalkerGenerator.cs:280-283, :435-439): out[r] = E0[codes[r][0]] + E1[codes[r][1]] + ... +
 * E_{groups-1}[codes[r][groups-1]] (+ addend[r] when d_addend is not NULL), left to right in fp32.
 * E0 = d_codec_table [vocab][hidden]; E_g = d_cp_tables + (g-1) * cp_vocab * hidden, g >= 1, the
 * code predictor's tables stored back to back. Code g of frame r is d_codes[r * ld_codes +
 * g * group_stride]: a [rows][groups] matrix has ld_codes = groups, group_stride = 1; the ids of one
 * sampling call per codebook, stage g at d_codes + g * rows, have ld_codes = 1, group_stride = rows.
 */
VXS_API int vxs_frame_embed_device(vxs_ctx* ctx, int rows, int groups, int hidden, const int32_t* d_codes,
                                   int64_t ld_codes, int64_t group_stride, const uint16_t* d_codec_table, int vocab,
                                   const uint16_t* d_cp_tables, int cp_vocab, const float* d_addend,
                                   int64_t ld_addend, float* d_out, int64_t ld_out, int32_t* d_status);

/*
 * Attention over a paged cache of keys and values: the layer between the embedding of the sampled ids
 * and the logit heads, for callers whose transformer runs on this GPU too. The reference keeps one
 * contiguous cache per sequence (KvCache, src/Voxwerk/Talker/DecoderStack.cs:21-50) and attends with
 * src/Voxwerk/Numerics/Attention.cs:15-118 and Rope.cs; here a layer's cache is a pool of pages that
 * all sequences share.
 */

/* Element types of the attention entry points. */
#define VXS_F32 0
#define VXS_BF16 1
#define VXS_F16 2

/* flag of vxs_shared_prefix */
#define VXS_FLAG_SHARE_ALWAYS (1u << 12)

/*
 * One layer's cache: keys and values of `pages` pages of `page_size` tokens each. Token t of slot s
 * (a sequence) lies in page p = table[s * ld_table + t / page_size], its key of head h at
 *   k + p * page_stride + h * head_stride + (t % page_size) * token_stride   (elements),
 * its value likewise in v; head_dim contiguous entries each. [pages][kv_heads][page_size][head_dim]
 * has token_stride = head_dim, head_stride = page_size * head_dim, page_stride = kv_heads * head_stride.
 * A host struct; k, v and table are device memory of the caller's, which also owns the choice of
 * pages (several slots may hold the same page). page_size is a power of two from 16 to 65536, head_dim
 * 64, 128 or 256, the strides are multiples of 8 (token_stride below 2^25, page_stride below 2^31), k and v
 * 16-byte aligned (else VXS_ERR_UNSUPPORTED).
 */
typedef struct vxs_kv_cache {
    void* k;
    void* v;
    const int32_t* table; /* [slots][ld_table] page numbers; entries past a sequence's end are not used */
    int64_t ld_table;
    int64_t page_stride;
    int64_t head_stride;
    int64_t token_stride;
    int32_t slots;
    int32_t pages;
    int32_t page_size;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t dtype; /* VXS_BF16 or VXS_F16 */
} vxs_kv_cache;

/*
 * What happens to a query or key head before attention: an RMS norm over its entries (weights fp32
 * [head_dim] in device memory; NULL: none), then the rotation of its first rot_dim entries in pairs:
 * entries i and i + rot_dim / 2 (interleaved 0) or 2i and 2i + 1 (interleaved 1) turn by
 * position * inv_freq[i] radians, inv_freq fp32 [rot_dim / 2] in device memory (rot_dim 0: no
 * rotation). rope_scale multiplies both cosine and sine (1, or the magnitude that a scaling for
 * long contexts asks for). rot_dim is a multiple of 8.
 */
typedef struct vxs_kv_prep {
    const float* q_norm;
    const float* k_norm;
    const float* inv_freq;
    float eps;
    float rope_scale;
    int32_t rot_dim;
    int32_t interleaved;
} vxs_kv_prep;

/*
 * The projections of `tokens` new tokens on their way to attention, in one pass: each query and key head
 * is normed and rotated (prep; NULL: neither), queries go to q_out, keys and values to their pages.
 *   q, k, v    [tokens] rows of q_heads, kv_heads and kv_heads heads of head_dim entries, of in_dtype, with
 *              leading dimensions ldq, ldk, ldv in elements (a packed projection passes three places of one
 *              buffer); q or k and v may be NULL: only the others are done
 *   d_pos      int32 [tokens] positions of the rotation; may be NULL where nothing rotates and d_index is given
 *   d_slots    int32 [tokens] each token's slot; NULL: token t belongs to slot t (one new token per sequence)
 *   d_index    int32 [tokens] each token's place in its sequence; NULL: d_pos
 *   q_out      [tokens] rows of the cache's dtype, leading dimension ldqo
 *   d_status   NULL or int32 [tokens]: 0, or VXS_ERR_ID_OUT_OF_RANGE for a token whose slot, place or page lies
 *              outside the cache: its key and value are not written
 * Norms, angles and products are fp32 or wider, rounded once, to nearest even. Pointers 16-byte (fp32) or 8-byte
 * (bf16, fp16) aligned, leading dimensions multiples of 4 (q_out: 8-byte, 4), else VXS_ERR_UNSUPPORTED. Two tokens
 * of one call with the same place leave entries of either; tokens is below 2^24. Asynchronous on the context stream.
 */
VXS_API int vxs_kv_append_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                 int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                 const int32_t* d_pos, const int32_t* d_slots, const int32_t* d_index,
                                 const vxs_kv_cache* cache, void* q_out, int64_t ldqo, int32_t* d_status);

/*
 * Causal attention of packed sequences over their pages: sequence i (slot d_slots[i]; NULL: slot i) has new tokens
 * [d_q_off[i], d_q_off[i + 1]) of the `tokens` query rows and d_kv_len[i] tokens in the cache, the new ones last
 * (appended before): its j-th of n new tokens sees the keys up to and with d_kv_len[i] - n + j. For each query head
 * h (key head h / (q_heads / kv_heads)):
 *   out[t][h] = sum_s softmax_s(scale * q[t][h] . k[s]) v[s]
 * A token that sees no key gets zeros; keys that a token does not see do not touch its result, whatever they hold. Where it sees a
 * value that is infinite or NaN, that entry of its result is infinite or NaN.
 * q is of the cache's dtype, out of that or VXS_F32 (leading dimensions in elements, multiples of 8, 16-byte
 * aligned, else VXS_ERR_UNSUPPORTED); scale is positive and finite, q_heads a multiple of kv_heads. Sums and softmax
 * statistics are fp32. The weights are rounded for the matrix cores: to the cache's type, for fp32 outputs to 24 bits (bf16 caches)
 * or 22 (fp16). Fp16's range ends this below 2^-21 of a row's largest weight: from there on a weight's error is up to 2^-32 of that
 * largest one, for fp32 outputs up to 2^-44. bf16's does not end within fp32's. Rows outside every sequence are not written; a slot outside
 * the cache has no keys, a length above the table's is cut to it. Asynchronous on the context stream.
 */
VXS_API int vxs_attn_prompt_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                   const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                   const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype);

/*
 * A prefix that groups of rows share (the same voice or instructions): rows [d_off[g], d_off[g + 1]) hold the same
 * pages, or copies of the same entries, for their first d_len[g] tokens. Those are read once for all of them, from the
 * first row's pages, where that is faster than each row's reading its own. d_off int32 [groups + 1] (ascending) and d_len
 * int32 [groups] in device memory; max_len: no d_len is longer. Rows outside every group share nothing.
 */
typedef struct vxs_shared_prefix {
    const int32_t* d_off;
    const int32_t* d_len;
    int32_t groups;
    int32_t max_len;
    uint32_t flags; /* VXS_FLAG_NONE, or VXS_FLAG_SHARE_ALWAYS: also where each row's reading its own is faster */
} vxs_shared_prefix;

/*
 * Attention of one token per sequence: row r's query heads over the first d_kv_len[r] tokens of its slot
 * (d_slots[r]; NULL: slot r), its own among them. Results, types and layouts as vxs_attn_prompt_device; a row of
 * length 0 gets zeros. max_len: no length is longer (the work is divided for it, and for the prefix's: longer
 * or much shorter ones cost time, not correctness). prefix: NULL, or the rows' shared prefixes.
 * A few new tokens of one long sequence can be rows too: the same slot, a length each, their context as a shared prefix.
 *
 * work: device memory of vxs_attn_step_workspace bytes, 16-byte aligned, zeroed once before its first use; calls
 * leave it ready for the next, of whatever sizes and types. One call at a time may use it (calls on one stream are
 * in order). Zero it again after a call whose prefix d_off was not ascending or that the device did not finish.
 * NULL: each row's keys are read by one workgroup per key head, with no sharing.
 * Asynchronous on the context stream; may be captured.
 */
VXS_API int vxs_attn_step_device(vxs_ctx* ctx, int rows, int q_heads, const void* q, int64_t ldq,
                                 const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_kv_len, int max_len,
                                 const vxs_shared_prefix* prefix, float scale, void* out, int64_t ldo, int out_dtype,
                                 void* work, int64_t work_bytes);

/* The workspace of vxs_attn_step_device calls of at most these rows, max_len and prefix lengths (prefix NULL: calls without
 * one) over caches of these head sizes, in bytes; negative: an error code. */
VXS_API int64_t vxs_attn_step_workspace(vxs_ctx* ctx, int rows, int q_heads, const vxs_kv_cache* cache, int max_len,
                                        const vxs_shared_prefix* prefix);

/*
 * Cross attention of packed tokens to another sequence's states (an encoder's): as vxs_attn_prompt_device, but every token
 * [d_q_off[i], d_q_off[i + 1]) sees all d_kv_len[i] tokens of its slot, of which it is none. Both lengths are of any size. One
 * token per sequence, or a few over many states, are a step's rows too: vxs_attn_step_device's see their whole slot. A few tokens
 * of few sequences over long states are faster so, with each sequence a group (d_q_off) that shares all its states (d_kv_len),
 * VXS_FLAG_SHARE_ALWAYS: 4 times 4 tokens over 4000 to 8000 states of head size 128 take 20 us, not 83; 24 times 4 over 1000 to
 * 2000 of head size 64 take 29, not 19.
 */
VXS_API int vxs_attn_cross_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                  const vxs_kv_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                  const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype);

/*
 * Positions of several axes for the rotation of queries and keys (time, height and width of images and video between text):
 * frequency i of vxs_kv_prep turns by the token's position on axis d_axis[i], which is d_pos[d_axis[i] * ld_pos + token].
 * d_axis int32 [rot_dim / 2] in device memory, 16-byte aligned, entries in [0, axes) (one outside counts as the nearest inside);
 * ld_pos at least the call's tokens.
 */
typedef struct vxs_rope_axes {
    const int32_t* d_axis;
    int64_t ld_pos;
    int32_t axes;
} vxs_rope_axes;

/* vxs_kv_append_device with d_pos int32 [axes][ld_pos]; d_index, each token's place in its sequence, is needed with k and v.
 * axes NULL: vxs_kv_append_device. */
VXS_API int vxs_kv_append_axes_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                      int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                      const vxs_rope_axes* axes, const int32_t* d_pos, const int32_t* d_slots,
                                      const int32_t* d_index, const vxs_kv_cache* cache, void* q_out, int64_t ldqo,
                                      int32_t* d_status);

/*
 * One layer's cache in 8 bits: as vxs_kv_cache with entries of one byte (OCP e4m3: 4 significant bits, up to 448 in size) and a
 * scale for each block of 16 tokens and key head, for keys and values apart. Block b of a slot is its tokens 16 b .. 16 b + 15;
 * its scale of head h is the byte (page * kv_heads + h) * (page_size / 16) + (16 b % page_size) / 16 of k_scale, which stands for
 * 2^(byte - 127) (E8M0; 1 to 254), and its entries for e4m3 * 2^(byte - 127). Strides in entries, multiples of 16, k and v
 * 16-byte aligned, k_scale and v_scale 4-byte aligned (else VXS_ERR_UNSUPPORTED). Scales are read in whole aligned 4-byte words: the
 * memory of each array is a multiple of four bytes long, up to three more than pages * kv_heads * page_size / 16.
 * q_dtype: the type of queries, VXS_BF16 or VXS_F16.
 */
typedef struct vxs_kv8_cache {
    void* k;
    void* v;
    uint8_t* k_scale; /* [pages][kv_heads][page_size / 16] */
    uint8_t* v_scale;
    const int32_t* table;
    int64_t ld_table;
    int64_t page_stride;
    int64_t head_stride;
    int64_t token_stride;
    int32_t slots;
    int32_t pages;
    int32_t page_size;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t q_dtype;
} vxs_kv8_cache;

/*
 * vxs_kv_append_device and vxs_kv_append_axes_device (axes NULL: one position a token) for an 8-bit cache; queries go to q_out in
 * q_dtype. A block's scale is the least power of two (from 2^-126) with which none of its finite entries, as they are in fp32
 * after norm and rotation, passes 448; entries are divided by it and rounded once, to nearest even, infinite ones and NaN
 * become NaN. A token at the first place of a block begins it anew: what the block held counts for nothing. Tokens at other
 * places join what is there: where they need a larger scale, the entries at the block's other places are divided by the
 * quotient, a power of two, which changes none but those that fall below 2^-6 of the new scale (rounded to its 2^-9).
 * Tokens of one block in one call are consecutive rows (of two with the same place the later one stays); where they are not,
 * what that block holds after the call is unspecified, as where two slots that share its page append to it.
 */
VXS_API int vxs_kv8_append_device(vxs_ctx* ctx, int tokens, int q_heads, const void* q, int64_t ldq, const void* k,
                                  int64_t ldk, const void* v, int64_t ldv, int in_dtype, const vxs_kv_prep* prep,
                                  const vxs_rope_axes* axes, const int32_t* d_pos, const int32_t* d_slots,
                                  const int32_t* d_index, const vxs_kv8_cache* cache, void* q_out, int64_t ldqo,
                                  int32_t* d_status);

/*
 * vxs_attn_prompt_device, vxs_attn_cross_device, vxs_attn_step_device and vxs_attn_step_workspace over an 8-bit cache: the same
 * but for the cache; q is of its q_dtype, out of that or VXS_F32. Keys and values enter the products as they are (e4m3 has fewer
 * bits than bf16 and fp16), values times their scale; the weights are rounded to 8 significant bits for bf16 outputs, 16 for fp16,
 * 24 for fp32; sums are fp32, whose range ends: outputs may be off by 2^-116 whatever the scales. A NaN entry that a token sees
 * makes its result NaN (a key's: all of it, a value's: that entry). A workspace serves steps over both kinds of cache.
 */
VXS_API int vxs_attn8_prompt_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                    const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                    const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype);
VXS_API int vxs_attn8_cross_device(vxs_ctx* ctx, int seqs, int tokens, int q_heads, const void* q, int64_t ldq,
                                   const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_q_off,
                                   const int32_t* d_kv_len, float scale, void* out, int64_t ldo, int out_dtype);
VXS_API int vxs_attn8_step_device(vxs_ctx* ctx, int rows, int q_heads, const void* q, int64_t ldq,
                                  const vxs_kv8_cache* cache, const int32_t* d_slots, const int32_t* d_kv_len, int max_len,
                                  const vxs_shared_prefix* prefix, float scale, void* out, int64_t ldo, int out_dtype,
                                  void* work, int64_t work_bytes);
VXS_API int64_t vxs_attn8_step_workspace(vxs_ctx* ctx, int rows, int q_heads, const vxs_kv8_cache* cache, int max_len,
                                         const vxs_shared_prefix* prefix);

#ifdef __cplusplus
}
#endif

#endif /* VXS_SAMPLER_H */
