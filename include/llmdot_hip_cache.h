/*
 * llmdot_hip_cache.h -- operators over device memory for serving loops: a
 * quantised KV cache, attention over it, and the verification of drafted tokens.
 *
 * The conventions of llmdot_hip.h hold (status codes, llmdot_hip_last_error, no
 * C++ exception crosses the ABI).  Besides them:
 *   - `_dev` pointers are HBM addresses on the context's device.  Float arrays
 *     are 16-byte aligned (LLMDOT_E_INVALID otherwise).
 *   - Calls enqueue kernels on the context's stream and return; they allocate
 *     nothing, copy nothing and record no memset, so they can be captured into
 *     a HIP graph on that stream and replayed with new contents of their
 *     arrays.  Work on other streams is ordered by the caller
 *     (llmdot_hip_stream).
 *   - What the host can see is checked before anything is enqueued.  Slots,
 *     positions, counts and token ids live in HBM and are checked by the
 *     kernels: nothing outside the cache or the arrays is read or written.
 *   - A workspace belongs to one call until that call's kernels have run: calls
 *     in the order of one stream may share it, graphs replayed at the same time
 *     may not.  It is zeroed once before its first call (llmdot_hip_device_alloc
 *     does that); every call leaves it fit for the next, whatever its sizes and
 *     whichever of these operators it is for.
 *   - No counterpart in the reference, whose cache is fp32 and whose loop holds
 *     one sequence (src/Llmdot.Core/Inference/KvCache.cs).
 */
#ifndef LLMDOT_HIP_CACHE_H
#define LLMDOT_HIP_CACHE_H

#include "llmdot_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The context's hipStream_t, for events, capture and copies of the caller's own. */
int32_t llmdot_hip_stream(llmdot_hip_ctx* ctx, void** stream);

/* ---- quantised KV cache ---------------------------------------------------
 * `slots` sequences of `capacity` positions, kv_heads x head_dim keys and as
 * many values each, in blocks of 32 along head_dim: Q8_0 or Q4_0 with the
 * integers and fp16 scales that llmdot_hip_quantize gives for the same row
 * (a scale past fp16's largest is held as the largest, and a NaN as 0, so
 * that no hidden position can reach a result).  head_dim is 64, 96, 128 or 256
 * (LLMDOT_E_UNSUPPORTED otherwise).  A new cache reads as zeros. */
typedef struct llmdot_hip_kv_cache llmdot_hip_kv_cache;
typedef struct llmdot_hip_kv_cache_desc {
    int32_t slots, kv_heads, head_dim, capacity;
    uint32_t k_type, v_type;     /* ggml types: Q8_0 = 8 or Q4_0 = 2 */
} llmdot_hip_kv_cache_desc;
int32_t llmdot_hip_kv_cache_create(llmdot_hip_ctx* ctx, const llmdot_hip_kv_cache_desc* desc,
                                   llmdot_hip_kv_cache** out);
/* Waits for the context's stream.  The context outlives its caches as it does its models. */
int32_t llmdot_hip_kv_cache_destroy(llmdot_hip_kv_cache* cache);

/* The tokens of one call: sequence b's are positions starts[b] ..
 * starts[b] + counts[b] - 1 of slot slots[b], and rows b * tokens .. of the
 * call's arrays.  Rows past a sequence's count, of a slot outside the cache or
 * at positions outside [0, capacity) are neither read nor written. */
typedef struct llmdot_hip_token_batch {
    int32_t batch;               /* sequences (at most 4096) */
    int32_t tokens;              /* rows per sequence */
    const int32_t* slots_dev;    /* [batch] */
    const int32_t* starts_dev;   /* [batch] */
    const int32_t* counts_dev;   /* [batch], values past `tokens` count as tokens; NULL: tokens each */
} llmdot_hip_token_batch;

/* Quantises the rows k_dev, v_dev [batch * tokens][kv_heads * head_dim] into
 * the cache.  Strides are floats from row to row (0: packed; multiples of 4).
 * Where two sequences of a call name the same position of the same slot, the
 * later one's row is kept. */
int32_t llmdot_hip_kv_cache_write(llmdot_hip_kv_cache* cache, const float* k_dev, int64_t k_stride,
                                  const float* v_dev, int64_t v_stride, const llmdot_hip_token_batch* rows);
/* The values the cache holds at those positions, as fp32 (scale x integer, exact). */
int32_t llmdot_hip_kv_cache_read(llmdot_hip_kv_cache* cache, float* k_dev, int64_t k_stride, float* v_dev,
                                 int64_t v_stride, const llmdot_hip_token_batch* rows);

/* Attention of the call's tokens, whose own rows are already in the cache.
 * Token i of sequence b attends to the prefix, then to positions 0 ..
 * starts[b] + i of its slot:
 *   out = sum_t softmax_t(scale q . k_t) v_t
 * per query head, heads / kv_heads of them to a kv head.  With a prefix, rows
 * 0 .. prefix_len - 1 of one slot of `prefix` (the same cache or another of
 * the same context, shape and types) come before every sequence's own and are
 * read once for all of them; a slot's position p then stands at prefix_len + p.
 * window > 0 keeps the last `window` positions, the token's own included.
 * fp32 results: scores, softmax statistics and sums are held in 32 bits,
 * probabilities and queries enter the products with 22-bit significands. */
typedef struct llmdot_hip_attention {
    int32_t heads;               /* a multiple of kv_heads */
    int32_t window;              /* 0: every earlier position */
    float scale;                 /* 0: 1 / sqrt(head_dim); at most 2e38 */
    const llmdot_hip_kv_cache* prefix;   /* NULL: none */
    int32_t prefix_slot, prefix_len;
    int64_t q_stride, out_stride;        /* as above */
} llmdot_hip_attention;
int32_t llmdot_hip_kv_cache_attention(llmdot_hip_kv_cache* cache, const float* q_dev, float* out_dev,
                                      const llmdot_hip_token_batch* rows, const llmdot_hip_attention* opt,
                                      void* workspace_dev, size_t workspace_bytes);
/* Bytes that suffice for such a call, with or without a prefix of any length. */
int32_t llmdot_hip_kv_cache_attention_workspace(const llmdot_hip_kv_cache* cache, int32_t heads, int32_t batch,
                                                int32_t tokens, int32_t has_prefix, size_t* bytes);

/* ---- verification of drafted tokens ---------------------------------------
 * Speculative sampling for `batch` sequences of up to `drafts` drafted tokens.
 * target_dev [batch][drafts + 1][vocab]: the target model's logits before each
 * draft and after the last; draft_dev [batch][drafts][vocab]: the draft model's
 * (NULL: drafts that came with certainty, as from a lookup); p = softmax(target
 * / temperature), q = softmax(draft / temperature), in 64 bits.  counts_dev
 * [batch]: each sequence's drafts (NULL: all).
 *   Draft i stands if uniforms[b][i] q(d_i) < p(d_i); accepted_dev[b] counts
 *   the leading ones that do.  The next token is drawn with
 *   uniforms[b][drafts] from max(p - q, 0) at the first that does not (from p
 *   if that leaves nothing), else from p after the last: the first token whose
 *   cumulative mass exceeds the draw.
 *   temperature <= 0: a draft stands if it is the first maximum of its row, and
 *   the next token is the row's first maximum.
 * tokens_dev [batch][drafts + 1]: the standing drafts, the next token, then -1.
 * NaN logits have no mass (a row with no mass gives no token: -1), +infinity
 * takes all of it, and drafted ids outside the vocabulary do not stand.  The
 * sampler's top_k, top_p and repeat penalty have no part in this. */
int32_t llmdot_hip_verify_drafts(llmdot_hip_ctx* ctx, const float* target_dev, const float* draft_dev,
                                 const int32_t* drafts_dev, const int32_t* counts_dev, const float* uniforms_dev,
                                 int32_t batch, int32_t drafts, int32_t vocab, float temperature,
                                 int32_t* tokens_dev, int32_t* accepted_dev, void* workspace_dev,
                                 size_t workspace_bytes);
int32_t llmdot_hip_verify_drafts_workspace(llmdot_hip_ctx* ctx, int32_t batch, int32_t drafts, int32_t vocab,
                                           size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif
