/*
 * zq_kv.h -- C ABI of the 4-bit KV cache: rows of keys and values held in HBM
 * as Q4_0 values, written by an append, read by an attention over one or many
 * query tokens a sequence, and evicted by the attention weight they have
 * drawn.  The decoder of zq_model.h runs on it after zq_model_set_kv_cache().
 * No counterpart in the reference, whose caches are fp32.
 *
 * Every call takes device pointers and a hipStream_t (as void*, NULL = the
 * null stream), only enqueues kernels (no allocation, copy or memset: it may be
 * captured into a graph) and never synchronises.  Lengths are read on the
 * device, so a captured step replays while the cache grows.  Status codes are
 * those of zq_hip.h.  Work runs on the device that holds the cache.
 *
 * One row is one token of one kv head: head_dim / 32 blocks of 32 elements with
 * an fp16 scale d each, value = (code - 8) * d, byte j of a block's 16 bytes =
 * elements j (low nibble) and j + 16 (high), as in a Q4_0 weight block; the
 * scales lie in planes of their own.  Scales carry 8 significant bits and
 * |d| <= 4096, so every value is exact in fp16.
 */
#ifndef ZQ_KV_H
#define ZQ_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The arrays of one cache.  The caller owns them; nothing needs to start at any
 * value: rows past a sequence's length are never used.  capacity is a multiple
 * of 32 (at most 2^24), head_dim 64, 128 or 256, seqs * kv_heads at most 2^20; k, v,
 * k_scale and v_scale are 16-byte aligned.  One call takes at most 2^25 (sequence,
 * token, head) rows. */
typedef struct zq_kv_q4 {
    uint8_t* k;        /* [seqs][kv_heads][capacity][head_dim / 2] codes */
    uint8_t* v;
    uint16_t* k_scale; /* [seqs][kv_heads][head_dim / 32][capacity] fp16 */
    uint16_t* v_scale;
    float* weight;     /* [seqs][kv_heads][capacity] attention weight drawn, or NULL */
    int32_t* pos;      /* [seqs][kv_heads][capacity] positions of the rows' tokens, or NULL */
    size_t seqs;
    size_t kv_heads;
    size_t head_dim;
    size_t capacity;
} zq_kv_q4;

/* Bytes that one sequence's rows take for `capacity` slots (k, v and their
 * scales, without weight and pos); 0 for a shape the cache does not take. */
size_t zq_kv_q4_bytes(size_t kv_heads, size_t head_dim, size_t capacity);

/* ---- append --------------------------------------------------------------
 * Quantises the new tokens' keys and values into slots lens[s] ... of every
 * sequence.  k and v: [seqs][tokens][stride] fp32, kv_heads * head_dim used
 * (stride in floats, 0 = kv_heads * head_dim; a multiple of 4, 16-byte aligned:
 * columns of a packed Q|K|V output will do).  lens [seqs]: rows held before the
 * call.  counts [seqs] (NULL: tokens): how many of a sequence's tokens are real;
 * the others, and tokens past the capacity, are not written.  pos gets
 * first_pos[s] + t (NULL: lens[s] + t) and weight 0, where the cache has them.
 * A sequence of negative length gets nothing, as one that is full.
 * A block's scale is d = fp16(bf16(m / -8)) of its element m of largest
 * magnitude (the first of equals), at most 4096 in magnitude; the code is the
 * nearest to x / d (ties to even) in -8 .. 7, plus 8.  A token whose key or
 * value holds a NaN or an infinity is held as NaN keys and zero values, so that
 * the queries that see it give NaN and no others do. */
int zq_hip_kv_q4_append_dev(const zq_kv_q4* cache, const float* k, const float* v, size_t tokens, size_t stride,
                            const int32_t* lens, const int32_t* counts, const int32_t* first_pos, void* stream);

/* Rows first[s] ... first[s] + counts[s] (NULL: tokens) of every sequence as
 * fp32, [seqs][tokens][kv_heads * head_dim], 16-byte aligned; k or v may be NULL.
 * Rows past the count or the capacity are left as they were. */
int zq_hip_kv_q4_read_dev(const zq_kv_q4* cache, float* k, float* v, size_t tokens, const int32_t* first,
                          const int32_t* counts, void* stream);

/* ---- attention -----------------------------------------------------------
 * out[s][t][h] = sum_p softmax_p(scale * q . k_p) v_p, h of kv head h / (heads /
 * kv_heads).  The held values are exact operands, q has 22 bits, scores, exponentials
 * and sums are fp32: over n rows an output is off by at most (n / 2 + 128) * 2^-24 of
 * the largest |v|, and by what 2^-21 of the largest sum of |scale q k| moves the
 * softmax.  Nearly all calls are far below the first term: it needs rows of equal
 * weight, and so many queries that the rows are not split over workgroups (1,000,003
 * equal rows: 4e-4 of the largest |v| with 512 tokens of 4 heads a kv head at head_dim
 * 64, 1.2e-3 with 2048 tokens at 256, 2e-7 with one token; of unequal weight: 7e-7 at
 * most).  q: [seqs][tokens]
 * [stride] fp32, heads * head_dim used (stride as above, 0 = heads * head_dim); out:
 * [seqs][tokens][heads * head_dim], 16-byte aligned, not overlapping q.  lens and counts
 * as in the append that came before: query t sees the slots below lens[s] + t +
 * 1, its own token's row the last.  With ZQ_ATTN_Q4_FULL every query sees the
 * lens[s] held rows and no others; where there are none its output is 0.  A length
 * below 0 counts as 0, one past the capacity as the capacity.  Outputs
 * of tokens past a sequence's count are left as they were.
 * ZQ_ATTN_Q4_WEIGHTS: weight[s][kv head][p] of every row that a query of the call
 * sees becomes the sum over the queries and the kv head's heads of their softmax
 * weights; with ZQ_ATTN_Q4_ADD as well, that is added to it.
 * workspace: zq_hip_attention_q4_workspace_bytes() bytes, 16-byte aligned, of any
 * contents (calls that may run at the same time need one each); with less, the
 * call fails with ZQ_ERR_ARG. */
#define ZQ_ATTN_Q4_FULL 1
#define ZQ_ATTN_Q4_WEIGHTS 2
#define ZQ_ATTN_Q4_ADD 4
size_t zq_hip_attention_q4_workspace_bytes(const zq_kv_q4* cache, size_t tokens, size_t heads, int flags);
int zq_hip_attention_q4_dev(const zq_kv_q4* cache, const float* q, float* out, size_t tokens, size_t heads,
                            size_t stride, const int32_t* lens, const int32_t* counts, float scale, int flags,
                            void* workspace, size_t workspace_bytes, void* stream);

/* ---- eviction ------------------------------------------------------------
 * Keeps min(lens[s], keep) rows of every (sequence, kv head): first those whose
 * pos is at least next_pos[s] - recent (next_pos NULL: lens[s]) or in 0 ... first -
 * 1, then those of the largest weight (a NaN counts as the lowest); of equal ones
 * those in the lower slots.  first + recent <= keep.  Kept rows in slots below the
 * new length stay where they are; the free slots there, in order, take the kept
 * rows from above it, in order, with their weight and pos (no order of the slots
 * is needed: attention does not depend on it).  Sequences then hold min(lens[s],
 * keep) rows; the caller keeps lens.
 * dst NULL (or of the same arrays): in place, and the slots from the new length to
 * the old get weight -inf and pos -1.  Otherwise the rows go to the same slots of
 * dst (on the same device; the cache's seqs, kv_heads and head_dim; a capacity of at
 * least keep or the cache's; no array shared) and the cache stays as it is.  Both need
 * weight and pos.  Lengths count as in the attention.  At most 2^30 kept rows in all
 * (seqs * kv_heads * keep), else ZQ_ERR_ARG.
 * workspace: zq_hip_kv_q4_evict_workspace_bytes(), 16-byte aligned. */
size_t zq_hip_kv_q4_evict_workspace_bytes(const zq_kv_q4* cache, size_t keep);
int zq_hip_kv_q4_evict_dev(const zq_kv_q4* cache, const zq_kv_q4* dst, const int32_t* lens, size_t keep, size_t recent,
                           size_t first, const int32_t* next_pos, void* workspace, size_t workspace_bytes,
                           void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ZQ_KV_H */
