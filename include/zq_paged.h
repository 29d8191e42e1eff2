/*
 * zq_paged.h -- C ABI of the paged KV cache: a pool of pages that many
 * sequences share, the tables that say which pages a sequence has, an append
 * by slot, attention of single query tokens over a sequence's pages, and the
 * choice of the pages that a query attends to.  For callers that serve many
 * sequences with a decoder of their own.  No counterpart in the reference,
 * whose caches hold one sequence.
 *
 * Every call takes device pointers and a hipStream_t (as void*, NULL = the
 * null stream), only enqueues kernels (no allocation, copy or memset: it may be
 * captured into a graph) and never synchronises.  Lengths, tables and counts
 * are read on the device, so a captured step replays while sequences come, grow
 * and go.  Status codes are those of zq_hip.h.  Work runs on the device that
 * holds the cache (or the table).  Equal calls give equal bits.
 *
 * One serving step, for sequences that hold lens[s] tokens and bring counts[s]:
 *   zq_hip_page_tables_step_dev()   pages for the new tokens, their slots
 *   zq_hip_kv_paged_append_dev()    their keys and values into the slots
 *   zq_hip_page_select_dev()        (long contexts) the pages worth reading
 *   zq_hip_attention_paged_dev()    their queries over the rows held
 * after which the caller adds granted[s] to lens[s].
 */
#ifndef ZQ_PAGED_H
#define ZQ_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- page tables -----------------------------------------------------------
 * Token p of sequence s lies in page table[s][p / page_size], at row p %
 * page_size of it: its slot is page * page_size + row.  Entries past a
 * sequence's pages are not used.  free_pages is a stack: free_pages[0 ..
 * *free_count) are the free pages, the next one to be taken last.  seqs is at
 * most 8192, pages 2^24, page_size 16, 32, 64, 128 or 256, width * page_size at
 * most 2^24.  free_pages may be NULL where only attention and selection use the
 * tables.  Numbers of pages outside 0 .. pages - 1 are never followed: a token
 * there gets no slot (-1), and a query sees no rows there (so that -1 stands for
 * pages that were given up). */
typedef struct zq_page_tables {
    int32_t* table;      /* [seqs][width] */
    int32_t* free_pages; /* [pages] */
    size_t seqs;
    size_t width;
    size_t pages;
    size_t page_size;
} zq_page_tables;

/* Room for counts[s] new tokens behind the lens[s] held ones of every sequence.
 * A sequence fits if lens + counts <= width * page_size.  In order of s, each
 * fitting one takes the pages it lacks from the top of the stack; from the first
 * one on for which pages, or the `tokens` rows of the outputs, do not suffice,
 * none is served.  granted[s] is counts[s] or 0 (may be the counts array);
 * start[s] = sum of granted before s (start[seqs]: of all).  The new tokens are
 * packed: row r = start[s] + i of the outputs is token lens[s] + i of s, with
 * its slot, position and sequence; rows from start[seqs] on get -1 in all three.
 * positions and seq_of may be NULL.  table gets the new pages, *free_left what
 * is left of *free_count (may be the same address).  lens are not changed.
 * Lengths and counts below 0 count as 0, a length past the table as its end. */
int zq_hip_page_tables_step_dev(const zq_page_tables* tables, const int32_t* lens, const int32_t* counts,
                                const int32_t* free_count, int32_t* free_left, int32_t* granted, int32_t* start,
                                int64_t* slots, int32_t* positions, int32_t* seq_of, size_t tokens, void* stream);

/* Gives back the pages that sequences of lens[s] tokens do not need for their
 * first keep[s] (0: all of them; lens[s] or more: none), in the order that makes
 * the release of what the last step took its inverse.  table is not changed (its
 * entries past the kept pages are no longer the sequence's); *free_left =
 * *free_count plus the pages given back, at most `pages` (may be the same
 * address).  Entries outside 0 .. pages - 1 (given up before) are left out; a page
 * that stands in several entries comes back as often. */
int zq_hip_page_tables_release_dev(const zq_page_tables* tables, const int32_t* lens, const int32_t* keep,
                                   const int32_t* free_count, int32_t* free_left, void* stream);

/* ---- the cache ---------------------------------------------------------------
 * Nothing needs to start at any value: rows past a sequence's length are never
 * used.  head_dim is 64, 128 or 256, kv_heads at most 1024; k, v and bounds are
 * 16-byte aligned.  bounds and bounds_exp, both or neither: for a page of which
 * rows 0 .. r - 1 are held, with k as held, e is the least exponent in -50 .. 50
 * with max |k| <= 127 * 2^e (50 if there is none, -50 if all are 0), and element d has
 * the bounds floor(min k_d / 2^e) and ceil(max k_d / 2^e), within -127 .. 127.  A
 * NaN among the keys counts as no key there (no key at all: 0 and 0). */
#define ZQ_KV_F32 0
#define ZQ_KV_F16 1
#define ZQ_KV_BF16 2
typedef struct zq_kv_paged {
    void* k; /* [pages][kv_heads][page_size][head_dim] */
    void* v;
    int8_t* bounds;     /* [pages][kv_heads][2][head_dim]: least, greatest; or NULL */
    int8_t* bounds_exp; /* [pages][kv_heads]; or NULL */
    size_t pages;
    size_t kv_heads;
    size_t head_dim;
    size_t page_size;
    int type; /* ZQ_KV_* of k and v */
} zq_kv_paged;

/* Keys and values of `tokens` rows [tokens][stride] fp32 (kv_heads * head_dim
 * used; stride in floats, 0 = kv_heads * head_dim; a multiple of 4, at most 2^31;
 * 16-byte aligned) into slots[r], rounded to the cache's type (to nearest, ties to
 * even; past its range to infinity).  Rows whose slot is outside 0 .. pages *
 * page_size - 1 are not written.  Slots of a call differ.
 * With bounds, those of every page that gets a row are made anew of the page's
 * rows up to the last one written.  A page's rows of one call have to be
 * neighbours in it and ascend, as a step's do: consecutive slots in consecutive
 * rows (of other orders the rows are right and the bounds need not be).
 * At most 2^24 tokens a call, and tokens * kv_heads 2^25. */
int zq_hip_kv_paged_append_dev(const zq_kv_paged* cache, const float* k, const float* v, size_t tokens, size_t stride,
                               const int64_t* slots, void* stream);

/* ---- attention -----------------------------------------------------------------
 * out[i][h] = sum_p softmax_p(scale * q_i . k_p) v_p, h of kv head h / (heads /
 * kv_heads), for `queries` rows q [queries][stride] fp32 (heads * head_dim used;
 * stride as above, 0 = heads * head_dim); out: [queries][heads * head_dim],
 * 16-byte aligned, not overlapping q.
 * Query i belongs to sequence seq_of[i] (NULL: i, queries <= seqs) and sees its
 * first lens[i] + counts[i] rows (counts NULL: lens[i] + 1, its own token the
 * last; with ZQ_ATTN_PAGED_FULL: lens[i] rows; at most width * page_size).  A
 * decode step passes the lens and granted counts of its sequences; prompts and
 * drafted tokens the positions and seq_of of a step, with counts NULL.  A query
 * with counts[i] <= 0 or a seq_of outside 0 .. seqs - 1 is idle: its output is
 * left as it was.  Lengths below 0 count as 0.  One that sees no rows gets 0.
 * select [queries][kv_heads][keep] (NULL: all pages): of every kv head, the
 * pages that the query attends to, by their place in the sequence; of these the
 * first min(keep, pages of the rows seen) entries count, and those outside the
 * pages seen hold nothing.  A page named twice counts twice.  keep is at most 2^20.
 * Scores, exponentials and sums are fp32; q and the softmax weights have 24
 * bits with an fp32 or bf16 cache and 22 with an fp16 one (weights below 2^-17 of
 * the largest are off by 2^-39 of that at most), and the held rows are exact.
 * Before the division by their sum weights go up to 2^14 (fp32 and bf16 caches):
 * values of 2^-14 of fp32's range, all rows of a sequence together, may overflow.
 * NaN and infinities of rows that are not seen do not matter.  A seen key that
 * makes a score of NaN or +infinity gives no numbers in that head's output; one
 * that makes -infinity does too, or the row has no weight.  A seen NaN or infinity
 * of the values gives a NaN or an infinity in its element of the outputs.
 * At most 8192 queries a call and 1024 heads; workspace:
 * zq_hip_attention_paged_workspace_bytes(), 16-byte aligned, of any contents (calls
 * that may run at the same time need one each); with less, the call fails with
 * ZQ_ERR_ARG. */
#define ZQ_ATTN_PAGED_FULL 1
size_t zq_hip_attention_paged_workspace_bytes(const zq_kv_paged* cache, const zq_page_tables* tables, size_t queries,
                                              size_t heads);
int zq_hip_attention_paged_dev(const zq_kv_paged* cache, const zq_page_tables* tables, const float* q, float* out,
                               size_t queries, size_t heads, size_t stride, const int32_t* seq_of, const int32_t* lens,
                               const int32_t* counts, const int32_t* select, size_t keep, float scale, int flags,
                               void* workspace, size_t workspace_bytes, void* stream);

/* ---- selection -------------------------------------------------------------------
 * For every query (as above) and kv head, the pages that it attends to: all of
 * the n that hold the rows it sees, or, of more than `keep`, the `first` first and
 * `recent` last ones (first + recent <= keep) and then those of the largest score,
 * of equal ones the earlier; written in ascending order, -1 behind them.  The score
 * bounds q . k over the page's rows from above, for a query held in 8 bits:
 *   max over the kv head's heads of 2^(eq + e) * sum_d max(c_d * least_d, c_d * greatest_d)
 * with eq the least exponent in -50 .. 50 with max |q| <= 127 * 2^eq and c_d = q_d /
 * 2^eq rounded to the nearest whole number (ties to even; a NaN counts as 0).
 * Scores are whole numbers below 2^23 times a power of two, so the choice does
 * not depend on an order of summation.  Pages outside the pool score lowest.  Idle queries'
 * entries are left as they were.  For scale > 0. */
size_t zq_hip_page_select_workspace_bytes(const zq_kv_paged* cache, const zq_page_tables* tables, size_t queries,
                                          size_t heads, size_t keep);
int zq_hip_page_select_dev(const zq_kv_paged* cache, const zq_page_tables* tables, const float* q, int32_t* select,
                           size_t queries, size_t heads, size_t stride, const int32_t* seq_of, const int32_t* lens,
                           const int32_t* counts, size_t keep, size_t recent, size_t first, int flags, void* workspace,
                           size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ZQ_PAGED_H */
