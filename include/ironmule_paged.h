/*
 * ironmule_paged.h — C ABI of the paged KV cache and of beam selection on MI355X (gfx950), in
 * libironmule_qmv.so: requests whose keys and values lie in pages shared out on the device, attention
 * of any number of new tokens per request over them, and the choice of the next tokens of beams.
 *
 * Contract (as for ironmule_qmv.h): device pointers allocated by the caller, work queued on `stream`,
 * no allocation or synchronisation per call, int32 return codes with imq_last_error() for the
 * message.  Nothing is kept between calls; every call can be captured in a HIP graph, and calls that
 * share no memory may run at the same time.
 *
 * A cache of `requests` requests (row r of every array is request r):
 *   tables    int32 (requests, columns): the page of each page_size tokens of a request, -1 none
 *   lengths   int32 (requests): tokens held
 *   refs      int32 (pages): the table entries that hold each page (0: free)
 *   pages     bf16 (pages, kv_heads, page_size, head_dim) per layer for the keys and for the values
 * Only imq_paged_reserve and imq_paged_reorder change tables and refs; the caller adds accepted
 * tokens to the lengths (lengths = ends) between steps.  A page is held by more than one request only
 * after imq_paged_reorder, in the same column of each, and only where tokens are held.
 */
#ifndef IRONMULE_PAGED_H
#define IRONMULE_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "ironmule_qmv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define IMQ_PAGED_MAX_REQUESTS 1024
#define IMQ_PAGED_MAX_COLUMNS (1 << 20)
#define IMQ_PAGED_MAX_ROWS (1 << 20)
#define IMQ_PAGED_MIN_PAGE 16   /* a page holds a power of two tokens */
#define IMQ_PAGED_MAX_PAGE 1024
#define IMQ_PAGED_MAX_HEADS 1024

typedef struct {
  int32_t* tables;
  int32_t* lengths;
  int32_t* refs;
  int32_t requests, columns, pages, page_size;
} imq_paged_cache;

/* What imq_paged_reserve gives the rows of a step, all int32: starts (requests + 1), the rows of
 * request r being starts[r] .. starts[r + 1] - 1; ends (requests), its tokens with the new ones;
 * status (requests); positions and slots (rows), the row's token position and its place
 * page * page_size + offset, both -1 in rows past starts[requests]; copies (requests, 2), the page
 * copied from and to, -1 where none was. */
typedef struct {
  int32_t* starts;
  int32_t* ends;
  int32_t* status;
  int32_t* positions;
  int32_t* slots;
  int32_t* copies;
  int32_t rows;
} imq_paged_chunk;

/* Gives the next counts[r] tokens of every request their pages, rows and slots: tokens lengths[r] ..
 * lengths[r] + counts[r] - 1.  Where a page has to be had, requests in order and a request's pages
 * in order take the lowest-numbered free ones; pages had already (an earlier reservation) are kept.
 * Where the first of these tokens falls into a page that other requests hold too, the request gets
 * a page of its own instead, and if it holds tokens of that page their page is copied in all
 * `planes` planes of `pool` (plane p of page i at pool + (p * pages + i) * page_bytes; pool may be
 * null, then the caller copies).  A request is taken whole or refused: status 0 taken (or no new
 * tokens), 1 not enough pages, 2 malformed (a negative count or length, more tokens than its columns,
 * a shared page past its tokens), 3 not enough rows.  Pages and rows count as asked for by every
 * well-formed request up to it, refused ones too, so the first request that does not fit ends the
 * taking of pages (of rows).  A request that is malformed for a shared page past its tokens (found while
 * the pages are counted) counts like a well-formed one; the other malformed ones ask for nothing.  A refused request keeps its pages and gets no rows; ends[r] = lengths[r].
 * The lengths are not changed.
 * Takes the place of the admission of a request into a KV pool slot (ironmule/dense_plan.py:297-301). */
IMQ_API int32_t imq_paged_reserve(const imq_paged_cache* cache, const int32_t* counts, const imq_paged_chunk* chunk,
                                  void* pool, int32_t planes, int64_t page_bytes, void* stream);

/* Request r becomes a copy of request parents[r] as it was before the call: its tokens' pages are
 * shared, what r held before is given back.  -1: r becomes empty.  A parent that is r itself, or
 * outside -1 .. requests - 1, leaves r as it is.  Serves forks, the reordering of beams and the end
 * of requests. */
IMQ_API int32_t imq_paged_reorder(const imq_paged_cache* cache, const int32_t* parents, void* stream);

/* Per row and head: q and k heads get the per-head RMSNorm (q_norm / k_norm weights of head_dim
 * values, rounded to bf16) and the non-interleaved rotary embedding at positions[row] with base
 * theta; q goes to q_out (rows ldo apart; q itself, or memory of its own), k and the untouched v to the pages at slots[row].
 * q, k, v: rows of heads * head_dim values ldq, ldk, ldv apart.  head_dim 128 or 256.  A row whose
 * slot is outside the pages (padding, a refused request) is left out: nothing is written for it.
 * Slots of one call are distinct.  The paged form of imq_qk_norm_rope. */
IMQ_API int32_t imq_paged_write(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk, const uint16_t* v,
                                int64_t ldv, const uint16_t* q_norm, const uint16_t* k_norm,
                                const int32_t* positions, const int32_t* slots, uint16_t* q_out, int64_t ldo,
                                uint16_t* k_pages, uint16_t* v_pages, int32_t rows, int32_t Hq, int32_t Hkv,
                                int32_t head_dim, int32_t pages, int32_t page_size, double theta, float eps,
                                void* stream);

/* Row i of request r, at position p = ends[r] - (starts[r + 1] - starts[r]) + i, attends over its
 * request's positions max(0, p - window + 1) .. p (window 0: from 0):
 *   out[row][h] = softmax(scale q[row][h] . K[h / (Hq / Hkv)]) V[h / (Hq / Hkv)]
 * with fp32 scores, maxima and sums.  For the product with V a probability is two terms of bf16 (2^-15 of it
 * are lost at most, about as in imq_attention_decode) for a request of up to 32 / (Hq / Hkv) new tokens, and rounded to one
 * (2^-8) where it has more, which are less than imq_prompt_layer keeps; in a batch whose requests have that
 * many on average all have two terms.
 * One token per request is a decode step, many a chunk of a prompt over what is cached already; a
 * batch may mix them.  q and out: `rows` rows, ldq and ldo apart, scale > 0, head_dim 128 or 256.
 * Rows outside every request are left as they were; a row that sees nothing gets zeros.  Keys in a
 * table entry outside 0 .. pages - 1 are left out.  Entries past a row's position are never used,
 * whatever they hold.  Starts ascend; values outside 0 .. rows are taken as the nearest bound.
 * max_context: a bound on `ends` by which the launch is planned (the results do not depend on it
 * beyond the order of sums; the tables' capacity will do).  `workspace`: imq_paged_attention_workspace
 * bytes (may be 0) for the same max_context, 16-byte aligned, no preparation; calls that share one must not
 * overlap.
 * The paged, many-row form of imq_attention_decode (ironmule/dense_plan.py:258-274). */
IMQ_API size_t imq_paged_attention_workspace(int32_t rows, int32_t requests, int32_t Hq, int32_t Hkv, int32_t head_dim,
                                             int32_t max_context, int32_t window);
IMQ_API int32_t imq_paged_attention(const uint16_t* q, int64_t ldq, const uint16_t* k_pages, const uint16_t* v_pages,
                                    const int32_t* tables, const int32_t* starts, const int32_t* ends, uint16_t* out,
                                    int64_t ldo, int32_t rows, int32_t requests, int32_t columns, int32_t pages,
                                    int32_t page_size, int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t max_context,
                                    int32_t window, float scale, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* The `count` best continuations of each group of `beams` beams (rows group * beams ..):
 *   key(b, v) = scores[b] + logits[b][v] - log(sum_u exp(logits[b][u]))      over all b, v of a group
 * compared in double (inside a beam: the logits themselves), ties to the lowest (b, v).  The log sum is good
 * to a few units of 2^-24 whatever the size of the logits, which may be masked with the lowest finite
 * value of their type as well as with -inf.  logits: fp32 or bf16 rows of `vocab` values, ld apart.  `finished` (may be null): a beam with a non-zero flag offers only itself, token eos with
 * its score.  Values that are NaN or -inf, and beams whose score or sum is not finite, offer nothing.
 * Outputs (groups, count), the best first: the key as fp32, the parent row (over all groups), the
 * token, and whether the continuation is finished (its parent was, or the token is eos); where there
 * are fewer continuations -inf, -1, -1, 0.  The workspace needs no preparation. */
#define IMQ_BEAM_MAX_COUNT 64
#define IMQ_BEAM_MAX_BEAMS 64
#define IMQ_BEAM_MAX_GROUPS 4096
IMQ_API size_t imq_beam_select_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t count);
IMQ_API int32_t imq_beam_select(const void* logits, int64_t ld, int32_t dtype, const float* scores,
                                const int32_t* finished, int32_t eos, int32_t groups, int32_t beams, int32_t vocab,
                                int32_t count, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                                int32_t* out_finished, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* IRONMULE_PAGED_H */
