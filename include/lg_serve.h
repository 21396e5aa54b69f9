/* lg_serve.h -- operators of a decode step of many requests: block tables and cache slots, a paged K / V cache, attention over it,
 * and sampling.  The calls take device pointers, enqueue on the caller's stream, allocate nothing, keep nothing from one call to
 * the next and wait for nothing; they can be captured into a graph, which reads lengths, tables and parameters when it runs.
 * They have no counterpart in the reference, whose sessions hold one sequence.
 *
 * A call returns 0, or a negative code with a message on stderr and nothing enqueued: -1 bad arguments (out of range, a NULL or
 * misaligned pointer, one that is not device memory, pointers of two devices), -2 sizes that the kernels do not hold, -3 a workspace
 * that is too small, -6 the launch failed.  The work runs on the device that holds the memory, whichever device is current; the
 * stream (a cudaStream_t, or NULL) belongs to that device.  What only the device can see -- page ids, slots, lengths, row starts -- is
 * checked by the kernels: a bad value is left out as the call describes it and raises a bit in the cache's status word.
 */
#ifndef LG_SERVE_H
#define LG_SERVE_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

struct model;
struct kvcache;

/* Bits of the status word: a request that was not served for want of pages, of columns in the block table, of rows in the
 * step's outputs; a page id or a length outside the cache; a slot outside the cache; rows of a request that an attention call does
 * not cover. */
enum { LG_PAGED_NO_PAGES = 1, LG_PAGED_TOO_LONG = 2, LG_PAGED_NO_ROWS = 4, LG_PAGED_BAD_PAGE = 8, LG_PAGED_BAD_SLOT = 16, LG_PAGED_BAD_ROWS = 32 };

#define LG_PAGED_MAX_REQ 8192          /* requests of one step */
#define LG_PAGED_MAX_NEW 8             /* new tokens of a request in one attention call: the widest verify block */

/* A cache of many requests in pages of page_size rows.  The caller owns all of it.  Element (page, row, head, d) of k is
 * k[page * page_stride + row * row_stride + head * head_stride + d], the same for v: rows or heads may come first, and k and v may
 * lie in one array.  Strides are in elements and multiples of 8, as head_dim is (at most 512); k and v are 16-byte aligned; a request has
 * at most 2^30 rows (max_pages * page_size), the cache at most 2^31 - 1. */
struct lg_paged_cache {
    void *k, *v;
    long long page_stride, row_stride, head_stride;
    int type;                          /* of k and v: 0 f32, 1 f16, 30 bf16 */
    int n_pages, page_size, n_kv_heads, head_dim;
    int max_req, max_pages, table_stride;
    int *table;                        /* [max_req][table_stride >= max_pages]: page ids of each request, in the order of its rows */
    int *len;                          /* [max_req]: rows that each request has */
    int *free_pages, *n_free;          /* stack of free page ids, n_pages entries, and its height; NULL: no steps */
    int *status;                       /* or NULL; the caller clears it */
};

/* Where the kernels look for a row of a page and a head: elements from the beginning of k (or v), -1 where the cache has no such row.  Needs no GPU. */
long long lg_debug_paged_place(const struct lg_paged_cache *c, int page, int row, int head);

/* One step of requests 0 .. n_req-1: request r keeps its first d_keep[r] rows (NULL: all of them) and gets d_new[r] new ones behind
 * them.  Pages that this takes come from the top of the stack, in the order of the requests and of their rows; pages that it
 * gives up go back in the opposite order, so that a step which rolls a step back leaves the stack as it was.  Updated: table
 * (-1 behind the last page given back), len, the stack.  Written: d_start [n_req + 1], first new token of each request in the step's token rows; for
 * each row its position, its slot (page * page_size + row in the page) and its request, in d_pos, d_slot, d_req [cap] (each may be
 * NULL; without any of them cap is only the limit below, up to 2^31 - 1), -1 in rows behind the last token.
 * Who is served is settled in this order.  One that would have more than max_pages pages is not.  Then pages, in the order of the requests: the first that
 * needs more than are left is not served, and neither is a later one that needs any (pages given up in a step can be taken from the next on).  Then rows (cap), among those that have their pages: the first
 * whose tokens do not fit is not, and neither is a later one with tokens; pages set aside for such a request stay on the stack and are not offered to
 * another.  A request that is not served stays as it is, with no token in the step and a status bit; one that needs neither is always served.
 * Values of d_keep above len count as len, negative ones as 0.  An entry of the table that is no page goes onto the
 * stack as -1, and whoever takes that has rows without slots.  Tables and outputs do not overlap. */
int  lg_paged_step(const struct lg_paged_cache *c, int n_req, const int *d_keep, const int *d_new, int cap, int *d_start, int *d_pos,
                   int *d_slot, int *d_req, void *stream);

/* Rows into the cache: row i of k and v ([n][n_kv_heads][head_dim], ld_k / ld_v elements from row to row) to slot d_slot[i].  type: 0 f32
 * (rounded to the cache's type, to nearest even) or the cache's own.  Rows with slot -1 are skipped, other slots outside the cache too, with a status
 * bit.  The slots of one call differ from each other. */
int  lg_paged_append(const struct lg_paged_cache *c, const void *d_k, const void *d_v, int type, long long ld_k, long long ld_v, int n,
                     const int *d_slot, void *stream);

/* Attention of the newest rows of requests 0 .. n_req-1 over the cache.  q and out are [n_rows][n_heads][head_dim], ld_q / ld_out elements from row to row,
 * both of one type: 0 f32 or the cache's own.  n_heads is a multiple of n_kv_heads; query head h reads KV head h / (n_heads / n_kv_heads).
 * d_start NULL: request r has rows r * n_new .. of exactly n_new tokens (n_rows = n_req * n_new); otherwise rows d_start[r] .. d_start[r + 1] - 1
 * as lg_paged_step wrote them, at most n_new of them (rows beyond are left as they are, with a status bit), and rows from d_start[n_req] on are left as
 * they are.  The last of a request's m rows is the query at position len - 1, row t the one at len - m + t; it sees the rows at its position and
 * before, with window > 0 the nearest `window` of them.  A query that sees nothing (a length of 0, pages that are not in the cache) gives
 * zeros.  scale 0: 1 / sqrt(head_dim).  What a query does not see does not reach it, inf and NaN included.  V rows that it sees may hold any
 * numbers: inf gives inf, inf of both signs or NaN give NaN, and a mean of large numbers is none larger; such calls take several times as long.  q and the
 * K rows that it sees are finite, below 2^127 where they are f32.
 * Every sum is held in f32 and has an order that the call's sizes and lengths fix: the same call gives the same bits.  The work of a call is cut over all
 * its requests, so a request's answer can have other last bits beside other requests, and a token in a block others than alone.  Products are of
 * 16-bit numbers: an f32 query enters with 22 bits of its row's largest element over an f16 cache, with 24 over others; f32 K and V with 24; the weights with
 * 22 bits over f16 and 24 over others, but 16 for bf16 answers.  f32 answers are 1e-7 to 7e-7 of their norm off 64-bit ones, as 32-bit sums are; 16-bit
 * answers are off by their rounding.
 * d_work: lg_paged_attn_work bytes, 16-byte aligned, this call's alone until the call's work has ended: calls and graphs that may
 * overlap have workspaces of their own. */
long long lg_paged_attn_work(const struct lg_paged_cache *c, int n_req, int n_new, int n_heads);
int  lg_paged_attn(const struct lg_paged_cache *c, const void *d_q, int type, long long ld_q, int n_req, int n_new, int n_rows, const int *d_start,
                   int n_heads, float scale, int window, void *d_out, long long ld_out, void *d_work, long long work_bytes, void *stream);

/* One token from each row of logits ([rows][vocab], ld elements from row to row; type 0 f32, 1 f16, 30 bf16).  Each parameter has
 * one value a row, or is NULL: temperature 1, the others off.
 *   order: larger logits first, the lower index first where they are equal; -inf and NaN are never drawn
 *   weight of a token: exp((logit - largest) / temperature); where the largest is +inf, 1 for those and 0 for the others
 *   top_k  > 0: the first top_k tokens of that order
 *   top_p  < 1: of these the shortest beginning that has top_p of their weight (at least one token)
 *   min_p  > 0: of these the tokens whose weight is at least min_p (at least the first)
 *   the draw: in vocabulary order, the first kept token at which the running weight passes d_u[row] (in [0, 1)) of the kept weight
 * temperature <= 0 or NaN: the first token of the order, as the greedy calls choose.  d_token: the token, -1 where nothing can be drawn; d_prob
 * (or NULL): its share of the kept weight, 0 with -1.  Weights are summed as 64-bit integers of 2^-40 or finer, so a result does not
 * depend on the order of any sum. */
int  lg_sample(const void *d_logits, int type, long long ld, int rows, int vocab, const float *d_temperature, const int *d_top_k,
               const float *d_top_p, const float *d_min_p, const float *d_u, int *d_token, float *d_prob, void *stream);

/* model_forward_next with a drawn token in place of the greedy one: one forward of `token` at `pos`, then a draw from its logits on the device with
 * these parameters (top_k <= 0, top_p >= 1, min_p <= 0: off) and the random number u.  Returns the token; prob (or NULL) receives its
 * probability.  Positions and failures as in model_forward_next. */
int  lg_forward_sample(struct model *m, struct kvcache *kv, int token, int pos, float temperature, int top_k, float top_p, float min_p,
                       float u, float *prob);

#ifdef __cplusplus
}
#endif
#endif /* LG_SERVE_H */
