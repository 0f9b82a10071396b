/*
 * Serving operators beside MhcPre for AMD Instinct MI355X (gfx950): C ABI.
 *
 * What a serving step of a model with multi-stream residual blocks calls
 * between MhcPre's hIn and the attention layer's output projection:
 *
 *   mhcQkNormRope        norms of queries and keys per head and their rotary
 *                        positions in one pass, keys and values written into
 *                        the pages of a cache or to tensors;
 *   mhcPagedAttention    attention of one new token per sequence over a paged
 *                        key-value cache;
 *   mhcDraftAttention    attention of several new tokens per sequence: a tree of
 *                        drafted tokens, or a chain (a prompt's chunk);
 *   mhcDraftAccept       the path of a drafted tree that the model's choices confirm;
 *   mhcCacheKeep         the confirmed tokens' keys and values to their places;
 *   mhcSparseAttention   attention of one new token per sequence over the pages that
 *                        a score ranks highest;
 *   mhcCacheBounds       the bounds of every page's keys, which that score reads;
 *   mhcCacheUpdate       a step's page table: keep, fork, reorder, end and
 *                        extend sequences, private copies of shared pages;
 *   mhcCacheCompact      the moves that bring the pages in use to the front;
 *   mhcCacheCopyPages    copies the contents of pages.
 *
 * Every operator has the two phases of mhcPre: a GetWorkspaceSize call
 * validates the tensors on the host, sizes the device workspace and returns an
 * executor bound to the tensors' addresses; the second call enqueues it on a
 * stream and returns without waiting.  An executor may be launched any number
 * of times, captured into a HIP graph, and used from several host threads as
 * long as launches that run at the same time do not share a workspace, which
 * is 256-byte aligned and whose contents need not be preserved.  A workspace
 * of 0 bytes may be NULL.  No launch waits for other launches or workgroups.
 * Status codes are those of mhc_pre.h (mhcPreStatusString names them); no
 * function aborts.
 *
 * A paged cache.  Keys and values live in two tensors [pages, pageSize,
 * kvHeads, d].  A sequence's token t is in slot t % pageSize of page
 * pageTable[row, t / pageSize].  What the host cannot check is checked where
 * it is used: a page number outside [0, pages) is a hole, whose keys no query
 * sees, a length below 0 counts as 0 and one above the table's width *
 * pageSize as that.
 */
#ifndef MHC_SERVE_H
#define MHC_SERVE_H

#include "mhc_pre.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Further element types, with the values of the reference stack's aclDataType. */
#define MHC_DTYPE_INT32 3
#define MHC_DTYPE_INT64 9
#define MHC_DTYPE_DOUBLE 11

/* A tensor over caller-owned device memory with its own order: strides are in
 * elements, that of the last dimension must be 1.  Dimensions of size 1 may
 * have any stride. */
typedef struct mhcStridedTensor {
    void *data;
    int32_t dtype;
    int32_t ndim;
    int64_t dims[MHC_MAX_DIMS];
    int64_t strides[MHC_MAX_DIMS];
} mhcStridedTensor;

typedef struct mhcServeExecutor mhcServeExecutor;

MHC_API int mhcServeExecutorDestroy(mhcServeExecutor *executor);

/*
 * Norms of queries and keys per head, rotary positions, and the cache write.
 * For every row x in R^d of a head of token t, with w the weight of queries or
 * keys (qWeight, kWeight: both given or both NULL, then there is no norm):
 *
 *   y = x * w / sqrt(mean(x^2) + eps)
 *   out = y with each pair (a, b) of its first `rot` values turned:
 *         (a cos - b sin, a sin + b cos) * amplitude,
 *         angle = positions[t] * invFreq[i], pair i < rot/2
 *
 * computed in fp32 and rounded once; the angle is a product in 64 bits, so
 * that positions of any size keep their phase.  Pair i is (i, i + rot/2), or
 * (2i, 2i + 1) with `interleaved`.
 *
 *   q         fp16 | bf16     [T, heads, d]     k, v: same type [T, kvHeads, d]
 *   positions int32 | int64   [T]
 *   invFreq   double          [rot/2], rot even, rot <= d; or NULL: no rotation
 *   qWeight, kWeight  fp32    [d], or both NULL
 *   qOut      type of q       [T, heads, d]
 *   kOut      type of q       [T, kvHeads, d], and no v, slots and caches; or NULL:
 *   slots     int64           [T]: page * pageSize + slot of the token, where its
 *                             keys and values go; negative or beyond the cache:
 *                             nowhere (a batch's padding).  No two tokens share one.
 *   kCache, vCache  type of q [pages, pageSize, kvHeads, d]
 *
 * d is even and at most 1024.  qOut may be q and kOut k (the same memory and
 * order); other overlaps of outputs with inputs are the caller's error.
 */
MHC_API int mhcQkNormRopeGetWorkspaceSize(
    const mhcStridedTensor *q, const mhcStridedTensor *k, const mhcStridedTensor *v,
    const mhcTensor *positions, const mhcTensor *invFreq, const mhcTensor *qWeight,
    const mhcTensor *kWeight, float eps, int32_t interleaved, float amplitude,
    const mhcTensor *slots, const mhcStridedTensor *qOut, const mhcStridedTensor *kOut,
    const mhcStridedTensor *kCache, const mhcStridedTensor *vCache, uint64_t *workspaceSize,
    mhcServeExecutor **executor);

MHC_API int mhcQkNormRope(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                          hipStream_t stream);

/*
 * The inverse frequencies (radians per position) of rotary positions, in host
 * memory: base^(-2i/rot) for i < rot/2, changed for contexts longer than a
 * model was trained on:
 *
 *   MHC_ROTARY_PLAIN       as they are
 *   MHC_ROTARY_LINEAR      divided by `factor`
 *   MHC_ROTARY_BASE        base * factor^(rot/(rot - 2)) in base's place, which
 *                          leaves the fastest pair and divides the slowest by
 *                          `factor` (rot > 2)
 *   MHC_ROTARY_RAMP        pairs that turn more than `high` times in
 *                          `trainedLength` positions as they are, less than `low`
 *                          times divided by `factor`, and in between a mean of
 *                          the two, weighted linearly in the number of turns
 *   MHC_ROTARY_INDEX_RAMP  the same with weights that are linear in the pair's
 *                          index between the (real) indices where the pairs turn
 *                          `high` and `low` times, rounded outward to whole ones
 *                          within [0, rot - 1]
 *
 * low, high and trainedLength are read by the two ramps only (0 < low < high).
 */
#define MHC_ROTARY_PLAIN 0
#define MHC_ROTARY_LINEAR 1
#define MHC_ROTARY_BASE 2
#define MHC_ROTARY_RAMP 3
#define MHC_ROTARY_INDEX_RAMP 4

MHC_API int mhcRotaryFrequencies(int32_t rot, double base, int32_t kind, double factor, double low,
                                 double high, double trainedLength, double *invFreq);

/*
 * Attention of one new token per sequence over a paged cache:
 *
 *   s_t = scale * q . k_t,  t in [max(0, L - window), L)  (window 0: all)
 *   out = sum_t exp(s_t - lse) v_t,  lse = log sum_t exp(s_t)
 *
 * with query head h reading kv head h / (heads / kvHeads), in fp32, out rounded
 * once.  (In fp16 the weights are held in 21 bits, small ones to 2^-39 of the
 * largest.)  A row that sees no key (L = 0, holes only) has out 0 and lse -inf.
 * What a row does not see may be infinite or NaN; an infinite value that it sees
 * is infinite in out.  (So may finite ones in bf16 be whose sum, weighted by exp(s_t -
 * max s), is 2^128 or more.)
 *
 *   q          fp16 | bf16   [B, heads, d]
 *   kCache, vCache  same     [pages, pageSize, kvHeads, d]
 *   pageTable  int32         [B, width]      lengths  int32 [B], the new token included
 *   out        type of q     [B, heads, d]   lse      fp32  [B, heads], or NULL
 *
 * d is one of 32, 64, 80, 96, 112, 128, 160, 192, 256; q, the caches and out
 * are 16-byte aligned with strides (other than the last) of multiples of 8
 * elements; heads is a multiple of kvHeads; B * kvHeads * (width * pageSize / 128
 * + 2) is below 2^31, with kvHeads counted ceil(heads / kvHeads / 32) times where
 * more than 16 query heads share one.  The same call gives the same bits again;
 * how a row's sums are cut depends on the batch's lengths, so that in another batch
 * they may differ in their last bits, by roundings in fp32.
 */
MHC_API int mhcPagedAttentionGetWorkspaceSize(
    const mhcStridedTensor *q, const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
    const mhcTensor *pageTable, const mhcTensor *lengths, float scale, int64_t window,
    const mhcStridedTensor *out, const mhcTensor *lse, uint64_t *workspaceSize,
    mhcServeExecutor **executor);

MHC_API int mhcPagedAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                              hipStream_t stream);

/*
 * Attention of several new tokens per sequence over a paged cache.  Row b's last
 * n = min(max(drafted[b], 0), S, L) of L = lengths[b] cached tokens are new: node
 * i < n is token c + i, c = L - n.  It sees the context, tokens t < c, and of the
 * new tokens itself and its ancestors:
 *
 *   parents given: node i's parent is parents[b, i] where 0 <= parents[b, i] < i;
 *     any other value: it has none and hangs under the context.  Positions are
 *     c + (number of ancestors);
 *   parents NULL: a chain, node i hangs under node i - 1 (a prompt's chunk).
 *
 * With a window w a node at position p sees tokens at positions above p - w only
 * (context token t is at position t).  Then, for the tokens t that node i sees,
 *
 *   s_t = scale * q_i . k_t,  out_i = sum_t exp(s_t - lse_i) v_t,
 *   lse_i = log sum_t exp(s_t)
 *
 * with query head h reading kv head h / (heads / kvHeads), in fp32, out rounded
 * once.  (The weights are held in 16 bits in bf16 and in 22 in fp16, there small
 * ones to 2^-34 of the largest.)  Nodes i >= n, and nodes that see no key, have out
 * 0 and lse -inf.  What a node does not see may be infinite or NaN; an infinite
 * value that it sees is infinite in its output, and finite ones are never.
 *
 *   q          fp16 | bf16   [B, S, heads, d]
 *   kCache, vCache  same     [pages, pageSize, kvHeads, d]
 *   pageTable  int32         [B, width]
 *   lengths    int32         [B], the new tokens included
 *   drafted    int32         [B]
 *   parents    int32         [B, S], S <= 256; or NULL
 *   out        type of q     [B, S, heads, d]   lse      fp32  [B, S, heads], or NULL
 *
 * Sizes, alignments and strides as for mhcPagedAttention; the units of work,
 * B * kvHeads * ceil(S * heads / kvHeads / 32) * (width * pageSize / 32 + 5), are
 * below 2^31.  The same call gives the same bits again; in another batch sums may be
 * cut elsewhere and differ by roundings in fp32.
 */
MHC_API int mhcDraftAttentionGetWorkspaceSize(
    const mhcStridedTensor *q, const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
    const mhcTensor *pageTable, const mhcTensor *lengths, const mhcTensor *drafted,
    const mhcTensor *parents, float scale, int64_t window, const mhcStridedTensor *out,
    const mhcTensor *lse, uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcDraftAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                              hipStream_t stream);

/*
 * What the model confirms of a drafted tree (nodes, parents and n as for
 * mhcDraftAttention, with L = max(lengths[b], 0)).  chosen[b, i] is the token that
 * the model puts behind node i: its likeliest, or one drawn from its distribution
 * (what is accepted then follows that distribution).  The path begins at node 0, the
 * row's last known token, which always stays, and goes on from node i to its first
 * child j < n with tokens[b, j] = chosen[b, i], as long as there is one.
 *
 *   path       int32 [B, S]: the path's nodes, ascending, then -1
 *   accepted   int32 [B]: how many (0 where n = 0)
 *   next       type of tokens [B]: chosen at the path's last node, the row's next
 *              token; -1 where n = 0
 *   newLengths int32 [B]: L - n + accepted, the row's length once mhcCacheKeep has
 *              put the path's tokens behind the context
 *
 *   tokens, chosen  int32 | int64 [B, S], S <= 256; parents int32 [B, S] or NULL (a
 *   chain); drafted, lengths int32 [B]
 */
MHC_API int mhcDraftAcceptGetWorkspaceSize(
    const mhcTensor *tokens, const mhcTensor *parents, const mhcTensor *drafted,
    const mhcTensor *chosen, const mhcTensor *lengths, const mhcTensor *path,
    const mhcTensor *accepted, const mhcTensor *next, const mhcTensor *newLengths,
    uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcDraftAccept(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                           hipStream_t stream);

/*
 * Keys and values of a path's nodes to the places behind the context, in place: with
 * c and n as for mhcDraftAttention and L clamped to the table, token c + path[b, k]
 * goes to place c + k, for k = 0, 1, ... as long as path[b, k] is a node (0 <=
 * path[b, k] < n) above path[b, k - 1].  Where either place is in a hole nothing is
 * moved.  lengths is the one that mhcDraftAttention and mhcDraftAccept were given.
 * Pages that the moves touch must be held by one row only (mhcCacheUpdate sees to
 * that for rows that append).  vCache may be kCache; else they share no element.
 *
 *   kCache, vCache  fp16 | bf16 | fp32 [pages, pageSize, kvHeads, d]
 *   pageTable int32 [B, width]   lengths, drafted int32 [B]   path int32 [B, S], S <= 2^30
 */
MHC_API int mhcCacheKeepGetWorkspaceSize(
    const mhcStridedTensor *kCache, const mhcStridedTensor *vCache, const mhcTensor *pageTable,
    const mhcTensor *lengths, const mhcTensor *drafted, const mhcTensor *path,
    uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcCacheKeep(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                         hipStream_t stream);

/*
 * The smallest and the largest value, per kv head and dimension, of each page's keys:
 * lo, hi [pages, kvHeads, d].  For the pages that hold row b's last
 * min(max(counts[b], 0), tokens, L) tokens (L: lengths[b] clamped to the table), in
 * place:
 *
 *   lo = min over these tokens in the page, and of the old lo if the page also holds
 *   tokens of the row in front of them; hi likewise.
 *
 * So counts = what a step appended keeps the bounds of a growing cache, and counts =
 * L makes them anew.  After tokens were taken away (mhcCacheKeep) the last page's
 * bounds may be wider than need be; counts that reach back to the page's start mend
 * that.  A NaN among the keys, or in the old bounds that count, makes both bounds NaN.
 * -0 is below 0.  No two rows' new tokens lie in one page.
 *
 *   kCache  fp16 | bf16 [pages, pageSize, kvHeads, d]   lo, hi  same [pages, kvHeads, d]
 *   pageTable int32 [B, width]   lengths, counts int32 [B]   tokens >= 0
 *
 * d, alignments and strides as for mhcPagedAttention.  cache_copy_pages copies bounds
 * too: they are caches with pages of one slot.
 */
MHC_API int mhcCacheBoundsGetWorkspaceSize(
    const mhcStridedTensor *kCache, const mhcTensor *pageTable, const mhcTensor *lengths,
    const mhcTensor *counts, int64_t tokens, const mhcStridedTensor *lo,
    const mhcStridedTensor *hi, uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcCacheBounds(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                           hipStream_t stream);

/*
 * Attention of one new token per sequence over `top` pages for each of its kv heads.
 * Row b holds its table's first ceil(L / pageSize) columns (L: lengths[b] clamped to
 * the table); holes are left out.  Of these columns kv head g takes those among the
 * first `first` and the last `last` that are no holes, and of the others those with
 * the highest scores, until it has `top` (or all); of equal scores the lower column.
 * With the query heads h that share g
 *
 *   score = sum_h sum_i max(q_hi lo_i, q_hi hi_i)
 *         = sum_i (sum_h max(q_hi, 0)) hi_i + (sum_h min(q_hi, 0)) lo_i,
 *
 * the largest value that the sum of the heads' products with a key between the bounds
 * lo and hi can have, in 64 bits as the second line has it (with bounds that are
 * infinite a sum of 0 makes NaN); a score that is NaN is above all others.  Over the
 * tokens of these pages
 *
 *   s_t = scale * q . k_t,  out = sum_t exp(s_t - lse) v_t,  lse = log sum_t exp(s_t)
 *
 * as mhcPagedAttention computes it, with its limits, holes and exceptional values.
 *
 *   q          fp16 | bf16   [B, heads, d]
 *   kCache, vCache  same     [pages, pageSize, kvHeads, d]
 *   lo, hi     same          [pages, kvHeads, d], 16-byte aligned rows
 *   pageTable  int32         [B, width]      lengths  int32 [B], the new token included
 *   out        type of q     [B, heads, d]   lse      fp32  [B, heads], or NULL
 *   columns    int32         [B, kvHeads, top]: the columns taken, ascending, then -1
 *
 * 0 <= first, last; first + last <= top; top >= 1; top * pageSize below 2^31; width at
 * most 2^30; B * kvHeads at most 2^20.
 */
MHC_API int mhcSparseAttentionGetWorkspaceSize(
    const mhcStridedTensor *q, const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
    const mhcStridedTensor *lo, const mhcStridedTensor *hi, const mhcTensor *pageTable,
    const mhcTensor *lengths, int64_t top, int64_t first, int64_t last, float scale,
    const mhcStridedTensor *out, const mhcTensor *lse, const mhcTensor *columns,
    uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcSparseAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                               hipStream_t stream);

/*
 * A step's page table.  Row r of the new state goes on from row parents[r] of
 * the old one (r: keep; another row: fork or reorder; outside [0, rows): a new,
 * empty sequence) and then gets counts[r] tokens (clamped to [0, tokens]).
 * There is no other state: a page is free if no row of the new state holds it.
 *
 *   - A row holds its parent's first ceil(length / pageSize) pages, shared with
 *     every other row that holds them.
 *   - A row that appends into a partly filled page that another row holds too
 *     gets a free page in its place: src[r] is the shared page, dst[r] the
 *     private one, whose contents the caller copies (mhcCacheCopyPages); else
 *     both are -1.  Where all rows that hold the page append, all of them get one
 *     and the page itself falls free: a page and a copy more than they need.
 *   - Free pages are given out in ascending order, to rows in ascending order;
 *     within a row first the private copy, then the pages it grows by.
 *   - A row gets what it asked for (granted[r] = counts[r]) or, if the rows up
 *     to it need more pages than are free (and it needs one), or its pages
 *     exceed the table's width, nothing: granted[r] = 0, its state as its
 *     parent's.
 *
 *   pageTable  int32 [rows, width]    lengths  int32 [rows]
 *   parents    int32 [rows]           counts   int32 [rows]
 *   newTable   int32 [rows, width], -1 where no page is held
 *   newLengths int32 [rows]
 *   slots      int64 [rows, tokens]: page * pageSize + slot of each new token, -1
 *              beyond granted[r]
 *   granted, src, dst  int32 [rows]
 *
 * The new state's tensors must not overlap the old one's.  width * pageSize
 * must be below 2^31.
 */
MHC_API int mhcCacheUpdateGetWorkspaceSize(
    const mhcTensor *pageTable, const mhcTensor *lengths, const mhcTensor *parents,
    const mhcTensor *counts, int64_t pages, int64_t pageSize, const mhcTensor *newTable,
    const mhcTensor *newLengths, const mhcTensor *slots, const mhcTensor *granted,
    const mhcTensor *src, const mhcTensor *dst, uint64_t *workspaceSize,
    mhcServeExecutor **executor);

MHC_API int mhcCacheUpdate(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                           hipStream_t stream);

/*
 * Compaction's plan: with U pages held by the rows, the k-th held page >= U
 * moves to the k-th free page < U, so that pages [0, U) are held.
 *
 *   newTable  int32 [rows, width]: the table after the moves, -1 where no page is held
 *   src, dst  int32 [pages / 2]: the moves, in ascending order, then -1
 *   used      int32 [1]: U
 *
 * The caller copies the contents (mhcCacheCopyPages; no page is both a source
 * and a destination).
 */
MHC_API int mhcCacheCompactGetWorkspaceSize(const mhcTensor *pageTable, const mhcTensor *lengths,
                                            int64_t pages, int64_t pageSize,
                                            const mhcTensor *newTable, const mhcTensor *src,
                                            const mhcTensor *dst, const mhcTensor *used,
                                            uint64_t *workspaceSize, mhcServeExecutor **executor);

MHC_API int mhcCacheCompact(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                            hipStream_t stream);

/*
 * Copies page src[i] of both caches to page dst[i], for every i with both in
 * [0, pages).  No page may be a destination twice, or both a source and a
 * destination.  The caches are of any type of 2 bytes or 4 (fp16, bf16, fp32).
 *
 *   kCache, vCache  [pages, pageSize, kvHeads, d]     src, dst  int32 [n]
 */
MHC_API int mhcCacheCopyPagesGetWorkspaceSize(const mhcStridedTensor *kCache,
                                              const mhcStridedTensor *vCache, const mhcTensor *src,
                                              const mhcTensor *dst, uint64_t *workspaceSize,
                                              mhcServeExecutor **executor);

MHC_API int mhcCacheCopyPages(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor,
                              hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MHC_SERVE_H */
