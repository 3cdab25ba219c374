/* gpann_blocks.h — C-ABI of the block operators of libgpann_hip.so: the route-then-scan path over a KEY/VALUE CACHE whose answer is not the ids of
 * the best rows but their softmax-weighted read-out (attention), its gradients, and the eviction of the rows that no query weighs.
 *
 * A cache sequence is cut into BLOCKS of `block_rows` consecutive rows — the shards of this path.  gpann_blocks_summarize keeps one centroid per block,
 * gpann_blocks_route ranks the blocks of every query row by it (as gpann_router_query_batch ranks shards) and gpann_blocks_attend reads the PROBED
 * blocks only (as gpann_scan_buckets does).  Formulas, for query row t of a sequence with n = kv_len cache rows and m = q_len query rows, key/value head h
 * shared by the G = q_heads / kv_heads query heads of its group, position pos = n - m + t (the query rows are the sequence's last m):
 *
 *   visible    cache row r is visible iff 0 <= r < n and, with GPANN_BLOCKS_CAUSAL, r <= pos
 *   centroid   c[h][j] = mean of the keys of the rows r < n of block j           (binary64 sum, one rounding to binary32)
 *   score      s[t][h][j] = sum_d (sum_{heads of the group} q[t][head][d]) * c[h][j][d]                                   (binary64)
 *   probes     of the blocks that hold a visible row: the first `first`, the last `last`, and the best-scored others up to nprobe in all (equal scores:
 *              lowest block; a NaN score ranks below every number), written in ascending block order, -1 in unused slots
 *   attention  x[r] = scale * <q[t][head], k[h][r]> over the visible rows of the probed blocks;  lse = ln sum_r exp x[r];
 *              out[t][head] = sum_r exp(x[r] - lse) v[h][r].  A row that sees nothing (no probe, n = 0, pos < 0): out = 0, lse = -inf
 *   gradients  p[r] = exp(x[r] - lse);  dp[r] = <dout, v[r]>;  ds[r] = p[r] (dp[r] - <dout, out>);
 *              dq = scale * sum_r ds[r] k[r];  dk[r] = scale * sum_{t, heads} ds q;  dv[r] = sum_{t, heads} p dout      (over the heads of the group)
 *   weight     mass_out[h][r] = mass_in[h][r] + sum_{t, heads of the group} p[r]
 *
 * Conventions: those of gpann.h (status codes, gpann_last_error, nothing throws).  All tensors are DEVICE pointers on `device` and stay the caller's; every
 * call only enqueues work on `stream` (a hipStream_t of `device`, NULL = its default stream) and returns: nothing is synchronised, allocated or kept, so a
 * call may be captured into a graph.  Scratch memory is the caller's `workspace` (gpann_blocks_workspace_bytes; 16-byte aligned, contents undefined before
 * and after): one workspace serves calls that run one after the other; calls that may run AT THE SAME TIME — from two threads, on two streams, two
 * captured graphs — need one each.  The calling thread's current device is left as it was.
 *
 * Rows of a batch beyond q_len[b] are neither read nor written by route and attend (their probes, out and lse stay as they were); gradients are written
 * over the whole tensors, zero where no query reaches.  Cache rows beyond kv_len[b] are never read.  A probe outside the sequence's blocks (negative, too
 * large, not visible) and a page outside [0, n_pages) are skipped; a block probed twice by one row counts once.  What a call writes must not overlap what it
 * reads, but for gpann_blocks_weigh in place.
 *
 * Rounding: logits, sums, softmax statistics and masses are binary32, centroids and scores as above; weights and ds are rounded once to the tensors' type
 * where they enter a matrix product, so in GPANN_BLOCKS_FP16 a weight below 2^-32 of a row's largest counts as 0 in out, one below 2^-40 in dv, and a ds
 * below 2^-25 in dq and dk (scale a loss whose gradients are that small).  A ds that GPANN_BLOCKS_FP16 does not hold (above 65504) costs time, not the
 * result: the sums it enters are done again, row by row.  So are sums that a value which is not finite enters: it reaches the rows and keys that see it
 * and no others.
 *
 * Refused, besides what the arguments' comments say: backward and weigh (of more than one query row) of more than 65535 (sequence, key/value head) pairs or
 * 65535 * 128 query rows; backward of 2^32 - 1 (query row, head) rows; route of fewer than 4 query rows, or over more than 4096 blocks, of more than 65535
 * pairs or 2^22 query rows; any call of more than 2^23 workgroups (GPANN_ERR_UNSUPPORTED). */
#ifndef GPANN_BLOCKS_H
#define GPANN_BLOCKS_H

#include "gpann.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    GPANN_BLOCKS_BF16 = 0, /* element type of q, k, v, out and their gradients */
    GPANN_BLOCKS_FP16 = 1
};

enum {
    GPANN_BLOCKS_CAUSAL = 1 << 0 /* gpann_blocks_layout.flags */
};

enum { /* calls a workspace is meant for (gpann_blocks_workspace_bytes) */
    GPANN_BLOCKS_ROUTE = 1 << 0,
    GPANN_BLOCKS_ATTEND = 1 << 1,
    GPANN_BLOCKS_BACKWARD = 1 << 2,
    GPANN_BLOCKS_WEIGH = 1 << 3,
    GPANN_BLOCKS_EVICT = 1 << 4
};

#define GPANN_BLOCKS_MAX_PROBE 64u    /* probes of a query row are held one per wavefront lane */
#define GPANN_BLOCKS_MAX_BLOCKS 16384u /* blocks of a sequence: ceil(kv_rows / block_rows) */

/* The tensors of a call: q, out, dout, dq are [batch][q_rows][q_heads][head_dim]; k, v, dk, dv are [batch][kv_rows][kv_heads][head_dim] or, with a
 * page table, [n_pages][block_rows][kv_heads][head_dim] — a block is a page.  Strides are in elements, {batch or page, row, head}, the last dimension is
 * contiguous; a gradient has the strides of its tensor and dout those of out.  Strides have to be multiples of 8, at most 2^22 of a row, 2^31 of a head
 * and 2^40 of a batch or page, tensors 16-byte aligned, and a tensor that is written must not overlap itself. */
typedef struct gpann_blocks_layout {
    uint32_t struct_bytes;        /* sizeof(gpann_blocks_layout) of the caller's header */
    int32_t device;
    int32_t dtype;                /* GPANN_BLOCKS_BF16 | GPANN_BLOCKS_FP16 */
    uint32_t flags;
    uint32_t batch;
    uint32_t q_rows;              /* query rows the tensors hold per sequence */
    uint32_t kv_rows;             /* cache rows per sequence: with a page table the most a sequence can have */
    uint32_t q_heads, kv_heads;   /* q_heads a multiple of kv_heads */
    uint32_t head_dim;            /* 64, 96, 128, 192 or 256 */
    uint32_t block_rows;          /* a multiple of 16 up to 256 */
    float scale;                  /* finite, below 2^127; of the logits, usually 1 / sqrt(head_dim) */
    const int32_t* q_len;         /* device [batch], clamped to [0, q_rows]; NULL: q_rows */
    const int32_t* kv_len;        /* device [batch], clamped to [0, kv_rows]; NULL: kv_rows */
    const int32_t* page_table;    /* device [batch][page_stride]: page of every block; NULL: contiguous cache */
    uint32_t page_stride;         /* >= ceil(kv_rows / block_rows) */
    uint32_t n_pages;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
} gpann_blocks_layout;

/* Bytes of workspace that any of `calls` (GPANN_BLOCKS_ROUTE | ...) needs for this layout; 0 where a call needs none (`workspace` may be NULL then; route and
 * evict need none today).  Gradients need the most: they have room for every probe list that the layout allows (8192 rows of 32 heads, 8 key/value heads of 128
 * dimensions, 16 probes: 131 MiB; 131072 rows, 64 probes: 8.3 GiB). */
gpann_status gpann_blocks_workspace_bytes(const gpann_blocks_layout* layout, uint32_t nprobe, uint32_t calls, size_t* out_bytes);

/* Centroids of the blocks that hold one of the last `new_rows` rows of each sequence (0: of all its blocks).  Others stay as they were.
 *   summary   [batch][kv_heads][ceil(kv_rows / block_rows)][head_dim] float32 */
gpann_status gpann_blocks_summarize(const gpann_blocks_layout* layout, const void* k, uint32_t new_rows, float* summary, void* stream);

/* Probes of every query row.  1 <= nprobe <= GPANN_BLOCKS_MAX_PROBE; first + last <= nprobe; with GPANN_BLOCKS_CAUSAL last >= 1 (the centroid of a row's
 * own block may hold rows after it: that block is probed by position, never by score).
 *   probes    [batch][q_rows][kv_heads][nprobe] int32 */
gpann_status gpann_blocks_route(const gpann_blocks_layout* layout, const void* q, const float* summary, uint32_t nprobe, uint32_t first, uint32_t last,
                                int32_t* probes, void* workspace, size_t workspace_bytes, void* stream);

/* Attention over the probed blocks.
 *   out       as q, strides out_stride;  lse  [batch][q_rows][q_heads] float32, natural logarithm (may be NULL) */
gpann_status gpann_blocks_attend(const gpann_blocks_layout* layout, const void* q, const void* k, const void* v, const int32_t* probes, uint32_t nprobe,
                                 void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* Gradients of gpann_blocks_attend, from its out and lse, or this call's part of the gradients of attention that was joined over several calls (other probes,
 * other rows of a longer cache), from the joined out and lse.  <dout, out> is corrected for the rounding of out where the weights' own sum tells it, by 1.25
 * times what that rounding can have come to at most.  Contiguous caches only.  Every sum has one order: results repeat bit for bit. */
gpann_status gpann_blocks_attend_backward(const gpann_blocks_layout* layout, const void* q, const void* k, const void* v, const int32_t* probes,
                                          uint32_t nprobe, const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                                          void* workspace, size_t workspace_bytes, void* stream);

/* Adds the attention weights of this call's query rows to the weights of the cache rows.  Every sum has one order.
 *   lse       of gpann_blocks_attend on the same q, k, probes
 *   mass_in, mass_out   [batch][kv_heads][kv_rows] float32; the same pointer: in place; all of mass_out is written */
gpann_status gpann_blocks_weigh(const gpann_blocks_layout* layout, const void* q, const void* k, const int32_t* probes, uint32_t nprobe, const float* lse,
                                const float* mass_in, float* mass_out, void* workspace, size_t workspace_bytes, void* stream);

/* Keeps min(keep, kv_len) rows of every sequence and head — the first `first`, the last `last` (first + last <= keep), and the heaviest others (equal
 * masses: lowest row; NaN below every number) — and copies them, in cache order, to the front of k_out / v_out: a contiguous cache of `keep` rows whose
 * heads hold rows of their own.  Slots beyond the count stay as they were.  The outputs must not overlap the cache.
 *   mass      [batch][kv_heads][kv_rows] float32
 *   rows      [batch][kv_heads][keep] int32: which rows stayed;  count [batch][kv_heads] int32
 *   k_out, v_out   [batch][keep][kv_heads][head_dim], strides out_kv_stride (elements, multiples of 8); both NULL: select only
 *   mass_out  [batch][kv_heads][keep] float32 (may be NULL) */
gpann_status gpann_blocks_evict(const gpann_blocks_layout* layout, const void* k, const void* v, const float* mass, uint32_t keep, uint32_t first,
                                uint32_t last, int32_t* rows, int32_t* count, void* k_out, void* v_out, const int64_t out_kv_stride[3], float* mass_out,
                                void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GPANN_BLOCKS_H */
