/*
 * qf_attn.h -- the key/value cache of a layer's sequences and the attention of
 * their newest rows over it: what fork rows (up to 64 drafted tokens of one
 * sequence, a tree or a chain; one decoded token is a tree of one) need beside
 * the MoE layer that runs the same rows (qf_moe.h). No counterpart in the
 * reference's MoE path: entry points and layouts are this library's own.
 *
 * Cache rows are quantised as they are written, per token and head:
 *   amax = max_d |v[d]|,  s = amax * (1 / 127) (E4M3: amax * (1 / 448)), 1 where that is 0
 *   INT8 code = rint(v / s) clamped to +-127,  E4M3 code = e4m3(v / s) clamped to +-448
 *   (fp32 operations, ties to even; the scale by the rule of qf8_i8_x8);  value = code * s
 * A row that holds a NaN or an infinity is stored as codes 0 with s = NaN: it
 * reads back as NaN, and a query that sees it gets NaN.
 *
 * Conventions as in qf_moe.h: asynchronous, stream-ordered, no allocation, no
 * host synchronisation, graph-capturable; 0 on success, -1 for a rejected
 * argument (nothing launched), -3 for a launch error; messages through
 * qfm_last_error(). Launches go to the current device, where every buffer has
 * to be. Indices that live in device memory (sequences, positions, pages) are
 * checked by the kernels, which pass over what is out of range.
 */
#ifndef QF_ATTN_H
#define QF_ATTN_H
#include "qf_moe.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

#define QFM_KV_INT8 0
#define QFM_KV_E4M3 1
/* element types of rows */
#define QFM_DT_F32  0
#define QFM_DT_BF16 1
#define QFM_DT_F16  2

/* A layer's pool of pages. page: tokens a page, 16, 32, 64, 128 or 256;
 * head_dim D: 64, 128 or 256; kv_heads up to 1024.
 *   k  codes [n_pages][kv_heads][page][D]
 *   v  codes [n_pages][kv_heads][page / 4][D][4]: four tokens of one channel
 *      side by side, so that attention's second product, whose inner dimension
 *      is the tokens, loads its operand as it lies
 *   ks, vs  fp32 scales [n_pages][kv_heads][page]
 * k, v, ks and vs 16-byte aligned. Pages need no initialisation. */
typedef struct {
    void  *k, *v;
    float *ks, *vs;
    int    n_pages, page, kv_heads, head_dim, fmt;
} qfm_kv_cache;

/* The sequences' pages: position p of sequence s lies in page
 * table[s][p / page] (device, int32 [n_seq][max_pages]) at token p % page. A
 * page id outside [0, n_pages) is no page: rows there are neither written nor
 * read, and attention does not see them. Up to 65535 sequences. */
typedef struct {
    const int *table;
    int        n_seq, max_pages;
} qfm_kv_seqs;

/* T rows of keys and values (k and v: element (t, h, d) at t * row_stride +
 * h * head_stride + d, type dtype) into positions pos[t] of the sequences
 * seq[t] (device int32 [T]). Strides are multiples of 8 and not negative, k and
 * v 16-byte aligned, T up to 2^24. A row whose sequence, position or page does not exist
 * (pos -1, say) is passed over. Rows of one call name different places: of two
 * that name the same one, codes and scale may be from either. */
int qfm_kv_write(const qfm_kv_cache *c, const qfm_kv_seqs *sq, const void *k, const void *v, int dtype,
                 long row_stride, long head_stride, const int *seq, const int *pos, int T, hipStream_t s);

/* The same rows back as values (code * scale, rounded once to dtype) into k
 * and v, either of which may be NULL. Strides as above and at least D. A row
 * that does not exist is left as it was. */
int qfm_kv_read(const qfm_kv_cache *c, const qfm_kv_seqs *sq, void *k, void *v, int dtype, long row_stride,
                long head_stride, const int *seq, const int *pos, int T, hipStream_t s);

/* Attention of the newest rows of every sequence over its cached keys and
 * values. Sequence s has the rows row_start[s] .. row_start[s + 1] - 1 of q
 * (device int32 [n_seq + 1], ascending, at most max_nodes <= 64 a sequence) and
 * ctx[s] tokens before them; its row i, node i of a tree of drafted tokens,
 * lies at position ctx[s] + i of the cache, written there before this call.
 * Row i sees every position below ctx[s], and node j of its own sequence where
 * bit j of tree[row_start[s] + i] is set (its ancestors and, as a rule, itself);
 * tree NULL: the nodes are a chain, row i sees nodes 0..i. One decoded token
 * is max_nodes 1, its mask 1 or NULL.
 *   out(t, h) = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q(t, h) . k_j - max)
 * over the positions that row t sees, with the keys and values of head
 * h / (q_heads / kv_heads). A row that sees nothing gets zeros; a row of q that
 * is not finite gets NaN. Of a sequence's positions the first 2^31 - 2^16 are seen. Scores, maxima,
 * sums and results are held in fp32. Q and p times the value's scale enter the
 * products as fp16 scaled by powers of two, the codes exactly: q as one number
 * (F32 rows: two, 22 bits), p as one for BF16 rows and two for F16 and F32.
 *   q, out  element (t, h, d) at t * row_stride + h * head_stride + d, type
 *           dtype; strides multiples of 8 and not negative (out: at least D),
 *           16-byte aligned. Rows of out that no sequence has are left.
 *   T       rows of q, up to 2^22; row_start beyond it is cut there
 *   q_heads a multiple of kv_heads, up to 4096; kv_heads times the blocks of 16
 *           rows that max_nodes q_heads / kv_heads rows make, up to 65535
 *   max_ctx the largest ctx the host expects: it sets how many workgroups the
 *           keys are split over, nothing else (longer ones are right, too). Up to
 *           256 sequences share them by length, so that where the sums of one are
 *           split, and how they round, depends on the others' lengths.
 *   scale   > 0
 *   ws      at least qfm_tree_attn_ws_bytes of the same arguments, 16-byte
 *           aligned, no initialisation; calls that share it must not overlap.
 *           0 bytes: ws may be NULL. */
size_t qfm_tree_attn_ws_bytes(const qfm_kv_cache *c, int n_seq, int T, int q_heads, int max_nodes, int max_ctx);
int    qfm_tree_attn(const qfm_kv_cache *c, const qfm_kv_seqs *sq, const void *q, void *out, int dtype, int q_heads,
                     long q_row_stride, long q_head_stride, long out_row_stride, long out_head_stride,
                     const int *row_start, const int *ctx, const uint64_t *tree, int T, int max_nodes, int max_ctx,
                     float scale, void *ws, size_t ws_bytes, hipStream_t s);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif
#endif
