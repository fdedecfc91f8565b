/*
 * apus_attn_gcuda.h — attention over batches of sequences (sm_100a): a 4-bit
 * key/value cache (written, read back, attended to) and causal prompt
 * attention over packed sequences.  No counterpart in the reference, whose
 * attention keeps one sequence's BF16 rows (c/gdsa.h:451-517, :612-626).
 *
 * Rules of every entry point here:
 *   - Device pointers, a cudaStream_t passed as void*, the current device.
 *     0 on success; -1 with the reason in apus_gcuda_last_error().  Bad
 *     arguments are refused before anything is launched; where a launch itself
 *     fails, the outputs are not complete.
 *   - No allocation, no synchronisation, no state kept between calls: every
 *     entry can be captured into a CUDA graph, and calls on different streams
 *     may overlap as long as their outputs and workspaces do not.
 *   - Scales are positive and finite; head dims are 64, 128 or 256.
 *   - The structs are read during the call; the device arrays they point to
 *     are read by the kernels, so they must live until those have run.
 *   - What the host cannot see is checked on the device: a page id, a length
 *     or a row range that is out of bounds is never followed.  It is left out
 *     (below, at each entry) and reported by apus_gcuda_kernel_error():
 *     41 page id, 42 length or row range (43: a wait inside a kernel gave up,
 *     and that call's outputs are incomplete).
 */
#ifndef APUS_ATTN_GCUDA_H
#define APUS_ATTN_GCUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* BF16 codes of rows of heads: dim d of head h of row r is
 * p[r * row_stride + h * head_stride + d].  Strides in elements, multiples of
 * 8; p 16-byte aligned.  Rows or heads may be the outer axis, and keys and
 * values may lie interleaved; an output's rows and heads must not overlap. */
typedef struct {
    uint16_t *p;
    size_t rows, heads;
    size_t row_stride, head_stride;
} ApusHeadRows;

/* ---- the 4-bit cache ----------------------------------------------------- */

#define APUS_KV4_PAGE 64     /* positions of a page */
#define APUS_KV4_GROUP 32    /* neighbouring dims that share a scale */

/* Pages of `heads` key/value heads of `dim` (64, 128 or 256) dims:
 * [num_pages][heads][72 * dim] bytes, 16-byte aligned.  A head's block holds
 * the key codes [64][dim / 2], the value codes [64][dim / 2], the key scales
 * [64][dim / 32] and the value scales [64][dim / 32] (BF16).
 *
 * A group of 32 dims has the scale s = bf16(amax / 7); a code is
 * clamp(rint(x / s), -7, 7) + 8 and stands for (code - 8) * s.  So a held
 * value is off by at most s / 2 (where the rounding of s makes 7 s smaller
 * than amax, by at most amax / 256 more).  A group whose scale rounds to 0
 * holds zeros; a group with a NaN or an infinity holds NaN (s = NaN).
 *
 * Where a code stands (32-bit words of a position's row, eight codes each,
 * code i of a word in bits 4i .. 4i + 3; p the position in the page,
 * j = d / 32):
 *   keys, word of dim d, code d % 8, with q = d % 32 / 8:
 *     dim 64:  2 q + j         dim 128: 4 q + j
 *     dim 256: 16 ((j / 4) ^ (p / 4 % 2)) + 4 q + j % 4
 *   values, code 4 (j % 2) + d % 4, with g = d % 32 / 4:
 *     dim 64:  g               dim 128: 2 (g ^ 4 (p / 2 % 2)) + d / 64
 *     dim 256: 4 (g ^ 2 (p % 4)) + d / 64
 * (the order in which the tensor-core fragments of the attention read them). */
typedef struct {
    void *pages;
    size_t num_pages;
    size_t heads, dim;
} ApusKv4Cache;

/* Sequences over a cache.  Sequence s has the rows cu_rows[s] ..
 * cu_rows[s + 1] - 1 of the row arrays; they are its last positions: row
 * cu_rows[s] + i stands at position kv_len[s] - n + i, n its number of rows.
 * Position p is in page page_table[s * table_stride + p / 64].  max_rows and
 * max_len bound the rows and the length of any sequence (max_len <=
 * 64 * table_stride).  A sequence may have no rows or no positions (padding of
 * a batch).  Out of bounds, a length counts as 0 and a row range as no rows.
 * cu_rows ascends: where it does not, a range is out of bounds and reported, and
 * append and read, which look a row's sequence up, may also leave out rows of
 * other sequences. */
typedef struct {
    const int32_t *cu_rows;      /* [nseq + 1] */
    const int32_t *kv_len;       /* [nseq], this call's rows included */
    const int32_t *page_table;   /* [nseq][table_stride] */
    size_t table_stride;
    size_t nseq;
    size_t max_rows, max_len;
} ApusKv4Batch;

/* Bytes of one page of `heads` heads: heads * 72 * dim; 0 for another dim. */
size_t apus_gcuda_kv4_page_bytes(size_t heads, size_t dim);

/* Quantise the batch's rows of k and v into the cache.  Rows before position
 * 0 and rows whose page id is out of range are not written.  Two rows of one
 * call must not stand at the same place of the cache. */
int apus_gcuda_kv4_append_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *k,
                              const ApusHeadRows *v, void *stream);

/* Read the batch's rows back into k and v: what append wrote for the same
 * batch, rounded to BF16 ((code - 8) * s has up to 11 bits).  With cu_rows
 * spaced by kv_len it reads whole sequences.  Rows behind cu_rows[nseq] are
 * left as they are; rows before position 0 and rows whose page id is out of
 * range read as zeros. */
int apus_gcuda_kv4_read_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *k,
                            const ApusHeadRows *v, void *stream);

/* Attention of the batch's rows over the cache: out = softmax(scale q k^T) v,
 * query head h over cache head h / (q->heads / cache->heads), row i of a
 * sequence of n rows over the positions up to its own (so the rows of a verify
 * step see one another causally).  The cache must hold those rows already.
 *
 * sel (optional, NULL: all positions) keeps pools of `pool` (1..128) positions,
 * as the indexer selects them: row r sees position j of its sequence when
 * sel[r * sel_stride + j / pool] != 0 (0 beyond sel_stride), and always the
 * positions of its own last, incomplete pool.
 *
 * Scores, softmax statistics and sums are fp32, and the sum of the weights goes
 * by the scores alone, however large or small the values are.  For the output a
 * weight w is rounded to f16 as it is and once more times its value's scale s,
 * for the tensor cores, in units of a power of two that keep the row's largest
 * w s in f16's range; scales are f16 too, relative to their position's largest
 * (exact from 2^-17 of that on).  So a term w s c (c the code) is off by 2^-10
 * of itself, plus 21 * 2^-30 of the row's largest w s in any group, plus
 * 7 * 2^-25 of the largest w s of its position: groups of dims 2^14 and more
 * below their neighbours lose bits, and at 2^25 below they count as zeros.
 * Query elements are exact down to 2^-24 of their row's largest and held to
 * 2^-35 of it below; a row whose largest magnitude times scale is 2^117 or more
 * may be NaN.  Positions in a page whose id
 * is out of range count as unseen; a row that sees nothing gives zeros.  What
 * stands at unseen positions has no influence, NaN and infinities included; a
 * NaN or an infinity in a query row makes that row NaN, and a group of values
 * that holds NaN those dims of every row that sees it.  Rows behind
 * cu_rows[nseq] are left as they are.
 * workspace: 16-byte aligned, at least apus_gcuda_kv4_attn_workspace bytes (0:
 * none needed, or bad arguments: apus_gcuda_last_error() tells), private to the
 * call until it has run; its contents need no initialisation.  The bytes go by
 * the batch's bounds (nseq, max_rows, max_len) and grow with each, so one
 * workspace for the largest serves all. */
size_t apus_gcuda_kv4_attn_workspace(const ApusKv4Cache *cache, const ApusKv4Batch *batch, size_t q_heads);
int apus_gcuda_kv4_attn_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *q,
                            const ApusHeadRows *out, float scale, const uint8_t *sel, size_t sel_stride, size_t pool,
                            void *workspace, size_t workspace_bytes, void *stream);

/* ---- prompt attention ---------------------------------------------------- */

/* Packed sequences: rows cu_q[s] .. cu_q[s + 1] - 1 of q and out, rows
 * cu_k[s] .. cu_k[s + 1] - 1 of k and v.  Row i of n queries over m keys sees
 * the keys 0 .. m - n + i (n = m: a whole prompt; n < m: the last n rows of a
 * prompt, its earlier keys read back from a cache, say).  max_rows bounds the
 * queries of any sequence. */
typedef struct {
    const int32_t *cu_q, *cu_k;  /* [nseq + 1] */
    size_t nseq;
    size_t max_rows;
} ApusPromptBatch;

/* out = softmax(scale q k^T) v, causal, query head h over head
 * h / (q->heads / k->heads) of k and v; dim 64, 128 or 256.  Scores, softmax
 * statistics and sums are fp32, the weights are rounded to BF16 for the tensor
 * cores.  A row that sees no key gives zeros; keys and values that a row does
 * not see have no influence on it, NaN and infinities included; rows behind
 * cu_q[nseq] are left as they are.  Out of bounds, a sequence's range counts
 * as no queries or no keys.  Scores are bounded by fp32 before the scale is
 * applied, and so are the weighted sums before they are divided, in which a
 * weight counts up to 2^8: with values of 2^120 / keys and more (10^32 at 10^4
 * keys) they may overflow, and the row then holds infinities or NaN. */
int apus_gcuda_prompt_attn_dev(const ApusPromptBatch *batch, const ApusHeadRows *q, const ApusHeadRows *k,
                               const ApusHeadRows *v, const ApusHeadRows *out, size_t dim, float scale, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* APUS_ATTN_GCUDA_H */
