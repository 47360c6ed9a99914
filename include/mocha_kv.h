/* Paged key/value cache operators of libmocha_b200.so.
 *
 * A cache is a pool of pages; a sequence's position t lives at row t % page_size of page
 * table[seq][t / page_size].  mocha_kv_append rotates new queries and keys and writes
 * keys and values to their pages, mocha_kv_decode attends from one new token per
 * sequence, mocha_kv_prefill from a ragged batch of prompt pieces whose keys have been
 * appended before.  No reference counterpart: the reference keeps one flat cache of 1024
 * positions (src/minimind.cu:71,85-88).
 *
 * Every pointer is a device pointer of `device` unless it is said to be on the host.  The
 * calls enqueue their kernels on `stream` (NULL: the default stream) and return; they
 * neither allocate nor wait, so they can be captured into graphs, and lengths, tables and
 * positions are read on the device at replay.  They may be made with any device current
 * and leave it as it was; outputs must not overlap inputs but where that is said to be
 * allowed.  They return 0 on success and 1 on an error, with a message on
 * stderr and nothing enqueued.
 *
 * Types: the pages, the rotated queries and the attention's queries and outputs have one
 * type, fp32, fp16 or bf16; products are summed in fp32 and softmax statistics are fp32.  On
 * 16-bit pages mocha_kv_prefill rounds the softmax weights to the pages' type for the product
 * with the values, which adds up to 40 % to the error that the outputs' own rounding makes;
 * mocha_kv_decode keeps twice the bits of them, and on fp32 pages they are fp32.
 * Alignment: the base pointers of pages, queries, keys, values and outputs are multiples
 * of 16 bytes, their strides multiples of 16 bytes, and a head's values are contiguous.
 * head_dim is a multiple of 32 up to 128, page_size a multiple of 8 up to 65536. */
#ifndef MOCHA_KV_H
#define MOCHA_KV_H

#ifdef __cplusplus
extern "C" {
#endif

enum { MOCHA_KV_F32 = 0, MOCHA_KV_F16 = 1, MOCHA_KV_BF16 = 2 };

/* The page pool.  Element (page, kv head, row, i) of k and of v is at
 * page * page_stride + head * head_stride + row * token_stride + i, in elements. */
typedef struct {
    int device, type;
    int pages, page_size, kv_heads, head_dim;
    long long page_stride, head_stride, token_stride;
    void *k, *v;
} mocha_kv_pages;

/* The sequences.  table[s * table_stride + i], i < table_width, is the page of positions
 * [i * page_size, (i + 1) * page_size) of sequence s; entries of positions that no call
 * needs are not used.  A sequence has at most 2^30 positions.  A needed page id outside [0, pages) reads as a page of zeros and is
 * not written.  Where `status` is not NULL, *status becomes at least 1 when such a page, or
 * an append position that the table or the angles do not hold, was met, and 2 when a
 * bounded wait inside a kernel ran out (it is never reset); the rows concerned, outputs and
 * lse, are then NaN, so that a call without `status` shows it too. */
typedef struct {
    int seqs, table_width;
    long long table_stride;
    const int *table;
    const int *kv_len; /* [seqs] positions held, this call's included; attention only */
    int *status;       /* or NULL */
} mocha_kv_seqs;

/* Rows of heads: element (row, head, i) at row * row_stride + head * head_stride + i. */
typedef struct {
    void *data;
    long long row_stride, head_stride;
} mocha_kv_rows;

/* Rotary positions.  A pair (a, b) of the first `dims` values of a head becomes
 * (a cos - b sin, a sin + b cos) with cos[pos * stride + i], sin[pos * stride + i];
 * pair i is values (i, i + dims / 2), or (2i, 2i + 1) when interleaved.  The other values
 * are kept.  dims is a multiple of 16 up to head_dim; 0 rotates nothing. */
typedef struct {
    const float *cos, *sin;
    long long stride; /* floats between positions, a multiple of 4 */
    int positions;    /* rows of the tables */
    int dims, interleaved;
} mocha_kv_rope;

/* Scores of query head h at position p with key j, its kv head being
 * h / (heads / kv_heads):  z = scale * (q . k);  z = cap * tanh(z / cap) when cap > 0;
 * z -= slopes[h] * |p - j| when slopes is not NULL.  Key j is visible when
 * j < kv_len and (j <= p and (window == 0 or p - j < window), or j < prefix[s]): a prefix
 * is seen by every query, also by those before its end and past the window.
 * heads / kv_heads is at most 64, scale within 2^40, a cap from 2^-40 to 2^40. */
typedef struct {
    int heads, window;
    float scale, cap;
    const int *prefix;   /* [seqs] or NULL */
    const float *slopes; /* [heads] or NULL */
} mocha_kv_scores;

/* Row i (i < rows) holds the new token of sequence seq[i] at position pos[i]: q rotated
 * goes to q_out, k rotated and v go to the page row.  A row with a seq outside [0, seqs),
 * a negative position, or a position past the table or the angles is skipped: its q_out
 * and the pages stay as they were (rows of a padded batch have seq -1).  q, k and v have
 * type in_type, q_out the pages' type; each value is rounded once.  q and q_out may both
 * be NULL.  q_out may be q itself when the types and strides agree.  Of rows that name
 * the same sequence and position, each 8 or 16 values are those of one of them. */
int mocha_kv_append(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, int rows, const int *seq, const int *pos,
                    int in_type, int heads, const mocha_kv_rows *q, const mocha_kv_rows *k, const mocha_kv_rows *v,
                    const mocha_kv_rows *q_out, const mocha_kv_rope *rope, void *stream);

/* Bytes of workspace (a host pointer) that decode (prefill = 0) or prefill (1) calls on
 * these pages need with `heads` query heads.  The workspace needs no initial contents
 * and must be 16-byte aligned; calls, or replays of graphs, that share one must not
 * overlap on the GPU. */
int mocha_kv_workspace(const mocha_kv_pages *pages, int heads, int prefill, unsigned long long *bytes);

/* Attention of one query row per sequence, row s at position kv_len[s] - 1, which must
 * have been appended.  out[s][h] = sum over visible keys of softmax(z) v, and
 * lse[s * heads + h] = log(sum of exp z) where lse is not NULL.  A row that sees no key
 * (kv_len <= 0), or whose visible scores are all -infinity, gives zeros and -infinity. */
int mocha_kv_decode(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                    const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse, void *workspace,
                    unsigned long long workspace_bytes, void *stream);

/* Attention of rows q_start[s] .. q_start[s+1] - 1 of q for each sequence s (q_start has
 * seqs + 1 values, not falling; a sequence may have no rows), which stand at the last
 * positions of the sequence: row i at kv_len[s] - (q_start[s+1] - q_start[s]) +
 * (i - q_start[s]).  Outputs and lse[row * heads + h] as in mocha_kv_decode; a row whose
 * position is negative sees at most the prefix.  Rows outside the sequences' ranges (all
 * ranges lie in [0, rows)) are left as they were.  Values of keys that a row does not see
 * never reach it, infinite or NaN ones included. */
int mocha_kv_prefill(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores, int rows,
                     const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse,
                     void *workspace, unsigned long long workspace_bytes, void *stream);

/* mocha_kv_prefill for tests of status 2: waits give up after wait_polls polls of 4 us, in
 * place of as many as take a second, and on 16-bit pages, where drop is not 0, CTA b does not copy the
 * values of its (b % drop)-th tile of keys, which its other warps then wait for. */
int mocha_kv_prefill_check(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                           int rows, const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse,
                           void *workspace, unsigned long long workspace_bytes, void *stream, int wait_polls,
                           int drop);

#ifdef __cplusplus
}
#endif
#endif
