/*
 * m27b_paged.h — a paged key/value cache for several sequences: rotary
 * positions with the append to the cache, attention of new tokens over it,
 * and the upkeep of its pages.
 *
 * The reference keeps one contiguous fp32 cache of one sequence
 * (k_mrope_and_cache, src/mono27b_executor.cu:1180-1229; the attention pair
 * :1339-1484); these entries have no counterpart there.
 *
 * The cache of a layer is two pools of pages in 16 bits: element d of kv head
 * j at slot s of page p is k[p * page_stride + (s * n_kv + j) * head_dim + d]
 * (within a page the order of the reference's cache).  A table of page ids
 * says which page holds which positions: position i of the sequence in table
 * row r is slot i % page_size of page table[r * n_cols + i / page_size], and
 * lens[r] is the number of positions the sequence has.  Pages may be shared
 * by several rows; ref[p] counts the rows that hold page p, and a page with
 * ref[p] <= 0 is free.
 *
 * Conventions of m27b_qmv.h: bool + error buffer; device pointers on the
 * current device; the work is enqueued on `stream` and nothing is
 * synchronised or allocated, so every entry can be captured in a CUDA graph.
 * Lengths, tables and page ids are read on the device, so a captured graph
 * serves every state of the cache.  What only the device can see to be wrong
 * (a table row, page id or position out of range) is reported through
 * m27b_device_status (code 6): nothing outside the buffers is read or written,
 * and each entry says what it does instead.
 */
#ifndef M27B_PAGED_H
#define M27B_PAGED_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime_api.h>

#include "m27b_qmv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ggml's code of bfloat16 (f16 is M27B_TYPE_F16, f32 M27B_TYPE_F32). */
#define M27B_TYPE_BF16 30u

/* One layer's pools and the page table. */
typedef struct M27BPagedKV {
    void *k, *v;           /* pools, 16-byte aligned */
    const int *table;      /* n_rows rows of n_cols page ids */
    uint32_t type;         /* M27B_TYPE_F16 or M27B_TYPE_BF16 */
    int n_pages;
    int page_size;         /* positions per page: 16, 32, 64, 128 or 256 */
    int n_kv, head_dim;    /* kv heads; 64, 128 or 256 values each */
    int n_rows, n_cols;
    long long page_stride; /* values from a page to the next: a multiple of 8,
                              at least page_size * n_kv * head_dim */
} M27BPagedKV;

/* The new tokens of a batch: sequence b's are rows cu_q[b] .. cu_q[b + 1] - 1
 * of the token buffers (cu_q ascending from >= 0, at most n_tok; a sequence
 * may have none), and are the last positions of its lens[row] positions: row
 * i of sequence b is position lens[row] - (cu_q[b + 1] - cu_q[b]) + i. */
typedef struct M27BPagedBatch {
    const int *cu_q; /* n_seq + 1 offsets */
    const int *lens; /* positions of each TABLE ROW, the new ones included */
    const int *rows; /* table row of each sequence, or NULL: sequence b is row b */
    int n_seq;
    int n_tok; /* rows of the token buffers; rows of no sequence are left alone */
} M27BPagedBatch;

/* ---- rotary positions ---- */

enum { M27B_ROPE_NONE = 0, M27B_ROPE_LINEAR = 1, M27B_ROPE_YARN = 2 };

/* How positions are stretched for long contexts (NULL or M27B_ROPE_NONE: not).
 *   linear: every frequency divided by `factor`.
 *   yarn:   pair j's frequency is f_j / factor * r_j + f_j * (1 - r_j) with the
 *           ramp r_j = clamp((j - lo) / max(hi - lo, 0.001), 0, 1), lo and hi
 *           the pairs that turn beta_fast and beta_slow times over
 *           `original_ctx` positions (rounded outwards), and the factors are
 *           multiplied by `attn_factor` (<= 0: 0.1 ln(factor) + 1). */
typedef struct M27BRopeScaling {
    int kind;
    float factor;        /* >= 1 */
    int original_ctx;    /* yarn */
    float beta_fast;     /* yarn: 32 */
    float beta_slow;     /* yarn: 1 */
    float attn_factor;   /* yarn */
} M27BRopeScaling;

/* table[p][j] = {cos, sin}(p * f_j) of positions p < n_pos and pairs j <
 * n_rot / 2, f_j = theta^(-2j / n_rot) with the scaling applied: angles in
 * fp64, stored as fp32 (8-byte aligned). */
M27B_API bool m27b_rope_table(float *table, int n_pos, int n_rot, double theta, const M27BRopeScaling *scaling,
                              cudaStream_t stream, char *err, size_t err_cap);

typedef struct M27BRope {
    const float *table; /* of m27b_rope_table, 16-byte aligned */
    int n_pos, n_rot;   /* n_rot <= head_dim, a multiple of 16 */
    int interleaved;    /* pairs (2j, 2j + 1); 0: (j, j + n_rot / 2) */
    const int *positions; /* rotary position of each token row, or NULL: its position in the cache */
} M27BRope;

/* The projections of the new tokens: head h of token t at q + t * q_stride +
 * h * head_dim (values), likewise k and v; all of type src_type (F32, or the
 * cache's type).  Base pointers 16-byte aligned, strides multiples of 16
 * bytes. */
typedef struct M27BHeads {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    uint32_t src_type;
    int n_q;
    const float *q_norm, *k_norm; /* head RMSNorm weights (head_dim, 16-byte aligned), or NULL: no norm */
    float eps;
} M27BHeads;

/* For every new token: RMSNorm of its q and k heads (where weights are given),
 * rotation of their first n_rot values, rounding once to the cache's type; q
 * to q_out (q_out + t * q_out_stride + h * head_dim), k and the unrotated v to
 * the token's slot in the cache.  All arithmetic in fp32.  q_out may be q
 * itself when the types agree.  n_q = 0 appends only.  A token whose position
 * or page is out of range is left out (status 6).  In f16 a value above 65504
 * becomes an infinity, and rows that attend to it may become NaN. */
M27B_API bool m27b_rope_append(const M27BPagedKV *kv, const M27BPagedBatch *batch, const M27BRope *rope,
                               const M27BHeads *heads, void *q_out, long long q_out_stride, cudaStream_t stream,
                               char *err, size_t err_cap);

/* ---- attention ---- */

/* Scratch of m27b_paged_attn, contents free; calls that may overlap need one
 * each.  0 for an invalid shape. */
M27B_API size_t m27b_paged_attn_scratch_bytes(int n_q, int n_kv, int head_dim);

/* out[t][h] = softmax(scale * q[t][h] . K) V over the positions that token t
 * sees: p and everything before it, p its own position; with window > 0 only
 * the last `window` of those.  q and out: the cache's type, head h of token t
 * at q + t * q_stride + h * head_dim (16-byte aligned, strides multiples of 8
 * values).  n_q is a multiple of n_kv, at most 128 query heads per kv head.
 * lse, if given, receives log(sum(exp(scale * q . k))) at lse[t * n_q + h].  A
 * row that sees nothing (a sequence with fewer positions than new tokens)
 * gets zeros and -inf.  Scores, softmax statistics and sums are fp32; the
 * weights are rounded to the cache's type for their product with V.  Slots
 * that no row of the sequence sees may hold anything, infinities and NaN
 * included; a position that the sequence holds must be finite.  A row of q with
 * a NaN gets NaN in out and lse, and so does a row that sees one in K.
 * scale is positive.
 * Status 6: a page out of range that a row sees counts as keys and values of
 * zero, a length beyond the table as the table's, a table row out of range as
 * one without positions.  The rows of that sequence are then of no use; those of
 * other sequences are right. */
M27B_API bool m27b_paged_attn(const M27BPagedKV *kv, const M27BPagedBatch *batch, const void *q, long long q_stride,
                              int n_q, float scale, int window, void *out, long long out_stride, float *lse,
                              void *scratch, cudaStream_t stream, char *err, size_t err_cap);

/* ---- pages ---- */

/* Page counts and tables of a cache.  Row r holds ceil(lens[r] / page_size)
 * pages in its first entries; the others are -1. */
typedef struct M27BPages {
    int *ref;   /* n_pages */
    int *table; /* n_rows x n_cols */
    int *lens;  /* n_rows */
    int n_pages, page_size, n_rows, n_cols;
} M27BPages;

/* The data that page ids name: page p of plane i (a layer's keys or values)
 * is the page_bytes bytes at base + i * plane_stride + p * page_stride.  All
 * multiples of 16. */
typedef struct M27BPagePool {
    void *base;
    int n_planes;
    size_t plane_stride, page_stride, page_bytes;
} M27BPagePool;

#define M27B_MAX_POOLS 2

/* What a refused call writes to its `status` word (which a successful call
 * leaves alone): too few free pages; a row, length or request out of range,
 * or a row named twice.  A refused call changes nothing else. */
enum { M27B_PAGES_FULL = 1, M27B_PAGES_BAD = 2 };

/* Scratch of the entries below for n requests (0 for compact), 16-byte
 * aligned, contents free; calls that may overlap need one each. */
M27B_API size_t m27b_pages_scratch_bytes(int n_pages, int n_rows, int n);

/* Set the lengths of n rows to new_lens (device).  A row that grows takes the
 * lowest free pages, request by request; if its last page is half-filled and
 * shared, the row first gets a copy of its own (the next append writes
 * there).  A row that shrinks gives up its last pages.  After a refused call the
 * lengths are the old ones: an append of the new tokens would then overwrite the
 * last positions, also in pages that other rows hold, so *status is to be read
 * first. */
M27B_API bool m27b_pages_resize(const M27BPages *pages, const M27BPagePool *pools, int n_pools, const int *rows,
                                const int *new_lens, int n, void *scratch, int *status, cudaStream_t stream, char *err,
                                size_t err_cap);

/* Fork n rows: row dst[i] (empty before, named once, no src[j]) becomes a copy
 * of row src[i] that shares its full pages and gets its own copy of a
 * half-filled last page, in the lowest free page, request by request. */
M27B_API bool m27b_pages_fork(const M27BPages *pages, const M27BPagePool *pools, int n_pools, const int *src,
                              const int *dst, int n, void *scratch, int *status, cudaStream_t stream, char *err,
                              size_t err_cap);

/* Empty n rows: their pages lose a reference, their lengths become 0 (a row
 * named twice is freed once; a row out of range is skipped, status 6). */
M27B_API bool m27b_pages_free(const M27BPages *pages, const int *rows, int n, cudaStream_t stream, char *err,
                              size_t err_cap);

/* Move the pages in use together: with L pages in use, the pages >= L in use,
 * in ascending order, move into the free pages < L, in ascending order; data,
 * counts and tables follow.  n_live, if given, receives L. */
M27B_API bool m27b_pages_compact(const M27BPages *pages, const M27BPagePool *pools, int n_pools, int *n_live,
                                 void *scratch, cudaStream_t stream, char *err, size_t err_cap);

/* Copy page src[i] to page dst[i] in every plane, i < n (a pair with an id out
 * of range is skipped, status 6).  No page is both a source and a target, and
 * none is a target twice. */
M27B_API bool m27b_pages_copy(const M27BPagePool *pools, int n_pools, int n_pages, const int *src, const int *dst,
                              int n, cudaStream_t stream, char *err, size_t err_cap);

#ifdef __cplusplus
}
#endif

#endif /* M27B_PAGED_H */
