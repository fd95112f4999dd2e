/*
 * gr_paged.h -- paged KV cache and attention over packed batches, beside the
 * contiguous caches and single-sequence calls of gr_attn.h.  For serving loops that
 * keep activations in HBM: device pointers only, work is enqueued on the caller's HIP
 * stream (which belongs to the current device, where every buffer lives), nothing is
 * allocated and nothing synchronises, so the calls can be captured into a HIP graph.
 * Status codes, element types and gr_last_error() are those of gr_attn.h.
 *
 * No counterpart in the reference, whose cache is one contiguous array per sequence
 * (src/engine/types.rs:745-809).  What a row stores and what a token sees are the
 * reference's: rows after QK norm and RoPE (kv_write_token, inference.rs:1877-1965),
 * the visible keys of attention.rs:74-96, quantize_row_q8's scale and codes
 * (inference.rs:249-268).
 *
 * Lengths, row offsets and page tables are read from device memory when the kernels
 * run; the host only sees upper bounds.  Whatever they hold, nothing outside the
 * buffers described here is read or written: offsets are clamped to [0, n_rows],
 * lengths to [0, table_pages * page_size], and a page id outside [0, n_pages) names a
 * page that holds no rows (see each call).
 */
#ifndef GR_PAGED_H
#define GR_PAGED_H

#include "gr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* K and V pages of one layer.  Element i of KV head g in row r of page p is at
 * p*page_stride + r*row_stride + g*head_stride + i of k_pages / v_pages, so a page may
 * be [row][head][dim] (row_stride = n_kv_heads*head_dim, head_stride = head_dim) or
 * [head][row][dim].  Position t of a sequence is row t % page_size of its page
 * t / page_size.  Rows no sequence owns may hold anything. */
typedef struct gr_paged_cache {
    int32_t n_pages;
    int32_t page_size;    /* rows per page: a power of two, 16 or more */
    int32_t n_kv_heads;
    int32_t head_dim;     /* 64, 128 or 256 */
    int32_t kv_dtype;     /* GR_DTYPE_F16, GR_DTYPE_BF16 or GR_DTYPE_Q8 */
    void* k_pages;        /* 16-byte aligned, as v_pages */
    void* v_pages;
    int64_t page_stride;  /* elements, as row_stride and head_stride: multiples of 16 bytes; */
    int64_t row_stride;   /* row_stride at most 2^22 */
    int64_t head_stride;
    /* GR_DTYPE_Q8 only (NULL / 0 otherwise): int8 codes and one f32 scale per (row, KV
     * head), at p*scale_page_stride + r*scale_row_stride + g*scale_head_stride; the
     * element is code * scale.  Scales are finite and positive. */
    float* k_scale;
    float* v_scale;
    int64_t scale_page_stride;
    int64_t scale_row_stride;
    int64_t scale_head_stride;
} gr_paged_cache;

/* The rows of a step: sequence s has the rows row_start[s] .. row_start[s + 1] - 1 of
 * the step's row arrays, which are its last positions kv_len[s] - (number of its rows)
 * .. kv_len[s] - 1.  One row per sequence is a decode step, many are a prompt or a
 * chunk of one, and a batch may mix them.  Rows in front of row_start[0] and from
 * row_start[n_seq] on (a padded batch) belong to no sequence: calls leave what they
 * would write for them as it was.  A row whose position would be negative (more rows
 * than kv_len) has no place in the cache. */
typedef struct gr_paged_batch {
    int32_t n_seq;
    int32_t n_rows;             /* rows of the row arrays */
    int32_t max_rows;           /* the most rows of a sequence, and the largest kv_len: they */
    int32_t max_len;            /* choose kernels; a wrong value costs time, not results */
    const int32_t* row_start;   /* device [n_seq + 1], not decreasing */
    const int32_t* kv_len;      /* device [n_seq]: cached positions, the step's rows included */
    const int32_t* page_table;  /* device [n_seq][table_stride]: pages of each sequence in order */
    int64_t table_stride;
    int32_t table_pages;        /* entries of a table row; * page_size at most 2^30 */
} gr_paged_batch;

/* K and V rows outside the cache: element i of head g of row r is at
 * r*row_stride + g*head_stride + i; 16-byte aligned, strides multiples of 16 bytes. */
typedef struct gr_paged_rows {
    int32_t dtype;        /* GR_DTYPE_F32, GR_DTYPE_F16 or GR_DTYPE_BF16 */
    void* k;
    void* v;
    int64_t row_stride;   /* elements */
    int64_t head_stride;
} gr_paged_rows;

/* Store the batch's rows in their pages.  16-bit pages: rounded to nearest even.  Q8
 * pages: per (row, head), amax = max |x|; scale = amax * (1/127); code = clamp(round(x *
 * (127 * (1/amax))), -127, 127), halves away from zero, every quotient and product
 * rounded to f32 (quantize_row_q8 over one head's row, with reciprocals); an amax below
 * 2^-100 counts as 0: scale 1, codes 0.  A NaN stores as 0; an infinity makes its head
 * row read as NaN. A row whose page id names no page is
 * dropped.  Sequences may share pages they only read; no two rows of a call may name
 * the same place.  At most 2^26 rows, as a read. */
int gr_paged_kv_write(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_rows* rows, void* stream);

/* The reverse: the batch's positions read out of their pages into rows (with kv_len
 * rows per sequence, whole sequences), each element rounded once to rows->dtype.  A row
 * whose page id names no page, or whose position is negative, reads as zeros. */
int gr_paged_kv_read(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_rows* rows, void* stream);

/* Attention of the batch's rows over their pages, which hold those rows' K and V
 * already (gr_paged_kv_write): the row at position p sees keys max(0, p + 1 - window)
 * (0 for window 0) .. p of its own sequence.  Grouped heads: query head h reads KV head
 * h / (n_heads / n_kv_heads).  Scores, softmax and sums are f32; the weights enter the
 * product with V rounded to dtype (f16 over Q8 pages), the result is rounded once.  A
 * row that sees no key (negative position, pages that hold no rows) gets zeros.  Keys a
 * row does not see have no influence on it, whatever they hold (inf and NaN too).  More
 * work than can be numbered in 31 bits of tiles is refused. */
typedef struct gr_paged_attention_args {
    int32_t n_heads;        /* a multiple of the cache's n_kv_heads */
    int32_t dtype;          /* of q and out: GR_DTYPE_F16 or GR_DTYPE_BF16; the pages' type unless they are Q8 */
    int32_t window;         /* 0 = every key up to the row's own, W > 0 = the last W of them */
    float score_scale;      /* finite and positive, usually 1/sqrt(head_dim) */
    const void* q;          /* row r, head h, dim i at r*q_row_stride + h*q_head_stride + i; */
    int64_t q_row_stride;   /* 16-byte aligned, strides multiples of 8 elements */
    int64_t q_head_stride;
    void* out;              /* as q */
    int64_t out_row_stride;
    int64_t out_head_stride;
    void* workspace;        /* gr_paged_attention_workspace_size() bytes, 256-byte aligned; one call at a time */
} gr_paged_attention_args;

/* Bytes of workspace for these sizes (0 when an argument is invalid).  It depends on
 * the sizes, types and upper bounds only, not on device data. */
size_t gr_paged_attention_workspace_size(const gr_paged_cache* c, const gr_paged_batch* b,
                                         const gr_paged_attention_args* a);
int gr_paged_attention(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_attention_args* a, void* stream);

/* Causal attention inside each of n_seq prompts that lie one after another in q, k and
 * v: prompt s is rows seq_start[s] .. seq_start[s + 1] - 1 and sees nothing of the
 * others.  No cache is read or written.  Windows, heads, arithmetic, padding rows and
 * rows outside every prompt as gr_paged_attention. */
typedef struct gr_packed_args {
    int32_t n_seq;
    int32_t n_rows;           /* rows of q, k, v and out */
    int32_t max_rows;         /* the longest prompt: chooses kernels */
    int32_t n_heads;          /* a multiple of n_kv_heads */
    int32_t n_kv_heads;
    int32_t head_dim;         /* 64, 128 or 256 */
    int32_t dtype;            /* of q, k, v and out: GR_DTYPE_F16 or GR_DTYPE_BF16 */
    int32_t window;
    float score_scale;
    const int32_t* seq_start; /* device [n_seq + 1], not decreasing */
    const void* q;            /* layouts and alignment as gr_paged_attention_args; k and v share strides, */
    int64_t q_row_stride;     /* kv_row_stride at most 2^22 */
    int64_t q_head_stride;
    const void* k;
    const void* v;
    int64_t kv_row_stride;
    int64_t kv_head_stride;
    void* out;
    int64_t out_row_stride;
    int64_t out_head_stride;
    void* workspace;          /* gr_packed_attention_workspace_size() bytes, 256-byte aligned; one call at a time */
} gr_packed_args;

size_t gr_packed_attention_workspace_size(const gr_packed_args* a);
int gr_packed_attention(const gr_packed_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GR_PAGED_H */
