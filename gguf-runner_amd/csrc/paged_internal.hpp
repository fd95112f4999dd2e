// Launch descriptors of the paged KV cache and the packed-batch attention, shared
// between the C-ABI layer (api_paged.cpp) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gr_common.hpp"
#include "gr_paged.h"

namespace gr {

// Sequences of a step and where their rows and keys are (gr_paged_batch; packed
// prompts: kv_len and page_table null, a sequence's keys are its own rows).
struct PagedSeqs {
    int n_seq, n_rows;
    const int32_t* row_start;
    const int32_t* kv_len;
    const int32_t* page_table;
    int64_t table_stride;
    int page_shift;  // log2(page_size)
    int n_pages;
    int max_len;     // table_pages * page_size (packed: n_rows): lengths are clamped to it
};

struct PagedKvLaunch {
    PagedSeqs seqs;
    int n_kv_heads, head_dim, kv_dtype, rows_dtype;
    void* pages[2];       // K, V
    float* scale[2];
    void* rows[2];
    int64_t page_stride, row_stride, head_stride;
    int64_t scale_page_stride, scale_row_stride, scale_head_stride;
    int64_t rows_row_stride, rows_head_stride;
};

hipError_t launch_paged_kv_write(const PagedKvLaunch& p, hipStream_t st);
hipError_t launch_paged_kv_read(const PagedKvLaunch& p, hipStream_t st);

struct PagedAttnLaunch {
    PagedSeqs seqs;
    int n_heads, n_kv_heads, head_dim;
    int group;             // query heads per KV head
    uint32_t group_magic;  // ceil(2^32 / group), 0 for 1
    int dtype;     // q, out
    int kv_dtype;  // pages (packed: dtype)
    int window;
    float scale_log2;  // score_scale * log2(e)
    const void* q;
    void* out;
    int64_t q_row_stride, q_head_stride, out_row_stride, out_head_stride;
    const void* k;
    const void* v;
    int64_t page_stride, row_stride, head_stride;  // packed: page_stride 0
    const float* k_scale;
    const float* v_scale;
    int64_t scale_page_stride, scale_row_stride, scale_head_stride;
    int max_rows, max_len;  // the caller's bounds, for the choice of kernels
    void* workspace;
};

// Whether the launch's work can be numbered.
bool paged_attn_fits(const PagedAttnLaunch& p);
size_t paged_attn_ws_bytes(const PagedAttnLaunch& p);
hipError_t launch_paged_attn(const PagedAttnLaunch& p, hipStream_t st);

// ---------------------------------------------------------------- device helpers

// r / group for 0 <= r < 2^31: the product with ceil(2^32 / group) is at most one too high.
__device__ __forceinline__ int div_group(const PagedAttnLaunch& p, int r) {
    if (p.group == 1) return r;
    const int q = (int)__umulhi((uint32_t)r, p.group_magic);
    return q - ((uint32_t)q * (uint32_t)p.group > (uint32_t)r ? 1 : 0);
}

// Row offset i of the batch, clamped to the row arrays.
__device__ __forceinline__ int seq_row(const PagedSeqs& s, int i) {
    return min(max(s.row_start[i], 0), s.n_rows);
}

// The sequence whose rows hold `row` (wave-uniform; every lane of the wave calls it),
// or -1 for a row of none: a 64-ary search of row_start, one load per level.
__device__ __forceinline__ int seq_of_row(const PagedSeqs& s, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = s.n_seq + 1;  // the last i in [lo, hi) with row_start[i] <= row
    if (row < s.row_start[0]) return -1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const int n = __popcll(__ballot(i < hi && s.row_start[min(i, s.n_seq)] <= row));
        const int at = lo + max(n - 1, 0) * step;
        hi = min(at + step, hi);
        lo = at;
    }
    return lo < s.n_seq ? lo : -1;
}

__device__ __forceinline__ int seq_len(const PagedSeqs& s, int seq, int rows) {
    return s.kv_len ? min(max(s.kv_len[seq], 0), s.max_len) : rows;
}

}  // namespace gr
