// C-ABI entry points of the paged KV cache and of the attention over packed batches
// (gr_paged.h): argument validation and dispatch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "gr_api_util.hpp"
#include "gr_attn.h"
#include "gr_paged.h"
#include "paged_internal.hpp"

namespace gr {

namespace {

constexpr int64_t kMaxRowStride = (int64_t)1 << 22;  // a tile's byte offsets stay in 31 bits
constexpr int64_t kMaxPositions = (int64_t)1 << 30;  // positions plus a tile stay in 31 bits
constexpr int kMaxKvRows = 1 << 26;  // rows of a write or read: its threads are numbered in 32 bits

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
int elem_bytes(int dtype) { return dtype == GR_DTYPE_F32 ? 4 : dtype == GR_DTYPE_Q8 ? 1 : 2; }
bool dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

int check_cache(const char* fn, const gr_paged_cache* c) {
    if (!c) return fail(GR_ERR_ARG, "%s: null cache", fn);
    if (!dim_ok(c->head_dim)) return fail(GR_ERR_ARG, "%s: head_dim %d unsupported (64, 128, 256)", fn, c->head_dim);
    if (c->n_kv_heads < 1) return fail(GR_ERR_ARG, "%s: n_kv_heads %d must be positive", fn, c->n_kv_heads);
    if (c->n_pages < 1) return fail(GR_ERR_ARG, "%s: n_pages %d must be positive", fn, c->n_pages);
    if (c->page_size < 16 || c->page_size > kMaxPositions || (c->page_size & (c->page_size - 1)))
        return fail(GR_ERR_ARG, "%s: page_size %d must be a power of two, 16 or more", fn, c->page_size);
    if (c->kv_dtype != GR_DTYPE_F16 && c->kv_dtype != GR_DTYPE_BF16 && c->kv_dtype != GR_DTYPE_Q8)
        return fail(GR_ERR_ARG, "%s: kv_dtype %d unsupported (F16, BF16, Q8)", fn, c->kv_dtype);
    if (!c->k_pages || !c->v_pages) return fail(GR_ERR_ARG, "%s: null k_pages or v_pages", fn);
    if (!aligned16(c->k_pages) || !aligned16(c->v_pages))
        return fail(GR_ERR_ARG, "%s: k_pages and v_pages must be 16-byte aligned", fn);
    const int64_t unit = 16 / elem_bytes(c->kv_dtype);
    for (int64_t s : {c->page_stride, c->row_stride, c->head_stride})
        if (s < c->head_dim || s % unit)
            return fail(GR_ERR_ARG, "%s: cache strides must be at least head_dim and multiples of 16 bytes", fn);
    if (c->row_stride > kMaxRowStride)
        return fail(GR_ERR_ARG, "%s: row_stride %lld above 2^22", fn, (long long)c->row_stride);
    if (c->kv_dtype == GR_DTYPE_Q8) {
        if (!c->k_scale || !c->v_scale) return fail(GR_ERR_ARG, "%s: Q8 pages need k_scale and v_scale", fn);
        if (c->scale_page_stride < 1 || c->scale_row_stride < 1 || c->scale_head_stride < 1)
            return fail(GR_ERR_ARG, "%s: Q8 scale strides must be positive", fn);
    } else if (c->k_scale || c->v_scale) {
        return fail(GR_ERR_ARG, "%s: k_scale and v_scale belong to Q8 pages", fn);
    }
    return GR_OK;
}

// *none: nothing to do (no sequence or no row).
int check_batch(const char* fn, const gr_paged_cache* c, const gr_paged_batch* b, bool* none) {
    if (!b) return fail(GR_ERR_ARG, "%s: null batch", fn);
    if (b->n_seq < 0 || b->n_rows < 0)
        return fail(GR_ERR_ARG, "%s: negative sizes: n_seq %d, n_rows %d", fn, b->n_seq, b->n_rows);
    *none = b->n_seq == 0 || b->n_rows == 0;
    if (*none) return GR_OK;
    if (b->n_seq >= kMaxPositions) return fail(GR_ERR_ARG, "%s: n_seq %d above 2^30", fn, b->n_seq);
    if (b->max_rows < 1 || b->max_len < 1)
        return fail(GR_ERR_ARG, "%s: max_rows %d and max_len %d must be positive", fn, b->max_rows, b->max_len);
    if (!b->row_start || !b->kv_len || !b->page_table)
        return fail(GR_ERR_ARG, "%s: null row_start, kv_len or page_table", fn);
    if (b->table_pages < 1 || b->table_stride < b->table_pages)
        return fail(GR_ERR_ARG, "%s: table_pages %d must be positive and at most table_stride %lld", fn, b->table_pages,
                    (long long)b->table_stride);
    if ((int64_t)b->table_pages * c->page_size > kMaxPositions)
        return fail(GR_ERR_ARG, "%s: table_pages * page_size above 2^30", fn);
    return GR_OK;
}

PagedSeqs seqs_of(const gr_paged_cache* c, const gr_paged_batch* b) {
    PagedSeqs s{};
    s.n_seq = b->n_seq;
    s.n_rows = b->n_rows;
    s.row_start = b->row_start;
    s.kv_len = b->kv_len;
    s.page_table = b->page_table;
    s.table_stride = b->table_stride;
    s.page_shift = __builtin_ctz((unsigned)c->page_size);
    s.n_pages = c->n_pages;
    s.max_len = b->table_pages * c->page_size;
    return s;
}

int kv_call(const char* fn, const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_rows* r, void* stream,
            hipError_t (*launch)(const PagedKvLaunch&, hipStream_t)) {
    clear_error();
    int rc = check_cache(fn, c);
    bool none = false;
    if (!rc) rc = check_batch(fn, c, b, &none);
    if (rc || none) return rc;
    if (!r) return fail(GR_ERR_ARG, "%s: null rows", fn);
    if (b->n_rows > kMaxKvRows) return fail(GR_ERR_ARG, "%s: n_rows %d above 2^26: divide the batch", fn, b->n_rows);
    if (r->dtype != GR_DTYPE_F32 && r->dtype != GR_DTYPE_F16 && r->dtype != GR_DTYPE_BF16)
        return fail(GR_ERR_ARG, "%s: rows dtype %d unsupported (F32, F16, BF16)", fn, r->dtype);
    if (!r->k || !r->v) return fail(GR_ERR_ARG, "%s: null k or v rows", fn);
    const int64_t unit = 16 / elem_bytes(r->dtype);
    if (!aligned16(r->k) || !aligned16(r->v) || r->row_stride % unit || r->head_stride % unit)
        return fail(GR_ERR_ARG, "%s: rows must be 16-byte aligned, with strides of multiples of 16 bytes", fn);
    if (r->row_stride < c->head_dim || r->head_stride < c->head_dim)
        return fail(GR_ERR_ARG, "%s: row strides must be at least head_dim", fn);
    PagedKvLaunch p{};
    p.seqs = seqs_of(c, b);
    p.n_kv_heads = c->n_kv_heads;
    p.head_dim = c->head_dim;
    p.kv_dtype = c->kv_dtype;
    p.rows_dtype = r->dtype;
    p.pages[0] = c->k_pages, p.pages[1] = c->v_pages;
    p.scale[0] = c->k_scale, p.scale[1] = c->v_scale;
    p.rows[0] = r->k, p.rows[1] = r->v;
    p.page_stride = c->page_stride, p.row_stride = c->row_stride, p.head_stride = c->head_stride;
    p.scale_page_stride = c->scale_page_stride, p.scale_row_stride = c->scale_row_stride;
    p.scale_head_stride = c->scale_head_stride;
    p.rows_row_stride = r->row_stride, p.rows_head_stride = r->head_stride;
    const hipError_t e = launch(p, (hipStream_t)stream);
    return e == hipSuccess ? GR_OK : hip_fail(e, fn);
}

int check_heads(const char* fn, int n_heads, int n_kv_heads, int dtype, int window, float scale, int64_t n_rows) {
    if (n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads)
        return fail(GR_ERR_ARG, "%s: n_heads %d must be a positive multiple of n_kv_heads %d", fn, n_heads, n_kv_heads);
    if (dtype != GR_DTYPE_F16 && dtype != GR_DTYPE_BF16)
        return fail(GR_ERR_ARG, "%s: dtype %d unsupported (F16, BF16)", fn, dtype);
    if (window < 0) return fail(GR_ERR_ARG, "%s: negative window %d", fn, window);
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return fail(GR_ERR_ARG, "%s: score_scale must be finite and positive", fn);
    if (n_rows * n_heads > kMaxPositions) return fail(GR_ERR_ARG, "%s: n_rows * n_heads above 2^30", fn);
    return GR_OK;
}

int check_qo(const char* fn, const void* q, const void* out, int head_dim, int64_t qr, int64_t qh, int64_t outr,
             int64_t outh) {
    if (!q || !out) return fail(GR_ERR_ARG, "%s: null q or out", fn);
    if (!aligned16(q) || !aligned16(out)) return fail(GR_ERR_ARG, "%s: q and out must be 16-byte aligned", fn);
    for (int64_t s : {qr, qh, outr, outh})
        if (s < head_dim || s % 8)
            return fail(GR_ERR_ARG, "%s: q and out strides must be at least head_dim and multiples of 8", fn);
    return GR_OK;
}

int check_fits(const char* fn, PagedAttnLaunch& p) {
    p.group = p.n_heads / p.n_kv_heads;
    p.group_magic = p.group == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + p.group - 1) / p.group);
    if (!paged_attn_fits(p))
        return fail(GR_ERR_ARG, "%s: rows, sequences and positions beyond 2^31 tiles of work: divide the batch", fn);
    return GR_OK;
}

int check_ws(const char* fn, const void* ws) {
    if (!ws) return fail(GR_ERR_ARG, "%s: null workspace", fn);
    if ((uintptr_t)ws % 256) return fail(GR_ERR_ARG, "%s: workspace must be 256-byte aligned", fn);
    return GR_OK;
}

int paged_attn_args(const char* fn, const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_attention_args* a,
                    PagedAttnLaunch* p, bool* none) {
    int rc = check_cache(fn, c);
    if (!rc) rc = check_batch(fn, c, b, none);
    if (rc || *none) return rc;
    if (!a) return fail(GR_ERR_ARG, "%s: null args", fn);
    rc = check_heads(fn, a->n_heads, c->n_kv_heads, a->dtype, a->window, a->score_scale, b->n_rows);
    if (!rc && c->kv_dtype != GR_DTYPE_Q8 && a->dtype != c->kv_dtype)
        rc = fail(GR_ERR_ARG, "%s: q of dtype %d over pages of dtype %d", fn, a->dtype, c->kv_dtype);
    if (!rc)
        rc = check_qo(fn, a->q, a->out, c->head_dim, a->q_row_stride, a->q_head_stride, a->out_row_stride,
                      a->out_head_stride);
    if (rc) return rc;
    p->seqs = seqs_of(c, b);
    p->n_heads = a->n_heads;
    p->n_kv_heads = c->n_kv_heads;
    p->head_dim = c->head_dim;
    p->dtype = a->dtype;
    p->kv_dtype = c->kv_dtype;
    p->window = a->window;
    p->scale_log2 = a->score_scale * kLog2e;
    p->q = a->q;
    p->out = a->out;
    p->q_row_stride = a->q_row_stride, p->q_head_stride = a->q_head_stride;
    p->out_row_stride = a->out_row_stride, p->out_head_stride = a->out_head_stride;
    p->k = c->k_pages, p->v = c->v_pages;
    p->page_stride = c->page_stride, p->row_stride = c->row_stride, p->head_stride = c->head_stride;
    p->k_scale = c->k_scale, p->v_scale = c->v_scale;
    p->scale_page_stride = c->scale_page_stride, p->scale_row_stride = c->scale_row_stride;
    p->scale_head_stride = c->scale_head_stride;
    p->max_rows = b->max_rows, p->max_len = b->max_len;
    p->workspace = a->workspace;
    return check_fits(fn, *p);
}

int packed_args(const char* fn, const gr_packed_args* a, PagedAttnLaunch* p, bool* none) {
    if (!a) return fail(GR_ERR_ARG, "%s: null args", fn);
    if (!dim_ok(a->head_dim)) return fail(GR_ERR_ARG, "%s: head_dim %d unsupported (64, 128, 256)", fn, a->head_dim);
    if (a->n_seq < 0 || a->n_rows < 0)
        return fail(GR_ERR_ARG, "%s: negative sizes: n_seq %d, n_rows %d", fn, a->n_seq, a->n_rows);
    *none = a->n_seq == 0 || a->n_rows == 0;
    if (*none) return GR_OK;
    if (a->n_seq >= kMaxPositions) return fail(GR_ERR_ARG, "%s: n_seq %d above 2^30", fn, a->n_seq);
    if (a->max_rows < 1) return fail(GR_ERR_ARG, "%s: max_rows %d must be positive", fn, a->max_rows);
    int rc = check_heads(fn, a->n_heads, a->n_kv_heads, a->dtype, a->window, a->score_scale, a->n_rows);
    if (!rc && !a->seq_start) rc = fail(GR_ERR_ARG, "%s: null seq_start", fn);
    if (!rc)
        rc = check_qo(fn, a->q, a->out, a->head_dim, a->q_row_stride, a->q_head_stride, a->out_row_stride,
                      a->out_head_stride);
    if (rc) return rc;
    if (!a->k || !a->v) return fail(GR_ERR_ARG, "%s: null k or v", fn);
    if (!aligned16(a->k) || !aligned16(a->v)) return fail(GR_ERR_ARG, "%s: k and v must be 16-byte aligned", fn);
    for (int64_t s : {a->kv_row_stride, a->kv_head_stride})
        if (s < a->head_dim || s % 8)
            return fail(GR_ERR_ARG, "%s: k and v strides must be at least head_dim and multiples of 8", fn);
    if (a->kv_row_stride > kMaxRowStride)
        return fail(GR_ERR_ARG, "%s: kv_row_stride %lld above 2^22", fn, (long long)a->kv_row_stride);
    p->seqs.n_seq = a->n_seq;
    p->seqs.n_rows = a->n_rows;
    p->seqs.row_start = a->seq_start;
    p->seqs.max_len = a->n_rows;
    p->n_heads = a->n_heads;
    p->n_kv_heads = a->n_kv_heads;
    p->head_dim = a->head_dim;
    p->dtype = a->dtype;
    p->kv_dtype = a->dtype;
    p->window = a->window;
    p->scale_log2 = a->score_scale * kLog2e;
    p->q = a->q;
    p->out = a->out;
    p->q_row_stride = a->q_row_stride, p->q_head_stride = a->q_head_stride;
    p->out_row_stride = a->out_row_stride, p->out_head_stride = a->out_head_stride;
    p->k = a->k, p->v = a->v;
    p->row_stride = a->kv_row_stride, p->head_stride = a->kv_head_stride;
    p->max_rows = a->max_rows, p->max_len = a->max_rows;
    p->workspace = a->workspace;
    return check_fits(fn, *p);
}

}  // namespace

}  // namespace gr

extern "C" int gr_paged_kv_write(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_rows* rows,
                                 void* stream) {
    return gr::kv_call("gr_paged_kv_write", c, b, rows, stream, gr::launch_paged_kv_write);
}

extern "C" int gr_paged_kv_read(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_rows* rows,
                                void* stream) {
    return gr::kv_call("gr_paged_kv_read", c, b, rows, stream, gr::launch_paged_kv_read);
}

extern "C" size_t gr_paged_attention_workspace_size(const gr_paged_cache* c, const gr_paged_batch* b,
                                                    const gr_paged_attention_args* a) {
    gr::clear_error();
    gr::PagedAttnLaunch p{};
    bool none = false;
    if (gr::paged_attn_args("gr_paged_attention_workspace_size", c, b, a, &p, &none) || none) return 0;
    return gr::paged_attn_ws_bytes(p);
}

extern "C" int gr_paged_attention(const gr_paged_cache* c, const gr_paged_batch* b, const gr_paged_attention_args* a,
                                  void* stream) {
    gr::clear_error();
    gr::PagedAttnLaunch p{};
    bool none = false;
    int rc = gr::paged_attn_args("gr_paged_attention", c, b, a, &p, &none);
    if (rc || none) return rc;
    if ((rc = gr::check_ws("gr_paged_attention", a->workspace))) return rc;
    const hipError_t e = gr::launch_paged_attn(p, (hipStream_t)stream);
    return e == hipSuccess ? GR_OK : gr::hip_fail(e, "gr_paged_attention launch");
}

extern "C" size_t gr_packed_attention_workspace_size(const gr_packed_args* a) {
    gr::clear_error();
    gr::PagedAttnLaunch p{};
    bool none = false;
    if (gr::packed_args("gr_packed_attention_workspace_size", a, &p, &none) || none) return 0;
    return gr::paged_attn_ws_bytes(p);
}

extern "C" int gr_packed_attention(const gr_packed_args* a, void* stream) {
    gr::clear_error();
    gr::PagedAttnLaunch p{};
    bool none = false;
    int rc = gr::packed_args("gr_packed_attention", a, &p, &none);
    if (rc || none) return rc;
    if ((rc = gr::check_ws("gr_packed_attention", a->workspace))) return rc;
    const hipError_t e = gr::launch_paged_attn(p, (hipStream_t)stream);
    return e == hipSuccess ? GR_OK : gr::hip_fail(e, "gr_packed_attention launch");
}
