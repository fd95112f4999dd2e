// Attention of a ragged batch's rows over a paged KV cache, or over the batch's own
// packed K / V rows.  One wave per (row, query head): a key at a time, online softmax.
#include "gr_common.hpp"
#include "paged_internal.hpp"

namespace gr {

template <typename T, int D, int KV>  // KV: 0 packed rows, 1 16-bit pages, 2 Q8 pages
__global__ __launch_bounds__(64) void paged_attn_kernel(const PagedAttnLaunch p) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x;
    const int row = blockIdx.x, h = blockIdx.y;
    const int seq = seq_of_row(p.seqs, row);
    if (seq < 0) return;
    const int beg = seq_row(p.seqs, seq), end = seq_row(p.seqs, seq + 1);
    const int pos = seq_len(p.seqs, seq, end - beg) - (end - row);
    const int lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
    const int g = h / (p.n_heads / p.n_kv_heads);
    float q[E], o[E];
    const uint16_t* qr = (const uint16_t*)p.q + (int64_t)row * p.q_row_stride + h * p.q_head_stride;
#pragma unroll
    for (int e = 0; e < E; e++) q[e] = to_f32<T>(qr[lane * E + e]), o[e] = 0.0f;
    float m = -1e30f, l = 0.0f;
    for (int t = lo; t <= pos; t++) {
        int64_t at, sc = 0;
        if constexpr (KV == 0) {
            at = (int64_t)(beg + t) * p.row_stride;
        } else {
            const int id = p.seqs.page_table[(int64_t)seq * p.seqs.table_stride + (t >> p.seqs.page_shift)];
            if ((unsigned)id >= (unsigned)p.seqs.n_pages) continue;
            const int r = t & ((1 << p.seqs.page_shift) - 1);
            at = (int64_t)id * p.page_stride + (int64_t)r * p.row_stride;
            sc = (int64_t)id * p.scale_page_stride + (int64_t)r * p.scale_row_stride + g * p.scale_head_stride;
        }
        at += g * p.head_stride + lane * E;
        float k[E], v[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            if constexpr (KV == 2) {
                k[e] = (float)((const int8_t*)p.k)[at + e];
                v[e] = (float)((const int8_t*)p.v)[at + e];
            } else {
                k[e] = to_f32<T>(((const uint16_t*)p.k)[at + e]);
                v[e] = to_f32<T>(((const uint16_t*)p.v)[at + e]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s += q[e] * k[e];
        s = wave_sum<64>(s) * p.scale_log2;
        float vs = 1.0f;
        if constexpr (KV == 2) s *= p.k_scale[sc], vs = p.v_scale[sc];
        const float mn = fmaxf(m, s);
        const float a = exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * a + w;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * a + w * vs * v[e];
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    uint16_t* out = (uint16_t*)p.out + (int64_t)row * p.out_row_stride + h * p.out_head_stride;
#pragma unroll
    for (int e = 0; e < E; e++) out[lane * E + e] = from_f32<T>(o[e] * inv);
}

size_t paged_attn_ws_bytes(const PagedAttnLaunch&) { return 256; }

template <typename T, int D>
static hipError_t launch_attn(const PagedAttnLaunch& p, hipStream_t st) {
    const dim3 grid((unsigned)p.seqs.n_rows, (unsigned)p.n_heads);
    if (!p.seqs.page_table) paged_attn_kernel<T, D, 0><<<grid, 64, 0, st>>>(p);
    else if (p.kv_dtype != GR_DTYPE_Q8) paged_attn_kernel<T, D, 1><<<grid, 64, 0, st>>>(p);
    else paged_attn_kernel<T, D, 2><<<grid, 64, 0, st>>>(p);
    return hipGetLastError();
}

template <typename T>
static hipError_t launch_attn_d(const PagedAttnLaunch& p, hipStream_t st) {
    return p.head_dim == 64 ? launch_attn<T, 64>(p, st)
                            : p.head_dim == 128 ? launch_attn<T, 128>(p, st) : launch_attn<T, 256>(p, st);
}

hipError_t launch_paged_attn(const PagedAttnLaunch& p, hipStream_t st) {
    return p.dtype == GR_DTYPE_F16 ? launch_attn_d<F16>(p, st) : launch_attn_d<BF16>(p, st);
}

}  // namespace gr
