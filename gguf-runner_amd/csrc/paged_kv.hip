// Paged KV cache: storing a ragged batch's rows in their pages (rounded to 16 bits or
// quantised to Q8) and reading rows back.
//
// Both are copies bound by HBM: rows * n_kv_heads * head_dim elements in and out, for K
// and V.  A row's K (or V) is n_kv_heads * head_dim / 8 pieces of 8 elements, and a wave
// takes one row (several when a row has fewer than 64 pieces) of K or V, a piece per
// lane, so both sides move in whole lines.  The wave finds its row's sequence by a
// 64-ary search of row_start (one load for up to 63 sequences), then its page id; a wave whose
// rows are all of one sequence reads that sequence's sizes once.
//
// Calls that fill the GPU (kPagedKvFull) take U = 4 rows per wave, all requested before the
// first is used: one row leaves too few bytes in flight (Q8 pages of 3 x 20k .. 32k rows read
// as bf16: 107 us with one, 60 with 4, 71 with 2, 60 with 8), four in a small call leave CUs
// idle.  They move what no cache will hold, so whole-line stores and the pages that are read
// carry the nontemporal hint (that read: 59.3 -> 53.8 us = 5.3 TB/s; f16 pages, 4 x 16k rows:
// 105 -> 91 us; 4 x 8k rows written: 54 -> 52).  Not so the rows of a write, just computed
// (with it 4 prompts requantised and read back: 36.5 -> 38.4 us), the 8-byte stores of codes,
// half a line a row (36.5 -> 39.2), and small calls (20 x 300 rows read: 9.2 -> 11.5 us).
// Steps of a few rows are bound by the launch and three dependent loads (48 rows: 3.6 - 4.2 us).
#include "gr_common.hpp"
#include "paged_internal.hpp"

namespace gr {

constexpr int kPagedKvThreads = 256;
constexpr int kPagedKvFull = 1024;  // workgroups (four per CU) from which on a wave takes more rows

// 8 or 16 bytes; ONCE: with the nontemporal hint.
template <typename V>
using PkVec = uint32_t __attribute__((ext_vector_type(sizeof(V) / 4)));
template <typename V, bool ONCE>
__device__ __forceinline__ V pk_load(const void* p) {
    if constexpr (ONCE) return __builtin_bit_cast(V, __builtin_nontemporal_load((const PkVec<V>*)p));
    else return *(const V*)p;
}
template <bool ONCE, typename V>
__device__ __forceinline__ void pk_put(void* p, const V& x) {
    if constexpr (ONCE) __builtin_nontemporal_store(__builtin_bit_cast(PkVec<V>, x), (PkVec<V>*)p);
    else *(V*)p = x;
}

// 8 consecutive elements as they are stored: 8 (codes), 16 or 32 bytes.
template <int BYTES>
struct PkRaw {
    using V = std::conditional_t<BYTES == 8, uint2, uint4>;
    V w[BYTES == 32 ? 2 : 1];
    template <bool ONCE>
    __device__ __forceinline__ void load(const void* p) {
        w[0] = pk_load<V, ONCE>(p);
        if constexpr (BYTES == 32) w[1] = pk_load<V, ONCE>((const V*)p + 1);
    }
    template <typename T>
    __device__ __forceinline__ void floats(float* x) const {
        unpack16<T>(w[0], x);
        if constexpr (BYTES == 32) unpack16<T>(w[1], x + 4);
    }
};

template <typename T, bool ONCE>
__device__ __forceinline__ void pk_store8(typename T::storage* dst, const float* x) {
    if constexpr (T::bytes == 4) {
        pk_put<ONCE>(dst, make_float4(x[0], x[1], x[2], x[3]));
        pk_put<ONCE>(dst + 4, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = (uint32_t)from_f32<T>(x[2 * i]) | ((uint32_t)from_f32<T>(x[2 * i + 1]) << 16);
        pk_put<ONCE>(dst, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// Where a row of the batch is in the cache: page (or -1: nowhere) and row of it.
struct PagedPlace {
    int page, row;
};

// Row `row` of the lane's, seq: the sequence of a row at or before it in the wave.
__device__ __forceinline__ PagedPlace pk_place(const PagedSeqs& s, int row, int seq) {
    PagedPlace at{-1, 0};
    while (seq < s.n_seq && row >= s.row_start[seq + 1]) seq++;
    if (seq >= s.n_seq) return {-2, 0};
    const int end = seq_row(s, seq + 1);
    const int n = end - seq_row(s, seq);
    const int pos = seq_len(s, seq, n) - (end - row);
    if (pos < 0) return at;
    const int id = s.page_table[(int64_t)seq * s.table_stride + (pos >> s.page_shift)];
    at.page = (unsigned)id < (unsigned)s.n_pages ? id : -1;
    at.row = pos & ((1 << s.page_shift) - 1);
    return at;
}

// Head rows below this magnitude (2^-100) store as zeros: their scale would leave f32's normal range.
constexpr float kQ8Least = 7.8886091e-31f;

// code of x: round(x * inv) with halves away from zero, as quantize_row_q8
// (inference.rs:249-268); a NaN becomes 0, as Rust's saturating `as i8`.
__device__ __forceinline__ uint32_t pk_code(float x, float inv) {
    float r = roundf(x * inv);
    if (r < -127.0f) r = -127.0f;
    if (r > 127.0f) r = 127.0f;
    return (uint32_t)(uint8_t)(int8_t)(int)r;
}

struct KvQ8 {};

// lanes_per_row lanes (a power of two up to 64) share a row, 64 / lanes_per_row rows a wave, U
// times over: the U rows of a lane are requested together.
template <int D, typename ROWS, typename KV, bool WRITE, int U>
__global__ __launch_bounds__(kPagedKvThreads) void paged_kv_kernel(const PagedKvLaunch p, const int lanes_per_row) {
    constexpr int CPH = D / 8;  // pieces per head
    constexpr bool q8 = std::is_same_v<KV, KvQ8>;
    constexpr bool kStoreOnce = U > 1, kLoadOnce = U > 1 && !WRITE;
    using RT = typename ROWS::storage;
    const int lane = threadIdx.x & 63;
    const int unit = (int)blockIdx.x * (kPagedKvThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rpw = 64 / lanes_per_row;
    const int first = (unit >> 1) * rpw * U;  // the wave's first row; units alternate between K and V
    const int which = unit & 1;
    if (first >= p.seqs.n_rows) return;
    const int n_pieces = p.n_kv_heads * CPH;
    const int seq0 = seq_of_row(p.seqs, first);  // -1: in front of every sequence, or behind
    const int row_beg = p.seqs.row_start[0];
    if (seq0 < 0 && first >= row_beg) return;
    PagedPlace at[U];
    const int wave_end = min(first + rpw * U, p.seqs.n_rows);
    if (seq0 >= 0 && wave_end <= p.seqs.row_start[seq0 + 1]) {
        // all of one sequence (most waves of long ones): its sizes once, then the rows' page ids together
        const int end = seq_row(p.seqs, seq0 + 1);
        const int p0 = seq_len(p.seqs, seq0, 0) - end;  // position less row
        int id[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = min(first + u * rpw + lane / lanes_per_row, p.seqs.n_rows - 1);
            id[u] = p.seqs.page_table[(int64_t)seq0 * p.seqs.table_stride + (max(p0 + row, 0) >> p.seqs.page_shift)];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = first + u * rpw + lane / lanes_per_row;
            const bool there = p0 + row >= 0 && (unsigned)id[u] < (unsigned)p.seqs.n_pages;
            at[u].page = row >= p.seqs.n_rows ? -2 : there ? id[u] : -1;
            at[u].row = (p0 + row) & ((1 << p.seqs.page_shift) - 1);
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = first + u * rpw + lane / lanes_per_row;
            at[u] = PagedPlace{-2, 0};
            if (row < p.seqs.n_rows && row >= row_beg) at[u] = pk_place(p.seqs, row, max(seq0, 0));
        }
    }
    for (int c = lane % lanes_per_row; c < n_pieces; c += lanes_per_row) {
        const int g = c / CPH, i = (c % CPH) * 8;
        // every row's piece is requested before the first is used (rows without a place: some valid one)
        using ST = std::conditional_t<WRITE, ROWS, std::conditional_t<q8, F16, KV>>;
        PkRaw<WRITE ? ROWS::bytes * 8 : q8 ? 8 : ST::bytes * 8> raw[U];
        float sc[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = min(first + u * rpw + lane / lanes_per_row, p.seqs.n_rows - 1);
            const int64_t page = max(at[u].page, 0);
            if constexpr (WRITE) {
                raw[u].template load<kLoadOnce>((const RT*)p.rows[which] + (int64_t)row * p.rows_row_stride + g * p.rows_head_stride + i);
            } else {
                const int64_t e = page * p.page_stride + (int64_t)at[u].row * p.row_stride + g * p.head_stride + i;
                if constexpr (q8) {
                    raw[u].template load<kLoadOnce>((const int8_t*)p.pages[which] + e);
                    sc[u] = p.scale[which][page * p.scale_page_stride + (int64_t)at[u].row * p.scale_row_stride +
                                           g * p.scale_head_stride];
                } else {
                    raw[u].template load<kLoadOnce>((const typename ST::storage*)p.pages[which] + e);
                }
            }
        }
        float x[U][8];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if constexpr (!WRITE && q8) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[u][j] = (float)(int8_t)(raw[u].w[0].x >> (8 * j)) * sc[u];
                    x[u][j + 4] = (float)(int8_t)(raw[u].w[0].y >> (8 * j)) * sc[u];
                }
            } else {
                raw[u].template floats<ST>(x[u]);
            }
            if (at[u].page < 0) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[u][j] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int row = first + u * rpw + lane / lanes_per_row;
            if constexpr (!WRITE) {
                if (at[u].page != -2)
                    pk_store8<ROWS, kStoreOnce>((RT*)p.rows[which] + (int64_t)row * p.rows_row_stride + g * p.rows_head_stride + i, x[u]);
            } else {
                const int64_t e = (int64_t)at[u].page * p.page_stride + (int64_t)at[u].row * p.row_stride + g * p.head_stride + i;
                if constexpr (q8) {
                    float amax = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(x[u][j]));
                    // a head's CPH pieces are CPH adjacent lanes (lanes_per_row is a multiple of CPH)
#pragma unroll
                    for (int m = CPH / 2; m >= 1; m >>= 1) amax = fmaxf(amax, shfl_xor(amax, m));
                    if (at[u].page < 0) continue;
                    if (amax < kQ8Least) amax = 0.0f;
                    const float inv = amax == 0.0f ? 0.0f : __fdiv_rn(1.0f, amax) * 127.0f;
                    uint32_t w0 = 0, w1 = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        w0 |= pk_code(x[u][j], inv) << (8 * j);
                        w1 |= pk_code(x[u][j + 4], inv) << (8 * j);
                    }
                    *(uint2*)((int8_t*)p.pages[which] + e) = make_uint2(w0, w1);
                    if (i == 0)
                        p.scale[which][(int64_t)at[u].page * p.scale_page_stride + (int64_t)at[u].row * p.scale_row_stride +
                                       g * p.scale_head_stride] = amax == 0.0f ? 1.0f : amax * (1.0f / 127.0f);
                } else if (at[u].page >= 0) {
                    pk_store8<KV, kStoreOnce>((typename KV::storage*)p.pages[which] + e, x[u]);
                }
            }
        }
    }
}

template <int D, typename ROWS, typename KV, bool WRITE>
static hipError_t launch_kv(const PagedKvLaunch& p, hipStream_t st) {
    const int pieces = p.n_kv_heads * (D / 8);
    int lpr = 64;
    while (lpr > D / 8 && lpr / 2 >= pieces) lpr /= 2;
    auto wgs = [&](int rows) {  // for waves of that many rows
        const int64_t units = 2 * (((int64_t)p.seqs.n_rows + rows - 1) / rows);
        return (units + kPagedKvThreads / 64 - 1) / (kPagedKvThreads / 64);
    };
    constexpr int U = 4;
    const int rows = 64 / lpr;
    if (wgs(rows * U) >= kPagedKvFull)
        paged_kv_kernel<D, ROWS, KV, WRITE, U><<<dim3((unsigned)wgs(rows * U)), kPagedKvThreads, 0, st>>>(p, lpr);
    else
        paged_kv_kernel<D, ROWS, KV, WRITE, 1><<<dim3((unsigned)wgs(rows)), kPagedKvThreads, 0, st>>>(p, lpr);
    return hipGetLastError();
}

template <int D, typename ROWS, bool WRITE>
static hipError_t launch_kv_d(const PagedKvLaunch& p, hipStream_t st) {
    switch (p.kv_dtype) {
        case GR_DTYPE_F16: return launch_kv<D, ROWS, F16, WRITE>(p, st);
        case GR_DTYPE_BF16: return launch_kv<D, ROWS, BF16, WRITE>(p, st);
        default: return launch_kv<D, ROWS, KvQ8, WRITE>(p, st);
    }
}

template <typename ROWS, bool WRITE>
static hipError_t launch_kv_rows(const PagedKvLaunch& p, hipStream_t st) {
    switch (p.head_dim) {
        case 64: return launch_kv_d<64, ROWS, WRITE>(p, st);
        case 128: return launch_kv_d<128, ROWS, WRITE>(p, st);
        default: return launch_kv_d<256, ROWS, WRITE>(p, st);
    }
}

template <bool WRITE>
static hipError_t launch_kv_any(const PagedKvLaunch& p, hipStream_t st) {
    switch (p.rows_dtype) {
        case GR_DTYPE_F32: return launch_kv_rows<F32, WRITE>(p, st);
        case GR_DTYPE_F16: return launch_kv_rows<F16, WRITE>(p, st);
        default: return launch_kv_rows<BF16, WRITE>(p, st);
    }
}

hipError_t launch_paged_kv_write(const PagedKvLaunch& p, hipStream_t st) { return launch_kv_any<true>(p, st); }
hipError_t launch_paged_kv_read(const PagedKvLaunch& p, hipStream_t st) { return launch_kv_any<false>(p, st); }

}  // namespace gr
