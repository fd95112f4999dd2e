// Attention of a ragged batch's rows over a paged KV cache, or over the batch's own packed
// K / V rows, on the matrix cores.
//
// Rows of a sequence and KV head g are packed (token, query head of g's group): row r is
// token r / group, head g * group + r % group, so a K / V tile is read once for the whole
// group and one token of a wide group fills a wave.  A block is BM = 32 * RW of them.  A
// workgroup is RW row groups of 32 rows times KH key parts: with KH > 1 (few rows) its waves
// take alternate 32-key sub-tiles of every BN-key tile and merge at the end.  As in the
// contiguous prefill, S^T = K Q^T and O^T += V^T P^T run on v_mfma_f32_32x32x16 with one row
// per lane column, K and V row-major in LDS, 16-byte chunks XOR-swizzled, V read through the
// transposing LDS loads.  16-bit tiles go from HBM straight into LDS, each wave's run of rows
// from its page; Q8 codes go through registers and become exact f16 values on the way.
//
// The online softmax is in log2 units, m and l in f32:
//   s = c q.k  (c = score_scale * log2 e, applied in f32: the operands are the caller's exact
//   16-bit values),  p = 2^(s - m),  o = sum p v / sum p.
// Q8: with weights w = p * v_scale the products are sum w * code and sum w / v_scale, so m is
// the maximum of s + log2(v_scale) and w is what is rounded to f16, in f16's range whatever
// the scales are.  Rounding p (w) to 16 bits is what the matrix product costs: half a step
// per weight, errors that average out over the keys; the sum uses the rounded weights too
// (16-bit pages), so that a common factor cancels.
//
// Two schedules.  ORDERED: one block per workgroup, longest first.  STREAM: the blocks'
// tiles, one after another, are cut into one equal range per workgroup; a block that a cut
// divides leaves unnormalised partials (O, m, l) which paged_combine_kernel joins.
#pragma once

#include <type_traits>

#include "gr_common.hpp"
#include "paged_internal.hpp"

namespace gr {

typedef _Float16 pa_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_half2 __attribute__((ext_vector_type(2)));
typedef float pa_float2 __attribute__((ext_vector_type(2)));
typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x16 __attribute__((ext_vector_type(16)));
typedef short pa_i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short pa_u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int pa_u32x4 __attribute__((ext_vector_type(4)));
#define GR_PA_LDS __attribute__((address_space(3)))

template <typename DT>
struct PaMat;
template <>
struct PaMat<F16> {
    static constexpr uint32_t kInf = 0x7c00u;
    static __device__ __forceinline__ pa_f32x16 mma(const uint4& a, const uint4& b, const pa_f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pa_half8, a), __builtin_bit_cast(pa_half8, b),
                                                      c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(pa_float2{lo, hi}, pa_half2));
    }
    // c + both halves of w
    static __device__ __forceinline__ float add2(uint32_t w, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(pa_half2, w), pa_half2{1.0f16, 1.0f16}, c, false);
    }
};
template <>
struct PaMat<BF16> {
    static constexpr uint32_t kInf = 0x7f80u;
    static __device__ __forceinline__ pa_f32x16 mma(const uint4& a, const uint4& b, const pa_f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pa_bf16x8, a),
                                                       __builtin_bit_cast(pa_bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
    static __device__ __forceinline__ float add2(uint32_t w, float c) {
        return c + (__uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u));
    }
};

enum PaSrc { kPaPacked = 0, kPaPages = 1, kPaPagesQ8 = 2 };

// Tiles of a kernel: RW row groups x KH key parts, BN keys, waves per SIMD it is built for.
template <int D_, int RW_, int KH_, int BN_, int OCC_>
struct PaTile {
    static constexpr int D = D_, RW = RW_, KH = KH_, BN = BN_, OCC = OCC_;
    static constexpr int NW = RW * KH, NT = NW * 64, BM = RW * 32;
    static_assert(BN % (32 * KH) == 0, "every key part has its sub-tiles");
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t pa_rsrc(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)0xffffffff, 0x00020000);
}
__device__ __forceinline__ void pa_dma16(__amdgpu_buffer_rsrc_t r, uint16_t* lds, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (GR_PA_LDS void*)lds, 16, voff, 0, 0, 0);
#endif
}
__device__ __forceinline__ uint4 pa_load16(__amdgpu_buffer_rsrc_t r, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0));
#else
    return uint4{};
#endif
}
__device__ __forceinline__ void pa_wait_vmem() { __builtin_amdgcn_s_waitcnt(0x0F70); }
__device__ __forceinline__ float pa_xmax32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_xsum32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Position of 16-byte chunk c of tile row r: c ^ pa_swz<D>(r & 15).  K reads (16 consecutive
// rows, one chunk) and V transpose reads (4 rows x 4 chunks) then touch distinct banks; a
// head_dim-64 row is 8 chunks, half the banks, hence its own 3-bit form.
template <int D>
__device__ __forceinline__ int pa_swz(int r) {
    if constexpr (D == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r << 2) ^ (r << 1) ^ (r >> 2)) & 15;
}

// 8 int8 codes -> 8 exact f16: sign bit flipped, u = code + 128 becomes the f16 1024 + u
// under the exponent byte 0x64, less 1152.
__device__ __forceinline__ uint4 pa_cvt8(uint32_t x, uint32_t y) {
    const pa_half2 bias = {1152.0f16, 1152.0f16};
    auto two = [&](uint32_t w, uint32_t sel) {
        const uint32_t spread = __builtin_amdgcn_perm(0x64646464u, w, sel);
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(pa_half2, spread) - bias);
    };
    const uint32_t a = x ^ 0x80808080u, b = y ^ 0x80808080u;
    return make_uint4(two(a, 0x04010400u), two(a, 0x04030402u), two(b, 0x04010400u), two(b, 0x04030402u));
}

constexpr float kPaNone = -1e30f;     // m of a row that has seen no key
constexpr float kPaLazy = 8.0f;       // m is only raised for tile maxima this far above it: p <= 2^8
constexpr float kPaLeastScale = 7.8886091e-31f;  // 2^-100: smaller v_scales count as this in m and l

// ---------------------------------------------------------------- schedules

// One block's place: rows [row0, row0 + n_pr) packed, keys.
struct PaBlock {
    int seq, rb, g;
    int beg, n, p0;      // first row, rows, position of the first row
    int t_first, kend;   // keys [.., kend), tiles start at t_first
    int n_tiles;
};

template <int BM, int BN>
__device__ __forceinline__ void pa_block(const PagedAttnLaunch& p, PaBlock& b) {
    const int group = p.n_heads / p.n_kv_heads;
    b.beg = seq_row(p.seqs, b.seq);
    b.n = seq_row(p.seqs, b.seq + 1) - b.beg;
    const int len = seq_len(p.seqs, b.seq, b.n);
    b.p0 = len - b.n;
    const int tok0 = b.rb * BM / group, tok1 = (min((b.rb + 1) * BM, b.n * group) - 1) / group;
    b.kend = max(b.p0 + tok1 + 1, 0);
    const int lo = p.window > 0 ? max(b.p0 + tok0 + 1 - p.window, 0) : 0;
    b.t_first = lo / BN * BN;
    b.n_tiles = b.kend > b.t_first ? (b.kend - b.t_first + BN - 1) / BN : 0;
}

// Blocks of sequence s and the tiles that each of them counts in the stream (at least its
// longest one's, so that the cuts fall evenly: 1 for a sequence of no keys).
template <int BM, int BN>
__device__ __forceinline__ void pa_counts(const PagedAttnLaunch& p, int s, int& nb, int& vt) {
    nb = vt = 0;
    if (s >= p.seqs.n_seq) return;
    const int group = p.n_heads / p.n_kv_heads;
    const int n = max(seq_row(p.seqs, s + 1) - seq_row(p.seqs, s), 0);
    nb = (n * group + BM - 1) / BM;
    const int len = seq_len(p.seqs, s, n);
    vt = (len + BN - 1) / BN;
    if (p.window > 0) {
        const int64_t most = ((int64_t)p.window + (BM + group - 1) / group + BN - 1) / BN + 1;
        if (vt > most) vt = (int)most;
    }
    vt = max(vt, 1);
}

__device__ __forceinline__ int64_t pa_scan(int64_t x) {  // inclusive, over the wave
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
}

// The stream: sequence s takes cost(s) = n_kv_heads * nb(s) * vt(s) places, in that order.
template <int BM, int BN>
__device__ __forceinline__ int64_t pa_stream_total(const PagedAttnLaunch& p) {
    int64_t t = 0;
    for (int s0 = 0; s0 < p.seqs.n_seq; s0 += 64) {
        int nb, vt;
        pa_counts<BM, BN>(p, s0 + (threadIdx.x & 63), nb, vt);
        t += __shfl(pa_scan((int64_t)nb * vt * p.n_kv_heads), 63, 64);
    }
    return t;
}

// Where place x (< total) of the stream is: block, its vt and x's offset in it.
struct PaPlace {
    int seq, rb, g, vt;
    int64_t at;
};
template <int BM, int BN>
__device__ __forceinline__ PaPlace pa_stream_find(const PagedAttnLaunch& p, int64_t x) {
    PaPlace r{0, 0, 0, 1, 0};
    for (int s0 = 0; s0 < p.seqs.n_seq; s0 += 64) {
        int nb, vt;
        pa_counts<BM, BN>(p, s0 + (threadIdx.x & 63), nb, vt);
        const int64_t cost = (int64_t)nb * vt * p.n_kv_heads;
        const int64_t incl = pa_scan(cost);
        const int64_t all = __shfl(incl, 63, 64);
        if (x < all) {
            const int l = __ffsll((unsigned long long)__ballot(x < incl)) - 1;
            const int64_t in = x - __shfl(incl - cost, l, 64);
            r.seq = __builtin_amdgcn_readfirstlane(s0 + l);
            nb = __builtin_amdgcn_readfirstlane(__shfl(nb, l, 64));
            r.vt = __builtin_amdgcn_readfirstlane(__shfl(vt, l, 64));
            const int64_t blk = in / r.vt;
            r.at = in - blk * r.vt;
            r.g = __builtin_amdgcn_readfirstlane((int)(blk / nb));
            r.rb = __builtin_amdgcn_readfirstlane((int)(blk - (int64_t)r.g * nb));
            break;
        }
        x -= all;
    }
    return r;
}

// Workgroup b of a stream launch as a place among them: XCD b % 8 gets a run of
// neighbouring ranges (the blocks of a sequence's KV head share its tiles in one L2).
__device__ __forceinline__ int pa_stream_rank(int b, int g) {
    const int per = g / 8;  // workgroups of a launch: a multiple of 8
    return (b & 7) * per + (b >> 3);
}
__device__ __forceinline__ int64_t pa_stream_q(int64_t total, int g) { return (total + g - 1) / g; }

// The real tiles [a, b) of a block of n_tiles for virtual ones [va, vb) of vt.
__device__ __forceinline__ int pa_real(int64_t v, int n_tiles, int vt) { return (int)(v * n_tiles / vt); }

// ---------------------------------------------------------------- the kernel

template <typename DT, typename T, int SRC, bool STREAM>
__global__ __launch_bounds__(T::NT, T::OCC) void paged_attn_kernel(const PagedAttnLaunch p) {
    constexpr int D = T::D, BN = T::BN, BM = T::BM, RW = T::RW, KH = T::KH, NT = T::NT;
    constexpr bool kQ8 = SRC == kPaPagesQ8;
    using M = PaMat<DT>;
    constexpr int CPR = D / 8;              // 16-byte chunks per tile row
    constexpr int SCPR = kQ8 ? D / 16 : CPR;  // chunks per source row
    constexpr int LD = BN * SCPR / NT;      // source chunks per thread per K (or V) tile
    constexpr int RPU = NT / SCPR;          // rows filled by one round of the workgroup
    constexpr int RPV = 64 / SCPR;          // ... of a wave: inside one run of 16 rows, so one page
    constexpr int EB = kQ8 ? 1 : 2;         // bytes per stored element
    static_assert(LD >= 1 && LD <= 32 && BN * SCPR % NT == 0 && BN / 16 <= 32 && BN <= NT, "tile shape");

    __shared__ __attribute__((aligned(16))) uint16_t Ks0[BN * D];
    __shared__ __attribute__((aligned(16))) uint16_t Ks1[BN * D];
    __shared__ __attribute__((aligned(16))) uint16_t Vs0[BN * D];
    __shared__ __attribute__((aligned(16))) uint16_t Vs1[BN * D];
    // Q8: c * k_scale, log2 v_scale, 1 / v_scale of the tile's keys
    __shared__ __attribute__((aligned(16))) float Sc0[kQ8 ? 3 * BN : 4];
    __shared__ __attribute__((aligned(16))) float Sc1[kQ8 ? 3 * BN : 4];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = KH > 1 ? wave % RW : wave, kh = KH > 1 ? wave / RW : 0;
    const int ln = lane & 31, lg = lane >> 5;
    const int group = p.n_heads / p.n_kv_heads;
    const int ps1 = (1 << p.seqs.page_shift) - 1;

    // this thread's source chunks: row wave * RPV + lane / SCPR + u * RPU of the tile
    const int lrow = lane / SCPR;
    int col[LD];  // byte offset in the source row
#pragma unroll
    for (int u = 0; u < LD; u++) {
        const int r = wave * RPV + lrow + u * RPU;
        col[u] = kQ8 ? lane % SCPR * 16 : ((lane % SCPR) ^ pa_swz<D>(r & 15)) * 16;
    }
    const int rsb = (int)p.row_stride * EB;
    const int swz_k = pa_swz<D>(ln & 15);
    const int gi = lane & 15;
    const int v_chunk = 2 * ((lane >> 4) & 1) + ((gi & 3) >> 1);
    int v_base[2], v_swz[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int r = 8 * b + 4 * lg + (gi >> 2);
        v_base[b] = r * D + (gi & 1) * 4;
        v_swz[b] = pa_swz<D>(r & 15);
    }

    // ------------------------------------------------ the workgroup's range
    int64_t pos = 0, stop = 1;  // STREAM: places of the stream
    int64_t total = 0, q_len = 0;
    int rank = 0;
    PaPlace pl{};
    if constexpr (STREAM) {
        total = pa_stream_total<BM, BN>(p);
        rank = pa_stream_rank(blockIdx.x, gridDim.x);
        q_len = pa_stream_q(total, gridDim.x);
        pos = rank * q_len;
        stop = min(total, pos + q_len);
    }

    while (pos < stop) {
        PaBlock blk;
        int it0 = 0, it1 = 0;
        bool whole = true;
        int slot = 0;
        if constexpr (STREAM) {
            pl = pa_stream_find<BM, BN>(p, pos);
            blk.seq = pl.seq, blk.rb = pl.rb, blk.g = pl.g;
            pa_block<BM, BN>(p, blk);
            const int64_t vb = min((int64_t)pl.vt, pl.at + (stop - pos));
            whole = pl.at == 0 && vb == pl.vt;
            slot = 2 * rank + (pl.at == 0 ? 1 : 0);
            it0 = pa_real(pl.at, blk.n_tiles, pl.vt);
            it1 = pa_real(vb, blk.n_tiles, pl.vt);
            pos += vb - pl.at;
            if (!whole && it0 == it1) continue;  // the joining kernel knows that this piece is empty
        } else {
            pos = 1;
            // the item's place in the order
            const int hx = p.n_kv_heads;
            int idx, g;
            const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
            if (8 % hx == 0) {  // 8 / hx XCDs take the blocks of one KV head
                g = x % hx;
                idx = i * (8 / hx) + x / hx;
            } else if (hx % 8 == 0) {
                g = x + 8 * (i % (hx / 8));
                idx = i / (hx / 8);
            } else {
                g = blockIdx.x % hx;
                idx = blockIdx.x / hx;
            }
            int seq = -1, rb = 0;
            if (p.seqs.n_seq <= 64) {
                // longest first: blocks by their number from the highest, C(l) = blocks numbered l or more
                int nb, vt;
                pa_counts<BM, BN>(p, lane, nb, vt);
                auto count = [&](int l) {
                    int c = max(nb - l, 0);
#pragma unroll
                    for (int m = 32; m >= 1; m >>= 1) c += __shfl_xor(c, m, 64);
                    return __builtin_amdgcn_readfirstlane(c);
                };
                if (idx >= count(0)) return;
                int lo = 0, hi = 1;  // the highest l with C(l) > idx
                while (count(hi) > idx) hi *= 2;
                while (hi - lo > 1) {
                    const int mid = lo + (hi - lo) / 2;
                    if (count(mid) > idx) lo = mid;
                    else hi = mid;
                }
                rb = lo;
                int k = idx - count(lo + 1);  // the k-th sequence with a block of this number
                const uint64_t has = __ballot(nb > lo);
                const int before = __popcll(has & ((1ull << lane) - 1));
                seq = __ffsll((unsigned long long)__ballot(nb > lo && before == k)) - 1;
            } else {
                for (int s0 = 0; s0 < p.seqs.n_seq; s0 += 64) {
                    int nb, vt;
                    pa_counts<BM, BN>(p, s0 + lane, nb, vt);
                    const int incl = (int)pa_scan(nb);
                    const int all = __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64));
                    if (idx < all) {
                        const int l = __ffsll((unsigned long long)__ballot(idx < incl)) - 1;
                        seq = s0 + l;
                        rb = __builtin_amdgcn_readfirstlane(__shfl(incl, l, 64)) - 1 - idx;  // its last block first
                        break;
                    }
                    idx -= all;
                }
                if (seq < 0) return;
            }
            blk.seq = __builtin_amdgcn_readfirstlane(seq);
            blk.rb = rb;
            blk.g = g;
            pa_block<BM, BN>(p, blk);
            it1 = blk.n_tiles;
        }

        const int n_pr = blk.n * group;
        const int r0 = blk.rb * BM;
        const int wr0 = r0 + rw * 32;
        const bool wave_active = wr0 < n_pr;
        const int my_row = wr0 + ln;
        const bool row_ok = my_row < n_pr;
        const int row_c = min(my_row, n_pr - 1);
        const int my_tok = row_c / group;
        const int my_h = blk.g * group + (row_c - my_tok * group);
        const int my_pos = blk.p0 + my_tok;
        const int my_lo = p.window > 0 ? max(my_pos + 1 - p.window, 0) : 0;
        const unsigned my_seen = (unsigned)max(my_pos + 1 - my_lo, 0);
        // the wave's rows: positions rise with the row
        const int hi_min = __builtin_amdgcn_readfirstlane(my_pos);
        const int hi_max = __builtin_amdgcn_readlane(my_pos, 31);
        const int lo_min = __builtin_amdgcn_readfirstlane(my_lo);
        const int lo_max = __builtin_amdgcn_readlane(my_lo, 31);

        const int t_begin = blk.t_first + it0 * BN;
        const int n_tiles = it1 - it0;
        const int last = blk.kend - 1;
        const int32_t* table = SRC == kPaPacked ? nullptr : p.seqs.page_table + (int64_t)blk.seq * p.seqs.table_stride;
        const char* const kb0 = (const char*)p.k + (int64_t)blk.g * p.head_stride * EB;
        const char* const vb0 = (const char*)p.v + (int64_t)blk.g * p.head_stride * EB;

        // Page ids of a tile: lane u < LD the page of this wave's rows of round u, lane 32 + j
        // that of keys 16 j .. 16 j + 15.
        auto load_ids = [&](int t0) {
            if constexpr (SRC == kPaPacked) return 0;
            const int key = t0 + (lane < 32 ? wave * RPV + lane * RPU : (lane - 32) * 16);
            return table[min(key, last) >> p.seqs.page_shift];
        };
        // Q8: the page of key t0 + tid
        auto load_key_id = [&](int t0) {
            if constexpr (!kQ8) return 0;
            return table[min(t0 + tid, last) >> p.seqs.page_shift];
        };
        // 16-key runs of the tile whose page is not there
        auto bad_runs = [&](int ids) {
            if constexpr (SRC == kPaPacked) return 0u;
            return (unsigned)(__ballot((unsigned)ids >= (unsigned)p.seqs.n_pages) >> 32) & ((1u << (BN / 16)) - 1);
        };

        // For round u of the tile at t0: the scalar byte offset of this wave's run of rows, and
        // the rows the lane's offset is clamped to (rows past the last key repeat it: they are
        // masked, and must not be read).
        auto run_of = [&](int t0, int ids, int u, int& room) __attribute__((always_inline)) {
            const int f = t0 + wave * RPV + u * RPU;
            const int fc = min(f, last);
            room = last - fc;
            if constexpr (SRC == kPaPacked) {
                return (int64_t)(blk.beg + fc) * p.row_stride * EB;
            } else {
                int id = __builtin_amdgcn_readlane(ids, u);
                if ((unsigned)id >= (unsigned)p.seqs.n_pages) id = 0;
                return ((int64_t)id * p.page_stride + (int64_t)(fc & ps1) * p.row_stride) * EB;
            }
        };
        auto dma_tile = [&](int t0, int ids, uint16_t* kd, uint16_t* vd) __attribute__((always_inline)) {
            const bool full = t0 + BN - 1 <= last;
#pragma unroll
            for (int u = 0; u < LD; u++) {
                int room;
                const int64_t at = run_of(t0, ids, u, room);
                const int off = (full ? lrow : min(lrow, room)) * rsb + col[u];
                const int dst = (wave * 64 + u * NT) * 8;
                pa_dma16(pa_rsrc(kb0 + at), kd + dst, off);
                pa_dma16(pa_rsrc(vb0 + at), vd + dst, off);
            }
        };
        uint4 kr[kQ8 ? LD : 1], vr[kQ8 ? LD : 1];
        float ks_r = 0.0f, vs_r = 1.0f;
        auto load_q8 = [&](int t0, int ids, int key_id) __attribute__((always_inline)) {
            if constexpr (kQ8) {
                const bool full = t0 + BN - 1 <= last;
#pragma unroll
                for (int u = 0; u < LD; u++) {
                    int room;
                    const int64_t at = run_of(t0, ids, u, room);
                    const int off = (full ? lrow : min(lrow, room)) * rsb + col[u];
                    kr[u] = pa_load16(pa_rsrc(kb0 + at), off);
                    vr[u] = pa_load16(pa_rsrc(vb0 + at), off);
                }
                if (tid < BN) {
                    const int id = (unsigned)key_id < (unsigned)p.seqs.n_pages ? key_id : 0;
                    const int64_t at = (int64_t)id * p.scale_page_stride +
                                       (int64_t)(min(t0 + tid, last) & ps1) * p.scale_row_stride +
                                       (int64_t)blk.g * p.scale_head_stride;
                    ks_r = p.k_scale[at];
                    vs_r = p.v_scale[at];
                }
            }
        };
        auto store_q8 = [&](uint16_t* kd, uint16_t* vd, float* sc) __attribute__((always_inline)) {
            if constexpr (kQ8) {
#pragma unroll
                for (int u = 0; u < LD; u++) {
                    const int r = wave * RPV + lrow + u * RPU;
                    const int c = lane % SCPR * 2;
                    const int s = pa_swz<D>(r & 15);
                    *(uint4*)(kd + r * D + ((c ^ s) << 3)) = pa_cvt8(kr[u].x, kr[u].y);
                    *(uint4*)(kd + r * D + (((c + 1) ^ s) << 3)) = pa_cvt8(kr[u].z, kr[u].w);
                    *(uint4*)(vd + r * D + ((c ^ s) << 3)) = pa_cvt8(vr[u].x, vr[u].y);
                    *(uint4*)(vd + r * D + (((c + 1) ^ s) << 3)) = pa_cvt8(vr[u].z, vr[u].w);
                }
                if (tid < BN) {
                    const float vs = fmaxf(vs_r, kPaLeastScale);
                    sc[tid] = ks_r * p.scale_log2;
                    sc[BN + tid] = __builtin_amdgcn_logf(vs);
                    sc[2 * BN + tid] = 1.0f / vs;
                }
            }
        };

        __syncthreads();  // the block before is done with every LDS buffer
        int ids = 0, key_id = 0;
        unsigned bad0 = 0, bad1 = 0;
        if (n_tiles > 0) {
            ids = load_ids(t_begin);
            key_id = load_key_id(t_begin);
            bad0 = bad_runs(ids);
            if constexpr (kQ8) load_q8(t_begin, ids, key_id);
            else dma_tile(t_begin, ids, Ks0, Vs0);
            if (n_tiles > 1) {
                ids = load_ids(t_begin + BN);
                key_id = load_key_id(t_begin + BN);
            }
        }

        // ------------------------------------------------ Q: B operands, one row per lane column
        uint4 qf[D / 16];
        float q_mul = 1.0f;  // Q8: what the scores are multiplied by (bf16 rows are put in f16's range)
        {
            const uint16_t* qr = (const uint16_t*)p.q + (int64_t)(blk.beg + my_tok) * p.q_row_stride +
                                 (int64_t)my_h * p.q_head_stride;
#pragma unroll
            for (int c = 0; c < D / 16; c++) qf[c] = *(const uint4*)(qr + 16 * c + 8 * lg);
            if constexpr (kQ8) {
                if (p.dtype == GR_DTYPE_BF16) {
                    // bf16's 8 significant bits fit f16's 11: exact but for values 2^-24 below the row's largest
                    float big = 0.0f;
#pragma unroll
                    for (int c = 0; c < D / 16; c++) {
                        float x[8];
                        unpack16<BF16>(qf[c], x);
#pragma unroll
                        for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[e]));
                    }
                    big = pa_xmax32(big);
                    const int ex = max((int)((__float_as_uint(big) >> 23) & 0xffu) - 127, -100);
                    const int sh = min(ex, 100);
                    const float down = __uint_as_float((uint32_t)(127 - sh) << 23);
                    q_mul = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
                    for (int c = 0; c < D / 16; c++) {
                        float x[8];
                        unpack16<BF16>(qf[c], x);
                        qf[c] = make_uint4(M::pack2(x[0] * down, x[1] * down), M::pack2(x[2] * down, x[3] * down),
                                           M::pack2(x[4] * down, x[5] * down), M::pack2(x[6] * down, x[7] * down));
                    }
                }
            }
        }

        pa_f32x16 o[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[dt][e] = 0.0f;
        float mrow = kPaNone, lrow_sum = 0.0f;
        const float c2 = p.scale_log2;

        // One 32-key sub-tile: keys ts .. ts + 31, rows 32 sb .. of the tile; bad: its two
        // 16-key runs that are not there.
        auto subtile = [&](const uint16_t* kb, const uint16_t* vb, const float* sc, int sb, int ts, unsigned bad) __attribute__((always_inline)) {
            const pa_f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            __builtin_amdgcn_s_setprio(1);
            pa_f32x16 s;
            const uint16_t* krow = kb + (32 * sb + ln) * D;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const uint4 a = *(const uint4*)(krow + (((2 * i + lg) ^ swz_k) << 3));
                s = M::mma(a, qf[i], i == 0 ? zero : s);
            }
            auto load_va = [&](int dt, int t) __attribute__((always_inline)) {
                pa_i16x4 part[2];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int off = (32 * sb + 16 * t) * D + v_base[b] + (((4 * dt + v_chunk) ^ v_swz[b]) << 3);
                    part[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GR_PA_LDS pa_i16x4*)(vb + off));
                }
                const uint2 lo = __builtin_bit_cast(uint2, part[0]);
                const uint2 hi = __builtin_bit_cast(uint2, part[1]);
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            constexpr bool kPreV = D <= 128;
            uint4 va[kPreV ? D / 32 : 1][2];
            if constexpr (kPreV) {
#pragma unroll
                for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                    for (int t = 0; t < 2; t++) va[dt][t] = load_va(dt, t);
            }
            __builtin_amdgcn_s_setprio(0);
            // element e is key ts + 8 (e / 4) + 4 lg + e % 4
            if constexpr (kQ8) {
                const float4* ks4 = (const float4*)(sc + 32 * sb + 4 * lg);
                const float4* lv4 = (const float4*)(sc + BN + 32 * sb + 4 * lg);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 a = ks4[2 * j], b = lv4[2 * j];
                    s[4 * j + 0] = fmaf(s[4 * j + 0] * q_mul, a.x, b.x);
                    s[4 * j + 1] = fmaf(s[4 * j + 1] * q_mul, a.y, b.y);
                    s[4 * j + 2] = fmaf(s[4 * j + 2] * q_mul, a.z, b.z);
                    s[4 * j + 3] = fmaf(s[4 * j + 3] * q_mul, a.w, b.w);
                }
            }
            const bool need_mask = ts + 31 > hi_min || ts < lo_max || bad;
            unsigned seen = 0xffffu;  // bit e: the lane's row sees the key of element e
            if (need_mask) {
                const int kb0_ = ts + 4 * lg - my_lo;
                seen = 0;
#pragma unroll
                for (int e = 0; e < 16; e++)
                    seen |= ((unsigned)(kb0_ + 8 * (e >> 2) + (e & 3)) < my_seen ? 1u : 0u) << e;
                if (bad & 1) seen &= 0xff00u;
                if (bad & 2) seen &= 0x00ffu;
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = seen >> e & 1 ? s[e] : -INFINITY;
            }
            float mx = fmaxf(s[0], s[1]);
#pragma unroll
            for (int e = 2; e < 16; e++) mx = fmaxf(mx, s[e]);
            mx = pa_xmax32(mx);
            if constexpr (!kQ8) mx *= c2;
            if (__any(mx > mrow + kPaLazy)) {
                const float mnew = fmaxf(mrow, mx);
                const float alpha = __builtin_amdgcn_exp2f(mrow - mnew);
                mrow = mnew;
                lrow_sum *= alpha;
#pragma unroll
                for (int dt = 0; dt < D / 32; dt++) {
                    if constexpr (D == 256) asm volatile("" : "+v"(o[dt]));  // moved to VGPRs here only
                    o[dt] *= alpha;
                    if constexpr (D == 256) asm volatile("" : "+a"(o[dt]));
                }
            }
            float w[16];
#pragma unroll
            for (int e = 0; e < 16; e++)
                w[e] = __builtin_amdgcn_exp2f(kQ8 ? s[e] - mrow : fmaf(s[e], c2, -mrow));
            uint4 pf[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                pf[t].x = M::pack2(w[8 * t + 0], w[8 * t + 1]);
                pf[t].y = M::pack2(w[8 * t + 2], w[8 * t + 3]);
                pf[t].z = M::pack2(w[8 * t + 4], w[8 * t + 5]);
                pf[t].w = M::pack2(w[8 * t + 6], w[8 * t + 7]);
            }
            if constexpr (kQ8) {
                const float4* iv4 = (const float4*)(sc + 2 * BN + 32 * sb + 4 * lg);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 a = iv4[2 * j];
                    lrow_sum = fmaf(w[4 * j + 0], a.x, lrow_sum);
                    lrow_sum = fmaf(w[4 * j + 1], a.y, lrow_sum);
                    lrow_sum = fmaf(w[4 * j + 2], a.z, lrow_sum);
                    lrow_sum = fmaf(w[4 * j + 3], a.w, lrow_sum);
                }
            } else {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    lrow_sum = M::add2(pf[t].x, lrow_sum);
                    lrow_sum = M::add2(pf[t].y, lrow_sum);
                    lrow_sum = M::add2(pf[t].z, lrow_sum);
                    lrow_sum = M::add2(pf[t].w, lrow_sum);
                }
            }
            // A hidden key's weight is 0, and 0 * inf is not: V elements that are not finite leave the
            // product, and reach the rows that see them through counts of +inf, -inf and NaN.
            if constexpr (!kQ8) {
                if (need_mask) {
                    pa_u16x2 top = {0, 0};
#pragma unroll
                    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            const uint4 a = kPreV ? va[kPreV ? dt : 0][t] : load_va(dt, t);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const uint32_t x = (i == 0 ? a.x : i == 1 ? a.y : i == 2 ? a.z : a.w) & 0x7fff7fffu;
                                top = __builtin_elementwise_max(top, __builtin_bit_cast(pa_u16x2, x));
                            }
                        }
                    if (__any(top[0] >= M::kInf || top[1] >= M::kInf)) {
#pragma unroll
                        for (int dt = 0; dt < D / 32; dt++) {
                            pa_f32x16 cnt = zero;
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                const uint4 a = kPreV ? va[kPreV ? dt : 0][t] : load_va(dt, t);
                                uint32_t fin[4], code[4], see[4];
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const uint32_t x = i == 0 ? a.x : i == 1 ? a.y : i == 2 ? a.z : a.w;
                                    fin[i] = code[i] = see[i] = 0;
#pragma unroll
                                    for (int j = 0; j < 2; j++) {
                                        const uint32_t h = x >> (16 * j) & 0xffffu, mag = h & 0x7fffu;
                                        const float what = mag < M::kInf ? 0.0f : mag > M::kInf ? 4096.0f : h >> 15 ? 64.0f : 1.0f;
                                        if (mag < M::kInf) fin[i] |= h << (16 * j);
                                        code[i] |= (M::pack2(what, 0.0f) & 0xffffu) << (16 * j);
                                        if (seen >> (8 * t + 2 * i + j) & 1) see[i] |= (M::pack2(1.0f, 0.0f) & 0xffffu) << (16 * j);
                                    }
                                }
                                o[dt] = M::mma(make_uint4(fin[0], fin[1], fin[2], fin[3]), pf[t], o[dt]);
                                cnt = M::mma(make_uint4(code[0], code[1], code[2], code[3]),
                                             make_uint4(see[0], see[1], see[2], see[3]), cnt);
                            }
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const int c = (int)cnt[e];
                                float add = c & 63 ? INFINITY : 0.0f;
                                if (c >> 6 & 63) add -= INFINITY;
                                if (c >> 12) add = NAN;
                                o[dt][e] += add;
                            }
                        }
                        return;
                    }
                }
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint4 a = kPreV ? va[kPreV ? dt : 0][t] : load_va(dt, t);
                    o[dt] = M::mma(a, pf[t], o[dt]);
                }
            __builtin_amdgcn_s_setprio(0);
        };
        auto compute_tile = [&](const uint16_t* kb, const uint16_t* vb, const float* sc, int t0, unsigned bad) __attribute__((always_inline)) {
#pragma unroll 1
            for (int sb = kh; sb < BN / 32; sb += KH) {
                const int ts = t0 + 32 * sb;
                if (!(wave_active && ts <= hi_max && ts + 31 >= lo_min)) continue;
                subtile(kb, vb, sc, sb, ts, bad >> (2 * sb) & 3);
            }
        };

        // Double-buffered tiles; ids are those of the tile after the one in flight.
        if constexpr (kQ8) {
            if (n_tiles > 0) store_q8(Ks0, Vs0, Sc0);
            __syncthreads();
            for (int it = 0; it < n_tiles; it += 2) {
                const int t0 = t_begin + it * BN;
                if (it + 1 < n_tiles) {
                    bad1 = bad_runs(ids);
                    load_q8(t0 + BN, ids, key_id);
                    if (it + 2 < n_tiles) ids = load_ids(t0 + 2 * BN), key_id = load_key_id(t0 + 2 * BN);
                }
                compute_tile(Ks0, Vs0, Sc0, t0, bad0);
                if (it + 1 >= n_tiles) break;
                store_q8(Ks1, Vs1, Sc1);
                __syncthreads();
                if (it + 2 < n_tiles) {
                    bad0 = bad_runs(ids);
                    load_q8(t0 + 2 * BN, ids, key_id);
                    if (it + 3 < n_tiles) ids = load_ids(t0 + 3 * BN), key_id = load_key_id(t0 + 3 * BN);
                }
                compute_tile(Ks1, Vs1, Sc1, t0 + BN, bad1);
                if (it + 2 < n_tiles) store_q8(Ks0, Vs0, Sc0);
                __syncthreads();
            }
        } else {
            for (int it = 0; it < n_tiles; it += 2) {
                const int t0 = t_begin + it * BN;
                pa_wait_vmem();   // this thread's part of tile it is in LDS
                __syncthreads();  // ... everyone's, and tile it - 1's buffers are free
                if (it + 1 < n_tiles) {
                    bad1 = bad_runs(ids);
                    dma_tile(t0 + BN, ids, Ks1, Vs1);
                    if (it + 2 < n_tiles) ids = load_ids(t0 + 2 * BN);
                }
                compute_tile(Ks0, Vs0, Sc0, t0, bad0);
                if (it + 1 >= n_tiles) break;
                pa_wait_vmem();
                __syncthreads();
                if (it + 2 < n_tiles) {
                    bad0 = bad_runs(ids);
                    dma_tile(t0 + 2 * BN, ids, Ks0, Vs0);
                    if (it + 3 < n_tiles) ids = load_ids(t0 + 3 * BN);
                }
                compute_tile(Ks1, Vs1, Sc1, t0 + BN, bad1);
            }
        }

        // ------------------------------------------------ key parts join, then out
        float lsum = pa_xsum32(lrow_sum);
        if constexpr (KH > 1) {
            // key parts 1 .. hand (O, m, l) of their rows to part 0, one part after another,
            // through the tile buffers: O = O0 2^(m0 - m) + O1 2^(m1 - m), m = max(m0, m1)
            constexpr int NO = D / 32 * 16;
            static_assert(RW * NO * 64 * 4 <= 2 * BN * D * 2 && RW * 2 * 64 * 4 <= BN * D * 2, "merge buffers");
#pragma unroll 1
            for (int part = 1; part < KH; part++) {
                __syncthreads();
                float* const half0 = (float*)Ks0;
                float* const half1 = (float*)Ks1;
                float* const ml = (float*)Vs0 + rw * 128;
                constexpr int NH = BN * D * 2 / 4;  // floats per buffer
                auto at = [&](int i) -> float& {
                    const int x = (rw * NO + i) * 64 + lane;
                    return x < NH ? half0[x] : half1[x - NH];
                };
                if (kh == part) {
#pragma unroll
                    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                        for (int e = 0; e < 16; e++) at(dt * 16 + e) = o[dt][e];
                    ml[lane] = mrow;
                    ml[64 + lane] = lsum;
                }
                __syncthreads();
                if (kh == 0) {
                    const float m1 = ml[lane], l1 = ml[64 + lane];
                    const float mm = fmaxf(mrow, m1);
                    const float a0 = __builtin_amdgcn_exp2f(mrow - mm), a1 = __builtin_amdgcn_exp2f(m1 - mm);
                    mrow = mm;
                    lsum = lsum * a0 + l1 * a1;
#pragma unroll
                    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[dt][e] = o[dt][e] * a0 + at(dt * 16 + e) * a1;
                }
            }
        }
        if (kh != 0 || !wave_active) continue;
        if constexpr (STREAM) {
            if (!whole) {
                float* const ws = (float*)p.workspace + (int64_t)(slot * RW + rw) * (32 * D + 64);
                if (row_ok) {
#pragma unroll
                    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                        for (int jb = 0; jb < 4; jb++)
                            *(float4*)(ws + ((4 * dt + jb) * 64 + lane) * 4) =
                                make_float4(o[dt][4 * jb + 0], o[dt][4 * jb + 1], o[dt][4 * jb + 2], o[dt][4 * jb + 3]);
                    if (lg == 0) {
                        ws[32 * D + ln] = mrow;
                        ws[32 * D + 32 + ln] = lsum;
                    }
                }
                continue;
            }
        }
        if (row_ok) {
            const float inv = lsum != 0.0f ? 1.0f / lsum : 0.0f;
            uint16_t* orow = (uint16_t*)p.out + (int64_t)(blk.beg + my_tok) * p.out_row_stride +
                             (int64_t)my_h * p.out_head_stride;
            const bool f16 = p.dtype == GR_DTYPE_F16;
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                for (int jb = 0; jb < 4; jb++) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = o[dt][4 * jb + e] * inv;
                    uint2 r;
                    if (kQ8 ? f16 : std::is_same_v<DT, F16>)
                        r = make_uint2(PaMat<F16>::pack2(x[0], x[1]), PaMat<F16>::pack2(x[2], x[3]));
                    else
                        r = make_uint2(PaMat<BF16>::pack2(x[0], x[1]), PaMat<BF16>::pack2(x[2], x[3]));
                    *(uint2*)(orow + 32 * dt + 8 * jb + 4 * lg) = r;
                }
        }
    }
}

// Joins the pieces of the block that boundary w (the start of range w) is the first to cut;
// blockIdx.y: a row group of it.
template <typename T>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedAttnLaunch p, const int n_ranges) {
    constexpr int D = T::D, RW = T::RW, BM = T::BM, BN = T::BN;
    const int64_t total = pa_stream_total<BM, BN>(p);
    const int64_t q = pa_stream_q(total, n_ranges);
    const int w0 = (int)blockIdx.x;  // the range before the boundary
    const int64_t x = (w0 + 1) * q;
    if (x >= total) return;
    const PaPlace pl = pa_stream_find<BM, BN>(p, x);
    if (pl.at == 0 || pl.at > q) return;  // no cut here, or an earlier boundary was in this block
    PaBlock blk;
    blk.seq = pl.seq, blk.rb = pl.rb, blk.g = pl.g;
    pa_block<BM, BN>(p, blk);
    const int group = p.n_heads / p.n_kv_heads;
    const int r0 = blk.rb * BM + (int)blockIdx.y * 32;
    const int nr = min(32, blk.n * group - r0);
    if (nr <= 0) return;
    const int64_t start = x - pl.at;                 // the block's first place
    const int n_pieces = (int)((start + pl.vt - 1) / q) - w0 + 1;
    constexpr int kUnit = 32 * D + 64;
    const float* const ws = (const float*)p.workspace;
    // piece i: range w0 + i; its slot and whether it has tiles
    auto piece = [&](int i) -> const float* {
        const int w = w0 + i;
        const int64_t a = max((int64_t)w * q, start) - start, b = min((int64_t)(w + 1) * q, start + pl.vt) - start;
        if (pa_real(a, blk.n_tiles, pl.vt) == pa_real(b, blk.n_tiles, pl.vt)) return nullptr;
        return ws + ((int64_t)(2 * w + (a == 0 ? 1 : 0)) * RW + (int)blockIdx.y) * kUnit;
    };
    for (int i = threadIdx.x; i < nr * (D / 4); i += 256) {
        const int r = i % nr, c = i / nr;            // row, float4 c of it: (c >> 1)-th group of 8, lane half c & 1
        float m = kPaNone;
        for (int k = 0; k < n_pieces; k++) {
            const float* u = piece(k);
            if (u) m = fmaxf(m, u[32 * D + r]);
        }
        float l = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < n_pieces; k++) {
            const float* u = piece(k);
            if (!u) continue;
            const float a = __builtin_amdgcn_exp2f(u[32 * D + r] - m);
            const float4 v = *(const float4*)(u + ((c >> 1) * 64 + (c & 1) * 32 + r) * 4);
            l = fmaf(u[32 * D + 32 + r], a, l);
            o.x = fmaf(v.x, a, o.x), o.y = fmaf(v.y, a, o.y), o.z = fmaf(v.z, a, o.z), o.w = fmaf(v.w, a, o.w);
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const int tok = (r0 + r) / group, h = blk.g * group + (r0 + r) % group;
        uint16_t* out = (uint16_t*)p.out + (int64_t)(blk.beg + tok) * p.out_row_stride + (int64_t)h * p.out_head_stride + 4 * c;
        uint2 y;
        if (p.dtype == GR_DTYPE_F16)
            y = make_uint2(PaMat<F16>::pack2(o.x * inv, o.y * inv), PaMat<F16>::pack2(o.z * inv, o.w * inv));
        else
            y = make_uint2(PaMat<BF16>::pack2(o.x * inv, o.y * inv), PaMat<BF16>::pack2(o.z * inv, o.w * inv));
        *(uint2*)out = y;
    }
}

// ---------------------------------------------------------------- launches

// Blocks of a launch at most: every sequence's last block may be partly filled.
template <typename T>
int64_t pa_max_blocks(const PagedAttnLaunch& p) {
    const int64_t rows = (int64_t)p.seqs.n_rows * (p.n_heads / p.n_kv_heads);
    return (rows / T::BM + std::min<int64_t>(p.seqs.n_seq, p.seqs.n_rows)) * p.n_kv_heads;
}

template <typename T>
size_t pa_ws_bytes(int ranges) { return (size_t)2 * ranges * T::RW * (32 * T::D + 64) * 4; }

template <typename DT, typename T, int SRC>
hipError_t pa_launch_ordered(const PagedAttnLaunch& p, hipStream_t st) {
    // whole rounds of the XCDs for every KV head
    const int64_t per = (pa_max_blocks<T>(p) / p.n_kv_heads + 7) / 8 * 8;
    paged_attn_kernel<DT, T, SRC, false><<<dim3((unsigned)(per * p.n_kv_heads)), T::NT, 0, st>>>(p);
    return hipGetLastError();
}

template <typename DT, typename T, int SRC>
hipError_t pa_launch_stream(const PagedAttnLaunch& p, int ranges, hipStream_t st) {
    paged_attn_kernel<DT, T, SRC, true><<<dim3((unsigned)ranges), T::NT, 0, st>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    paged_combine_kernel<T><<<dim3((unsigned)(ranges - 1), T::RW), 256, 0, st>>>(p, ranges);
    return hipGetLastError();
}

// One (element type, source) of a head_dim: the tiles it is built for and which it takes.
size_t paged_attn_ws_d64(const PagedAttnLaunch& p);
size_t paged_attn_ws_d128(const PagedAttnLaunch& p);
size_t paged_attn_ws_d256(const PagedAttnLaunch& p);
hipError_t launch_paged_attn_d64(const PagedAttnLaunch& p, hipStream_t st);
hipError_t launch_paged_attn_d128(const PagedAttnLaunch& p, hipStream_t st);
hipError_t launch_paged_attn_d256(const PagedAttnLaunch& p, hipStream_t st);

// Few: blocks of few rows, key parts; Mid, Big: whole row blocks.
template <typename Few, typename Mid, typename Big>
struct PaKernels {
    enum Kind { kFew, kMidStream, kMid, kBig };
    static constexpr int kCus = 256;
    static constexpr int few_ranges = kCus * std::max(1, Few::OCC * 4 / Few::NW);
    static constexpr int mid_ranges = kCus * std::max(1, Mid::OCC * 4 / Mid::NW);

    static Kind kind(const PagedAttnLaunch& p) {
        const int64_t group = p.n_heads / p.n_kv_heads;
        if (std::min<int64_t>(p.max_rows, p.seqs.n_rows) * group <= Few::BM) return kFew;
        const int64_t rows = (int64_t)p.seqs.n_rows * group * p.n_kv_heads;
        if (rows >= (int64_t)2 * kCus * Big::BM) return kBig;
        if (rows >= (int64_t)2 * kCus * Mid::BM) return kMid;
        return kMidStream;
    }
    static size_t ws(const PagedAttnLaunch& p) {
        switch (kind(p)) {
            case kFew: return pa_ws_bytes<Few>(few_ranges);
            case kMidStream: return pa_ws_bytes<Mid>(mid_ranges);
            default: return 256;
        }
    }
    template <typename DT, int SRC>
    static hipError_t launch(const PagedAttnLaunch& p, hipStream_t st) {
        switch (kind(p)) {
            case kFew: return pa_launch_stream<DT, Few, SRC>(p, few_ranges, st);
            case kMidStream: return pa_launch_stream<DT, Mid, SRC>(p, mid_ranges, st);
            case kMid: return pa_launch_ordered<DT, Mid, SRC>(p, st);
            default: return pa_launch_ordered<DT, Big, SRC>(p, st);
        }
    }
    static hipError_t launch_any(const PagedAttnLaunch& p, hipStream_t st) {
        if (!p.seqs.page_table)
            return p.dtype == GR_DTYPE_F16 ? launch<F16, kPaPacked>(p, st) : launch<BF16, kPaPacked>(p, st);
        if (p.kv_dtype == GR_DTYPE_Q8) return launch<F16, kPaPagesQ8>(p, st);
        return p.dtype == GR_DTYPE_F16 ? launch<F16, kPaPages>(p, st) : launch<BF16, kPaPages>(p, st);
    }
};

}  // namespace gr
