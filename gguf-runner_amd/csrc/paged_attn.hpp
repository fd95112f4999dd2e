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
//
// What bounds the kernels, on one MI355X:
//   few rows (up to 32 per sequence and KV head): HBM.  16 tokens of 1k .. 32k keys, f16, 32 / 4
//     heads, head_dim 128: 97 us = 5.5 TB/s; Q8 pages, 24 sequences of 0.3k .. 12k keys, 1 - 5 rows:
//     101 us = 3.5 TB/s, where turning codes into f16 takes VALU time of the size of the softmax.  One
//     tile on its way and one wave per SIMD measured better than more of either (129 against 111 us
//     with four tiles in LDS, 188 against 108 us for Q8 at two waves per SIMD, which spills).
//   many rows: the matrix units and the softmax between them (VALU).  Three prompts of 1001 .. 8192
//     rows, f16, 32 / 8 heads, head_dim 128: 1213 us = 965 TFLOP/s; one of 8192 rows, 8 / 4
//     heads, head_dim 256: 300 us = 900 TFLOP/s (409 us before its LDS reads went four products
//     ahead of their use); 40 prompts of 9 .. 777 rows, bf16, 14 / 2 heads, head_dim 64: 36 us, a third
//     of it short blocks' starts and ends.  At head_dim 256 a block's O, Q and S take a whole SIMD's
//     registers; two waves per SIMD spill (2900 us).
#pragma once

#include <algorithm>
#include <cmath>
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
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pa_bf16x2, w), pa_bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
#else
        return c;
#endif
    }
};

enum PaMode { kPaFull, kPaMasked, kPaEither };
enum PaSrc { kPaPacked = 0, kPaPages = 1, kPaPagesQ8 = 2 };

// The launch's arguments (its kernel's only parameter), read anew from here on: what a block uses
// before or after its tiles does not stay in scalar registers through them.
__device__ __forceinline__ const PagedAttnLaunch& pa_again() {
#if defined(__HIP_DEVICE_COMPILE__)
    auto at = (const __attribute__((address_space(4))) PagedAttnLaunch*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const PagedAttnLaunch*)at;
#else
    return *(const PagedAttnLaunch*)nullptr;
#endif
}

// Tiles of a kernel: RW row groups x KH key parts, BN keys, NBUF tiles in LDS (with two, one
// is on its way), waves per SIMD it is built for.
template <int D_, int RW_, int KH_, int BN_, int NBUF_, int OCC_>
struct PaTile {
    static constexpr int D = D_, RW = RW_, KH = KH_, BN = BN_, NBUF = NBUF_, OCC = OCC_;
    static constexpr int NW = RW * KH, NT = NW * 64, BM = RW * 32;
    static_assert(BN % (32 * KH) == 0, "every key part has its sub-tiles");
    static constexpr int kLds = 4 * NBUF * BN * D + 2048 + 24 * BN + (KH > 1 ? 512 * NW : 0) + 64;  // at most (page ids, Q8 scales, m and l)
    // workgroups a CU holds: by waves, and by its 160 KB of LDS
    static constexpr int kPerCu = OCC * 4 / NW < 163840 / kLds ? (OCC * 4 / NW < 1 ? 1 : OCC * 4 / NW) : 163840 / kLds;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t pa_rsrc(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)0xffffffff, 0x00020000);
}
// ONCE: no other workgroup reads it (nontemporal)
template <bool ONCE>
__device__ __forceinline__ void pa_dma16(__amdgpu_buffer_rsrc_t r, uint16_t* lds, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (GR_PA_LDS void*)lds, 16, voff, 0, 0, ONCE ? 2 : 0);
#endif
}
template <bool ONCE>
__device__ __forceinline__ uint4 pa_load16(__amdgpu_buffer_rsrc_t r, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, ONCE ? 2 : 0));
#else
    return uint4{};
#endif
}
// s_waitcnt vmcnt(0): the wave's vector memory operations are done
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

// Asks the scheduler for this order of the products in front of it: the LDS reads of the first
// four (READS each), then a product and the reads of the one four later, so that a single wave
// does not wait for every read.
template <int N, int READS>
__device__ __forceinline__ void pa_pipeline() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4 * READS, 0);
#pragma unroll
    for (int i = 0; i < N - 4; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    __builtin_amdgcn_sched_barrier(0);
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

// The magnitudes of two 16-bit floats; the finite ones of eight (others 0).
__device__ __forceinline__ pa_u16x2 pa_mag(uint32_t x) { return __builtin_bit_cast(pa_u16x2, x & 0x7fff7fffu); }
template <typename M>
__device__ __forceinline__ uint4 pa_finite(const uint4& a) {
    auto two = [](uint32_t x) {
        const uint32_t lo = (x & 0x7fffu) < M::kInf ? 0xffffu : 0u, hi = (x >> 16 & 0x7fffu) < M::kInf ? 0xffff0000u : 0u;
        return x & (lo | hi);
    };
    return make_uint4(two(a.x), two(a.y), two(a.z), two(a.w));
}

// ---------------------------------------------------------------- schedules

// What a sequence has: rows, keys, blocks, and the tiles that each of its blocks counts in
// the stream (its longest block's, at least 1).  0 blocks behind the last sequence.
struct PaSeq {
    int beg, n, len, nb, vt;
};
template <int BM, int BN>
__device__ __forceinline__ PaSeq pa_seq(const PagedAttnLaunch& p, int s) {
    PaSeq r{0, 0, 0, 0, 0};
    if (s >= p.seqs.n_seq) return r;
    const int group = p.group;
    r.beg = seq_row(p.seqs, s);
    r.n = max(seq_row(p.seqs, s + 1) - r.beg, 0);
    r.len = seq_len(p.seqs, s, r.n);
    r.nb = (r.n * group + BM - 1) / BM;
    r.vt = (r.len + BN - 1) / BN;
    if (p.window > 0) r.vt = min(r.vt, (min(p.window, r.len) + div_group(p, BM) + BN - 1) / BN + 1);
    r.vt = max(r.vt, 1);
    return r;
}

// Inclusive sum over the wave's lanes: four shifts inside rows of 16 lanes, then each row's
// last lane is added to the rows behind it.
__device__ __forceinline__ int pa_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return x;
}
__device__ __forceinline__ int pa_last(int x) { return __builtin_amdgcn_readlane(x, 63); }

// One block: KV head g, block rb of sequence seq, its rows and keys.
struct PaBlock {
    int seq, rb, g;
    int beg, n, p0;           // first row, rows, position of the first row
    int nb, vt;
    int t_first, kend;        // keys [.., kend); tiles start at t_first
    int all_lo, all_hi;       // every row sees keys all_lo .. all_hi (as far as their pages are there)
    int n_tiles;
};
template <int BM, int BN>
__device__ __forceinline__ void pa_keys(const PagedAttnLaunch& p, PaBlock& b) {
    const int group = p.group;
    const int tok0 = div_group(p, b.rb * BM), tok1 = div_group(p, min((b.rb + 1) * BM, b.n * group) - 1);
    b.kend = max(b.p0 + tok1 + 1, 0);
    const int lo = p.window > 0 ? max(b.p0 + tok0 + 1 - p.window, 0) : 0;
    b.all_lo = p.window > 0 ? max(b.p0 + tok1 + 1 - p.window, 0) : 0;
    b.all_hi = b.p0 + tok0;
    b.t_first = lo / BN * BN;
    b.n_tiles = b.kend > b.t_first ? (b.kend - b.t_first + BN - 1) / BN : 0;
}
__device__ __forceinline__ void pa_take(PaBlock& b, const PaSeq& c, int s0, int l) {
    b.seq = s0 + l;
    b.beg = __builtin_amdgcn_readlane(c.beg, l);
    b.n = __builtin_amdgcn_readlane(c.n, l);
    b.p0 = __builtin_amdgcn_readlane(c.len, l) - b.n;
    b.nb = __builtin_amdgcn_readlane(c.nb, l);
    b.vt = __builtin_amdgcn_readlane(c.vt, l);
}

// The stream: sequence s takes n_kv_heads * nb * vt places (the host bounds their sum by
// 2^31), KV head by KV head, block by block; place v of a block is its tile v.
template <int BM, int BN>
__device__ __forceinline__ int pa_stream_total(const PagedAttnLaunch& p, const PaSeq& c0) {
    int t = pa_last(pa_scan(c0.nb * c0.vt * p.n_kv_heads));
    for (int s0 = 64; s0 < p.seqs.n_seq; s0 += 64) {
        const PaSeq c = pa_seq<BM, BN>(p, s0 + (threadIdx.x & 63));
        t += pa_last(pa_scan(c.nb * c.vt * p.n_kv_heads));
    }
    return t;
}
// The block that place x (< total) belongs to; returns x's offset in it, -1 for none (only
// rows that overlap, which sum up to more than 2^31 places).  c0: pa_seq of the lane.
template <int BM, int BN>
__device__ __forceinline__ int pa_stream_find(const PagedAttnLaunch& p, const PaSeq& c0, int x, PaBlock& b) {
    for (int s0 = 0; s0 < p.seqs.n_seq; s0 += 64) {
        const PaSeq c = s0 == 0 ? c0 : pa_seq<BM, BN>(p, s0 + (threadIdx.x & 63));
        const int cost = c.nb * c.vt * p.n_kv_heads;
        const int incl = pa_scan(cost);
        const int all = pa_last(incl);
        if (x < all) {
            const int l = __ffsll((unsigned long long)__ballot(x < incl)) - 1;
            x -= __builtin_amdgcn_readlane(incl - cost, l);
            pa_take(b, c, s0, l);
            const int i = x / b.vt;
            b.g = i / b.nb;
            b.rb = i - b.g * b.nb;
            if ((unsigned)b.g >= (unsigned)p.n_kv_heads) return -1;
            pa_keys<BM, BN>(p, b);
            return x - i * b.vt;
        }
        x -= all;
    }
    return -1;
}

// Workgroup b of a stream launch as a place among them: XCD b % 8 gets a run of
// neighbouring ranges (the blocks of a sequence's KV head share its tiles in one L2).
// Launches are multiples of 8 workgroups.
__device__ __forceinline__ int pa_stream_rank(int b, int n) { return (b & 7) * (n / 8) + (b >> 3); }
// Places per range: an equal share.
__device__ __forceinline__ int pa_stream_q(int total, int n) { return (int)(((int64_t)total + n - 1) / n); }

// ORDERED: item idx of one KV head, longest blocks first: blocks by their number counted
// from a sequence's first, the highest numbers first (up to 64 sequences); more sequences:
// one after another, each one's last block first.  False: no such item.
template <int BM, int BN>
__device__ __forceinline__ bool pa_ordered_find(const PagedAttnLaunch& p, const PaSeq& c0, int idx, PaBlock& b) {
    const int lane = threadIdx.x & 63;
    if (p.seqs.n_seq <= 64) {
        auto count = [&](int l) { return pa_last(pa_scan(max(c0.nb - l, 0))); };  // blocks numbered l or more
        if (idx >= count(0)) return false;
        int lo = 0, hi = 1;  // lo: the highest l with count(l) > idx
        while (count(hi) > idx) hi *= 2;
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (count(mid) > idx) lo = mid;
            else hi = mid;
        }
        const int k = idx - count(lo + 1);  // the k-th sequence that has a block of this number
        const bool has = c0.nb > lo;
        const int before = __popcll(__ballot(has) & ((1ull << lane) - 1));
        const int l = __ffsll((unsigned long long)__ballot(has && before == k)) - 1;
        pa_take(b, c0, 0, l);
        b.rb = lo;
    } else {
        int s0 = 0;
        for (;; s0 += 64) {
            if (s0 >= p.seqs.n_seq) return false;
            const PaSeq c = s0 == 0 ? c0 : pa_seq<BM, BN>(p, s0 + lane);
            const int incl = pa_scan(c.nb);
            const int all = pa_last(incl);
            if (idx < all) {
                const int l = __ffsll((unsigned long long)__ballot(idx < incl)) - 1;
                pa_take(b, c, s0, l);
                b.rb = __builtin_amdgcn_readlane(incl, l) - 1 - idx;
                break;
            }
            idx -= all;
        }
    }
    pa_keys<BM, BN>(p, b);
    return true;
}

// ---------------------------------------------------------------- the kernel

template <typename DT, typename T, int SRC, bool STREAM>
__global__ __launch_bounds__(T::NT, T::OCC) void paged_attn_kernel(const PagedAttnLaunch p) {
    constexpr int D = T::D, BN = T::BN, BM = T::BM, RW = T::RW, KH = T::KH, NT = T::NT, NBUF = T::NBUF;
    constexpr bool kQ8 = SRC == kPaPagesQ8;
    using M = PaMat<DT>;
    constexpr int CPR = D / 8;              // 16-byte chunks per tile row
    constexpr int SCPR = kQ8 ? D / 16 : CPR;  // chunks per source row
    constexpr int LD = BN * SCPR / NT;      // source chunks per thread per K (or V) tile
    constexpr int RPU = NT / SCPR;          // rows filled by one round of the workgroup
    constexpr int RPV = 64 / SCPR;          // ... of a wave: inside one run of 16 rows, so one page
    constexpr int EB = kQ8 ? 1 : 2;         // bytes per stored element
    // A call of few rows has one block per sequence and KV head: its tiles are read once, with the
    // nontemporal hint if a row fills a 128-byte line (16 tokens after 1k .. 32k keys, f16, 32 / 4
    // heads d128: 111 -> 97 us; Q8, 24 sequences to 12k keys: 104 -> 101; 64-byte rows, Q8 d64, 64 tokens
    // after 4k keys: 24.6 -> 25.7, not taken).  More rows share tiles in L2.
    constexpr bool kOnce = RW == 1 && D * EB >= 128;
    static_assert(LD >= 1 && LD <= 32 && BN * SCPR % NT == 0 && BN / 16 <= 32 && BN <= NT, "tile shape");
    static_assert(kQ8 ? NBUF <= 2 : NBUF == 2, "buffers");

    // distinct arrays, so that the compiler sees that filling one never aliases reading another
    __shared__ __attribute__((aligned(16))) uint16_t Ks0[BN * D];
    __shared__ __attribute__((aligned(16))) uint16_t Ks1[NBUF > 1 ? BN * D : 8];
    __shared__ __attribute__((aligned(16))) uint16_t Vs0[BN * D];
    __shared__ __attribute__((aligned(16))) uint16_t Vs1[NBUF > 1 ? BN * D : 8];
    // Q8: c * k_scale, log2 v_scale, 1 / v_scale of the tile's keys
    __shared__ __attribute__((aligned(16))) float Sc0[kQ8 ? 3 * BN : 4];
    __shared__ __attribute__((aligned(16))) float Sc1[kQ8 && NBUF > 1 ? 3 * BN : 4];
    // Page ids of a run of tiles (-1: not there): read from the table once per run, so that
    // no load of a tile waits for another
    constexpr int kIds = 512;
    __shared__ float Ml[KH > 1 ? T::NW * 128 : 1];  // the key parts' m and l
    __shared__ int Ids[SRC == kPaPacked ? 1 : kIds];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = KH > 1 ? wave % RW : wave, kh = KH > 1 ? wave / RW : 0;
    const int ln = lane & 31, lg = lane >> 5;
    const int shift = p.seqs.page_shift;
    const int ps1 = (1 << shift) - 1;

    // this thread's source chunks: row wave * RPV + lane / SCPR + u * RPU of the tile
    const int lrow = lane / SCPR;
    auto col = [&](int u) {  // byte offset in the source row
        const int r = wave * RPV + lrow + (RPU % 16 ? u * RPU : 0);
        return kQ8 ? lane % SCPR * 16 : ((lane % SCPR) ^ pa_swz<D>(r & 15)) * 16;
    };
    const int rsb = (int)p.row_stride * EB;
    // K fragments: row ln of a sub-tile, chunk 2 i + lg; V^T fragments (ds_read_b64_tr_b16): lane i
    // of a 16-lane group supplies row i / 4, columns 4 (i % 4) .. +3 of a 4 x 16 block (b) of O^T
    // tile dt and receives its column i.  Byte offsets, the V ones less where the V arrays start
    // in LDS (kVAt), which keeps every other part of an address within the instruction's 16-bit
    // offset.  The chunk number only touches the bits of an offset below the row size, so
    // offset(i) = offset(0) ^ 32 i and offset(dt) = offset(0) ^ 64 dt.  head_dim 256, which has no
    // registers to keep them all, makes them where they are used (an xor each); the empty asm
    // statements keep the compiler from taking offsets apart or moving them out of the loop.
    constexpr bool kMakeOff = D == 256, kEither = D == 256;
    constexpr int kVAt = NBUF * BN * D * 2;
    const int gi = lane & 15;
    const int v_chunk = 2 * ((lane >> 4) & 1) + ((gi & 3) >> 1);
    int k_off[kMakeOff ? 1 : D / 16], v_off[kMakeOff ? 1 : D / 32][2];
#pragma unroll
    for (int i = 0; i < (kMakeOff ? 1 : D / 16); i++) {
        k_off[i] = (2 * (ln * D + ((lg ^ pa_swz<D>(ln & 15)) << 3))) ^ (32 * i);
        asm volatile("" : "+v"(k_off[i]));
    }
#pragma unroll
    for (int dt = 0; dt < (kMakeOff ? 1 : D / 32); dt++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int r = 8 * b + 4 * lg + (gi >> 2);
            v_off[dt][b] = (kVAt + 2 * (r * D + (gi & 1) * 4 + ((v_chunk ^ pa_swz<D>(r & 15)) << 3))) ^ (64 * dt);
            asm volatile("" : "+v"(v_off[dt][b]));
        }

    // ------------------------------------------------ the workgroup's range
    const PaSeq c0 = pa_seq<BM, BN>(p, lane);
    int pos = 0, stop = 1, rank = 0;  // STREAM: places of the stream
    if constexpr (STREAM) {
        const int total = pa_stream_total<BM, BN>(p, c0);
        rank = pa_stream_rank(blockIdx.x, gridDim.x);
        const int q = pa_stream_q(total, gridDim.x);
        if ((int64_t)rank * q >= total) return;
        pos = rank * q;
        stop = min((int64_t)total, (int64_t)pos + q);
    }

    while (pos < stop) {
        const PagedAttnLaunch& p = pa_again();
        PaBlock blk;
        int it0 = 0, it1 = 0;
        bool whole = true;
        int slot = 0;
        if constexpr (STREAM) {
            const int at = pa_stream_find<BM, BN>(p, c0, pos, blk);
            if (at < 0) return;
            const int to = min(blk.vt, at + (stop - pos));
            whole = at == 0 && to == blk.vt;
            slot = 2 * rank + (at == 0 ? 1 : 0);
            it0 = min(at, blk.n_tiles);
            it1 = min(to, blk.n_tiles);
            pos += to - at;
            if (!whole && it0 == it1) continue;  // the joining kernel knows that this piece is empty
        } else {
            pos = 1;
            const int hx = p.n_kv_heads;
            const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
            int idx;
            if (8 % hx == 0) {  // 8 / hx XCDs take the blocks of one KV head
                blk.g = x % hx;
                idx = i * (8 / hx) + x / hx;
            } else if (hx % 8 == 0) {
                blk.g = x + 8 * (i % (hx / 8));
                idx = i / (hx / 8);
            } else {
                blk.g = blockIdx.x % hx;
                idx = blockIdx.x / hx;
            }
            if (!pa_ordered_find<BM, BN>(p, c0, idx, blk)) return;
            it1 = blk.n_tiles;
        }

        const int n_pr = blk.n * p.group;
        const int wr0 = blk.rb * BM + rw * 32;
        const bool wave_active = wr0 < n_pr;
        // the lane's row, its token and position
        const int my_tok = div_group(p, min(wr0 + ln, n_pr - 1));
        const int my_pos = blk.p0 + my_tok;
        const int my_lo = p.window > 0 ? max(my_pos + 1 - p.window, 0) : 0;
        const unsigned my_seen = (unsigned)max(my_pos + 1 - my_lo, 0);
        // the wave's rows: positions rise with the row
        const int hi_min = __builtin_amdgcn_readfirstlane(my_pos);
        const int hi_max = __builtin_amdgcn_readlane(my_pos, 31);
        const int lo_min = __builtin_amdgcn_readfirstlane(my_lo);
        const int lo_max = __builtin_amdgcn_readlane(my_lo, 31);

        const int last = blk.kend - 1;
        const char* kb0 = (const char*)p.k + (int64_t)blk.g * p.head_stride * EB;
        const char* vb0 = (const char*)p.v + (int64_t)blk.g * p.head_stride * EB;
        int64_t page_bytes = p.page_stride * EB, row_bytes = p.row_stride * EB;
        if constexpr (T::OCC == 1 && SRC != kPaPacked) asm volatile("" : "+v"(kb0), "+v"(vb0), "+v"(page_bytes), "+v"(row_bytes));
        int page0 = 0;        // the page Ids[0] is of
        bool some_bad = false, ever_bad = false;  // in the run, in a run so far

        // Pages: lane u has where in K and V this wave's run of rows of round u is.  One product in
        // vector registers for all rounds: a scalar one for every round, and every round's place in
        // LDS kept in scalar registers through the loop, spilled them, and the scheduler gave up the LDS
        // reads ahead of their products that a single wave per SIMD lives on (head_dim 256, 8000-token
        // prompt of 8 / 4 heads: 416 -> 312 us).
        struct Runs {
            uint64_t k, v;
        };
        auto tile_runs = [&](int t0) __attribute__((always_inline)) {
            if constexpr (SRC == kPaPacked) {
                return Runs{};
            } else {
                const int key = min(t0 + wave * RPV + min(lane, LD - 1) * RPU, last);
                const int id = max(Ids[(key >> shift) - page0], 0);
                const int64_t at = (int64_t)id * page_bytes + (int64_t)(key & ps1) * row_bytes;
                return Runs{(uint64_t)(kb0 + at), (uint64_t)(vb0 + at)};
            }
        };
        auto lane_at = [&](uint64_t x, int u) __attribute__((always_inline)) {
            return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), u) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)x, u));
        };
        auto round_wave = [&]() __attribute__((always_inline)) {
            int w = wave;
            if constexpr (T::OCC == 1) asm volatile("" : "+s"(w));
            return w;
        };
        // Round u's run in K and V (scalar) and the lane's offset in it: rows past the last key repeat it
        // (they are masked, and must not be read).
        auto round_of = [&](int t0, const Runs& runs, int w, int u, const char*& k, const char*& v) __attribute__((always_inline)) {
            const int fc = min(t0 + w * RPV + u * RPU, last);
            if constexpr (SRC == kPaPacked) {
                const int64_t at = (int64_t)(blk.beg + fc) * row_bytes;
                k = kb0 + at;
                v = vb0 + at;
            } else {
                k = lane_at(runs.k, u);
                v = lane_at(runs.v, u);
            }
            return (t0 + BN - 1 <= last ? lrow : min(lrow, last - fc)) * rsb + col(u);
        };
        // 16-key runs of the tile whose page is not there
        auto bad_runs = [&](int t0) __attribute__((always_inline)) {
            if (SRC == kPaPacked || !some_bad) return 0u;
            const int key = min(t0 + min(lane, BN / 16 - 1) * 16, last);
            return (unsigned)__ballot(Ids[(key >> shift) - page0] < 0) & ((1u << (BN / 16)) - 1);
        };
        auto dma_tile = [&](int t0, uint16_t* kd, uint16_t* vd) __attribute__((always_inline)) {
            const Runs runs = tile_runs(t0);
            const int w = round_wave();
#pragma unroll
            for (int u = 0; u < LD; u++) {
                const char *k, *v;
                const int off = round_of(t0, runs, w, u, k, v);
                const int dst = (w * 64 + u * NT) * 8;
                pa_dma16<kOnce>(pa_rsrc(k), kd + dst, off);
                pa_dma16<kOnce>(pa_rsrc(v), vd + dst, off);
            }
        };
        uint4 kr[kQ8 ? LD : 1], vr[kQ8 ? LD : 1];
        float ks_r = 0.0f, vs_r = 1.0f;
        auto load_q8 = [&](int t0) __attribute__((always_inline)) {
            if constexpr (kQ8) {
                const Runs runs = tile_runs(t0);
                const int w = round_wave();
#pragma unroll
                for (int u = 0; u < LD; u++) {
                    const char *k, *v;
                    const int off = round_of(t0, runs, w, u, k, v);
                    kr[u] = pa_load16<kOnce>(pa_rsrc(k), off);
                    vr[u] = pa_load16<kOnce>(pa_rsrc(v), off);
                }
                if (tid < BN) {
                    const int key = min(t0 + tid, last);
                    const int id = max(Ids[(key >> shift) - page0], 0);
                    const int64_t at = (int64_t)id * p.scale_page_stride + (int64_t)(key & ps1) * p.scale_row_stride +
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

        // ------------------------------------------------ Q: B operands, one row per lane column
        uint4 qf[D / 16];
        float q_mul = 1.0f;  // Q8: what the scores are multiplied by (bf16 rows are put in f16's range)
        {
            const int h = blk.g * p.group + (min(wr0 + ln, n_pr - 1) - my_tok * p.group);
            const uint16_t* qr = (const uint16_t*)p.q + (int64_t)(blk.beg + my_tok) * p.q_row_stride +
                                 (int64_t)h * p.q_head_stride;
#pragma unroll
            for (int c = 0; c < D / 16; c++) qf[c] = *(const uint4*)(qr + 16 * c + 8 * lg);
        }
        // Q is in its registers from here on: without a use in front of the tile loop its first
        // product would wait for every load in flight, the next tile's among them.
        auto settle_q = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < D / 16; c++)
                asm volatile("" : "+v"(qf[c].x), "+v"(qf[c].y), "+v"(qf[c].z), "+v"(qf[c].w));
        };
        auto prepare_q = [&]() __attribute__((always_inline)) {
            if constexpr (kQ8) {
                if (pa_again().dtype == GR_DTYPE_BF16) {
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
        };

        pa_f32x16 o[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[dt][e] = 0.0f;
        float mrow = kPaNone, lrow_sum = 0.0f;
        bool odd = false;  // V elements that are not finite were left out of some tile
        const float c2 = p.scale_log2;

        // One 32-key sub-tile: keys ts .. ts + 31, rows 32 sb .. of the tile; mode kPaFull: every row of
        // the wave sees all of them, kPaMasked: some do not (bad: its two 16-key runs that are not
        // there), kPaEither: decided here (one body for both, where O cannot change its registers).
        auto subtile = [&](auto mode, const uint16_t* kb, const uint16_t* vb, const float* sc, int sb, int ts,
                           unsigned bad) __attribute__((always_inline)) {
            constexpr bool kMasked = decltype(mode)::value != kPaFull;
            const bool need = decltype(mode)::value == kPaMasked || ts + 31 > hi_min || ts < lo_max || bad;
            __builtin_amdgcn_sched_barrier(0);  // sub-tiles are not interleaved: the registers hold one
            if constexpr (kMakeOff) asm volatile("" : "+v"(k_off[0]), "+v"(v_off[0][0]), "+v"(v_off[0][1]));
            const pa_f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            __builtin_amdgcn_s_setprio(1);
            pa_f32x16 s;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const uint4 a = *(const uint4*)((const char*)kb + (kMakeOff ? (k_off[0] + 64 * sb * D) ^ (32 * i) : 64 * sb * D + k_off[kMakeOff ? 0 : i]));
                s = M::mma(a, qf[i], i == 0 ? zero : s);
            }
            if constexpr (D == 256) {
                pa_pipeline<D / 16, 1>();
                asm volatile("" : "+v"(s));
            }
            auto load_va = [&](int dt, int t) __attribute__((always_inline)) {
                pa_i16x4 part[2];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int off = kMakeOff ? (v_off[0][b] + 64 * sb * D) ^ (64 * dt) : 64 * sb * D + v_off[kMakeOff ? 0 : dt][b];
                    const char* at = (const char*)vb - kVAt + 32 * t * D + off;
                    part[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GR_PA_LDS pa_i16x4*)at);
                }
                const uint2 lo = __builtin_bit_cast(uint2, part[0]);
                const uint2 hi = __builtin_bit_cast(uint2, part[1]);
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            constexpr bool kPreV = D <= 128 && !(kQ8 && RW > 1);
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
            if constexpr (kMasked) {
                if (need) {
                    const int k0 = ts + 4 * lg - my_lo;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const bool seen = (unsigned)(k0 + 8 * (e >> 2) + (e & 3)) < my_seen && !(bad >> (e >> 3) & 1);
                        s[e] = seen ? s[e] : -INFINITY;
                    }
                }
            }
            if constexpr (D == 256) asm volatile("" : "+v"(s));
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
                    if constexpr (D == 256 && T::OCC == 1) asm volatile("" : "+v"(o[dt]));  // moved to VGPRs here only
                    o[dt] *= alpha;
                    if constexpr (D == 256 && T::OCC == 1) asm volatile("" : "+a"(o[dt]));
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
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint4 a = kPreV ? va[kPreV ? dt : 0][t] : load_va(dt, t);
                    o[dt] = M::mma(a, pf[t], o[dt]);
                }
            if constexpr (D == 256) pa_pipeline<D / 16, 2>();
            __builtin_amdgcn_s_setprio(0);
        };
        auto compute_tile = [&](const uint16_t* kb, const uint16_t* vb, const float* sc, int t0, unsigned bad) __attribute__((always_inline)) {
            if (!wave_active) return;
            using std::integral_constant;
            if (!kEither && t0 + BN - 1 <= hi_min && t0 >= lo_max && !bad) {
#pragma unroll
                for (int i = 0; i < BN / 32 / KH; i++)
                    subtile(integral_constant<int, kPaFull>{}, kb, vb, sc, KH * i + kh, t0 + 32 * (KH * i + kh), 0u);
                return;
            }
#pragma unroll(kEither ? BN / 32 / KH : 1)
            for (int sb = kh; sb < BN / 32; sb += KH) {
                const int ts = t0 + 32 * sb;
                if (ts <= hi_max && ts + 31 >= lo_min)
                    subtile(integral_constant<int, kEither ? kPaEither : kPaMasked>{}, kb, vb, sc, sb, ts, bad >> (2 * sb) & 3);
            }
        };

        // Whether some row of the block does not see every key of the tile.
        auto partly = [&](int t0, bool bad) __attribute__((always_inline)) {
            return t0 + BN - 1 > blk.all_hi || t0 < blk.all_lo || bad;
        };
        // A hidden key's weight is 0, but 0 * inf is not: V elements of a partly hidden tile that are not
        // finite become zeros (each thread looks at what it brought), and the rows that see them get
        // them after the last tile.  Called by the whole workgroup, the tile is in LDS.
        auto finite_only = [&](uint16_t* vd) __attribute__((always_inline)) {
            uint4* const mine = (uint4*)(vd + (wave * 64 + lane) * 8);
            pa_u16x2 top = {0, 0};
#pragma unroll
            for (int u = 0; u < LD; u++) {
                const uint4 a = mine[u * NT];
                top = __builtin_elementwise_max(top, __builtin_elementwise_max(pa_mag(a.x), pa_mag(a.y)));
                top = __builtin_elementwise_max(top, __builtin_elementwise_max(pa_mag(a.z), pa_mag(a.w)));
            }
            if (!__syncthreads_or(top[0] >= M::kInf || top[1] >= M::kInf)) return;
            odd = true;
#pragma unroll 1
            for (int u = 0; u < LD; u++) mine[u * NT] = pa_finite<M>(mine[u * NT]);
            __syncthreads();
        };

        // The tiles, run of page ids by run.
        const int run_tiles = SRC == kPaPacked ? it1 - it0 : (int)min(((int64_t)(kIds - 1) << shift) / BN, (int64_t)1 << 30);
        for (int rt = it0; rt < it1; rt += run_tiles) {
            const int t_begin = blk.t_first + rt * BN;
            const int n_tiles = min(it1 - rt, run_tiles);
            __syncthreads();  // what ran before is done with every LDS array
            if constexpr (SRC != kPaPacked) {
                const PagedAttnLaunch& p = pa_again();
                const int32_t* table = p.seqs.page_table + (int64_t)blk.seq * p.seqs.table_stride;
                page0 = t_begin >> shift;
                const int n_ids = (min(last, t_begin + n_tiles * BN - 1) >> shift) - page0 + 1;
                int bad = 0;
                for (int i = tid; i < n_ids; i += NT) {
                    const int id = table[page0 + i];
                    const bool there = (unsigned)id < (unsigned)p.seqs.n_pages;
                    Ids[i] = there ? id : -1;
                    bad |= !there;
                }
                some_bad = __syncthreads_or(bad);
                ever_bad |= some_bad;
            }
            if constexpr (kQ8) {
                load_q8(t_begin);
                settle_q();
                if (rt == it0) prepare_q();
                store_q8(Ks0, Vs0, Sc0);
                __syncthreads();
                // the next tile's codes are on their way to registers while this one is used; one tile in
                // LDS takes two barriers a tile, but leaves room for other workgroups
                for (int it = 0; NBUF == 1 && it < n_tiles; it++) {
                    const int t0 = t_begin + it * BN;
                    if (it + 1 < n_tiles) load_q8(t0 + BN);
                    compute_tile(Ks0, Vs0, Sc0, t0, bad_runs(t0));
                    if (it + 1 >= n_tiles) break;
                    __syncthreads();
                    store_q8(Ks0, Vs0, Sc0);
                    __syncthreads();
                }
                for (int it = 0; NBUF == 2 && it < n_tiles; it += 2) {
                    const int t0 = t_begin + it * BN;
                    if (it + 1 < n_tiles) load_q8(t0 + BN);
                    compute_tile(Ks0, Vs0, Sc0, t0, bad_runs(t0));
                    if (it + 1 >= n_tiles) break;
                    store_q8(Ks1, Vs1, Sc1);
                    __syncthreads();
                    if (it + 2 < n_tiles) load_q8(t0 + 2 * BN);
                    compute_tile(Ks1, Vs1, Sc1, t0 + BN, bad_runs(t0 + BN));
                    if (it + 2 < n_tiles) store_q8(Ks0, Vs0, Sc0);
                    __syncthreads();
                }
            } else {
                // tile it: wait until it is in LDS, send for the next one, compute
                auto step = [&](uint16_t* kd, uint16_t* vd, uint16_t* next_kd, uint16_t* next_vd, int it) __attribute__((always_inline)) {
                    const int t0 = t_begin + it * BN;
                    pa_wait_vmem();
                    __syncthreads();  // everyone's part of it is, and tile it - 1's buffer is free
                    if (it + 1 < n_tiles) dma_tile(t0 + BN, next_kd, next_vd);
                    const unsigned bad = bad_runs(t0);
                    if (partly(t0, bad)) finite_only(vd);
                    compute_tile(kd, vd, Sc0, t0, bad);
                };
                dma_tile(t_begin, Ks0, Vs0);
                settle_q();
                for (int it = 0; it < n_tiles; it += 2) {
                    step(Ks0, Vs0, Ks1, Vs1, it);
                    if (it + 1 >= n_tiles) break;
                    step(Ks1, Vs1, Ks0, Vs0, it + 1);
                }
            }
        }

        // V elements that are not finite, left out of the partly hidden tiles, a key at a time: p * inf is
        // inf of that sign for every row that sees the key, two signs or a NaN make NaN.  With key
        // parts, each part takes the keys whose scores it had: its maximum is a number then, and the
        // merge does not multiply the infinity by 0.
        const PagedAttnLaunch& pe = pa_again();
        if (!kQ8 && odd) {
#pragma unroll 1
            for (int it = it0; it < it1; it++) {
                const int t0 = blk.t_first + it * BN;
                if (!partly(t0, SRC == kPaPages && ever_bad)) continue;
#pragma unroll 1
                for (int i = 0; i < BN / KH; i++) {
                    const int key = t0 + 32 * (KH * (i / 32) + kh) + i % 32;
                    if (key > last) break;
                    int64_t at;
                    if constexpr (SRC == kPaPacked) {
                        at = (int64_t)(blk.beg + key) * pe.row_stride;
                    } else {
                        const int id = pe.seqs.page_table[(int64_t)blk.seq * pe.seqs.table_stride + (key >> shift)];
                        if ((unsigned)id >= (unsigned)pe.seqs.n_pages) continue;
                        at = (int64_t)id * pe.page_stride + (int64_t)(key & ps1) * pe.row_stride;
                    }
                    const uint16_t* v = (const uint16_t*)vb0 + at + 4 * lg;
                    if ((unsigned)(key - my_lo) < my_seen) {
#pragma unroll
                        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const uint16_t x = v[32 * dt + 8 * (e >> 2) + (e & 3)];
                                if ((x & 0x7fffu) >= M::kInf) o[dt][e] += to_f32<DT>(x);
                            }
                    }
                }
            }
        }

        // ------------------------------------------------ key parts join, then out
        float lsum = pa_xsum32(lrow_sum);
        // the rows again (not kept through the loop)
        int ln2 = ln;
        asm volatile("" : "+v"(ln2));
        const int row = wr0 + ln2;
        const bool row_ok = row < n_pr;
        const int tok = div_group(pe, min(row, n_pr - 1));
        if constexpr (KH > 1) {
            // Every key part leaves (O, m, l) of its rows in the tile buffers; part k then adds up its
            // 1 / KH of the row group's O: O = sum O_k 2^(m_k - m), m = max m_k.
            constexpr int NO = 32 * D;            // floats of a wave's O
            constexpr int NH = BN * D / 2;        // floats of a buffer
            static_assert(RW * KH * NO <= 2 * NBUF * NH && NH % NO == 0 && D / 8 % KH == 0, "merge buffers");
            auto part_o = [&](int k) __attribute__((always_inline)) {
                const int x = (k * RW + rw) * NO, i = x / NH;
                if constexpr (NBUF == 1) return (float*)(i == 0 ? Ks0 : Vs0) + x % NH;
                else return (float*)(i == 0 ? Ks0 : i == 1 ? Ks1 : i == 2 ? Vs0 : Vs1) + x % NH;
            };
            float* const ml = Ml + rw * 128;      // part k's at + k * RW * 128
            __syncthreads();
            float* const mine = part_o(kh);
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    *(float4*)(mine + ((4 * dt + j) * 64 + lane) * 4) =
                        make_float4(o[dt][4 * j + 0], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]);
            ml[kh * RW * 128 + lane] = mrow;
            ml[kh * RW * 128 + 64 + lane] = lsum;
            __syncthreads();
            float mk[KH];
            mrow = kPaNone;
#pragma unroll
            for (int k = 0; k < KH; k++) mk[k] = ml[k * RW * 128 + lane], mrow = fmaxf(mrow, mk[k]);
            lsum = 0.0f;
#pragma unroll
            for (int k = 0; k < KH; k++) {
                mk[k] = __builtin_amdgcn_exp2f(mk[k] - mrow);
                lsum = fmaf(ml[k * RW * 128 + 64 + lane], mk[k], lsum);
            }
            constexpr int SH = D / 8 / KH;  // float4s of a part's share
#pragma unroll
            for (int i = 0; i < SH; i++) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < KH; k++) {
                    const float4 y = *(const float4*)(part_o(k) + ((kh * SH + i) * 64 + lane) * 4);
                    x.x = fmaf(y.x, mk[k], x.x), x.y = fmaf(y.y, mk[k], x.y);
                    x.z = fmaf(y.z, mk[k], x.z), x.w = fmaf(y.w, mk[k], x.w);
                }
                o[i / 4][i % 4 * 4 + 0] = x.x, o[i / 4][i % 4 * 4 + 1] = x.y;
                o[i / 4][i % 4 * 4 + 2] = x.z, o[i / 4][i % 4 * 4 + 3] = x.w;
            }
        }
        if (!wave_active || !row_ok) continue;
        constexpr int N4 = D / 8 / KH;         // float4s of the row that this lane has ...
        const int first4 = KH > 1 ? kh * N4 : 0;  // ... from this one on
        if constexpr (STREAM) {
            if (!whole) {
                float* const ws = (float*)pe.workspace + (int64_t)(slot * RW + rw) * (32 * D + 64);
#pragma unroll
                for (int i = 0; i < N4; i++)
                    *(float4*)(ws + ((first4 + i) * 64 + lane) * 4) =
                        make_float4(o[i / 4][i % 4 * 4 + 0], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2],
                                    o[i / 4][i % 4 * 4 + 3]);
                if (lg == 0 && kh == 0) {
                    ws[32 * D + ln] = mrow;
                    ws[32 * D + 32 + ln] = lsum;
                }
                continue;
            }
        }
        const float inv = lsum != 0.0f ? __builtin_amdgcn_rcpf(lsum) : 0.0f;  // within an ulp: nothing beside 16 bits
        uint16_t* orow = (uint16_t*)pe.out + (int64_t)(blk.beg + tok) * pe.out_row_stride +
                         (int64_t)(blk.g * pe.group + (row - tok * pe.group)) * pe.out_head_stride;
        const bool f16 = kQ8 ? pe.dtype == GR_DTYPE_F16 : std::is_same_v<DT, F16>;
#pragma unroll
        for (int i = 0; i < N4; i++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = o[i / 4][i % 4 * 4 + e] * inv;
            uint2 r;
            if (f16) r = make_uint2(PaMat<F16>::pack2(x[0], x[1]), PaMat<F16>::pack2(x[2], x[3]));
            else r = make_uint2(PaMat<BF16>::pack2(x[0], x[1]), PaMat<BF16>::pack2(x[2], x[3]));
            *(uint2*)(orow + 8 * (first4 + i) + 4 * lg) = r;
        }
    }
}

// Joins the pieces of the block that boundary w (the start of range w) is the first to cut;
// blockIdx.y: a row group of it, blockIdx.z: a share of its rows' elements.  Thread (row, 4
// elements) runs over the pieces, four at once; with more than four and threads to spare,
// several take a row's pieces among them and add up in LDS (a token after 16000 keys, 32 / 4
// heads d128: 127 pieces a block, 41 -> 24 us a call; after 1000 keys 13.6 -> 12.2).  Bound by latency: 4 us after a token's split kernel, 10
// after that of 501 rows after 7690 keys (256 ranges of 256-row blocks, 33 MB of partials).
template <typename T>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedAttnLaunch p, const int n_ranges) {
    constexpr int D = T::D, RW = T::RW, BM = T::BM, BN = T::BN;
    constexpr int kUnit = 32 * D + 64;
    __shared__ __attribute__((aligned(16))) float4 So[256];
    __shared__ float Sl[256];
    __shared__ float Sm[256];
    const PaSeq c0 = pa_seq<BM, BN>(p, threadIdx.x & 63);
    const int total = pa_stream_total<BM, BN>(p, c0);
    const int q = pa_stream_q(total, n_ranges);
    const int w0 = (int)blockIdx.x;  // the range before the boundary
    if ((int64_t)(w0 + 1) * q >= total) return;
    PaBlock blk;
    const int at = pa_stream_find<BM, BN>(p, c0, (w0 + 1) * q, blk);
    if (at <= 0 || at > q) return;  // no cut here, or an earlier boundary was in this block
    const int group = p.group;
    const int r0 = blk.rb * BM + (int)blockIdx.y * 32;
    const int nr = min(32, blk.n * group - r0);
    if (nr <= 0) return;
    // piece k is range w0 + k's: tiles [k q - (q - at), (k + 1) q - (q - at)) of the block, those in
    // [0, n_tiles); the first one started inside its range (slot 1 of it), the others at its start
    const int lead = q - at;
    const int n_pieces = blk.n_tiles > 0 ? (blk.n_tiles + lead - 1) / q + 1 : 0;
    const float* const ws = (const float*)p.workspace + (int64_t)blockIdx.y * kUnit;
    auto piece = [&](int k) { return ws + (int64_t)(2 * (w0 + k) + (k == 0 ? 1 : 0)) * RW * kUnit; };
    const int tid = threadIdx.x;
    const int n_items = nr * (D / 4);
    const int my_items = (n_items + (int)gridDim.z - 1) / (int)gridDim.z;
    int parts = 1;  // threads per item, a power of two
    constexpr int U = 4;  // pieces at once
    while (my_items * parts * 2 <= 256 && parts * U < n_pieces) parts *= 2;
    const int per = 256 / parts;  // items at once
    const int my_part = tid / per;
    for (int i0 = (int)blockIdx.z * per; i0 < n_items; i0 += (int)gridDim.z * per) {
        const int i = i0 + tid % per;
        const bool mine = i < n_items;
        const int r = mine ? i % nr : 0, c = mine ? i / nr : 0;  // row; float4 c: 8-group c / 2, half c & 1
        const int e = ((c >> 1) * 64 + (c & 1) * 32 + r) * 4;
        float m = kPaNone, l = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine) {
            for (int k0 = my_part; k0 < n_pieces; k0 += U * parts) {
                float4 v[U];
                float mk[U], lk[U];
                float top = m;
#pragma unroll
                for (int j = 0; j < U; j++) {
                    const float* u = piece(min(k0 + j * parts, n_pieces - 1));
                    v[j] = *(const float4*)(u + e);
                    mk[j] = k0 + j * parts < n_pieces ? u[32 * D + r] : -INFINITY;
                    lk[j] = u[32 * D + 32 + r];
                    top = fmaxf(top, mk[j]);
                }
                const float a = __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= a, o.x *= a, o.y *= a, o.z *= a, o.w *= a;
#pragma unroll
                for (int j = 0; j < U; j++) {
                    const float b = __builtin_amdgcn_exp2f(mk[j] - top);
                    if (k0 + j * parts < n_pieces) {
                        l = fmaf(lk[j], b, l);
                        o.x = fmaf(v[j].x, b, o.x), o.y = fmaf(v[j].y, b, o.y);
                        o.z = fmaf(v[j].z, b, o.z), o.w = fmaf(v[j].w, b, o.w);
                    }
                }
            }
        }
        if (parts > 1) {  // my_items * parts <= 256: one round
            So[tid] = o, Sl[tid] = l, Sm[tid] = m;
            __syncthreads();
            if (my_part != 0 || !mine) return;
            float top = m;
            for (int k = 1; k < parts; k++) top = fmaxf(top, Sm[tid + k * per]);
            float a = __builtin_amdgcn_exp2f(m - top);
            l *= a, o.x *= a, o.y *= a, o.z *= a, o.w *= a;
            for (int k = 1; k < parts; k++) {
                const float4 v = So[tid + k * per];
                a = __builtin_amdgcn_exp2f(Sm[tid + k * per] - top);
                l = fmaf(Sl[tid + k * per], a, l);
                o.x = fmaf(v.x, a, o.x), o.y = fmaf(v.y, a, o.y), o.z = fmaf(v.z, a, o.z), o.w = fmaf(v.w, a, o.w);
            }
        }
        if (!mine) continue;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const int tok = div_group(p, r0 + r), h = blk.g * group + (r0 + r - tok * group);
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

// Blocks of a KV head in a launch at most: every sequence's last block may be partly filled.
template <typename T>
int64_t pa_max_blocks(const PagedAttnLaunch& p) {
    const int64_t rows = (int64_t)p.seqs.n_rows * p.group;
    return rows / T::BM + std::min<int64_t>(p.seqs.n_seq, p.seqs.n_rows);
}
// Places of the stream at most.
template <typename T>
int64_t pa_max_places(const PagedAttnLaunch& p) {
    return pa_max_blocks<T>(p) * p.n_kv_heads * (p.seqs.max_len / T::BN + 1);
}

template <typename T>
size_t pa_ws_bytes(int ranges) { return (size_t)2 * ranges * T::RW * (32 * T::D + 64) * 4; }

template <typename DT, typename T, int SRC>
hipError_t pa_launch_ordered(const PagedAttnLaunch& p, hipStream_t st) {
    // whole rounds of the XCDs for every KV head
    const int64_t per = (pa_max_blocks<T>(p) + 7) / 8 * 8;
    paged_attn_kernel<DT, T, SRC, false><<<dim3((unsigned)(per * p.n_kv_heads)), T::NT, 0, st>>>(p);
    return hipGetLastError();
}

template <typename DT, typename T, int SRC>
hipError_t pa_launch_stream(const PagedAttnLaunch& p, int ranges, hipStream_t st) {
    paged_attn_kernel<DT, T, SRC, true><<<dim3((unsigned)ranges), T::NT, 0, st>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // few blocks have many pieces each: their elements are shared among more workgroups (64 rows of 8 / 4
    // heads after 4000 keys, d256: 113 -> 40 us); many blocks: each one more costs a
    // look at the stream (twice as many: 501 rows after 7690 keys, d128, 94.5 -> 97.7 us; up to 16 of
    // a token after 8000 keys, 32 / 4 heads, 19.8 -> 22.3)
    const int64_t blocks = pa_max_blocks<T>(p) * p.n_kv_heads;
    const unsigned share = (unsigned)std::min<int64_t>(std::max<int64_t>(1024 / (blocks * T::RW), 1), T::D / 32);
    paged_combine_kernel<T><<<dim3((unsigned)(ranges - 1), T::RW, share), 256, 0, st>>>(p, ranges);
    return hipGetLastError();
}

bool paged_attn_fits_d64(const PagedAttnLaunch& p);
bool paged_attn_fits_d128(const PagedAttnLaunch& p);
bool paged_attn_fits_d256(const PagedAttnLaunch& p);
size_t paged_attn_ws_d64(const PagedAttnLaunch& p);
size_t paged_attn_ws_d128(const PagedAttnLaunch& p);
size_t paged_attn_ws_d256(const PagedAttnLaunch& p);
hipError_t launch_paged_attn_d64(const PagedAttnLaunch& p, hipStream_t st);
hipError_t launch_paged_attn_d128(const PagedAttnLaunch& p, hipStream_t st);
hipError_t launch_paged_attn_d256(const PagedAttnLaunch& p, hipStream_t st);

// What a kernel's workgroup takes, us measured on MI355X: for a tile alone on its CU, for a tile
// of the CU's time when the CU is full, and of that for its start and end.
struct PaTime {
    float alone, shared, start;
};

// The kernels of a head_dim and which of them a call takes.  Few: blocks of few rows, key
// parts (FewQ8 over Q8 pages), always cut; Wide: the same with larger tiles, for few and long
// blocks, whose pieces are then fewer (Few where a head_dim has none); Mid, Big: one block per workgroup (kMid, kBig), or
// Cut: the tiles of all blocks in equal ranges (kCut: a tile, cutting and joining included;
// kCutFixed: the launches of it).  Fitted to calls timed all three ways; head_dim 256, us for
// Mid / Big / Cut: a prompt of 8000 rows 397 / 312 / 548, 512 rows after 2000 keys 68 / 94 / 37,
// 8 x 500 rows after 3000 keys 178 / 143 / 148, 24 x 64 rows in a window of 1024 49 / 61 / 60,
// 4000 rows over Q8 pages 148 / 192 / 194: the rule took the least of the three in each.
template <typename Few, typename FewQ8, typename Wide, typename Mid, typename Big, typename Cut, typename Costs>
struct PaKernels {
    enum Kind { kFew, kWide, kMid, kBig, kCut };
    static constexpr int kCus = 256;
    template <typename T>
    static constexpr int ranges = kCus * T::kPerCu;

    // Uncut, a launch lasts as long as its longest block alone, or as its tiles take on full CUs,
    // whole rounds of workgroups where all blocks are about as long and one round does not hold them;
    // cut, as its places (each block counts its sequence's longest) and the join.
    static Kind kind(const PagedAttnLaunch& p) {
        const int group = p.group;
        const double len = std::min(p.max_len, p.seqs.max_len);
        if (std::min<int64_t>(p.max_rows, p.seqs.n_rows) * group <= Few::BM) {
            // one block per sequence and KV head; Few / Wide, f16, d128, us: 1 x 16000 keys, 4 KV heads 23.6 /
            // 18.7, 4 x 4000 20.3 / 16.4, 1 x 4000, 8 KV heads 15.8 / 14.0; but 1 x 1000 12.3 / 12.9, 16 x 1k ..
            // 32k, 4 KV heads 97 / 98 - 100, and Q8 pages of 24 sequences to 12k keys, 8 KV heads 101 / 112
            const int64_t n = (int64_t)std::min(p.seqs.n_seq, p.seqs.n_rows) * p.n_kv_heads;
            return !std::is_same_v<Wide, Few> && n <= kCus / 8 && len >= 16 * Wide::BN ? kWide : kFew;
        }
        const double rows = std::min<double>(p.max_rows, len);
        const bool even = p.window > 0 ? len > 2.0 * p.window : rows < 0.4 * len;
        auto blocks = [&](int bm) {  // half of every sequence's last block is empty
            return ((double)p.seqs.n_rows * group / bm + 0.5 * std::min(p.seqs.n_seq, p.seqs.n_rows)) * p.n_kv_heads;
        };
        auto tiles = [&](double keys, int bm, int bn) {
            return p.window > 0 ? std::min(keys / bn, (double)(p.window + bm / group) / bn + 1) : keys / bn;
        };
        auto uncut = [&](auto t, PaTime c) {
            using T = decltype(t);
            double n = blocks(T::BM);
            if (even && n > ranges<T>) n = std::ceil(n / ranges<T> - 0.15) * ranges<T>;
            return std::max(tiles(len, T::BM, T::BN) * c.alone,
                            n * (tiles(len - rows / 2, T::BM, T::BN) * c.shared + c.start) / kCus);
        };
        const double mid = uncut(Mid{}, Costs::kMid), big = uncut(Big{}, Costs::kBig);
        const double cut = Costs::kCutFixed + blocks(Cut::BM) * tiles(len, Cut::BM, Cut::BN) * Costs::kCut.shared / kCus;
        return cut < std::min(mid, big) ? kCut : big < mid ? kBig : kMid;
    }
    // Workgroups of a stream launch: what the GPU holds at once, or the places there are by the
    // caller's bounds, in eights.
    template <typename T>
    static int n_ranges(const PagedAttnLaunch& p) {
        const int64_t tiles = (std::min(p.max_len, p.seqs.max_len) + T::BN - 1) / T::BN;
        const int64_t places = pa_max_blocks<T>(p) * p.n_kv_heads * std::max<int64_t>(tiles, 1);
        return (int)std::min<int64_t>(ranges<T>, (places + 7) / 8 * 8);
    }
    static size_t ws(const PagedAttnLaunch& p) {
        switch (kind(p)) {
            case kFew: return p.kv_dtype == GR_DTYPE_Q8 ? pa_ws_bytes<FewQ8>(n_ranges<FewQ8>(p)) : pa_ws_bytes<Few>(n_ranges<Few>(p));
            case kWide: return pa_ws_bytes<Wide>(n_ranges<Wide>(p));
            case kCut: return pa_ws_bytes<Cut>(n_ranges<Cut>(p));
            default: return 256;
        }
    }
    // Whether a cut call's places can be numbered in 31 bits, an uncut one's threads in 32.
    static bool fits(const PagedAttnLaunch& p) {
        constexpr int64_t kMost = INT32_MAX;
        switch (kind(p)) {
            case kFew: return std::max(pa_max_places<Few>(p), pa_max_places<FewQ8>(p)) < kMost;
            case kWide: return pa_max_places<Wide>(p) < kMost;
            case kCut: return pa_max_places<Cut>(p) < kMost;
            case kMid: return (pa_max_blocks<Mid>(p) + 8) * p.n_kv_heads * Mid::NT < 2 * kMost;
            default: return (pa_max_blocks<Big>(p) + 8) * p.n_kv_heads * Big::NT < 2 * kMost;
        }
    }
    template <typename DT, int SRC>
    static hipError_t launch(const PagedAttnLaunch& p, hipStream_t st) {
        using F = std::conditional_t<SRC == kPaPagesQ8, FewQ8, Few>;
        switch (kind(p)) {
            case kFew: return pa_launch_stream<DT, F, SRC>(p, n_ranges<F>(p), st);
            case kWide:
                if constexpr (!std::is_same_v<Wide, Few>) return pa_launch_stream<DT, Wide, SRC>(p, n_ranges<Wide>(p), st);
                return hipErrorInvalidValue;
            case kCut: return pa_launch_stream<DT, Cut, SRC>(p, n_ranges<Cut>(p), st);
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
