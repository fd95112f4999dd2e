// head_dim 256 of the attention over pages and packed rows (paged_attn.hpp).
//
// A wave's O, Q and S fill a SIMD's registers, so one wave per SIMD: LDS reads are sent ahead of
// their products by hand (pa_pipeline).  Few rows over Q8 pages: one tile in LDS instead of
// two, so that two workgroups share a CU and one converts codes while the other multiplies
// (16 tokens of 30k keys, 8 / 4 heads: 343 -> 199 us; f16 pages come by DMA and keep two).
#include "paged_attn.hpp"

namespace gr {

struct Costs256 {
    static constexpr PaTime kMid{2.0f, 1.75f, 11.0f}, kBig{3.05f, 2.6f, 11.0f}, kCut{3.0f, 3.0f, 0.0f};
    static constexpr float kCutFixed = 24.0f;
};
using K256 = PaKernels<PaTile<256, 1, 2, 64, 2, 1>, PaTile<256, 1, 2, 64, 1, 1>,
                       PaTile<256, 1, 2, 64, 2, 1>, PaTile<256, 2, 2, 64, 2, 1>,
                       PaTile<256, 4, 1, 64, 2, 1>, PaTile<256, 4, 1, 64, 2, 1>, Costs256>;

bool paged_attn_fits_d256(const PagedAttnLaunch& p) { return K256::fits(p); }
size_t paged_attn_ws_d256(const PagedAttnLaunch& p) { return K256::ws(p); }
hipError_t launch_paged_attn_d256(const PagedAttnLaunch& p, hipStream_t st) { return K256::launch_any(p, st); }

}  // namespace gr
