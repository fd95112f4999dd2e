// head_dim 64 of the attention over pages and packed rows (paged_attn.hpp).
//
// Short rows make the softmax the larger part of a tile, so several small workgroups share a
// CU and hide each other's: 128-row blocks, three waves per SIMD (40 prompts of 9 .. 777 rows,
// bf16, 14 / 2 heads: 35.1 us; four waves 35.2, 64-row blocks 43.6, 256-row blocks 36 - 41).
// One kernel is both Mid and Big.
#include "paged_attn.hpp"

namespace gr {

struct Costs64 {
    static constexpr PaTime kMid{1.0f, 0.74f, 3.0f}, kBig{1.0f, 0.74f, 3.0f}, kCut{2.4f, 2.4f, 0.0f};
    static constexpr float kCutFixed = 18.0f;
};
using K64 = PaKernels<PaTile<64, 1, 4, 128, 2, 2>, PaTile<64, 1, 4, 128, 2, 2>,
                      PaTile<64, 1, 4, 128, 2, 2>, PaTile<64, 4, 1, 64, 2, 3>,
                      PaTile<64, 4, 1, 64, 2, 3>, PaTile<64, 8, 1, 128, 2, 2>, Costs64>;

bool paged_attn_fits_d64(const PagedAttnLaunch& p) { return K64::fits(p); }
size_t paged_attn_ws_d64(const PagedAttnLaunch& p) { return K64::ws(p); }
hipError_t launch_paged_attn_d64(const PagedAttnLaunch& p, hipStream_t st) { return K64::launch_any(p, st); }

}  // namespace gr
