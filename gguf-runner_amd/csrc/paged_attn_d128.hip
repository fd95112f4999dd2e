// head_dim 128 of the attention over pages and packed rows (paged_attn.hpp).
//
// Eight waves of 32 rows share a 128-key tile where there are blocks enough (one workgroup per
// CU, two waves per SIMD: a wave's softmax runs under the other's products), four waves of a
// 64-key tile where there are not.  Cut calls take the large block: 501 rows after 7690 keys,
// 32 / 8 heads, f16: 92 us, 124 with the small one, whose blocks leave twice the partials.
#include "paged_attn.hpp"

namespace gr {

struct Costs128 {
    static constexpr PaTime kMid{1.6f, 1.2f, 5.0f}, kBig{4.0f, 4.4f, 10.0f}, kCut{4.4f, 4.4f, 0.0f};
    static constexpr float kCutFixed = 18.0f;
};
using K128 = PaKernels<PaTile<128, 1, 2, 64, 2, 1>, PaTile<128, 1, 2, 64, 2, 1>,
                       PaTile<128, 1, 4, 128, 2, 1>, PaTile<128, 4, 1, 64, 2, 2>,
                       PaTile<128, 8, 1, 128, 2, 2>, PaTile<128, 8, 1, 128, 2, 2>, Costs128>;

bool paged_attn_fits_d128(const PagedAttnLaunch& p) { return K128::fits(p); }
size_t paged_attn_ws_d128(const PagedAttnLaunch& p) { return K128::ws(p); }
hipError_t launch_paged_attn_d128(const PagedAttnLaunch& p, hipStream_t st) { return K128::launch_any(p, st); }

}  // namespace gr
