// head_dim 128 of the attention over pages and packed rows (paged_attn.hpp).
#include <algorithm>

#include "paged_attn.hpp"

namespace gr {

using K128 = PaKernels<PaTile<128, 1, 2, 64, 4, 1>, PaTile<128, 1, 4, 128, 2, 1>, PaTile<128, 4, 1, 64, 2, 2>, PaTile<128, 8, 1, 128, 2, 2>>;

bool paged_attn_fits_d128(const PagedAttnLaunch& p) { return K128::fits(p); }
size_t paged_attn_ws_d128(const PagedAttnLaunch& p) { return K128::ws(p); }
hipError_t launch_paged_attn_d128(const PagedAttnLaunch& p, hipStream_t st) { return K128::launch_any(p, st); }

}  // namespace gr
