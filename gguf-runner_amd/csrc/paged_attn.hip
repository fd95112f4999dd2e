// Attention over pages and packed rows: dispatch by head_dim (paged_attn.hpp).
#include "paged_attn.hpp"

namespace gr {

bool paged_attn_fits(const PagedAttnLaunch& p) {
    return p.head_dim == 64 ? paged_attn_fits_d64(p) : p.head_dim == 128 ? paged_attn_fits_d128(p) : paged_attn_fits_d256(p);
}

size_t paged_attn_ws_bytes(const PagedAttnLaunch& p) {
    return p.head_dim == 64 ? paged_attn_ws_d64(p) : p.head_dim == 128 ? paged_attn_ws_d128(p) : paged_attn_ws_d256(p);
}

hipError_t launch_paged_attn(const PagedAttnLaunch& p, hipStream_t st) {
    return p.head_dim == 64 ? launch_paged_attn_d64(p, st)
                            : p.head_dim == 128 ? launch_paged_attn_d128(p, st) : launch_paged_attn_d256(p, st);
}

}  // namespace gr
