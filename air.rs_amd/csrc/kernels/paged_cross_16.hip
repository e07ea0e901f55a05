// Cross attention with operands rounded to bf16: bf16 queries and outputs over bf16 or 1-byte
// pages (paged_cross_kernel.hpp).
#include "paged_cross_kernel.hpp"

namespace airkv {

hipError_t launch_cross_16(const CrossArgs &a, int head_dim, bool few, hipStream_t s) {
    if (a.dtype == AIR_KV_BF16) return few ? launch_cross_shape<1, false, true>(a, head_dim, s) : launch_cross_shape<1, false, false>(a, head_dim, s);
    return few ? launch_cross_shape<1, true, true>(a, head_dim, s) : launch_cross_shape<1, true, false>(a, head_dim, s);
}

int cross_rows_16(int head_dim, bool few) {
    // (1-byte pages are staged as bf16: the same shape)
    return few ? cross_rows_shape<1, false, true>(head_dim) : cross_rows_shape<1, false, false>(head_dim);
}

}  // namespace airkv
