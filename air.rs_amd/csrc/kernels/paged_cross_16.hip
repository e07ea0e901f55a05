// Cross attention with 16-bit operands: bf16 queries and outputs over bf16 or 1-byte pages
// (paged_cross_kernel.hpp).
#include "paged_cross_kernel.hpp"

namespace airkv {

hipError_t launch_cross_16(const CrossArgs &a, int head_dim, bool few, hipStream_t s) {
    if (a.dtype == AIR_KV_BF16) return few ? launch_cross_shape<kBf16, true>(a, head_dim, s) : launch_cross_shape<kBf16, false>(a, head_dim, s);
    return few ? launch_cross_shape<kCodes, true>(a, head_dim, s) : launch_cross_shape<kCodes, false>(a, head_dim, s);
}

CrossBlocks cross_blocks_16(int head_dim, bool codes, bool few) {
    if (codes) return few ? cross_blocks_shape<kCodes, true>(head_dim) : cross_blocks_shape<kCodes, false>(head_dim);
    return few ? cross_blocks_shape<kBf16, true>(head_dim) : cross_blocks_shape<kBf16, false>(head_dim);
}

}  // namespace airkv
