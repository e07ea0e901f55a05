// Cross attention at f32 precision: f32 queries or outputs over any pages, or f32 pages
// (paged_cross_kernel.hpp).
#include "paged_cross_kernel.hpp"

namespace airkv {

hipError_t launch_cross_f32(const CrossArgs &a, int head_dim, bool few, hipStream_t s) {
    if (a.dtype == AIR_KV_BF16) return few ? launch_cross_shape<kParts, true>(a, head_dim, s) : launch_cross_shape<kParts, false>(a, head_dim, s);
    return few ? launch_cross_shape<kWide, true>(a, head_dim, s) : launch_cross_shape<kWide, false>(a, head_dim, s);
}

CrossBlocks cross_blocks_f32(int head_dim, bool wide, bool few) {
    if (wide) return few ? cross_blocks_shape<kWide, true>(head_dim) : cross_blocks_shape<kWide, false>(head_dim);
    return few ? cross_blocks_shape<kParts, true>(head_dim) : cross_blocks_shape<kParts, false>(head_dim);
}

}  // namespace airkv
