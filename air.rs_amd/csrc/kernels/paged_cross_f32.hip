// Cross attention at f32 precision: f32 queries or outputs over any pages, or f32 pages
// (paged_cross_kernel.hpp).
#include "paged_cross_kernel.hpp"

namespace airkv {

hipError_t launch_cross_f32(const CrossArgs &a, int head_dim, bool few, hipStream_t s) {
    if (a.dtype == AIR_KV_BF16) return few ? launch_cross_shape<kParts, true>(a, head_dim, s) : launch_cross_shape<kParts, false>(a, head_dim, s);
    if (a.dtype == AIR_KV_F32) return few ? launch_cross_shape<kFloats, true>(a, head_dim, s) : launch_cross_shape<kFloats, false>(a, head_dim, s);
    return few ? launch_cross_shape<kWide, true>(a, head_dim, s) : launch_cross_shape<kWide, false>(a, head_dim, s);
}

CrossBlocks cross_blocks_f32(int head_dim, bool wide, bool few) {
    // (kFloats and kWide have the same shapes)
    if (wide) return few ? cross_blocks_shape<kFloats, true>(head_dim) : cross_blocks_shape<kFloats, false>(head_dim);
    return few ? cross_blocks_shape<kParts, true>(head_dim) : cross_blocks_shape<kParts, false>(head_dim);
}

}  // namespace airkv
