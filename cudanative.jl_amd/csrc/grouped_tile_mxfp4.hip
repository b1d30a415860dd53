// Microscaled 4-bit instances of the tiled kernel for products grouped by expert, and plain ones (one group).
#include "grouped_tile_launch.hpp"

namespace miw {

hipError_t launch_grouped_tile_mxfp4(const grouped_params &p, grouped_tile_size t, int d_type, hipStream_t s)
{
    if (d_type == TYPE_BF16) return launch_tile<op_mxfp4, bf16_t>(p, t, d_type, false, s);
    return launch_tile<op_mxfp4, f16_t>(p, t, d_type, false, s);
}

}  // namespace miw
