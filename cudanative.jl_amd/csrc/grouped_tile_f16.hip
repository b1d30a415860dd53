// Float16 instances of the tiled kernel for products grouped by expert.
#include "grouped_tile_launch.hpp"

namespace miw {

hipError_t launch_grouped_tile_f16(const grouped_params &p, grouped_tile_size t, int d_type, bool ragged_sum, hipStream_t s)
{
    return launch_tile<op_f16, f16_t>(p, t, d_type, ragged_sum, s);
}

}  // namespace miw
