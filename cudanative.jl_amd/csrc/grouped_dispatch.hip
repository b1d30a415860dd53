// Which kernel runs a product grouped by expert.
#include "experts.hpp"
#include <cstdlib>

namespace miw {

static grouped_tile_size pick(const grouped_params &p)
{
    if (const char *e = getenv("MIW_TILE")) return (grouped_tile_size)atoi(e);
    return p.I > 128 && p.rows / p.groups > 64 ? TILE_256x128 : TILE_128x64;
}

hipError_t launch_grouped(const grouped_params &p, int dtype, int d_type, bool ragged_sum, hipStream_t s)
{
    if (!p.vector || 256 * p.ldx >= 1l << 31) return launch_grouped_plain(p, dtype, d_type, ragged_sum, s);
    return (dtype == TYPE_F16 ? launch_grouped_tile_f16 : launch_grouped_tile_bf16)(p, pick(p), d_type, ragged_sum, s);
}

hipError_t launch_grouped_mxfp4(const grouped_params &p, int d_type, hipStream_t s)
{
    if (256 * p.ldx >= 1l << 31) return launch_grouped_mxfp4_plain(p, d_type, s);
    return launch_grouped_tile_mxfp4(p, pick(p), d_type, s);
}

}  // namespace miw
