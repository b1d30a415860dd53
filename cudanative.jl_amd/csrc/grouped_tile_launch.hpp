// Instances of k_grouped_tile for one element type and their launch.
#pragma once
#include "grouped_tile.hpp"

#include <algorithm>
#include <type_traits>

namespace miw {

template <class OP, int BI, int BJ, int WI, int WJ, int NX, int NY, int FORM, class DT>
static hipError_t launch_tile_instance(grouped_params p, hipStream_t s)
{
    constexpr int lds = grouped_lds_bytes(BI, BJ, NX, NY, OP::scaled, FORM);
    const void *fn = (const void *)k_grouped_tile<OP, BI, BJ, WI, WJ, NX, NY, FORM, DT>;
    static const hipError_t allowed = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (allowed != hipSuccess) return allowed;
    constexpr bool walks = grouped_walks(OP::scaled, FORM);
    const long blocks = grouped_blocks(p, BI, BJ, grouped_sums(FORM));
    if (walks ? blocks >= MOST_WALKED_TILES : !grid_fits(blocks, 512)) return hipErrorInvalidConfiguration;
    p.most_tiles = (int)blocks;
    // Workgroups that walk their tiles request the next one's first slots ahead of the stores (16384 rows, 8 groups, 4096 x 4096, bf16:
    // 456 us -> 433).  A ragged sum's sums are shorter than its stores, which the loop's loads then wait for (vmcnt counts in
    // order): 238 us -> 291 for 8198 rows, 16 groups, 2048 x 4096.  With 4 bits the registers do not suffice in the largest tile.
    hipLaunchKernelGGL((k_grouped_tile<OP, BI, BJ, WI, WJ, NX, NY, FORM, DT>), dim3((unsigned)(walks ? std::min(blocks, 256l) : blocks)), dim3(512), lds, s, p);
    return hipGetLastError();
}

template <class OP, int FORM, class DT>
static hipError_t launch_tile_size(const grouped_params &p, grouped_tile_size t, hipStream_t s)
{
    switch (t) {
    case TILE_256x256: return launch_tile_instance<OP, 256, 256, 2, 4, OP::scaled || FORM == RAGGED_SUM ? 2 : 3, 2, FORM, DT>(p, s);
    case TILE_256x128:
        if constexpr (FORM == RAGGED_SUM) return launch_tile_instance<OP, 256, 128, 4, 2, 3, 3, RAGGED_SUM_32, DT>(p, s);
        else return launch_tile_instance<OP, 256, 128, 4, 2, 3, 3, FORM, DT>(p, s);
    case TILE_128x128:
        if constexpr (FORM == RAGGED_SUM) return launch_tile_instance<OP, 128, 128, 4, 2, 2, 2, RAGGED_SUM, DT>(p, s);
        else return launch_tile_instance<OP, 128, 128, 4, 2, 4, 4, FORM, DT>(p, s);
    default: return launch_tile_instance<OP, 128, 64, 4, 2, 6, 6, FORM, DT>(p, s);
    }
}

// T: the 16-bit type of results that are not Float32.
template <class OP, class T>
static hipError_t launch_tile(const grouped_params &p, grouped_tile_size t, int d_type, bool ragged_sum, hipStream_t s)
{
    auto go = [&](auto type) {
        using DT = decltype(type);
        if constexpr (OP::scaled) {
            return launch_tile_size<OP, ROWS_X_K, DT>(p, t, s);
        } else {
            if (ragged_sum) return launch_tile_size<OP, RAGGED_SUM, DT>(p, t, s);
            return p.x_k_major ? launch_tile_size<OP, ROWS_X_K, DT>(p, t, s) : launch_tile_size<OP, ROWS_X_I, DT>(p, t, s);
        }
    };
    if (d_type == TYPE_F32) return go(float{});
    return go(T{});
}

}  // namespace miw
