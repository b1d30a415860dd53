// The products of the loss for one element type: the grouped kernels with the loss's ends, chosen as grouped products are.
//
// Scores z = x . w of all rows by the vocabulary's vectors; again, of those that count, for the probabilities, share (exp(z - lse) - [target]); and these by the vectors (the rows' gradients) and
// by the rows (the vectors').  Bound by the matrix cores under the power cap where there is work: 4096 rows, 32768 x 4096 bf16: 750, 810 to 820, 700 to 715 and 780 us, 1.27 to 1.49
// PFLOP/s, the probabilities the slowest with their exponentials and 268 MB of stores.  Few rows: by HBM (16 rows: 48 to 52 us for 268 MB).  Few hundred rows: by latency, 11
// to 16 us each (356 rows, 4999 x 720).
#pragma once
#include "grouped_narrow.hpp"
#include "grouped_plain.hpp"
#include "grouped_tile_launch.hpp"
#include "loss_ends.hpp"

namespace miw {

// The element types of the loss's products, so that its instances have names of their own.
struct loss_f16 : op_f16 {
    using plain = mfma_f16;
};
struct loss_bf16 : op_bf16 {
    using plain = mfma_bf16;
};

template <class OP, class DT, class END>
static hipError_t launch_loss_narrow(const loss_params &p, grouped_narrow_form f, hipStream_t s)
{
    const dim3 grid((unsigned)((p.I + 16 * f.wt - 1) / (16 * f.wt))), block((unsigned)(64 * f.waves));
    if (f.mt == 2) hipLaunchKernelGGL((k_grouped_narrow<OP, 2, 1, 8, 2, DT, END>), grid, block, 0, s, p);
    else if (f.waves == 2) hipLaunchKernelGGL((k_grouped_narrow<OP, 1, 2, 2, 2, DT, END>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((k_grouped_narrow<OP, 1, 2, 4, 2, DT, END>), grid, block, 0, s, p);
    return hipGetLastError();
}

template <class OP, class DT, bool RAGGED_SUM, class END>
static hipError_t launch_loss_plain(loss_params p, hipStream_t s)
{
    const long blocks = RAGGED_SUM ? (long)p.groups * ((p.I + PLAIN - 1) / PLAIN) * ((p.J + PLAIN - 1) / PLAIN) : grouped_blocks(p, PLAIN, PLAIN, false);
    if (!grid_fits(blocks, 256)) return hipErrorInvalidConfiguration;
    p.most_tiles = (int)blocks;
    hipLaunchKernelGGL((k_grouped_plain<typename OP::plain, DT, RAGGED_SUM, END>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    return hipGetLastError();
}

// Rows of Y by X with k contiguous in both.
template <class OP, class DT, class END>
static hipError_t launch_loss_rows(const loss_params &p, int cus, hipStream_t s)
{
    const grouped_choice c = choose_loss_rows(p, cus);
    if (c.kernel == GROUPED_PLAIN) return launch_loss_plain<OP, DT, false, END>(p, s);
    if (c.kernel == GROUPED_NARROW) return launch_loss_narrow<OP, DT, END>(p, c.narrow, s);
    return launch_tile_size<OP, ROWS_X_K, DT, END>(p, (grouped_tile_size)c.tile, s);
}
// Rows of Y by X with i contiguous, on the tile of cut_loss_rows.
template <class OP, class DT, class END>
static hipError_t launch_loss_turned(const loss_params &p, int cus, hipStream_t s)
{
    const grouped_choice c = choose_grouped(p, false, false, cus);
    if (c.kernel == GROUPED_PLAIN) return launch_loss_plain<OP, DT, false, END>(p, s);
    return launch_tile_size<OP, ROWS_X_I, DT, END>(p, (grouped_tile_size)p.tile, s);
}
// Sums over the rows.  Large ones (p.dense) are over rows that lie one behind the other in both operands: no row has to be looked up in the loop, and LDS
// has room for a third slot of X.
template <class OP, class DT, class END>
static hipError_t launch_loss_sum(const loss_params &p, int cus, hipStream_t s)
{
    if (p.dense) return launch_tile_instance<OP, 256, 256, 2, 4, 3, 2, DENSE_SUM, DT, END>(p, s);
    const grouped_choice c = choose_grouped(p, false, true, cus);
    if (c.kernel == GROUPED_PLAIN) return launch_loss_plain<OP, DT, true, END>(p, s);
    switch (c.tile) {
    case TILE_256x256:  // (probabilities at too large a pitch)
    case TILE_256x128: return launch_tile_instance<OP, 256, 128, 4, 2, 3, 3, RAGGED_SUM_32, DT, END>(p, s);
    case TILE_128x128: return launch_tile_instance<OP, 128, 128, 4, 2, 2, 2, RAGGED_SUM, DT, END>(p, s);
    default: return launch_tile_instance<OP, 128, 64, 4, 2, 6, 6, RAGGED_SUM, DT, END>(p, s);
    }
}

}  // namespace miw
