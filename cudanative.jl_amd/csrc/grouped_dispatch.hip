// Which kernel runs a product grouped by expert.
//
// How many rows a group has is not known on the host: the rules go by the mean, rows / groups.  Their numbers come from some 400
// products timed on every kernel (1 to 128 groups, 512 to 4096 wide, 0.5 to 2048 rows a group whose loads differ by up to three
// times, f16 with k or i contiguous in the weights and 4 bits, weights from HBM): the rule's kernel takes 1.007 (f16) and 1.012 (4 bits)
// of the fastest one's time in the geometric mean, at worst 1.38 and 1.52 (loads that happen to make a round more or less).
#include "experts.hpp"

#include <algorithm>
#include <cmath>

namespace miw {

static long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Groups of few rows are read through registers (grouped_narrow.hpp) where that is faster than a tile:
//   Few workgroups at 32 rows of weights each (a single projection): 16 rows and eight wavefronts that share k, up to 64 rows.  1
//     group, 4096 x 4096, f16, 8 rows: 10.2 us, 13.7 with 32 rows and four wavefronts, 28.8 on 128 x 64 tiles; 64 rows 22.5, tiles 29.8.
//   Otherwise up to ten rows a group, 16 at a time (64 groups, 1024 x 2048, f16: 4 rows 51.0 us, tiles 65.5; 14 rows 77.5 and
//     64.8), on as many wavefronts as have two chunks of k or more each: 4 bits, 64 groups, 768 x 512 (two chunks): two
//     wavefronts 6.0 us, four 9.2; f16, 1024 x 2048 (32 chunks): 54.5 and 51.0.  Eight where k is long and the groups are few (8 groups, 4096 x
//     4096, f16: 49.2 us, four wavefronts 63.1; 64 groups, 1024 x 2048: 63.4 and 51.0).
// Loads far from even are not seen here: a group of more rows reads its weights once for every 16.  64 groups, 640 rows, 1024 x 2048, f16: 55 us even, 142 with half of
// them in one group, 223 with all; 4 bits, 2048 x 2048: 30, 60 and 78.
static grouped_narrow_form pick_narrow(const grouped_params &p, int slot_k)
{
    const double per_group = (double)p.rows / p.groups;
    const long workgroups = p.groups * ceil_div(p.I, 32), chunks = ceil_div(p.K, slot_k);
    if (!p.x_k_major || p.source_rows * p.ldy >= 1l << 32) return {0, 0, 0};  // (its offsets are 32 bits; the weights' rows are contiguous along k)
    if (workgroups <= 256 && per_group <= 64) return {per_group <= 16 ? 1 : per_group <= 32 ? 2 : 4, 1, 8};
    if (per_group > 10) return {0, 0, 0};
    if (chunks >= 64 && workgroups <= 1024) return {1, 1, 8};
    const int waves = chunks >= 16 ? 4 : 2;
    if (!grid_fits(workgroups, 64 * waves)) return {0, 0, 0};  // (it has a workgroup for every group, with rows or without; a tile's launch has not)
    return {1, 2, waves};
}

struct tile_price {
    grouped_tile_size size;
    int bi, bj;
    double f16_slot, f16_tile, mxfp4_slot, mxfp4_tile;  // microseconds for a slot of k and for a tile's start and end
};
static const tile_price g_tiles[] = {
    {TILE_256x256, 256, 256, 1.35, 6.4, 1.33, 12.0},
    {TILE_256x128, 256, 128, 0.92, 3.6, 0.89, 7.2},
    {TILE_128x128, 128, 128, 0.58, 6.3, 0.57, 6.0},
    {TILE_128x64, 128, 64, 0.36, 3.3, 0.50, 4.4},
};

// Ragged rows: the tile with the shortest estimated launch, rounds of tiles over the CUs at the measured price of each.  A group's
// last tile is half full in the mean, and off that by 0.29 of a tile (the root of 1/12): a round is counted where there are tiles for it beyond what
// that makes of all groups together.
static grouped_tile_size pick_rows_tile(const grouped_params &p, int slot_k, int cus)
{
    const double per_group = (double)p.rows / p.groups, slots = (double)ceil_div(p.K, slot_k);
    const tile_price *best = nullptr;
    double best_us = 0.0;
    for (const tile_price &t : g_tiles) {
        if (best && slot_k == 256 && !grid_fits(grouped_blocks(p, t.bi, t.bj, false), 512)) continue;  // (4 bits: no walk)
        const double high = p.groups == 1 ? (double)ceil_div(p.rows, t.bj) : per_group <= 0.5 * t.bj ? 1.0 : per_group / t.bj + 0.5;
        const double rounds = (double)std::min(p.groups, p.rows) * high * (double)ceil_div(p.I, t.bi) / cus;
        const double spread = p.groups > 1 && per_group > 0.5 * t.bj ? std::sqrt(p.groups / 12.0) * (double)ceil_div(p.I, t.bi) / cus : 0.0;
        const double whole = rounds >= 8 ? rounds + 0.5 : std::max(1.0, (double)(long)std::max(rounds + 0.995 - spread, 0.0));
        const double us = whole * (slot_k == 64 ? t.f16_tile + slots * t.f16_slot : t.mxfp4_tile + slots * t.mxfp4_slot);
        if (!best || us < best_us) {
            best = &t;
            best_us = us;
        }
    }
    // Weights with i contiguous are read in whole lines by the wider tile: 64 groups of 8 rows, 2048 x 1024: 44.5 us, 51.4 with 128 x 64.
    if (best->size == TILE_128x64 && !p.x_k_major && p.groups * ceil_div(p.I, 256) >= cus) return TILE_256x128;
    return best->size;
}

// Ragged sums, priced in the same way: a tile's start and end with its stores, and 64 rows of its sum, where a CU holds one workgroup (256 x 256,
// 128 x 64) or two.  105 sums (1 to 128 groups, 304 to 4096 wide, 1 to 2048 rows a group): 1.01 of the fastest tile's time in the mean, 1.17 at worst.
// 16 groups, 2048 x 4096, Float32: 128 rows 142 us on 256 x 128 with slots of 32, 154 on 256 x 256; 8 groups of 2048 rows, 4096 x 4096: 618 and
// 560; 7 groups of 330 rows, 3040 x 336: 16.4 us on 128 x 128, 21.4 on 256 x 128; one group of 2048 rows, 1024 x 1024: 22 on 128 x 64, 30 on 128 x 128.
struct sum_price {
    grouped_tile_size size;
    int bi, bj, together;
    double tile, slot;
};
static const sum_price g_sums[] = {
    {TILE_256x256, 256, 256, 1, 9.1, 1.40},
    {TILE_256x128, 256, 128, 2, 6.6, 1.55},
    {TILE_128x128, 128, 128, 2, 4.7, 0.88},
    {TILE_128x64, 128, 64, 1, 4.7, 0.39},
};
static grouped_tile_size pick_sum_tile(const grouped_params &p, int cus)
{
    const double slots = (double)p.rows / p.groups / 64 + (p.groups > 1 ? 0.5 : 0.0);
    const sum_price *best = nullptr;
    double best_us = 0.0;
    for (const sum_price &t : g_sums) {
        if (best && !grid_fits(grouped_blocks(p, t.bi, t.bj, true), 512)) continue;
        const double rounds = (double)p.groups * (double)ceil_div(p.I, t.bi) * (double)ceil_div(p.J, t.bj) / (t.together * cus);
        const double us = (rounds >= 3 ? rounds + 0.25 : std::max(1.0, (double)(long)(rounds + 0.95))) * (t.tile + slots * t.slot);
        if (!best || us < best_us) {
            best = &t;
            best_us = us;
        }
    }
    return best->size;
}

grouped_choice choose_grouped(const grouped_params &p, bool mxfp4, bool ragged_sum, int cus)
{
    // (lane offsets of 256 rows, or of 64 along k, are 32 bits; a sum over no rows has none to fetch)
    if (!p.vector || 256 * p.ldx >= 1l << 31 || p.rows == 0) return {GROUPED_PLAIN, {0, 0, 0}, 0, 0};
    const int slot_k = mxfp4 ? 256 : 64;
    if (!ragged_sum)
        if (const grouped_narrow_form f = pick_narrow(p, slot_k); f.mt) return {GROUPED_NARROW, f, 0, p.groups * ceil_div(p.I, 16 * f.wt)};
    const grouped_tile_size size = ragged_sum ? pick_sum_tile(p, cus) : pick_rows_tile(p, slot_k, cus);
    const tile_price &t = *std::find_if(std::begin(g_tiles), std::end(g_tiles), [&](const tile_price &x) { return x.size == size; });
    return {GROUPED_TILE, {0, 0, 0}, size, grouped_blocks(p, t.bi, t.bj, ragged_sum)};
}

hipError_t launch_grouped(const grouped_params &p, int dtype, int d_type, bool ragged_sum, int cus, hipStream_t s)
{
    const grouped_choice c = choose_grouped(p, false, ragged_sum, cus);
    if (c.kernel == GROUPED_PLAIN) return launch_grouped_plain(p, dtype, d_type, ragged_sum, s);
    if (c.kernel == GROUPED_NARROW) return launch_grouped_narrow(p, c.narrow, dtype, d_type, s);
    return (dtype == TYPE_F16 ? launch_grouped_tile_f16 : launch_grouped_tile_bf16)(p, (grouped_tile_size)c.tile, d_type, ragged_sum, s);
}

hipError_t launch_grouped_mxfp4(const grouped_params &p, int d_type, int cus, hipStream_t s)
{
    const grouped_choice c = choose_grouped(p, true, false, cus);
    if (c.kernel == GROUPED_PLAIN) return launch_grouped_mxfp4_plain(p, d_type, s);
    if (c.kernel == GROUPED_NARROW) return launch_grouped_mxfp4_narrow(p, c.narrow, d_type, s);
    return launch_grouped_tile_mxfp4(p, (grouped_tile_size)c.tile, d_type, s);
}

}  // namespace miw
