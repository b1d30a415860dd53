// Scores of the loss: logits that are summed up where they are made.
#include "loss_products.hpp"

#include <algorithm>
#include <cmath>

namespace miw {

static long ceil_div(long a, long b) { return (a + b - 1) / b; }

// As grouped products are, but for a few rows: the vocabulary is one group of many columns, read once, and what counts is how much of it is on the way
// (bf16, weights of repeated calls; microseconds with the join).
//   Up to sixteen rows go straight into registers: from HBM, 16 rows, 32768 x 4096 57 on four wavefronts a workgroup, 62 on 128 x 64 tiles.  Two wavefronts where
//     the sums are short (3 rows, 40000 x 256: 10.8, four 12.8); eight, on sixteen columns each, where the columns would leave CUs idle and the sums are not
//     short (3 rows, 800 x 4096: 11.3, four 13.7).
//   Up to 64 rows for the same reason (48 rows, 800 x 720: 8.3, 128 x 64 tiles 11.6; 3000 x 4096: 26.6 and 28.7), and 32 up to twice the columns.
//   Otherwise tiles: 128 x 64, or 256 x 128 where the CUs would take more than one of those (48 rows, 40000 x 4096: 83 and 99; 32768 x 4096: 68 and 63).
grouped_choice choose_loss_rows(const grouped_params &p, int cus)
{
    const grouped_choice c = choose_grouped(p, false, false, cus);
    const long columns = p.I, chunks = (p.K + 63) / 64;
    if (c.kernel == GROUPED_PLAIN) return c;
    if (p.source_rows * p.ldy < 1l << 32) {  // (the narrow kernel's offsets are 32 bits)
        const bool few = columns <= 16l * cus;
        if (p.rows <= 16 && !(few && chunks >= 24)) return {GROUPED_NARROW, {1, 2, chunks <= 4 ? 2 : 4}, 0, (columns + 31) / 32};
        if ((p.rows <= 64 && few) || (p.rows <= 32 && columns <= 32l * cus)) return {GROUPED_NARROW, {2, 1, 8}, 0, (columns + 15) / 16};
    }
    if (c.kernel == GROUPED_TILE && p.rows > 64) return c;
    const grouped_tile_size t = columns > 128l * cus ? TILE_256x128 : TILE_128x64;
    return {GROUPED_TILE, {0, 0, 0}, t, grouped_blocks(p, t == TILE_128x64 ? 128 : 256, t == TILE_128x64 ? 64 : 128, false)};
}

loss_slices loss_score_slices(const grouped_params &p, int cus)
{
    const grouped_choice c = choose_loss_rows(p, cus);
    auto slices = [&](int tile, int waves) { return loss_slices{tile / waves, (p.I + tile - 1) / tile * waves}; };
    if (c.kernel == GROUPED_PLAIN) return slices(PLAIN, 2);
    if (c.kernel == GROUPED_NARROW) return slices(16 * c.narrow.wt, c.narrow.wt);
    switch (c.tile) {
    case TILE_256x256: return slices(256, 2);
    case TILE_256x128: return slices(256, 4);
    default: return slices(128, 4);
    }
}

// 2^24 of them, 128 MiB, or those of 256 tokens where that is more.  A tile of 256 x 256 makes slices of 128 columns, so 16384 tokens by 128256 words are one run, and more
// runs cost nothing that can be seen (x 1024 bf16: 3.36 ms, 65536 tokens in four runs 13.1; 20000 in two of 10240 4.10).
static long all_stats(long tokens, long vocabulary)
{
    // (the most that any kernel makes of so many tokens or fewer: sixteen columns a slice up to 64 of them, 32 beyond)
    return std::max(std::min(tokens, 64l) * (ceil_div(vocabulary, 16) + 8), tokens * (ceil_div(vocabulary, 32) + 8));
}
long loss_stats(long tokens, long vocabulary) { return std::min(all_stats(tokens, vocabulary), std::max((long)LOSS_STATS, all_stats(LOSS_RUN, vocabulary))); }
long loss_run(grouped_params p, int cus)
{
    const long tokens = p.rows, room = loss_stats(tokens, p.I);
    for (long runs = 1;;) {
        const long run = runs == 1 ? tokens : std::min(tokens, ceil_div(ceil_div(tokens, runs), LOSS_RUN) * LOSS_RUN);
        p.rows = p.source_rows = (int)run;
        const long need = run * loss_score_slices(p, cus).count;
        if (need <= room) return run;
        runs = std::max(runs + 1, runs * need / room);
    }
}

// Tile and slices of the rows' gradients, priced as other products' tiles are, rounds of tiles over the CUs, and each slice for the values that it adds to write
// and read.  150 sizes (3 to 3000 tokens, 800 to 40000 words, 256 to 4096 wide): 1.01 of the fastest combination's time in the geometric mean, 1.12 at
// worst.  The gradient to the rows of 3 tokens, 40000 x 256: 251 us in one slice, 51 in eight, 34 in 32; 700 tokens, 3000 x 4096: 78 in one, 88 in two.
struct cut_price {
    int tile, bi, bj;
    double start, slot;  // microseconds for a tile's start and end, and for 64 columns
};
static const cut_price g_cuts[] = {
    {TILE_256x256, 256, 256, 11.4, 1.20},
    {TILE_256x128, 256, 128, 5.1, 0.85},
    {TILE_128x128, 128, 128, 2.5, 0.75},
    {TILE_128x64, 128, 64, 2.4, 0.64},
};
loss_cut cut_loss_rows(long tokens, long width, long columns, int cus)
{
    const long most = std::max(1l, std::min({(long)LOSS_SLICES, (long)LOSS_SLICED / (tokens * width), columns / 128}));
    loss_cut best{1, TILE_256x256};
    double best_us = 0.0;
    for (const cut_price &t : g_cuts)
        for (long n = 1; n <= most; n++) {
            const long slots = ((columns + n - 1) / n + 63) / 64, slices = (columns + 64 * slots - 1) / (64 * slots);
            const double rounds = (double)(slices * ((tokens + t.bj - 1) / t.bj) * ((width + t.bi - 1) / t.bi)) / cus;
            const double us = (rounds >= 8 ? rounds + 0.5 : std::ceil(rounds)) * (t.start + slots * t.slot) + slices * (0.35 + 2.7e-6 * (double)(tokens * width));
            if (best_us == 0.0 || us < best_us) {
                best = {(int)slices, t.tile};
                best_us = us;
            }
        }
    return best;
}

// Sums that the largest tiles would take are over rows that lie one behind the other: the copy that this needs is 2 bytes read and written for each of X's
// values, the tile loop no longer looks up rows.  (8192 rows, 8192 x 4096 bf16: 368 to 390 us and
// 21 for the copy, 430 with the look; nine tenths of the time left is the loop of MFMAs.  Lane offsets of 64 rows are 32 bits.)
bool loss_sum_is_dense(const grouped_params &p, int cus)
{
    const grouped_choice c = choose_grouped(p, false, true, cus);
    return c.kernel == GROUPED_TILE && c.tile == TILE_256x256 && 64 * p.ldy < 1l << 31;
}

hipError_t launch_loss_scores(const loss_params &p, int dtype, int cus, hipStream_t s)
{
    return dtype == TYPE_F16 ? launch_loss_rows<loss_f16, float, loss_score_end>(p, cus, s) : launch_loss_rows<loss_bf16, float, loss_score_end>(p, cus, s);
}

}  // namespace miw
