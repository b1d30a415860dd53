// What the grouped kernels share: where a group's rows lie, which tile a workgroup takes, and the store of results.
#pragma once
#include "experts.hpp"
#include "gemm_tiled.hpp"
#include "vec_types.hpp"

namespace miw {

// First and last + 1 sorted position of a group, inside 0 .. rows whatever the offsets say; without offsets there is one group.
struct group_rows {
    int first, last;
};
template <class PARAMS>
__device__ inline group_rows rows_of_group(const PARAMS &p, int g)
{
    if (!p.offsets) return {0, p.rows};
    const int first = min(max(p.offsets[g], 0), p.rows), last = min(max(p.offsets[g + 1], 0), p.rows);
    return {first, max(first, last)};
}
// Row of the gathered operand at a sorted position.
template <class PARAMS>
__device__ inline int source_row(const PARAMS &p, int position)
{
    const int row = p.gather ? p.gather[position] : position;
    return min(max(row, 0), p.source_rows - 1);
}

// Tiles of BJ rows over all groups: a group has ceil(rows / BJ), and how many there are is only known on the device.
// The launch has as many workgroups as there can be at most (rows / BJ + groups, times the tiles along i) and each
// finds its own from the offsets: every wavefront sums the groups' tile counts 64 at a time, without LDS.
// Within a group eight tiles of rows share the way along i, and an XCD's CUs take 32 tiles that follow one another, so that
// they read few panels of weights and few of rows at a time.
constexpr int GROUP_J_TILES = 8;
// Workgroup -> tile, or -1.  Workgroups go round-robin over the eight XCDs; 256 tiles at a time are cut into eight runs.  (One run
// of all tiles for each XCD gives it whole groups, and the XCD with the longest ones ends last: the gradient to the
// weights of 16 uneven groups, 4096 x 2048 each, took 314 us like that.)
__device__ inline int tile_of_workgroup(int total, int workgroup)
{
    const int xcd = workgroup & 7, loc = workgroup >> 3;
    const int whole = total >> 8, rest = total & 255;
    if (loc < whole * 32) return (loc >> 5) * 256 + xcd * 32 + (loc & 31);
    const int run = (rest + 7) >> 3, at = loc - whole * 32, tile = xcd * run + at;
    return at < run && tile < rest ? whole * 256 + tile : -1;
}
struct grouped_tile {
    int group, first, last, j0, i0;  // first, last: the group's rows; j0: first row of the tile; group -1: no tile
};
template <class PARAMS>
__device__ inline grouped_tile find_tile(const PARAMS &p, int bi, int bj, int workgroup)
{
    const int lane = (int)threadIdx.x & 63;
    const int tiles_i = (p.I + bi - 1) / bi;
    auto count = [&](int g) MIW_INLINE {
        if (g >= p.groups) return 0;
        const group_rows r = rows_of_group(p, g);
        return (r.last - r.first + bj - 1) / bj;
    };
    int c = count(lane), upto = wave_scan(c);
    int total = __builtin_amdgcn_readlane(upto, 63);
    for (int g0 = 64; g0 < p.groups; g0 += 64) total += __builtin_amdgcn_readlane(wave_scan(count(g0 + lane)), 63);
    total = min(max(total, 0) * tiles_i, p.most_tiles);
    int id = tile_of_workgroup(total, workgroup);
    if (id < 0) return {-1, 0, 0, 0, 0};
    const int row_tile = id / tiles_i;  // (of all groups; a group's tiles are numbered together)
    int g0 = 0, before = 0;
    unsigned long beyond = __ballot(upto > row_tile);
    while (!beyond) {
        before += __builtin_amdgcn_readlane(upto, 63);
        g0 += 64;
        if (g0 >= p.groups) return {-1, 0, 0, 0, 0};
        c = count(g0 + lane);
        upto = wave_scan(c);
        beyond = __ballot(before + upto > row_tile);
    }
    const int at = __builtin_ctzl(beyond);
    const int tiles = __builtin_amdgcn_readlane(c, at);
    before += __builtin_amdgcn_readlane(upto, at) - tiles;
    const group_rows rows = rows_of_group(p, g0 + at);
    id -= before * tiles_i;
    // (offsets that do not rise make sums that are not the launch's: nothing is read or written outside for them)
    if (tiles <= 0 || id < 0 || id >= tiles * tiles_i) return {-1, 0, 0, 0, 0};
    const int band = id / (GROUP_J_TILES * tiles_i), in = id - band * GROUP_J_TILES * tiles_i;
    const int height = min(GROUP_J_TILES, tiles - band * GROUP_J_TILES);
    const int i = in / height, j = band * GROUP_J_TILES + in - i * height;
    return {g0 + at, __builtin_amdgcn_readfirstlane(rows.first), __builtin_amdgcn_readfirstlane(rows.last),
            __builtin_amdgcn_readfirstlane(rows.first) + j * bj, i * bi};
}
// Stores the four results i .. i + 3 of row j; those from I on are left out.  In the gated form they are two pairs of gate and
// value, and two results are stored (I counts the columns before that).
template <class DT, class PARAMS>
__device__ inline void store_results(const PARAMS &p, DT *row, int i, f32x4 v)
{
    if (i >= p.I) return;
    if (p.gated) {
        row += i / 2;
        const f32x2 w = {gated_silu(v[0], v[1]), gated_silu(v[2], v[3])};
        if (p.d_vector && i + 2 < p.I) {
            *(vec<DT, 2> *)row = __builtin_convertvector(w, vec<DT, 2>);
        } else {
            row[0] = (DT)w[0];
            if (i + 2 < p.I) row[1] = (DT)w[1];
        }
        return;
    }
    row += i;
    if (p.d_vector && i + 3 < p.I) {
        vec<DT, 4> *to = (vec<DT, 4> *)row;
        if (p.accumulate) v += __builtin_convertvector(*to, f32x4);
        *to = __builtin_convertvector(v, vec<DT, 4>);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (i + e < p.I) row[e] = (DT)(p.accumulate ? v[e] + (float)row[e] : v[e]);
    }
}

// The matrix instruction of an element type: fragments of 16 bytes a lane.
struct mfma_f16 {
    static __device__ inline f32x4 mac(u32x4 x, u32x4 y, f32x4 acc)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec<_Float16, 8>, x), __builtin_bit_cast(vec<_Float16, 8>, y), acc, 0, 0, 0);
    }
};
struct mfma_bf16 {
    static __device__ inline f32x4 mac(u32x4 x, u32x4 y, f32x4 acc)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec<__bf16, 8>, x), __builtin_bit_cast(vec<__bf16, 8>, y), acc, 0, 0, 0);
    }
};
// 32 values of e2m1 a lane, with one scale each for its 32 of X and of Y in byte BYTE.
template <int BYTE>
__device__ inline f32x4 mac_mxfp4(u32x4 x, u32x4 y, f32x4 acc, unsigned xs, unsigned ys)
{
    typedef int i32x8 __attribute__((ext_vector_type(8)));
    const i32x8 a = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}, b = {(int)y[0], (int)y[1], (int)y[2], (int)y[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4 /* e2m1 */, 4, BYTE, (int)xs, BYTE, (int)ys);
}

}  // namespace miw
