// Declarations shared by the experts' kernels, the 4-bit conversions and their C ABI layer.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace miw {

// Element types, numbered as MIW_F16, MIW_F32, MIW_BF16.
enum { TYPE_F16 = 0, TYPE_F32 = 1, TYPE_BF16 = 2 };

// A matrix of more than this is streamed past the caches by the kernels that touch every element once: it, the result and what
// the calls before and after work on no longer share the last-level cache (256 MiB).  Each kernel says what it measured.
constexpr long STREAM_BYTES = 96l << 20;

// --- route.hip
struct route_params {
    const void *logits;
    int *chosen;
    float *gates;
    int *offsets, *rows, *place;
    int *counts;  // workspace: choices of each expert in each chunk of tokens
    int tokens, experts, top, over_all;
    long ld;
    int chunks, chunk;  // chunks of `chunk` tokens
};
// The most chunks that up to so many tokens are cut into; 1: one workgroup does everything and there is no workspace.
int route_most_chunks(long tokens);
hipError_t launch_route(route_params p, int dtype, hipStream_t s);
struct route_grad_params {
    const void *logits;
    const int *chosen;
    const float *gates, *dgates;
    void *dlogits;
    int tokens, experts, top, over_all;
    long ld, ldd;
};
hipError_t launch_route_grad(const route_grad_params &p, int dtype, hipStream_t s);

// --- combine.hip
struct combine_params {
    const void *H, *dY;
    const float *gates;  // or null: 1
    const int *place;
    void *out;      // Y, or dH
    float *dgates;  // or null
    int tokens, top, rows;
    long n, ldh, ldy, lddh;
    int vector;  // 16-byte accesses: pointers, pitches and n allow them
};
hipError_t launch_combine(const combine_params &p, int dtype, hipStream_t s);
hipError_t launch_combine_grad(const combine_params &p, int dtype, hipStream_t s);

// --- gated.hip
struct gated_params {
    const void *Z, *dA;  // dA null: the forward pass
    void *out;           // A, or dZ
    long rows, n, ldz, ldda, ldo;
    int vector;       // 16-byte accesses to Z and dZ, 8-byte ones to A and dA
    int column_bits;  // set by the launch
};
hipError_t launch_gated_silu(gated_params p, int dtype, hipStream_t s);

// --- mxfp4_convert.hip
struct mxfp4_convert_params {
    const void *in;
    void *out;
    uint8_t *codes, *scales;
    long rows, k, ld, ldq, lds;
    int vector;  // 16-byte accesses to the matrix
};
hipError_t launch_mxfp4_quantize(const mxfp4_convert_params &p, int dtype, hipStream_t s);
hipError_t launch_mxfp4_dequantize(const mxfp4_convert_params &p, int dtype, hipStream_t s);

// --- grouped_*.hip
// D[j][i] = sum over k of X_g[i][k] * Y[j][k]: i runs along D's rows (contiguous), j over rows of D.
//   Rows are ragged (miw_grouped_gemm): X is the group's weights, Y the rows of A that gather names.
//   The sum is ragged (miw_grouped_wgrad): k runs over a group's rows, X is B (gathered), Y is A, D the group's own.
struct grouped_params {
    const char *X, *Y;
    const uint8_t *xs, *ys;  // scales of 4-bit operands
    const int *offsets, *gather;
    void *D;
    int groups, rows, source_rows;  // source_rows: of the operand that gather names
    int I, J, K;                    // J: only where the sum is ragged; K: only where the rows are
    long ldx, ldy, ldd;             // X, Y: bytes; D: elements
    long sx, sd, sxs;               // from group to group: X and scales in bytes, D in elements
    long lxs, lys;                  // rows of a panel of scales
    int x_k_major;                  // k contiguous in X
    int gated, accumulate;
    int vector;   // 16-byte accesses to the operands
    int d_vector; // aligned stores of four elements
    int most_tiles;  // workgroups that the tiles need, one each, rounded up to whole eighths; set by the launch
};
enum grouped_tile_size { TILE_256x256, TILE_256x128, TILE_128x128, TILE_128x64 };
hipError_t launch_grouped_tile_f16(const grouped_params &p, grouped_tile_size t, int d_type, bool ragged_sum, hipStream_t s);
hipError_t launch_grouped_tile_bf16(const grouped_params &p, grouped_tile_size t, int d_type, bool ragged_sum, hipStream_t s);
hipError_t launch_grouped_tile_mxfp4(const grouped_params &p, grouped_tile_size t, int d_type, hipStream_t s);
hipError_t launch_grouped_plain(grouped_params p, int dtype, int d_type, bool ragged_sum, hipStream_t s);
hipError_t launch_grouped_mxfp4_plain(grouped_params p, int d_type, hipStream_t s);
// Groups of few rows.  mt: 16-row tiles taken together; wt: 16-row tiles of weights a workgroup.  There are mt 1 with wt 2 on 2 or 4 wavefronts,
// and mt 1, 2 and 4 with wt 1 on 8.
struct grouped_narrow_form {
    int mt, wt, waves;
};
hipError_t launch_grouped_narrow(const grouped_params &p, grouped_narrow_form f, int dtype, int d_type, hipStream_t s);
hipError_t launch_grouped_mxfp4_narrow(const grouped_params &p, grouped_narrow_form f, int d_type, hipStream_t s);
// --- grouped_dispatch.hip: the kernel that runs a product.
enum grouped_kernel { GROUPED_PLAIN, GROUPED_NARROW, GROUPED_TILE };
struct grouped_choice {
    int kernel;
    grouped_narrow_form narrow;  // GROUPED_NARROW
    int tile;                    // GROUPED_TILE
    long workgroups;             // that it asks for, or tiles where workgroups walk them (not set for GROUPED_PLAIN)
};
grouped_choice choose_grouped(const grouped_params &p, bool mxfp4, bool ragged_sum, int cus);
hipError_t launch_grouped(const grouped_params &p, int dtype, int d_type, bool ragged_sum, int cus, hipStream_t s);
hipError_t launch_grouped_mxfp4(const grouped_params &p, int d_type, int cus, hipStream_t s);

// Workgroups of a launch over tiles of bi x bj: at most ceil(rows / bj) and one more for each group, or the sums' own number; whole eighths, since
// an XCD's share may be one more than that.
inline long grouped_blocks(const grouped_params &p, long bi, long bj, bool ragged_sum)
{
    const long tiles_i = (p.I + bi - 1) / bi;
    const long tiles_j = ragged_sum ? (long)p.groups * ((p.J + bj - 1) / bj) : p.rows / bj + (p.groups < p.rows ? p.groups : p.rows);
    return (tiles_i * tiles_j + 7) / 8 * 8;
}
// A launch has fewer than 2^32 threads; tiles that workgroups walk are counted in an int.
constexpr bool grid_fits(long workgroups, long threads) { return workgroups < (1l << 32) / threads; }
constexpr long MOST_WALKED_TILES = 1l << 30;

}  // namespace miw
