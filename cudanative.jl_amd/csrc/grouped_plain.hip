// Products grouped by expert without any demand on sizes, pitches or alignment.
//
// A workgroup takes 64 x 64 results, element by element through LDS in steps of 32 along the sum; what lies beyond an edge is
// zero there.  It runs what the kernels with 16-byte loads cannot.
//
// Bound by the issue of two-byte loads and LDS writes, sixteen of each a thread and step: 16384 rows, 8 groups, 1001 x 1001 (f16, Float32 results):
// 248 us (132 TFLOP/s), the ragged sum 226 (145); 578 and 586 where a step's loads began after the step before.  Sums are Float32 in the MFMA
// accumulators and are rounded once, when they are stored.
#include "grouped_common.hpp"

namespace miw {

constexpr int PLAIN = 64, PLAIN_K = 32, PLAIN_PITCH = PLAIN_K + 8;

template <class MFMA, class DT, bool RAGGED_SUM>
__global__ __launch_bounds__(256) void k_grouped_plain(grouped_params p)
{
    __shared__ __attribute__((aligned(16))) unsigned short xs[PLAIN * PLAIN_PITCH], ys[PLAIN * PLAIN_PITCH];
    __shared__ long source[PLAIN];
    int i0, j0, rows, length, group;
    group_rows range;
    if constexpr (RAGGED_SUM) {
        const int tiles_i = (p.I + PLAIN - 1) / PLAIN, tiles_j = (p.J + PLAIN - 1) / PLAIN;
        group = (int)blockIdx.x / (tiles_i * tiles_j);
        const int at = (int)blockIdx.x % (tiles_i * tiles_j);
        i0 = at % tiles_i * PLAIN;
        j0 = at / tiles_i * PLAIN;
        range = rows_of_group(p, group);
        rows = p.J - j0;
        length = range.last - range.first;
        if (length == 0 && p.accumulate) return;
    } else {
        const grouped_tile t = find_tile(p, PLAIN, PLAIN, (int)blockIdx.x);
        if (t.group < 0) return;
        group = t.group;
        i0 = t.i0;
        j0 = t.j0;
        range = {t.first, t.last};
        rows = t.last - t.j0;
        length = p.K;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, r = lane & 15;
    const int wi = (wave & 1) * 32, wj = (wave >> 1) * 32;
    const unsigned short *X = (const unsigned short *)(p.X + (RAGGED_SUM ? 0 : (long)group * p.sx));
    const unsigned short *Y = (const unsigned short *)p.Y;
    const long ldx = p.ldx / 2, ldy = p.ldy / 2;
    f32x4 acc[2][2] = {};
    const bool k_first = !RAGGED_SUM && p.x_k_major;
    // A step's elements are in registers while the step before is multiplied: PER of each operand a thread, asked for without a branch,
    // from the nearest place inside where theirs lies beyond an edge.  source: rows of this step's X and of the next's.
    constexpr int PER = PLAIN * PLAIN_K / 256;
    unsigned short vx[PER], vy[PER];
    auto find_sources = [&](int k0) {
        if (RAGGED_SUM && tid < PLAIN_K) source[(k0 / PLAIN_K & 1) * PLAIN_K + tid] = (long)source_row(p, min(range.first + k0 + tid, range.last - 1)) * ldx;
    };
    auto fetch = [&](int k0) {
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int at = tid + 256 * n;
            const int i = k_first ? at / PLAIN_K : at % PLAIN, kx = k_first ? at % PLAIN_K : at / PLAIN;
            const int j = RAGGED_SUM ? at % PLAIN : at / PLAIN_K, ky = RAGGED_SUM ? at / PLAIN : at % PLAIN_K;
            const long xi = min(i0 + i, p.I - 1), xk = min(k0 + kx, length - 1), yk = min(k0 + ky, length - 1);
            if constexpr (RAGGED_SUM) {
                vx[n] = X[source[(k0 / PLAIN_K & 1) * PLAIN_K + kx] + xi];
                vy[n] = Y[(range.first + yk) * ldy + j0 + min(j, rows - 1)];
            } else {
                vx[n] = X[k_first ? xi * ldx + xk : xk * ldx + xi];
                vy[n] = Y[source[j] + yk];
            }
        }
    };
    if (length) {
        if constexpr (!RAGGED_SUM) {
            if (tid < PLAIN) source[tid] = (long)source_row(p, min(j0 + tid, range.last - 1)) * ldy;
        }
        find_sources(0);
        find_sources(PLAIN_K);
        __syncthreads();
        fetch(0);
    }
    for (int k0 = 0; k0 < length; k0 += PLAIN_K) {
        __syncthreads();  // (the step before has been read)
#pragma unroll
        for (int n = 0; n < PER; n++) {
            const int at = tid + 256 * n;
            const int i = k_first ? at / PLAIN_K : at % PLAIN, kx = k_first ? at % PLAIN_K : at / PLAIN;
            const int j = RAGGED_SUM ? at % PLAIN : at / PLAIN_K, ky = RAGGED_SUM ? at / PLAIN : at % PLAIN_K;
            xs[i * PLAIN_PITCH + kx] = i0 + i < p.I && k0 + kx < length ? vx[n] : 0;
            ys[j * PLAIN_PITCH + ky] = j < rows && k0 + ky < length ? vy[n] : 0;
        }
        __syncthreads();
        if (k0 + PLAIN_K < length) fetch(k0 + PLAIN_K);
        u32x4 x[2], y[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            x[t] = *(const u32x4 *)&xs[(wi + 16 * t + r) * PLAIN_PITCH + 8 * q];
            y[t] = *(const u32x4 *)&ys[(wj + 16 * t + r) * PLAIN_PITCH + 8 * q];
        }
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int b = 0; b < 2; b++) acc[a][b] = MFMA::mac(x[a], y[b], acc[a][b]);
        find_sources(k0 + 2 * PLAIN_K);  // (into the places of this step's, which nobody reads any more)
    }
    DT *D = (DT *)p.D + (RAGGED_SUM ? (long)group * p.sd : 0);
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int j = wj + 16 * b + r;
        if (j >= rows) continue;
#pragma unroll
        for (int a = 0; a < 2; a++) store_results<DT>(p, D + (long)(j0 + j) * p.ldd, i0 + wi + 16 * a + 4 * q, acc[a][b]);
    }
}

hipError_t launch_grouped_plain(grouped_params p, int dtype, int d_type, bool ragged_sum, hipStream_t s)
{
    const long blocks = ragged_sum ? (long)p.groups * ((p.I + PLAIN - 1) / PLAIN) * ((p.J + PLAIN - 1) / PLAIN) : grouped_blocks(p, PLAIN, PLAIN, false);
    if (!grid_fits(blocks, 256)) return hipErrorInvalidConfiguration;
    p.most_tiles = (int)blocks;
    const dim3 grid((unsigned)blocks), block(256);
    auto go = [&](auto mfma, auto type) {
        using M = decltype(mfma);
        using D = decltype(type);
        if (ragged_sum) hipLaunchKernelGGL((k_grouped_plain<M, D, true>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_grouped_plain<M, D, false>), grid, block, 0, s, p);
    };
    if (dtype == TYPE_F16 && d_type == TYPE_F16) go(mfma_f16{}, f16_t{});
    else if (dtype == TYPE_F16) go(mfma_f16{}, float{});
    else if (d_type == TYPE_BF16) go(mfma_bf16{}, bf16_t{});
    else go(mfma_bf16{}, float{});
    return hipGetLastError();
}

// 4-bit operands: one wavefront per 16 x 16 results, fragments straight from memory.
template <class DT>
__global__ __launch_bounds__(64) void k_grouped_mxfp4_plain(grouped_params p)
{
    const grouped_tile t = find_tile(p, 16, 16, (int)blockIdx.x);
    if (t.group < 0) return;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int i = min(t.i0 + r, p.I - 1), j = source_row(p, min(t.j0 + r, t.last - 1));
    const char *x = p.X + (long)t.group * p.sx + (long)i * p.ldx, *y = p.Y + (long)j * p.ldy;
    const uint8_t *xs = p.xs + (long)t.group * p.sxs + (long)i * 8, *ys = p.ys + (long)j * 8;
    const int blocks = (p.K + 31) / 32;
    f32x4 acc = {};
    for (int b0 = 0; b0 < blocks; b0 += 4) {
        const int b = b0 + q;
        u32x4 xv = {}, yv = {};
        unsigned sx = 127, sy = 127;
        if (b < blocks) {
            xv = *(const u32x4 *)(x + 16l * b);
            yv = *(const u32x4 *)(y + 16l * b);
            sx = xs[(long)(b / 8) * p.lxs * 8 + b % 8];
            sy = ys[(long)(b / 8) * p.lys * 8 + b % 8];
        }
        acc = mac_mxfp4<0>(xv, yv, acc, sx, sy);
    }
    if (t.j0 + r < t.last) store_results<DT>(p, (DT *)p.D + (long)(t.j0 + r) * p.ldd, t.i0 + 4 * q, acc);
}

hipError_t launch_grouped_mxfp4_plain(grouped_params p, int d_type, hipStream_t s)
{
    const long blocks = grouped_blocks(p, 16, 16, false);
    if (!grid_fits(blocks, 64)) return hipErrorInvalidConfiguration;
    p.most_tiles = (int)blocks;
    const dim3 grid((unsigned)blocks), block(64);
    if (d_type == TYPE_F32) hipLaunchKernelGGL(k_grouped_mxfp4_plain<float>, grid, block, 0, s, p);
    else if (d_type == TYPE_F16) hipLaunchKernelGGL(k_grouped_mxfp4_plain<f16_t>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(k_grouped_mxfp4_plain<bf16_t>, grid, block, 0, s, p);
    return hipGetLastError();
}

}  // namespace miw
