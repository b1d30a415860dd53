// Products grouped by expert where a group has few rows: a decoding step, whose time is that of reading the used experts'
// weights from HBM once.
//
// Nothing goes through LDS on the way in.  A workgroup takes 16 WT rows of one group's weights (k contiguous) and all of the
// group's rows, 16 MT at a time; its wavefronts take the 128-byte chunks of k in turn, a lane loads its 16 bytes of a weight row
// straight into an MFMA fragment, DEPTH chunks ahead, and the partial sums are added in wavefront order through LDS: no second
// kernel, the same bits every time.  Which group and which weights a workgroup has is its number: a group without rows costs a
// look at two offsets.  Registers hold DEPTH * 2 * (WT + MT) * 16 bytes a lane; 16 wavefronts a CU keep some 200 KB on the way.
// Bound by HBM: 64 rows over 64 groups, 1024 x 2048 (f16): 30 to 35 us for 165 MB, 4.7 to 5.6 TB/s; 4 bits, 128 rows over 64 groups, 2048 x 2048:
// 22 to 24 us for 125 MB.  One group of 4096 x 4096: 8 rows 9.8 us in f16, 4.7 in 4 bits (weights partly in the last-level cache).  Partial sums are Float32, rounded once when they are stored.
#pragma once
#include "grouped_tile.hpp"
#include <type_traits>

namespace miw {

static __device__ const u32x4 g_zeros = {0, 0, 0, 0};

template <class OP, int MT, int WT, int WAVES, int DEPTH, class DT>
__global__ __launch_bounds__(64 * WAVES) void k_grouped_narrow(grouped_params p)
{
    constexpr bool SCALED = OP::scaled;
    __shared__ f32x4 part[WAVES][WT * MT][64];
    const int tiles_i = (p.I + 16 * WT - 1) / (16 * WT);
    const int group = (int)blockIdx.x / tiles_i, i0 = (int)blockIdx.x % tiles_i * 16 * WT;
    const group_rows rows = rows_of_group(p, group);
    if (rows.first >= rows.last) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, r = lane & 15;
    const int chunks = (p.K + OP::slot_k - 1) / OP::slot_k;
    // 16-byte pieces of a row: those from `pieces` on are zeros
    const int pieces = SCALED ? (p.K + 31) / 32 : p.K / 8;
    // Every address is a uniform one and an offset of 32 bits for the lane.
    MIW_GLOBAL const char *const W = (MIW_GLOBAL const char *)(uintptr_t)p.X + (long)group * p.sx + (long)i0 * p.ldx;
    MIW_GLOBAL const char *const WS = (MIW_GLOBAL const char *)(uintptr_t)p.xs + (long)group * p.sxs;
    unsigned wo[WT], wso[SCALED ? WT : 1];
#pragma unroll
    for (int t = 0; t < WT; t++) {
        const int i = min(16 * t + r, p.I - 1 - i0);
        wo[t] = (unsigned)(i * (int)p.ldx + 16 * q);
        if constexpr (SCALED) wso[t] = 8u * (unsigned)(i0 + i);
    }
    unsigned yo[MT], yso[SCALED ? MT : 1];
    const unsigned own_bytes = (unsigned)(q | (4 + q) << 8 | 0x0c0c0000);
    (void)own_bytes;

    u32x4 fw[DEPTH][WT][2], fy[DEPTH][MT][2];
    u32x2 sw[DEPTH][SCALED ? WT : 1], sy[DEPTH][SCALED ? MT : 1];
    // What lies behind a row's end, whole chunks among it, is fetched from zeros elsewhere: every load is made in any case.  (With
    // conditions on them, or fragments zeroed behind the loads, the compiler keeps a second set of registers.)
    using bytes = MIW_GLOBAL const char;
    auto piece = [&](bytes *rows, unsigned lane_offset, int chunk, int h) MIW_INLINE {
        bytes *from = rows + (unsigned)(lane_offset + 128u * (unsigned)chunk + 64u * (unsigned)h);
        return *(MIW_GLOBAL const u32x4 *)(8 * chunk + 4 * h + q < pieces ? from : (bytes *)(uintptr_t)&g_zeros);
    };
    auto scales = [&](bytes *first, long panel, unsigned lane_offset, int chunk) MIW_INLINE {
        return *(MIW_GLOBAL const u32x2 *)(first + 8l * min(chunk, chunks - 1) * panel + lane_offset);
    };
    bytes *const Y = (bytes *)(uintptr_t)p.Y, *const YS = (bytes *)(uintptr_t)p.ys;
    auto load_w = [&]<int D>(std::integral_constant<int, D>, int chunk) MIW_INLINE {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int t = 0; t < WT; t++) fw[D][t][h] = piece(W, wo[t], chunk, h);
        if constexpr (SCALED)
#pragma unroll
            for (int t = 0; t < WT; t++) sw[D][t] = scales(WS, p.lxs, wso[t], chunk);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load_y = [&]<int D>(std::integral_constant<int, D>, int chunk) MIW_INLINE {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int m = 0; m < MT; m++) fy[D][m][h] = piece(Y, yo[m], chunk, h);
        if constexpr (SCALED)
#pragma unroll
            for (int m = 0; m < MT; m++) sy[D][m] = scales(YS, p.lys, yso[m], chunk);
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4 acc[WT][MT];
    auto multiply = [&]<int D>(std::integral_constant<int, D>, int chunk) MIW_INLINE {
        unsigned xs[SCALED ? WT : 1], yss[SCALED ? MT : 1];
        if constexpr (SCALED) {
#pragma unroll
            for (int t = 0; t < WT; t++) xs[t] = __builtin_amdgcn_perm(sw[D][t][1], sw[D][t][0], own_bytes);
#pragma unroll
            for (int m = 0; m < MT; m++) yss[m] = __builtin_amdgcn_perm(sy[D][m][1], sy[D][m][0], own_bytes);
        }
        if constexpr (SCALED) {
            // (the scales of blocks behind the row's end are anybody's)
            const unsigned mine = (8 * chunk + q < pieces ? 0xffu : 0u) | (8 * chunk + 4 + q < pieces ? 0xff00u : 0u);
#pragma unroll
            for (int t = 0; t < WT; t++) xs[t] &= mine;
#pragma unroll
            for (int m = 0; m < MT; m++) yss[m] &= mine;
        }
#pragma unroll
        for (int t = 0; t < WT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if constexpr (SCALED) {
                    acc[t][m] = mac_mxfp4<0>(fw[D][t][0], fy[D][m][0], acc[t][m], xs[t], yss[m]);
                    acc[t][m] = mac_mxfp4<1>(fw[D][t][1], fy[D][m][1], acc[t][m], xs[t], yss[m]);
                } else {
                    acc[t][m] = OP::mac(fw[D][t][0], fy[D][m][0], acc[t][m]);
                    acc[t][m] = OP::mac(fw[D][t][1], fy[D][m][1], acc[t][m]);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Chunks wave, wave + WAVES, ...: DEPTH of them on the way, the weights' ahead of the look at which rows there are.
    const int rounds = (chunks + WAVES * DEPTH - 1) / (WAVES * DEPTH);
    auto each = [&]<int... D>(std::integer_sequence<int, D...>, auto f) MIW_INLINE { (f(std::integral_constant<int, D>{}), ...); };
    constexpr std::make_integer_sequence<int, DEPTH> all{};
    for (int j0 = rows.first; j0 < rows.last; j0 += 16 * MT) {
        each(all, [&](auto d) MIW_INLINE { load_w(d, wave + WAVES * d); });
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int j = source_row(p, min(j0 + 16 * m + r, rows.last - 1));
            yo[m] = (unsigned)j * (unsigned)p.ldy + 16u * q;
            if constexpr (SCALED) yso[m] = 8u * (unsigned)j;
        }
        each(all, [&](auto d) MIW_INLINE { load_y(d, wave + WAVES * d); });
#pragma unroll
        for (int t = 0; t < WT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        int chunk = wave;
        for (int n = 1; n < rounds; n++) {
            each(all, [&](auto d) MIW_INLINE {
                multiply(d, chunk + WAVES * d);
                load_w(d, chunk + WAVES * (d + DEPTH));
                load_y(d, chunk + WAVES * (d + DEPTH));
            });
            chunk += WAVES * DEPTH;
        }
        each(all, [&](auto d) MIW_INLINE { multiply(d, chunk + WAVES * d); });
#pragma unroll
        for (int t = 0; t < WT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) part[wave][t * MT + m][lane] = acc[t][m];
        __syncthreads();
        for (int x = wave; x < WT * MT; x += WAVES) {
            const int t = x / MT, m = x % MT, j = j0 + 16 * m + r;
            f32x4 v = part[0][x][lane];
#pragma unroll
            for (int o = 1; o < WAVES; o++) v += part[o][x][lane];
            if (j < rows.last) store_results<DT>(p, (DT *)p.D + (long)j * p.ldd, i0 + 16 * t + 4 * q, v);
        }
        __syncthreads();
    }
}

template <class OP, class DT>
static hipError_t launch_narrow_type(const grouped_params &p, grouped_narrow_form f, hipStream_t s)
{
    const long blocks = (long)p.groups * ((p.I + 16 * f.wt - 1) / (16 * f.wt));
    const dim3 grid((unsigned)blocks), block((unsigned)(64 * f.waves));
    if (f.wt == 2 && f.waves == 2) hipLaunchKernelGGL((k_grouped_narrow<OP, 1, 2, 2, 2, DT>), grid, block, 0, s, p);
    else if (f.wt == 2) hipLaunchKernelGGL((k_grouped_narrow<OP, 1, 2, 4, 2, DT>), grid, block, 0, s, p);
    else if (f.mt == 1) hipLaunchKernelGGL((k_grouped_narrow<OP, 1, 1, 8, 2, DT>), grid, block, 0, s, p);
    else if (f.mt == 2) hipLaunchKernelGGL((k_grouped_narrow<OP, 2, 1, 8, 2, DT>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((k_grouped_narrow<OP, 4, 1, 8, 2, DT>), grid, block, 0, s, p);
    return hipGetLastError();
}

template <class OP, class T>
static hipError_t launch_narrow(const grouped_params &p, grouped_narrow_form f, int d_type, hipStream_t s)
{
    if (d_type == TYPE_F32) return launch_narrow_type<OP, float>(p, f, s);
    return launch_narrow_type<OP, T>(p, f, s);
}

}  // namespace miw
