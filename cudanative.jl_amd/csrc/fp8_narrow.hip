// Products of 8-bit matrices where a group has few rows: a decoding step, whose time is that of reading the used weights from HBM once.
//
// As grouped_narrow.hpp: a workgroup takes 16 WT rows of one group's weights and all of the group's rows, 16 MT at a time; its wavefronts take the
// 128-byte blocks of k in turn, a lane loads its 32 bytes of a weight row straight into an MFMA fragment, DEPTH blocks ahead, and the partial
// sums are added in wavefront order through LDS: no second kernel, the same bits every time.  A block's scale comes with the row's four of its panel.
// Bound by HBM: 128 rows over 56 of 64 groups, 2048 x 2048, 235 MB in 36 to 41 us (5.7 to 6.4 TB/s, partly from the last-level cache); one group of 16 rows, 32768 x 8192, 54 to 56 us for 270 MB.
// Float32 results, by way of bfloat16, are nearly as fast: the 64 groups 39.7 us (38.8 with 16-bit ones), 16 rows, 8192 x 8192 16.8 (15.8), 64 rows 42 (35.5).
#include "fp8_common.hpp"

namespace miw {

static __device__ const u32x4 g_fp8_zeros = {0, 0, 0, 0};

template <int MT, int WT, int WAVES, int DEPTH, int FORMAT, class DT>
__global__ __launch_bounds__(64 * WAVES) void k_fp8_narrow(grouped_params p)
{
    __shared__ f32x4 part[WAVES][WT * MT][64];
    const int tiles_i = (p.I + 16 * WT - 1) / (16 * WT);
    const int group = (int)blockIdx.x / tiles_i, i0 = (int)blockIdx.x % tiles_i * 16 * WT;
    const group_rows rows = rows_of_group(p, group);
    if (rows.first >= rows.last) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, r = lane & 15;
    const int blocks = (p.K + 127) / 128;
    // Every address is a uniform one and an offset of 32 bits for the lane.
    using bytes = MIW_GLOBAL const char;
    bytes *const W = (bytes *)(uintptr_t)p.X + (long)group * p.sx + (long)i0 * p.ldx, *const WS = (bytes *)(uintptr_t)p.xs + (long)group * p.sxs;
    bytes *const Y = (bytes *)(uintptr_t)p.Y, *const YS = (bytes *)(uintptr_t)p.ys;
    unsigned wo[WT], wso[WT], yo[MT], yso[MT];
#pragma unroll
    for (int t = 0; t < WT; t++) {
        const int i = min(16 * t + r, p.I - 1 - i0);
        wo[t] = (unsigned)(i * (int)p.ldx + 16 * q);
        wso[t] = 4u * (unsigned)(i0 + i);
    }
    u32x4 fw[DEPTH][WT][2], fy[DEPTH][MT][2];
    unsigned sw[DEPTH][WT], sy[DEPTH][MT];
    // Blocks behind the last are fetched from zeros elsewhere: every load is made in any case.  (With conditions on them the compiler
    // keeps a second set of registers.)
    auto piece = [&](bytes *from, unsigned lane_offset, int block, int h) MIW_INLINE {
        bytes *at = from + (unsigned)(lane_offset + 128u * (unsigned)block + 64u * (unsigned)h);
        return *(MIW_GLOBAL const u32x4 *)(block < blocks ? at : (bytes *)(uintptr_t)&g_fp8_zeros);
    };
    auto scale = [&](bytes *first, long panel, unsigned lane_offset, int block) MIW_INLINE {
        return *(MIW_GLOBAL const unsigned *)(first + 4l * (min(block, blocks - 1) >> 2) * panel + lane_offset);
    };
    // Rows of a multiple of 4 KiB would have all workgroups read the same of HBM's channels at a time: each begins at a block of its own (16 rows, f16: 8192 x 8192
    // 20.8 -> 14.9 us, 32768 x 8192 66 -> 56; with rows of 2 KiB it is 3% slower, 32768 x 2048 13.9 and 14.4).
    const int turn = p.ldx % 4096 == 0 ? 9 * ((int)blockIdx.x % blocks) % blocks : 0;
    auto turned = [&](int block) MIW_INLINE { return block < blocks ? (block + turn < blocks ? block + turn : block + turn - blocks) : block; };
    auto load_w = [&]<int D>(std::integral_constant<int, D>, int block) MIW_INLINE {
        block = turned(block);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int t = 0; t < WT; t++) fw[D][t][h] = piece(W, wo[t], block, h);
#pragma unroll
        for (int t = 0; t < WT; t++) sw[D][t] = scale(WS, p.lxs, wso[t], block);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load_y = [&]<int D>(std::integral_constant<int, D>, int block) MIW_INLINE {
        block = turned(block);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int m = 0; m < MT; m++) fy[D][m][h] = piece(Y, yo[m], block, h);
#pragma unroll
        for (int m = 0; m < MT; m++) sy[D][m] = scale(YS, p.lys, yso[m], block);
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4 acc[WT][MT];
    auto multiply = [&]<int D>(std::integral_constant<int, D>, int block) MIW_INLINE {
        block = turned(block);
        const int shift = 8 * (block & 3);
        // (a block behind the last has zeros, and must not have the scale that stands for NaN)
        const unsigned mask = block < blocks ? 255u : 0u;
#pragma unroll
        for (int t = 0; t < WT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const unsigned xs = sw[D][t] >> shift & mask, ys = sy[D][m] >> shift & mask;
                if constexpr (std::is_same_v<DT, float>) acc[t][m] = mac_fp8_wide<FORMAT>(fw[D][t][0], fw[D][t][1], fy[D][m][0], fy[D][m][1], acc[t][m], xs, ys);
                else acc[t][m] = mac_fp8<FORMAT>(fw[D][t][0], fw[D][t][1], fy[D][m][0], fy[D][m][1], acc[t][m], xs, ys);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Blocks wave, wave + WAVES, ...: DEPTH of them on the way, the weights' ahead of the look at which rows there are.
    const int rounds = (blocks + WAVES * DEPTH - 1) / (WAVES * DEPTH);
    auto each = [&]<int... D>(std::integer_sequence<int, D...>, auto f) MIW_INLINE { (f(std::integral_constant<int, D>{}), ...); };
    constexpr std::make_integer_sequence<int, DEPTH> all{};
    for (int j0 = rows.first; j0 < rows.last; j0 += 16 * MT) {
        each(all, [&](auto d) MIW_INLINE { load_w(d, wave + WAVES * d); });
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int j = source_row(p, min(j0 + 16 * m + r, rows.last - 1));
            yo[m] = (unsigned)j * (unsigned)p.ldy + 16u * q;
            yso[m] = 4u * (unsigned)j;
        }
        each(all, [&](auto d) MIW_INLINE { load_y(d, wave + WAVES * d); });
#pragma unroll
        for (int t = 0; t < WT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        int block = wave;
        for (int n = 1; n < rounds; n++) {
            each(all, [&](auto d) MIW_INLINE {
                multiply(d, block + WAVES * d);
                load_w(d, block + WAVES * (d + DEPTH));
                load_y(d, block + WAVES * (d + DEPTH));
            });
            block += WAVES * DEPTH;
        }
        each(all, [&](auto d) MIW_INLINE { multiply(d, block + WAVES * d); });
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

hipError_t launch_fp8_narrow(const grouped_params &p, grouped_narrow_form f, int format, int d_type, hipStream_t s)
{
    const long blocks = (long)p.groups * ((p.I + 16 * f.wt - 1) / (16 * f.wt));
    const dim3 grid((unsigned)blocks), block((unsigned)(64 * f.waves));
    auto with = [&](auto fmt, auto type) {
        constexpr int F = decltype(fmt)::value;
        using DT = decltype(type);
        if (f.wt == 2 && f.waves == 2) hipLaunchKernelGGL((k_fp8_narrow<1, 2, 2, 2, F, DT>), grid, block, 0, s, p);
        else if (f.wt == 2) hipLaunchKernelGGL((k_fp8_narrow<1, 2, 4, 2, F, DT>), grid, block, 0, s, p);
        else if (f.mt == 1) hipLaunchKernelGGL((k_fp8_narrow<1, 1, 8, 2, F, DT>), grid, block, 0, s, p);
        else if (f.mt == 2) hipLaunchKernelGGL((k_fp8_narrow<2, 1, 8, 2, F, DT>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_fp8_narrow<4, 1, 8, 2, F, DT>), grid, block, 0, s, p);
        return hipGetLastError();
    };
    auto go = [&](auto type) {
        return format == FORMAT_E4M3 ? with(std::integral_constant<int, FORMAT_E4M3>{}, type) : with(std::integral_constant<int, FORMAT_E5M2>{}, type);
    };
    if (d_type == TYPE_F32) return go(float{});
    if (d_type == TYPE_F16) return go(f16_t{});
    return go(bf16_t{});
}

}  // namespace miw
