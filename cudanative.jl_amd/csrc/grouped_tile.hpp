// LDS-tiled products grouped by expert: f16, bf16 and microscaled 4-bit operands, ragged rows or a ragged sum.
//
// The loop is that of the ping-pong kernel with 64-k clusters (gemm_pingpong.hpp): of the two wavefronts of a SIMD one
// issues nothing but the MFMAs of a slot while the other reads its fragments of the next slot and requests a later one, and
// a barrier swaps them.  What is the same for every type is the movement of bytes: a slot is 128 bytes of k a row, which are
// 64 elements of 16 bits (two MFMA steps of 32) or 256 of 4 bits (two of 128), and a lane's fragment is 16 bytes of its row in
// either case.  So 4-bit operands run through the same loaders and readers, with their scales, eight bytes a row and slot,
// as two more loads.
//   Ragged rows: Y's rows are a tile of one group's, through gather; the lanes' addresses are full ones.  Rows behind the
//     group's last repeat it and are not stored.  X is the group's weights, k contiguous or i contiguous.
//   Ragged sum: both operands have i (j) contiguous and k runs over a group's rows.  X's rows come through gather, whose
//     entries travel to LDS NSLOT - 1 slots ahead of the slot that they are for.
// Where the sum ends inside a slot, lanes fetch the last valid chunk (row) again and its values are zeroed in both operands'
// fragments, in a copy of the loop body that only the last slot runs.
#pragma once
#include "grouped_common.hpp"

namespace miw {

enum grouped_form { ROWS_X_K = 0, ROWS_X_I = 1, RAGGED_SUM = 2 };

struct op_f16 : mfma_f16 {
    static constexpr bool scaled = false;
    static constexpr int slot_k = 64;
};
struct op_bf16 : mfma_bf16 {
    static constexpr bool scaled = false;
    static constexpr int slot_k = 64;
};
struct op_mxfp4 {
    static constexpr bool scaled = true;
    static constexpr int slot_k = 256;
};

// Direct-to-LDS loads with a full address per lane; a wavefront's 16 (4) bytes a lane land at lds_base + DST.
template <int DST>
__device__ inline void lds_load16(const char *lane_address, unsigned lds_base)
{
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_base), "v"(lane_address), "n"(DST) : "memory", "m0", "scc");
}
template <int DST>
__device__ inline void lds_load4(const char *lane_address, unsigned lds_base)
{
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_base), "v"(lane_address), "n"(DST) : "memory", "m0", "scc");
}

constexpr int grouped_slot_bytes(int bi, int bj, bool scaled) { return (bi + bj) * (128 + (scaled ? 8 : 0)); }
constexpr int grouped_lds_bytes(int bi, int bj, int nslot, bool scaled, int form)
{
    return nslot * grouped_slot_bytes(bi, bj, scaled) + (form == RAGGED_SUM ? 2 * nslot * 256 : 0);
}

// Tile of a ragged sum: groups one after the other, in runs over the XCDs, eight tiles along j together.
__device__ inline grouped_tile find_sum_tile(const grouped_params &p, int bi, int bj)
{
    const int tiles_i = (p.I + bi - 1) / bi, tiles_j = (p.J + bj - 1) / bj;
    int id = (int)blockIdx.x;
    const int per = (int)gridDim.x >> 3, rem = (int)gridDim.x & 7, xcd = id & 7, loc = id >> 3;
    id = xcd < rem ? xcd * (per + 1) + loc : rem * (per + 1) + (xcd - rem) * per + loc;
    const int group = id / (tiles_i * tiles_j);
    id -= group * tiles_i * tiles_j;
    const group_rows rows = rows_of_group(p, group);
    const int band = id / (GROUP_J_TILES * tiles_i), in = id - band * GROUP_J_TILES * tiles_i;
    const int height = min(GROUP_J_TILES, tiles_j - band * GROUP_J_TILES);
    const int i = in / height, j = band * GROUP_J_TILES + in - i * height;
    return {group, __builtin_amdgcn_readfirstlane(rows.first), __builtin_amdgcn_readfirstlane(rows.last), j * bj, i * bi};
}

// Zeroes the values of a lane's 16-byte fragment of 16-bit elements from `keep` on.
__device__ inline void keep_first(u32x4 &f, int keep)
{
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] &= keep >= 2 * e + 2 ? 0xffffffffu : keep == 2 * e + 1 ? 0xffffu : 0u;
}

template <class OP, int BI, int BJ, int WI, int WJ, int NSLOT, int FORM, class DT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void k_grouped_tile(grouped_params p)
{
    constexpr int NT = 512;
    static_assert(WI * WJ == 8, "two wavefronts per SIMD");
    constexpr bool XK = FORM == ROWS_X_K, YK = FORM != RAGGED_SUM, SUM = FORM == RAGGED_SUM, SCALED = OP::scaled;
    static_assert(!SCALED || XK, "4-bit operands have k contiguous");
    constexpr int WTI = BI / WI, WTJ = BJ / WJ, TI = WTI / 16, TJ = WTJ / 16;
    constexpr int XBYTES = BI * 128, YBYTES = BJ * 128, SLOT = grouped_slot_bytes(BI, BJ, SCALED);
    constexpr int XS = XBYTES + YBYTES, YS = XS + BI * 8, INDEX = NSLOT * SLOT;  // scales in the slot; the ring of gathered rows
    static_assert(grouped_lds_bytes(BI, BJ, NSLOT, SCALED, FORM) <= 160 * 1024 && NSLOT >= 3, "ring does not fit in LDS");
    constexpr int NLX = BI / 64, NLY = BJ / 64, EXTRA = SCALED ? 2 : SUM ? 1 : 0, LPAIR = NLX + NLY + EXTRA;
    constexpr int NFRAG = 2 * (TI + TJ);
    static_assert(BI % 128 == 0 && BJ % 64 == 0 && WTI % 16 == 0 && WTJ % 16 == 0, "tile");

    extern __shared__ __attribute__((aligned(128))) char smem[];
    MIW_LDS char *lds = (MIW_LDS char *)smem;
    const grouped_tile at = SUM ? find_sum_tile(p, BI, BJ) : find_tile(p, BI, BJ);
    if (at.group < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = wave % WI, wj = wave / WI, q = lane >> 4, r = lane & 15;
    const bool late_group = wave >= 4;
    const int length = SUM ? at.last - at.first : p.K;  // of the sum
    const int NP = (length + OP::slot_k - 1) / OP::slot_k;
    if (SUM && NP == 0 && p.accumulate) return;

    // This thread's chunk of a load: row (k) tid / 8, and the 16 bytes of it that go to place tid % 8.
    const int line = tid >> 3, place = tid & 7;
    const int k_chunk = place ^ ((line >> 1) & 7), i_chunk = place ^ (2 * i_major_swizzle(line));
    // Chunks of 16 bytes (8 values of k) that the last slot has: all lanes fetch valid ones.
    const int last_values = length - (NP - 1) * OP::slot_k;
    const int last_chunks = SCALED ? (last_values + 31) / 32 : (last_values + 7) / 8;

    const char *X = p.X + (SUM ? 0 : (long)at.group * p.sx);
    const char *Y = p.Y;
    // X: a uniform origin that moves with the slots and a lane offset for each load.
    unsigned xvo[NLX];
    const char *yp[NLY];
    if constexpr (XK) {
        X += (long)at.i0 * p.ldx;
#pragma unroll
        for (int i = 0; i < NLX; i++) xvo[i] = (unsigned)(min(line + 64 * i, p.I - 1 - at.i0) * (int)p.ldx + k_chunk * 16);
    } else {
        X += 2l * at.i0;
#pragma unroll
        for (int i = 0; i < NLX; i++) xvo[i] = (SUM ? 0u : (unsigned)(line * (int)p.ldx)) + 2u * (unsigned)min(64 * i + i_chunk * 8, p.I - 8 - at.i0);
    }
    if constexpr (YK) {
#pragma unroll
        for (int i = 0; i < NLY; i++) yp[i] = Y + (long)source_row(p, min(at.j0 + line + 64 * i, at.last - 1)) * p.ldy + k_chunk * 16;
    } else {
#pragma unroll
        for (int i = 0; i < NLY; i++) yp[i] = Y + 2l * (at.j0 + min(64 * i + i_chunk * 8, p.J - 8 - at.j0));
    }
    const int x_scale_wave = wave % (BI / 128), y_scale_wave = wave % (BJ / 32);
    const char *xsp = nullptr, *ysp = nullptr;
    if constexpr (SCALED) {
        xsp = (const char *)p.xs + (long)at.group * p.sxs + 8l * min((long)at.i0 + x_scale_wave * 128 + 2 * lane, p.lxs - 2);
        const int dword = y_scale_wave * 64 + lane;
        ysp = (const char *)p.ys + 8l * source_row(p, min(at.j0 + (dword >> 1), at.last - 1)) + 4 * (dword & 1);
    }
    const long x_step = XK ? 128 : 64 * p.ldx, xs_step = 8 * p.lxs, ys_step = 8 * p.lys;

    const unsigned wave_dst = (unsigned)(uintptr_t)lds + (unsigned)wave * 1024u;
    const unsigned lds0 = (unsigned)(uintptr_t)lds;
    int next = 0;       // slot to request
    unsigned woff = 0;  // its place in the ring
    unsigned xw = 0, yw = 0;  // (ragged sum: the lane's rows of the slot, in bytes from the operands)
    long xrow = 0, yrow = 0;
    (void)xw; (void)yw;
    auto last_slot_begins = [&]() MIW_INLINE {
        if constexpr (XK) {
            const unsigned back = 16u * (unsigned)max(0, k_chunk - (last_chunks - 1));
#pragma unroll
            for (int i = 0; i < NLX; i++) xvo[i] -= back;
        } else if constexpr (!SUM) {
            const unsigned back = (unsigned)(max(0, line - (last_values - 1)) * (int)p.ldx);
#pragma unroll
            for (int i = 0; i < NLX; i++) xvo[i] -= back;
        }
        if constexpr (YK) {
            const int back = 16 * max(0, k_chunk - (last_chunks - 1));
#pragma unroll
            for (int i = 0; i < NLY; i++) yp[i] -= back;
        }
    };
    // Ragged sum: where this lane's row of slot `next` lies in both operands.
    auto find_rows = [&](int gathered) MIW_INLINE {
        const int position = min(at.first + next * 64 + line, at.last - 1);
        yrow = (long)position * p.ldy;
        xrow = (long)gathered * p.ldx;
    };
    auto direct_row = [&]() MIW_INLINE { return source_row(p, min(at.first + next * 64 + line, at.last - 1)); };
    auto index_entry = [&](int slot) MIW_INLINE { return (unsigned)(slot % (2 * NSLOT)) * 256u; };
    auto request_one = [&]<int N>(std::integral_constant<int, N>) MIW_INLINE {
        const unsigned dst = wave_dst + woff;
        if constexpr (N < NLX) {
            if constexpr (SUM) lds_load16<N * NT * 16>(X + xvo[N] + xrow, dst);
            else lds_dma16_at<N * NT * 16, 0>(X, xvo[N], dst);
        } else if constexpr (N < NLX + NLY) {
            constexpr int M = N - NLX;
            if constexpr (SUM) lds_load16<XBYTES + M * NT * 16>(yp[M] + yrow, dst);
            else lds_load16<XBYTES + M * NT * 16>(yp[M], dst);
        } else if constexpr (SCALED) {
            if constexpr (N == NLX + NLY) lds_load16<XS>(xsp, lds0 + woff + (unsigned)x_scale_wave * 1024u);
            else lds_load4<YS>(ysp, lds0 + woff + (unsigned)y_scale_wave * 256u);
        } else if constexpr (SUM) {
            // the rows of the slot NSLOT - 1 further on, by every wavefront to the same place
            const int position = min(at.first + min(next + NSLOT - 1, NP - 1) * 64 + lane, at.last - 1);
            lds_load4<INDEX>((const char *)(p.gather ? p.gather + position : p.offsets), lds0 + index_entry(next + NSLOT - 1));
        }
    };
    auto end_request = [&]() MIW_INLINE {
        woff = woff + SLOT == NSLOT * SLOT ? 0 : woff + SLOT;
        if constexpr (SUM) {
            next++;
        } else if (next < NP - 1) {
            next++;
            X += x_step;
#pragma unroll
            for (int i = 0; i < NLY; i++) yp[i] += 128;
            if constexpr (SCALED) {
                xsp += xs_step;
                ysp += ys_step;
            }
            if (next == NP - 1) last_slot_begins();
        }
    };

    frag_reader<BI, XK> xr;
    frag_reader<BJ, YK> yr;
    xr.init(wi * WTI, lane);
    yr.init(wj * WTJ, lane);
    f32x4 acc[TI][TJ];
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (NP > 0) {
        if (NP == 1) last_slot_begins();
#pragma unroll
        for (int s = 0; s < NSLOT - 1; s++) {
            if constexpr (SUM) find_rows(direct_row());
            [&]<int... I>(std::integer_sequence<int, I...>) { (request_one(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, LPAIR>{});
            end_request();
        }
        wait_loads_and_barrier<(NSLOT - 2) * LPAIR>();

        u32x4 fx[2][TI], fy[2][TJ];
        u32x2 sx[SCALED ? TI : 1], sy[SCALED ? TJ : 1];
        unsigned roff = 0;
        auto cluster_unit = [&]<int U>(MIW_LDS const char *slot, std::integral_constant<int, U>) MIW_INLINE {
            [&]<int... N>(std::integer_sequence<int, N...>) {
                (([&] {
                     if constexpr (N * NFRAG / LPAIR == U) {
                         request_one(std::integral_constant<int, N>{});
                         __builtin_amdgcn_sched_barrier(0);
                     }
                 }()),
                 ...);
            }(std::make_integer_sequence<int, LPAIR>{});
            constexpr int H = U / (TI + TJ), V = U % (TI + TJ);
            if constexpr (V < TI) fx[H][V] = __builtin_bit_cast(u32x4, xr.template read<V, H>(slot));
            else fy[H][V - TI] = __builtin_bit_cast(u32x4, yr.template read<V - TI, H>(slot + XBYTES));
            __builtin_amdgcn_sched_barrier(0);
        };
        auto memory_cluster = [&]() MIW_INLINE {
            MIW_LDS const char *slot = lds + roff;
            if constexpr (SUM) {
                const int row = p.gather ? min(max(*(MIW_LDS const int *)(lds + INDEX + index_entry(next) + 4 * line), 0), p.source_rows - 1)
                                         : min(at.first + next * 64 + line, at.last - 1);
                find_rows(row);
            }
            if constexpr (SCALED) {
#pragma unroll
                for (int a = 0; a < TI; a++) sx[a] = *(MIW_LDS const u32x2 *)(slot + XS + (wi * WTI + 16 * a + r) * 8);
#pragma unroll
                for (int b = 0; b < TJ; b++) sy[b] = *(MIW_LDS const u32x2 *)(slot + YS + (wj * WTJ + 16 * b + r) * 8);
            }
            [&]<int... U>(std::integer_sequence<int, U...>) { (cluster_unit(slot, std::integral_constant<int, U>{}), ...); }(std::make_integer_sequence<int, NFRAG>{});
            end_request();
            roff = roff + SLOT == NSLOT * SLOT ? 0 : roff + SLOT;
            __builtin_amdgcn_sched_barrier(0);
        };
        auto compute_cluster = [&]() MIW_INLINE {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int m = 0; m < TI * TJ; m++) {
                    const int a = m / TJ, b = serpentine_column(m, TJ);
                    if constexpr (SCALED) acc[a][b] = mac_mxfp4(fx[h][a], fy[h][b], acc[a][b], sx[a][h] >> (8 * q), sy[b][h] >> (8 * q));
                    else acc[a][b] = OP::mac(fx[h][a], fy[h][b], acc[a][b]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        };
        // Zeroes what the last slot's lanes fetched again; a block's scale that goes with it becomes 1.
        auto mask_tail = [&]() MIW_INLINE {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (SCALED) {
                    const bool in = 4 * h + q < last_chunks;
#pragma unroll
                    for (int a = 0; a < TI; a++) {
                        if (!in) fx[h][a] = u32x4{0, 0, 0, 0};
                        sx[a][h] = in ? sx[a][h] : 0x7f7f7f7fu;
                    }
#pragma unroll
                    for (int b = 0; b < TJ; b++) {
                        if (!in) fy[h][b] = u32x4{0, 0, 0, 0};
                        sy[b][h] = in ? sy[b][h] : 0x7f7f7f7fu;
                    }
                } else {
                    const int keep = last_values - (32 * h + 8 * q);
#pragma unroll
                    for (int a = 0; a < TI; a++) keep_first(fx[h][a], keep);
#pragma unroll
                    for (int b = 0; b < TJ; b++) keep_first(fy[h][b], keep);
                }
            }
        };
        if (late_group) __builtin_amdgcn_s_barrier();
        for (int s = 0; s < NP - 1; s++) {
            memory_cluster();
            wait_loads_and_barrier<(NSLOT - 2) * LPAIR>();
            compute_cluster();
            __builtin_amdgcn_s_barrier();
        }
        memory_cluster();
        wait_loads_and_barrier<(NSLOT - 2) * LPAIR>();
        mask_tail();
        compute_cluster();
        __builtin_amdgcn_s_barrier();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may outlive the workgroup's LDS
        if (!late_group) __builtin_amdgcn_s_barrier();
    }

    DT *D = (DT *)p.D + (SUM ? (long)at.group * p.sd : 0);
    const int end_j = SUM ? p.J : at.last;
#pragma unroll
    for (int b = 0; b < TJ; b++) {
        const int j = at.j0 + wj * WTJ + 16 * b + r;
        if (j < end_j) {
            DT *row = D + (long)j * p.ldd;
#pragma unroll
            for (int a = 0; a < TI; a++) store_results<DT>(p, row, at.i0 + wi * WTI + 16 * a + 4 * q, acc[a][b]);
        }
    }
}

}  // namespace miw
