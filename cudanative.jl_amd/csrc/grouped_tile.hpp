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

// Tile of a ragged sum: groups one after the other, eight tiles along j together.
__device__ inline grouped_tile find_sum_tile(const grouped_params &p, int bi, int bj)
{
    const int tiles_i = (p.I + bi - 1) / bi, tiles_j = (p.J + bj - 1) / bj;
    int id = tile_of_workgroup(p.groups * tiles_i * tiles_j);
    if (id < 0) return {-1, 0, 0, 0, 0};
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
    static_assert(grouped_lds_bytes(BI, BJ, NSLOT, SCALED, FORM) <= 160 * 1024 && NSLOT >= 2, "ring does not fit in LDS");
    constexpr bool HALVES = NSLOT == 2;  // a cluster is one MFMA step of the slot, otherwise both
    constexpr int XSW = BI / 128, YSW = BJ / 32;  // wavefronts' loads that a slot's scales take
    constexpr bool SHARED_SCALES = XSW + YSW <= 8;
    constexpr int NLX = BI / 64, NLY = BJ / 64, EXTRA = SCALED ? (SHARED_SCALES ? 1 : 2) : SUM ? 1 : 0, LPAIR = NLX + NLY + EXTRA;
    constexpr int NFRAG = (HALVES ? 1 : 2) * (TI + TJ);  // of a cluster
    static_assert(BI % 128 == 0 && BJ % 64 == 0 && WTI % 32 == 0 && WTJ % 16 == 0, "tile");

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
    // Scales: X's are fetched 16 bytes (two rows) a lane, Y's, whose rows may lie anywhere, four bytes a lane.  Where the
    // wavefronts suffice the first ones fetch X's and the others Y's, one load each; otherwise every one fetches a part of
    // both.  All count the same: those that are left over repeat another's.
    static_assert(!SCALED || (XSW <= 8 && YSW <= 8), "loads of scales");
    const bool x_scales = SHARED_SCALES && wave < XSW;
    const int x_part = wave % XSW, y_part = SHARED_SCALES ? (wave + YSW - XSW % YSW) % YSW : wave % YSW;
    const char *xsp = nullptr, *ysp = nullptr;
    if constexpr (SCALED) {
        xsp = (const char *)p.xs + (long)at.group * p.sxs + 8l * min((long)at.i0 + x_part * 128 + 2 * lane, p.lxs - 2);
        const int dword = y_part * 64 + lane;
        ysp = (const char *)p.ys + 8l * source_row(p, min(at.j0 + (dword >> 1), at.last - 1)) + 4 * (dword & 1);
    }
    const long x_step = XK ? 128 : 64 * p.ldx;

    const unsigned wave_dst = (unsigned)(uintptr_t)lds + (unsigned)wave * 1024u;
    const unsigned lds0 = (unsigned)(uintptr_t)lds;
    int next = 0;       // slot to request
    unsigned woff = 0;  // its place in the ring
    long xrow = 0, yrow = 0;  // (ragged sum: the lane's rows of the slot, in bytes from the operands)
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
            const bool x_turn = SHARED_SCALES ? x_scales : N == NLX + NLY;
            if (x_turn) lds_load16<XS>(xsp, lds0 + woff + (unsigned)x_part * 1024u);
            else lds_load4<YS>(ysp, lds0 + woff + (unsigned)y_part * 256u);
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
                xsp += 8 * p.lxs;
                ysp += 8 * p.lys;
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
        // The first slots (a sum that is shorter than the ring asks for its last slot again, which nobody reads).
#pragma unroll
        for (int s = 0; s < NSLOT - 1; s++) {
            if constexpr (SUM) find_rows(direct_row());
            [&]<int... I>(std::integer_sequence<int, I...>) { (request_one(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, LPAIR>{});
            end_request();
        }
        wait_loads_and_barrier<(NSLOT - 2) * LPAIR>();

        constexpr int FSETS = HALVES ? 1 : 2;
        u32x4 fx[FSETS][TI], fy[FSETS][TJ];
        unsigned lane_sx[SCALED ? TI : 1], lane_sy[SCALED ? TJ : 1];  // this lane's scales of steps 0 and 1 in the low bytes
        const unsigned own_bytes = (unsigned)(q | (4 + q) << 8 | 0x0c0c0000);
        (void)own_bytes;
        unsigned roff = 0;
        constexpr std::integral_constant<int, 0> step0{};
        constexpr std::integral_constant<int, 1> step1{};
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        // Memory cluster H (of one: 0): its fragments, and with REQUEST the loads of the slot NSLOT - 1 further on, all in cluster
        // 0, at even distances between the reads.  REQUEST is false where the sum has no such slot.
        auto memory_cluster = [&]<int H, bool REQUEST>(std::integral_constant<int, H>, std::bool_constant<REQUEST>) MIW_INLINE {
            constexpr bool FIRST = H == 0, LAST = !HALVES || H == 1;
            MIW_LDS const char *slot = lds + roff;
            if constexpr (SUM && FIRST && REQUEST) {
                const int row = p.gather ? min(max(*(MIW_LDS const int *)(lds + INDEX + index_entry(next) + 4 * line), 0), p.source_rows - 1)
                                         : min(at.first + next * 64 + line, at.last - 1);
                find_rows(row);
            }
            u32x2 sx[SCALED ? TI : 1], sy[SCALED ? TJ : 1];  // a row's eight scales of the slot
            if constexpr (SCALED && FIRST) {
#pragma unroll
                for (int a = 0; a < TI; a++) sx[a] = *(MIW_LDS const u32x2 *)(slot + XS + (wi * WTI + 16 * a + r) * 8);
#pragma unroll
                for (int b = 0; b < TJ; b++) sy[b] = *(MIW_LDS const u32x2 *)(slot + YS + (wj * WTJ + 16 * b + r) * 8);
            }
            auto unit = [&]<int U>(std::integral_constant<int, U>) MIW_INLINE {
                if constexpr (FIRST && REQUEST)
                    [&]<int... N>(std::integer_sequence<int, N...>) {
                        (([&] {
                             if constexpr (N * NFRAG / LPAIR == U) {
                                 request_one(std::integral_constant<int, N>{});
                                 __builtin_amdgcn_sched_barrier(0);
                             }
                         }()),
                         ...);
                    }(std::make_integer_sequence<int, LPAIR>{});
                constexpr int S = HALVES ? 0 : U / (TI + TJ), T = HALVES ? H : S, V = U % (TI + TJ);
                if constexpr (V < TI) fx[S][V] = __builtin_bit_cast(u32x4, xr.template read<V, T>(slot));
                else fy[S][V - TI] = __builtin_bit_cast(u32x4, yr.template read<V - TI, T>(slot + XBYTES));
                __builtin_amdgcn_sched_barrier(0);
            };
            [&]<int... U>(std::integer_sequence<int, U...>) { (unit(std::integral_constant<int, U>{}), ...); }(std::make_integer_sequence<int, NFRAG>{});
            if constexpr (FIRST && REQUEST) end_request();
            if constexpr (LAST) roff = roff + SLOT == NSLOT * SLOT ? 0 : roff + SLOT;
            if constexpr (SCALED && FIRST) {
#pragma unroll
                for (int a = 0; a < TI; a++) lane_sx[a] = __builtin_amdgcn_perm(sx[a][1], sx[a][0], own_bytes);
#pragma unroll
                for (int b = 0; b < TJ; b++) lane_sy[b] = __builtin_amdgcn_perm(sy[b][1], sy[b][0], own_bytes);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto multiply = [&]<int S, int T>(std::integral_constant<int, S>, std::integral_constant<int, T>) MIW_INLINE {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < TI * TJ; m++) {
                const int a = m / TJ, b = serpentine_column(m, TJ);
                if constexpr (SCALED) acc[a][b] = mac_mxfp4<T>(fx[S][a], fy[S][b], acc[a][b], lane_sx[a], lane_sy[b]);
                else acc[a][b] = OP::mac(fx[S][a], fy[S][b], acc[a][b]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Zeroes what the last slot's lanes fetched again; a block's scale that goes with it becomes 1.
        auto mask_tail = [&]<int S, int T>(std::integral_constant<int, S>, std::integral_constant<int, T>) MIW_INLINE {
            if constexpr (SCALED) {
                const bool in = 4 * T + q < last_chunks;
                constexpr unsigned one = 0x7fu << (8 * T), others = ~(0xffu << (8 * T));
#pragma unroll
                for (int a = 0; a < TI; a++) {
                    if (!in) fx[S][a] = u32x4{0, 0, 0, 0};
                    if (!in) lane_sx[a] = (lane_sx[a] & others) | one;
                }
#pragma unroll
                for (int b = 0; b < TJ; b++) {
                    if (!in) fy[S][b] = u32x4{0, 0, 0, 0};
                    if (!in) lane_sy[b] = (lane_sy[b] & others) | one;
                }
            } else {
                const int keep = last_values - (32 * T + 8 * q);
#pragma unroll
                for (int a = 0; a < TI; a++) keep_first(fx[S][a], keep);
#pragma unroll
                for (int b = 0; b < TJ; b++) keep_first(fy[S][b], keep);
            }
        };
        // One slot.  At the end of its last memory cluster the wavefront lets the NSLOT - 2 youngest slots stay in flight (none where
        // the sum's last ones are being used up): the next slot has landed, and the barriers that follow publish it.
        auto one_slot = [&]<bool REQUEST, bool MASK>(std::bool_constant<REQUEST> request, std::bool_constant<MASK>) MIW_INLINE {
            constexpr int INFLIGHT = REQUEST ? (NSLOT - 2) * LPAIR : 0;
            memory_cluster(step0, request);
            if constexpr (HALVES) {
                wait_loads_and_barrier<63>();  // (the fragments alone)
                if constexpr (MASK) mask_tail(step0, step0);
                multiply(step0, step0);
                __builtin_amdgcn_s_barrier();
                memory_cluster(step1, request);
                wait_loads_and_barrier<INFLIGHT>();
                if constexpr (MASK) mask_tail(step0, step1);
                multiply(step0, step1);
            } else {
                wait_loads_and_barrier<INFLIGHT>();
                if constexpr (MASK) {
                    mask_tail(step0, step0);
                    mask_tail(step1, step1);
                }
                multiply(step0, step0);
                multiply(step1, step1);
            }
            __builtin_amdgcn_s_barrier();
        };
        if (late_group) __builtin_amdgcn_s_barrier();
        int s = 0;
        for (; s < NP - (NSLOT - 1); s++) one_slot(yes, no);
        for (; s < NP - 1; s++) one_slot(no, no);
        one_slot(no, yes);
        if (!late_group) __builtin_amdgcn_s_barrier();
    }

    // Neighbouring lanes hold neighbouring rows: they exchange the results of two MFMA tiles, so that a row's 32 go out together
    // (128 bytes of Float32) from eight lanes, first the even rows and then the odd ones.
    DT *D = (DT *)p.D + (SUM ? (long)at.group * p.sd : 0);
    const int end_j = SUM ? p.J : at.last;
    const bool odd = r & 1;
#pragma unroll
    for (int b = 0; b < TJ; b++) {
        const int j = at.j0 + wj * WTJ + 16 * b + (r & ~1);
        DT *row = D + (long)j * p.ldd;
#pragma unroll
        for (int a = 0; a < TI; a += 2) {
            float4_t v0 = acc[a][b], v1 = acc[a + 1][b];
            pair_exchange(odd, v0, v1);
            const int i = at.i0 + wi * WTI + 16 * (a + odd) + 4 * q;
            if (j < end_j) store_results<DT>(p, row, i, v0);
            if (j + 1 < end_j) store_results<DT>(p, row + p.ldd, i, v1);
        }
    }
}

}  // namespace miw
