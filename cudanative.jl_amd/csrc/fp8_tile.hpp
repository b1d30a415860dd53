// LDS-tiled products of 8-bit matrices, plain and grouped by expert.
//
// The loop is that of grouped_tile.hpp: of the two wavefronts of a SIMD one issues nothing but the MFMAs of a cluster while the other reads its
// fragments of the next one and requests a later slot, and a barrier swaps them.  A slot is 128 bytes of k a row, which is one block: rows are
// padded with zeros to whole blocks, so there is no tail, and the scales of a slot are one byte a row.  They come as the four bytes that a
// row has in a panel, one load of 64 rows a wavefront, and are shifted to the slot's byte when its fragments are read.
//   16-bit results: one MFMA of 128 k takes both 16-byte pieces that a lane has of a row's slot, and applies the scales.
//   Float32 results: the pieces become bfloat16 with their scale, eight values at a time (fp8_common.hpp says why).
//
// Bound by the power cap where tiles are many (256 x 256, half a wavefront's rows at a time: 4096 x 4096 x 4096 57 us, 2.4 PFLOP/s, x 8192 102 to 104; the latter with zeros for data 83,
// of which the MFMAs beside LDS reads alone take 70 and the loads alone 72), by latency where they are few: 509 x 656 x 720 with Float32 results is 48 tiles of 128 x 64 on 256 CUs, each a
// chain of six slots that are widened: 8 us, where a launch takes 3.5 (smaller tiles, or wavefronts that share k, are not there). Float32
// results on 256 x 128: 4096 x 4096 x 8192 218 us, 1.26 PFLOP/s, nine tenths of what the 16-bit instructions reach in products of 16 bits.
#pragma once
#include "fp8_common.hpp"

#include <type_traits>

namespace miw {

constexpr int fp8_slot_bytes(int rows) { return rows * (128 + 4); }
constexpr int fp8_lds_bytes(int bi, int bj, int slots) { return slots * (fp8_slot_bytes(bi) + fp8_slot_bytes(bj)); }

// Direct-to-LDS loads with a full address per lane; a wavefront's 16 (4) bytes a lane land at lds_base + DST.
template <int DST>
__device__ inline void fp8_load16(const char *lane_address, unsigned lds_base)
{
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_base), "v"(lane_address), "n"(DST) : "memory", "m0", "scc");
}
__device__ inline void fp8_load4(const char *lane_address, unsigned lds_at)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_at), "v"(lane_address) : "memory", "m0");
}

// NS slots in LDS.  Three or more: a cluster is a whole slot; the slot NS - 1 further on is requested in a slot's memory cluster, into
// the place of the one before, and at its end the NS - 2 youngest stay in flight.  Two (tiles of 256 x 256): a cluster is half of the
// wavefront's rows of X, the next slot is requested in the first memory cluster and has to have landed at the end of the second.
template <int BI, int BJ, int WI, int WJ, int NS, int FORMAT, class DT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void k_fp8_tile(grouped_params p)
{
    constexpr int NT = 512;
    static_assert(WI * WJ == 8, "two wavefronts per SIMD");
    constexpr bool WIDE = std::is_same_v<DT, float>, HALVES = NS == 2;
    constexpr int WTI = BI / WI, WTJ = BJ / WJ, TI = WTI / 16, TJ = WTJ / 16, PARTS = HALVES ? 2 : 1, TP = TI / PARTS;
    constexpr int XBYTES = BI * 128, YBYTES = BJ * 128, XSLOT = fp8_slot_bytes(BI), YSLOT = fp8_slot_bytes(BJ), XRING = NS * XSLOT, YRING = NS * YSLOT;
    static_assert(fp8_lds_bytes(BI, BJ, NS) <= 160 * 1024, "rings do not fit in LDS");
    constexpr int NLX = BI / 64, NLY = BJ / 64, LSLOT = NLX + NLY + 1;  // loads a thread and slot
    constexpr int XSW = BI / 64, YSW = BJ / 64;                         // wavefronts' loads that a slot's scales take
    static_assert(XSW + YSW <= 8, "one load of scales a wavefront");
    static_assert(BI % 64 == 0 && BJ % 64 == 0 && WTI % 32 == 0 && WTJ % 16 == 0 && TI % PARTS == 0, "tile");

    extern __shared__ __attribute__((aligned(128))) char smem[];
    MIW_LDS char *lds = (MIW_LDS char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = wave % WI, wj = wave / WI, r = lane & 15;
    const bool late_group = wave >= 4;
    // Between tiles the arguments are read again and what hangs on the thread's number is made again: kept through the K loop
    // they would take more registers than there are.
    auto arguments = [] MIW_INLINE {
        auto a = (const __attribute__((address_space(4))) grouped_params *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };
    auto thread = [] MIW_INLINE {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    };
    // The first wavefronts fetch X's scales, the others Y's; those that are left over repeat another's.
    const bool x_scales = wave < XSW;
    const int part = x_scales ? wave : (wave - XSW) % YSW;

    struct walked_tile {
        grouped_tile at;
        int rows[NLY];  // of this thread's lines of Y
        int scale_row;  // of its scale of Y
    };
    auto find = [&](int workgroup) MIW_INLINE {
        walked_tile t;
        const auto a = arguments();
        const int me = thread(), line = me >> 3;
        const grouped_tile at = find_tile(*a, BI, BJ, workgroup);
        t.at = {__builtin_amdgcn_readfirstlane(at.group), __builtin_amdgcn_readfirstlane(at.first), __builtin_amdgcn_readfirstlane(at.last),
                __builtin_amdgcn_readfirstlane(at.j0), __builtin_amdgcn_readfirstlane(at.i0)};
        t.scale_row = 0;
#pragma unroll
        for (int i = 0; i < NLY; i++) t.rows[i] = 0;
        if (t.at.group >= 0) {
#pragma unroll
            for (int i = 0; i < NLY; i++) t.rows[i] = source_row(*a, min(t.at.j0 + line + 64 * i, t.at.last - 1));
            t.scale_row = source_row(*a, min(t.at.j0 + 64 * part + (me & 63), t.at.last - 1));
        }
        return t;
    };
    int workgroup = (int)blockIdx.x;
    walked_tile tile = find(workgroup);
    if (tile.at.group < 0) return;
    grouped_tile at = tile.at;

    const int NP = (p.K + 127) / 128;
    const char *X;  // a uniform origin that moves with the slots, and a lane offset for each load
    unsigned xvo[NLX];
    const char *yp[NLY];
    const char *scales;  // of this wavefront's load
    const unsigned lds0 = (unsigned)(uintptr_t)lds, wave_dst = lds0 + (unsigned)wave * 1024u;
    const long scale_step = 4 * (x_scales ? p.lxs : p.lys);
    int next;              // slot to request
    unsigned xwoff, ywoff;  // its places in the rings
    auto request_one = [&]<int N>(std::integral_constant<int, N>) MIW_INLINE {
        if constexpr (N < NLX) lds_dma16_at<N * NT * 16, 0>(X, xvo[N], wave_dst + xwoff);
        else if constexpr (N < NLX + NLY) fp8_load16<XRING + (N - NLX) * NT * 16>(yp[N - NLX], wave_dst + ywoff);
        else fp8_load4(scales, lds0 + (unsigned)part * 256u + (x_scales ? XBYTES + xwoff : XRING + YBYTES + ywoff));
    };
    // (beyond the last slot it is asked for again, which nobody reads)
    auto end_request = [&]() MIW_INLINE {
        xwoff = xwoff + XSLOT == XRING ? 0 : xwoff + XSLOT;
        ywoff = ywoff + YSLOT == YRING ? 0 : ywoff + YSLOT;
        if (next < NP - 1) {
            next++;
            X += 128;
#pragma unroll
            for (int i = 0; i < NLY; i++) yp[i] += 128;
            if ((next & 3) == 0) scales += scale_step;
        }
    };
    // Turns to a tile and requests its first slots.
    auto start = [&](const walked_tile &t) MIW_INLINE {
        const auto a = arguments();
        const int me = thread(), line = me >> 3, chunk = (me & 7) ^ ((me >> 4) & 7);
        at = t.at;
        next = 0;
        xwoff = ywoff = 0;
        X = a->X + (long)at.group * a->sx + (long)at.i0 * a->ldx;
#pragma unroll
        for (int i = 0; i < NLX; i++) xvo[i] = (unsigned)(min(line + 64 * i, a->I - 1 - at.i0) * (int)a->ldx + chunk * 16);
#pragma unroll
        for (int i = 0; i < NLY; i++) yp[i] = a->Y + (long)t.rows[i] * a->ldy + chunk * 16;
        scales = x_scales ? (const char *)a->xs + (long)at.group * a->sxs + 4l * min(at.i0 + 64 * part + (me & 63), a->I - 1) : (const char *)a->ys + 4l * t.scale_row;
#pragma unroll
        for (int s = 0; s < NS - 1; s++) {
            [&]<int... N>(std::integer_sequence<int, N...>) { (request_one(std::integral_constant<int, N>{}), ...); }(std::make_integer_sequence<int, LSLOT>{});
            end_request();
        }
    };

    frag_reader<BI, true> xr;
    frag_reader<BJ, true> yr;
    xr.init(wi * WTI, lane);
    yr.init(wj * WTJ, lane);
    f32x4 acc[TI][TJ];

    // Neighbouring lanes hold neighbouring rows: they exchange the results of two MFMA tiles, so that a row's 32 go out together
    // from eight lanes, first the even rows and then the odd ones.  True: by TI * TJ instructions of each wavefront.
    auto store_tile = [&](const grouped_tile &t) MIW_INLINE {
        const auto args = arguments();
        const int me = thread(), q = (me & 63) >> 4, r = me & 15;
        DT *D = (DT *)args->D;
        const bool odd = r & 1;
        const bool whole = args->d_vector && !args->gated && t.i0 + BI <= args->I && t.j0 + BJ <= t.last;
#pragma unroll
        for (int b = 0; b < TJ; b++) {
            const int j = t.j0 + wj * WTJ + 16 * b + (r & ~1);
            DT *row = D + (long)j * args->ldd;
#pragma unroll
            for (int a = 0; a < TI; a += 2) {
                float4_t v0 = acc[a][b], v1 = acc[a + 1][b];
                pair_exchange(odd, v0, v1);
                const int i = t.i0 + wi * WTI + 16 * (a + odd) + 4 * q;
                __builtin_amdgcn_sched_barrier(0);  // (two tiles' registers at a time)
                if (whole) {
                    *(vec<DT, 4> *)(row + i) = __builtin_convertvector(v0, vec<DT, 4>);
                    *(vec<DT, 4> *)(row + args->ldd + i) = __builtin_convertvector(v1, vec<DT, 4>);
                } else {
                    if (j < t.last) store_results<DT>(*args, row, i, v0);
                    if (j + 1 < t.last) store_results<DT>(*args, row + args->ldd, i, v1);
                }
            }
        }
        return whole;
    };

    start(tile);
    workgroup += (int)gridDim.x;
    tile = find(workgroup);
    wait_loads_and_barrier<0>();
    for (;;) {
    float zero = 0.f;
    asm volatile("" : "+s"(zero));  // (otherwise a zero vector is kept in registers through the tiles)
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++) acc[a][b] = f32x4{zero, zero, zero, zero};
    {
        u32x4 fx[TP][2], fy[TJ][2];
        unsigned sx[TP], sy[TJ];  // the slot's scale in the low byte
        unsigned xroff = 0, yroff = 0, shift = 0;  // the slot that is read
        // Memory cluster H of PARTS: its fragments, with the requests at even distances between the reads.
        auto memory_cluster = [&]<int H, bool REQUEST>(std::integral_constant<int, H>, std::bool_constant<REQUEST>) MIW_INLINE {
            constexpr bool FIRST = H == 0, LAST = H == PARTS - 1;
            constexpr int READS = 2 * (TP + (FIRST ? TJ : 0)), COUNT = REQUEST && FIRST ? LSLOT : 0;
            MIW_LDS const char *xs = lds + xroff, *ys = lds + XRING + yroff;
#pragma unroll
            for (int a = 0; a < TP; a++) sx[a] = *(MIW_LDS const unsigned *)(xs + XBYTES + (wi * WTI + 16 * (H * TP + a) + r) * 4);
            if constexpr (FIRST)
#pragma unroll
                for (int b = 0; b < TJ; b++) sy[b] = *(MIW_LDS const unsigned *)(ys + YBYTES + (wj * WTJ + 16 * b + r) * 4);
            auto unit = [&]<int U>(std::integral_constant<int, U>) MIW_INLINE {
                [&]<int... N>(std::integer_sequence<int, N...>) {
                    (([&] {
                         if constexpr (N * READS / (COUNT ? COUNT : 1) == U) {
                             request_one(std::integral_constant<int, N>{});
                             __builtin_amdgcn_sched_barrier(0);
                         }
                     }()),
                     ...);
                }(std::make_integer_sequence<int, COUNT>{});
                constexpr int S = U % 2, V = U / 2;
                if constexpr (V < TP) fx[V][S] = __builtin_bit_cast(u32x4, xr.template read<H * TP + V, S>(xs));
                else fy[V - TP][S] = __builtin_bit_cast(u32x4, yr.template read<V - TP, S>(ys));
                __builtin_amdgcn_sched_barrier(0);
            };
            [&]<int... U>(std::integer_sequence<int, U...>) { (unit(std::integral_constant<int, U>{}), ...); }(std::make_integer_sequence<int, READS>{});
            if constexpr (COUNT > 0) end_request();
#pragma unroll
            for (int a = 0; a < TP; a++) sx[a] >>= shift;
            if constexpr (FIRST)
#pragma unroll
                for (int b = 0; b < TJ; b++) sy[b] >>= shift;
            if constexpr (LAST) {
                xroff = xroff + XSLOT == XRING ? 0 : xroff + XSLOT;
                yroff = yroff + YSLOT == YRING ? 0 : yroff + YSLOT;
                shift = (shift + 8) & 31;
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto multiply = [&]<int H>(std::integral_constant<int, H>) MIW_INLINE {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!WIDE) {
#pragma unroll
                for (int m = 0; m < TP * TJ; m++) {
                    const int a = m / TJ, b = serpentine_column(m, TJ);
                    acc[H * TP + a][b] = mac_fp8<FORMAT>(fx[a][0], fx[a][1], fy[b][0], fy[b][1], acc[H * TP + a][b], sx[a], sy[b]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // 32 of the slot's 128 at a time
                [&]<int... T>(std::integer_sequence<int, T...>) {
                    (([&] {
                         constexpr int S = T / 2, E = T % 2 * 2;
                         u32x4 wx[TP], wy[TJ];
#pragma unroll
                         for (int a = 0; a < TP; a++) wx[a] = widened<FORMAT_E4M3>(fx[a][S][E], fx[a][S][E + 1], sx[a]);
#pragma unroll
                         for (int b = 0; b < TJ; b++) wy[b] = widened<FORMAT>(fy[b][S][E], fy[b][S][E + 1], sy[b]);
                         __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                         for (int m = 0; m < TP * TJ; m++) {
                             const int a = m / TJ, b = serpentine_column(m, TJ);
                             acc[H * TP + a][b] = mfma_bf16::mac(wx[a], wy[b], acc[H * TP + a][b]);
                         }
                         __builtin_amdgcn_sched_barrier(0);
                     }()),
                     ...);
                }(std::make_integer_sequence<int, 4>{});
            }
        };
        constexpr std::integral_constant<int, 0> first{};
        constexpr std::integral_constant<int, PARTS - 1> second{};
        // One slot.  At the end of its last memory cluster the next slot's loads have landed, what is younger stays in flight, and
        // the barriers that follow publish them.
        auto one_slot = [&]<bool REQUEST>(std::bool_constant<REQUEST> request) MIW_INLINE {
            memory_cluster(first, request);
            if constexpr (HALVES) {
                wait_loads_and_barrier<63>();  // (the fragments alone)
                multiply(first);
                __builtin_amdgcn_s_barrier();
                memory_cluster(second, request);
                wait_loads_and_barrier<0>();
                multiply(second);
            } else {
                wait_loads_and_barrier<REQUEST ? (NS - 2) * LSLOT : 0>();
                multiply(first);
            }
            __builtin_amdgcn_s_barrier();
        };
        if (late_group) __builtin_amdgcn_s_barrier();
        int s = 0;
        for (; s < NP - (NS - 1); s++) one_slot(std::true_type{});
        for (; s < NP; s++) one_slot(std::false_type{});
        if (!late_group) __builtin_amdgcn_s_barrier();
    }

    const grouped_tile done = at;
    const bool more = tile.at.group >= 0;
    if (more) {
        start(tile);
        workgroup += (int)gridDim.x;
        tile = find(workgroup);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool whole = store_tile(done);
    __builtin_amdgcn_sched_barrier(0);
    if (!more) break;
    // (the stores of a whole tile, younger than the requests, may stay in flight)
    if (whole) wait_loads_and_barrier<TI * TJ>();
    else wait_loads_and_barrier<0>();
    }
}

}  // namespace miw
