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
//     entries travel to LDS NY - 1 slots ahead of the slot that they are for.  A slot is 64 along k, or 32, where half the LDS then
//     suffices for a tile of 256 x 128 and a CU holds two workgroups: while one waits for its first slot the other multiplies.  Stores
//     and products add up all the same: 8198 rows, 16 groups, 2048 x 4096 (bf16, Float32 results): without stores 136 to 147 us, stores
//     alone 111 to 118, both 238 to 258 on 256 x 256 with slots of 64; 221 to 243 on 256 x 128 with slots of 32.  Added to D: 301, for the 537 MB
//     more that are read.
//
// Sums are Float32 in the accumulators and are rounded once, when they are stored (gated ones after the activation).  Measured, back to back on several cards: 16384 rows, 8
// groups of uneven size, 4096 x 4096 (bf16): 427 to 460 us, 1.20 to 1.29 PFLOP/s, matrix cores busy 65 to 67 % of the cycles at some 1.75 GHz, which is what the power
// cap leaves a dense product too (even groups: 400 us; gated 410).  The gradient to 8198 rows, 16 groups, 2048 x 4096 (i contiguous): 157 to 172 us, 0.80 to 0.87 PFLOP/s for 40 tiles
// of rows where 32 would do.  4 bits, 4096 x 4096 x 8192: 64 to 69 us, 4.0 to 4.3 PFLOP/s, gated 73; cores 41 to 43 %, the memory cluster is the longer one (without loads 55 us, without
// MFMAs 43).  4 bits, 16384 rows, 8 even groups, 4096 x 4096: 156 us, 3.5 PFLOP/s, gated 174; 2048 rows, 16 groups, 2048 x 2048: 15.6, gated 17.9 (f16 42 and 45).
//
// Where the sum ends inside a slot, lanes fetch the last valid chunk (row) again and its values are zeroed in both operands'
// fragments, in a copy of the loop body that only the last slot runs.
#pragma once
#include "grouped_common.hpp"

#include <type_traits>

namespace miw {

enum grouped_form { ROWS_X_K = 0, ROWS_X_I = 1, RAGGED_SUM = 2, RAGGED_SUM_32 = 3 };  // (the last: in slots of 32 along k)
constexpr bool grouped_sums(int form) { return form >= RAGGED_SUM; }

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

// A slot of one operand: its rows' 128 bytes, then their scales.
constexpr int grouped_slot_bytes(int rows, bool scaled, int form) { return rows * ((form == RAGGED_SUM_32 ? 64 : 128) + (scaled ? 8 : 0)); }
constexpr int grouped_lds_bytes(int bi, int bj, int nx, int ny, bool scaled, int form)
{
    return nx * grouped_slot_bytes(bi, scaled, form) + ny * grouped_slot_bytes(bj, scaled, form) + (grouped_sums(form) ? 2 * ny * 256 : 0);
}

// X's scales of a tile are fetched 16 bytes, two rows, a lane, 128 rows a wavefront's load: the first row, of the matrix' I, of such a
// pair.  Rows behind the matrix' last pair repeat it: panels may hold other matrices' rows there, or end.
constexpr int scale_pair(int i0, int part, int lane, int I)
{
    const int row = i0 + part * 128 + 2 * lane, last = I + (I & 1) - 2;
    return row < last ? row : last;
}

// Workgroups that a CU holds together.
constexpr int grouped_workgroups(int bi, int bj, int nx, int ny, bool scaled, int form)
{
    return grouped_lds_bytes(bi, bj, nx, ny, scaled, form) <= 80 * 1024 ? 2 : 1;
}
// Do workgroups walk several tiles?
constexpr bool grouped_walks(bool scaled, int form) { return !scaled && !grouped_sums(form); }

// Tile of a ragged sum: groups one after the other, eight tiles along j together.
template <class PARAMS>
__device__ inline grouped_tile find_sum_tile(const PARAMS &p, int bi, int bj, int workgroup)
{
    const int tiles_i = (p.I + bi - 1) / bi, tiles_j = (p.J + bj - 1) / bj;
    int id = tile_of_workgroup(p.groups * tiles_i * tiles_j, workgroup);
    if (id < 0) return {-1, 0, 0, 0, 0};
    const int group = id / (tiles_i * tiles_j);
    id -= group * tiles_i * tiles_j;
    const group_rows rows = rows_of_group(p, group);
    const int band = id / (GROUP_J_TILES * tiles_i), in = id - band * GROUP_J_TILES * tiles_i;
    const int height = min(GROUP_J_TILES, tiles_j - band * GROUP_J_TILES);
    const int i = in / height, j = band * GROUP_J_TILES + in - i * height;
    return {group, __builtin_amdgcn_readfirstlane(rows.first), __builtin_amdgcn_readfirstlane(rows.last), j * bj, i * bi};
}

// Fragments of a slot of 32 along k whose rows have i contiguous: as frag_reader, with 32 rows to each 64 along i.
struct short_reader {
    int base[4];
    __device__ inline void init(int wave_row0, int lane)
    {
        const int j = lane & 15, q = lane >> 4, jq = j >> 2, jr = j & 3;
        const int g = ((jq >> 1) & 1) | ((q & 1) << 1);  // i_major_swizzle of this lane's k
        const int w16 = wave_row0 / 16;
#pragma unroll
        for (int m = 0; m < 4; m++) base[m] = (w16 / 4) * 4096 + (8 * q + jq) * 128 + jr * 8 + ((((w16 & 3) + m) & 3) ^ g) * 32;
    }
    template <int T, int H>
    __device__ inline half8_t read(MIW_LDS const char *slot) const
    {
        static_assert(H == 0, "one step");
        const int off = base[T & 3] + (T >> 2) * 4096;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((MIW_LDS fp16x4_t *)(slot + off)));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((MIW_LDS fp16x4_t *)(slot + off + 512)));
        return __builtin_bit_cast(half8_t, u32x4{lo[0], lo[1], hi[0], hi[1]});
    }
};

// Zeroes the values of a lane's 16-byte fragment of 16-bit elements from `keep` on.
__device__ inline void keep_first(u32x4 &f, int keep)
{
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] &= keep >= 2 * e + 2 ? 0xffffffffu : keep == 2 * e + 1 ? 0xffffu : 0u;
}

// NX, NY: slots of X and of Y in LDS.
//   Three or more, as many of both: a cluster is a whole slot.  The slot NX - 1 further on is requested in a slot's memory
//     cluster, into the place of the one before, and at its end the NX - 2 youngest stay in flight.
//   Two of Y (tiles of 256 x 256): a cluster is one MFMA step, half a slot.  Y's next slot is requested in the first memory cluster and
//     has to have landed at the end of the second; X's goes with it, or, with three slots of X, the one after that in the
//     second cluster, so that X, the weights, which come from HBM where the rows mostly come from caches, has twice the time.
template <class OP, int BI, int BJ, int WI, int WJ, int NX, int NY, int FORM, class DT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2 * grouped_workgroups(BI, BJ, NX, NY, OP::scaled, FORM))))
void k_grouped_tile(grouped_params p)
{
    constexpr int NT = 512;
    static_assert(WI * WJ == 8, "two wavefronts per SIMD");
    constexpr bool XK = FORM == ROWS_X_K, SUM = grouped_sums(FORM), YK = !SUM, SCALED = OP::scaled;
    constexpr bool SHORT = FORM == RAGGED_SUM_32;
    constexpr int SLOT_K = SHORT ? 32 : OP::slot_k, LOAD_I = SHORT ? 128 : 64;  // LOAD_I: rows of a tile that one load takes
    static_assert(!SCALED || XK, "4-bit operands have k contiguous");
    constexpr int WTI = BI / WI, WTJ = BJ / WJ, TI = WTI / 16, TJ = WTJ / 16;
    constexpr int XBYTES = BI * 128, YBYTES = BJ * 128, XSLOT = grouped_slot_bytes(BI, SCALED, FORM), YSLOT = grouped_slot_bytes(BJ, SCALED, FORM);
    constexpr int XRING = NX * XSLOT, YRING = NY * YSLOT, INDEX = XRING + YRING;  // X's ring, Y's, that of the gathered rows
    static_assert(grouped_lds_bytes(BI, BJ, NX, NY, SCALED, FORM) <= 160 * 1024, "rings do not fit in LDS");
    constexpr bool HALVES = NY == 2, SPLIT = HALVES && NX == 3;
    static_assert((SPLIT ? !SCALED && !SUM : NX == NY) && !(HALVES && SHORT), "slots");
    constexpr int XSW = BI / 128, YSW = BJ / 32;  // wavefronts' loads that a slot's scales take
    constexpr bool SHARED_SCALES = XSW + YSW <= 8;
    constexpr int NLX = BI / LOAD_I, NLY = BJ / LOAD_I, EXTRA = SCALED ? (SHARED_SCALES ? 1 : 2) : SUM ? 1 : 0;
    constexpr int LPAIR = NLX + NLY + EXTRA;  // loads a thread and slot
    constexpr int NFRAG = (HALVES || SHORT ? 1 : 2) * (TI + TJ);  // of a cluster
    static_assert(BI % 128 == 0 && BJ % LOAD_I == 0 && WTI % 32 == 0 && WTJ % 16 == 0, "tile");

    extern __shared__ __attribute__((aligned(128))) char smem[];
    MIW_LDS char *lds = (MIW_LDS char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = wave % WI, wj = wave / WI, q = lane >> 4, r = lane & 15;
    const bool late_group = wave >= 4;
    // This thread's row (k) of a load; with slots of 32 a load takes two times 64 along i.
    auto line_of = [](int t) MIW_INLINE { return SHORT ? (t >> 3) & 31 : t >> 3; };
    const int line = line_of(tid);
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
    // The 16 bytes of a load's row that go to place t % 8 of it, where k is contiguous and where i is.
    auto k_chunk_of = [](int t) MIW_INLINE { return (t & 7) ^ ((t >> 4) & 7); };
    auto i_chunk_of = [](int t) MIW_INLINE { return (t & 7) ^ (2 * i_major_swizzle(t >> 3)); };
    // Scales: X's are fetched 16 bytes (two rows) a lane, Y's, whose rows may lie anywhere, four bytes a lane.  Where the
    // wavefronts suffice the first ones fetch X's and the others Y's, one load each; otherwise every one fetches a part of
    // both.  All count the same: those that are left over repeat another's.
    static_assert(!SCALED || (XSW <= 8 && YSW <= 8), "loads of scales");
    const bool x_scales = SHARED_SCALES && wave < XSW;
    const int x_part = wave % XSW, y_part = SHARED_SCALES ? (wave + YSW - XSW % YSW) % YSW : wave % YSW;

    // A workgroup walks tiles.  Which one is next, and the rows that its first requests need, is looked up while the first slots of
    // the one before are on the way, and these are requested ahead of the stores of the one before that: what is left
    // of a tile's start is the wait for its first slot.
    constexpr int ROWS = YK ? NLY : NY - 1;
    struct walked_tile {
        grouped_tile at;
        int rows[ROWS];  // ragged rows: of this thread's lines of Y; ragged sum: of its line of the first slots of X
        int scale_row;
    };
    auto find = [&](int workgroup) MIW_INLINE {
        walked_tile t;
        const auto a = arguments();
        const int me = thread(), line = line_of(me);
        grouped_tile at;
        if constexpr (SUM) at = find_sum_tile(*a, BI, BJ, workgroup);
        else at = find_tile(*a, BI, BJ, workgroup);
        t.at = {__builtin_amdgcn_readfirstlane(at.group), __builtin_amdgcn_readfirstlane(at.first), __builtin_amdgcn_readfirstlane(at.last),
                __builtin_amdgcn_readfirstlane(at.j0), __builtin_amdgcn_readfirstlane(at.i0)};
        t.scale_row = 0;
#pragma unroll
        for (int i = 0; i < ROWS; i++) t.rows[i] = 0;
        if (t.at.group >= 0 && t.at.first < t.at.last) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) t.rows[i] = source_row(*a, min((YK ? t.at.j0 : t.at.first) + line + (SHORT ? 32 : 64) * i, t.at.last - 1));
            if constexpr (SCALED) t.scale_row = source_row(*a, min(t.at.j0 + 32 * y_part + ((me & 63) >> 1), t.at.last - 1));
        }
        return t;
    };
    int workgroup = (int)blockIdx.x;
    walked_tile tile = find(workgroup);
    if (tile.at.group < 0) return;
    grouped_tile at = tile.at;

    int length, NP, last_values, last_chunks;  // of the sum, in values and slots; values and 16-byte chunks that its last slot has
    const char *X;           // a uniform origin that moves with the slots, and a lane offset for each load
    unsigned xvo[NLX];
    const char *yp[NLY];
    const char *xsp = nullptr, *ysp = nullptr;
    const long x_step = XK ? 128 : 64 * p.ldx;
    const unsigned wave_dst = (unsigned)(uintptr_t)lds + (unsigned)wave * 1024u;
    const unsigned lds0 = (unsigned)(uintptr_t)lds;
    int xnext, ynext;       // slots to request (one number, ynext, without SPLIT)
    unsigned xwoff, ywoff;  // their places in the rings
    long xrow = 0, yrow = 0;     // (ragged sum: the lane's rows of the slot, in bytes from the operands)
    auto x_last_begins = [&]() MIW_INLINE {
        if constexpr (SUM) return;
        const int me = thread(), line = line_of(me), k_chunk = k_chunk_of(me);
        const unsigned back = XK ? 16u * (unsigned)max(0, k_chunk - (last_chunks - 1)) : (unsigned)(max(0, line - (last_values - 1)) * (int)p.ldx);
#pragma unroll
        for (int i = 0; i < NLX; i++) xvo[i] -= back;
    };
    auto y_last_begins = [&]() MIW_INLINE {
        if constexpr (SUM) return;
        const int k_chunk = k_chunk_of(thread());
        const int back = 16 * max(0, k_chunk - (last_chunks - 1));
#pragma unroll
        for (int i = 0; i < NLY; i++) yp[i] -= back;
    };
    // Ragged sum: where this lane's row of slot `ynext` lies in both operands.
    auto find_rows = [&](int gathered) MIW_INLINE {
        const int position = max(min(at.first + ynext * SLOT_K + line, at.last - 1), 0);
        yrow = (long)position * p.ldy;
        xrow = (long)gathered * p.ldx;
    };
    auto index_entry = [&](int slot) MIW_INLINE { return (unsigned)(slot % (2 * NY)) * 256u; };
    // Load N of a slot: X's, Y's, then what goes with them.
    auto request_one = [&]<int N>(std::integral_constant<int, N>) MIW_INLINE {
        if constexpr (N < NLX) {
            const unsigned dst = wave_dst + xwoff;
            if constexpr (SUM) lds_load16<N * NT * 16>(X + xvo[N] + xrow, dst);
            else lds_dma16_at<N * NT * 16, 0>(X, xvo[N], dst);
        } else if constexpr (N < NLX + NLY) {
            constexpr int M = N - NLX;
            const unsigned dst = wave_dst + ywoff;
            if constexpr (SUM) lds_load16<XRING + M * NT * 16>(yp[M] + yrow, dst);
            else lds_load16<XRING + M * NT * 16>(yp[M], dst);
        } else if constexpr (SCALED) {
            const bool x_turn = SHARED_SCALES ? x_scales : N == NLX + NLY;
            if (x_turn) lds_load16<XBYTES>(xsp, lds0 + xwoff + (unsigned)x_part * 1024u);
            else lds_load4<XRING + YBYTES>(ysp, lds0 + ywoff + (unsigned)y_part * 256u);
        } else if constexpr (SUM) {
            // the rows of the slot NY - 1 further on, by every wavefront to the same place
            const int position = max(min(at.first + min(ynext + NY - 1, NP - 1) * SLOT_K + lane, at.last - 1), 0);
            lds_load4<INDEX>((const char *)(p.gather ? p.gather + position : p.offsets), lds0 + index_entry(ynext + NY - 1));
        }
    };
    // FROM .. TO - 1, in one go.
    auto request_all = [&]<int FROM, int TO>(std::integral_constant<int, FROM>, std::integral_constant<int, TO>) MIW_INLINE {
        [&]<int... I>(std::integer_sequence<int, I...>) { (request_one(std::integral_constant<int, FROM + I>{}), ...); }(std::make_integer_sequence<int, TO - FROM>{});
    };
    auto x_end_request = [&]() MIW_INLINE {
        xwoff = xwoff + XSLOT == XRING ? 0 : xwoff + XSLOT;
        if constexpr (!SUM)
            if (xnext < NP - 1) {
                xnext++;
                X += x_step;
                if constexpr (SCALED) xsp += 8 * p.lxs;
                if (xnext == NP - 1) x_last_begins();
            }
    };
    auto y_end_request = [&]() MIW_INLINE {
        ywoff = ywoff + YSLOT == YRING ? 0 : ywoff + YSLOT;
        if constexpr (SUM) {
            ynext++;
        } else if (ynext < NP - 1) {
            ynext++;
#pragma unroll
            for (int i = 0; i < NLY; i++) yp[i] += 128;
            if constexpr (SCALED) ysp += 8 * p.lys;
            if (ynext == NP - 1) y_last_begins();
        }
    };

    // Turns to a tile and requests its first slots (a sum that is shorter than the rings asks for its last slot again, which
    // nobody reads, and one of no rows for the row before).  The rings are empty then, and start at their beginnings.
    auto start = [&](const walked_tile &t) MIW_INLINE {
        const auto a = arguments();
        const int me = thread(), line = line_of(me), k_chunk = k_chunk_of(me), i_offset = 8 * i_chunk_of(me) + (SHORT ? 64 * (me >> 8) : 0);
        at = t.at;
        length = SUM ? at.last - at.first : a->K;
        NP = (length + SLOT_K - 1) / SLOT_K;
        last_values = length - (NP - 1) * SLOT_K;
        last_chunks = SCALED ? (last_values + 31) / 32 : (last_values + 7) / 8;
        xnext = ynext = 0;
        xwoff = ywoff = 0;
        X = a->X + (SUM ? 0 : (long)at.group * a->sx);
        if constexpr (XK) {
            X += (long)at.i0 * a->ldx;
#pragma unroll
            for (int i = 0; i < NLX; i++) xvo[i] = (unsigned)(min(line + 64 * i, a->I - 1 - at.i0) * (int)a->ldx + k_chunk * 16);
        } else {
            X += 2l * at.i0;
#pragma unroll
            for (int i = 0; i < NLX; i++) xvo[i] = (SUM ? 0u : (unsigned)(line * (int)a->ldx)) + 2u * (unsigned)min(LOAD_I * i + i_offset, a->I - 8 - at.i0);
        }
#pragma unroll
        for (int i = 0; i < NLY; i++) {
            if constexpr (YK) yp[i] = a->Y + (long)t.rows[i] * a->ldy + k_chunk * 16;
            else yp[i] = a->Y + 2l * (at.j0 + min(LOAD_I * i + i_offset, a->J - 8 - at.j0));
        }
        if constexpr (SCALED) {
            xsp = (const char *)a->xs + (long)at.group * a->sxs + 8l * scale_pair(at.i0, x_part, me & 63, a->I);
            ysp = (const char *)a->ys + 8l * t.scale_row + 4 * (me & 1);
        }
        if (NP == 1) {
            x_last_begins();
            y_last_begins();
        }
        constexpr std::integral_constant<int, 0> first_load{};
        constexpr std::integral_constant<int, NLX> x_loads{};
        constexpr std::integral_constant<int, LPAIR> all_loads{};
#pragma unroll
        for (int s = 0; s < NY - 1; s++) {
            if constexpr (SUM) find_rows(t.rows[s]);
            request_all(first_load, all_loads);
            x_end_request();
            y_end_request();
        }
        if constexpr (SPLIT) {
            request_all(first_load, x_loads);
            x_end_request();
        }
    };

    std::conditional_t<SHORT, short_reader, frag_reader<BI, XK>> xr;
    std::conditional_t<SHORT, short_reader, frag_reader<BJ, YK>> yr;
    xr.init(wi * WTI, lane);
    yr.init(wj * WTJ, lane);
    f32x4 acc[TI][TJ];

    // Neighbouring lanes hold neighbouring rows: they exchange the results of two MFMA tiles, so that a row's 32 go out together
    // (128 bytes of Float32) from eight lanes, first the even rows and then the odd ones.  Whole tiles are stored by TI * TJ
    // instructions of each wavefront; true is returned then.
    auto store_tile = [&](const grouped_tile &t) MIW_INLINE {
        const auto args = arguments();
        const int me = thread(), q = (me & 63) >> 4, r = me & 15;
        if (SUM && args->accumulate && t.first >= t.last) return false;
        DT *D = (DT *)args->D + (SUM ? (long)t.group * args->sd : 0);
        const int end_j = SUM ? args->J : t.last;
        const bool odd = r & 1;
        const bool whole = args->d_vector && !args->gated && !args->accumulate && t.i0 + BI <= args->I && t.j0 + BJ <= end_j;
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
                    if (j < end_j) store_results<DT>(*args, row, i, v0);
                    if (j + 1 < end_j) store_results<DT>(*args, row + args->ldd, i, v1);
                }
            }
        }
        return whole;
    };

    constexpr bool WALKS = grouped_walks(SCALED, FORM);
    start(tile);
    if constexpr (WALKS) {
        workgroup += (int)gridDim.x;
        tile = find(workgroup);
    }
    wait_loads_and_barrier<0>();
    for (;;) {
    float zero = 0.f;
    asm volatile("" : "+s"(zero));  // (otherwise a zero vector is kept in registers through the tiles)
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++) acc[a][b] = f32x4{zero, zero, zero, zero};
    if (NP > 0) {
        constexpr int FSETS = HALVES || SHORT ? 1 : 2;
        u32x4 fx[FSETS][TI], fy[FSETS][TJ];
        unsigned lane_sx[SCALED ? TI : 1], lane_sy[SCALED ? TJ : 1];  // this lane's scales of steps 0 and 1 in the low bytes
        const unsigned own_bytes = (unsigned)(q | (4 + q) << 8 | 0x0c0c0000);
        (void)own_bytes;
        unsigned xroff = 0, yroff = 0;  // the slot that is read, in the rings
        constexpr std::integral_constant<int, 0> step0{};
        constexpr std::integral_constant<int, 1> step1{};
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        // Memory cluster H (of one: 0): its fragments, and its requests at even distances between the reads.  REQUEST_X, REQUEST_Y:
        // whether the sum has the slots that are next.
        auto memory_cluster = [&]<int H, bool REQUEST_X, bool REQUEST_Y>(std::integral_constant<int, H>, std::bool_constant<REQUEST_X>,
                                                                         std::bool_constant<REQUEST_Y>) MIW_INLINE {
            constexpr bool FIRST = H == 0, LAST = !HALVES || H == 1;
            constexpr bool X_HERE = REQUEST_X && (SPLIT ? H == 1 : H == 0), Y_HERE = REQUEST_Y && H == 0;
            constexpr int FROM = X_HERE ? 0 : NLX, TO = Y_HERE ? LPAIR : X_HERE ? NLX : FROM, COUNT = TO - FROM;
            MIW_LDS const char *xs = lds + xroff, *ys = lds + XRING + yroff;
            if constexpr (SUM && Y_HERE) {
                const int row = p.gather ? min(max(*(MIW_LDS const int *)(lds + INDEX + index_entry(ynext) + 4 * line), 0), p.source_rows - 1)
                                         : min(at.first + ynext * SLOT_K + line, at.last - 1);
                find_rows(row);
            }
            u32x2 sx[SCALED ? TI : 1], sy[SCALED ? TJ : 1];  // a row's eight scales of the slot
            if constexpr (SCALED && FIRST) {
#pragma unroll
                for (int a = 0; a < TI; a++) sx[a] = *(MIW_LDS const u32x2 *)(xs + XBYTES + (wi * WTI + 16 * a + r) * 8);
#pragma unroll
                for (int b = 0; b < TJ; b++) sy[b] = *(MIW_LDS const u32x2 *)(ys + YBYTES + (wj * WTJ + 16 * b + r) * 8);
            }
            auto unit = [&]<int U>(std::integral_constant<int, U>) MIW_INLINE {
                [&]<int... N>(std::integer_sequence<int, N...>) {
                    (([&] {
                         if constexpr (N * NFRAG / (COUNT ? COUNT : 1) == U) {
                             request_one(std::integral_constant<int, FROM + N>{});
                             __builtin_amdgcn_sched_barrier(0);
                         }
                     }()),
                     ...);
                }(std::make_integer_sequence<int, COUNT>{});
                constexpr int S = HALVES ? 0 : U / (TI + TJ), T = HALVES ? H : S, V = U % (TI + TJ);
                if constexpr (V < TI) fx[S][V] = __builtin_bit_cast(u32x4, xr.template read<V, T>(xs));
                else fy[S][V - TI] = __builtin_bit_cast(u32x4, yr.template read<V - TI, T>(ys));
                __builtin_amdgcn_sched_barrier(0);
            };
            [&]<int... U>(std::integer_sequence<int, U...>) { (unit(std::integral_constant<int, U>{}), ...); }(std::make_integer_sequence<int, NFRAG>{});
            if constexpr (X_HERE) x_end_request();
            if constexpr (Y_HERE) y_end_request();
            if constexpr (LAST) {
                xroff = xroff + XSLOT == XRING ? 0 : xroff + XSLOT;
                yroff = yroff + YSLOT == YRING ? 0 : yroff + YSLOT;
            }
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
        // One slot.  At the end of its last memory cluster the next slot's loads have landed, what is younger stays in flight, and
        // the barriers that follow publish them.
        auto one_slot = [&]<bool REQUEST_X, bool REQUEST_Y, bool MASK>(std::bool_constant<REQUEST_X> want_x, std::bool_constant<REQUEST_Y> want_y,
                                                                       std::bool_constant<MASK>) MIW_INLINE {
            constexpr int INFLIGHT = SPLIT ? (REQUEST_X ? NLX : 0) : REQUEST_Y ? (NY - 2) * LPAIR : 0;
            memory_cluster(step0, want_x, want_y);
            if constexpr (HALVES) {
                wait_loads_and_barrier<63>();  // (the fragments alone)
                if constexpr (MASK) mask_tail(step0, step0);
                multiply(step0, step0);
                __builtin_amdgcn_s_barrier();
                memory_cluster(step1, want_x, want_y);
                wait_loads_and_barrier<INFLIGHT>();
                if constexpr (MASK) mask_tail(step0, step1);
                multiply(step0, step1);
            } else {
                wait_loads_and_barrier<INFLIGHT>();
                if constexpr (MASK) {
                    mask_tail(step0, step0);
                    if constexpr (!SHORT) mask_tail(step1, step1);
                }
                multiply(step0, step0);
                if constexpr (!SHORT) multiply(step1, step1);
            }
            __builtin_amdgcn_s_barrier();
        };
        if (late_group) __builtin_amdgcn_s_barrier();
        int s = 0;
        for (; s < NP - (NX - 1); s++) one_slot(yes, yes, no);
        if constexpr (SPLIT) {
            if (s < NP - 1) {
                one_slot(no, yes, no);
                s++;
            }
        }
        for (; s < NP - 1; s++) one_slot(no, no, no);
        one_slot(no, no, yes);
        if (!late_group) __builtin_amdgcn_s_barrier();
    }

    const grouped_tile done = at;
    const bool more = WALKS && tile.at.group >= 0;
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
