// What the loss does with the sums of its four products, in place of storing them.
//
// acc[a][b]: results i .. i + 3 (i = i0 + 16 a + 4 (lane / 16)) of row j0 + 16 b + lane % 16.
#pragma once
#include "grouped_common.hpp"
#include "loss.hpp"

#include <type_traits>
#include <utility>

namespace miw {

constexpr float LOG2E = 1.4426950408889634f;
// exp(x): the argument is scaled in one rounding, |x| 2^-24 of the result, and what lies below 2^-126 is 0.
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// Among the four lanes that hold a row's results.
__device__ inline float across_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float across_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

struct loss_end {
    using params = loss_params;
    // Few rows: vectors a multiple of 4 KiB apart would have all workgroups read the same of HBM's channels at a time; each begins at a chunk of its own (16 rows,
    // 32768 x 4096: 56.6 us, all from the first chunk on 64.7; 1 row, 50000 x 2048: 44 and 53; 2 KiB apart, 65536 x 1024, 37 and 36).
    static constexpr bool turns = true;
    template <class PARAMS>
    static __device__ inline int first_chunk(const PARAMS &p, int workgroup, int chunks)
    {
        return p.ldx % 4096 == 0 ? 9 * (workgroup % chunks) % chunks : 0;
    }
    template <class PARAMS>
    static __device__ inline int sum_length(const PARAMS &p, int)
    {
        return p.K;
    }
    template <class PARAMS>
    static __device__ inline long y_offset(const PARAMS &, int)
    {
        return 0;
    }
};

// Which of the columns from i on a target is.  Targets are any Int32: those outside the vocabulary lie behind all columns (of at most 2^26 and a tile).
constexpr unsigned target_column(int target, int i) { return (unsigned)target - (unsigned)i; }
static_assert(target_column(70, 64) == 6 && target_column(63, 64) > 1u << 30 && target_column(-2147483647 - 1, (1 << 26) + 256) > 1u << 30 && target_column(-1, 0) > 1u << 30 &&
              target_column(2147483647, (1 << 26) + 256) > 1u << 30);

// Scores: of a wavefront's columns, the largest and the sum of the exponentials of the differences to it; and of the target, where it is among them, its score and that sum
// without it.  Nothing else of the scores is kept.  (The loss is log(1 + the others' exponentials over the target's); in a sum that has the target's too, 1 where its score is the
// largest, what is far below 1 is lost.)
struct loss_score_end : loss_end {
    template <class DT, class PARAMS, int TI, int TJ>
    static __device__ __forceinline__ void finish(const PARAMS &p, const grouped_tile &t, f32x4 (&acc)[TI][TJ], int i0, int j0, int lane)
    {
        const int q = lane >> 4, r = lane & 15, i = i0 + 4 * q;
        float *stats = p.stats + 2 * (long)(i0 / (16 * TI)) * p.stat_rows;
#pragma unroll
        for (int b = 0; b < TJ; b++) {
            const int j = j0 + 16 * b + r;
            const bool here = j < t.last;
            const unsigned goal = here ? target_column(p.goal[j], i) : ~0u;
            float most = -__builtin_inff();
#pragma unroll
            for (int a = 0; a < TI; a++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = i + 16 * a + e < p.I ? acc[a][b][e] : -__builtin_inff();
                    acc[a][b][e] = v;
                    most = fmaxf(most, v);
                }
            most = across_max(most);
            // (a slice of -inf alone has no exponentials)
            const float from = most == -__builtin_inff() ? 0.f : most;
            float sum = 0.f;
#pragma unroll
            for (int a = 0; a < TI; a++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum += exp_of(acc[a][b][e] - from);
            sum = across_sum(sum);
            if (here && q == 0) *(f32x2 *)(stats + 2 * (long)j) = f32x2{most, sum};
            const bool mine = goal < 16 * TI && (goal & 15) < 4;
            if (!__any(mine)) continue;  // (few wavefronts have a target of their rows among their columns)
            float score = 0.f, others = 0.f;
#pragma unroll
            for (int a = 0; a < TI; a++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool target = goal == 16u * a + e;
                    score = target ? acc[a][b][e] : score;
                    others += target ? 0.f : exp_of(acc[a][b][e] - from);
                }
            others = across_sum(others);
            if (mine) *(f32x2 *)(p.goals + 2 * (long)j) = f32x2{score, others};
        }
    }
};

// Probabilities: share * (exp(score - lse) - [the target]), rounded to the operands' type, for the two products that follow.
struct loss_probability_end : loss_end {
    template <class DT, class PARAMS>
    static __device__ inline void store(const PARAMS &p, int j, int i, f32x4 v)
    {
        const float lse = p.lse[j], share = p.share[j];
        const long goal = p.goal[j] - p.first - i;
        DT *row = (DT *)p.D + (long)j * p.ldd + i;
        f32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = share * (exp_of(v[e] - lse) - (goal == e ? 1.f : 0.f));
        if (i + 3 < p.I) {
            *(vec<DT, 4> *)row = __builtin_convertvector(w, vec<DT, 4>);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + e < p.I) row[e] = (DT)w[e];
        }
    }
    template <class DT, class PARAMS, int TI, int TJ>
    static __device__ __forceinline__ void finish(const PARAMS &p, const grouped_tile &t, f32x4 (&acc)[TI][TJ], int i0, int j0, int lane)
    {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (TI == 1) {
#pragma unroll
            for (int b = 0; b < TJ; b++)
                if (j0 + 16 * b + r < t.last) store<DT>(p, j0 + 16 * b + r, i0 + 4 * q, acc[0][b]);
        } else {
            // (neighbouring lanes exchange results as in grouped_tile.hpp, so that 64 bytes of a row go out together)
            const bool odd = r & 1;
#pragma unroll
            for (int b = 0; b < TJ; b++) {
                const int j = j0 + 16 * b + (r & ~1);
#pragma unroll
                for (int a = 0; a < TI; a += 2) {
                    float4_t v0 = acc[a][b], v1 = acc[a + 1][b];
                    pair_exchange(odd, v0, v1);
                    const int i = i0 + 16 * (a + odd) + 4 * q;
                    if (j < t.last) store<DT>(p, j, i, v0);
                    if (j + 1 < t.last) store<DT>(p, j + 1, i, v1);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
};

// Calls f with 0, 1, ... N - 1 as constants (a loop of this many stores is not unrolled by itself, and the results would go to memory to be indexed).
template <int N, class F>
__device__ __forceinline__ void each_of(F f)
{
    [&]<int... I>(std::integer_sequence<int, I...>) MIW_INLINE { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// Sums in Float32, or rounded, to rows below `end`, times `by`.
template <class DT, class PARAMS, int TI, int TJ>
__device__ __forceinline__ void store_scaled(const PARAMS &p, int end, float by, f32x4 (&acc)[TI][TJ], int i0, int j0, int lane)
{
    const int q = lane >> 4, r = lane & 15;
    const bool odd = r & 1;
    each_of<TJ>([&](auto b) MIW_INLINE {
        const int j = j0 + 16 * b + (r & ~1);
        DT *row = (DT *)p.D + (long)j * p.ldd;
        each_of<TI / 2>([&](auto pair) MIW_INLINE {
            constexpr int a = 2 * pair;
            float4_t v0 = by * acc[a][b], v1 = by * acc[a + 1][b];
            pair_exchange(odd, v0, v1);
            const int i = i0 + 16 * (a + odd) + 4 * q;
            if (j < end) store_results<DT>(p, row, i, v0);
            if (j + 1 < end) store_results<DT>(p, row + p.ldd, i, v1);
            __builtin_amdgcn_sched_barrier(0);
        });
    });
}

// Gradient to the rows: partial sums over slices of the vocabulary.  Groups are the same rows of Y, from their slice's column on.
struct loss_rows_end : loss_end {
    template <class PARAMS>
    static __device__ inline int sum_length(const PARAMS &p, int group)
    {
        return min(p.slice, p.K - group * p.slice);
    }
    template <class PARAMS>
    static __device__ inline long y_offset(const PARAMS &p, int group)
    {
        return 2l * group * p.slice;
    }
    template <class DT, class PARAMS, int TI, int TJ>
    static __device__ __forceinline__ void finish(const PARAMS &p, const grouped_tile &t, f32x4 (&acc)[TI][TJ], int i0, int j0, int lane)
    {
        store_scaled<DT>(p, t.last, 1.f, acc, i0, j0, lane);
    }
};

// Gradient to the vocabulary's vectors.  (Nothing is added to them where no token counts.)
struct loss_vectors_end : loss_end {
    template <class DT, class PARAMS, int TI, int TJ>
    static __device__ __forceinline__ void finish(const PARAMS &p, const grouped_tile &t, f32x4 (&acc)[TI][TJ], int i0, int j0, int lane)
    {
        if (p.accumulate && t.first >= t.last) return;
        store_scaled<DT>(p, p.store_j, p.unscale ? *p.unscale : 1.f, acc, i0, j0, lane);
    }
};

}  // namespace miw
