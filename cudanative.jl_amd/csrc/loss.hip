// Softmax cross entropy over a large vocabulary: the join of the scores' statistics; for the gradient the tokens that count, and the join of the rows' gradients.
// The products are in loss_products.hpp.
//
// All of it is small beside them: the look 3.9 to 5 us for 509 to 4096 tokens, one workgroup's chain of loads and barriers; the join 4.2 to 7 (2048 slices of 16 tokens 5.5; 252 of 8192, 16 MB, 6.4 to 7);
// the rows' gradients 3.8 (356 rows x 720, five slices) to 38 (8192 x 4096, 200 MB, 5.3 TB/s); the copy 12 (4096 x 4096, 64 MB) and 21 (8192 x 4096).
#include "loss_ends.hpp"

#include <type_traits>

namespace miw {

// Which tokens count, in one workgroup: a token whose target is outside the vocabulary has no row in any product of the gradient.  8192 tokens at a time, every
// wavefront 64 neighbours in each of eight turns, so that all loads and nearly all stores are whole lines; the counts of the 128
// runs of 64 are summed up in LDS, so rows keep the tokens' order.
constexpr int LOOK_THREADS = 1024, LOOK_TURNS = 8, LOOK_WAVES = LOOK_THREADS / 64;
__global__ __launch_bounds__(LOOK_THREADS) void k_loss_look(loss_look_params p)
{
    __shared__ int upto[LOOK_TURNS * LOOK_WAVES];
    __shared__ unsigned largest[LOOK_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float scale = 1.f;
    if (p.scaled) {
        // The power of two that brings the largest finite share to 2^14 .. 2^15: shares times probabilities then use Float16's whole range.
        unsigned most = 0;
        for (int t = tid; t < p.tokens; t += LOOK_THREADS) {
            const int target = p.targets[t];
            const unsigned m = __builtin_bit_cast(unsigned, p.shares[t]) & 0x7fffffffu;
            if (target >= 0 && target < p.vocabulary && m < 0x7f800000u) most = max(most, m);
        }
        most = wave_max(most);
        if (lane == 0) largest[wave] = most;
        __syncthreads();
        for (int w = 0; w < LOOK_WAVES; w++) most = max(most, largest[w]);
        const int up = most ? max(-126, min(126, 127 + 14 - (int)(most >> 23))) : 0;
        scale = __builtin_ldexpf(1.f, up);
        if (tid == 0) {
            p.rows.scale[0] = scale;
            p.rows.scale[1] = __builtin_ldexpf(1.f, -up);
        }
    }
    int before = 0;
    for (int t0 = 0; t0 < p.tokens; t0 += LOOK_THREADS * LOOK_TURNS) {
        int target[LOOK_TURNS];
        float lse[LOOK_TURNS], share[LOOK_TURNS];
#pragma unroll
        for (int e = 0; e < LOOK_TURNS; e++) {
            const int t = min(t0 + e * LOOK_THREADS + tid, p.tokens - 1);
            target[e] = p.targets[t];
            lse[e] = p.lse[t];
            share[e] = p.shares[t];
        }
        unsigned long counted[LOOK_TURNS];
#pragma unroll
        for (int e = 0; e < LOOK_TURNS; e++) {
            if (target[e] >= p.vocabulary || t0 + e * LOOK_THREADS + tid >= p.tokens) target[e] = -1;
            counted[e] = __ballot(target[e] >= 0);
        }
        __syncthreads();  // (the sums before have been read)
        if (lane == 0) {
#pragma unroll
            for (int e = 0; e < LOOK_TURNS; e++) upto[e * LOOK_WAVES + wave] = __popcll(counted[e]);
        }
        __syncthreads();
        if (wave == 0) {
            const int low = upto[2 * lane], high = upto[2 * lane + 1], sum = wave_scan(low + high);
            upto[2 * lane] = sum - high;
            upto[2 * lane + 1] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < LOOK_TURNS; e++) {
            const int t = t0 + e * LOOK_THREADS + tid, run = e * LOOK_WAVES + wave;
            if (t >= p.tokens) continue;
            const int row = before + upto[run] - __popcll(counted[e]) + __popcll(counted[e] & ((1ul << lane) - 1));
            p.rows.place[t] = target[e] >= 0 ? row : -1;
            if (target[e] < 0) continue;
            p.rows.list[row] = t;
            p.rows.goal[row] = target[e];
            p.rows.lse[row] = lse[e];
            p.rows.share[row] = share[e] * scale;
        }
        before += upto[LOOK_TURNS * LOOK_WAVES - 1];
    }
    if (tid == 0) {
        p.rows.offsets[0] = 0;
        p.rows.offsets[1] = before;
    }
    if (p.slices > 1) {
        for (int g = 0; g <= p.slices; g++) {
            if (tid == 0) p.rows.slice_offsets[g] = g * before;
            if (g < p.slices)
                for (int r = tid; r < before; r += LOOK_THREADS) p.rows.slice_rows[g * before + r] = r;
        }
    }
}

hipError_t launch_loss_look(const loss_look_params &p, hipStream_t s)
{
    hipLaunchKernelGGL(k_loss_look, dim3(1), dim3(LOOK_THREADS), 0, s, p);
    return hipGetLastError();
}

__global__ __launch_bounds__(256) void k_loss_copy(loss_copy_params p)
{
    const long all = p.offsets[1] * p.pieces;
    for (long unit = (long)blockIdx.x * 256 + threadIdx.x; unit < all; unit += (long)gridDim.x * 256) {
        const long row = unit / p.pieces, piece = unit % p.pieces;
        ((u32x4 *)p.copy)[unit] = ((const u32x4 *)p.X)[p.list[row] * p.ldx + piece];
    }
}

hipError_t launch_loss_copy(const loss_copy_params &p, hipStream_t s)
{
    const long blocks = (p.tokens * p.pieces + 255) / 256;
    hipLaunchKernelGGL(k_loss_copy, dim3((unsigned)(blocks < 1 << 14 ? blocks : 1 << 14)), dim3(256), 0, s, p);
    return hipGetLastError();
}

// Sums of exponentials, over the largest of their scores: of all words, and of those that are not the target.
struct loss_sum {
    float most, all, others;
};
// Two of them as one.
__device__ inline loss_sum joined(const loss_sum &a, const loss_sum &b)
{
    const float most = fmaxf(a.most, b.most), from = most == -__builtin_inff() ? 0.f : most, fa = exp_of(a.most - from), fb = exp_of(b.most - from);
    return {most, a.all * fa + b.all * fb, a.others * fa + b.others * fb};
}
// COLUMNS tokens a workgroup, THREADS / COLUMNS lanes each over the slices; those of a wavefront meet by exchanges, the wavefronts in LDS in their order.
// (Four tokens a workgroup where they are few: 16 tokens, 2048 slices 9.9 us with sixteen.)
template <int THREADS, int COLUMNS>
__global__ __launch_bounds__(THREADS) void k_loss_join(loss_join_params p)
{
    constexpr int LANES = THREADS / COLUMNS, WAVES = THREADS / 64;
    __shared__ loss_sum parts[WAVES][COLUMNS];
    const int tid = threadIdx.x, column = tid % COLUMNS, lane = tid / COLUMNS;
    const int token = (int)blockIdx.x * COLUMNS + column;
    const int target = token < p.tokens ? p.targets[token] : -1;
    const bool counts = target >= 0 && target < p.vocabulary;
    const f32x2 goal = counts ? *(const f32x2 *)(p.goals + 2l * token) : f32x2{0.f, 0.f};
    loss_sum sum = {-__builtin_inff(), 0.f, 0.f};
    if (token < p.tokens) {
        const int goal_slice = counts ? target / p.slice : -1;
        for (int n = lane; n < p.slices; n += 8 * LANES) {
            // eight on the way at a time
            f32x2 v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = *(const f32x2 *)(p.stats + 2 * ((long)min(n + e * LANES, p.slices - 1) * p.stat_rows + token));
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (n + e * LANES < p.slices) sum = joined(sum, {v[e][0], v[e][1], n + e * LANES == goal_slice ? goal[1] : v[e][1]});
        }
    }
#pragma unroll
    for (int step = COLUMNS; step < 64; step *= 2) sum = joined(sum, {__shfl_xor(sum.most, step), __shfl_xor(sum.all, step), __shfl_xor(sum.others, step)});
    if ((tid & 63) < COLUMNS) parts[tid >> 6][column] = sum;
    __syncthreads();
    if (lane || token >= p.tokens) return;
    for (int n = 1; n < WAVES; n++) sum = joined(sum, parts[n][column]);
    const float lse = (sum.most == -__builtin_inff() ? 0.f : sum.most) + logf(sum.all);
    // (a row of padding that nobody filled may hold anything: no NaN comes of it)
    p.lse[token] = !counts && lse != lse ? 0.f : lse;
    // Where the target's score is the largest the loss is log1p of the others' sum, which keeps the digits of a loss far below 1.
    const float over = sum.most - goal[0];
    p.losses[token] = !counts ? 0.f : over == 0.f ? log1pf(sum.others) : over + logf(sum.all);
}

hipError_t launch_loss_join(const loss_join_params &p, hipStream_t s)
{
    auto grid = [&](int columns) { return dim3((unsigned)((p.tokens + columns - 1) / columns)); };
    if (p.slices <= 256) hipLaunchKernelGGL((k_loss_join<256, 16>), grid(16), dim3(256), 0, s, p);
    else if (p.tokens > 256) hipLaunchKernelGGL((k_loss_join<1024, 16>), grid(16), dim3(1024), 0, s, p);
    else hipLaunchKernelGGL((k_loss_join<1024, 4>), grid(4), dim3(1024), 0, s, p);
    return hipGetLastError();
}

// A lane takes eight columns of a token; the slices are added in their order.
template <class T, bool VECTOR>
__global__ __launch_bounds__(256) void k_loss_dx(loss_dx_params p)
{
    const long eights = (p.width + 7) / 8;
    const long rows = p.offsets[1];
    const float by = p.unscale ? *p.unscale : 1.f;
    for (long unit = (long)blockIdx.x * 256 + threadIdx.x; unit < eights * p.tokens; unit += (long)gridDim.x * 256) {
        const long token = unit / eights, c = unit % eights * 8;
        const int count = (int)min(8l, p.width - c), row = p.place[token];
        f32x8 v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row >= 0) {
            // (four on the way at a time)
#pragma unroll 4
            for (int n = 0; n < p.slices; n++) v += load8<float, VECTOR>(p.partial + (n * rows + row) * p.width + c, count);
            v *= by;
        }
        store8<T, VECTOR>((T *)p.dX + token * p.lddx + c, v, count);
    }
}

hipError_t launch_loss_dx(const loss_dx_params &p, int dtype, hipStream_t s)
{
    const long blocks = ((p.width + 7) / 8 * p.tokens + 255) / 256;
    const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), block(256);
    auto go = [&](auto type) {
        using T = decltype(type);
        if (p.vector) hipLaunchKernelGGL((k_loss_dx<T, true>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_loss_dx<T, false>), grid, block, 0, s, p);
    };
    if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
    return hipGetLastError();
}

}  // namespace miw
