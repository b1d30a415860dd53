// The experts' answers joined by their weights, and the gradients to answers and weights.
//
// Bound by HBM: every row of H is read once and every row of the result written once, in 16-byte pieces.  8191 tokens, 4
// choices, 4096 columns (bf16): 56 to 57 us (336 MB, 5.9 TB/s), gradients 105 to 107 us (604 MB, 5.7 TB/s); a large copy reaches 4.8 to 5.4.
// 16 tokens: 2.9 to 3.2 us, a launch's latency and two dependent reads.  Sums run over a
// token's choices in order, in Float32, and are rounded once.
#include "experts.hpp"
#include "vec_types.hpp"

#include <type_traits>

namespace miw {

constexpr int COMBINE_THREADS = 256;
constexpr int COMBINE_TOGETHER = 4;  // rows of H that a thread has on the way

// Y[t] = sum over j of gates[t][j] H[place[t][j]].  A workgroup takes 2048 columns of one token.
template <class T, bool VECTOR, bool STREAM>
__global__ __launch_bounds__(COMBINE_THREADS) void k_combine(combine_params p)
{
    const int token = blockIdx.x;
    const long c = ((long)blockIdx.y * COMBINE_THREADS + threadIdx.x) * 8;
    if (c >= p.n) return;
    const int count = (int)min(8l, p.n - c);
    const int *place = p.place + (long)token * p.top;
    const float *gates = p.gates ? p.gates + (long)token * p.top : nullptr;
    const T *H = (const T *)p.H + c;
    f32x8 sum = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < p.top; j0 += COMBINE_TOGETHER) {
        f32x8 h[COMBINE_TOGETHER];
        float g[COMBINE_TOGETHER];
        bool has[COMBINE_TOGETHER];
#pragma unroll
        for (int j = 0; j < COMBINE_TOGETHER; j++) {
            const int at = j0 + j < p.top ? place[j0 + j] : -1;
            has[j] = at >= 0 && at < p.rows;
            if (has[j]) {
                h[j] = load8<T, VECTOR, STREAM>(H + (long)at * p.ldh, count);
                g[j] = gates ? gates[j0 + j] : 1.f;
            }
        }
#pragma unroll
        for (int j = 0; j < COMBINE_TOGETHER; j++)
            if (has[j])
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] = __builtin_fmaf(g[j], h[j][e], sum[e]);
    }
    store8<T, VECTOR, STREAM>((T *)p.out + (long)token * p.ldy + c, sum, count);
}

// dH[place[t][j]] = gates[t][j] dY[t] and dgates[t][j] = dY[t] . H[place[t][j]].  A workgroup takes a token; a thread's parts of
// the dot products meet through LDS in a fixed order.
template <class T, bool VECTOR, bool DOTS, bool STREAM>
__global__ __launch_bounds__(COMBINE_THREADS) void k_combine_grad(combine_params p)
{
    constexpr int WAVES = COMBINE_THREADS / 64;
    __shared__ float parts[WAVES][COMBINE_TOGETHER];
    const int token = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int *place = p.place + (long)token * p.top;
    const T *dY = (const T *)p.dY + (long)token * p.ldy;
    for (int j0 = 0; j0 < p.top; j0 += COMBINE_TOGETHER) {
        int at[COMBINE_TOGETHER];
        float g[COMBINE_TOGETHER], dot[COMBINE_TOGETHER];
#pragma unroll
        for (int j = 0; j < COMBINE_TOGETHER; j++) {
            const int x = j0 + j < p.top ? place[j0 + j] : -1;
            at[j] = x < p.rows ? x : -1;
            g[j] = at[j] >= 0 && p.gates ? p.gates[(long)token * p.top + j0 + j] : 1.f;
            dot[j] = 0.f;
        }
        for (long c = threadIdx.x * 8; c < p.n; c += COMBINE_THREADS * 8) {
            const int count = (int)min(8l, p.n - c);
            const f32x8 dy = load8<T, VECTOR>(dY + c, count);
            f32x8 h[COMBINE_TOGETHER];
            if constexpr (DOTS)
#pragma unroll
                for (int j = 0; j < COMBINE_TOGETHER; j++)
                    if (at[j] >= 0) h[j] = load8<T, VECTOR, STREAM>((const T *)p.H + (long)at[j] * p.ldh + c, count);
#pragma unroll
            for (int j = 0; j < COMBINE_TOGETHER; j++) {
                if (at[j] < 0) continue;
                f32x8 d;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    d[e] = g[j] * dy[e];
                    if constexpr (DOTS) dot[j] = __builtin_fmaf(dy[e], h[j][e], dot[j]);
                }
                store8<T, VECTOR, STREAM>((T *)p.out + (long)at[j] * p.lddh + c, d, count);
            }
        }
        if constexpr (DOTS) {
#pragma unroll
            for (int j = 0; j < COMBINE_TOGETHER; j++) {
                const float sum = wave_sum(dot[j]);
                if (lane == 0) parts[wave][j] = sum;
            }
            __syncthreads();
            if (threadIdx.x < COMBINE_TOGETHER && j0 + (int)threadIdx.x < p.top) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; w++) sum += parts[w][threadIdx.x];
                p.dgates[(long)token * p.top + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

// Writing H, joining it, its gradients and reading those, 4 choices and 4096 columns (bf16), streamed and not: 823 and 841 us at 537 MB
// of H, 411 and 427 at 268 MB (join and gradients alone, call after call: 164 and 185), 211 and 214 at 134 MB; but 116 and 112 at 67 MB and
// 70 and 62 at 34 MB, where the next kernel finds in a cache what was not streamed.
static bool streams(const combine_params &p) { return p.vector && 2l * p.tokens * p.top * p.n > STREAM_BYTES; }

hipError_t launch_combine(const combine_params &p, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)p.tokens, (unsigned)((p.n + 8 * COMBINE_THREADS - 1) / (8 * COMBINE_THREADS))), block(COMBINE_THREADS);
    auto go = [&](auto type) {
        using T = decltype(type);
        if (streams(p)) hipLaunchKernelGGL((k_combine<T, true, true>), grid, block, 0, s, p);
        else if (p.vector) hipLaunchKernelGGL((k_combine<T, true, false>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_combine<T, false, false>), grid, block, 0, s, p);
    };
    if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
    return hipGetLastError();
}

hipError_t launch_combine_grad(const combine_params &p, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)p.tokens), block(COMBINE_THREADS);
    auto go = [&](auto type) {
        using T = decltype(type);
        auto dots = [&](auto wanted) {
            constexpr bool DOTS = decltype(wanted)::value;
            if (streams(p)) hipLaunchKernelGGL((k_combine_grad<T, true, DOTS, true>), grid, block, 0, s, p);
            else if (p.vector) hipLaunchKernelGGL((k_combine_grad<T, true, DOTS, false>), grid, block, 0, s, p);
            else hipLaunchKernelGGL((k_combine_grad<T, false, DOTS, false>), grid, block, 0, s, p);
        };
        if (p.dgates) dots(std::true_type{});
        else dots(std::false_type{});
    };
    if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
    return hipGetLastError();
}

}  // namespace miw
