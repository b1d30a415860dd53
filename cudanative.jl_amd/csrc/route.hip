// Routing of tokens to experts: the choice, its weights, and the order of the rows by expert; the gradient to the logits.
//
// Choice.  One wavefront per token, a lane holds logits lane, lane + 64, ...  as unsigned keys in the order of the
// values (0: never chosen).  The largest key of the wavefront comes from a reduction without LDS, and the lowest expert
// that has it from one ballot per register, so equal logits go to the lowest expert.
// Order.  Counting sort: choices are counted per expert and chunk of tokens (integers: no order matters), every chunk
// then starts at (choices of lower experts) + (choices of this expert in earlier chunks), and one wavefront hands out
// its chunk's positions in token order.  64 choices at a time find the earlier ones of the same expert by one ballot
// for each bit of the expert's number.
//
// Bound by latency throughout (16 tokens: the launch; 16384 x 128: two launches, and the choice's chain of reductions).
#include "experts.hpp"
#include "vec_types.hpp"

#include <type_traits>

namespace miw {

constexpr int ROUTE_THREADS = 512, ROUTE_WAVES = ROUTE_THREADS / 64;
constexpr int ROUTE_EXPERTS = 1024;
constexpr float LARGEST = 3.4028234663852886e38f;

// Key of a logit: the order of the keys is that of the values, -0 equals 0, and what is never chosen has key 0.
__device__ inline unsigned order_key(float z)
{
    const unsigned u = __builtin_bit_cast(unsigned, z + 0.0f);  // (-0 becomes 0)
    const unsigned key = u & 0x80000000u ? ~u : u | 0x80000000u;
    return z > -__builtin_inff() ? key : 0u;  // (false for NaN)
}
__device__ inline float key_value(unsigned key)
{
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// R: registers that hold a token's logits, ceil(experts / 64).
template <class T, int R>
__device__ inline void choose(const route_params &p, int token, int *hist)
{
    const int lane = threadIdx.x & 63;
    const T *z = (const T *)p.logits + (long)token * p.ld;
    unsigned key[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int e = lane + 64 * i;
        key[i] = e < p.experts ? order_key((float)z[e]) : 0u;
    }
    unsigned all[R];
#pragma unroll
    for (int i = 0; i < R; i++) all[i] = key[i];
    int mine = -1;           // lane j: choice j
    float value = 0.f, largest = 0.f;
    for (int j = 0; j < p.top; j++) {
        unsigned most = key[0];
#pragma unroll
        for (int i = 1; i < R; i++) most = max(most, key[i]);
        most = wave_max(most);
        if (most == 0) break;
        int expert = -1;
#pragma unroll
        for (int i = R - 1; i >= 0; i--) {
            const unsigned long has = __ballot(key[i] == most);
            if (has) expert = 64 * i + __builtin_ctzl(has);
        }
#pragma unroll
        for (int i = 0; i < R; i++)
            if (expert == lane + 64 * i) key[i] = 0;
        const float v = fminf(key_value(most), LARGEST);
        if (j == 0) largest = v;
        if (lane == j) {
            mine = expert;
            value = v;
        }
    }
    const float part = mine >= 0 ? __expf(value - largest) : 0.f;
    float sum = part;
    if (p.over_all) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (all[i]) sum += __expf(fminf(key_value(all[i]), LARGEST) - largest);
    }
    sum = wave_sum(sum);
    if (lane < p.top) {
        const long at = (long)token * p.top + lane;
        p.chosen[at] = mine;
        p.gates[at] = mine >= 0 ? part / sum : 0.f;
        if (mine >= 0) atomicAdd(&hist[mine], 1);
    }
}

// Positions of a chunk's choices.  start: in LDS, the next position of each expert.  One wavefront.
__device__ inline void place_chunk(const route_params &p, int first, int last, int *start)
{
    const int lane = threadIdx.x & 63;
    for (int at = first * p.top; at < last * p.top; at += 64) {
        const int i = at + lane;
        const bool in = i < last * p.top;
        const int expert = in ? p.chosen[i] : -1;
        unsigned long same = __ballot(expert >= 0);
        for (int bit = 0; (p.experts - 1) >> bit; bit++) {
            const bool set = (expert >> bit) & 1;
            const unsigned long with = __ballot(set);
            same &= set ? with : ~with;
        }
        const int before = __builtin_popcountl(same & ((1ul << lane) - 1));
        int position = -1;
        if (expert >= 0) {
            position = start[expert] + before;
            p.rows[position] = i / p.top;
        }
        if (in) p.place[i] = position;
        __builtin_amdgcn_wave_barrier();
        if (expert >= 0 && (same >> lane) == 1ul) start[expert] = position + 1;  // (the last of them)
        __builtin_amdgcn_wave_barrier();
    }
}

// Turns counts per expert, in LDS, into the first position of each; one wavefront.  Returns the number of choices.
__device__ inline int first_positions(int experts, int *counts)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = e0 + lane, c = e < experts ? counts[e] : 0;
        const int upto = wave_scan(c) + before;
        if (e < experts) counts[e] = upto - c;
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return before;
}

// WHOLE: one workgroup for all tokens, choice and order in one launch.  A prompt's worth of tokens takes two: the
// chunks' counts have to be there before any position is known.
template <class T, int R, bool WHOLE>
__global__ __launch_bounds__(ROUTE_THREADS) void k_route_choose(route_params p)
{
    __shared__ int hist[ROUTE_EXPERTS];
    __shared__ int total;
    const int wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < p.experts; e += ROUTE_THREADS) hist[e] = 0;
    __syncthreads();
    const int first = WHOLE ? 0 : blockIdx.x * p.chunk, last = WHOLE ? p.tokens : min(p.tokens, first + p.chunk);
    for (int t = first + wave; t < last; t += ROUTE_WAVES) choose<T, R>(p, t, hist);
    __syncthreads();
    if constexpr (WHOLE) {
        if (wave == 0) {
            const int n = first_positions(p.experts, hist);
            if (threadIdx.x == 0) total = n;
            __threadfence_block();
            for (int e = threadIdx.x; e < p.experts; e += 64) p.offsets[e] = hist[e];
            if (threadIdx.x == 0) p.offsets[p.experts] = n;
            place_chunk(p, first, last, hist);
        }
        __syncthreads();
        for (int i = total + (int)threadIdx.x; i < p.tokens * p.top; i += ROUTE_THREADS) p.rows[i] = -1;
    } else {
        for (int e = threadIdx.x; e < p.experts; e += ROUTE_THREADS) p.counts[(long)blockIdx.x * p.experts + e] = hist[e];
    }
}

__global__ __launch_bounds__(ROUTE_THREADS) void k_route_place(route_params p)
{
    __shared__ int counts[ROUTE_EXPERTS], earlier[ROUTE_EXPERTS];
    __shared__ int total;
    const int wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < p.experts; e += ROUTE_THREADS) counts[e] = earlier[e] = 0;
    __syncthreads();
    // Several threads add up an expert's chunks where there are fewer experts than threads.
    const int lanes = ROUTE_THREADS / p.experts < 1 ? 1 : ROUTE_THREADS / p.experts;
    for (int i = threadIdx.x; i < p.experts * lanes; i += ROUTE_THREADS) {
        const int e = i % p.experts;
        int all = 0, before = 0;
        for (int c = i / p.experts; c < p.chunks; c += lanes) {
            const int n = p.counts[(long)c * p.experts + e];
            all += n;
            if (c < (int)blockIdx.x) before += n;
        }
        atomicAdd(&counts[e], all);
        atomicAdd(&earlier[e], before);
    }
    __syncthreads();
    if (wave == 0) {
        const int n = first_positions(p.experts, counts);
        if (threadIdx.x == 0) total = n;
        if (blockIdx.x == 0) {
            for (int e = threadIdx.x; e < p.experts; e += 64) p.offsets[e] = counts[e];
            if (threadIdx.x == 0) p.offsets[p.experts] = n;
        }
        for (int e = threadIdx.x; e < p.experts; e += 64) earlier[e] += counts[e];
        __builtin_amdgcn_wave_barrier();
        const int first = blockIdx.x * p.chunk;
        place_chunk(p, first, min(p.tokens, first + p.chunk), earlier);
    }
    __syncthreads();
    for (int i = total + (int)(blockIdx.x * ROUTE_THREADS + threadIdx.x); i < p.tokens * p.top; i += (int)(gridDim.x * ROUTE_THREADS)) p.rows[i] = -1;
}

// dz over the chosen: g (dg - sum g dg); over all: p_e (dg_e - sum g dg), dg_e zero where e is not chosen.  A wavefront per token.
template <class T>
__global__ __launch_bounds__(256) void k_route_grad(route_grad_params p)
{
    const int lane = threadIdx.x & 63, token = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= p.tokens) return;
    const long at = (long)token * p.top + lane;
    int expert = -1;
    float gate = 0.f, dgate = 0.f;
    if (lane < p.top) {
        expert = p.chosen[at];
        gate = p.gates[at];
        if (expert >= 0) dgate = p.dgates[at];  // (what a choice without an expert gets is not looked at)
    }
    const float inner = wave_sum(gate * dgate);
    const T *z = (const T *)p.logits + (long)token * p.ld;
    T *dz = (T *)p.dlogits + (long)token * p.ldd;
    // The softmax over all logits from its largest: choice 0 is the largest logit.
    const int first = __builtin_amdgcn_readlane(expert, 0);
    const bool all = p.over_all && first >= 0 && first < p.experts;
    float largest = 0.f, total = 1.f;
    if (all) {
        largest = fminf((float)z[first], LARGEST);
        float sum = 0.f;
        for (int e = lane; e < p.experts; e += 64) {
            const float v = (float)z[e];
            if (v > -__builtin_inff()) sum += __expf(fminf(v, LARGEST) - largest);
        }
        total = wave_sum(sum);
    }
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
        const int e = e0 + lane;
        float own = 0.f;
        bool chosen = false;
        for (int j = 0; j < p.top; j++) {
            const int x = __builtin_amdgcn_readlane(expert, j);
            const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p.over_all ? gate * dgate : gate * (dgate - inner)), j));
            if (x == e) {
                own = v;
                chosen = true;
            }
        }
        if (e >= p.experts) continue;
        float d = chosen ? own : 0.f;
        if (all) {
            const float v = (float)z[e];
            if (v > -__builtin_inff()) d -= __expf(fminf(v, LARGEST) - largest) / total * inner;
        }
        dz[e] = (T)d;
    }
}

// One workgroup as long as its wavefronts have no more than eight tokens each and its one placing wavefront sixteen rounds.
int route_chunks(long tokens, int top)
{
    if (tokens <= 8 * ROUTE_WAVES && tokens * top <= 1024) return 1;
    const long chunk = (tokens + 255) / 256 > ROUTE_WAVES ? (tokens + 255) / 256 : ROUTE_WAVES;
    return (int)((tokens + chunk - 1) / chunk);
}

hipError_t launch_route(route_params p, int dtype, hipStream_t s)
{
    p.chunks = route_chunks(p.tokens, p.top);
    p.chunk = (p.tokens + p.chunks - 1) / p.chunks;
    const int r = (p.experts + 63) / 64;
    auto go = [&](auto type, auto regs) {
        using T = decltype(type);
        constexpr int R = decltype(regs)::value;
        if (p.chunks == 1) hipLaunchKernelGGL((k_route_choose<T, R, true>), dim3(1), dim3(ROUTE_THREADS), 0, s, p);
        else hipLaunchKernelGGL((k_route_choose<T, R, false>), dim3((unsigned)p.chunks), dim3(ROUTE_THREADS), 0, s, p);
    };
    auto typed = [&](auto type) {
        if (r == 1) go(type, std::integral_constant<int, 1>{});
        else if (r == 2) go(type, std::integral_constant<int, 2>{});
        else if (r <= 4) go(type, std::integral_constant<int, 4>{});
        else go(type, std::integral_constant<int, 16>{});
    };
    if (dtype == TYPE_F32) typed(float{});
    else if (dtype == TYPE_F16) typed(f16_t{});
    else typed(bf16_t{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)p.chunks), dim3(ROUTE_THREADS), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_route_grad(const route_grad_params &p, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)((p.tokens + 3) / 4)), block(256);
    if (dtype == TYPE_F32) hipLaunchKernelGGL(k_route_grad<float>, grid, block, 0, s, p);
    else if (dtype == TYPE_F16) hipLaunchKernelGGL(k_route_grad<f16_t>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(k_route_grad<bf16_t>, grid, block, 0, s, p);
    return hipGetLastError();
}

}  // namespace miw
