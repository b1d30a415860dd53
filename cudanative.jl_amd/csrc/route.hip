// Routing of tokens to experts: the choice, its weights, and the order of the rows by expert; the gradient to the logits.
//
// Choice.  A lane holds logits as unsigned keys in the order of the values (0: never chosen).  Up to 256 experts a token has sixteen
// lanes, four tokens a wavefront: the largest key and the lowest expert that has it are two reductions over a row of lanes by
// data-parallel moves, so equal logits go to the lowest expert; 16-bit logits carry the expert in the key's low half, and one reduction does.  What bounds it is the number of instructions: with a wavefront for every
// token, forty of them a choice in place of fourteen, the first launch of the case below took 12.4 us.  Beyond 256 experts a token has a
// wavefront, and a ballot per register finds the expert.
// Order.  Counting sort in two launches over at most 256 chunks of tokens (one launch for up to 64 tokens).  The first counts its chunk's
// choices of each expert and ranks them: 64 at a time, a wavefront finds the earlier ones of the same expert by one ballot for each
// bit of the expert's number, and what the 64s before it have is added from a table in LDS.  The second adds up the counts of
// lower experts and earlier chunks and writes the positions.  Counts are integers: no order of theirs matters.
//
// Bound by latency throughout: 16381 tokens, 128 experts, 8 choices (bf16), 4.2 MB of logits and 1.6 MB of results, where the bytes alone take one to two
// microseconds a launch: back to back choice and order 16.5 us and gradient 6.2 (8.4 MB in and out); under the profiler, medians, choose 9.0, place 8.5 to 9.8,
// gradient 6.4 to 7.3.  (When they were tried: choose 8.5, 9.4 with two reductions; gradient 6.0, 7.8 with a wavefront a token.)  16 tokens of 64 experts, 4
// choices: one launch of 3.2 to 3.4 us.  A wavefront a token: 16381 tokens of 512 experts (f32) 70 us, gradient over all 24; of 1024 (bf16) 102 and 35.
#include "experts.hpp"
#include "vec_types.hpp"

#include <type_traits>

namespace miw {

constexpr int ROUTE_THREADS = 1024, ROUTE_WAVES = ROUTE_THREADS / 64;
constexpr int ROUTE_EXPERTS = 1024, ROUTE_TOP = 16;
constexpr int ROUTE_TOKENS = 64;                                      // tokens that a workgroup chooses for at a time
constexpr int ROUTE_SEGMENTS = ROUTE_TOKENS * ROUTE_TOP / 64;         // of 64 choices
static_assert(ROUTE_SEGMENTS <= ROUTE_WAVES, "a wavefront for each");
constexpr float LARGEST = 3.4028234663852886e38f;

// Key of a logit: the order of the keys is that of the values, -0 equals 0, +inf the largest finite Float32, and what is never
// chosen has key 0.
__device__ inline unsigned order_key(float z)
{
    const unsigned u = __builtin_bit_cast(unsigned, fminf(z, LARGEST) + 0.0f);  // (-0 becomes 0)
    const unsigned key = u & 0x80000000u ? ~u : u | 0x80000000u;
    return z > -__builtin_inff() ? key : 0u;  // (false for NaN)
}
__device__ inline float key_value(unsigned key)
{
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Logits of 16 bits have keys of 16, and the expert fits beside them: the largest such number names the largest logit and, of equal ones,
// the lowest expert, by one reduction.  (No finite one equals Float32's largest, which +inf counts as.)
template <class T>
__device__ inline unsigned packed_key(T z, int expert)
{
    const unsigned u = z == (T)0.f ? 0u : __builtin_bit_cast(unsigned short, z);
    const unsigned key = u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
    return (float)z > -__builtin_inff() ? key << 16 | (0xffffu - (unsigned)expert) : 0u;
}
template <class T>
__device__ inline float packed_value(unsigned packed)
{
    const unsigned key = packed >> 16;
    return (float)__builtin_bit_cast(T, (unsigned short)(key & 0x8000u ? key & 0x7fffu : ~key));
}

// exp of x <= 0, -inf among them, to two units in the last place: 2^t with t = x log2 e rounded, times what the rounding left out, which for x
// near -80 is up to 2^-18 of the result.  Results below 2^-126 are zeros.  (Gradient of 16381 tokens of 1024 experts over all, bf16: 33.7 us with 2^t alone,
// 34.7 so, 36.9 with expf.)
__device__ inline float exp_below(float x)
{
    constexpr float LOG2E = 1.44269504f, REST = (float)(1.4426950408889634074 - (double)LOG2E), LN2 = 0.69314718f;
    x = fmaxf(x, -200.f);
    const float t = x * LOG2E, left = __builtin_fmaf(x, REST, __builtin_fmaf(x, LOG2E, -t)), e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, LN2 * left, e);
}

// Over the sixteen lanes of a row, to all of them; sums pair the same lanes in every lane.
template <class F>
__device__ inline int row_reduce(int v, F join)
{
    v = join(v, __builtin_amdgcn_update_dpp(0, v, 0x128 /* row_ror:8 */, 0xf, 0xf, true));
    v = join(v, __builtin_amdgcn_update_dpp(0, v, 0x124, 0xf, 0xf, true));
    v = join(v, __builtin_amdgcn_update_dpp(0, v, 0x122, 0xf, 0xf, true));
    return join(v, __builtin_amdgcn_update_dpp(0, v, 0x121, 0xf, 0xf, true));
}
__device__ inline unsigned row_max(unsigned v) { return (unsigned)row_reduce((int)v, [](int a, int b) { return (int)max((unsigned)a, (unsigned)b); }); }
__device__ inline int row_min(int v) { return row_reduce(v, [](int a, int b) { return min(a, b); }); }
__device__ inline float row_sum(float v)
{
    return __builtin_bit_cast(float, row_reduce(__builtin_bit_cast(int, v), [](int a, int b) { return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)); }));
}

// Writes choice `lane` of a token (lanes below top), its gate, and the choice into LDS.
__device__ inline void write_choice(const route_params &p, int base, int token, int lane, int expert, float part, float sum, int *kept)
{
    if (lane >= p.top) return;
    const int at = token * p.top + lane;
    p.chosen[at] = expert;
    p.gates[at] = expert >= 0 ? part / sum : 0.f;
    kept[(token - base) * p.top + lane] = expert;
}

// Sixteen lanes a token: tokens first .. first + 3, those below last.  R: registers that hold a token's logits, ceil(experts / 16).
// `kept`: the choices in LDS, those of token `base` first.
template <class T, int R>
__device__ inline void choose_row(const route_params &p, int base, int first, int last, int *kept)
{
    const int lane = threadIdx.x & 15, token = first + ((threadIdx.x & 63) >> 4);
    const bool in = token < last;
    const T *z = (const T *)p.logits + (long)(in ? token : first) * p.ld;
    constexpr bool PACKED = sizeof(T) == 2;
    auto value_of = [](unsigned k) {
        if constexpr (PACKED) return fminf(packed_value<T>(k), LARGEST);
        else return key_value(k);
    };
    unsigned key[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int e = lane + 16 * i;
        if constexpr (PACKED) key[i] = e < p.experts ? packed_key(z[e], e) : 0u;
        else key[i] = e < p.experts ? order_key(z[e]) : 0u;
    }
    int mine = -1;  // lane j: choice j
    float value = 0.f, largest = 0.f, every = 0.f;
    for (int j = 0; j < p.top; j++) {
        unsigned most = key[0];
#pragma unroll
        for (int i = 1; i < R; i++) most = max(most, key[i]);
        most = row_max(most);
        const float v = value_of(most);
        if (j == 0) {
            largest = v;
            if (p.over_all)
#pragma unroll
                for (int i = 0; i < R; i++) every += exp_below(key[i] ? value_of(key[i]) - v : -__builtin_inff());
        }
        int expert;
        if constexpr (PACKED) {
            expert = 0xffff - (int)(most & 0xffffu);
#pragma unroll
            for (int i = 0; i < R; i++) key[i] = key[i] == most ? 0u : key[i];
        } else {
            expert = 1 << 30;
#pragma unroll
            for (int i = R - 1; i >= 0; i--) expert = key[i] == most ? lane + 16 * i : expert;
            expert = row_min(expert);
            const int hit = (expert & 15) == lane ? expert >> 4 : -1;
#pragma unroll
            for (int i = 0; i < R; i++) key[i] = hit == i ? 0u : key[i];
        }
        if (lane == j && most) {
            mine = expert;
            value = v;
        }
    }
    const float part = mine >= 0 ? exp_below(value - largest) : 0.f;
    const float sum = row_sum(p.over_all ? every : part);
    if (in) write_choice(p, base, token, lane, mine, part, sum, kept);
}

// A wavefront for the token.  R: ceil(experts / 64).
template <class T, int R>
__device__ inline void choose_wave(const route_params &p, int base, int token, int *kept)
{
    const int lane = threadIdx.x & 63;
    const T *z = (const T *)p.logits + (long)token * p.ld;
    unsigned key[R];
#pragma unroll
    for (int i = 0; i < R; i++) key[i] = lane + 64 * i < p.experts ? order_key((float)z[lane + 64 * i]) : 0u;
    int mine = -1;
    float value = 0.f, largest = 0.f, every = 0.f;
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
        const float v = key_value(most);
        if (j == 0) {
            largest = v;
            if (p.over_all)
#pragma unroll
                for (int i = 0; i < R; i++) every += exp_below(key[i] ? key_value(key[i]) - v : -__builtin_inff());
        }
#pragma unroll
        for (int i = 0; i < R; i++)
            if (expert == lane + 64 * i) key[i] = 0;
        if (lane == j) {
            mine = expert;
            value = v;
        }
    }
    const float part = mine >= 0 ? exp_below(value - largest) : 0.f;
    write_choice(p, base, token, lane, mine, part, wave_sum(p.over_all ? every : part), kept);
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

// WHOLE: one workgroup for all tokens, choice and order in one launch.  ROW: sixteen lanes a token, or a wavefront.
template <class T, int R, bool ROW, bool WHOLE>
__global__ __launch_bounds__(ROUTE_THREADS) void k_route_choose(route_params p)
{
    __shared__ int kept[ROUTE_TOKENS * ROUTE_TOP];
    __shared__ unsigned short table[ROUTE_SEGMENTS][ROUTE_EXPERTS];  // choices of each expert in each 64
    __shared__ int running[ROUTE_EXPERTS];
    __shared__ int total;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int first = WHOLE ? 0 : blockIdx.x * p.chunk, last = WHOLE ? p.tokens : min(p.tokens, first + p.chunk);
    for (int e = tid; e < p.experts; e += ROUTE_THREADS) running[e] = 0;
    for (int base = first; base < last; base += ROUTE_TOKENS) {
        const int end = min(last, base + ROUTE_TOKENS), choices = (end - base) * p.top, segments = (choices + 63) / 64;
        for (int i = tid; i < segments * p.experts; i += ROUTE_THREADS) table[i / p.experts][i % p.experts] = 0;
        if constexpr (ROW) {
            if (base + 4 * wave < end) choose_row<T, R>(p, base, base + 4 * wave, end, kept);
        } else {
            for (int t = base + wave; t < end; t += ROUTE_WAVES) choose_wave<T, R>(p, base, t, kept);
        }
        __syncthreads();
        const int i = wave * 64 + lane;
        int expert = -1, before = 0;
        if (wave < segments) {
            expert = i < choices ? kept[i] : -1;
            unsigned long same = __ballot(expert >= 0);
            for (int bit = 0; (p.experts - 1) >> bit; bit++) {
                const bool set = (expert >> bit) & 1;
                const unsigned long with = __ballot(set);
                same &= set ? with : ~with;
            }
            before = __builtin_popcountl(same & ((1ul << lane) - 1));
            if (expert >= 0 && (same >> lane) == 1ul) table[wave][expert] = (unsigned short)(before + 1);  // (the last of them)
        }
        __syncthreads();
        if (i < choices) {
            int rank = -1;
            if (expert >= 0) {
                rank = running[expert] + before;
                for (int s = 0; s < wave; s++) rank += table[s][expert];
            }
            if constexpr (WHOLE) kept[i] = rank;  // (read and written by this thread alone)
            else p.place[base * p.top + i] = rank;
        }
        __syncthreads();
        for (int e = tid; e < p.experts; e += ROUTE_THREADS) {
            int sum = running[e];
            for (int s = 0; s < segments; s++) sum += table[s][e];
            running[e] = sum;
        }
        if constexpr (WHOLE) {
            __syncthreads();
            if (wave == 0) {
                const int n = first_positions(p.experts, running);
                if (tid == 0) total = n;
            }
            __syncthreads();
            for (int e = tid; e < p.experts; e += ROUTE_THREADS) p.offsets[e] = running[e];
            if (tid == 0) p.offsets[p.experts] = total;
            if (i < choices) {
                const int position = expert >= 0 ? running[expert] + kept[i] : -1;
                p.place[i] = position;
                if (position >= 0) p.rows[position] = i / p.top;
            }
            for (int at = total + tid; at < p.tokens * p.top; at += ROUTE_THREADS) p.rows[at] = -1;
        } else {
            __syncthreads();
        }
    }
    if constexpr (WHOLE) {
        if (p.tokens == 0)
            for (int e = tid; e <= p.experts; e += ROUTE_THREADS) p.offsets[e] = 0;
    } else {
        for (int e = tid; e < p.experts; e += ROUTE_THREADS) p.counts[(long)blockIdx.x * p.experts + e] = running[e];
    }
}

__global__ __launch_bounds__(ROUTE_THREADS) void k_route_place(route_params p)
{
    __shared__ int counts[ROUTE_EXPERTS], earlier[ROUTE_EXPERTS];
    __shared__ int total;
    const int tid = threadIdx.x;
    const int first = blockIdx.x * p.chunk * p.top, last = min(p.tokens, (int)(blockIdx.x + 1) * p.chunk) * p.top;
    // This thread's first choice is asked for ahead of the counts.
    int expert = -1, rank = 0;
    if (first + tid < last) {
        expert = p.chosen[first + tid];
        rank = p.place[first + tid];
    }
    for (int e = tid; e < p.experts; e += ROUTE_THREADS) counts[e] = earlier[e] = 0;
    __syncthreads();
    // Several threads add up an expert's chunks, eight loads on the way.
    const int columns = (p.experts + 63) & ~63, slices = ROUTE_THREADS / columns;
    const int e = tid % columns, slice = tid / columns;
    if (e < p.experts && slice < slices) {
        int all = 0, before = 0;
        for (int c0 = slice; c0 < p.chunks; c0 += 8 * slices) {
            int n[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int c = c0 + u * slices;
                n[u] = c < p.chunks ? p.counts[(long)c * p.experts + e] : 0;
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                all += n[u];
                before += c0 + u * slices < (int)blockIdx.x ? n[u] : 0;
            }
        }
        atomicAdd(&counts[e], all);
        atomicAdd(&earlier[e], before);
    }
    __syncthreads();
    if (tid < 64) {
        const int n = first_positions(p.experts, counts);
        if (tid == 0) total = n;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = tid; i < p.experts; i += ROUTE_THREADS) p.offsets[i] = counts[i];
        if (tid == 0) p.offsets[p.experts] = total;
    }
    for (int at = first + tid; at < last; at += ROUTE_THREADS) {
        if (at != first + tid) {
            expert = p.chosen[at];
            rank = p.place[at];
        }
        if (expert < 0) continue;
        const int position = counts[expert] + earlier[expert] + rank;
        p.place[at] = position;
        p.rows[position] = at / p.top;
    }
    for (int i = total + (int)(blockIdx.x * ROUTE_THREADS) + tid; i < p.tokens * p.top; i += (int)(gridDim.x * ROUTE_THREADS)) p.rows[i] = -1;
}

// dz over the chosen: g (dg - sum g dg); over all: p_e (dg_e - sum g dg), dg_e zero where e is not chosen.  LANES (16 up to 256 experts,
// or 64) have a token; its logits, R registers a lane, are asked for together with what it chose.
template <class T, int R, int LANES>
__global__ __launch_bounds__(256) void k_route_grad(route_grad_params p)
{
    const int lane = threadIdx.x & (LANES - 1);
    for (long token = ((long)blockIdx.x * 256 + threadIdx.x) / LANES; token < p.tokens; token += (long)gridDim.x * (256 / LANES)) {
        const T *z = (const T *)p.logits + token * p.ld;
        T *dz = (T *)p.dlogits + token * p.ldd;
        float v[R];
        if (p.over_all)
#pragma unroll
            for (int i = 0; i < R; i++) v[i] = lane + LANES * i < p.experts ? (float)z[lane + LANES * i] : -__builtin_inff();
        const long at = token * p.top + lane;
        int expert = -1;
        float gate = 0.f, dgate = 0.f;
        if (lane < p.top) {
            expert = p.chosen[at];
            gate = p.gates[at];
            dgate = p.dgates[at];
        }
        if (expert < 0) gate = dgate = 0.f;  // (what a choice without an expert gets is not looked at)
        const float inner = LANES == 16 ? row_sum(gate * dgate) : wave_sum(gate * dgate);
        const float direct = p.over_all ? gate * dgate : gate * (dgate - inner);
        float scale = 0.f;
        if (p.over_all) {
            // The softmax over all logits from its largest.
            unsigned most = 0;
#pragma unroll
            for (int i = 0; i < R; i++) most = max(most, order_key(v[i]));
            most = LANES == 16 ? row_max(most) : wave_max(most);
            const float largest = most ? key_value(most) : 0.f;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < R; i++) {
                v[i] = exp_below(v[i] > -__builtin_inff() ? fminf(v[i], LARGEST) - largest : -__builtin_inff());  // (NaN: 0)
                sum += v[i];
            }
            const float total = LANES == 16 ? row_sum(sum) : wave_sum(sum);
            if (total > 0.f) scale = -inner / total;
        }
        float d[R];
#pragma unroll
        for (int i = 0; i < R; i++) d[i] = p.over_all ? v[i] * scale : 0.f;
        for (int j = 0; j < p.top; j++) {
            const int x = __shfl(expert, j, LANES);
            const float add = __shfl(direct, j, LANES);
            const int hit = (x & (LANES - 1)) == lane ? x >> (LANES == 16 ? 4 : 6) : -1;  // (-1 stays -1)
#pragma unroll
            for (int i = 0; i < R; i++) d[i] += hit == i ? add : 0.f;
        }
#pragma unroll
        for (int i = 0; i < R; i++)
            if (lane + LANES * i < p.experts) dz[lane + LANES * i] = (T)d[i];
    }
}

// At most 256 chunks of sixteen tokens (one a wavefront) or more; one workgroup as long as it has its tokens together.
constexpr int ROUTE_CHUNKS = 256;
static int route_chunk(long tokens)
{
    const long chunk = (tokens + ROUTE_CHUNKS - 1) / ROUTE_CHUNKS;
    return (int)(chunk < ROUTE_WAVES ? ROUTE_WAVES : chunk);
}
// (The number of chunks falls where the chunk becomes a token longer.)
int route_most_chunks(long tokens)
{
    const long chunks = (tokens + ROUTE_WAVES - 1) / ROUTE_WAVES;
    return tokens <= ROUTE_TOKENS ? 1 : (int)(chunks < ROUTE_CHUNKS ? chunks : ROUTE_CHUNKS);
}
static int route_chunks(long tokens)
{
    return tokens <= ROUTE_TOKENS ? 1 : (int)((tokens + route_chunk(tokens) - 1) / route_chunk(tokens));
}

// Registers that hold a token's logits on sixteen lanes (up to 256 experts); a wavefront has sixteen for up to 1024.
template <class F>
static void with_registers(int experts, F go)
{
    if (experts <= 64) go(std::integral_constant<int, 4>{});
    else if (experts <= 128) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}
template <class F>
static void with_type(int dtype, F go)
{
    if (dtype == TYPE_F32) go(float{});
    else if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
}

hipError_t launch_route(route_params p, int dtype, hipStream_t s)
{
    p.chunks = route_chunks(p.tokens);
    p.chunk = route_chunk(p.tokens);
    with_type(dtype, [&](auto type) {
        using T = decltype(type);
        auto go = [&](auto regs, auto row) {
            constexpr int R = decltype(regs)::value;
            constexpr bool ROW = decltype(row)::value;
            if (p.chunks == 1) hipLaunchKernelGGL((k_route_choose<T, R, ROW, true>), dim3(1), dim3(ROUTE_THREADS), 0, s, p);
            else hipLaunchKernelGGL((k_route_choose<T, R, ROW, false>), dim3((unsigned)p.chunks), dim3(ROUTE_THREADS), 0, s, p);
        };
        if (p.experts > 256) go(std::integral_constant<int, 16>{}, std::false_type{});
        else with_registers(p.experts, [&](auto regs) { go(regs, std::true_type{}); });
    });
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)p.chunks), dim3(ROUTE_THREADS), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_route_grad(const route_grad_params &p, int dtype, hipStream_t s)
{
    const bool row = p.experts <= 256;
    const long blocks = (p.tokens + (row ? 15l : 3l)) / (row ? 16 : 4);
    const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), block(256);
    with_type(dtype, [&](auto type) {
        using T = decltype(type);
        if (row) with_registers(p.experts, [&](auto regs) {
            hipLaunchKernelGGL((k_route_grad<T, decltype(regs)::value, 16>), grid, block, 0, s, p);
        });
        else hipLaunchKernelGGL((k_route_grad<T, 16, 64>), grid, block, 0, s, p);
    });
    return hipGetLastError();
}

}  // namespace miw
