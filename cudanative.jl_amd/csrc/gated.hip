// The gated SiLU of the products' epilogue by itself, and its gradient: a pair (u, v) of neighbouring columns becomes
// a = u s v with s = 1 / (1 + exp(-u)), and da becomes du = da v s (1 + u (1 - s)), dv = da u s.
//
// Bound by HBM: forward 2 + 1 elements a pair, gradient 2 + 1 + 2, each touched once.  A lane takes four pairs: 16 bytes of Z, 8
// of A.  Everything between a load and its one rounding is Float32.  32768 rows of 2 x 4096 (bf16):
// 135 us forward (6.0 TB/s), 213 us gradient (6.3 TB/s); a copy of Z reaches 5.2 TB/s.
#include "experts.hpp"
#include "vec_types.hpp"

#include <type_traits>

namespace miw {

constexpr int GATED_THREADS = 256;

// Four elements, as load8 and store8 do eight.
template <class T, bool VECTOR, bool STREAM>
__device__ inline f32x4 load4(const T *p, int count)
{
    if constexpr (VECTOR) return __builtin_convertvector(load_vector<STREAM>((const vec<T, 4> *)p), f32x4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < count) v[e] = (float)p[e];
    return v;
}
template <class T, bool VECTOR, bool STREAM>
__device__ inline void store4(T *p, f32x4 v, int count)
{
    if constexpr (VECTOR) store_vector<STREAM>((vec<T, 4> *)p, __builtin_convertvector(v, vec<T, 4>));
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < count) p[e] = (T)v[e];
}

// 2^p.column_bits lanes of a workgroup lie along a row, the others along the rows.
template <class T, bool VECTOR, bool GRAD, bool STREAM>
__global__ __launch_bounds__(GATED_THREADS) void k_gated_silu(gated_params p)
{
    const int bits = p.column_bits;
    const long c = ((long)blockIdx.y * GATED_THREADS + (threadIdx.x & ((1 << bits) - 1))) * 8;
    if (c >= p.n) return;
    const int count = (int)min(8l, p.n - c);
    for (long row = ((long)blockIdx.x * GATED_THREADS + threadIdx.x) >> bits; row < p.rows; row += (long)gridDim.x * (GATED_THREADS >> bits)) {
        const f32x8 z = load8<T, VECTOR, STREAM>((const T *)p.Z + row * p.ldz + c, count);
        if constexpr (!GRAD) {
            f32x4 a;
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = gated_silu(z[2 * e], z[2 * e + 1]);
            store4<T, VECTOR, STREAM>((T *)p.out + row * p.ldo + c / 2, a, count / 2);
        } else {
            const f32x4 da = load4<T, VECTOR, STREAM>((const T *)p.dA + row * p.ldda + c / 2, count / 2);
            f32x8 dz;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float u = z[2 * e], v = z[2 * e + 1], s = 1.f / (1.f + __expf(-u));
                dz[2 * e] = da[e] * v * s * (1.f + u * (1.f - s));
                dz[2 * e + 1] = da[e] * u * s;
            }
            store8<T, VECTOR, STREAM>((T *)p.out + row * p.ldo + c, dz, count);
        }
    }
}

hipError_t launch_gated_silu(gated_params p, int dtype, hipStream_t s)
{
    const long pieces = (p.n + 7) / 8;
    p.column_bits = 0;
    while (p.column_bits < 8 && (1 << p.column_bits) < pieces) p.column_bits++;
    const long rows = GATED_THREADS >> p.column_bits, blocks = (p.rows + rows - 1) / rows;
    const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), (unsigned)((pieces + GATED_THREADS - 1) / GATED_THREADS)), block(GATED_THREADS);
    // Writing Z, A from it, reading A, dZ, reading dZ, 2 x 4096 columns (bf16), streamed and not: 439 and 477 us at 268 MB of Z, 225 and 240 at
    // 134 MB; 123 and 115 at 67 MB.
    const bool streams = p.vector && 2 * p.rows * p.n > STREAM_BYTES;
    auto go = [&](auto type) {
        using T = decltype(type);
        auto form = [&](auto grad) {
            constexpr bool GRAD = decltype(grad)::value;
            if (streams) hipLaunchKernelGGL((k_gated_silu<T, true, GRAD, true>), grid, block, 0, s, p);
            else if (p.vector) hipLaunchKernelGGL((k_gated_silu<T, true, GRAD, false>), grid, block, 0, s, p);
            else hipLaunchKernelGGL((k_gated_silu<T, false, GRAD, false>), grid, block, 0, s, p);
        };
        if (p.dA) form(std::true_type{});
        else form(std::false_type{});
    };
    if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
    return hipGetLastError();
}

}  // namespace miw
