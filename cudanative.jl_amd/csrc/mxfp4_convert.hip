// Microscaled 4-bit floating point: a matrix into codes and scales, and back.
//
// A lane has eight values of a block, four lanes the block, 32 lanes a row's piece of one panel of scales (256 values); the
// largest magnitude meets in the four lanes by data-parallel moves.  The scale is a power of two, so dividing by it is
// exact, and v_cvt_scalef32_pk_fp4_f32 rounds to the nearest code, ties to the even one, and saturates.
// Bound by HBM: a Float16 matrix is read once (2 bytes a value) and 17/32 of a byte written.  8192 x 8192 (Float16): 33 to 35 us
// (170 MB, 4.8 to 5.2 TB/s), back to bfloat16 25 us (170 MB, 6.8 TB/s: the codes are still in a cache).
#include "experts.hpp"
#include "vec_types.hpp"

namespace miw {

constexpr int CONVERT_THREADS = 256;

// 2^n for n in -127 .. 127.
__device__ inline float power_of_two(int n) { return __builtin_ldexpf(1.f, n); }

template <class T, bool VECTOR, bool STREAM>
__global__ __launch_bounds__(CONVERT_THREADS) void k_mxfp4_quantize(mxfp4_convert_params p)
{
    const long panels = (p.k + 255) / 256;
    const int sub = threadIdx.x & 31;  // place in the panel's piece: block sub / 4
    for (long unit = ((long)blockIdx.x * CONVERT_THREADS + threadIdx.x) >> 5; unit < panels * p.rows; unit += (long)gridDim.x * (CONVERT_THREADS / 32)) {
        const long row = unit / panels, panel = unit % panels;
        const long k0 = panel * 256 + sub * 8;
        const int count = (int)max(0l, min(8l, p.k - k0));
        f32x8 v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (count == 8) v = load8<T, VECTOR, STREAM>((const T *)p.in + row * p.ld + k0, 8);
        else if (count > 0) v = load8<T, false>((const T *)p.in + row * p.ld + k0, count);
        // Magnitudes as unsigned numbers have their order, infinities and NaN above all others.
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = v[e];  // (a bit cast of the vector's element itself takes element 0)
            most = max(most, __builtin_bit_cast(unsigned, x) & 0x7fffffffu);
        }
        most = max(most, (unsigned)__builtin_amdgcn_mov_dpp((int)most, 0xB1 /* quad_perm:[1,0,3,2] */, 0xf, 0xf, true));
        most = max(most, (unsigned)__builtin_amdgcn_mov_dpp((int)most, 0x4E /* quad_perm:[2,3,0,1] */, 0xf, 0xf, true));
        // floor(log2) - 2, biased by 127; below 2^-125 (Float32 subnormals among them) the smallest scale.
        const int field = (int)(most >> 23);
        const int scale = field == 255 ? 255 : max(field - 2, 0);
        unsigned codes = 0;
        if (scale != 255) {
            const float up = power_of_two(127 - scale);
            f32x8 w;
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = v[e] * up;
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, w[0], w[1], 1.f, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, w[2], w[3], 1.f, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, w[4], w[5], 1.f, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, w[6], w[7], 1.f, 3);
        }
        if (k0 / 32 * 32 < p.k) *(unsigned *)(p.codes + row * p.ldq + k0 / 2) = codes;
        // Four blocks' scales meet in the last lane of 16.
        unsigned word = (unsigned)scale << (8 * ((sub >> 2) & 3));
        word |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x114 /* row_shr:4 */, 0xf, 0xf, true);
        word |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x118 /* row_shr:8 */, 0xf, 0xf, true);
        if ((sub & 15) == 15) *(unsigned *)(p.scales + ((panel * p.lds + row) * 8 + (sub >> 4) * 4)) = word;
    }
}

template <class T, bool VECTOR, bool STREAM>
__global__ __launch_bounds__(CONVERT_THREADS) void k_mxfp4_dequantize(mxfp4_convert_params p)
{
    const long eights = (p.k + 7) / 8;
    for (long unit = (long)blockIdx.x * CONVERT_THREADS + threadIdx.x; unit < eights * p.rows; unit += (long)gridDim.x * CONVERT_THREADS) {
        const long row = unit / eights, k0 = unit % eights * 8;
        const int count = (int)min(8l, p.k - k0);
        const unsigned codes = *(const unsigned *)(p.codes + row * p.ldq + k0 / 2);
        const int scale = p.scales[((k0 >> 8) * p.lds + row) * 8 + ((k0 >> 5) & 7)];
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1),
                    c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
        const float by = scale == 255 ? __builtin_nanf("") : power_of_two(scale - 127);
        const f32x8 v = {a[0] * by, a[1] * by, b[0] * by, b[1] * by, c[0] * by, c[1] * by, d[0] * by, d[1] * by};
        T *to = (T *)p.out + row * p.ld + k0;
        if (count == 8) store8<T, VECTOR, STREAM>(to, v, 8);
        else store8<T, false>(to, v, count);
    }
}

template <class F>
static hipError_t typed(int dtype, F go)
{
    if (dtype == TYPE_F32) go(float{});
    else if (dtype == TYPE_F16) go(f16_t{});
    else go(bf16_t{});
    return hipGetLastError();
}
// The matrix streams past the caches, codes and scales stay.  Writing X, its codes, reading them, back, reading that, 8192 columns (bf16),
// streamed and not: 338 and 387 us at 268 MB of X, 178 and 195 at 134 MB; 101 and 99 at 67 MB.
template <class T>
static bool streams(const mxfp4_convert_params &p) { return p.vector && (long)sizeof(T) * p.rows * p.k > STREAM_BYTES; }

static dim3 convert_grid(long threads)
{
    const long blocks = (threads + CONVERT_THREADS - 1) / CONVERT_THREADS;
    return dim3((unsigned)(blocks < 256 * 64 ? blocks : 256 * 64));
}

hipError_t launch_mxfp4_quantize(const mxfp4_convert_params &p, int dtype, hipStream_t s)
{
    const dim3 grid = convert_grid((p.k + 255) / 256 * 32 * p.rows), block(CONVERT_THREADS);
    return typed(dtype, [&](auto type) {
        using T = decltype(type);
        if (streams<T>(p)) hipLaunchKernelGGL((k_mxfp4_quantize<T, true, true>), grid, block, 0, s, p);
        else if (p.vector) hipLaunchKernelGGL((k_mxfp4_quantize<T, true, false>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_mxfp4_quantize<T, false, false>), grid, block, 0, s, p);
    });
}

hipError_t launch_mxfp4_dequantize(const mxfp4_convert_params &p, int dtype, hipStream_t s)
{
    const dim3 grid = convert_grid((p.k + 7) / 8 * p.rows), block(CONVERT_THREADS);
    return typed(dtype, [&](auto type) {
        using T = decltype(type);
        if (streams<T>(p)) hipLaunchKernelGGL((k_mxfp4_dequantize<T, true, true>), grid, block, 0, s, p);
        else if (p.vector) hipLaunchKernelGGL((k_mxfp4_dequantize<T, true, false>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((k_mxfp4_dequantize<T, false, false>), grid, block, 0, s, p);
    });
}

}  // namespace miw
