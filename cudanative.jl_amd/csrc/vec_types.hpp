// Element types of the experts' operators on the device: loads and stores of eight elements, conversions to and from Float32.
#pragma once
#include <hip/hip_runtime.h>

namespace miw {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <class T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// A whole vector; STREAM: the caches are told that it is not used again soon.
template <bool STREAM, class V>
__device__ inline V load_vector(const V *p)
{
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool STREAM, class V>
__device__ inline void store_vector(V *p, V v)
{
    if constexpr (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
}

// Eight consecutive elements as Float32; VECTOR: one or two 16-byte loads, otherwise `count` single ones and zeros behind them.
template <class T, bool VECTOR, bool STREAM = false>
__device__ inline f32x8 load8(const T *p, int count)
{
    if constexpr (VECTOR) {
        if constexpr (sizeof(T) == 2) {
            return __builtin_convertvector(load_vector<STREAM>((const vec<T, 8> *)p), f32x8);
        } else {
            const f32x4 a = load_vector<STREAM>((const f32x4 *)p), b = load_vector<STREAM>((const f32x4 *)p + 1);
            return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    } else {
        f32x8 v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < count) v[e] = (float)p[e];
        return v;
    }
}
// Rounded to T (nearest, ties to even) and stored.
template <class T, bool VECTOR, bool STREAM = false>
__device__ inline void store8(T *p, f32x8 v, int count)
{
    if constexpr (VECTOR) {
        if constexpr (sizeof(T) == 2) {
            store_vector<STREAM>((vec<T, 8> *)p, __builtin_convertvector(v, vec<T, 8>));
        } else {
            store_vector<STREAM>((f32x4 *)p, f32x4{v[0], v[1], v[2], v[3]});
            store_vector<STREAM>((f32x4 *)p + 1, f32x4{v[4], v[5], v[6], v[7]});
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < count) p[e] = (T)v[e];
    }
}

// The gate of a gated SiLU times its value.  __expf scales its argument in one rounding: the result is off by |gate| 2^-24 of itself and a few units
// more, twenty of Float32's last place at a gate of -40, as much as half a unit of the gate, a rounded sum, makes; the rounding to 16 bits that mostly follows
// is far above that.  Gates below -88.7 give zeros.
__device__ inline float gated_silu(float gate, float value) { return gate / (1.f + __expf(-gate)) * value; }

// Reductions over a wavefront by data-parallel primitives: no LDS, some fifty cycles.  The result is uniform.
__device__ inline unsigned wave_max(unsigned v)
{
#define MIW_STEP(ctrl, rows) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, true))
    MIW_STEP(0x111, 0xf);  // from the lane 1, 2, 4, 8 below in a row of 16
    MIW_STEP(0x112, 0xf);
    MIW_STEP(0x114, 0xf);
    MIW_STEP(0x118, 0xf);
    MIW_STEP(0x142, 0xa);  // from the last lane of the row below
    MIW_STEP(0x143, 0xc);  // from lane 31
#undef MIW_STEP
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ inline float wave_sum(float v)
{
#define MIW_STEP(ctrl, rows) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, true))
    MIW_STEP(0x111, 0xf);
    MIW_STEP(0x112, 0xf);
    MIW_STEP(0x114, 0xf);
    MIW_STEP(0x118, 0xf);
    MIW_STEP(0x142, 0xa);
    MIW_STEP(0x143, 0xc);
#undef MIW_STEP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// Sum over this lane and those below it.
__device__ inline int wave_scan(int v)
{
#define MIW_STEP(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, true)
    MIW_STEP(0x111, 0xf);
    MIW_STEP(0x112, 0xf);
    MIW_STEP(0x114, 0xf);
    MIW_STEP(0x118, 0xf);
    MIW_STEP(0x142, 0xa);
    MIW_STEP(0x143, 0xc);
#undef MIW_STEP
    return v;
}

}  // namespace miw
