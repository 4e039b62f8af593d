// Element types, vector loads and activations shared by the layer kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "turbinator/training/hip_layers.h"

namespace layer {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Raw storage of B bytes, loaded and stored in one instruction.
template <int B>
struct Raw;
template <>
struct Raw<16> { typedef u32x4 type; };
template <>
struct Raw<8> { typedef u32x2 type; };
template <>
struct Raw<4> { typedef unsigned type; };
template <>
struct Raw<2> { typedef unsigned short type; };

// B bytes of elements of type T as floats and back, rounded to nearest even.
template <class T, int B>
struct Vec {
    static constexpr int n = B / (int)sizeof(T);
    typedef typename Raw<B>::type raw;
    typedef T elems __attribute__((ext_vector_type(n)));
    typedef float floats __attribute__((ext_vector_type(n)));

    static __device__ __forceinline__ void unpack(raw r, float (&v)[n]) {
        const floats f = __builtin_convertvector(__builtin_bit_cast(elems, r), floats);
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = f[i];
    }
    static __device__ __forceinline__ raw pack(const float (&v)[n]) {
        floats f;
#pragma unroll
        for (int i = 0; i < n; ++i) f[i] = v[i];
        return __builtin_bit_cast(raw, __builtin_convertvector(f, elems));
    }
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLow = 1.92596299112661887e-8f;  // log2(e) - kLog2e
constexpr float kLn2 = 0.69314718055994530942f;

// e^x.  v_exp_f32 is 2^x to 1 ulp; the rounding of x log2(e) alone would cost
// |x| 2^-24, which a result rounded to 16 bits does not show.  With FINE the
// product's remainder r is put back as the factor 1 + r ln 2, which keeps
// about 2 ulp while e^x and its inverse are normal.
template <bool FINE>
__device__ __forceinline__ float exp_of(float x) {
    const float p = x * kLog2e;
    const float e = __builtin_amdgcn_exp2f(p);
    if constexpr (!FINE) return e;
    const float r = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -p));
    // Further out e may be 0 or inf and r NaN.
    return __builtin_fabsf(p) < 126.0f ? fmaf(e, r * kLn2, e) : e;
}

// 1 / (1 + e^-z); v_rcp_f32 is within 1 ulp.
template <bool FINE>
__device__ __forceinline__ float sigmoid_of(float z) {
    return __builtin_amdgcn_rcpf(1.0f + exp_of<FINE>(-z));
}

// The normal distribution below z, and e^(-z^2/2) on the way.  Below 0 it is
// erfc(|z| / sqrt 2) / 2 in the form e^(-z^2/2) t P(t), t = 1 / (1 + 0.21 |z|)
// (Abramowitz and Stegun 7.1.26's, with a longer P): relative digits stay as
// far as the result is a normal number, where 1 + erf(z / sqrt 2) cancels (4%
// of GELU off at -5, all of it from -6 on).  P is the polynomial of degree 8
// with the least relative error, 0.2 units of 2^-24, for |z| up to 13.3, from
// where on the exponential is 0 or subnormal; with it the result is within 12
// units for z above -3 and z^2 (16-bit results: 2 z^2) further out.
// 4,096 x 1,024 x 64 bf16 through GELU in group norm, forward: 292 us, and 451
// with erfcf; gradient of 1,024 x 2,048 x 64: 318 and 505.
struct Normal {
    float below, bell;
};
template <bool FINE>
__device__ __forceinline__ Normal normal_of(float z) {
    const float bell = exp_of<FINE>(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.21f, __builtin_fabsf(z), 1.0f));
    float p = -0.072194494f;
    p = fmaf(p, t, 0.2862464f);
    p = fmaf(p, t, -0.3358655f);
    p = fmaf(p, t, 0.35600975f);
    p = fmaf(p, t, -0.09866595f);
    p = fmaf(p, t, 0.12699148f);
    p = fmaf(p, t, 0.068616636f);
    p = fmaf(p, t, 0.085155666f);
    p = fmaf(p, t, 0.083706014f);
    const float tail = p * t * bell;
    return {z < 0.0f ? tail : 1.0f - tail, bell};
}

template <bool FINE, int ACT>
__device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == TB_HIP_ACT_SILU) return z * sigmoid_of<FINE>(z);
    if constexpr (ACT == TB_HIP_ACT_GELU) return z * normal_of<FINE>(z).below;
    return z;
}

// The derivative of act_of.
template <bool FINE, int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == TB_HIP_ACT_SILU) {
        const float s = sigmoid_of<FINE>(z);
        return fmaf(z, fmaf(-s, s, s), s);
    }
    if constexpr (ACT == TB_HIP_ACT_GELU) {
        const Normal n = normal_of<FINE>(z);
        return fmaf(z, 0.39894228040143267794f * n.bell, n.below);
    }
    return 1.0f;
}

// Sum over the wave's lanes up to this one: shifts within sixteen lanes, then
// the last lane of the rows before.
__device__ __forceinline__ int running_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 15, 15, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 15, 15, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 15, 15, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 15, 15, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 10, 15, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 12, 15, false);
}

// Calls f with the activation as a compile-time constant.
template <int N>
struct Int {
    static constexpr int value = N;
};
template <class F>
inline void with_act(int act, F f) {
    if (act == TB_HIP_ACT_SILU)
        f(Int<TB_HIP_ACT_SILU>());
    else if (act == TB_HIP_ACT_GELU)
        f(Int<TB_HIP_ACT_GELU>());
    else
        f(Int<TB_HIP_ACT_NONE>());
}

// The value of the lane `N` to the left within its sixteen lanes, around.
template <int N>
__device__ __forceinline__ int rotated(int v) {
    return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 15, 15, true);
}

// f over v and the value of the partner 16 or 32 lanes away.
template <class F>
__device__ __forceinline__ int across(int v, bool far, F f) {
    const auto r = far ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                       : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f((int)r[0], (int)r[1]);
}

template <class T>
constexpr bool kFine = sizeof(T) == 4;

__host__ __device__ inline int type_size(int dtype) { return dtype == TB_HIP_F32 ? 4 : 2; }
inline bool known_type(int dtype) {
    return dtype == TB_HIP_F32 || dtype == TB_HIP_BF16 || dtype == TB_HIP_F16;
}
inline bool known_act(int act) { return act >= TB_HIP_ACT_NONE && act <= TB_HIP_ACT_GELU; }
inline bool multiple_of(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace layer
