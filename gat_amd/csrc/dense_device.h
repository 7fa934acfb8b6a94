// Device-side building blocks of the dense operators (linear.hip, group_norm.hip, embedding.hip,
// dropout.hip): element types, vector access at element alignment, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/gat_mi355.h"
#include "attn_device.h"

namespace gatmi {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <int V> struct VecF { float e[V]; };

// V elements as one access.  The address only needs the element's own alignment: rows of odd widths and
// sliced tensors start anywhere, and a global load or store of up to 16 bytes takes that as it is.
template <class T, int V> __device__ __forceinline__ VecF<V> ldv(const T *p) {
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef vec uvec __attribute__((aligned(sizeof(T))));
    VecF<V> r;
    if constexpr (V == 1) {
        r.e[0] = (float)p[0];
    } else {
        const vec v = *reinterpret_cast<const uvec *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) r.e[i] = (float)v[i];
    }
    return r;
}
// f32 -> T rounds to nearest even, once
template <class T, int V> __device__ __forceinline__ void stv(T *p, const VecF<V> &r) {
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef vec uvec __attribute__((aligned(sizeof(T))));
    if constexpr (V == 1) {
        p[0] = (T)r.e[0];
    } else {
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)r.e[i];
        *reinterpret_cast<uvec *>(p) = v;
    }
}

// Division of a 32-bit number by a divisor fixed at launch: one high multiply instead of a division
// (round-up multiplier with the carry kept in the shift, exact for every 32-bit numerator).
struct FastDiv {
    uint32_t d, m, s;
};
inline FastDiv make_fast_div(uint32_t d) {
    FastDiv f;
    f.d = d;
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) ++l;
    f.m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
    f.s = l;
    return f;
}
__device__ __forceinline__ uint32_t fdiv(const FastDiv &f, uint32_t n) {
    const uint32_t t = __umulhi(f.m, n);
    return f.s == 0 ? n : (t + ((n - t) >> 1)) >> (f.s - 1);
}

// ---- activations: value and derivative at z, f32.  EXACT: to a few steps of f32, for f32 tensors.  Otherwise
// (results are rounded to 16 bits) v_exp_f32 and v_rcp_f32 forms, whose error of at most 2^-17 of the value is small
// beside that rounding (2^-11 for f16, 2^-8 for bf16), where the value itself is small too.
template <bool EXACT> __device__ __forceinline__ float act_exp(float v) {
    if constexpr (EXACT) return expf(v);   // of either sign
    return __builtin_amdgcn_exp2f(v * 1.44269502162933349609375f);
}

// exp(z) for z <= 0, to a few of its own steps down to the smallest normal number, then 0; NaN for NaN.  EXACT: as exp_fast, whose
// end at -87 applies to the correction alone here.
template <bool EXACT> __device__ __forceinline__ float act_exp_neg(float z) {
    if constexpr (!EXACT) return act_exp<false>(z);
    const float L2E = 1.44269502162933349609375f, L2E_LO = 1.925963033500011e-8f;
    const float c = fmaxf(z, -87.0f);
    const float r = fmaf(c, L2E_LO, fmaf(c, L2E, -(c * L2E)));
    const float e = __builtin_amdgcn_exp2f(z * L2E);
    return fmaf(e, r * 0.693147182464599609375f, e);
}

// exp(z) - 1 for z <= 0, from exp(z)
template <bool EXACT> __device__ __forceinline__ float act_expm1(float z, float e) {
    if constexpr (EXACT) {
        // above -0.35 the series to z^8 / 8! (what follows is below 2^-30 of the sum); below it exp(z) <= 0.705
        // and the subtraction leaves an error of exp's own 1.5 steps of at most 2^-24 against 0.295 or more
        float s = fmaf(z, 2.4801587e-5f, 1.9841270e-4f);
        s = fmaf(z, s, 1.3888889e-3f);
        s = fmaf(z, s, 8.3333333e-3f);
        s = fmaf(z, s, 4.1666668e-2f);
        s = fmaf(z, s, 1.6666667e-1f);
        s = fmaf(z, s, 0.5f);
        s = fmaf(z * z, s, z);
        return z < -0.35f ? e - 1.0f : s;      // NaN: s
    }
    // next to 0 the subtraction would cancel: z + z^2/2 + z^3/6, off by z^3/24 relative, 2^-19.7 at -0.03
    const float s = z * fmaf(z, fmaf(z, 0.16666667f, 0.5f), 1.0f);
    return z < -0.03f ? e - 1.0f : s;
}

// The normal distribution function, its lower tail relative to itself, not as 1 + erf, which is nothing where erf
// rounds to -1 and has lost half its digits by z = -3: exp(-z^2/2) times a polynomial in t = 1 / (1 + p |z|), fitted to
// erfc(a) exp(a^2) / 2 (a = |z| / sqrt 2, up to 10) for the smallest relative error.  EXACT: degree 9, 2^-25.6, with
// 1 / (1 + p |z|) corrected by its residual and z^2 by what its rounding left; 8 f32 steps in all (the library's erfc
// costs twice the arithmetic: group norm with GELU of [100000, 8 x 30] f32 52 us forward).  16-bit results: degree 6,
// 2^-17.9; v_exp adds z^2 2^-24 of its argument's rounding.  `gauss` = exp(-z^2/2).
template <bool EXACT> __device__ __forceinline__ float act_phi(float z, float &gauss) {
    float tail;
    if constexpr (EXACT) {
        const float a = fminf(fabsf(z), 20.0f);                 // the tail is 0 from 14.2 on; a^2 stays finite
        const float h = a * a, e = act_exp_neg<true>(-0.5f * h);
        gauss = fmaf(-0.5f * fmaf(a, a, -h), e, e);
        float t = __builtin_amdgcn_rcpf(fmaf(0.26870057f, a, 1.0f));
        t = fmaf(t, fmaf(-(t * a), 0.26870057f, 1.0f - t), t);
        float q = fmaf(t, 0.0294948481f, -0.131197944f);
        q = fmaf(t, q, 0.18205376f);
        q = fmaf(t, q, -0.0808761716f);
        q = fmaf(t, q, 0.115118489f);
        q = fmaf(t, q, 0.0692774951f);
        q = fmaf(t, q, 0.101966202f);
        q = fmaf(t, q, 0.106957726f);
        q = fmaf(t, q, 0.1072056f);
        tail = q * t * gauss;
    } else {
        gauss = act_exp<false>(-0.5f * z * z);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.308308125f, fabsf(z), 1.0f));
        float q = fmaf(t, -0.07528124f, 0.188420862f);
        q = fmaf(t, q, 0.00836186484f);
        q = fmaf(t, q, 0.136160269f);
        q = fmaf(t, q, 0.119097903f);
        q = fmaf(t, q, 0.123238377f);
        tail = q * t * gauss;
    }
    return z > 0.f ? 1.0f - tail : tail;
}

template <int ACT, bool EXACT> __device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == GATMI_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if constexpr (ACT == GATMI_ACT_ELU) return z > 0.f ? z : act_expm1<EXACT>(z, act_exp_neg<EXACT>(z));
    if constexpr (ACT == GATMI_ACT_SILU) {
        const float d = 1.0f + act_exp<EXACT>(-z);   // +inf for z far below 0: the quotient is -0
        return EXACT ? z / d : z * __builtin_amdgcn_rcpf(d);
    }
    if constexpr (ACT == GATMI_ACT_GELU) {
        float g;
        return z * act_phi<EXACT>(z, g);
    }
    return z;
}

// (value, derivative)
template <int ACT, bool EXACT> __device__ __forceinline__ float act_both(float z, float &d) {
    if constexpr (ACT == GATMI_ACT_RELU) {
        d = z > 0.f ? 1.f : (z != z ? z : 0.f);
        return z > 0.f ? z : (z != z ? z : 0.f);
    }
    if constexpr (ACT == GATMI_ACT_ELU) {
        const float e = act_exp_neg<EXACT>(z);
        d = z > 0.f ? 1.f : e;            // not (exp(z) - 1) + 1, which is good to a step of 1 only
        return z > 0.f ? z : act_expm1<EXACT>(z, e);
    }
    if constexpr (ACT == GATMI_ACT_SILU) {
        const float q = 1.0f + act_exp<EXACT>(-z);
        const float s = EXACT ? 1.0f / q : __builtin_amdgcn_rcpf(q);
        d = s * (1.0f + z * (1.0f - s));
        return EXACT ? z / q : z * s;
    }
    if constexpr (ACT == GATMI_ACT_GELU) {
        float g;
        const float phi = act_phi<EXACT>(z, g);
        d = fmaf(z * 0.3989422804014327f, g, phi);
        return z * phi;
    }
    d = 1.f;
    return z;
}

template <class T> struct IsF32 { static constexpr bool value = false; };
template <> struct IsF32<float> { static constexpr bool value = true; };

// f(integral_constant V) for a vector of v elements: 16 bytes, or less where a row is shorter
template <class T, class F> void with_vec(int v, F f) {
    constexpr int VM = 16 / sizeof(T);
    if (v == VM) f(std::integral_constant<int, VM>{});
    else if (v == 1) f(std::integral_constant<int, 1>{});
    else if (v == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
}
// the widest vector, in elements, that a row of n elements takes
inline int vec_of(int dtype, long long n) {
    int v = dtype == GATMI_F32 ? 4 : 8;
    while (v > n) v >>= 1;
    return v;
}

}  // namespace gatmi

// Runs BODY with `T` bound to the element type of a GATMI_F32 / _BF16 / _F16 code (checked before).
#define GATMI_WITH_TYPE(code, ...)                                                        \
    do {                                                                                  \
        if ((code) == GATMI_F32) { using T = float; __VA_ARGS__; }                        \
        else if ((code) == GATMI_BF16) { using T = gatmi::bf16_t; __VA_ARGS__; }          \
        else { using T = gatmi::f16_t; __VA_ARGS__; }                                     \
    } while (0)

// ... and with `ACT` bound to an activation code
#define GATMI_WITH_ACT(code, ...)                                                         \
    do {                                                                                  \
        switch (code) {                                                                   \
        case GATMI_ACT_RELU: { constexpr int ACT = GATMI_ACT_RELU; __VA_ARGS__; break; }  \
        case GATMI_ACT_ELU: { constexpr int ACT = GATMI_ACT_ELU; __VA_ARGS__; break; }    \
        case GATMI_ACT_SILU: { constexpr int ACT = GATMI_ACT_SILU; __VA_ARGS__; break; }  \
        case GATMI_ACT_GELU: { constexpr int ACT = GATMI_ACT_GELU; __VA_ARGS__; break; }  \
        default: { constexpr int ACT = GATMI_ACT_NONE; __VA_ARGS__; break; }              \
        }                                                                                 \
    } while (0)
