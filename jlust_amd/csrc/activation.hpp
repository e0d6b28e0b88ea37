// activation.hpp -- the activations gelu and silu beside relu, and their slopes.
#pragma once

#include "common.hpp"

namespace jlust {

// The normal distribution's density factor e = exp(-z^2/2) and its integral up
// to z.  16-bit values: erfc(x) = t (a1 + t (a2 + ... )) exp(-x^2) with
// t = 1/(1 + p x) for x >= 0 (Abramowitz and Stegun 7.1.26, off by at most
// 1.5e-7, a 2,000th of bfloat16's rounding and a 300th of half's at 1/2; of the
// integral itself by 5e-4 at z = -4, 0.4 % at -6, where gelu is -6e-9, and 4 % at
// -13, the end of bfloat16's range); the others call erfc.  A tile's 32,768 calls of erfc would take as long as its
// matrix products at k = 1,000.
template <bool FAST, typename A>
__device__ __forceinline__ A normal_cdf(A z, A *e)
{
    if constexpr (FAST) {
        const float x = fabsf(z) * 0.70710678f;
        *e = __expf(-x * x);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
        const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f),
                                 0.254829592f);
        const float half = 0.5f * q * *e;
        return z < 0 ? half : 1.0f - half;
    } else {
        // erfc's relative error grows as twice its argument times the
        // argument's own error, so the product's rounding is added back:
        // erfc(x + r) = erfc(x) - 2/sqrt(pi) exp(-x^2) r.
        constexpr A C = A(-0.70710678118654752440);
        constexpr A C_LO = sizeof(A) == 8 ? A(4.8336466567264567e-17) : A(-0.70710678118654752440 - double(C));
        const A x = z * C, r = fma(z, C, -x) + z * C_LO, d = exp(-x * x);
        *e = d;
        const A c = erfc(x);
        return A(0.5) * (d > A(0) ? c - A(1.12837916709551257390) * d * r : c);
    }
}

template <bool FAST, typename A>
__device__ __forceinline__ A logistic(A z)
{
    if constexpr (FAST) return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    return A(1) / (A(1) + exp(-z));
}

template <bool FAST, typename A>
__device__ __forceinline__ A activate(int act, A z)
{
    A e;
    switch (act) {
    case JLUST_FN_RELU: return z > A(0) ? z : (z != z ? z : A(0));
    case JLUST_FN_GELU: return z * normal_cdf<FAST>(z, &e);
    case JLUST_FN_SILU: return z * logistic<FAST>(z);
    default: return z;
    }
}

// V of them, the kind asked for once.
template <bool FAST, int V, typename A>
__device__ __forceinline__ void activate_all(int act, A *z)
{
    switch (act) {
    case JLUST_FN_RELU:
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = activate<FAST>(JLUST_FN_RELU, z[e]);
        break;
    case JLUST_FN_GELU:
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = activate<FAST>(JLUST_FN_GELU, z[e]);
        break;
    case JLUST_FN_SILU:
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = activate<FAST>(JLUST_FN_SILU, z[e]);
        break;
    default: break;
    }
}

// The activation's derivative at z.
template <bool FAST, typename A>
__device__ __forceinline__ A activate_slope(int act, A z)
{
    A e;
    switch (act) {
    case JLUST_FN_RELU: return z > A(0) ? A(1) : (z != z ? z : A(0));
    case JLUST_FN_GELU: {
        const A c = normal_cdf<FAST>(z, &e);
        return c + z * e * A(0.39894228040143267794);
    }
    case JLUST_FN_SILU: {
        const A s = logistic<FAST>(z);
        return s + s * (z - z * s);
    }
    default: return A(1);
    }
}

}  // namespace jlust
