// The logistic function and its kin, for one value and for several, two to an instruction.
#pragma once
#include "nkb_tcgen.cuh"

namespace nkb {

// exp(-|u|) and 1 / (1 + it), of which the others are made. The exponent's product with log2(e) is rounded to 2^-24 of itself; EXACT adds what that lost. What is not a number has to come with a factor of its own.
struct Fading { float e, r; };
template <bool EXACT> __device__ __forceinline__ Fading fading(float u) {
    const float a = fminf(fabsf(u), 100.f), t = a * -1.4426950408889634f;
    Fading f;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(f.e) : "f"(t));
    if (EXACT) f.e = fmaf(f.e, fmaf(a, -1.4426950408889634f, -t) * 0.6931471805599453f + a * -1.33498e-8f, f.e);       // the last: what log2(e) lost, 1.92596e-8, times ln(2)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f.r) : "f"(1.f + f.e));
    return f;
}
__device__ __forceinline__ float logistic(float u, Fading f) { return u >= 0.f ? f.r : f.e * f.r; }
__device__ __forceinline__ float one_less(float u, Fading f) { return u >= 0.f ? f.e * f.r : f.r; }             // 1 - logistic(u)
// Where 16 bits are the result: 1 / (1 + exp(-s)) at once. The exponential may be infinite, and the result 0, as it has to be next to an s of that size.
__device__ __forceinline__ float logistic_fast(float s) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(s * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}
template <bool EXACT> __device__ __forceinline__ float silu(float s) { return s * (EXACT ? logistic(s, fading<true>(s)) : logistic_fast(s)); }
// log(1 + exp(u)) = max(u, 0) + log(1 + e), the latter by the series of 2 artanh(e / (2 + e)): its argument is 1/3 at most, the first term left out 2^-26 of the sum.
__device__ __forceinline__ float softplus(float u, Fading f) {
    float most, q;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(most) : "f"(u));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(2.f + f.e));
    const float z = f.e * q, s = z * z;
    const float series = fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, 1.f / 13.f, 1.f / 11.f), 1.f / 9.f), 1.f / 7.f), 1.f / 5.f), 1.f / 3.f), 1.f);
    return fmaf(z + z, series, most);
}

// ---- several values, two to an instruction ---------------------------------------------------------------------------------
__device__ __forceinline__ Pair both(float v) { return pair_of(v, v); }
__device__ __forceinline__ float inverse_of(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// logistic_fast of two values
__device__ __forceinline__ Pair logistic_pair(Pair s) {
    float a, b, x, y;
    split(mul_pair(s, both(-1.4426950408889634f)), a, b);
    split(add_pair(pair_of(exp2_fast(a), exp2_fast(b)), both(1.f)), x, y);
    return pair_of(inverse_of(x), inverse_of(y));
}
// s = silu(s)
template <bool EXACT, int N> __device__ __forceinline__ void silu_all(float (&s)[N]) {
    if constexpr (!EXACT && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const Pair v = pair_of(s[k], s[k + 1]);
            split(mul_pair(v, logistic_pair(v)), s[k], s[k + 1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] = silu<EXACT>(s[k]);
    }
}
// by *= silu'(s), and where `value` is given value *= silu(s)
template <bool EXACT, int N> __device__ __forceinline__ void by_silu_slope(const float (&s)[N], float (&by)[N], float* value = nullptr) {
    if constexpr (!EXACT && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const Pair v = pair_of(s[k], s[k + 1]), r = logistic_pair(v), slope = mul_pair(r, fma_pair(v, fma_pair(r, both(-1.f), both(1.f)), both(1.f)));
            if (value != nullptr) split(mul_pair(pair_of(value[k], value[k + 1]), mul_pair(v, r)), value[k], value[k + 1]);
            split(mul_pair(pair_of(by[k], by[k + 1]), slope), by[k], by[k + 1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const Fading f = fading<EXACT>(s[k]);
            const float r = logistic(s[k], f);
            if (value != nullptr) value[k] *= s[k] * r;
            by[k] *= r * fmaf(s[k], one_less(s[k], f), 1.f);
        }
    }
}
// softplus of u, and where `slope` is given logistic(u)
template <int N> __device__ __forceinline__ void softplus_all(const float (&u)[N], float (&to)[N], float* slope = nullptr) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            float x, y, m, n;
            // fading<true>, its sign turned round
            const Pair a = pair_of(fminf(fabsf(u[k]), 100.f), fminf(fabsf(u[k + 1]), 100.f)), t = mul_pair(a, both(1.4426950408889634f));
            split(t, x, y);
            Pair e = pair_of(exp2_fast(-x), exp2_fast(-y));
            e = fma_pair(e, fma_pair(fma_pair(a, both(-1.4426950408889634f), t), both(0.6931471805599453f), mul_pair(a, both(-1.33498e-8f))), e);
            if (slope != nullptr) {
                split(add_pair(e, both(1.f)), x, y);
                const Pair r = pair_of(inverse_of(x), inverse_of(y));
                split(r, x, y);
                split(mul_pair(e, r), m, n);
                slope[k] = u[k] >= 0.f ? x : m;
                slope[k + 1] = u[k + 1] >= 0.f ? y : n;
            }
            split(add_pair(e, both(2.f)), x, y);
            const Pair z = mul_pair(e, pair_of(inverse_of(x), inverse_of(y))), s = mul_pair(z, z);
            Pair series = fma_pair(s, both(1.f / 13.f), both(1.f / 11.f));
            series = fma_pair(s, series, both(1.f / 9.f));
            series = fma_pair(s, series, both(1.f / 7.f));
            series = fma_pair(s, series, both(1.f / 5.f));
            series = fma_pair(s, series, both(1.f / 3.f));
            series = fma_pair(s, series, both(1.f));
            asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(m) : "f"(u[k]));
            asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(n) : "f"(u[k + 1]));
            split(fma_pair(add_pair(z, z), series, pair_of(m, n)), to[k], to[k + 1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const Fading f = fading<true>(u[k]);
            if (slope != nullptr) slope[k] = logistic(u[k], f);
            to[k] = softplus(u[k], f);                  // which may be u
        }
    }
}

}  // namespace nkb
