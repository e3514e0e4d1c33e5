// Loads, stores and small pieces that the sequence kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace nkb {

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = unsigned short; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
template <typename T, int N> using Raw = typename RawOf<sizeof(T) * N>::type;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// two 16-bit values at a time, the first one the low half (a recurrence of 131071 x 1024 in 161 and 270 us so, 178 and 285 with one at a time)
template <typename T> __device__ __forceinline__ float2 two_floats(uint32_t v);
template <> __device__ __forceinline__ float2 two_floats<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <> __device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ uint32_t two_of(float low, float high);
template <> __device__ __forceinline__ uint32_t two_of<__half>(float low, float high) { const __half2 v = __floats2half2_rn(low, high); return *reinterpret_cast<const uint32_t*>(&v); }
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float low, float high) { const __nv_bfloat162 v = __floats2bfloat162_rn(low, high); return *reinterpret_cast<const uint32_t*>(&v); }

template <typename T, int N> __device__ __forceinline__ Raw<T, N> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, N>*>(p); }
template <typename T, int N> __device__ __forceinline__ void unpack(const Raw<T, N>& raw, float (&v)[N]) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        const uint32_t* e = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float2 two = two_floats<T>(e[k / 2]);
            v[k] = two.x;
            v[k + 1] = two.y;
        }
    } else {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = to_float<T>(e[k]);
    }
}
template <typename T, int N> __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    Raw<T, N> raw;
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        uint32_t* e = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
        for (int k = 0; k < N; k += 2) e[k / 2] = two_of<T>(v[k], v[k + 1]);
    } else {
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int k = 0; k < N; ++k) e[k] = from_float<T>(v[k]);
    }
    *reinterpret_cast<Raw<T, N>*>(p) = raw;
}

// ---- logistic function and its kin -------------------------------------------------------------------------------------
// exp(-|u|) and 1 / (1 + it), of which the others are made. The exponent's product with log2(e) is rounded to 2^-24 of itself; EXACT adds what that lost. What is not a number has to come with a factor of its own.
struct Fading { float e, r; };
template <bool EXACT> __device__ __forceinline__ Fading fading(float u) {
    const float a = fminf(fabsf(u), 100.f), t = a * -1.4426950408889634f;
    Fading f;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(f.e) : "f"(t));
    if (EXACT) f.e = fmaf(f.e, fmaf(a, -1.4426950408889634f, -t) * 0.6931471805599453f + a * -1.3352e-8f, f.e);       // the last: log2(e)'s own rounding, 1.9263e-8, times ln(2)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f.r) : "f"(1.f + f.e));
    return f;
}
__device__ __forceinline__ float logistic(float u, Fading f) { return u >= 0.f ? f.r : f.e * f.r; }
__device__ __forceinline__ float one_less(float u, Fading f) { return u >= 0.f ? f.e * f.r : f.r; }             // 1 - logistic(u)
// Where 16 bits are the result: 1 / (1 + exp(-s)) at once, the exponential kept finite.
__device__ __forceinline__ float logistic_fast(float s) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(s * -1.4426950408889634f, 126.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}
template <bool EXACT> __device__ __forceinline__ float silu(float s) { return s * (EXACT ? logistic(s, fading<true>(s)) : logistic_fast(s)); }
template <bool EXACT> __device__ __forceinline__ float silu_slope(float s) {
    if (!EXACT) {
        const float r = logistic_fast(s);
        return r * fmaf(s, 1.f - r, 1.f);
    }
    const Fading f = fading<true>(s);
    return logistic(s, f) * fmaf(s, one_less(s, f), 1.f);
}
// log(1 + exp(u)) = max(u, 0) + log(1 + e), the latter by the series of 2 artanh(e / (2 + e)): its argument is 1/3 at most, the first term left out 2^-26 of the sum.
__device__ __forceinline__ float softplus(float u, Fading f) {
    float most, q;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(most) : "f"(u));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(2.f + f.e));
    const float z = f.e * q, s = z * z;
    const float series = fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, 1.f / 13.f, 1.f / 11.f), 1.f / 9.f), 1.f / 7.f), 1.f / 5.f), 1.f / 3.f), 1.f);
    return fmaf(z + z, series, most);
}

}  // namespace nkb
