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

// c += a b of 16 x 16 and 16 x 8, and 8 x 8 values of 16 bits turned over, a warp's each
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

}  // namespace nkb
