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

template <typename T, int N> __device__ __forceinline__ Raw<T, N> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, N>*>(p); }
template <typename T, int N> __device__ __forceinline__ void unpack(const Raw<T, N>& raw, float (&v)[N]) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = to_float<T>(e[k]);
}
template <typename T, int N> __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    Raw<T, N> raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = from_float<T>(v[k]);
    *reinterpret_cast<Raw<T, N>*>(p) = raw;
}

}  // namespace nkb
