// Gradients of an episode's first keys and values (sinks) from the queries that are too far away to see the keys around them: what the kernels of nkb_sinks.cu leave for the keys' kernel.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "nkb_sequence.h"

namespace nkb {

constexpr int kSinkRows = 8;                            // sinks of a product

// What there is to add to a row of 32-bit sums.
struct FarRow {
    const float* at = nullptr;
    // to columns c to c + 31
    __device__ __forceinline__ void add(uint32_t (&r)[32], int c) const {
        if (at == nullptr) return;
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(at + c + k);
            r[k] = __float_as_uint(__uint_as_float(r[k]) + v.x); r[k + 1] = __float_as_uint(__uint_as_float(r[k + 1]) + v.y);
            r[k + 2] = __float_as_uint(__uint_as_float(r[k + 2]) + v.z); r[k + 3] = __float_as_uint(__uint_as_float(r[k + 3]) + v.w);
        }
    }
};

// A tile of keys has far queries where its last key's episode has sinks in it and goes on behind what the window reaches; tiles with `least` of them have a slot, the keys' kernel works out the others itself.
struct FarSinks {
    int slots = 0, groups = 0, heads_k = 0, least = 1;             // slots: at most; groups: of kSinkRows sinks
    int64_t jobs = 0;                                   // there is room for, slots x groups x heads_k or more
    int32_t *slot_of = nullptr, *tile_of = nullptr, *count = nullptr;           // of tiles, of slots, and how many; behind it into how many parts each one's far queries are split
    float* sums = nullptr;                              // slots x groups x heads_k x splits x 2 x kSinkRows x DP: of keys, then values, not scaled; the splits joined in the first
    // Of row `row` of the tile's sinks.
    __device__ __forceinline__ FarRow row_of(int tile, int row, int head, int which, int dp) const {
        FarRow r;
        if (slots == 0 || row < 0 || row >= groups * kSinkRows) return r;
        const int slot = slot_of[tile];
        if (slot < 0) return r;
        r.at = sums + ((((int64_t)slot * groups + row / kSinkRows) * heads_k + head) * count[1] * 2 + which) * (kSinkRows * dp) + row % kSinkRows * dp;
        return r;
    }
};

uint64_t far_sinks_bytes(const nuka_b200_attention_t& d, int64_t sinks, int span, int tiles);
FarSinks far_sinks(const nuka_b200_attention_t& d, int64_t sinks, int span, int tiles, void* workspace);
cudaError_t launch_far_sinks(const nuka_b200_attention_t& d, int window, int sinks, int span, int tiles, int64_t pitch, const FarSinks& far, cudaStream_t stream);

}  // namespace nkb
