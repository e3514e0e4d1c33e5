// Attention of one token of each env over the env's cached history, the token's own key and value written to the cache on the way.
//
// The cache is read once and nothing else is of its size, so the bytes bound it: every load is 16 bytes to a lane straight into the operands of the
// 16 x 8 x 16 matrix instruction, without shared memory.  The order of a product's inner dimension is free as long as both operands agree, so a lane's 16 bytes of a key
// row stand for the four values that the instruction wants of it in each of two steps; for P V the lane holds 16 bytes of four neighbouring keys' rows and pairs them up,
// and the columns of the result are taken in the order that this gives.  The query heads of a key head are the instruction's 16 rows.
//
// An env's keys are dealt out over the block's warps and, where there are too few envs and key heads to fill the GPU, over several blocks, evenly
// over the keys that the env has.  The last block of an env to end joins their partial sums, in the order of the blocks, so the same call gives the same bits.
#include <cuda_runtime.h>
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"
#include "nkb_tcgen.cuh"

namespace nkb {

constexpr int kHistoryWarps = 4, kQueries = 16;
constexpr float kHistoryLog2e = 1.4426950408889634f;

struct HistoryParams {
    int64_t envs, capacity, q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride;
    int heads_q, heads_k, dim, splits, parts;           // parts: sets of 16 query heads of a key head
    float scale2;
    const void *q, *k, *v;
    void *keys, *values, *out;
    const int32_t* position;
    uint32_t* arrived;                                  // per env, key head and part; 0 between calls
    float* partial;                                     // per env, key head, part and split: 16 x (DP + 2)
};

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(kHistoryWarps * 32) history_kernel(const HistoryParams p) {
    constexpr int SETS = DP == 64 ? 2 : 1, KEYS = 16 * SETS, CHUNKS = DP / 32, COLUMNS = DP / 8, HALVES = DP / 64;
    __shared__ float sums[kHistoryWarps][kQueries][DP], tops[kHistoryWarps][kQueries], totals[kHistoryWarps][kQueries];
    __shared__ uint32_t order;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % p.splits;
    const int64_t job = blockIdx.x / p.splits;          // env, key head, part
    const int part = (int)(job % p.parts), head = (int)(job / p.parts % p.heads_k);
    const int64_t env = job / p.parts / p.heads_k;
    const int group = p.heads_q / p.heads_k, queries = min(kQueries, group - part * kQueries);
    const int32_t position = max(p.position[env], 0);
    const int slot = (int)(position % p.capacity), held = (int)min((int64_t)position + 1, p.capacity);
    const int each = (held + p.splits * 16 - 1) / (p.splits * 16) * 16, begin = min(held, split * each), end = min(held, begin + each);

    const int64_t row = (int64_t)p.heads_k * p.dim;     // between an env's keys
    T* const keys = static_cast<T*>(p.keys) + env * p.capacity * row + (int64_t)head * p.dim;
    T* const values = static_cast<T*>(p.values) + env * p.capacity * row + (int64_t)head * p.dim;
    const T* const new_key = static_cast<const T*>(p.k) + env * p.k_stride + head * p.k_head_stride;
    const T* const new_value = static_cast<const T*>(p.v) + env * p.v_stride + head * p.v_head_stride;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);

    uint4 q[CHUNKS][2];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int h = g + 8 * half;
            q[c][half] = h < queries && 32 * c + 8 * t < p.dim
                             ? load_raw<T, 8>(static_cast<const T*>(p.q) + env * p.q_stride + (head * group + part * kQueries + h) * p.q_head_stride + 32 * c + 8 * t) : none;
        }

    float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, o[COLUMNS][4] = {};
    for (int base = begin + warp * KEYS; base < end; base += kHistoryWarps * KEYS) {
        uint4 k[SETS][2][CHUNKS], v[SETS][4][HALVES];
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int key = base + 16 * s + 8 * half + g;
                const T* from = key == slot ? new_key : keys + key * row;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) k[s][half][c] = key < end && 32 * c + 8 * t < p.dim ? load_raw<T, 8>(from + 32 * c + 8 * t) : none;
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int key = base + 16 * s + 2 * t + (n & 1) + (n >> 1) * 8;
                const T* from = key == slot ? new_value : values + key * row;
                // keys that the env does not have are zeros: whatever an earlier episode left there meets no product
#pragma unroll
                for (int c = 0; c < HALVES; ++c) v[s][n][c] = key < end && 64 * c + 8 * g < p.dim ? load_raw<T, 8>(from + 64 * c + 8 * g) : none;
            }
        }
        float score[SETS][2][4] = {};
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    mma16816<T>(score[s][half], q[c][0].x, q[c][1].x, q[c][0].y, q[c][1].y, k[s][half][c].x, k[s][half][c].y);
                    mma16816<T>(score[s][half], q[c][0].z, q[c][1].z, q[c][0].w, q[c][1].w, k[s][half][c].z, k[s][half][c].w);
                }
#pragma unroll
        for (int r = 0; r < 2; ++r) {                   // query heads g and g + 8
            float best = top[r];
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = score[s][half][2 * r + e];
                        if (base + 16 * s + 8 * half + 2 * t + e >= end) x = -INFINITY;
                        best = fmaxf(best, x);
                    }
            best = fmaxf(best, __shfl_xor_sync(~0u, best, 1));
            best = fmaxf(best, __shfl_xor_sync(~0u, best, 2));
            const float by = best == top[r] ? 1.f : exp2_fast((top[r] - best) * p.scale2), shift = best == -INFINITY ? 0.f : best * p.scale2;
            top[r] = best;
            total[r] *= by;
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) { o[c][2 * r] *= by; o[c][2 * r + 1] *= by; }
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = score[s][half][2 * r + e];
                        x = exp2_fast(fmaf(x, p.scale2, -shift));
                        total[r] += x;
                    }
        }
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            const uint32_t a0 = pack<T>(score[s][0][0], score[s][0][1]), a1 = pack<T>(score[s][0][2], score[s][0][3]);
            const uint32_t a2 = pack<T>(score[s][1][0], score[s][1][1]), a3 = pack<T>(score[s][1][2], score[s][1][3]);
#pragma unroll
            for (int c = 0; c < HALVES; ++c) {
                const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&v[s][0][c]);
                const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&v[s][1][c]);
                const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&v[s][2][c]);
                const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&v[s][3][c]);
#pragma unroll
                for (int m = 0; m < 8; ++m) {
                    const uint32_t which = m & 1 ? 0x7632u : 0x5410u;
                    mma16816<T>(o[8 * c + m], a0, a1, a2, a3, __byte_perm(v0[m / 2], v1[m / 2], which), __byte_perm(v2[m / 2], v3[m / 2], which));
                }
            }
        }
    }
    // the slot is in one split's range, and nobody reads it from the cache in this launch
    if (part == 0 && slot >= begin && slot < end) {
        for (int c = threadIdx.x; c < p.dim / 8; c += blockDim.x) {
            *reinterpret_cast<uint4*>(keys + slot * row + 8 * c) = load_raw<T, 8>(new_key + 8 * c);
            *reinterpret_cast<uint4*>(values + slot * row + 8 * c) = load_raw<T, 8>(new_value + 8 * c);
        }
    }

    // the block's warps into one
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        total[r] += __shfl_xor_sync(~0u, total[r], 1);
        total[r] += __shfl_xor_sync(~0u, total[r], 2);
        const int h = g + 8 * r;
        if (t == 0) { tops[warp][h] = top[r]; totals[warp][h] = total[r]; }
#pragma unroll
        for (int c = 0; c < HALVES; ++c)
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                sums[warp][h][64 * c + 16 * t + m] = o[8 * c + m][2 * r];
                sums[warp][h][64 * c + 16 * t + 8 + m] = o[8 * c + m][2 * r + 1];
            }
    }
    __syncthreads();
    const bool alone = p.splits == 1;
    float* const partial = alone ? nullptr : p.partial + (job * p.splits + split) * (kQueries * (DP + 2));
    for (int x = threadIdx.x; x < queries * DP; x += blockDim.x) {
        const int h = x / DP, d = x % DP;
        float best = tops[0][h];
#pragma unroll
        for (int w = 1; w < kHistoryWarps; ++w) best = fmaxf(best, tops[w][h]);
        float sum = 0.f, all = 0.f;
#pragma unroll
        for (int w = 0; w < kHistoryWarps; ++w) {
            const float by = tops[w][h] == -INFINITY ? 0.f : exp2_fast((tops[w][h] - best) * p.scale2);
            sum = by == 0.f ? sum : fmaf(sums[w][h][d], by, sum);
            all = fmaf(totals[w][h], by, all);
        }
        if (!alone) {
            partial[h * (DP + 2) + d] = sum;
            if (d == 0) { partial[h * (DP + 2) + DP] = best; partial[h * (DP + 2) + DP + 1] = all; }
        } else if (d < p.dim) {
            static_cast<T*>(p.out)[(env * p.heads_q + head * group + part * kQueries + h) * p.dim + d] = from_float<T>(sum / all);
        }
    }
    if (alone) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) order = atomicAdd(p.arrived + job, 1u);
    __syncthreads();
    if (order != (uint32_t)p.splits - 1u) return;
    __threadfence();
    const float* all_partials = p.partial + job * p.splits * (kQueries * (DP + 2));
    for (int x = threadIdx.x; x < queries * DP; x += blockDim.x) {
        const int h = x / DP, d = x % DP;
        float best = -INFINITY;
        for (int s = 0; s < p.splits; ++s) best = fmaxf(best, all_partials[(s * kQueries + h) * (DP + 2) + DP]);
        float sum = 0.f, all = 0.f;
        for (int s = 0; s < p.splits; ++s) {
            const float* from = all_partials + (s * kQueries + h) * (DP + 2);
            const float by = from[DP] == -INFINITY ? 0.f : exp2_fast((from[DP] - best) * p.scale2);
            sum = by == 0.f ? sum : fmaf(from[d], by, sum);
            all = fmaf(from[DP + 1], by, all);
        }
        if (d < p.dim) static_cast<T*>(p.out)[(env * p.heads_q + head * group + part * kQueries + h) * p.dim + d] = from_float<T>(sum / all);
    }
    if (threadIdx.x == 0) p.arrived[job] = 0u;
}

__global__ void advance_kernel(int32_t* __restrict__ position, const uint8_t* __restrict__ fresh, int64_t envs) {
    const int64_t env = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (env < envs) position[env] = fresh != nullptr && fresh[env] != 0 ? 0 : max(position[env], -1) + 1;
}

cudaError_t launch_history_advance(int32_t* position, const uint8_t* fresh, int64_t envs, cudaStream_t stream) {
    if (envs != 0) advance_kernel<<<(unsigned)((envs + 127) / 128), 128, 0, stream>>>(position, fresh, envs);
    return cudaGetLastError();
}

static int history_parts(const nuka_b200_history_t& d) { return (int)((d.heads_q / d.heads_k + kQueries - 1) / kQueries); }
// Enough blocks for four to an SM, none with fewer than 64 keys of a full cache.
static int history_splits(const nuka_b200_history_t& d) {
    const int64_t jobs = d.envs * d.heads_k * history_parts(d);
    return (int)std::max<int64_t>(1, std::min<int64_t>((592 + jobs - 1) / jobs, d.capacity / 64));
}

uint64_t history_workspace(const nuka_b200_history_t& d) {
    const int splits = history_splits(d);
    if (splits == 1) return 0u;
    const uint64_t jobs = (uint64_t)(d.envs * d.heads_k * history_parts(d));
    return (jobs * 4 + 255) / 256 * 256 + jobs * splits * kQueries * ((d.dim <= 64 ? 64 : 128) + 2) * 4;
}

template <typename T, int DP> static void run_history(const HistoryParams& p, int64_t blocks, cudaStream_t stream) {
    history_kernel<T, DP><<<(unsigned)blocks, kHistoryWarps * 32, 0, stream>>>(p);
}

cudaError_t launch_history(const nuka_b200_history_t& d, cudaStream_t stream) {
    if (d.envs == 0) return cudaSuccess;
    HistoryParams p{};
    p.envs = d.envs; p.capacity = d.capacity; p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride;
    p.v_stride = d.v_stride; p.v_head_stride = d.v_head_stride; p.heads_q = (int)d.heads_q; p.heads_k = (int)d.heads_k; p.dim = (int)d.dim; p.splits = history_splits(d); p.parts = history_parts(d);
    p.scale2 = d.scale * kHistoryLog2e; p.q = d.q; p.k = d.k; p.v = d.v; p.keys = d.keys; p.values = d.values; p.out = d.out; p.position = d.position;
    const int64_t jobs = d.envs * d.heads_k * p.parts;
    if (p.splits > 1) {
        p.arrived = static_cast<uint32_t*>(d.workspace);
        p.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(d.workspace) + (jobs * 4 + 255) / 256 * 256);
    }
    const int64_t blocks = jobs * p.splits;
    if (d.dtype == NUKA_B200_F16) d.dim <= 64 ? run_history<__half, 64>(p, blocks, stream) : run_history<__half, 128>(p, blocks, stream);
    else d.dim <= 64 ? run_history<__nv_bfloat16, 64>(p, blocks, stream) : run_history<__nv_bfloat16, 128>(p, blocks, stream);
    return cudaGetLastError();
}

}  // namespace nkb
