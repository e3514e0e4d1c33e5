// Attention of one token of each env over the env's cached history, the token's own key and value written to the cache on the way.
//
// The cache is read once and nothing else is of its size, so the bytes bound it: every load is 16 bytes to a lane straight into the operands of the
// 16 x 8 x 16 matrix instruction, without shared memory: S^T = K Q^T and O^T = V^T P^T, the 8 columns being query heads of one key head. The order of a product's inner dimension is
// free as long as both operands agree, so a lane's 16 bytes of a key row stand for the values that the instruction wants of it in two steps; of V the lane holds 16
// bytes of four neighbouring keys' rows, pairs them up, and the rows of the result are taken in the order that this gives: 8 neighbouring columns of one head to a lane. Between the
// products P is transposed in registers, 8 x 8 at a time.
//
// With envs and key heads enough a warp has one of them to itself. Where they are too few to fill the GPU, an env's keys are dealt out over a block's
// warps, and over several blocks, evenly over the keys that the env has; the last block of an env to end joins their partial sums, always in the same order, so
// the same call gives the same bits.
//
// Measured, bf16, 8 heads, 2 of keys, dim 64: 4096 envs of up to 256 tokens 80 us, 5.2 TB/s of cached keys and values (0.79 of what a copy reaches; 89 us where the L2 holds what others wrote): a warp's
// loads under way are as many as its registers hold, and with at most 16 warps to an SM the memory idles between them (18 and 20 with spilled registers: 94 us).  One env of 8192 tokens 9.5 us, of which its 4 MB are 1: it is bound by the chain of launch, loads and join.
// The first tokens of an episode may have places of their own before the ring: which place a token takes is all that changes, the order of keys being free.
#include <cuda_runtime.h>
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"
#include "nkb_tcgen.cuh"

namespace nkb {

constexpr int kHistoryWarps = 4, kQueries = 8, kSplits = 32;
constexpr float kHistoryLog2e = 1.4426950408889634f;

struct HistoryParams {
    int64_t jobs, capacity, sinks, q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride;
    int heads_q, heads_k, dim, splits, parts;           // parts: sets of 8 query heads of a key head; jobs: envs x key heads x parts
    float scale2;
    const void *q, *k, *v;
    void *keys, *values, *out;
    const int32_t* position;
    uint32_t* arrived;                                  // per job; 0 between calls
    float* partial;                                     // per job and split: 8 x DP sums, 8 maxima, 8 totals
};

// WARPS: of a job and of a block. A warp with a job to itself is a block to itself, too: its place is then free when its own env's history ends, not the longest of four.
template <typename T, int DP, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (DP == 64 ? 4 : 3) * kHistoryWarps / WARPS) history_kernel(const HistoryParams p) {
    constexpr int SETS = DP == 64 ? 2 : 1, KEYS = 16 * SETS, CHUNKS = DP / 32, HALVES = DP / 64, ROW = DP + 2;
    __shared__ __align__(16) float sums[WARPS == 1 ? 1 : WARPS][kQueries][DP];
    __shared__ float tops[WARPS][kQueries], totals[WARPS][kQueries], weights[WARPS == 1 ? 1 : kSplits][kQueries];
    __shared__ uint32_t order;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, rank = WARPS == 1 ? 0 : warp;
    const int split = WARPS == 1 ? 0 : blockIdx.x % p.splits;
    const int64_t job = WARPS == 1 ? blockIdx.x : blockIdx.x / p.splits;
    const int part = (int)(job % p.parts), head = (int)(job / p.parts % p.heads_k);
    const int64_t env = job / p.parts / p.heads_k;
    const int group = p.heads_q / p.heads_k, queries = min(kQueries, group - part * kQueries), first = head * group + part * kQueries;
    const int32_t position = max(p.position[env], 0);
    // the first `sinks` tokens of an episode stay where they are, the others are a ring behind them
    const int slot = position < p.capacity ? position : (int)(p.sinks + (position - p.sinks) % (p.capacity - p.sinks)), held = (int)min((int64_t)position + 1, p.capacity);
    const int each = (held + p.splits * 16 - 1) / (p.splits * 16) * 16, begin = (int)min((int64_t)held, (int64_t)split * each), end = min(held, begin + each);

    const int64_t row = (int64_t)p.heads_k * p.dim;     // between an env's keys
    T* const keys = static_cast<T*>(p.keys) + env * p.capacity * row + (int64_t)head * p.dim;
    T* const values = static_cast<T*>(p.values) + env * p.capacity * row + (int64_t)head * p.dim;
    const T* const new_key = static_cast<const T*>(p.k) + env * p.k_stride + head * p.k_head_stride;
    const T* const new_value = static_cast<const T*>(p.v) + env * p.v_stride + head * p.v_head_stride;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);

    uint4 q[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        q[c] = g < queries && 32 * c + 8 * t < p.dim ? load_raw<T, 8>(static_cast<const T*>(p.q) + env * p.q_stride + (first + g) * p.q_head_stride + 32 * c + 8 * t) : none;

    // of the query heads 2 t and 2 t + 1; o[c][i]: columns 64 c + 8 g + 2 i and the next, of one head and the other
    float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, o[HALVES][4][4] = {};
    for (int base = begin + rank * KEYS; base < end; base += WARPS * KEYS) {
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
        float score[SETS][4] = {};                      // keys g and g + 8 of the two heads
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                mma16816<T>(score[s], k[s][0][c].x, k[s][1][c].x, k[s][0][c].y, k[s][1][c].y, q[c].x, q[c].y);
                mma16816<T>(score[s], k[s][0][c].z, k[s][1][c].z, k[s][0][c].w, k[s][1][c].w, q[c].z, q[c].w);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float best = top[h];
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float& x = score[s][2 * half + h];
                    if (base + 16 * s + 8 * half + g >= end) x = -INFINITY;
                    best = fmaxf(best, x);
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, d));
            const float by = best == top[h] ? 1.f : exp2_fast((top[h] - best) * p.scale2), shift = best == -INFINITY ? 0.f : best * p.scale2;
            top[h] = best;
            total[h] *= by;
#pragma unroll
            for (int c = 0; c < HALVES; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) { o[c][i][h] *= by; o[c][i][2 + h] *= by; }
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float& x = score[s][2 * half + h];
                    x = exp2_fast(fmaf(x, p.scale2, -shift));
                    total[h] += x;
                }
        }
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            // keys down, heads across -> heads down, keys 2 t and 2 t + 1 across, as the product's second operand
            const uint32_t b0 = transpose8(pack<T>(score[s][0], score[s][1])), b1 = transpose8(pack<T>(score[s][2], score[s][3]));
#pragma unroll
            for (int c = 0; c < HALVES; ++c) {
                const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&v[s][0][c]);
                const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&v[s][1][c]);
                const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&v[s][2][c]);
                const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&v[s][3][c]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma16816<T>(o[c][i], __byte_perm(v0[i], v1[i], 0x5410u), __byte_perm(v0[i], v1[i], 0x7632u), __byte_perm(v2[i], v3[i], 0x5410u), __byte_perm(v2[i], v3[i], 0x7632u), b0, b1);
            }
        }
    }
    // the slot is in one range of keys, and nobody reads it from the cache in this launch
    if (part == 0 && slot >= begin && slot < end)
        for (int c = WARPS == 1 ? lane : threadIdx.x; c < p.dim / 8; c += WARPS * 32) {
            *reinterpret_cast<uint4*>(keys + slot * row + 8 * c) = load_raw<T, 8>(new_key + 8 * c);
            *reinterpret_cast<uint4*>(values + slot * row + 8 * c) = load_raw<T, 8>(new_value + 8 * c);
        }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) total[h] += __shfl_xor_sync(~0u, total[h], d);
    T* const out = static_cast<T*>(p.out) + (env * p.heads_q + first) * p.dim;

    if constexpr (WARPS == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < HALVES; ++c)
                if (2 * t + h < queries && 64 * c + 8 * g < p.dim) {
                    const float by = 1.f / total[h];
                    float r[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { r[2 * i] = o[c][i][h] * by; r[2 * i + 1] = o[c][i][2 + h] * by; }
                    store<T, 8>(out + (2 * t + h) * p.dim + 64 * c + 8 * g, r);
                }
    } else {
        // the block's warps into one: a thread has four columns of a head
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (g == 0) { tops[warp][2 * t + h] = top[h]; totals[warp][2 * t + h] = total[h]; }
#pragma unroll
            for (int c = 0; c < HALVES; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(&sums[warp][2 * t + h][64 * c + 8 * g + 2 * i]) = make_float2(o[c][i][h], o[c][i][2 + h]);
        }
        __syncthreads();
        const bool alone = p.splits == 1;
        float* const partial = alone ? nullptr : p.partial + (job * p.splits + split) * (kQueries * ROW);
        auto give = [&](int h, int d, float4 sum, float all) {
            const float by = 1.f / all, r[4] = {sum.x * by, sum.y * by, sum.z * by, sum.w * by};
            if (h < queries && d < p.dim) store<T, 4>(out + h * p.dim + d, r);
        };
        auto join = [](float4& sum, float4 x, float by) {
            if (by != 0.f) { sum.x = fmaf(x.x, by, sum.x); sum.y = fmaf(x.y, by, sum.y); sum.z = fmaf(x.z, by, sum.z); sum.w = fmaf(x.w, by, sum.w); }
        };
        for (int x = threadIdx.x; x < kQueries * DP / 4; x += kHistoryWarps * 32) {
            const int h = x / (DP / 4), d = x % (DP / 4) * 4;
            float best = tops[0][h], all = 0.f;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) best = fmaxf(best, tops[w][h]);
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float by = tops[w][h] == -INFINITY ? 0.f : exp2_fast((tops[w][h] - best) * p.scale2);
                join(sum, *reinterpret_cast<const float4*>(&sums[w][h][d]), by);
                all = fmaf(totals[w][h], by, all);
            }
            if (alone) {
                give(h, d, sum, all);
            } else {
                *reinterpret_cast<float4*>(partial + h * DP + d) = sum;
                if (d == 0) { partial[kQueries * DP + h] = best; partial[kQueries * (DP + 1) + h] = all; }
            }
        }
        if (alone) return;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) order = atomicAdd(p.arrived + job, 1u);
        __syncthreads();
        if (order != (uint32_t)p.splits - 1u) return;
        __threadfence();
        // the env's blocks into one
        const float* const partials = p.partial + job * p.splits * (kQueries * ROW);
        for (int x = threadIdx.x; x < p.splits * kQueries; x += kHistoryWarps * 32) weights[x / kQueries][x % kQueries] = partials[x / kQueries * (kQueries * ROW) + kQueries * DP + x % kQueries];
        __syncthreads();
        for (int x = threadIdx.x; x < kQueries * DP / 4; x += kHistoryWarps * 32) {
            const int h = x / (DP / 4), d = x % (DP / 4) * 4;
            float best = -INFINITY, all = 0.f;
            for (int s = 0; s < p.splits; ++s) best = fmaxf(best, weights[s][h]);
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int s = 0; s < p.splits; ++s) {
                const float* const from = partials + s * (kQueries * ROW);
                const float by = weights[s][h] == -INFINITY ? 0.f : exp2_fast((weights[s][h] - best) * p.scale2);
                join(sum, *reinterpret_cast<const float4*>(from + h * DP + d), by);
                all = fmaf(from[kQueries * (DP + 1) + h], by, all);
            }
            give(h, d, sum, all);
        }
        if (threadIdx.x == 0) p.arrived[job] = 0u;
    }
}

__global__ void advance_kernel(int32_t* __restrict__ position, const uint8_t* __restrict__ fresh, int64_t envs) {
    const int64_t env = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (env < envs) position[env] = fresh != nullptr && fresh[env] != 0 ? 0 : max(position[env], -1) + 1;
}

cudaError_t launch_history_advance(int32_t* position, const uint8_t* fresh, int64_t envs, cudaStream_t stream) {
    if (envs != 0) advance_kernel<<<(unsigned)((envs + 127) / 128), 128, 0, stream>>>(position, fresh, envs);
    return cudaGetLastError();
}

static int64_t history_jobs(const nuka_b200_history_t& d) { return d.envs * d.heads_k * ((d.heads_q / d.heads_k + kQueries - 1) / kQueries); }
// A warp to itself where that gives every SM eight warps; else a block, and enough blocks for two to an SM, none with fewer than 128 keys of a full cache.
static bool history_by_warps(const nuka_b200_history_t& d) { return history_jobs(d) >= 8 * 148; }
static int history_splits(const nuka_b200_history_t& d) {
    if (history_by_warps(d)) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({(2 * 148 + history_jobs(d) - 1) / history_jobs(d), d.capacity / 128, kSplits}));
}

uint64_t history_workspace(const nuka_b200_history_t& d) {
    const int splits = history_splits(d);
    if (splits == 1) return 0u;
    const uint64_t jobs = (uint64_t)history_jobs(d);
    return (jobs * 4 + 255) / 256 * 256 + jobs * splits * kQueries * ((d.dim <= 64 ? 64 : 128) + 2) * 4;
}

template <typename T, int DP> static void run_history(const HistoryParams& p, bool by_warps, cudaStream_t stream) {
    if (by_warps) history_kernel<T, DP, 1><<<(unsigned)p.jobs, 32, 0, stream>>>(p);
    else history_kernel<T, DP, kHistoryWarps><<<(unsigned)(p.jobs * p.splits), kHistoryWarps * 32, 0, stream>>>(p);
}

cudaError_t launch_history(const nuka_b200_history_t& d, int64_t sinks, cudaStream_t stream) {
    if (d.envs == 0) return cudaSuccess;
    HistoryParams p{};
    p.jobs = history_jobs(d); p.capacity = d.capacity; p.sinks = sinks; p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride;
    p.v_stride = d.v_stride; p.v_head_stride = d.v_head_stride; p.heads_q = (int)d.heads_q; p.heads_k = (int)d.heads_k; p.dim = (int)d.dim; p.splits = history_splits(d);
    p.parts = (int)(p.jobs / d.envs / d.heads_k);
    p.scale2 = d.scale * kHistoryLog2e; p.q = d.q; p.k = d.k; p.v = d.v; p.keys = d.keys; p.values = d.values; p.out = d.out; p.position = d.position;
    if (p.splits > 1) {
        p.arrived = static_cast<uint32_t*>(d.workspace);
        p.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(d.workspace) + (p.jobs * 4 + 255) / 256 * 256);
    }
    const bool by_warps = history_by_warps(d);
    if (d.dtype == NUKA_B200_F16) d.dim <= 64 ? run_history<__half, 64>(p, by_warps, stream) : run_history<__half, 128>(p, by_warps, stream);
    else d.dim <= 64 ? run_history<__nv_bfloat16, 64>(p, by_warps, stream) : run_history<__nv_bfloat16, 128>(p, by_warps, stream);
    return cudaGetLastError();
}

}  // namespace nkb
