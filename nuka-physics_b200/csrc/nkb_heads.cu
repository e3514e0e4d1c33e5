// Norms of queries and keys for each head, with the rotation of positions in the same pass.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

// A token's heads are dim / 8 neighbouring lanes' work (rounded up to a power of two, LANES), one head after the other, the next ones' loads under way; a warp has 32 / LANES
// tokens. A lane holds 8 columns of each head, four whole pairs: with interleaved pairs 8 neighbouring columns, else 4 columns of the first half of
// the turned part and their partners in the second, so that no value crosses lanes and a lane works out the sines and cosines of its four pairs once for all heads of the token;
// columns behind the turned part lie as they are.
//
// Measured: 98304 tokens x 10 heads x 64, bf16, 63 us forwards (4.0 TB/s of its bytes) and 112 back (3.4 TB/s); 49999 x 20 x 128, f16, 108 us (4.7 TB/s) and 168 (4.6 TB/s).
// A value costs some ten instructions forwards and sixteen back, 2.9 and 2.5 of which are issued a cycle and SM (of 4), and the memory is 40 % busy: forwards the instructions leave no more of
// it, backwards the rows ahead, which fill the registers, leave 35 % of the warps' places in use.  Two values to an instruction need registers that are not there (128 and 204 us back).
constexpr int kThreads = 128;
constexpr int64_t kBlocksBack = 6 * 148;                // at most: they take their tokens in turn, and the weights' partial sums are as many

struct HeadsParams {
    const int32_t *first, *positions;
    const double* frequencies;
    int64_t tokens;
    int heads_q, heads_k, dim, turned;
    const void *q, *k;
    int64_t q_stride, q_head_stride, k_stride, k_head_stride;
    const float *q_weight, *k_weight;
    float eps;
    void *q_out, *k_out;
    const void *dq_out, *dk_out;
    void *dq, *dk;
    float* partial;                                     // blocks x 2 x dim, null where no weight's gradient is wanted
};

// EXACT: angles are products in 64 bits; a build of its own, since both forms in one cost the other's registers (49999 x 20 x 128: 346 us in place of 287)
template <typename T, int LANES, bool INTERLEAVED, bool BACKWARD, bool EXACT>
__global__ void __launch_bounds__(kThreads, BACKWARD ? (sizeof(T) == 4 ? 4 : 6) : sizeof(T) == 4 ? 8 : 10) heads_kernel(const HeadsParams p) {
    constexpr int TOKENS = kThreads / LANES;
    using R = Raw<T, 4>;
    const int group = threadIdx.x % LANES, half = p.turned / 2;
    const bool live = group * 8 < p.dim, turns = group * 8 < p.turned, split = turns && !INTERLEAVED;
    const int low = split ? group * 4 : group * 8, high = split ? half + group * 4 : group * 8 + 4;
    const float inverse = 1.f / (float)p.dim;
    float dw[2][BACKWARD ? 8 : 1] = {};

    // every lane makes every turn of every loop: the sums below go over a token's lanes
    for (int64_t t0 = (int64_t)blockIdx.x * TOKENS; t0 < p.tokens; t0 += (int64_t)gridDim.x * TOKENS) {
        const int64_t own = t0 + threadIdx.x / LANES, t = min(own, p.tokens - 1);
        const bool in = live && own < p.tokens;
        // the token's rows, queries first, and behind them its keys
        struct Row { R x[2], d[BACKWARD ? 2 : 1]; };
        const T *const q = static_cast<const T*>(p.q) + t * p.q_stride, *const k = static_cast<const T*>(p.k) + t * p.k_stride;
        auto fetch = [&](Row& r, int h) {
            const bool keys = h >= p.heads_q;
            const int i = keys ? h - p.heads_q : h;
            if (!in || i >= (keys ? p.heads_k : p.heads_q)) return;
            const T* const x = keys ? k + i * p.k_head_stride : q + i * p.q_head_stride;
            r.x[0] = load_raw<T, 4>(x + low);
            r.x[1] = load_raw<T, 4>(x + high);
            if constexpr (BACKWARD) {
                const T* const d = keys ? static_cast<const T*>(p.dk_out) + (t * p.heads_k + i) * p.dim : static_cast<const T*>(p.dq_out) + (t * p.heads_q + i) * p.dim;
                r.d[0] = load_raw<T, 4>(d + low);
                r.d[1] = load_raw<T, 4>(d + high);
            }
        };
        Row now{}, next{};
        fetch(now, 0);
        fetch(next, 1);
        float cosine[4], sine[4];
        const int32_t position = p.turned == 0 ? 0 : p.positions != nullptr ? p.positions[t] : (int32_t)(t - p.first[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cosine[i] = 1.f;
            sine[i] = 0.f;
            if (turns) {
                // The angle is the product in 32 bits unless asked otherwise, as programs have it that keep it in 32 bits: what they trained fits.  Of that angle in turns, taken
                // in 64 bits, only the fraction is kept, so its sine and cosine are exact to 32 bits however large it is.
                const double frequency = p.frequencies[group * 4 + i];
                double angle = (EXACT ? (double)position * frequency : (double)((float)position * (float)frequency)) * 0.15915494309189533577;
                angle -= rint(angle);
                sincospif(2.f * (float)angle, &sine[i], &cosine[i]);
            }
        }
#pragma unroll
        for (int keys = 0; keys < 2; ++keys) {
            const int heads = keys ? p.heads_k : p.heads_q;
            T* to = static_cast<T*>(BACKWARD ? (keys ? p.dk : p.dq) : (keys ? p.k_out : p.q_out)) + t * heads * p.dim;
            const float* const weight = keys ? p.k_weight : p.q_weight;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = weight != nullptr && live ? weight[i < 4 ? low + i : high + i - 4] : 1.f;
            // the body once, two rows ahead: four rows at a time, unrolled, outgrow the instruction cache (152 us in place of 106 forwards at 49999 x 20 x 128, f16)
#pragma unroll 1
            for (int h = 0; h < heads; ++h, to += p.dim) {
                Row after{};
                fetch(after, (keys ? p.heads_q : 0) + h + 2);
                float v[8], d[8];
                float (&v0)[4] = reinterpret_cast<float(&)[4]>(v[0]), (&v1)[4] = reinterpret_cast<float(&)[4]>(v[4]);
                float (&d0)[4] = reinterpret_cast<float(&)[4]>(d[0]), (&d1)[4] = reinterpret_cast<float(&)[4]>(d[4]);
                unpack<T, 4>(now.x[0], v0);             // zeros where the lane has no row
                unpack<T, 4>(now.x[1], v1);
                float square = 0.f, dot = 0.f;
                if constexpr (BACKWARD) {
                    unpack<T, 4>(now.d[0], d0);
                    unpack<T, 4>(now.d[1], d1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {       // the gradient turns back
                        float &a = d[INTERLEAVED ? 2 * i : i], &b = d[INTERLEAVED ? 2 * i + 1 : 4 + i];
                        const float a0 = a;
                        a = a0 * cosine[i] + b * sine[i];
                        b = b * cosine[i] - a0 * sine[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    square = fmaf(v[i], v[i], square);
                    if constexpr (BACKWARD) dot = fmaf(v[i], d[i] * w[i], dot);
                }
#pragma unroll
                for (int s = LANES / 2; s > 0; s >>= 1) {
                    square += __shfl_xor_sync(~0u, square, s);
                    if constexpr (BACKWARD) dot += __shfl_xor_sync(~0u, dot, s);
                }
                const float r = rsqrtf(fmaf(square, inverse, p.eps));
                if constexpr (BACKWARD) {
                    // dx = r (e - y mean(y e)) with y = x r, which stays within 32 bits where r^3 does not
                    const float pull = r * (dot * inverse);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float y = in ? v[i] * r : 0.f;        // without eps r is infinite where there is no row
                        dw[keys][i] = fmaf(d[i], y, dw[keys][i]);
                        d[i] = fmaf(-y, pull, d[i] * w[i]) * r;
                    }
                    if (in) { store<T, 4>(to + low, d0); store<T, 4>(to + high, d1); }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &a = v[INTERLEAVED ? 2 * i : i], &b = v[INTERLEAVED ? 2 * i + 1 : 4 + i];
                        const float a0 = a;
                        a = a0 * cosine[i] - b * sine[i];
                        b = a0 * sine[i] + b * cosine[i];
                    }
                    if (in) { store<T, 4>(to + low, v0); store<T, 4>(to + high, v1); }
                }
                now = next;
                next = after;
            }
        }
    }
    if constexpr (BACKWARD) {
        if (p.partial == nullptr) return;
        // every thread's sums into one per column, always in the same order
        __shared__ float sums[kThreads / 32][LANES * 8];
        for (int which = 0; which < 2; ++which) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float s = which ? dw[1][k] : dw[0][k];
#pragma unroll
                for (int d = 16; d >= LANES; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
                if (threadIdx.x % 32 < LANES) sums[threadIdx.x / 32][(split ? (k < 4 ? low + k : high + k - 4) : group * 8 + k)] = s;
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.dim; c += kThreads) {
                float s = 0.f;
                for (int w = 0; w < kThreads / 32; ++w) s += sums[w][c];
                p.partial[((int64_t)blockIdx.x * 2 + which) * p.dim + c] = s;
            }
            __syncthreads();
        }
    }
}

// The blocks' partial sums into the weights' gradients: a block per 32 columns, its 32 warps take every 32nd partial sum.
__global__ void __launch_bounds__(1024) weight_kernel(const float* __restrict__ partial, int blocks, int dim, float* dq_weight, float* dk_weight) {
    __shared__ float sums[32][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = blockIdx.x * 32 + lane, which = blockIdx.y;
    float* out = which ? dk_weight : dq_weight;
    if (out == nullptr) return;
    float s = 0.f;
    if (c < dim)
#pragma unroll 8
        for (int b = warp; b < blocks; b += 32) s += partial[((int64_t)b * 2 + which) * dim + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < dim) {
        for (int w = 1; w < 32; ++w) s += sums[w][lane];
        out[c] = s;
    }
}

// Tokens of a block's pass are kThreads / LANES; forwards every block has one.
static int64_t lanes_of(int64_t dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }
static int64_t blocks_of(int64_t tokens, int64_t dim, bool backward) {
    const int64_t blocks = (tokens * lanes_of(dim) + kThreads - 1) / kThreads;
    return backward ? std::min(blocks, kBlocksBack) : blocks;
}

uint64_t heads_workspace(int64_t tokens, int64_t dim) { return (uint64_t)(blocks_of(tokens, dim, true) * 2 * dim * 4); }

template <typename T, int LANES, bool INTERLEAVED> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    HeadsParams p{};
    p.first = d.first; p.positions = d.positions; p.frequencies = d.frequencies; p.tokens = d.tokens;
    p.heads_q = (int)d.heads_q; p.heads_k = (int)d.heads_k; p.dim = (int)d.dim; p.turned = (int)d.turned;
    p.q = d.q; p.k = d.k; p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride;
    p.q_weight = d.q_weight; p.k_weight = d.k_weight; p.eps = d.eps; p.q_out = d.q_out; p.k_out = d.k_out;
    p.dq_out = d.dq_out; p.dk_out = d.dk_out; p.dq = d.dq; p.dk = d.dk;
    const unsigned blocks = (unsigned)blocks_of(d.tokens, d.dim, backward);
    const bool exact = (d.interleaved & NUKA_B200_EXACT_ANGLES) != 0;
    if (!backward) {
        exact ? heads_kernel<T, LANES, INTERLEAVED, false, true><<<blocks, kThreads, 0, stream>>>(p) : heads_kernel<T, LANES, INTERLEAVED, false, false><<<blocks, kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const bool weights = d.dq_weight != nullptr || d.dk_weight != nullptr;
    p.partial = weights ? static_cast<float*>(d.workspace) : nullptr;
    exact ? heads_kernel<T, LANES, INTERLEAVED, true, true><<<blocks, kThreads, 0, stream>>>(p) : heads_kernel<T, LANES, INTERLEAVED, true, false><<<blocks, kThreads, 0, stream>>>(p);
    if (weights) weight_kernel<<<dim3((unsigned)((d.dim + 31) / 32), 2), 1024, 0, stream>>>(p.partial, (int)blocks, p.dim, d.dq_weight, d.dk_weight);
    return cudaGetLastError();
}

template <typename T, int LANES> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    return (d.interleaved & ~NUKA_B200_EXACT_ANGLES) != 0 ? run_heads<T, LANES, true>(d, backward, stream) : run_heads<T, LANES, false>(d, backward, stream);
}

template <typename T> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    const int64_t lanes = lanes_of(d.dim);
    return lanes == 4 ? run_heads<T, 4>(d, backward, stream) : lanes == 8 ? run_heads<T, 8>(d, backward, stream) : lanes == 16 ? run_heads<T, 16>(d, backward, stream) : run_heads<T, 32>(d, backward, stream);
}

cudaError_t launch_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    if (d.tokens == 0) {
        if (backward && d.dq_weight != nullptr) cudaMemsetAsync(d.dq_weight, 0, d.dim * 4, stream);
        if (backward && d.dk_weight != nullptr) cudaMemsetAsync(d.dk_weight, 0, d.dim * 4, stream);
        return cudaGetLastError();
    }
    return d.dtype == NUKA_B200_F32 ? run_heads<float>(d, backward, stream) : d.dtype == NUKA_B200_F16 ? run_heads<__half>(d, backward, stream) : run_heads<__nv_bfloat16>(d, backward, stream);
}

}  // namespace nkb
