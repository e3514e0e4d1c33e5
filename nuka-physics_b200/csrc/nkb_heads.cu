// Norms of queries and keys for each head, with the rotation of positions in the same pass.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

// A head's dim columns are taken in groups of 8 by dim / 8 neighbouring lanes (rounded up to a power of two, LANES), as many heads side by side as a
// warp has room for.  A group holds four whole pairs: with interleaved pairs 8 neighbouring columns, else 4 columns of the first half of
// the turned part and their partners in the second, so that no value crosses lanes; columns behind the turned part lie as they are.
// The angles' sines and cosines are worked out once per token into shared memory, for all of its heads.
constexpr int kTokens = 16;                             // of a block's pass
constexpr int kThreads = 256;
constexpr int64_t kBlocks = 592;                        // at most, four to an SM: they take their tokens in turn, and the weights' partial sums are as many

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

template <typename T, int LANES, bool INTERLEAVED, bool BACKWARD>
__device__ void turn_rows(const HeadsParams& p, const float2* angles, int64_t t0, int count, bool keys, float (&dw)[8]) {
    constexpr int ROWS = kThreads / LANES, AHEAD = BACKWARD ? 2 : 4;
    const int group = threadIdx.x % LANES, half = p.turned / 2;
    const bool live = group * 8 < p.dim, turns = group * 8 < p.turned, split = turns && !INTERLEAVED;
    const int low = split ? group * 4 : group * 8, high = split ? half + group * 4 : group * 8 + 4;
    const int heads = keys ? p.heads_k : p.heads_q, rows = count * heads;
    const T* x = static_cast<const T*>(keys ? p.k : p.q);
    const T* dy = static_cast<const T*>(keys ? p.dk_out : p.dq_out);
    T* y = static_cast<T*>(BACKWARD ? (keys ? p.dk : p.dq) : (keys ? p.k_out : p.q_out));
    const int64_t stride = keys ? p.k_stride : p.q_stride, head_stride = keys ? p.k_head_stride : p.q_head_stride;
    const float* weight = keys ? p.k_weight : p.q_weight;
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = weight != nullptr && live ? weight[k < 4 ? low + k : high + k - 4] : 1.f;
    const float inverse = 1.f / (float)p.dim;
    // every lane makes every turn of the loop: the sums below go over a row's lanes
    for (int base = threadIdx.x / LANES; base - (int)threadIdx.x / LANES < rows; base += ROWS * AHEAD) {
        Raw<T, 4> rx[AHEAD][2], rd[BACKWARD ? AHEAD : 1][2];
        int token[AHEAD];
        int64_t to[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int row = base + a * ROWS;
            token[a] = row / heads;
            const int head = row - token[a] * heads;
            to[a] = ((t0 + token[a]) * heads + head) * p.dim;
            if (row < rows && live) {
                const T* from = x + (t0 + token[a]) * stride + head * head_stride;
                rx[a][0] = load_raw<T, 4>(from + low);
                rx[a][1] = load_raw<T, 4>(from + high);
                if (BACKWARD) {
                    rd[a][0] = load_raw<T, 4>(dy + to[a] + low);
                    rd[a][1] = load_raw<T, 4>(dy + to[a] + high);
                }
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const bool in = base + a * ROWS < rows && live;
            float v[8], d[8];
            float (&v0)[4] = reinterpret_cast<float(&)[4]>(v[0]), (&v1)[4] = reinterpret_cast<float(&)[4]>(v[4]);
            float (&d0)[4] = reinterpret_cast<float(&)[4]>(d[0]), (&d1)[4] = reinterpret_cast<float(&)[4]>(d[4]);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = d[k] = 0.f;
            if (in) {
                unpack<T, 4>(rx[a][0], v0);
                unpack<T, 4>(rx[a][1], v1);
                if (BACKWARD) {
                    unpack<T, 4>(rd[a][0], d0);
                    unpack<T, 4>(rd[a][1], d1);
                }
            }
            float2 turn[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) turn[k] = make_float2(1.f, 0.f);
            if (in && turns)
#pragma unroll
                for (int k = 0; k < 4; ++k) turn[k] = angles[token[a] * half + group * 4 + k];
            if (BACKWARD)
#pragma unroll
                for (int k = 0; k < 4; ++k) {           // the gradient turns back
                    float &u = d[INTERLEAVED ? 2 * k : k], &s = d[INTERLEAVED ? 2 * k + 1 : 4 + k];
                    const float u0 = u;
                    u = u0 * turn[k].x + s * turn[k].y;
                    s = s * turn[k].x - u0 * turn[k].y;
                }
            float square = 0.f, dot = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                square = fmaf(v[k], v[k], square);
                if (BACKWARD) dot = fmaf(v[k], d[k] * w[k], dot);
            }
#pragma unroll
            for (int s = LANES / 2; s > 0; s >>= 1) {
                square += __shfl_xor_sync(~0u, square, s);
                if (BACKWARD) dot += __shfl_xor_sync(~0u, dot, s);
            }
            const float r = rsqrtf(fmaf(square, inverse, p.eps));
            if (BACKWARD) {
                const float pull = r * r * r * (dot * inverse);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    dw[k] = fmaf(d[k], v[k] * r, dw[k]);
                    d[k] = fmaf(d[k] * w[k], r, -v[k] * pull);
                }
                if (in) { store<T, 4>(y + to[a] + low, d0); store<T, 4>(y + to[a] + high, d1); }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = v[k] * r * w[k];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float &u = v[INTERLEAVED ? 2 * k : k], &s = v[INTERLEAVED ? 2 * k + 1 : 4 + k];
                    const float u0 = u;
                    u = u0 * turn[k].x - s * turn[k].y;
                    s = u0 * turn[k].y + s * turn[k].x;
                }
                if (in) { store<T, 4>(y + to[a] + low, v0); store<T, 4>(y + to[a] + high, v1); }
            }
        }
    }
}

template <typename T, int LANES, bool INTERLEAVED, bool BACKWARD>
__global__ void __launch_bounds__(kThreads) heads_kernel(const HeadsParams p) {
    __shared__ float2 angles[kTokens * 128];
    __shared__ float sums[kThreads / 32][LANES * 8];
    const int half = p.turned / 2;
    float dw[2][8] = {};
    for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < p.tokens; t0 += (int64_t)gridDim.x * kTokens) {
        const int count = (int)min((int64_t)kTokens, p.tokens - t0);
        for (int k = threadIdx.x; k < count * half; k += kThreads) {
            const int token = k / half;
            const int64_t t = t0 + token;
            const int32_t position = p.positions != nullptr ? p.positions[t] : (int32_t)(t - p.first[t]);
            // The angle is the product in 32 bits, as programs have it that keep it in 32 bits: what they trained fits.  Of that angle in turns, taken in 64 bits,
            // only the fraction is kept, so its sine and cosine are exact to 32 bits however large it is.
            double turns = (double)((float)position * (float)p.frequencies[k - token * half]) * 0.15915494309189533577;
            turns -= rint(turns);
            float s, c;
            sincospif(2.f * (float)turns, &s, &c);
            angles[k] = make_float2(c, s);
        }
        __syncthreads();
        turn_rows<T, LANES, INTERLEAVED, BACKWARD>(p, angles, t0, count, false, dw[0]);
        turn_rows<T, LANES, INTERLEAVED, BACKWARD>(p, angles, t0, count, true, dw[1]);
        __syncthreads();
    }
    if (!BACKWARD || p.partial == nullptr) return;
    // every thread's sums into one per column, always in the same order
    const int group = threadIdx.x % LANES;
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int s = 16; s >= LANES; s >>= 1) dw[which][k] += __shfl_xor_sync(~0u, dw[which][k], s);
        if (threadIdx.x % 32 < LANES)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool split = group * 8 < p.turned && !INTERLEAVED;
                const int column = split ? (k < 4 ? group * 4 + k : half + group * 4 + k - 4) : group * 8 + k;
                sums[threadIdx.x / 32][column] = dw[which][k];
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

// The blocks' partial sums into the weights' gradients: a block per 32 columns, its 8 warps take every eighth partial sum.
__global__ void weight_kernel(const float* __restrict__ partial, int blocks, int dim, float* dq_weight, float* dk_weight) {
    __shared__ float sums[8][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = blockIdx.x * 32 + lane, which = blockIdx.y;
    float* out = which ? dk_weight : dq_weight;
    if (out == nullptr) return;
    float s = 0.f;
    if (c < dim)
#pragma unroll 8
        for (int b = warp; b < blocks; b += 8) s += partial[((int64_t)b * 2 + which) * dim + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < dim) {
        for (int w = 1; w < 8; ++w) s += sums[w][lane];
        out[c] = s;
    }
}

static int64_t blocks_of(int64_t tokens) { return std::min((tokens + kTokens - 1) / kTokens, kBlocks); }

uint64_t heads_workspace(int64_t tokens, int64_t dim) { return (uint64_t)(blocks_of(tokens) * 2 * dim * 4); }

template <typename T, int LANES, bool INTERLEAVED> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    HeadsParams p{};
    p.first = d.first; p.positions = d.positions; p.frequencies = d.frequencies; p.tokens = d.tokens;
    p.heads_q = (int)d.heads_q; p.heads_k = (int)d.heads_k; p.dim = (int)d.dim; p.turned = (int)d.turned;
    p.q = d.q; p.k = d.k; p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride;
    p.q_weight = d.q_weight; p.k_weight = d.k_weight; p.eps = d.eps; p.q_out = d.q_out; p.k_out = d.k_out;
    p.dq_out = d.dq_out; p.dk_out = d.dk_out; p.dq = d.dq; p.dk = d.dk;
    const unsigned blocks = (unsigned)blocks_of(d.tokens);
    if (!backward) {
        heads_kernel<T, LANES, INTERLEAVED, false><<<blocks, kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const bool weights = d.dq_weight != nullptr || d.dk_weight != nullptr;
    p.partial = weights ? static_cast<float*>(d.workspace) : nullptr;
    heads_kernel<T, LANES, INTERLEAVED, true><<<blocks, kThreads, 0, stream>>>(p);
    if (weights) weight_kernel<<<dim3((unsigned)((d.dim + 31) / 32), 2), 256, 0, stream>>>(p.partial, (int)blocks, p.dim, d.dq_weight, d.dk_weight);
    return cudaGetLastError();
}

template <typename T, int LANES> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    return d.interleaved != 0 ? run_heads<T, LANES, true>(d, backward, stream) : run_heads<T, LANES, false>(d, backward, stream);
}

template <typename T> static cudaError_t run_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream) {
    const int64_t groups = d.dim / 8;
    return groups <= 4 ? run_heads<T, 4>(d, backward, stream) : groups <= 8 ? run_heads<T, 8>(d, backward, stream)
         : groups <= 16 ? run_heads<T, 16>(d, backward, stream) : run_heads<T, 32>(d, backward, stream);
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
