// The short causal convolution over episodes, channel by channel: forwards, backwards, and for one token of each env.
//
//   s_t = bias + sum over j of w_j x_{t - K + 1 + j},  y_t = s_t or silu(s_t);  ds_t = dy_t (silu'(s_t)),  dx_t = sum over j of w_j ds_{t + K - 1 - j},  dw_j = sum over t of ds_t x_{t - K + 1 + j}
//
// A few multiplications a value: the bytes bound it. A thread has VEC neighbouring channels, 16 bytes of them, and walks a stretch of tokens with the last K - 1 inputs in registers, so each
// input is read once and K - 1 of its neighbours' beside. An episode's begin empties those registers, a row's begin fills them from the row's initial inputs. Backwards one walk forwards, too: s is worked out again,
// and the sums that become the gradients of the last K inputs travel with them; the walk goes K - 1 tokens past its stretch (as far as the episode does) to complete them.
// Weights' gradients are summed in registers over all stretches of a thread, then over a block's warps, then over the blocks, always in the same order.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

constexpr int kLines = 8;                               // warps of a block: stretches side by side
constexpr int kSms = 148;

struct ConvolutionParams {
    nuka_b200_episodes_t plan;
    int64_t channels, x_stride, stretch, stretches;
    uint32_t tiles, across;                             // blocks side by side over the channels, and along the tokens
    const float *weight, *bias;
    const void *x, *initial, *dy, *dstate;
    void *y, *state, *dx, *dinitial;
    float* partial;                                     // of the weights' gradients: across x (K + 1) x channels
    bool act, sums;
};

template <typename T, int K, int VEC> struct Line {
    float w[K][VEC], bias[VEC];
    __device__ __forceinline__ Line(const ConvolutionParams& p, int64_t c) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
            for (int j = 0; j < K; ++j) w[j][v] = p.weight[(c + v) * K + j];
            bias[v] = p.bias != nullptr ? p.bias[c + v] : 0.f;
        }
    }
    // the sum for a window of inputs, the present one the last
    __device__ __forceinline__ void sum(const Raw<T, VEC> (&window)[K], float (&s)[VEC]) const {
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[v] = bias[v];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float x[VEC];
            unpack<T, VEC>(window[j], x);
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = fmaf(w[j][v], x[v], s[v]);
        }
    }
};

template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> nothing() {
    const float zero[VEC] = {};
    Raw<T, VEC> r;
    store<T, VEC>(reinterpret_cast<T*>(&r), zero);
    return r;
}

// The inputs before token t, which does not begin an episode: zeros before its first token, or what the row began with.
template <typename T, int K, int VEC> __device__ __forceinline__ void window_before(const ConvolutionParams& p, int64_t t, int64_t c, Raw<T, VEC> (&window)[K]) {
    const int64_t first = p.plan.first[t];
    const int32_t row = t - first < K - 1 ? p.plan.link[first] : -1;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const int64_t at = t - (K - 1) + j, early = at - first + K - 1;          // number among the row's initial inputs where below K - 1
        window[j + 1] = at >= first ? load_raw<T, VEC>(static_cast<const T*>(p.x) + at * p.x_stride + c)
                      : row >= 0 && p.initial != nullptr ? load_raw<T, VEC>(static_cast<const T*>(p.initial) + ((int64_t)row * (K - 1) + early) * p.channels + c) : nothing<T, VEC>();
    }
}
template <typename T, int K, int VEC> __device__ __forceinline__ void window_begins(const ConvolutionParams& p, int32_t row, int64_t c, Raw<T, VEC> (&window)[K]) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
        window[j + 1] = row >= 0 && p.initial != nullptr ? load_raw<T, VEC>(static_cast<const T*>(p.initial) + ((int64_t)row * (K - 1) + j) * p.channels + c) : nothing<T, VEC>();
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kLines * 32) convolution_kernel(const ConvolutionParams p) {
    constexpr int BATCH = 8;                            // tokens whose loads are under way
    const int64_t c = ((int64_t)(blockIdx.x % p.tiles) * 32 + threadIdx.x % 32) * VEC, C = p.channels;
    const int64_t line = (int64_t)(blockIdx.x / p.tiles) * kLines + threadIdx.x / 32;
    if (c >= C || line >= p.stretches) return;          // VEC divides the channels
    const Line<T, K, VEC> f(p, c);
    const T* const x = static_cast<const T*>(p.x) + c;
    const int64_t begin = line * p.stretch, end = min(begin + p.stretch, p.plan.tokens);
    Raw<T, VEC> window[K];                              // after the shift at the loop's begin: the last inputs, 0 the oldest
    if (p.plan.link[begin] == -1) window_before<T, K, VEC>(p, begin, c, window);
    for (int64_t t0 = begin; t0 < end; t0 += BATCH) {
        Raw<T, VEC> next[BATCH];
        int32_t link[BATCH], tail[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t t = min(t0 + i, end - 1);
            next[i] = load_raw<T, VEC>(x + t * p.x_stride);
            link[i] = p.plan.link[t];
            tail[i] = p.plan.tail[t];
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t t = t0 + i;
            if (t >= end) break;
            if (link[i] != -1) window_begins<T, K, VEC>(p, link[i], c, window);
#pragma unroll
            for (int j = 0; j < K - 1; ++j) window[j] = window[j + 1];
            window[K - 1] = next[i];
            float s[VEC];
            f.sum(window, s);
            if (p.act)
#pragma unroll
                for (int v = 0; v < VEC; ++v) s[v] = silu<sizeof(T) == 4>(s[v]);
            store<T, VEC>(static_cast<T*>(p.y) + t * C + c, s);
            if (tail[i] >= 0)
#pragma unroll
                for (int j = 0; j < K - 1; ++j) *reinterpret_cast<Raw<T, VEC>*>(static_cast<T*>(p.state) + ((int64_t)tail[i] * (K - 1) + j) * C + c) = window[j + 1];
        }
    }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kLines * 32) convolution_grad_kernel(const ConvolutionParams p) {
    __shared__ float sums[kLines / 2][(K + 1) * VEC * 32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t own = ((int64_t)(blockIdx.x % p.tiles) * 32 + lane) * VEC, C = p.channels;
    const bool live = own < C;
    const int64_t c = live ? own : 0;
    const Line<T, K, VEC> f(p, c);
    const T *const x = static_cast<const T*>(p.x) + c, *const dy = static_cast<const T*>(p.dy) + c;
    float dw[K][VEC] = {}, db[VEC] = {};
    for (int64_t line = (int64_t)(blockIdx.x / p.tiles) * kLines + warp; live && line < p.stretches; line += (int64_t)p.across * kLines) {
        const int64_t begin = line * p.stretch, end = min(begin + p.stretch, p.plan.tokens), past = min(end + K - 1, p.plan.tokens);
        Raw<T, VEC> window[K];
        float grad[K][VEC];                             // of the inputs in the window, as far as they are complete
        int64_t first = begin;                          // of the episode
        int32_t row = -1;                               // that it began, within this walk
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) grad[j][v] = 0.f;
        if (p.plan.link[begin] == -1) {
            window_before<T, K, VEC>(p, begin, c, window);
            first = p.plan.first[begin];
        }
        // the gradient of input number `at`, one of the row's initial ones where that is before the episode
        auto leave = [&](int64_t at, const float (&g)[VEC]) {
            if (at >= first) {
                if (at >= begin && at < end) store<T, VEC>(static_cast<T*>(p.dx) + at * C + c, g);
            } else if (row >= 0 && p.dinitial != nullptr) {
                const int64_t early = at - first + K - 1;
                if (early >= 0) store<T, VEC>(static_cast<T*>(p.dinitial) + ((int64_t)row * (K - 1) + early) * C + c, g);
            }
        };
        int64_t t = begin;
        constexpr int BATCH = 4;
        bool goes = true;
        for (int64_t t0 = begin; goes && t0 < past; t0 += BATCH) {
            Raw<T, VEC> xs[BATCH], dys[BATCH];
            int32_t link[BATCH], tail[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int64_t u = min(t0 + i, past - 1);
                xs[i] = load_raw<T, VEC>(x + u * p.x_stride);
                dys[i] = load_raw<T, VEC>(dy + u * C);
                link[i] = p.plan.link[u];
                tail[i] = p.plan.tail[u];
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                t = t0 + i;
                if (t >= past || (t >= end && link[i] != -1)) { goes = false; break; }
                if (link[i] != -1) {
                    if (t > begin)
#pragma unroll
                        for (int j = 0; j < K; ++j) leave(t - K + j, grad[j]);
                    window_begins<T, K, VEC>(p, link[i], c, window);
                    first = t;
                    row = link[i];
#pragma unroll
                    for (int j = 0; j < K; ++j)
#pragma unroll
                        for (int v = 0; v < VEC; ++v) grad[j][v] = 0.f;
                } else if (t > begin) {
                    leave(t - K, grad[0]);
                }
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {
                    window[j] = window[j + 1];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) grad[j][v] = grad[j + 1][v];
                }
                window[K - 1] = xs[i];
                float ds[VEC];
                unpack<T, VEC>(dys[i], ds);
                if (p.act) {
                    float s[VEC];
                    f.sum(window, s);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) ds[v] *= silu_slope<sizeof(T) == 4>(s[v]);
                }
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) grad[j][v] = fmaf(f.w[j][v], ds[v], j < K - 1 ? grad[j][v] : 0.f);
                if (p.sums && t < end) {
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        float xv[VEC];
                        unpack<T, VEC>(window[j], xv);
#pragma unroll
                        for (int v = 0; v < VEC; ++v) dw[j][v] = fmaf(ds[v], xv[v], dw[j][v]);
                    }
#pragma unroll
                    for (int v = 0; v < VEC; ++v) db[v] += ds[v];
                }
                if (tail[i] >= 0 && p.dstate != nullptr)
#pragma unroll
                    for (int j = 0; j < K - 1; ++j) {
                        float more[VEC];
                        unpack<T, VEC>(load_raw<T, VEC>(static_cast<const T*>(p.dstate) + ((int64_t)tail[i] * (K - 1) + j) * C + c), more);
#pragma unroll
                        for (int v = 0; v < VEC; ++v) grad[j + 1][v] += more[v];
                    }
            }
        }
        if (goes) t = past;                             // the token after the last one walked
#pragma unroll
        for (int j = 0; j < K; ++j) leave(t - K + j, grad[j]);
    }
    if (!p.sums) return;
    // the block's warps into one, half of them at a time
    auto place = [&](int w, int k) -> float& { return sums[w][k * 32 + lane]; };
#pragma unroll
    for (int half = kLines / 2; half > 0; half /= 2) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
#pragma unroll
                for (int j = 0; j < K; ++j) place(warp - half, j * VEC + v) = dw[j][v];
                place(warp - half, K * VEC + v) = db[v];
            }
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
#pragma unroll
                for (int j = 0; j < K; ++j) dw[j][v] += place(warp, j * VEC + v);
                db[v] += place(warp, K * VEC + v);
            }
        }
        __syncthreads();
    }
    if (warp == 0 && live) {
        float* const to = p.partial + (int64_t)(blockIdx.x / p.tiles) * (K + 1) * C + c;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
            for (int j = 0; j < K; ++j) to[j * C + v] = dw[j][v];
            to[K * C + v] = db[v];
        }
    }
}

// The blocks' sums into one: a warp row of 32 sums, its block's warps a share of the blocks each.
template <int K> __global__ void __launch_bounds__(1024) convolution_sums_kernel(const ConvolutionParams p, float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t C = p.channels, n = (K + 1) * C, at = (int64_t)blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (at < n)
        for (uint32_t b = warp; b < p.across; b += 32) sum += p.partial[b * n + at];
    part[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || at >= n) return;
    sum = 0.f;
    for (int w = 0; w < 32; ++w) sum += part[w][lane];
    const int64_t j = at / C, c = at % C;
    if (j < K) { if (dweight != nullptr) dweight[c * K + j] = sum; } else if (dbias != nullptr) dbias[c] = sum;
}

// Tokens of a walk: whole rows where they are of one short length, else 32, for which K - 1 are read twice.
static int64_t stretch_of(const nuka_b200_episodes_t& plan) {
    return plan.length > 0 && plan.length <= 64 ? plan.length * std::max<int64_t>(1, 32 / plan.length) : std::min<int64_t>(32, plan.tokens);
}

template <typename T, int VEC> static ConvolutionParams convolution_params(const nuka_b200_convolution_t& d) {
    ConvolutionParams p{};
    p.plan = *d.plan;
    p.channels = d.channels; p.x_stride = d.x_stride;
    p.stretch = stretch_of(p.plan);
    p.stretches = (p.plan.tokens + p.stretch - 1) / p.stretch;
    p.tiles = (uint32_t)((d.channels + 32 * VEC - 1) / (32 * VEC));
    p.across = (uint32_t)((p.stretches + kLines - 1) / kLines);
    p.weight = d.weight; p.bias = d.bias; p.act = d.silu != 0u;
    p.x = d.x; p.initial = d.initial; p.dy = d.dy; p.dstate = d.dstate;
    p.y = d.y; p.state = d.state; p.dx = d.dx; p.dinitial = d.dinitial;
    return p;
}

// Blocks along the tokens of the backward pass, each of which leaves a set of partial sums: four to an SM.
static int64_t convolution_across(const nuka_b200_episodes_t& plan, int64_t channels) {
    const int64_t stretches = (plan.tokens + stretch_of(plan) - 1) / stretch_of(plan), tiles = (channels + 255) / 256;
    return std::max<int64_t>(1, std::min<int64_t>((stretches + kLines - 1) / kLines, (4 * kSms + tiles - 1) / tiles));
}
uint64_t convolution_workspace(const nuka_b200_episodes_t& plan, int64_t channels, int64_t width) { return (uint64_t)(convolution_across(plan, channels) * (width + 1) * channels) * sizeof(float); }

template <typename T, int K, int VEC> static cudaError_t run_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    ConvolutionParams p = convolution_params<T, VEC>(d);
    if (!backward) {
        convolution_kernel<T, K, VEC><<<p.tiles * p.across, kLines * 32, 0, stream>>>(p);
        return cudaGetLastError();
    }
    p.sums = d.dweight != nullptr || d.dbias != nullptr;
    p.across = (uint32_t)convolution_across(p.plan, d.channels);
    p.partial = static_cast<float*>(d.workspace);
    convolution_grad_kernel<T, K, VEC><<<p.tiles * p.across, kLines * 32, 0, stream>>>(p);
    if (p.sums) convolution_sums_kernel<K><<<(unsigned)(((K + 1) * d.channels + 31) / 32), 1024, 0, stream>>>(p, d.dweight, d.dbias);
    return cudaGetLastError();
}

template <typename T, int VEC> static cudaError_t run_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    return d.width == 2 ? run_convolution<T, 2, VEC>(d, backward, stream) : d.width == 3 ? run_convolution<T, 3, VEC>(d, backward, stream) : run_convolution<T, 4, VEC>(d, backward, stream);
}

// 16 bytes to a thread where everything lies so, else a value.
template <typename T> static cudaError_t run_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    bool wide = d.channels % W == 0 && d.x_stride % W == 0;
    for (const void* p : {d.x, d.initial, d.dy, d.dstate, static_cast<const void*>(d.y), static_cast<const void*>(d.state), static_cast<const void*>(d.dx), static_cast<const void*>(d.dinitial)})
        wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    return wide ? run_convolution<T, W>(d, backward, stream) : run_convolution<T, 1>(d, backward, stream);
}

cudaError_t launch_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    if (d.plan->tokens == 0) {                          // weights' gradients are sums of nothing
        cudaError_t set = cudaSuccess;
        if (backward && d.dweight != nullptr) set = cudaMemsetAsync(d.dweight, 0, (size_t)(d.channels * d.width) * 4, stream);
        if (backward && d.dbias != nullptr && set == cudaSuccess) set = cudaMemsetAsync(d.dbias, 0, (size_t)d.channels * 4, stream);
        return set;
    }
    return d.dtype == NUKA_B200_F32 ? run_convolution<float>(d, backward, stream) : d.dtype == NUKA_B200_F16 ? run_convolution<__half>(d, backward, stream) : run_convolution<__nv_bfloat16>(d, backward, stream);
}

// ---- one token per env ---------------------------------------------------------------------------------------------
template <typename T, int K, int VEC>
__global__ void convolution_step_kernel(int64_t groups, uint32_t per_env, const nuka_b200_convolution_step_t d) {
    const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (g >= groups) return;
    const int64_t env = g / per_env, c = (g - env * per_env) * VEC;
    T* const state = static_cast<T*>(d.state) + env * (K - 1) * d.channels + c;
    const bool begins = d.fresh != nullptr && d.fresh[env] != 0;
    float sum[VEC], x[VEC];
    Raw<T, VEC> window[K];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) window[j] = begins ? nothing<T, VEC>() : load_raw<T, VEC>(state + j * d.channels);
    window[K - 1] = load_raw<T, VEC>(static_cast<const T*>(d.x) + env * d.x_stride + c);
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum[v] = d.bias != nullptr ? d.bias[c + v] : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        unpack<T, VEC>(window[j], x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] = fmaf(d.weight[(c + v) * K + j], x[v], sum[v]);
    }
    if (d.silu)
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] = silu<sizeof(T) == 4>(sum[v]);
    store<T, VEC>(static_cast<T*>(d.y) + env * d.channels + c, sum);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) *reinterpret_cast<Raw<T, VEC>*>(state + j * d.channels) = window[j + 1];
}

template <typename T, int VEC> static cudaError_t run_convolution_step(const nuka_b200_convolution_step_t& d, cudaStream_t stream) {
    const int64_t groups = d.envs * (d.channels / VEC);
    const unsigned blocks = (unsigned)((groups + 127) / 128);
    const uint32_t per_env = (uint32_t)(d.channels / VEC);
    if (d.width == 2) convolution_step_kernel<T, 2, VEC><<<blocks, 128, 0, stream>>>(groups, per_env, d);
    else if (d.width == 3) convolution_step_kernel<T, 3, VEC><<<blocks, 128, 0, stream>>>(groups, per_env, d);
    else convolution_step_kernel<T, 4, VEC><<<blocks, 128, 0, stream>>>(groups, per_env, d);
    return cudaGetLastError();
}

template <typename T> static cudaError_t run_convolution_step(const nuka_b200_convolution_step_t& d, cudaStream_t stream) {
    constexpr int W = 8 / sizeof(T);                    // 8 bytes: a batch of few envs then has more threads
    bool wide = d.channels % W == 0 && d.x_stride % W == 0;
    for (const void* p : {d.x, static_cast<const void*>(d.state), static_cast<const void*>(d.y)}) wide = wide && reinterpret_cast<uintptr_t>(p) % 8 == 0;
    return wide ? run_convolution_step<T, W>(d, stream) : run_convolution_step<T, 1>(d, stream);
}

cudaError_t launch_convolution_step(const nuka_b200_convolution_step_t& d, cudaStream_t stream) {
    return d.dtype == NUKA_B200_F32 ? run_convolution_step<float>(d, stream) : d.dtype == NUKA_B200_F16 ? run_convolution_step<__half>(d, stream) : run_convolution_step<__nv_bfloat16>(d, stream);
}

}  // namespace nkb
