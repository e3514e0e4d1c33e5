// The short causal convolution over episodes, channel by channel: forwards, backwards, and for one token of each env.
//
//   s_t = bias + sum over j of w_j x_{t - K + 1 + j},  y_t = s_t or silu(s_t);  ds_t = dy_t (silu'(s_t)),  dx_t = sum over j of w_j ds_{t + K - 1 - j},  dw_j = sum over t of ds_t x_{t - K + 1 + j}
//
// A few multiplications a value: the bytes bound it. A thread has four neighbouring channels and walks a stretch of tokens with the last K inputs in registers, so each
// input is read once and K - 1 of its neighbours' beside. An episode's begin empties those registers, a row's begin fills them from the row's initial inputs. Backwards one walk forwards, too: s is worked out again,
// and the sums that become the gradients of the last K inputs travel with them; the walk goes K - 1 tokens past its stretch (as far as the episode does) to complete them.
// Weights' gradients are summed in registers over all stretches of a thread, then over a block's warps, then over the blocks, always in the same order.
//
// Measured, K = 4 with silu: 4096 rows of 24 x 512, bf16, 51 us forwards (3.9 TB/s of its 2 tensors) and 86 back (3.5 TB/s of 3); 3 long rows, 131071 x 1024, f16, 112 us (4.8 TB/s) and 203 (4.0 TB/s); in f32 76, 135, 192 and 339. One token of 4096 envs x 512 22 us, in f32 15.
// The loads of the next tokens, and the plan's marks of the next 32, are under way while these are walked: with marks asked for by the batch, 55, 103, 133 and 243 us. Instructions, 1.9 to 2.0 of 4 a cycle, are some 15 a value
// forwards and 28 back, the exponentials' unit is busy for half of the time forwards and the multiplications' for 40 % back; 16 and 12 warps an SM is what the registers leave. More warps with four tokens ahead forwards: 52 and
// 124; back, four blocks to an SM spill (109 and 242), eight tokens ahead too (100 and 259). Eight channels to a thread were slower both ways (fewer warps), two slower back; blocks that take walks in turn forwards the same.
#include <algorithm>
#include "nkb_gates.cuh"
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

constexpr int kLines = 4;                               // warps of a block: stretches side by side
constexpr int kForthBlocks = 4, kBackBlocks = 3;        // blocks of an SM
constexpr int kForthBatch = 8, kBackBatch = 4;          // tokens whose loads are under way; a multiple of the longest window, so that its shift is a change of names
constexpr int kWide = 4;                                // channels of a thread
constexpr int kSms = 148;

struct ConvolutionParams {
    nuka_b200_episodes_t plan;
    int64_t channels, x_stride, stretch, stretches;
    uint32_t tiles, across;                             // blocks side by side over the channels, and along the tokens
    const float *weight, *bias;
    const void *x, *initial, *dy, *dstate;
    void *y, *state, *dx, *dinitial;
    float* partial;                                     // of the weights' gradients: across x (K + 1) x channels
    bool act, sums, whole, wide_weights;                // whole: every stretch ends with an episode; wide_weights: they lie on 16 bytes
};

// sum += a b, two values at a time where there are two
template <int N> __device__ __forceinline__ void add_products(float (&sum)[N], const float (&a)[N], const float (&b)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int v = 0; v < N; v += 2) split(fma_pair(pair_of(a[v], a[v + 1]), pair_of(b[v], b[v + 1]), pair_of(sum[v], sum[v + 1])), sum[v], sum[v + 1]);
    } else {
#pragma unroll
        for (int v = 0; v < N; ++v) sum[v] = fmaf(a[v], b[v], sum[v]);
    }
}

template <typename T, int K, int VEC> struct Line {
    float w[K][VEC], bias[VEC];
    __device__ __forceinline__ Line(const ConvolutionParams& p, int64_t c) {
        float all[VEC * K];
        if (VEC % 4 == 0 && p.wide_weights) {
#pragma unroll
            for (int k = 0; k < VEC * K; k += 4) { const float4 q = *reinterpret_cast<const float4*>(p.weight + c * K + k); all[k] = q.x; all[k + 1] = q.y; all[k + 2] = q.z; all[k + 3] = q.w; }
        } else {
#pragma unroll
            for (int k = 0; k < VEC * K; ++k) all[k] = p.weight[c * K + k];
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
            for (int j = 0; j < K; ++j) w[j][v] = all[v * K + j];
            bias[v] = p.bias != nullptr ? p.bias[c + v] : 0.f;
        }
    }
    // the sum for a window of inputs, the present one the last
    __device__ __forceinline__ void sum(const float (&window)[K][VEC], float (&s)[VEC]) const {
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[v] = bias[v];
#pragma unroll
        for (int j = 0; j < K; ++j) add_products(s, w[j], window[j]);
    }
};

// VEC inputs, or zeros.
template <typename T, int VEC> __device__ __forceinline__ void input(const void* from, int64_t at, bool there, float (&v)[VEC]) {
    if (there) {
        unpack<T, VEC>(load_raw<T, VEC>(static_cast<const T*>(from) + at), v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = 0.f;
    }
}

// The inputs before token t, which does not begin an episode: zeros before its first token, or what the row began with.
template <typename T, int K, int VEC> __device__ __forceinline__ void window_before(const ConvolutionParams& p, int64_t t, int64_t c, float (&window)[K][VEC]) {
    const int64_t first = p.plan.first[t];
    const int32_t row = t - first < K - 1 ? p.plan.link[first] : -1;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const int64_t at = t - (K - 1) + j, early = at - first + K - 1;          // number among the row's initial inputs where below K - 1
        if (at >= first) input<T, VEC>(p.x, at * p.x_stride + c, true, window[j + 1]);
        else input<T, VEC>(p.initial, ((int64_t)row * (K - 1) + early) * p.channels + c, row >= 0 && p.initial != nullptr, window[j + 1]);
    }
}
template <typename T, int K, int VEC> __device__ __forceinline__ void window_begins(const ConvolutionParams& p, int32_t row, int64_t c, float (&window)[K][VEC]) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) input<T, VEC>(p.initial, ((int64_t)row * (K - 1) + j) * p.channels + c, row >= 0 && p.initial != nullptr, window[j + 1]);
}

// 32 tokens of a warp's walk, number `lane` to a lane: which of them begin an episode, and which end a row. The next 32 are under way meanwhile, so that no batch waits for its own.
struct Marks {
    int32_t link, tail, next_link, next_tail;
    uint32_t begins, ends;
    __device__ __forceinline__ void ask(const ConvolutionParams& p, int64_t begin, int t0, int count) {
        const int t = t0 + threadIdx.x % 32;
        next_link = t < count ? p.plan.link[begin + t] : -1;
        next_tail = t < count ? p.plan.tail[begin + t] : -1;
    }
    __device__ __forceinline__ void turn(const ConvolutionParams& p, int64_t begin, int t0, int count) {
        link = next_link;
        tail = next_tail;
        begins = __ballot_sync(~0u, link != -1);
        ends = __ballot_sync(~0u, tail >= 0);
        ask(p, begin, t0 + 32, count);
    }
    __device__ __forceinline__ int32_t row_of(int t) const { return __shfl_sync(~0u, link, t & 31); }
    __device__ __forceinline__ int32_t end_of(int t) const { return __shfl_sync(~0u, tail, t & 31); }
};

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kLines * 32, kForthBlocks) convolution_kernel(const ConvolutionParams p) {
    constexpr int BATCH = kForthBatch;                  // tokens whose loads are under way
    constexpr uint32_t kBatchBits = (1u << BATCH) - 1u;
    const int64_t own = ((int64_t)(blockIdx.x % p.tiles) * 32 + threadIdx.x % 32) * VEC, C = p.channels;
    const int64_t line = (int64_t)(blockIdx.x / p.tiles) * kLines + threadIdx.x / 32;
    if (line >= p.stretches) return;
    const bool live = own < C;                          // VEC divides the channels; lanes behind the last read the first ones, and write nothing
    const int64_t c = live ? own : 0;
    const Line<T, K, VEC> f(p, c);
    const int64_t begin = line * p.stretch;
    const int count = (int)min(p.stretch, p.plan.tokens - begin);
    const T* const x = static_cast<const T*>(p.x) + begin * p.x_stride + c;
    T* y = static_cast<T*>(p.y) + begin * C + c;
    Raw<T, VEC> ahead[BATCH];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) ahead[i] = load_raw<T, VEC>(x + min(t0 + i, count - 1) * p.x_stride);
    };
    fetch(0);
    Marks marks;
    marks.ask(p, begin, 0, count);
    float window[K][VEC];                               // after the shift at a token's begin: the last inputs, 0 the oldest
    if (p.plan.link[begin] == -1) window_before<T, K, VEC>(p, begin, c, window);
    for (int t0 = 0; t0 < count; t0 += BATCH) {
        const int left = min(BATCH, count - t0);
        Raw<T, VEC> now[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) now[i] = ahead[i];
        if (t0 + BATCH < count) fetch(t0 + BATCH);
        if (t0 % 32 == 0) marks.turn(p, begin, t0, count);
        const uint32_t begins = marks.begins >> (t0 & 31) & kBatchBits, ends = marks.ends >> (t0 & 31) & kBatchBits;
        auto token = [&](int i) {
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
#pragma unroll
                for (int v = 0; v < VEC; ++v) window[j][v] = window[j + 1][v];
            unpack<T, VEC>(now[i], window[K - 1]);
            float s[VEC];
            f.sum(window, s);
            if (p.act) silu_all<sizeof(T) == 4>(s);
            if (live) store<T, VEC>(y, s);
            y += C;
        };
        auto begin_at = [&](int i) { window_begins<T, K, VEC>(p, marks.row_of(t0 + i), c, window); };
        auto end_at = [&](int i) {
            T* const to = static_cast<T*>(p.state) + (int64_t)marks.end_of(t0 + i) * (K - 1) * C + c;
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
                if (live) store<T, VEC>(to + j * C, window[j + 1]);
        };
        // mostly nothing begins or ends but at the edges
        if (left == BATCH && (begins & ~1u) == 0u && (ends & ~(1u << (BATCH - 1))) == 0u) {
            if (begins != 0u) begin_at(0);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) token(i);
            if (ends != 0u) end_at(BATCH - 1);
        } else {
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (i >= left) break;
                if (begins >> i & 1u) begin_at(i);
                token(i);
                if (ends >> i & 1u) end_at(i);
            }
        }
    }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kLines * 32, kBackBlocks) convolution_grad_kernel(const ConvolutionParams p) {
    __shared__ float sums[kLines / 2][(K + 1) * VEC * 32];
    constexpr int BATCH = kBackBatch;
    constexpr uint32_t kBatchBits = (1u << BATCH) - 1u;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t own = ((int64_t)(blockIdx.x % p.tiles) * 32 + lane) * VEC, C = p.channels;
    const bool live = own < C;
    const int64_t c = live ? own : 0;
    const Line<T, K, VEC> f(p, c);
    float dw[K][VEC] = {}, db[VEC] = {};
    for (int64_t line = (int64_t)(blockIdx.x / p.tiles) * kLines + warp; line < p.stretches; line += (int64_t)p.across * kLines) {
        // tokens by their number from the walk's first one
        const int64_t begin = line * p.stretch;
        const int end = (int)min(p.stretch, p.plan.tokens - begin), past = p.whole ? end : (int)min((int64_t)end + K - 1, p.plan.tokens - begin);
        float window[K][VEC], grad[K][VEC];             // grad: of the inputs in the window, as far as they are complete
        int first = 0, row = -1;                        // of the episode; the row that it began, within this walk
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) grad[j][v] = 0.f;
        if (p.plan.link[begin] == -1) {
            window_before<T, K, VEC>(p, begin, c, window);
            first = (int)max(p.plan.first[begin] - begin, (int64_t)-K);          // K before the walk is as far as any
        }
        const T *const x = static_cast<const T*>(p.x) + begin * p.x_stride + c, *const dy = static_cast<const T*>(p.dy) + begin * C + c;
        T* const dx = static_cast<T*>(p.dx) + begin * C + c;
        // the gradient of input number `at`, one of the row's initial ones where that is before the episode
        auto leave = [&](int at, const float (&g)[VEC]) {
            if (at >= first) {
                if (live && (unsigned)at < (unsigned)end) store<T, VEC>(dx + at * C, g);
            } else if (row >= 0 && p.dinitial != nullptr) {
                const int early = at - first + K - 1;
                if (live && early >= 0) store<T, VEC>(static_cast<T*>(p.dinitial) + ((int64_t)row * (K - 1) + early) * C + c, g);
            }
        };
        Raw<T, VEC> x_ahead[BATCH], dy_ahead[BATCH];
        auto fetch = [&](int t0) {
            const T *const xb = x + t0 * p.x_stride, *const dyb = dy + t0 * C;
            if (t0 + BATCH <= past) {                   // no clamps between the loads of a full batch
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    x_ahead[i] = load_raw<T, VEC>(xb + i * p.x_stride);
                    dy_ahead[i] = load_raw<T, VEC>(dyb + i * C);
                }
            } else {
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int t = min(i, past - 1 - t0);
                    x_ahead[i] = load_raw<T, VEC>(xb + t * p.x_stride);
                    dy_ahead[i] = load_raw<T, VEC>(dyb + t * C);
                }
            }
        };
        fetch(0);
        Marks marks;
        marks.ask(p, begin, 0, past);
        int last = past;                                // behind the last token walked
        for (int t0 = 0; t0 < past && last == past; t0 += BATCH) {
            const int left = min(BATCH, past - t0);
            Raw<T, VEC> xs[BATCH], dys[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) { xs[i] = x_ahead[i]; dys[i] = dy_ahead[i]; }
            if (t0 + BATCH < past) fetch(t0 + BATCH);
            if (t0 % 32 == 0) marks.turn(p, begin, t0, past);
            const uint32_t begins = marks.begins >> (t0 & 31) & kBatchBits, ends = marks.ends >> (t0 & 31) & kBatchBits;
            // one input further, whose gradient the others' are added to; own: the token is the walk's
            auto token = [&](int i, bool own) {
#pragma unroll
                for (int j = 0; j < K - 1; ++j)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) { window[j][v] = window[j + 1][v]; grad[j][v] = grad[j + 1][v]; }
                unpack<T, VEC>(xs[i], window[K - 1]);
                float ds[VEC];
                unpack<T, VEC>(dys[i], ds);
                if (p.act) {
                    float s[VEC];
                    f.sum(window, s);
                    by_silu_slope<sizeof(T) == 4>(s, ds);
                }
#pragma unroll
                for (int j = 0; j < K - 1; ++j) add_products(grad[j], f.w[j], ds);
#pragma unroll
                for (int v = 0; v < VEC; ++v) grad[K - 1][v] = f.w[K - 1][v] * ds[v];
                if (own) {
#pragma unroll
                    for (int j = 0; j < K; ++j) add_products(dw[j], ds, window[j]);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) db[v] += ds[v];
                }
            };
            auto end_at = [&](int i) {
                const int32_t ended = marks.end_of(t0 + i);
                if (p.dstate == nullptr) return;
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {
                    float more[VEC];
                    input<T, VEC>(p.dstate, ((int64_t)ended * (K - 1) + j) * C + c, true, more);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) grad[j + 1][v] += more[v];
                }
            };
            // an episode begins at token t: what the last one leaves, and an empty window
            auto begin_at = [&](int t) {
                if (t > 0)
#pragma unroll
                    for (int j = 0; j < K; ++j) leave(t - K + j, grad[j]);
                first = t;
                row = marks.row_of(t);
                window_begins<T, K, VEC>(p, row, c, window);
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) grad[j][v] = 0.f;
            };
            // mostly nothing begins or ends but at the edges, and what leaves is the walk's and the episode's, or the initial inputs' of the row that begins here
            const bool fresh = begins == 1u;
            if (t0 + BATCH <= end && (fresh || (begins == 0u && t0 >= K && first <= t0 - K)) && (ends & ~(1u << (BATCH - 1))) == 0u) {
                T* to = dx + (t0 - K) * C;
                if (fresh) {
                    begin_at(t0);
                    to = row >= 0 && p.dinitial != nullptr ? static_cast<T*>(p.dinitial) + ((int64_t)row * (K - 1) - 1) * C + c : nullptr;
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    if (i >= K ? live : live && to != nullptr && !(fresh && i == 0)) store<T, VEC>((i >= K ? dx + (t0 - K) * C : to) + i * C, grad[0]);
                    token(i, true);
                }
                if (ends != 0u) end_at(BATCH - 1);
                continue;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int t = t0 + i;
                if (i >= left) break;
                if (begins >> i & 1u) {
                    if (t >= end) { last = t; break; }
                    begin_at(t);
                } else if (t > 0) {
                    leave(t - K, grad[0]);
                }
                token(i, t < end);
                if (ends >> i & 1u) end_at(i);
            }
        }
#pragma unroll
        for (int j = 0; j < K; ++j) leave(last - K + j, grad[j]);
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

// Tokens of a walk. Whole rows where they are of one short length; else forwards as many as leave every SM sixty-four walks of 128 channels, 32 to 128, for which K - 1 are read twice; backwards, where a warp takes
// walks in turn, equal shares of about as many.
static int64_t walkers_of(int64_t channels) { return std::max<int64_t>(1, kBackBlocks * kSms / ((channels + 32 * kWide - 1) / (32 * kWide))) * kLines; }
static int64_t stretch_of(const nuka_b200_episodes_t& plan, int64_t channels, bool backward) {
    const int64_t tiles = (channels + 32 * kWide - 1) / (32 * kWide), fit = std::max<int64_t>(32, std::min<int64_t>(128, plan.tokens * tiles / (64 * kSms) / 4 * 4));
    if (plan.length > 0 && plan.length <= 64) return plan.length * std::max<int64_t>(1, ((backward ? 32 : fit) + plan.length / 2) / plan.length);
    if (!backward) return std::min<int64_t>(plan.tokens, fit);
    const int64_t walkers = walkers_of(channels), turns = (plan.tokens + 128 * walkers - 1) / (128 * walkers);
    return std::min<int64_t>(plan.tokens, std::max<int64_t>(32, (plan.tokens + turns * walkers - 1) / (turns * walkers)));
}

template <typename T, int VEC> static ConvolutionParams convolution_params(const nuka_b200_convolution_t& d, bool backward) {
    ConvolutionParams p{};
    p.plan = *d.plan;
    p.channels = d.channels; p.x_stride = d.x_stride;
    p.stretch = stretch_of(p.plan, d.channels, backward);
    p.stretches = (p.plan.tokens + p.stretch - 1) / p.stretch;
    p.tiles = (uint32_t)((d.channels + 32 * VEC - 1) / (32 * VEC));
    p.across = (uint32_t)((p.stretches + kLines - 1) / kLines);
    p.weight = d.weight; p.bias = d.bias; p.act = d.silu != 0u; p.whole = p.plan.length > 0 && p.stretch % p.plan.length == 0; p.wide_weights = reinterpret_cast<uintptr_t>(d.weight) % 16 == 0;
    p.x = d.x; p.initial = d.initial; p.dy = d.dy; p.dstate = d.dstate;
    p.y = d.y; p.state = d.state; p.dx = d.dx; p.dinitial = d.dinitial;
    return p;
}

// Blocks along the tokens of the backward pass, each of which leaves a set of partial sums: as many as run at a time, or several times that where a warp would sum more than kLongSum tokens one by one
// (n terms in 32 bits are off by up to n 2^-24 of their sizes).
constexpr int64_t kLongSum = 1024;
static int64_t convolution_across(const nuka_b200_episodes_t& plan, int64_t channels) {
    const int64_t stretch = stretch_of(plan, channels, true), stretches = (plan.tokens + stretch - 1) / stretch, walkers = walkers_of(channels);
    const int64_t tokens = (stretches + walkers - 1) / walkers * stretch;
    return std::min<int64_t>((stretches + kLines - 1) / kLines, walkers / kLines * ((tokens + kLongSum - 1) / kLongSum));
}
uint64_t convolution_workspace(const nuka_b200_episodes_t& plan, int64_t channels, int64_t width) { return (uint64_t)(convolution_across(plan, channels) * (width + 1) * channels) * sizeof(float); }

template <typename T, int K, int VEC> static cudaError_t run_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    ConvolutionParams p = convolution_params<T, VEC>(d, backward);
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

// kWide channels to a thread where everything lies on as many, else one.
template <typename T> static cudaError_t run_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream) {
    bool wide = d.channels % kWide == 0 && d.x_stride % kWide == 0;
    auto lies = [](const void* at) { return reinterpret_cast<uintptr_t>(at) % (kWide * sizeof(T)) == 0; };
    for (const void* p : {d.x, d.initial, static_cast<const void*>(d.y), static_cast<const void*>(d.state)}) wide = wide && lies(p);
    if (backward)
        for (const void* p : {d.dy, d.dstate, static_cast<const void*>(d.dx), static_cast<const void*>(d.dinitial)}) wide = wide && lies(p);
    return wide ? run_convolution<T, kWide>(d, backward, stream) : run_convolution<T, 1>(d, backward, stream);
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
    float sum[VEC], window[K][VEC];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) input<T, VEC>(state, j * d.channels, !begins, window[j]);
    input<T, VEC>(d.x, env * d.x_stride + c, true, window[K - 1]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sum[v] = d.bias != nullptr ? d.bias[c + v] : 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) sum[v] = fmaf(d.weight[(c + v) * K + j], window[j][v], sum[v]);
    }
    if (d.silu) silu_all<sizeof(T) == 4>(sum);
    store<T, VEC>(static_cast<T*>(d.y) + env * d.channels + c, sum);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) store<T, VEC>(state + j * d.channels, window[j + 1]);
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
