// The plan of episodes and the gated linear recurrence over them.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

// ---- plan ----------------------------------------------------------------------------------------------------------
__global__ void offsets_kernel(nuka_b200_episodes_t p, const int32_t* __restrict__ offsets) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= p.tokens) return;
    int64_t low = 0, high = p.rows;                 // the last row that begins at or before t
    while (high - low > 1) {
        const int64_t mid = (low + high) >> 1;
        if (offsets[mid] <= t) low = mid; else high = mid;
    }
    const int32_t first = min(max(offsets[low], 0), (int32_t)t), end = (int32_t)min(max((int64_t)offsets[low + 1], t + 1), p.tokens);
    p.first[t] = first;
    p.end[t] = end;
    p.link[t] = first == t ? (int32_t)low : -1;
    p.tail[t] = end == t + 1 ? (int32_t)low : -1;
}

// One block per row.  first: a running maximum over the places where an episode begins; end: a running minimum from the other side.
__global__ void done_kernel(nuka_b200_episodes_t p, const uint8_t* __restrict__ done, int32_t length) {
    __shared__ int32_t part[32];
    const int32_t row = blockIdx.x, base = row * length;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int back = 0; back < 2; ++back) {
        int32_t carry = back ? length : 0;
        for (int32_t at = 0; at < length; at += blockDim.x) {
            const int32_t s = at + threadIdx.x, k = back ? length - 1 - s : s;
            const bool in = s < length;
            // forwards: k where an episode begins, else 0; backwards: k + 1 where one ends, else the row's length
            int32_t v = back ? length : 0;
            if (in && !back) v = k > 0 && done[base + k - 1] ? k : 0;
            if (in && back) v = done[base + k] ? k + 1 : length;
            const int32_t own = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int32_t o = __shfl_up_sync(~0u, v, d);
                if (lane >= d) v = back ? min(v, o) : max(v, o);
            }
            if (lane == 31) part[warp] = v;
            __syncthreads();
            for (int w = 0; w < warp; ++w) v = back ? min(v, part[w]) : max(v, part[w]);
            v = back ? min(v, carry) : max(v, carry);
            int32_t all = carry;
            for (int w = 0; w < warps; ++w) all = back ? min(all, part[w]) : max(all, part[w]);
            carry = all;
            if (in && !back) {
                p.first[base + k] = base + v;
                p.link[base + k] = k == 0 ? row : own == k ? -2 : -1;
            }
            if (in && back) {
                p.end[base + k] = base + v;
                p.tail[base + k] = k == length - 1 ? row : -1;
            }
            __syncthreads();
        }
    }
}

cudaError_t launch_episodes_from_offsets(const nuka_b200_episodes_t& p, const int32_t* offsets, cudaStream_t stream) {
    if (p.tokens != 0) offsets_kernel<<<(unsigned)((p.tokens + 255) / 256), 256, 0, stream>>>(p, offsets);
    return cudaGetLastError();
}

cudaError_t launch_episodes_from_done(const nuka_b200_episodes_t& p, const uint8_t* done, cudaStream_t stream) {
    if (p.tokens == 0) return cudaSuccess;
    const int32_t length = (int32_t)(p.tokens / p.rows);
    done_kernel<<<(unsigned)p.rows, (unsigned)std::min(1024, (length + 31) / 32 * 32), 0, stream>>>(p, done, length);
    return cudaGetLastError();
}

// ---- recurrence ----------------------------------------------------------------------------------------------------
// Each token maps the state by h -> a h + b; two such maps in a row are one again, (A, B) after (a, b) = (A a, A b + B), which is what makes
// the scan parallel.  A token that begins an episode forgets the state whatever it was: such a map is *closed* and is never
// multiplied with what came before, so that an infinity or NaN stays in its episode.  Backwards the state is the gradient that goes on to the token before, m -> a (m + b).
//
// A warp walks a segment of tokens one by one, 32 * VEC channels wide, the next tokens' loads under way while it works on the present ones, so an element
// costs its sigmoid, two multiplications and its loads, and nothing waits for another warp.  Rows of one length that are short or give every SM its share of
// warps are the segments: each begins with a row, and that is all.  Otherwise the tokens are cut into as many equal segments as fill the GPU and walked twice: first for
// each segment's map alone, then, when a small scan over the maps has said what state each begins with, for the values.  The inputs are read twice that way (5 tensors' bytes in place
// of 3 forwards, 8 in place of 6 backwards); chunks that wait for one another's maps read them once, and were slower by more: their waits, a few microseconds for every chunk of 64 tokens, had
// nothing to hide under (131071 x 1024, bf16: 1.42 ms forwards, against 0.30 here).  All orders are fixed, so the same call gives the same bits.
//
// Measured: 4096 rows of 24 x 256 channels, bf16, 40 us forwards (3.8 TB/s of its 3 tensors) and 61 back (4.9 TB/s of 6); 1000 rows of 37 x 200, f32, 35 us (2.6 TB/s);
// 3 long rows, 131071 x 1024, bf16, 130 us for the maps, 5 for the scan over them and 161 for the values, back 131, 5 and 270 (4.1 to 6.0 TB/s of what each reads and writes).
// Neither the memory (half busy) nor the issue slots (2.1 to 2.3 of 4 a cycle) are full: sixteen warps an SM, as many as their loads' registers leave, wait for the chain of a token's
// sigmoid and step.

// Channels of a lane; tokens whose loads are under way.
template <typename T> constexpr int kWide = sizeof(T) == 4 ? 2 : 4;
template <bool BACKWARD> constexpr int kBatch = BACKWARD ? 4 : 8;
constexpr int kWalkers = 4;                             // warps of a block
constexpr float kClosed = -1.f;                         // in the place of A, which is never negative

struct RecurrenceParams {
    nuka_b200_episodes_t plan;
    int64_t channels, x_stride, gate_stride, segment, segments;
    const void *x, *gate, *dh;
    void *h, *dx, *dgate;
    const float *initial, *dstate;
    float *state, *dinitial;
    float2* maps;                                       // segments x channels; null where every segment is on its own
    float* carries;                                     // segments x channels: the state that a segment begins with, in scan order
    uint32_t tiles;
};

// 1 / (1 + exp(-g)) and 1 minus it, each without cancellation.  16-bit inputs and outputs leave the fast form's error, 2^-21 for small gates and, from the exponent's rounding, |g| 2^-24 for
// large ones (2^-20.5 at 11, 2^-17.7 at 80), far below their rounding; its clamp
// keeps exp(-g) finite, so that the product is 1 and not inf * 0 where the gate is closed.
template <bool EXACT> __device__ __forceinline__ void sigmoid(float g, float& a, float& rest) {
    if (EXACT) {
        const float e = expf(-fabsf(g)), r = 1.f / (1.f + e), s = e * r;         // NaN where g is
        a = g >= 0.f ? r : s;
        rest = g >= 0.f ? s : r;
    } else {
        float x, e;
        asm("max.NaN.f32 %0, %1, 0fC2A00000;" : "=f"(x) : "f"(g));               // -80
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(1.f + e));
        rest = e * a;
    }
}

// MAPS: only the segment's map
template <typename T, int VEC, bool BACKWARD, bool MAPS>
__global__ void __launch_bounds__(kWalkers * 32, 4) recurrence_kernel(const RecurrenceParams p) {
    constexpr int BATCH = kBatch<BACKWARD>;
    constexpr bool EXACT = sizeof(T) == 4, NEEDS_X = !BACKWARD || !MAPS, NEEDS_H = BACKWARD && !MAPS;
    using R = Raw<T, VEC>;
    const int lane = threadIdx.x & 31;
    const int64_t job = (int64_t)blockIdx.x * kWalkers + (threadIdx.x >> 5), segment = job / p.tiles, C = p.channels, c = (int64_t)(job % p.tiles) * (32 * VEC) + lane * VEC;
    if (segment >= p.segments) return;
    const bool live = c < C;                            // VEC divides the channels
    const int64_t lowest = segment * p.segment, count = min(p.segment, p.plan.tokens - lowest);
    const int64_t t0 = BACKWARD ? lowest + count - 1 : lowest, step = BACKWARD ? -1 : 1;
    const int64_t column = live ? c : 0;                // lanes behind the last channel read the first one's, and write nothing
    const T *const x = static_cast<const T*>(p.x) + column, *const gate = static_cast<const T*>(p.gate) + column;
    const T *const dh = static_cast<const T*>(p.dh) + column, *const hs = static_cast<const T*>(p.h) + column;

    struct Ahead {
        R x[NEEDS_X ? BATCH : 1], gate[BATCH], dh[BACKWARD ? BATCH : 1], h[NEEDS_H ? BATCH : 1];
        int32_t link, tail;                             // of token `lane` of the batch
    };
    // behind the segment's end the last token again: loaded, and not used
    auto fetch = [&](Ahead& b, int64_t k0) {
        const int64_t own = t0 + step * min(k0 + lane, count - 1);
        b.link = lane < BATCH ? p.plan.link[own] : -1;
        b.tail = lane < BATCH ? p.plan.tail[own] : -1;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t t = t0 + step * min(k0 + i, count - 1);
            if constexpr (NEEDS_X) b.x[i] = load_raw<T, VEC>(x + t * p.x_stride);
            b.gate[i] = load_raw<T, VEC>(gate + t * p.gate_stride);
            if constexpr (BACKWARD) b.dh[i] = load_raw<T, VEC>(dh + t * C);
            if constexpr (NEEDS_H) b.h[i] = load_raw<T, VEC>(hs + max((int64_t)0, t - 1) * C);
        }
    };
    float h[VEC], A[VEC];                               // the state or the gradient that goes on; of a map, B and A
    bool closed = false;
    const int64_t place = segment * C + column;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        h[v] = !MAPS && p.maps != nullptr ? p.carries[place + v] : 0.f;
        A[v] = 1.f;
    }
    auto row_of = [&](const float* values, int32_t row, float (&to)[VEC]) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) to[v] = values != nullptr ? values[row * C + column + v] : 0.f;
    };
    auto walk = [&](const Ahead& b, int64_t k0) {
        const uint32_t begins = __ballot_sync(~0u, b.link != -1), ends = __ballot_sync(~0u, b.tail >= 0);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            if (k0 + i >= count) break;
            const int64_t t = t0 + step * (k0 + i);
            const bool begin = begins >> i & 1u, end = ends >> i & 1u;
            float a[VEC], rest[VEC], gv[VEC], xv[VEC];
            unpack<T, VEC>(b.gate[i], gv);
            if constexpr (NEEDS_X) unpack<T, VEC>(b.x[i], xv);
#pragma unroll
            for (int v = 0; v < VEC; ++v) sigmoid<EXACT>(gv[v], a[v], rest[v]);
            if constexpr (!BACKWARD) {
                if (begin) {
                    const int32_t row = __shfl_sync(~0u, b.link, i);
                    if (row >= 0) {
                        row_of(p.initial, row, h);
                    } else {
#pragma unroll
                        for (int v = 0; v < VEC; ++v) h[v] = 0.f;
                    }
                    closed = true;
                }
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    h[v] = fmaf(a[v], h[v], rest[v] * xv[v]);
                    if (MAPS) A[v] *= a[v];
                }
                if constexpr (!MAPS) {
                    if (live) store<T, VEC>(static_cast<T*>(p.h) + t * C + c, h);
                    if (end) {
                        const int32_t row = __shfl_sync(~0u, b.tail, i);
                        if (live) store<float, VEC>(p.state + row * C + c, h);
                    }
                }
            } else {
                float dv[VEC];
                unpack<T, VEC>(b.dh[i], dv);
                if (end) {
                    const int32_t row = __shfl_sync(~0u, b.tail, i);
                    float more[VEC];
                    row_of(p.dstate, row, more);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) h[v] += more[v];
                }
                const int32_t row = begin ? __shfl_sync(~0u, b.link, i) : -1;
                if constexpr (!MAPS) {
                    float before[VEC], dx[VEC], dg[VEC];
                    unpack<T, VEC>(b.h[i], before);
                    if (begin) {
                        if (row >= 0) {
                            row_of(p.initial, row, before);
                        } else {
#pragma unroll
                            for (int v = 0; v < VEC; ++v) before[v] = 0.f;
                        }
                    }
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float grad = h[v] + dv[v];        // `before` was rounded to T: in 16 bits, where it is close to x, the difference below is mostly that
                        dx[v] = rest[v] * grad;
                        dg[v] = dx[v] * (before[v] - xv[v]) * a[v];
                        h[v] = a[v] * grad;
                    }
                    if (live) {
                        store<T, VEC>(static_cast<T*>(p.dx) + t * C + c, dx);
                        store<T, VEC>(static_cast<T*>(p.dgate) + t * C + c, dg);
                        if (row >= 0 && p.dinitial != nullptr) store<float, VEC>(p.dinitial + row * C + c, h);
                    }
                } else {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        h[v] = a[v] * (h[v] + dv[v]);
                        A[v] *= a[v];
                    }
                }
                if (begin) {                            // nothing goes on to another episode
                    closed = true;
#pragma unroll
                    for (int v = 0; v < VEC; ++v) h[v] = 0.f;
                }
            }
        }
    };
    Ahead one, two;
    fetch(one, 0);
    for (int64_t k = 0; k < count; k += 2 * BATCH) {
        fetch(two, k + BATCH);
        walk(one, k);
        if (k + BATCH >= count) break;
        fetch(one, k + 2 * BATCH);
        walk(two, k + BATCH);
    }
    if (MAPS && live)
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.maps[place + v] = make_float2(closed ? kClosed : A[v], h[v]);
}

// What each segment begins with: a block per 32 channels, its warps first join the maps of a run of segments each, then walk their run again.
template <bool BACKWARD> __global__ void __launch_bounds__(1024) recurrence_carries_kernel(const RecurrenceParams p) {
    __shared__ float2 runs[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t C = p.channels, c = (int64_t)blockIdx.x * 32 + lane, each = (p.segments + 31) / 32, begin = min(p.segments, warp * each), end = min(p.segments, begin + each);
    const bool live = c < C;
    auto at = [&](int64_t k) { return (BACKWARD ? p.segments - 1 - k : k) * C + (live ? c : 0); };
    float A = 1.f, B = 0.f;
    auto join = [&](float2 m) {
        if (m.x == kClosed) { A = kClosed; B = m.y; } else { B = fmaf(m.x, B, m.y); A = A == kClosed ? A : A * m.x; }
    };
#pragma unroll 8
    for (int64_t k = begin; k < end; ++k) join(p.maps[at(k)]);
    runs[warp][lane] = make_float2(A, B);
    __syncthreads();
    float h = 0.f;
    for (int w = 0; w < warp; ++w) h = runs[w][lane].x == kClosed ? runs[w][lane].y : fmaf(runs[w][lane].x, h, runs[w][lane].y);
#pragma unroll 8
    for (int64_t k = begin; k < end; ++k) {
        const float2 m = p.maps[at(k)];
        if (live) p.carries[at(k)] = h;
        h = m.x == kClosed ? m.y : fmaf(m.x, h, m.y);
    }
}

// Tokens of a segment.  Rows of one length where they give every SM sixteen warps, or are so short that a second walk would cost more than the
// first; else equal shares for sixteen warps an SM (by 128 channels of 16 bits, or 64 of 32), 32 tokens at least.
static int64_t segment_of(const nuka_b200_episodes_t& plan, int64_t channels) {
    const int64_t tiles = (channels + 127) / 128, wanted = 16 * 148;
    if (plan.length > 0 && (plan.length <= 64 || plan.rows * tiles >= wanted)) return plan.length;
    return plan.tokens <= 64 ? plan.tokens : std::max<int64_t>(32, (plan.tokens * tiles + wanted - 1) / wanted);
}
static bool on_its_own(int64_t segment, const nuka_b200_episodes_t& plan) { return plan.tokens <= segment || segment == plan.length; }

uint64_t recurrence_workspace(const nuka_b200_episodes_t& plan, int64_t channels) {
    const int64_t segment = segment_of(plan, channels);
    return on_its_own(segment, plan) ? 0u : (uint64_t)((plan.tokens + segment - 1) / segment * channels) * (sizeof(float2) + sizeof(float));
}

template <typename T, int VEC, bool BACKWARD> static cudaError_t run_recurrence(const nuka_b200_recurrence_t& d, cudaStream_t stream) {
    RecurrenceParams p{};
    p.plan = *d.plan;
    p.channels = d.channels; p.x_stride = d.x_stride; p.gate_stride = d.gate_stride;
    p.x = d.x; p.gate = d.gate; p.dh = d.dh; p.h = d.h; p.dx = d.dx; p.dgate = d.dgate;
    p.initial = d.initial; p.dstate = d.dstate; p.state = d.state; p.dinitial = d.dinitial;
    p.segment = segment_of(p.plan, d.channels);
    p.segments = (p.plan.tokens + p.segment - 1) / p.segment;
    p.tiles = (uint32_t)((d.channels + 32 * VEC - 1) / (32 * VEC));
    const unsigned blocks = (unsigned)((p.segments * p.tiles + kWalkers - 1) / kWalkers);
    if (!on_its_own(p.segment, p.plan)) {
        p.maps = static_cast<float2*>(d.workspace);
        p.carries = reinterpret_cast<float*>(p.maps + p.segments * d.channels);
        recurrence_kernel<T, VEC, BACKWARD, true><<<blocks, kWalkers * 32, 0, stream>>>(p);
        recurrence_carries_kernel<BACKWARD><<<(unsigned)((d.channels + 31) / 32), 1024, 0, stream>>>(p);
    }
    recurrence_kernel<T, VEC, BACKWARD, false><<<blocks, kWalkers * 32, 0, stream>>>(p);
    return cudaGetLastError();
}

template <typename T> static cudaError_t run_recurrence(const nuka_b200_recurrence_t& d, bool backward, cudaStream_t stream) {
    constexpr int W = kWide<T>;
    auto on = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    bool wide = d.channels % W == 0 && d.x_stride % W == 0 && d.gate_stride % W == 0;
    for (const void* p : {d.x, d.gate, static_cast<const void*>(d.h), d.dh, static_cast<const void*>(d.dx), static_cast<const void*>(d.dgate)}) wide = wide && on(p, W * sizeof(T));
    for (const float* p : {static_cast<const float*>(d.state), static_cast<const float*>(d.dinitial)}) wide = wide && on(p, W * sizeof(float));
    if (backward) return wide ? run_recurrence<T, W, true>(d, stream) : run_recurrence<T, 1, true>(d, stream);
    return wide ? run_recurrence<T, W, false>(d, stream) : run_recurrence<T, 1, false>(d, stream);
}

cudaError_t launch_recurrence(const nuka_b200_recurrence_t& d, bool backward, cudaStream_t stream) {
    if (d.plan->tokens == 0 || d.channels == 0) return cudaSuccess;
    return d.dtype == NUKA_B200_F32 ? run_recurrence<float>(d, backward, stream) : d.dtype == NUKA_B200_F16 ? run_recurrence<__half>(d, backward, stream) : run_recurrence<__nv_bfloat16>(d, backward, stream);
}

// ---- one token per env ---------------------------------------------------------------------------------------------
template <typename T, int VEC>
__global__ void recurrence_step_kernel(int64_t groups, uint32_t per_env, int64_t channels, const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gate, int64_t gate_stride,
                                       const uint8_t* __restrict__ fresh, float* __restrict__ state, T* __restrict__ h) {
    const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (g >= groups) return;
    const int64_t env = g / per_env, c = (g - env * per_env) * VEC, at = env * channels + c;
    float xv[VEC], gv[VEC], sv[VEC];
    unpack<T, VEC>(load_raw<T, VEC>(x + env * x_stride + c), xv);
    unpack<T, VEC>(load_raw<T, VEC>(gate + env * gate_stride + c), gv);
    unpack<float, VEC>(load_raw<float, VEC>(state + at), sv);
    const bool begins = fresh != nullptr && fresh[env] != 0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float a, rest;
        sigmoid<sizeof(T) == 4>(gv[v], a, rest);
        sv[v] = begins ? rest * xv[v] : fmaf(a, sv[v], rest * xv[v]);
    }
    store<float, VEC>(state + at, sv);
    store<T, VEC>(h + at, sv);
}

template <typename T> static cudaError_t run_step(int64_t n, int64_t channels, const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const uint8_t* fresh, float* state,
                                                  void* h, cudaStream_t stream) {
    auto fits = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    const bool four = channels % 4 == 0 && x_stride % 4 == 0 && gate_stride % 4 == 0 && fits(x, 4 * sizeof(T)) && fits(gate, 4 * sizeof(T)) && fits(h, 4 * sizeof(T)) && fits(state, 16);
    const int64_t groups = n * (four ? channels / 4 : channels);
    const unsigned blocks = (unsigned)((groups + 127) / 128);
    if (four) recurrence_step_kernel<T, 4><<<blocks, 128, 0, stream>>>(groups, (uint32_t)(channels / 4), channels, static_cast<const T*>(x), x_stride, static_cast<const T*>(gate), gate_stride, fresh, state, static_cast<T*>(h));
    else recurrence_step_kernel<T, 1><<<blocks, 128, 0, stream>>>(groups, (uint32_t)channels, channels, static_cast<const T*>(x), x_stride, static_cast<const T*>(gate), gate_stride, fresh, state, static_cast<T*>(h));
    return cudaGetLastError();
}

cudaError_t launch_recurrence_step(uint32_t dtype, int64_t n, int64_t channels, const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const uint8_t* fresh, float* state,
                                   void* h, cudaStream_t stream) {
    if (n == 0 || channels == 0) return cudaSuccess;
    return dtype == NUKA_B200_F32 ? run_step<float>(n, channels, x, x_stride, gate, gate_stride, fresh, state, h, stream)
         : dtype == NUKA_B200_F16 ? run_step<__half>(n, channels, x, x_stride, gate, gate_stride, fresh, state, h, stream)
                                  : run_step<__nv_bfloat16>(n, channels, x, x_stride, gate, gate_stride, fresh, state, h, stream);
}

}  // namespace nkb
