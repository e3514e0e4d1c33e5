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
// multiplied with what came before, so that an infinity or NaN stays in its episode.
//
// A block takes a chunk of tokens by 32 * VEC channels, a warp of it TOK tokens, all loaded before the first is used.  Warps join their maps through
// shared memory, chunks through words in global memory: a chunk's map is published as one 64-bit word per channel that is valid as
// soon as it is not the fill pattern, so that nobody has to order two stores.  A chunk walks back over the maps of its group of kGroup chunks, to the group's
// first or to the last closed one, and takes the state that the group before ended with.  Where a walk stops
// depends on the plan alone, so the same call gives the same bits.  Chunks are handed out by a ticket: a block waits only for chunks
// whose blocks run already.
constexpr int kWarps = 8, kGroup = 32;
constexpr int64_t kWaitCycles = 4000000000ll;           // about 2 s; then the chunk goes on with NaN, and the call ends
constexpr uint64_t kHeader = 256;                       // ticket

__host__ __device__ constexpr int recurrence_chunk(bool backward) { return kWarps * (backward ? 8 : 16); }

struct RecurrenceParams {
    nuka_b200_episodes_t plan;
    int64_t channels, x_stride, gate_stride, padded;
    const void *x, *gate, *dh;
    void *h, *dx, *dgate;
    const float *initial, *dstate;
    float *state, *dinitial;
    uint32_t* ticket;                                   // null where one chunk holds all tokens
    unsigned long long* maps;                           // chunks x padded
    uint32_t* ends;                                     // groups x padded: the state that a group's last chunk ends with
    uint32_t tiles, chunks;
};

// 1 / (1 + exp(-g)) and 1 minus it, each without cancellation.  16-bit inputs and outputs leave the fast forms' 2^-21 far below their rounding.
template <bool EXACT> __device__ __forceinline__ void sigmoid(float g, float& a, float& rest) {
    const float e = EXACT ? expf(-fabsf(g)) : __expf(-fabsf(g));
    const float r = EXACT ? 1.f / (1.f + e) : __fdividef(1.f, 1.f + e);
    const float s = e * r;
    a = g >= 0.f ? r : s;
    rest = g >= 0.f ? s : r;
    if (g != g) a = rest = g;
}

__device__ __forceinline__ unsigned long long load_word(const unsigned long long* p) {
    unsigned long long v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void store_word(unsigned long long* p, unsigned long long v) { asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory"); }
__device__ __forceinline__ uint32_t load_word(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void store_word(uint32_t* p, uint32_t v) { asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }
// NaN in one spelling: the fill pattern is a NaN, too
__device__ __forceinline__ uint32_t bits_of(float v) { return v != v ? 0x7fffffffu : __float_as_uint(v); }
constexpr float kClosed = -1.f;                         // in the place of A, which is never negative

template <typename Word> __device__ Word wait_word(const Word* p, bool& lost) {
    Word v = load_word(p);
    if (v != ~Word(0)) return v;
    const int64_t began = clock64();
    while ((v = load_word(p)) == ~Word(0)) {
        if (clock64() - began > kWaitCycles) { lost = true; return v; }
        __nanosleep(20);
    }
    return v;
}

template <typename T, int VEC, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32) recurrence_kernel(const RecurrenceParams p) {
    constexpr int TOK = recurrence_chunk(BACKWARD) / kWarps, WIDTH = 32 * VEC;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ float map_a[kWarps][WIDTH], map_b[kWarps][WIDTH], carried[WIDTH];
    __shared__ uint32_t cuts_of[kWarps], ticket;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t block = blockIdx.x;
    if (p.ticket != nullptr) {
        if (threadIdx.x == 0) ticket = atomicAdd(p.ticket, 1u) + 1u;
        __syncthreads();
        block = ticket;
    }
    const uint32_t chunk = block / p.tiles, tile = block % p.tiles;
    const int64_t C = p.channels, tokens = p.plan.tokens, c = (int64_t)tile * WIDTH + lane * VEC;
    const bool live = c < C;                            // VEC divides the channels
    const int64_t s0 = ((int64_t)chunk * kWarps + warp) * TOK;
    auto token = [&](int i) -> int64_t { return BACKWARD ? tokens - 1 - (s0 + i) : s0 + i; };
    const int here = (int)max((int64_t)0, min((int64_t)TOK, tokens - s0));

    // which of the warp's tokens take nothing from the one before them (in scan order), and the rows that begin or end there
    int32_t link = -1, tail = -1;
    bool cut = false;
    if (lane < here) {
        const int64_t t = token(lane);
        link = p.plan.link[t];
        tail = p.plan.tail[t];
        cut = BACKWARD ? p.plan.end[t] == t + 1 : link != -1;
    }
    const uint32_t cuts = __ballot_sync(~0u, cut);

    const T *x = static_cast<const T*>(p.x) + c, *gate = static_cast<const T*>(p.gate) + c;
    float a[TOK][VEC], b[TOK][VEC], rest[BACKWARD ? TOK : 1][VEC], gap[BACKWARD ? TOK : 1][VEC];
    {
        Raw<T, VEC> rx[TOK], rg[TOK], rd[BACKWARD ? TOK : 1], rh[BACKWARD ? TOK : 1];
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const int32_t row = __shfl_sync(~0u, link, i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) b[i][v] = 0.f;
            if (live && i < here) {
                const int64_t t = token(i);
                rx[i] = load_raw<T, VEC>(x + t * p.x_stride);
                rg[i] = load_raw<T, VEC>(gate + t * p.gate_stride);
                if (BACKWARD) {
                    rd[i] = load_raw<T, VEC>(static_cast<const T*>(p.dh) + t * C + c);
                    if (row == -1) rh[i] = load_raw<T, VEC>(static_cast<const T*>(p.h) + (t - 1) * C + c);
                }
                // the state before a row's first token; elsewhere an episode's first token has 0 before it
                if (row >= 0 && p.initial != nullptr)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) b[i][v] = p.initial[(int64_t)row * C + c + v];
            }
        }
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const int32_t row = __shfl_sync(~0u, link, i);
            float xv[VEC], gv[VEC], out[VEC];
            unpack<T, VEC>(rx[i], xv);
            unpack<T, VEC>(rg[i], gv);
            if (BACKWARD) {
                float hv[VEC], dv[VEC];
                unpack<T, VEC>(rh[i], hv);
                unpack<T, VEC>(rd[i], dv);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    sigmoid<EXACT>(gv[v], a[i][v], rest[i][v]);
                    gap[i][v] = (row == -1 ? hv[v] : b[i][v]) - xv[v];
                    b[i][v] = dv[v];
                }
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float z;
                    sigmoid<EXACT>(gv[v], z, out[v]);
                    a[i][v] = z;
                    b[i][v] = row >= 0 && p.initial != nullptr ? fmaf(z, b[i][v], out[v] * xv[v]) : out[v] * xv[v];
                }
            }
            if (!live || i >= here)
#pragma unroll
                for (int v = 0; v < VEC; ++v) { a[i][v] = 1.f; b[i][v] = 0.f; }
        }
    }
    if (BACKWARD && p.dstate != nullptr)
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const int32_t row = __shfl_sync(~0u, tail, i);
            if (row >= 0 && live)
#pragma unroll
                for (int v = 0; v < VEC; ++v) b[i][v] += p.dstate[(int64_t)row * C + c + v];
        }

    // the warp's map.  Forwards h -> a h + b; backwards m -> a (m + b), m the gradient that goes on to the token before.
    float A[VEC], B[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
    for (int i = 0; i < TOK; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const bool shut = (cuts >> i) & 1u;
            if (BACKWARD) B[v] = a[i][v] * (shut ? b[i][v] : B[v] + b[i][v]);
            else B[v] = shut ? b[i][v] : fmaf(a[i][v], B[v], b[i][v]);
            A[v] = shut ? 0.f : A[v] * a[i][v];
        }
#pragma unroll
    for (int v = 0; v < VEC; ++v) { map_a[warp][lane * VEC + v] = A[v]; map_b[warp][lane * VEC + v] = B[v]; }
    if (lane == 0) cuts_of[warp] = cuts;
    __syncthreads();

    if (warp == 0) {
        float carry[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) carry[v] = 0.f;
        if (p.ticket != nullptr) {
            bool closed = false;
#pragma unroll
            for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
            for (int w = 0; w < kWarps; ++w) {
                const bool shut = cuts_of[w] != 0u;
                closed |= shut;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float ma = map_a[w][lane * VEC + v], mb = map_b[w][lane * VEC + v];
                    B[v] = shut ? mb : fmaf(ma, B[v], mb);
                    A[v] *= ma;
                }
            }
            const int64_t word = (int64_t)chunk * p.padded + (int64_t)tile * WIDTH + lane * VEC;
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                store_word(p.maps + word + v, (unsigned long long)bits_of(closed ? kClosed : A[v]) << 32 | bits_of(B[v]));
            const bool needs = chunk != 0u && !(cuts & 1u);
            const int64_t group = chunk / kGroup;
            if (needs) {
                bool lost = false, shut = false;
                float P[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) P[v] = 1.f;
                constexpr int AHEAD = 8;
                for (int64_t m = (int64_t)chunk - 1; m >= group * kGroup && !shut; m -= AHEAD) {
                    unsigned long long got[AHEAD][VEC];
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                        for (int v = 0; v < VEC; ++v)
                            got[k][v] = m - k >= group * kGroup ? load_word(p.maps + (m - k) * p.padded + (int64_t)tile * WIDTH + lane * VEC + v) : 0ull;
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k) {
                        if (m - k < group * kGroup || shut) break;
                        bool last = false;
#pragma unroll
                        for (int v = 0; v < VEC; ++v) {
                            unsigned long long w = got[k][v];
                            if (w == ~0ull) w = wait_word(p.maps + (m - k) * p.padded + (int64_t)tile * WIDTH + lane * VEC + v, lost);
                            const float ma = __uint_as_float((uint32_t)(w >> 32)), mb = __uint_as_float((uint32_t)w);
                            carry[v] = fmaf(P[v], mb, carry[v]);
                            last = ma == kClosed;
                            P[v] *= ma;
                        }
                        shut = last;
                    }
                }
                if (!shut && group != 0)
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        carry[v] = fmaf(P[v], __uint_as_float(wait_word(p.ends + (group - 1) * p.padded + (int64_t)tile * WIDTH + lane * VEC + v, lost)), carry[v]);
                if (lost)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) carry[v] = __uint_as_float(0x7fffffffu);
            }
            if (chunk % kGroup == kGroup - 1 && chunk + 1 < p.chunks)
#pragma unroll
                for (int v = 0; v < VEC; ++v) store_word(p.ends + group * p.padded + (int64_t)tile * WIDTH + lane * VEC + v, bits_of(closed ? B[v] : fmaf(A[v], carry[v], B[v])));
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) carried[lane * VEC + v] = carry[v];
    }
    __syncthreads();

    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = carried[lane * VEC + v];
    for (int w = 0; w < warp; ++w) {
        const bool shut = cuts_of[w] != 0u;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float mb = map_b[w][lane * VEC + v];
            h[v] = shut ? mb : fmaf(map_a[w][lane * VEC + v], h[v], mb);
        }
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        const int32_t begins = __shfl_sync(~0u, link, i), ends = __shfl_sync(~0u, tail, i);
        if (i >= here || !live) continue;
        const int64_t at = token(i) * C + c;
        const bool shut = (cuts >> i) & 1u;
        if (BACKWARD) {
            float dx[VEC], dg[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float grad = shut ? b[i][v] : h[v] + b[i][v];
                dx[v] = rest[i][v] * grad;
                dg[v] = dx[v] * gap[i][v] * a[i][v];
                h[v] = a[i][v] * grad;
            }
            store<T, VEC>(static_cast<T*>(p.dx) + at, dx);
            store<T, VEC>(static_cast<T*>(p.dgate) + at, dg);
            if (begins >= 0 && p.dinitial != nullptr)
#pragma unroll
                for (int v = 0; v < VEC; ++v) p.dinitial[(int64_t)begins * C + c + v] = h[v];
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = shut ? b[i][v] : fmaf(a[i][v], h[v], b[i][v]);
            store<T, VEC>(static_cast<T*>(p.h) + at, h);
            if (ends >= 0)
#pragma unroll
                for (int v = 0; v < VEC; ++v) p.state[(int64_t)ends * C + c + v] = h[v];
        }
    }
}

static int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

static uint64_t workspace_of(bool backward, int64_t tokens, int64_t channels) {
    const int64_t chunks = (tokens + recurrence_chunk(backward) - 1) / recurrence_chunk(backward), padded = round_up(channels, 64);
    return chunks <= 1 ? 0 : kHeader + chunks * padded * 8 + (chunks + kGroup - 1) / kGroup * padded * 4;
}

uint64_t recurrence_workspace(uint32_t, int64_t tokens, int64_t channels) { return std::max(workspace_of(false, tokens, channels), workspace_of(true, tokens, channels)); }

template <typename T, int VEC> static cudaError_t run_recurrence(const nuka_b200_recurrence_t& d, bool backward, cudaStream_t stream) {
    RecurrenceParams p{};
    p.plan = *d.plan;
    p.channels = d.channels; p.x_stride = d.x_stride; p.gate_stride = d.gate_stride;
    p.x = d.x; p.gate = d.gate; p.dh = d.dh; p.h = d.h; p.dx = d.dx; p.dgate = d.dgate;
    p.initial = d.initial; p.dstate = d.dstate; p.state = d.state; p.dinitial = d.dinitial;
    p.tiles = (uint32_t)((d.channels + 32 * VEC - 1) / (32 * VEC));
    p.padded = round_up(d.channels, 64);
    p.chunks = (uint32_t)((p.plan.tokens + recurrence_chunk(backward) - 1) / recurrence_chunk(backward));
    if (p.chunks > 1u) {
        unsigned char* w = static_cast<unsigned char*>(d.workspace);
        p.ticket = reinterpret_cast<uint32_t*>(w);
        p.maps = reinterpret_cast<unsigned long long*>(w + kHeader);
        p.ends = reinterpret_cast<uint32_t*>(w + kHeader + (uint64_t)p.chunks * p.padded * 8);
        const cudaError_t filled = cudaMemsetAsync(w, 0xff, workspace_of(backward, p.plan.tokens, d.channels), stream);
        if (filled != cudaSuccess) return filled;
    }
    const unsigned blocks = p.tiles * p.chunks;
    if (backward) recurrence_kernel<T, VEC, true><<<blocks, kWarps * 32, 0, stream>>>(p);
    else recurrence_kernel<T, VEC, false><<<blocks, kWarps * 32, 0, stream>>>(p);
    return cudaGetLastError();
}

static bool even(const void* p, size_t size) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % (2 * size) == 0; }

template <typename T> static cudaError_t run_recurrence(const nuka_b200_recurrence_t& d, bool backward, cudaStream_t stream) {
    const bool pairs = d.channels % 2 == 0 && d.x_stride % 2 == 0 && d.gate_stride % 2 == 0 && even(d.x, sizeof(T)) && even(d.gate, sizeof(T)) && even(d.h, sizeof(T)) &&
                       even(d.dh, sizeof(T)) && even(d.dx, sizeof(T)) && even(d.dgate, sizeof(T));
    return pairs ? run_recurrence<T, 2>(d, backward, stream) : run_recurrence<T, 1>(d, backward, stream);
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
