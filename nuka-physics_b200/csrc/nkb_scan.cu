// The selective scan over episodes: forwards, backwards, and for one token of each env.
//
//   dt = softplus(delta + bias), a = exp(dt A_cn), h_t = a h_{t-1} + dt x B_n, y = sum over n of C_n h + D x, out = y silu(gate)
//   dy = dout silu(gate), m_t = C_n dy + a_{t+1} m_{t+1}, dA = sum of m a h_{t-1} dt, dB = sum over c of m dt x, dC = sum over c of dy h, ddt = sum over n of m (a h_{t-1} A + x B), dx = sum over n of m dt B + D dy
//
// A warp has 32 / LN groups of four channels and LN groups of four states, a lane one of each: sixteen states of its own, so that what a token's channels share of its states (dt, x, dy) and its states of their
// channels (B, C) comes 16 bytes at a time, and sums over the states or the channels are partly a lane's own and partly a few exchanges, in which lanes give away half of their values each time.
// It walks a segment of tokens, kChunk at a time: first what needs no state, value by value (rates, gates), into shared memory, then the states token by token, then the outputs.
// Segments and maps are as in the gated recurrence: rows where they are short or many, else equal shares, walked once for what each does to the state, (exp(A sum dt), h), and a second time for the values.
// For a gradient the states before each chunk are kept, in the lanes' order; backwards a chunk's states are worked out again from them, into shared memory, and its tokens then walked back.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"
#include "nkb_tcgen.cuh"

namespace nkb {

constexpr int kScanWarps = 4;                           // of a block
constexpr float kToBase2 = 1.4426950408889634f, kFromBase2 = 0.6931471805599453f;

// LN: lanes over the states
template <int LN> struct ScanTile {
    static constexpr int kChannelLanes = 32 / LN, kChannels = 4 * kChannelLanes, kStates = 4 * LN;
    static constexpr int kChunk = LN == 4 || LN == 8 ? 8 : 4;
    static constexpr int kEach = kChunk * kChannels / 32, kNarrow = kChunk * kStates / 32;          // of a lane: values of a chunk, and of its B
    static constexpr int kCells = kChunk * kChannels;
};

struct ScanParams {
    nuka_b200_episodes_t plan;
    int64_t channels, states, x_stride, delta_stride, gate_stride, b_stride, c_stride, segment, segments, chunks;           // chunks: of a segment
    uint32_t tiles, workers;                            // of the channels; warps of a tile backwards
    bool alone;                                         // every segment is whole rows
    const void *x, *delta, *gate, *b, *c, *dy;
    const float *decay, *skip, *delta_bias, *initial, *dstate;
    void *y, *dx, *ddelta, *dgate;
    float *state, *dinitial;
    float4* kept;                                       // segments x chunks x tiles x 4 x 32
    float *maps, *sums;                                 // segments x tiles x 512, and segments x tiles x channels of a tile; below 0 where what came before is forgotten
    float *db, *dc;                                     // tiles x tokens x states of a tile, each
    float *ddecay, *dskip, *dbias;                      // workers x tiles x 512, and workers x tiles x channels of a tile
};

__device__ __forceinline__ float softplus(float u) { return u > 20.f ? u : log1pf(expf(u)); }                 // above, exp(-u) is less than half a unit of u
__device__ __forceinline__ float logistic(float u) { return 1.f / (1.f + expf(-u)); }

// Sums over the LANES lanes that lie STRIDE apart: each time a lane keeps half of its values, as long as it has some to give. Afterwards it has max(1, COUNT / LANES) of them, from `first` on.
template <int COUNT, int LANES, int STRIDE> __device__ __forceinline__ void sum_lanes(float (&v)[COUNT], int lane) {
    int n = COUNT;
#pragma unroll
    for (int m = LANES / 2; m >= 1; m /= 2) {
        if (n > 1) {
            n /= 2;
            const bool upper = (lane & m * STRIDE) != 0;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
                v[i] = keep + __shfl_xor_sync(~0u, give, m * STRIDE);
            }
        } else {
            v[0] += __shfl_xor_sync(~0u, v[0], m * STRIDE);
        }
    }
}
template <int COUNT, int LANES> struct Kept {
    static constexpr int kCount = COUNT > LANES ? COUNT / LANES : 1, kShare = LANES > COUNT ? LANES / COUNT : 1;
    static __device__ __forceinline__ int first(int group) { return group / kShare * kCount; }
    static __device__ __forceinline__ bool owner(int group) { return group % kShare == 0; }
};

template <typename T, int LN> struct ScanLane {
    using S = ScanTile<LN>;
    int lane, nl, cl;
    int64_t c0;                                         // the tile's first channel
    int count, states;                                  // channels and states that there are of the tile
    float rate[4][4];                                   // A log2(e)
    __device__ __forceinline__ ScanLane(const ScanParams& p, int64_t tile) {
        lane = threadIdx.x % 32; nl = lane % LN; cl = lane / LN;
        c0 = tile * S::kChannels;
        count = (int)min((int64_t)S::kChannels, p.channels - c0); states = (int)p.states;
        each(p.decay, 0, rate);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) rate[j][i] *= kToBase2;
    }
    // the lane's values of row `row` of rows x channels x states; 0 where there are none
    __device__ __forceinline__ void each(const float* from, int64_t row, float (&v)[4][4], int64_t channels = 0) const {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * cl + j, n = 4 * nl + i;
                v[j][i] = from != nullptr && c < count && n < states ? from[(row * channels + c0 + c) * states + n] : 0.f;
            }
    }
    __device__ __forceinline__ void give(float* to, int64_t row, const float (&v)[4][4], int64_t channels) const {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * cl + j, n = 4 * nl + i;
                if (c < count && n < states) to[(row * channels + c0 + c) * states + n] = v[j][i];
            }
    }
    // value number k of the lane's share of a chunk: its token and channel; of B or C: its token and state
    __device__ __forceinline__ int token_of(int k) const { return (lane + 32 * k) / S::kChannels; }
    __device__ __forceinline__ int channel_of(int k) const { return (lane + 32 * k) % S::kChannels; }
    __device__ __forceinline__ int narrow_token(int k) const { return (lane + 32 * k) / S::kStates; }
    __device__ __forceinline__ int narrow_state(int k) const { return (lane + 32 * k) % S::kStates; }
    // tokens t0 to t0 + left - 1
    __device__ __forceinline__ void load(const void* from, int64_t stride, int64_t t0, int left, T (&v)[S::kEach]) const {
#pragma unroll
        for (int k = 0; k < S::kEach; ++k) {
            const int t = token_of(k), c = channel_of(k);
            v[k] = t < left && c < count ? static_cast<const T*>(from)[(t0 + t) * stride + c0 + c] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void load_narrow(const void* from, int64_t stride, int64_t t0, int left, T (&v)[S::kNarrow]) const {
#pragma unroll
        for (int k = 0; k < S::kNarrow; ++k) {
            const int t = narrow_token(k), n = narrow_state(k);
            v[k] = t < left && n < states ? static_cast<const T*>(from)[(t0 + t) * stride + n] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ float bias(const ScanParams& p, int k) const { const int c = channel_of(k); return p.delta_bias != nullptr && c < count ? p.delta_bias[c0 + c] : 0.f; }
    __device__ __forceinline__ float skip(const ScanParams& p, int k) const { const int c = channel_of(k); return p.skip != nullptr && c < count ? p.skip[c0 + c] : 0.f; }
    __device__ __forceinline__ bool there(int k, int left) const { return token_of(k) < left && channel_of(k) < count; }
};

// What a warp's states read of a chunk.
template <int LN> struct __align__(16) ScanShared {
    using S = ScanTile<LN>;
    float dt[S::kCells], in[S::kCells], out[S::kCells];
    float b[S::kChunk * S::kStates], c[S::kChunk * S::kStates];
};
__device__ __forceinline__ void four(const float* from, float (&v)[4]) {
    const float4 f = *reinterpret_cast<const float4*>(from);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}

// A segment's sums of dt, of each channel those that lie in the lanes and numbers that have it.
template <int LN> __device__ __forceinline__ void give_totals(const ScanParams& p, ScanShared<LN>& m, const float (&total)[ScanTile<LN>::kEach], int lane, int64_t map, bool closed) {
    using S = ScanTile<LN>;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < S::kEach; ++k) m.out[lane + 32 * k] = total[k];
    __syncwarp();
    for (int ch = lane; ch < S::kChannels; ch += 32) {
        float sum = 0.f;
        for (int t = 0; t < S::kChunk; ++t) sum += m.out[t * S::kChannels + ch];
        p.sums[map * S::kChannels + ch] = closed ? -1.f : sum;
    }
}

// ---- forwards ----------------------------------------------------------------------------------------------------------
// MAPS: only what the segment does to the state
template <typename T, int LN, bool MAPS>
__global__ void __launch_bounds__(kScanWarps * 32) scan_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    __shared__ ScanShared<LN> all[kScanWarps];
    ScanShared<LN>& m = all[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, segment = job / p.tiles, tile = job % p.tiles;
    if (segment >= p.segments) return;
    const ScanLane<T, LN> l(p, tile);
    const int64_t begin = segment * p.segment, end = min(begin + p.segment, p.plan.tokens);
    float h[4][4] = {}, total[S::kEach] = {};           // total: of dt, of the lane's own values
    bool closed = false;
    float4* const maps = p.alone ? nullptr : reinterpret_cast<float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane;
    if (!MAPS && maps != nullptr)
#pragma unroll
        for (int j = 0; j < 4; ++j) { const float4 v = maps[32 * j]; h[j][0] = v.x; h[j][1] = v.y; h[j][2] = v.z; h[j][3] = v.w; }
    T x[S::kEach], delta[S::kEach], gate[S::kEach], b[S::kNarrow], c[S::kNarrow];
    int32_t link, tail;                                 // of token number `lane` of the chunk
    auto fetch = [&](int64_t t0) {
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        if (left <= 0) return;
        l.load(p.x, p.x_stride, t0, left, x);
        l.load(p.delta, p.delta_stride, t0, left, delta);
        l.load_narrow(p.b, p.b_stride, t0, left, b);
        if (!MAPS) l.load_narrow(p.c, p.c_stride, t0, left, c);
        if (!MAPS && p.gate != nullptr) l.load(p.gate, p.gate_stride, t0, left, gate);
        link = l.lane < left ? p.plan.link[t0 + l.lane] : -1;
        tail = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
    };
    fetch(begin);
    int64_t chunk = segment * p.chunks;
    for (int64_t t0 = begin; t0 < end; t0 += S::kChunk, ++chunk) {
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        const uint32_t begins = __ballot_sync(~0u, link != -1), ends = __ballot_sync(~0u, tail >= 0);
        const int32_t links = link, tails = tail;
        float xs[S::kEach], zs[S::kEach];
#pragma unroll
        for (int k = 0; k < S::kEach; ++k) {
            xs[k] = to_float<T>(x[k]);
            if (!MAPS && p.gate != nullptr) zs[k] = to_float<T>(gate[k]);
            const float dt = l.there(k, left) ? softplus(to_float<T>(delta[k]) + l.bias(p, k)) : 0.f;
            if (MAPS) total[k] += dt;
            m.dt[l.lane + 32 * k] = dt;
            m.in[l.lane + 32 * k] = dt * xs[k];
        }
#pragma unroll
        for (int k = 0; k < S::kNarrow; ++k) {
            m.b[l.lane + 32 * k] = to_float<T>(b[k]);
            if (!MAPS) m.c[l.lane + 32 * k] = to_float<T>(c[k]);
        }
        __syncwarp();
        fetch(t0 + S::kChunk);
        if (!MAPS && p.kept != nullptr)
#pragma unroll
            for (int j = 0; j < 4; ++j) p.kept[((chunk * p.tiles + tile) * 4 + j) * 32 + l.lane] = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
#pragma unroll 2
        for (int t = 0; t < left; ++t) {
            if (begins >> t & 1u) {
                const int32_t row = __shfl_sync(~0u, links, t);
                l.each(row >= 0 ? p.initial : nullptr, row, h, p.channels);
                closed = true;
            }
            float dt[4], in[4], bs[4];
            four(m.dt + t * S::kChannels + 4 * l.cl, dt);
            four(m.in + t * S::kChannels + 4 * l.cl, in);
            four(m.b + t * S::kStates + 4 * l.nl, bs);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) h[j][i] = fmaf(exp2_fast(dt[j] * l.rate[j][i]), h[j][i], in[j] * bs[i]);
            if constexpr (!MAPS) {
                float cs[4], y[4] = {};
                four(m.c + t * S::kStates + 4 * l.nl, cs);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[j] = fmaf(cs[i], h[j][i], y[j]);
                sum_lanes<4, LN, 1>(y, l.lane);
                using K = Kept<4, LN>;
                if (K::owner(l.nl))
#pragma unroll
                    for (int i = 0; i < K::kCount; ++i) m.out[t * S::kChannels + 4 * l.cl + K::first(l.nl) + i] = y[i];
                if (ends >> t & 1u) l.give(p.state, __shfl_sync(~0u, tails, t), h, p.channels);
            }
        }
        __syncwarp();
        if constexpr (!MAPS)
#pragma unroll
            for (int k = 0; k < S::kEach; ++k)
                if (l.there(k, left)) {
                    float y = fmaf(l.skip(p, k), xs[k], m.out[l.lane + 32 * k]);
                    if (p.gate != nullptr) y *= zs[k] * logistic(zs[k]);
                    static_cast<T*>(p.y)[(t0 + l.token_of(k)) * p.channels + l.c0 + l.channel_of(k)] = from_float<T>(y);
                }
    }
    if constexpr (MAPS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) maps[32 * j] = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
        give_totals<LN>(p, m, total, l.lane, segment * p.tiles + tile, closed);
    }
}

// What each segment begins with (backwards: what goes back into its last token), in place of its map: a block per 32 of a tile's 512 states, its warps a run of segments each, joined, then walked again.
template <int LN, bool BACKWARD> __global__ void __launch_bounds__(1024) scan_carries_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    __shared__ float2 runs[32][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t tile = blockIdx.x / 16, place = (blockIdx.x % 16) * 32 + lane, each = (p.segments + 31) / 32, begin = min(p.segments, warp * each), end = min(p.segments, begin + each);
    const int j = (int)place / 128, of = (int)place % 128 / 4, c = 4 * (of / LN) + j, n = 4 * (of % LN) + (int)place % 4;
    const int64_t channel = tile * S::kChannels + c;
    const float rate = channel < p.channels && n < p.states ? p.decay[channel * p.states + n] * kToBase2 : 0.f;
    auto map_of = [&](int64_t k) -> float& { return p.maps[((BACKWARD ? p.segments - 1 - k : k) * p.tiles + tile) * 512 + place]; };
    auto sum_of = [&](int64_t k) { return p.sums[((BACKWARD ? p.segments - 1 - k : k) * p.tiles + tile) * S::kChannels + c]; };
    float sum = 0.f, h = 0.f;                           // of the run so far; below 0: forgotten
#pragma unroll 4
    for (int64_t k = begin; k < end; ++k) {
        const float s = sum_of(k), v = map_of(k);
        if (s < 0.f) { sum = -1.f; h = v; } else { h = fmaf(exp2_fast(s * rate), h, v); sum = sum < 0.f ? sum : sum + s; }
    }
    runs[warp][lane] = make_float2(sum, h);
    __syncthreads();
    h = 0.f;
    for (int w = 0; w < warp; ++w) h = runs[w][lane].x < 0.f ? runs[w][lane].y : fmaf(exp2_fast(runs[w][lane].x * rate), h, runs[w][lane].y);
#pragma unroll 4
    for (int64_t k = begin; k < end; ++k) {
        const float s = sum_of(k), v = map_of(k);
        map_of(k) = h;
        h = s < 0.f ? v : fmaf(exp2_fast(s * rate), h, v);
    }
}

// ---- backwards -----------------------------------------------------------------------------------------------------------
template <int LN> struct __align__(16) ScanGradShared {
    using S = ScanTile<LN>;
    float4 before[S::kChunk * 4 * 32];                  // the states before each token, in the lanes' order
    float dt[S::kCells], in[S::kCells], dy[S::kCells], out[S::kCells], by_b[S::kCells], by_a[S::kCells];
    float b[S::kChunk * S::kStates], c[S::kChunk * S::kStates];
};

// What goes back through a segment from 0: m_t = C dy + a_{t+1} m_{t+1}, times a_t of its first token
template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32) scan_back_maps_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    __shared__ ScanShared<LN> all[kScanWarps];
    ScanShared<LN>& m = all[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, segment = job / p.tiles, tile = job % p.tiles;
    if (segment >= p.segments) return;
    const ScanLane<T, LN> l(p, tile);
    const int64_t begin = segment * p.segment, end = min(begin + p.segment, p.plan.tokens), chunks = (end - begin + S::kChunk - 1) / S::kChunk;
    float back[4][4] = {}, total[S::kEach] = {};
    bool closed = false;
    T dy[S::kEach], delta[S::kEach], gate[S::kEach], c[S::kNarrow];
    int32_t link, tail;
    auto fetch = [&](int64_t k) {
        if (k < 0) return;
        const int64_t t0 = begin + k * S::kChunk;
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        l.load(p.dy, p.channels, t0, left, dy);
        l.load(p.delta, p.delta_stride, t0, left, delta);
        if (p.gate != nullptr) l.load(p.gate, p.gate_stride, t0, left, gate);
        l.load_narrow(p.c, p.c_stride, t0, left, c);
        link = l.lane < left ? p.plan.link[t0 + l.lane] : -1;
        tail = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
    };
    fetch(chunks - 1);
    for (int64_t k0 = chunks - 1; k0 >= 0; --k0) {
        const int64_t t0 = begin + k0 * S::kChunk;
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        const uint32_t begins = __ballot_sync(~0u, link != -1), ends = __ballot_sync(~0u, tail >= 0);
        const int32_t tails = tail;
#pragma unroll
        for (int k = 0; k < S::kEach; ++k) {
            const float dt = l.there(k, left) ? softplus(to_float<T>(delta[k]) + l.bias(p, k)) : 0.f;
            float d = to_float<T>(dy[k]);
            if (p.gate != nullptr) { const float z = to_float<T>(gate[k]); d *= z * logistic(z); }
            total[k] += dt;
            m.dt[l.lane + 32 * k] = dt;
            m.in[l.lane + 32 * k] = d;
        }
#pragma unroll
        for (int k = 0; k < S::kNarrow; ++k) m.c[l.lane + 32 * k] = to_float<T>(c[k]);
        __syncwarp();
        fetch(k0 - 1);
#pragma unroll 2
        for (int t = left - 1; t >= 0; --t) {
            if (ends >> t & 1u) {
                float more[4][4];
                l.each(p.dstate, __shfl_sync(~0u, tails, t), more, p.channels);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) back[j][i] += more[j][i];
            }
            float dt[4], d[4], cs[4];
            four(m.dt + t * S::kChannels + 4 * l.cl, dt);
            four(m.in + t * S::kChannels + 4 * l.cl, d);
            four(m.c + t * S::kStates + 4 * l.nl, cs);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) back[j][i] = exp2_fast(dt[j] * l.rate[j][i]) * fmaf(d[j], cs[i], back[j][i]);
            if (begins >> t & 1u) {
                closed = true;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) back[j][i] = 0.f;
            }
        }
        __syncwarp();
    }
    float4* const maps = reinterpret_cast<float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) maps[32 * j] = make_float4(back[j][0], back[j][1], back[j][2], back[j][3]);
    give_totals<LN>(p, m, total, l.lane, segment * p.tiles + tile, closed);
}

template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32) scan_grad_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    extern __shared__ __align__(16) unsigned char raw[];
    ScanGradShared<LN>& m = reinterpret_cast<ScanGradShared<LN>*>(raw)[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, worker = job / p.tiles, tile = job % p.tiles;
    if (worker >= p.workers) return;
    const ScanLane<T, LN> l(p, tile);
    constexpr int OWN = S::kChannels > 32 ? S::kChannels / 32 : 1;         // channels of a lane where it has values
    float ddecay[4][4] = {}, dskip[OWN] = {}, dbias[OWN] = {};
    for (int64_t segment = worker; segment < p.segments; segment += p.workers) {
        const int64_t begin = segment * p.segment, end = min(begin + p.segment, p.plan.tokens), chunks = (end - begin + S::kChunk - 1) / S::kChunk;
        float back[4][4] = {};                          // a_{t+1} m_{t+1}
        if (!p.alone) {
            const float4* const maps = reinterpret_cast<const float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane;
#pragma unroll
            for (int j = 0; j < 4; ++j) { const float4 v = maps[32 * j]; back[j][0] = v.x; back[j][1] = v.y; back[j][2] = v.z; back[j][3] = v.w; }
        }
        for (int64_t k0 = chunks - 1; k0 >= 0; --k0) {
            const int64_t t0 = begin + k0 * S::kChunk, chunk = segment * p.chunks + k0;
            const int left = (int)min((int64_t)S::kChunk, end - t0);
            T x[S::kEach], delta[S::kEach], gate[S::kEach], dy[S::kEach], b[S::kNarrow], c[S::kNarrow];
            l.load(p.x, p.x_stride, t0, left, x);
            l.load(p.delta, p.delta_stride, t0, left, delta);
            l.load(p.dy, p.channels, t0, left, dy);
            if (p.gate != nullptr) l.load(p.gate, p.gate_stride, t0, left, gate);
            l.load_narrow(p.b, p.b_stride, t0, left, b);
            l.load_narrow(p.c, p.c_stride, t0, left, c);
            const int32_t links = l.lane < left ? p.plan.link[t0 + l.lane] : -1, tails = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
            const uint32_t begins = __ballot_sync(~0u, links != -1), ends = __ballot_sync(~0u, tails >= 0);
            float h[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { const float4 v = p.kept[((chunk * p.tiles + tile) * 4 + j) * 32 + l.lane]; h[j][0] = v.x; h[j][1] = v.y; h[j][2] = v.z; h[j][3] = v.w; }
            float slope[S::kEach], silu[S::kEach];      // softplus'(delta + bias), silu(gate)
#pragma unroll
            for (int k = 0; k < S::kEach; ++k) {
                const bool there = l.there(k, left);
                const float u = to_float<T>(delta[k]) + l.bias(p, k), dt = there ? softplus(u) : 0.f;
                slope[k] = logistic(u);
                silu[k] = 1.f;
                if (p.gate != nullptr) { const float z = to_float<T>(gate[k]); silu[k] = z * logistic(z); }
                m.dt[l.lane + 32 * k] = dt;
                m.in[l.lane + 32 * k] = dt * to_float<T>(x[k]);
                m.dy[l.lane + 32 * k] = there ? to_float<T>(dy[k]) * silu[k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < S::kNarrow; ++k) { m.b[l.lane + 32 * k] = to_float<T>(b[k]); m.c[l.lane + 32 * k] = to_float<T>(c[k]); }
            __syncwarp();
#pragma unroll 2
            for (int t = 0; t < left; ++t) {
                if (begins >> t & 1u) {
                    const int32_t row = __shfl_sync(~0u, links, t);
                    l.each(row >= 0 ? p.initial : nullptr, row, h, p.channels);
                }
                float dt[4], in[4], bs[4];
                four(m.dt + t * S::kChannels + 4 * l.cl, dt);
                four(m.in + t * S::kChannels + 4 * l.cl, in);
                four(m.b + t * S::kStates + 4 * l.nl, bs);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m.before[(t * 4 + j) * 32 + l.lane] = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[j][i] = fmaf(exp2_fast(dt[j] * l.rate[j][i]), h[j][i], in[j] * bs[i]);
                }
            }
#pragma unroll 1
            for (int t = left - 1; t >= 0; --t) {
                if (ends >> t & 1u) {
                    float more[4][4];
                    l.each(p.dstate, __shfl_sync(~0u, tails, t), more, p.channels);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) back[j][i] += more[j][i];
                }
                float dt[4], in[4], d[4], bs[4], cs[4];
                four(m.dt + t * S::kChannels + 4 * l.cl, dt);
                four(m.in + t * S::kChannels + 4 * l.cl, in);
                four(m.dy + t * S::kChannels + 4 * l.cl, d);
                four(m.b + t * S::kStates + 4 * l.nl, bs);
                four(m.c + t * S::kStates + 4 * l.nl, cs);
                float y[4] = {}, by_b[4] = {}, by_a[4] = {}, narrow[8] = {};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float before[4];
                    four(reinterpret_cast<const float*>(m.before + (t * 4 + j) * 32 + l.lane), before);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float grad = fmaf(d[j], cs[i], back[j][i]), a = exp2_fast(dt[j] * l.rate[j][i]);
                        const float kept = a * before[i], now = fmaf(in[j], bs[i], kept), through = grad * kept;
                        y[j] = fmaf(cs[i], now, y[j]);
                        narrow[4 + i] = fmaf(d[j], now, narrow[4 + i]);
                        narrow[i] = fmaf(in[j], grad, narrow[i]);
                        by_b[j] = fmaf(grad, bs[i], by_b[j]);
                        by_a[j] = fmaf(through, l.rate[j][i], by_a[j]);
                        ddecay[j][i] = fmaf(through, dt[j], ddecay[j][i]);
                        back[j][i] = a * grad;
                    }
                }
                if (begins >> t & 1u) {
                    const int32_t row = __shfl_sync(~0u, links, t);
                    if (row >= 0 && p.dinitial != nullptr) l.give(p.dinitial, row, back, p.channels);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) back[j][i] = 0.f;
                }
                sum_lanes<4, LN, 1>(y, l.lane);
                sum_lanes<4, LN, 1>(by_b, l.lane);
                sum_lanes<4, LN, 1>(by_a, l.lane);
                using K = Kept<4, LN>;
                if (K::owner(l.nl))
#pragma unroll
                    for (int i = 0; i < K::kCount; ++i) {
                        const int at = t * S::kChannels + 4 * l.cl + K::first(l.nl) + i;
                        m.out[at] = y[i];
                        m.by_b[at] = by_b[i];
                        m.by_a[at] = by_a[i] * kFromBase2;
                    }
                sum_lanes<8, S::kChannelLanes, LN>(narrow, l.lane);
                using N = Kept<8, S::kChannelLanes>;
                if (N::owner(l.cl))
#pragma unroll
                    for (int i = 0; i < N::kCount; ++i) {
                        const int which = N::first(l.cl) + i;
                        float* const to = which < 4 ? p.db : p.dc;
                        to[(tile * p.plan.tokens + t0 + t) * S::kStates + 4 * l.nl + which % 4] = narrow[i];
                    }
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < S::kEach; ++k) {
                if (!l.there(k, left)) continue;
                const int at = l.lane + 32 * k;
                const int64_t to = (t0 + l.token_of(k)) * p.channels + l.c0 + l.channel_of(k);
                const float xv = to_float<T>(x[k]), dyv = m.dy[at], skip = l.skip(p, k);
                if (p.gate != nullptr) {
                    const float z = to_float<T>(gate[k]), r = logistic(z), y = fmaf(skip, xv, m.out[at]);
                    static_cast<T*>(p.dgate)[to] = from_float<T>(to_float<T>(dy[k]) * y * (r * fmaf(z, 1.f - r, 1.f)));
                }
                const float du = fmaf(m.by_b[at], xv, m.by_a[at]) * slope[k];
                static_cast<T*>(p.dx)[to] = from_float<T>(fmaf(m.by_b[at], m.dt[at], skip * dyv));
                static_cast<T*>(p.ddelta)[to] = from_float<T>(du);
                dskip[k % OWN] = fmaf(dyv, xv, dskip[k % OWN]);
                dbias[k % OWN] += du;
            }
            __syncwarp();
        }
    }
    // lanes that have values of one channel
#pragma unroll
    for (int d = S::kChannels; d < 32; d *= 2) {
        dskip[0] += __shfl_xor_sync(~0u, dskip[0], d);
        dbias[0] += __shfl_xor_sync(~0u, dbias[0], d);
    }
    const int64_t at = worker * p.tiles + tile;
#pragma unroll
    for (int k = 0; k < OWN; ++k)
        if (l.lane + 32 * k < S::kChannels) {
            p.dskip[at * S::kChannels + l.lane + 32 * k] = dskip[k];
            p.dbias[at * S::kChannels + l.lane + 32 * k] = dbias[k];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(p.ddecay)[at * 128 + j * 32 + l.lane] = make_float4(ddecay[j][0], ddecay[j][1], ddecay[j][2], ddecay[j][3]);
}

// The workers' sums into one: a block per 32 of a tile's 512 decays and their channels' other sums.
template <int LN> __global__ void __launch_bounds__(1024) scan_sums_kernel(const ScanParams p, float* __restrict__ ddecay, float* __restrict__ dskip, float* __restrict__ ddelta_bias) {
    using S = ScanTile<LN>;
    __shared__ float part[32][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr int PARTS = 16 + 2 * ((S::kChannels + 31) / 32);
    const int64_t tile = blockIdx.x / PARTS;
    const int which = blockIdx.x % PARTS, extra = which - 16, other = extra / 2 * 32 + lane;        // of the channels
    const float* from = which < 16 ? p.ddecay + tile * 512 + which * 32 + lane : (extra % 2 ? p.dbias : p.dskip) + tile * S::kChannels + other;
    const int64_t step = (int64_t)p.tiles * (which < 16 ? 512 : S::kChannels);
    const bool live = which < 16 || other < S::kChannels;
    float sum = 0.f;
    if (live)
        for (uint32_t w = warp; w < p.workers; w += 32) sum += from[w * step];
    part[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || !live) return;
    sum = 0.f;
    for (int w = 0; w < 32; ++w) sum += part[w][lane];
    if (which < 16) {
        const int place = which * 32 + lane, of = place % 128 / 4, n = 4 * (of % LN) + place % 4;
        const int64_t c = tile * S::kChannels + 4 * (of / LN) + place / 128;
        if (c < p.channels && n < p.states && ddecay != nullptr) ddecay[c * p.states + n] = sum;
    } else if (const int64_t c = tile * S::kChannels + other; c < p.channels) {
        float* const to = extra % 2 ? ddelta_bias : dskip;
        if (to != nullptr) to[c] = sum;
    }
}

// The tiles' sums of B's and C's gradients into one.
template <typename T> __global__ void __launch_bounds__(256) scan_narrow_kernel(const ScanParams p, int width, T* __restrict__ db, T* __restrict__ dc) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, n = p.plan.tokens * width;
    if (at >= n || at % width >= p.states) return;
    float b = 0.f, c = 0.f;
#pragma unroll 4
    for (uint32_t k = 0; k < p.tiles; ++k) { b += p.db[k * n + at]; c += p.dc[k * n + at]; }
    const int64_t to = at / width * p.states + at % width;
    db[to] = from_float<T>(b);
    dc[to] = from_float<T>(c);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static int scan_lanes(int64_t states) { return states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : 16; }
static int64_t scan_chunk(int lanes) { return lanes == 4 || lanes == 8 ? 8 : 4; }

struct ScanShape {
    int lanes;
    int64_t tiles, channels, states, chunk, segment, segments, chunks, workers;
    bool alone;
    ScanShape(const nuka_b200_episodes_t& plan, int64_t all_channels, int64_t all_states) {
        lanes = scan_lanes(all_states); states = 4 * lanes; channels = 128 / lanes; chunk = scan_chunk(lanes);
        tiles = (all_channels + channels - 1) / channels;
        // rows of one length where they give every SM sixteen warps, or are so short that a second walk would cost more than the first; else equal shares for sixteen warps an SM, 64 tokens at least
        const int64_t wanted = 16 * 148;
        if (plan.length > 0 && (plan.length <= 64 || plan.rows * tiles >= wanted)) segment = plan.length;
        else segment = plan.tokens <= 64 ? plan.tokens : std::max<int64_t>(64, (plan.tokens * tiles / wanted + 7) / 8 * 8);
        segments = (plan.tokens + segment - 1) / segment;
        alone = plan.tokens <= segment || segment == plan.length;
        chunks = (segment + chunk - 1) / chunk;
        workers = std::max<int64_t>(1, std::min<int64_t>(segments, (12 * 148 + tiles - 1) / tiles));
    }
    uint64_t kept() const { return (uint64_t)(segments * chunks * tiles) * 2048u; }
    uint64_t maps() const { return alone ? 0u : (uint64_t)(segments * tiles) * (512u + (uint64_t)channels) * 4u; }
    uint64_t grads(int64_t tokens) const { return (uint64_t)(tiles * tokens * states) * 8u + (uint64_t)(workers * tiles) * (512u + 2u * (uint64_t)channels) * 4u; }
};

uint64_t scan_kept(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states) { return ScanShape(plan, channels, states).kept(); }
uint64_t scan_workspace(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states, bool backward) {
    const ScanShape s(plan, channels, states);
    return s.maps() + (backward ? s.grads(plan.tokens) : 0u);
}
int64_t scan_blocks(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states) { const ScanShape s(plan, channels, states); return s.segments * s.tiles / kScanWarps + 1; }

template <typename T, int LN> static cudaError_t run_scan(const nuka_b200_scan_t& d, bool backward, cudaStream_t stream) {
    const ScanShape s(*d.plan, d.channels, d.states);
    ScanParams p{};
    p.plan = *d.plan;
    p.channels = d.channels; p.states = d.states; p.x_stride = d.x_stride; p.delta_stride = d.delta_stride; p.gate_stride = d.gate_stride; p.b_stride = d.b_stride; p.c_stride = d.c_stride;
    p.segment = s.segment; p.segments = s.segments; p.chunks = s.chunks; p.tiles = (uint32_t)s.tiles; p.workers = (uint32_t)s.workers; p.alone = s.alone;
    p.x = d.x; p.delta = d.delta; p.gate = d.gate; p.b = d.b; p.c = d.c; p.dy = d.dy;
    p.decay = d.decay; p.skip = d.skip; p.delta_bias = d.delta_bias; p.initial = d.initial; p.dstate = d.dstate;
    p.y = d.y; p.dx = d.dx; p.ddelta = d.ddelta; p.dgate = d.dgate; p.state = d.state; p.dinitial = d.dinitial;
    p.kept = static_cast<float4*>(d.kept);
    float* work = static_cast<float*>(d.workspace);
    if (!s.alone) { p.maps = work; p.sums = work + s.segments * s.tiles * 512; work += s.maps() / 4; }
    const unsigned jobs = (unsigned)((s.segments * s.tiles + kScanWarps - 1) / kScanWarps), carries = (unsigned)(s.tiles * 16);
    if (!backward) {
        if (!s.alone) {
            scan_kernel<T, LN, true><<<jobs, kScanWarps * 32, 0, stream>>>(p);
            scan_carries_kernel<LN, false><<<carries, 1024, 0, stream>>>(p);
        }
        scan_kernel<T, LN, false><<<jobs, kScanWarps * 32, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const int64_t narrow = s.tiles * p.plan.tokens * s.states;
    p.db = work; p.dc = work + narrow; p.ddecay = work + 2 * narrow; p.dskip = p.ddecay + s.workers * s.tiles * 512; p.dbias = p.dskip + s.workers * s.tiles * s.channels;
    constexpr int SHARED = sizeof(ScanGradShared<LN>) * kScanWarps;
    const cudaError_t set = cudaFuncSetAttribute(scan_grad_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHARED);
    if (set != cudaSuccess) return set;
    if (!s.alone) {
        scan_back_maps_kernel<T, LN><<<jobs, kScanWarps * 32, 0, stream>>>(p);
        scan_carries_kernel<LN, true><<<carries, 1024, 0, stream>>>(p);
    }
    scan_grad_kernel<T, LN><<<(unsigned)((s.workers * s.tiles + kScanWarps - 1) / kScanWarps), kScanWarps * 32, SHARED, stream>>>(p);
    scan_sums_kernel<LN><<<(unsigned)(s.tiles * (16 + 2 * ((s.channels + 31) / 32))), 1024, 0, stream>>>(p, d.ddecay, d.dskip, d.ddelta_bias);
    scan_narrow_kernel<T><<<(unsigned)((p.plan.tokens * s.states + 255) / 256), 256, 0, stream>>>(p, (int)s.states, static_cast<T*>(d.db), static_cast<T*>(d.dc));
    return cudaGetLastError();
}

template <typename T> static cudaError_t run_scan(const nuka_b200_scan_t& d, bool backward, cudaStream_t stream) {
    switch (scan_lanes(d.states)) {
        case 2: return run_scan<T, 2>(d, backward, stream);
        case 4: return run_scan<T, 4>(d, backward, stream);
        case 8: return run_scan<T, 8>(d, backward, stream);
        default: return run_scan<T, 16>(d, backward, stream);
    }
}

cudaError_t launch_scan(const nuka_b200_scan_t& d, bool backward, cudaStream_t stream) {
    if (d.plan->tokens == 0) {                          // weights' gradients are sums of nothing
        cudaError_t set = cudaSuccess;
        const struct { float* at; int64_t count; } sums[] = {{d.ddecay, d.channels * d.states}, {d.dskip, d.channels}, {d.ddelta_bias, d.channels}};
        for (const auto& s : sums)
            if (backward && s.at != nullptr && set == cudaSuccess) set = cudaMemsetAsync(s.at, 0, (size_t)s.count * 4, stream);
        return set;
    }
    return d.dtype == NUKA_B200_F32 ? run_scan<float>(d, backward, stream) : d.dtype == NUKA_B200_F16 ? run_scan<__half>(d, backward, stream) : run_scan<__nv_bfloat16>(d, backward, stream);
}

// ---- one token per env ---------------------------------------------------------------------------------------------
// The states' bytes bound it: four states of a channel to a lane, LN lanes to a channel.
template <typename T, int LN, bool FOUR> __global__ void __launch_bounds__(128) scan_step_kernel(int64_t cells, const nuka_b200_scan_step_t d) {
    const int64_t at = (int64_t)blockIdx.x * 128 + threadIdx.x, cell = at / LN;
    const int nl = threadIdx.x % LN;
    const bool live = cell < cells;
    const int64_t env = live ? cell / d.channels : 0, ch = live ? cell % d.channels : 0;
    const bool begins = d.fresh != nullptr && d.fresh[env] != 0;
    float* const state = d.state + (env * d.channels + ch) * d.states + 4 * nl;
    const float* const decay = d.decay + ch * d.states + 4 * nl;
    const T *const b = static_cast<const T*>(d.b) + env * d.b_stride + 4 * nl, *const c = static_cast<const T*>(d.c) + env * d.c_stride + 4 * nl;
    const int count = live ? min(4, (int)d.states - 4 * nl) : 0;                  // below 1: none
    float h[4], rate[4];
    if (FOUR && count > 0) {
        four(state, h);
        four(decay, rate);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { h[i] = i < count ? state[i] : 0.f; rate[i] = i < count ? decay[i] : 0.f; }
    }
    const float x = to_float<T>(static_cast<const T*>(d.x)[env * d.x_stride + ch]);
    const float dt = softplus(to_float<T>(static_cast<const T*>(d.delta)[env * d.delta_stride + ch]) + (d.delta_bias != nullptr ? d.delta_bias[ch] : 0.f));
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float bv = i < count ? to_float<T>(b[i]) : 0.f, cv = i < count ? to_float<T>(c[i]) : 0.f, into = dt * x * bv;
        h[i] = begins ? into : fmaf(exp2_fast(dt * (rate[i] * kToBase2)), h[i], into);
        if (i < count) y = fmaf(cv, h[i], y);
    }
#pragma unroll
    for (int m = 1; m < LN; m *= 2) y += __shfl_xor_sync(~0u, y, m);
    if (FOUR && count > 0) {
        *reinterpret_cast<float4*>(state) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) state[i] = h[i];
    }
    if (!live || nl != 0) return;
    if (d.skip != nullptr) y = fmaf(d.skip[ch], x, y);
    if (d.gate != nullptr) { const float z = to_float<T>(static_cast<const T*>(d.gate)[env * d.gate_stride + ch]); y *= z * logistic(z); }
    static_cast<T*>(d.y)[env * d.channels + ch] = from_float<T>(y);
}

template <typename T, int LN> static cudaError_t run_scan_step(const nuka_b200_scan_step_t& d, cudaStream_t stream) {
    const int64_t cells = d.envs * d.channels;
    const unsigned blocks = (unsigned)((cells * LN + 127) / 128);
    const bool by_four = d.states % 4 == 0 && reinterpret_cast<uintptr_t>(d.state) % 16 == 0 && reinterpret_cast<uintptr_t>(d.decay) % 16 == 0;
    if (by_four) scan_step_kernel<T, LN, true><<<blocks, 128, 0, stream>>>(cells, d);
    else scan_step_kernel<T, LN, false><<<blocks, 128, 0, stream>>>(cells, d);
    return cudaGetLastError();
}

template <typename T> static cudaError_t run_scan_step(const nuka_b200_scan_step_t& d, cudaStream_t stream) {
    switch (scan_lanes(d.states)) {
        case 2: return run_scan_step<T, 2>(d, stream);
        case 4: return run_scan_step<T, 4>(d, stream);
        case 8: return run_scan_step<T, 8>(d, stream);
        default: return run_scan_step<T, 16>(d, stream);
    }
}

cudaError_t launch_scan_step(const nuka_b200_scan_step_t& d, cudaStream_t stream) {
    return d.dtype == NUKA_B200_F32 ? run_scan_step<float>(d, stream) : d.dtype == NUKA_B200_F16 ? run_scan_step<__half>(d, stream) : run_scan_step<__nv_bfloat16>(d, stream);
}

}  // namespace nkb
