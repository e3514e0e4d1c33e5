// The selective scan over episodes: forwards, backwards, and for one token of each env.
//
//   dt = softplus(delta + bias), a = exp(dt A_cn), h_t = a h_{t-1} + dt x B_n, y = sum over n of C_n h + D x, out = y silu(gate)
//   dy = dout silu(gate), m_t = C_n dy + a_{t+1} m_{t+1}, dA = sum of m a h_{t-1} dt, dB = sum over c of m dt x, dC = sum over c of dy h, ddt = sum over n of m (a h_{t-1} A + x B), dx = sum over n of m dt B + D dy
//
// A warp has 32 / LN groups of four channels and LN groups of four states, a lane one of each: sixteen states of its own, so that what a token's channels share of its states (dt, x, dy) and its states of their
// channels (B, C) comes several at a time, and sums over the states or the channels are partly a lane's own and partly a few exchanges, in which lanes give away half of their values each time. Two neighbouring channels
// go through one instruction.
// It walks a segment of tokens, kChunk at a time: first what needs no state, eight values to a lane (rates, gates), into shared memory, then the states token by token, then the outputs, eight to a lane again.
// Segments and maps are as in the gated recurrence: rows where they are short or many, else equal shares, walked once for what each does to the state, (exp(A sum dt), h), and a second time for the values.
// For a gradient the states before each chunk are kept, in the lanes' order (2048 bytes for each chunk and tile: at 16 states 8 bytes for each value of x where rows are multiples of 8 tokens and channels of 32); backwards a chunk's states are worked out again from them, into shared memory, and its tokens then
// walked back. B's and C's gradients are sums over the channels: each tile leaves its own, in 32 bits, and a last kernel adds them up; so are A's and the other weights', by the warps' shares of the tokens. No atomics, every
// order is fixed.
//
// Measured, bf16, 16 states: 4096 rows of 24 x 512 370 us forwards and 1115 back, 51 more for B's and C's sums; 3 long rows, 32749 x 1024, 171 for the maps, 15 for the scan over them and 221 for the values, back 190, 17, 702 and 36;
// the same in f32 448, 1155 and 52, and 170, 17, 254, 213, 17, 721 and 36 (kernels of 8 and 16 states spill up to 80 bytes there); 1000 rows of 37 x 200, f32, 8 states 64 us; one token of 4096 envs x 512 63 us, 4.6 TB/s of its states.
// Exponentials bound it from below: one for each value and state forwards, two back, and a few for rates and gates, sixteen a cycle and SM, that is 224 us of the 370 and 414 of the 1115; their unit is busy for 61 % and 37 % of the time, the multiplying ones
// for 42 and 43 %. Forwards 16 warps share an SM, backwards 8 (201 KB of shared memory, with f32 and 64 states 214, and all registers), which leaves each warp's own chain of instructions in view: 1.9 of 4 a cycle.
#include <algorithm>
#include "nkb_gates.cuh"
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"

namespace nkb {

constexpr int kScanWarps = 4;                           // of a block
template <int N> struct Flag { static constexpr int value = N; };
constexpr float kToBase2 = 1.4426950408889634f, kFromBase2 = 0.6931471805599453f;
// Sums over tokens of one warp, term by term in 32 bits, are off by up to n 2^-24 of the terms' sizes. A warp with more than kLongSum tokens adds what it has to its share in memory every kFold tokens.
constexpr int64_t kLongSum = 4096;
constexpr int kFold = 1024;

// LN: lanes over the states
template <int LN> struct ScanTile {
    static constexpr int kChannelLanes = 32 / LN, kChannels = 4 * kChannelLanes, kStates = 4 * LN;
    static constexpr int kChunk = LN == 2 ? 4 : 8;
    // what a lane loads and works out of a chunk before and after the states: neighbouring channels of one token; of B and C neighbouring states
    static constexpr int kEach = kChunk * kChannels / 32, kNarrow = kChunk * kStates / 32;
    static constexpr int kRow = kChannels + 4;          // floats between a chunk's tokens in shared memory: neighbouring tokens' reads meet different banks
    static constexpr int kCells = kChunk * kRow;
};

struct ScanParams {
    nuka_b200_episodes_t plan;
    int64_t channels, states, x_stride, delta_stride, gate_stride, b_stride, c_stride, segment, segments, chunks;           // chunks: of a segment
    uint32_t tiles, workers;                            // of the channels; warps of a tile backwards
    bool alone;                                         // every segment is whole rows
    bool wide, wide_narrow, wide_states;                // a lane's loads and stores of a chunk go in one piece: of channels, and of B and C; those of states two at a time
    const void *x, *delta, *gate, *b, *c, *dy;
    const float *decay, *skip, *delta_bias, *initial, *dstate;
    void *y, *dx, *ddelta, *dgate;
    float *state, *dinitial;
    float4* kept;                                       // segments x chunks x tiles x 4 x 32
    float *maps, *sums;                                 // segments x tiles x 512, and segments x tiles x channels of a tile; below 0 where what came before is forgotten
    float* db;                                          // tiles x tokens x states of a tile, and the same of C
    int64_t dc_after;
    float *ddecay, *dskip, *dbias;                      // workers x tiles x 512, and workers x tiles x channels of a tile
};

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
// The same of four values whose first two are the lane's to keep (States).
template <int LN> __device__ __forceinline__ void sum_states(Pair low, Pair high, float (&v)[2], int lane) {
    float give[2];
    split(low, v[0], v[1]);
    split(high, give[0], give[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] += __shfl_xor_sync(~0u, give[i], LN / 2);
    sum_lanes<2, LN / 2, 1>(v, lane);
}
template <int COUNT, int LANES> struct Kept {
    static constexpr int kCount = COUNT > LANES ? COUNT / LANES : 1, kShare = LANES > COUNT ? LANES / COUNT : 1;
    static __device__ __forceinline__ int first(int group) { return group / kShare * kCount; }
    static __device__ __forceinline__ bool owner(int group) { return group % kShare == 0; }
};

// N neighbouring values, in pieces of at most 16 bytes.
template <typename T, int N> struct Piece {
    static constexpr int kPer = sizeof(T) * N > 16 ? 16 / sizeof(T) : N, kCount = N / kPer;
    Raw<T, kPer> raw[kCount];
    __device__ __forceinline__ void load(const T* from, int there, bool wide) {
        if (wide && there >= N) {
#pragma unroll
            for (int k = 0; k < kCount; ++k) raw[k] = load_raw<T, kPer>(from + k * kPer);
        } else {
            T v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = k < there ? from[k] : from_float<T>(0.f);
#pragma unroll
            for (int k = 0; k < kCount; ++k) {
                float f[kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) f[e] = to_float<T>(v[k * kPer + e]);
                nkb::store<T, kPer>(reinterpret_cast<T*>(&raw[k]), f);
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int k = 0; k < kCount; ++k) {
            float f[kPer];
            unpack<T, kPer>(raw[k], f);
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[k * kPer + e] = f[e];
        }
    }
    static __device__ __forceinline__ void store(T* to, const float (&v)[N], int there, bool wide) {
        if (wide && there >= N) {
#pragma unroll
            for (int k = 0; k < kCount; ++k) {
                float f[kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) f[e] = v[k * kPer + e];
                nkb::store<T, kPer>(to + k * kPer, f);
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k < there) to[k] = from_float<T>(v[k]);
        }
    }
};

// A lane's sixteen states: h[j][i] are those of its pair j of channels for its state i. The lanes of the upper half of a channel group have its two pairs in the other order, and those of the upper half of the
// channel groups the two halves of their four states: what a lane gives away first of its sums then lies in the same registers in all lanes.
struct States {
    Pair h[2][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i] = pair_of(0.f, 0.f);
    }
    // in the lanes' order: four times 32 x 16 bytes, one of each state
    __device__ __forceinline__ void load(const float4* from) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(from + 32 * i);
            h[0][i] = v.x; h[1][i] = v.y;
        }
    }
    __device__ __forceinline__ void store(float4* to) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<ulonglong2*>(to + 32 * i) = make_ulonglong2(h[0][i], h[1][i]);
    }
};
__device__ __forceinline__ Pair exp2_pair(Pair v) {
    float a, b;
    split(v, a, b);
    return pair_of(exp2_fast(a), exp2_fast(b));
}
// How a lane's own order goes through its channels and states: upper_j, upper_i 0 or 2.
struct Order {
    int upper_j, upper_i;
    __device__ __forceinline__ void two_pairs(const float* from, Pair (&v)[2]) const {
        v[0] = *reinterpret_cast<const Pair*>(from + upper_j); v[1] = *reinterpret_cast<const Pair*>(from + 2 - upper_j);
    }
};
// B and C of a chunk as they come, four states of each one behind the other, once in each of the two orders of a lane's states.
template <typename T, int LN> struct __align__(16) NarrowShared {
    T of[2][ScanTile<LN>::kChunk][LN][8];
    // what a lane has of B (which 0) or C (1), from state `first` of token `t` on
    template <int N> __device__ __forceinline__ void put(int which, int t, int first, const T (&v)[N]) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                T turned[4] = {v[k + 2], v[k + 3], v[k], v[k + 1]}, same[4] = {v[k], v[k + 1], v[k + 2], v[k + 3]};
                *reinterpret_cast<Raw<T, 4>*>(&of[0][t][first / 4 + k / 4][4 * which]) = *reinterpret_cast<const Raw<T, 4>*>(same);
                *reinterpret_cast<Raw<T, 4>*>(&of[1][t][first / 4 + k / 4][4 * which]) = *reinterpret_cast<const Raw<T, 4>*>(turned);
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int n = first + k;
                of[0][t][n / 4][4 * which + n % 4] = v[k];
                of[1][t][n / 4][4 * which + (n % 4 ^ 2)] = v[k];
            }
        }
    }
    // each twice, as it meets two channels
    __device__ __forceinline__ void get(int upper, int t, int nl, Pair (&b)[4], Pair (&c)[4]) const {
        float f[8];
        if constexpr (sizeof(T) == 2) {
            unpack<T, 8>(load_raw<T, 8>(of[upper][t][nl]), f);
        } else {
            take4(of[upper][t][nl], f);
            take4(of[upper][t][nl] + 4, f + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { b[i] = both(f[i]); c[i] = both(f[4 + i]); }
    }
    __device__ __forceinline__ void get(int which, int upper, int t, int nl, Pair (&v)[4]) const {
        float f[4];
        unpack<T, 4>(load_raw<T, 4>(of[upper][t][nl] + 4 * which), f);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = both(f[i]);
    }
    static __device__ __forceinline__ void take4(const float* from, float* v) {
        const float4 q = *reinterpret_cast<const float4*>(from);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    }
};

template <typename T, int LN> struct ScanLane {
    using S = ScanTile<LN>;
    using Each = Piece<T, S::kEach>;
    using Narrow = Piece<T, S::kNarrow>;
    int lane, nl, cl;
    int64_t c0;                                         // the tile's first channel
    int count, states;                                  // channels and states that there are of the tile
    int token, channel, own;                            // of the lane's share of a chunk: its token, its first channel, and how many there are
    int narrow_token, narrow_state, narrow_own;
    Order order;
    States rate;                                        // A log2(e)
    __device__ __forceinline__ ScanLane(const ScanParams& p, int64_t tile) {
        lane = threadIdx.x % 32; nl = lane % LN; cl = lane / LN;
        order.upper_j = nl / (LN / 2) * 2; order.upper_i = cl / (S::kChannelLanes / 2) * 2;
        c0 = tile * S::kChannels;
        count = (int)min((int64_t)S::kChannels, p.channels - c0); states = (int)p.states;
        token = lane * S::kEach / S::kChannels; channel = lane * S::kEach % S::kChannels; own = count - channel;
        narrow_token = lane * S::kNarrow / S::kStates; narrow_state = lane * S::kNarrow % S::kStates; narrow_own = states - narrow_state;
        each(p, p.decay, 0, rate);
        const Pair to = pair_of(kToBase2, kToBase2);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) rate.h[j][i] = mul_pair(rate.h[j][i], to);
    }
    // the lane's values of row `row` of rows x channels x states; 0 where there are none
    __device__ __forceinline__ void each(const ScanParams& p, const float* from, int64_t row, States& v) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float f[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = 4 * cl + (2 * j ^ order.upper_j) + e;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const int n = 4 * nl + (i ^ order.upper_i);
                    const float* const at = from + (row * p.channels + c0 + c) * states + n;
                    const int there = from != nullptr && c < count ? states - n : 0;
                    if (p.wide_states && there >= 2) {
                        const float2 q = *reinterpret_cast<const float2*>(at);
                        f[e][i] = q.x; f[e][i + 1] = q.y;
                    } else {
                        f[e][i] = there > 0 ? at[0] : 0.f; f[e][i + 1] = there > 1 ? at[1] : 0.f;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v.h[j][i] = pair_of(f[0][i], f[1][i]);
        }
    }
    __device__ __forceinline__ void give(const ScanParams& p, float* to, int64_t row, const States& v) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float f[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split(v.h[j][i], f[0][i], f[1][i]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = 4 * cl + (2 * j ^ order.upper_j) + e;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const int n = 4 * nl + (i ^ order.upper_i);
                    float* const at = to + (row * p.channels + c0 + c) * states + n;
                    const int there = c < count ? states - n : 0;
                    if (p.wide_states && there >= 2) {
                        *reinterpret_cast<float2*>(at) = make_float2(f[e][i], f[e][i + 1]);
                    } else {
                        if (there > 0) at[0] = f[e][i];
                        if (there > 1) at[1] = f[e][i + 1];
                    }
                }
            }
        }
    }
    // tokens t0 to t0 + left - 1
    __device__ __forceinline__ void load(const ScanParams& p, const void* from, int64_t stride, int64_t t0, int left, Each& v) const {
        v.load(static_cast<const T*>(from) + (t0 + token) * stride + c0 + channel, token < left ? own : 0, p.wide);
    }
    __device__ __forceinline__ void load_narrow(const ScanParams& p, const void* from, int64_t stride, int64_t t0, int left, Narrow& v) const {
        v.load(static_cast<const T*>(from) + (t0 + narrow_token) * stride + narrow_state, narrow_token < left ? narrow_own : 0, p.wide_narrow);
    }
    __device__ __forceinline__ void store(const ScanParams& p, void* to, int64_t t0, int left, const float (&v)[S::kEach]) const {
        Each::store(static_cast<T*>(to) + (t0 + token) * p.channels + c0 + channel, v, token < left ? own : 0, p.wide);
    }
    // values per channel, of the lane's
    __device__ __forceinline__ void of_channels(const float* from, float (&v)[S::kEach]) const {
#pragma unroll
        for (int k = 0; k < S::kEach; ++k) v[k] = from != nullptr && k < own ? from[c0 + channel + k] : 0.f;
    }
    __device__ __forceinline__ float* cell(float* of) const { return of + token * S::kRow + channel; }
    __device__ __forceinline__ void put_narrow(NarrowShared<T, LN>& to, int which, const Narrow& v) const {
        T f[S::kNarrow];
#pragma unroll
        for (int k = 0; k < S::kNarrow; ++k) f[k] = reinterpret_cast<const T*>(&v.raw)[k];
        to.put(which, narrow_token, narrow_state, f);
    }
};
template <int N> __device__ __forceinline__ void put(float* to, const float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(to + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) to[k] = v[k];
    }
}
template <int N> __device__ __forceinline__ void take(const float* from, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 4) { const float4 q = *reinterpret_cast<const float4*>(from + k); v[k] = q.x; v[k + 1] = q.y; v[k + 2] = q.z; v[k + 3] = q.w; }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = from[k];
    }
}

// What a warp's states read of a chunk, and what they give.
template <typename T, int LN> struct __align__(16) ScanShared {
    using S = ScanTile<LN>;
    float dt[S::kCells], in[S::kCells], out[S::kCells];
    NarrowShared<T, LN> narrow;
};

// A segment's sums of dt: of each channel those of the lanes that have it.
template <typename T, int LN> __device__ __forceinline__ void give_totals(const ScanParams& p, ScanShared<T, LN>& m, float* cell, const float (&total)[ScanTile<LN>::kEach], int lane, int64_t map, bool closed) {
    using S = ScanTile<LN>;
    __syncwarp();
    put(cell, total);
    __syncwarp();
    for (int ch = lane; ch < S::kChannels; ch += 32) {
        float sum = 0.f;
        for (int t = 0; t < S::kChunk; ++t) sum += m.out[t * S::kRow + ch];
        p.sums[map * S::kChannels + ch] = closed ? -1.f : sum;
    }
}

// ---- forwards ----------------------------------------------------------------------------------------------------------
// MAPS: only what the segment does to the state
template <typename T, int LN, bool MAPS>
__global__ void __launch_bounds__(kScanWarps * 32, 4) scan_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    constexpr int E = S::kEach;
    __shared__ ScanShared<T, LN> all[kScanWarps];
    ScanShared<T, LN>& m = all[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, segment = job / p.tiles, tile = job % p.tiles;
    if (segment >= p.segments) return;
    const ScanLane<T, LN> l(p, tile);
    const int64_t begin = segment * p.segment, end = min(begin + p.segment, p.plan.tokens);
    States h;
    h.clear();
    float total[E] = {}, bias[E], skip[E];              // total: of dt, of the lane's own values
    l.of_channels(p.delta_bias, bias);
    l.of_channels(p.skip, skip);
    bool closed = false;
    float4* const maps = p.alone ? nullptr : reinterpret_cast<float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane;
    if (!MAPS && maps != nullptr) h.load(maps);
    typename ScanLane<T, LN>::Each x, delta, gate;
    typename ScanLane<T, LN>::Narrow b, c;
    int32_t link, tail;                                 // of token number `lane` of the chunk
    auto fetch = [&](int64_t t0) {
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        if (left <= 0) return;
        l.load(p, p.x, p.x_stride, t0, left, x);
        l.load(p, p.delta, p.delta_stride, t0, left, delta);
        l.load_narrow(p, p.b, p.b_stride, t0, left, b);
        if (!MAPS) l.load_narrow(p, p.c, p.c_stride, t0, left, c);
        if (!MAPS && p.gate != nullptr) l.load(p, p.gate, p.gate_stride, t0, left, gate);
        link = l.lane < left ? p.plan.link[t0 + l.lane] : -1;
        tail = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
    };
    fetch(begin);
    int64_t chunk = segment * p.chunks;
    for (int64_t t0 = begin; t0 < end; t0 += S::kChunk, ++chunk) {
        const int left = (int)min((int64_t)S::kChunk, end - t0), there = l.token < left ? l.own : 0;
        const uint32_t begins = __ballot_sync(~0u, link != -1), ends = __ballot_sync(~0u, tail >= 0);
        const int32_t links = link, tails = tail;
        typename ScanLane<T, LN>::Each x_now = x, gate_now = gate;
        {
            float xs[E], us[E];
            x.get(xs);
            delta.get(us);
#pragma unroll
            for (int k = 0; k < E; ++k) us[k] += bias[k];
            softplus_all(us, us);
#pragma unroll
            for (int k = 0; k < E; ++k) {
                xs[k] *= us[k];
                if (MAPS && there > 0) total[k] += us[k];
            }
            put(l.cell(m.dt), us);
            put(l.cell(m.in), xs);
        }
        l.put_narrow(m.narrow, 0, b);
        if (!MAPS) l.put_narrow(m.narrow, 1, c);
        __syncwarp();
        fetch(t0 + S::kChunk);
        if (!MAPS && p.kept != nullptr) h.store(p.kept + (chunk * p.tiles + tile) * 128 + l.lane);
        auto begin_at = [&](int t) {
            const int32_t row = __shfl_sync(~0u, links, t);
            if (row >= 0) l.each(p, p.initial, row, h); else h.clear();
            closed = true;
        };
        auto token = [&](int t) {
            Pair dt[2], in[2], bs[4];
            l.order.two_pairs(m.dt + t * S::kRow + 4 * l.cl, dt);
            l.order.two_pairs(m.in + t * S::kRow + 4 * l.cl, in);
            Pair cs[4];
            if constexpr (MAPS) m.narrow.get(0, l.order.upper_i / 2, t, l.nl, bs); else m.narrow.get(l.order.upper_i / 2, t, l.nl, bs, cs);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) h.h[j][i] = fma_pair(exp2_pair(mul_pair(dt[j], l.rate.h[j][i])), h.h[j][i], mul_pair(in[j], bs[i]));
            if constexpr (!MAPS) {
                Pair sum[2];
                float y[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    sum[j] = mul_pair(cs[0], h.h[j][0]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) sum[j] = fma_pair(cs[i], h.h[j][i], sum[j]);
                }
                sum_states<LN>(sum[0], sum[1], y, l.lane);
                using K = Kept<4, LN>;
                if (K::owner(l.nl))
#pragma unroll
                    for (int i = 0; i < K::kCount; ++i) m.out[t * S::kRow + 4 * l.cl + K::first(l.nl) + i] = y[i];
            }
        };
        // most chunks are whole, and nothing begins or ends but at their edges
        if (left == S::kChunk && (begins & ~1u) == 0u && (ends & ~(1u << (S::kChunk - 1))) == 0u) {
            if (begins != 0u) begin_at(0);
#pragma unroll
            for (int t = 0; t < S::kChunk; ++t) token(t);
            if (!MAPS && ends != 0u) l.give(p, p.state, __shfl_sync(~0u, tails, S::kChunk - 1), h);
        } else {
#pragma unroll 1
            for (int t = 0; t < left; ++t) {
                if (begins >> t & 1u) begin_at(t);
                token(t);
                if (!MAPS && ends >> t & 1u) l.give(p, p.state, __shfl_sync(~0u, tails, t), h);
            }
        }
        __syncwarp();
        if constexpr (!MAPS) {
            float y[E], xs[E];
            take(l.cell(m.out), y);
            x_now.get(xs);
#pragma unroll
            for (int k = 0; k < E; ++k) y[k] = fmaf(skip[k], xs[k], y[k]);
            if (p.gate != nullptr) {
                float z[E];
                gate_now.get(z);
                silu_all<sizeof(T) == 4>(z);
#pragma unroll
                for (int k = 0; k < E; ++k) y[k] *= z[k];
            }
            l.store(p, p.y, t0, left, y);
            __syncwarp();
        }
    }
    if constexpr (MAPS) {
        h.store(maps);
        give_totals<T, LN>(p, m, l.cell(m.out), total, l.lane, segment * p.tiles + tile, closed);
    }
}

// Of the 512 states of a tile in the lanes' order, number `place`: its channel and state.
template <int LN> __device__ __forceinline__ void place_of(int place, int& c, int& n) {
    const int of = place % 128 / 4, upper_j = of % LN / (LN / 2) * 2, upper_i = of / LN / (16 / LN) * 2;
    c = 4 * (of / LN) + (place % 4 ^ upper_j);
    n = 4 * (of % LN) + (place / 128 ^ upper_i);
}

// What each segment begins with (backwards: what goes back into its last token), in place of its map: a block per 32 of a tile's 512 states, its warps a run of segments each, joined, then walked again.
template <int LN, bool BACKWARD> __global__ void __launch_bounds__(1024) scan_carries_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    __shared__ float2 runs[32][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t tile = blockIdx.x / 16, each = (p.segments + 31) / 32, begin = min(p.segments, warp * each), end = min(p.segments, begin + each);
    const int place = (int)(blockIdx.x % 16) * 32 + lane;
    int c, n;
    place_of<LN>(place, c, n);
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
template <typename T, int LN> struct __align__(16) ScanGradShared {
    using S = ScanTile<LN>;
    float4 before[S::kChunk * 4 * 32];                  // the states before each token, in the lanes' order
    float dt[S::kCells], dy[S::kCells], slope[S::kCells], gate[S::kCells], out[S::kCells], by_a[S::kCells];         // slope: of dt; gate: what y's gradient of the gate is multiplied with
    float in[S::kCells];                                // dt x, and when the token is done sum of m B
    float bias[S::kChannels], skip[S::kChannels];       // of the tile's channels
    NarrowShared<T, LN> narrow;
};

// What goes back through a segment from 0: m_t = C dy + a_{t+1} m_{t+1}, times a_t of its first token
template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32, 4) scan_back_maps_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    constexpr int E = S::kEach;
    __shared__ ScanShared<T, LN> all[kScanWarps];
    ScanShared<T, LN>& m = all[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, segment = job / p.tiles, tile = job % p.tiles;
    if (segment >= p.segments) return;
    const ScanLane<T, LN> l(p, tile);
    const int64_t begin = segment * p.segment, end = min(begin + p.segment, p.plan.tokens), chunks = (end - begin + S::kChunk - 1) / S::kChunk;
    States back;
    back.clear();
    float total[E] = {}, bias[E];
    l.of_channels(p.delta_bias, bias);
    bool closed = false;
    typename ScanLane<T, LN>::Each dy, delta, gate;
    typename ScanLane<T, LN>::Narrow c;
    int32_t link, tail;
    auto fetch = [&](int64_t k) {
        if (k < 0) return;
        const int64_t t0 = begin + k * S::kChunk;
        const int left = (int)min((int64_t)S::kChunk, end - t0);
        l.load(p, p.dy, p.channels, t0, left, dy);
        l.load(p, p.delta, p.delta_stride, t0, left, delta);
        if (p.gate != nullptr) l.load(p, p.gate, p.gate_stride, t0, left, gate);
        l.load_narrow(p, p.c, p.c_stride, t0, left, c);
        link = l.lane < left ? p.plan.link[t0 + l.lane] : -1;
        tail = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
    };
    fetch(chunks - 1);
    for (int64_t k0 = chunks - 1; k0 >= 0; --k0) {
        const int64_t t0 = begin + k0 * S::kChunk;
        const int left = (int)min((int64_t)S::kChunk, end - t0), there = l.token < left ? l.own : 0;
        const uint32_t begins = __ballot_sync(~0u, link != -1), ends = __ballot_sync(~0u, tail >= 0);
        const int32_t tails = tail;
        {
            float us[E], ds[E];
            delta.get(us);
            dy.get(ds);
#pragma unroll
            for (int k = 0; k < E; ++k) us[k] += bias[k];
            softplus_all(us, us);
            if (there > 0)
#pragma unroll
                for (int k = 0; k < E; ++k) total[k] += us[k];
            if (p.gate != nullptr) {
                float z[E];
                gate.get(z);
                silu_all<sizeof(T) == 4>(z);
#pragma unroll
                for (int k = 0; k < E; ++k) ds[k] *= z[k];
            }
            put(l.cell(m.dt), us);
            put(l.cell(m.in), ds);
        }
        l.put_narrow(m.narrow, 1, c);
        __syncwarp();
        fetch(k0 - 1);
        auto end_at = [&](int t) {
            const int32_t row = __shfl_sync(~0u, tails, t);
            if (p.dstate == nullptr) return;
            States more;
            l.each(p, p.dstate, row, more);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) back.h[j][i] = add_pair(back.h[j][i], more.h[j][i]);
        };
        auto back_through = [&](int t) {
            Pair dt[2], d[2], cs[4];
            l.order.two_pairs(m.dt + t * S::kRow + 4 * l.cl, dt);
            l.order.two_pairs(m.in + t * S::kRow + 4 * l.cl, d);
            m.narrow.get(1, l.order.upper_i / 2, t, l.nl, cs);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) back.h[j][i] = mul_pair(exp2_pair(mul_pair(dt[j], l.rate.h[j][i])), fma_pair(d[j], cs[i], back.h[j][i]));
        };
        if (left == S::kChunk && (begins & ~1u) == 0u && (ends & ~(1u << (S::kChunk - 1))) == 0u) {
            if (ends != 0u) end_at(S::kChunk - 1);
#pragma unroll
            for (int t = S::kChunk - 1; t >= 0; --t) back_through(t);
            if (begins != 0u) { closed = true; back.clear(); }
        } else {
#pragma unroll 1
            for (int t = left - 1; t >= 0; --t) {
                if (ends >> t & 1u) end_at(t);
                back_through(t);
                if (begins >> t & 1u) { closed = true; back.clear(); }
            }
        }
        __syncwarp();
    }
    back.store(reinterpret_cast<float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane);
    give_totals<T, LN>(p, m, l.cell(m.out), total, l.lane, segment * p.tiles + tile, closed);
}

// FOLD: the weights' sums go to memory every kFold tokens, not only at the end. The check after each chunk costs 2 % (4096 rows of 24 x 512 1574 us in all, forwards too, and 1541 without), so where sums are short it is left out.
template <typename T, int LN, bool FOLD>
__global__ void __launch_bounds__(kScanWarps * 32, 2) scan_grad_kernel(const ScanParams p) {
    using S = ScanTile<LN>;
    constexpr int E = S::kEach;
    extern __shared__ __align__(16) unsigned char raw[];
    ScanGradShared<T, LN>& m = reinterpret_cast<ScanGradShared<T, LN>*>(raw)[threadIdx.x / 32];
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, worker = job / p.tiles, tile = job % p.tiles;
    if (worker >= p.workers) return;
    const ScanLane<T, LN> l(p, tile);
    States ddecay;
    ddecay.clear();
    float dskip[E] = {}, dbias[E] = {};
    for (int ch = l.lane; ch < S::kChannels; ch += 32) {
        m.bias[ch] = p.delta_bias != nullptr && ch < l.count ? p.delta_bias[l.c0 + ch] : 0.f;
        m.skip[ch] = p.skip != nullptr && ch < l.count ? p.skip[l.c0 + ch] : 0.f;
    }
    __syncwarp();
    // a chunk's inputs and the states before it: asked for while the last one's outputs are worked out
    typename ScanLane<T, LN>::Each x, delta, gate, dy;
    typename ScanLane<T, LN>::Narrow b, c;
    int32_t links, tails;
    States h, back;                                     // back: a_{t+1} m_{t+1}
    auto end_of = [&](int64_t segment) { return min((segment + 1) * p.segment, p.plan.tokens); };
    auto last_of = [&](int64_t segment) { return (end_of(segment) - segment * p.segment + S::kChunk - 1) / S::kChunk - 1; };
    auto fetch = [&](int64_t segment, int64_t k) {
        const int64_t t0 = segment * p.segment + k * S::kChunk;
        const int left = (int)min((int64_t)S::kChunk, end_of(segment) - t0);
        l.load(p, p.x, p.x_stride, t0, left, x);
        l.load(p, p.delta, p.delta_stride, t0, left, delta);
        l.load(p, p.dy, p.channels, t0, left, dy);
        if (p.gate != nullptr) l.load(p, p.gate, p.gate_stride, t0, left, gate);
        l.load_narrow(p, p.b, p.b_stride, t0, left, b);
        l.load_narrow(p, p.c, p.c_stride, t0, left, c);
        links = l.lane < left ? p.plan.link[t0 + l.lane] : -1;
        tails = l.lane < left ? p.plan.tail[t0 + l.lane] : -1;
        h.load(p.kept + ((segment * p.chunks + k) * p.tiles + tile) * 128 + l.lane);
    };
    int since = 0;                                      // tokens in the weights' sums
    bool before = false;                                // some are in the warp's share already
    auto leave = [&]() {
        // lanes that have values of the same channels, which lie as many apart as a token has
        constexpr int APART = S::kChannels / E;
#pragma unroll
        for (int d = APART; d < 32; d *= 2)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                dskip[k] += __shfl_xor_sync(~0u, dskip[k], d);
                dbias[k] += __shfl_xor_sync(~0u, dbias[k], d);
            }
        const int64_t at = worker * p.tiles + tile;
        float4* const decays = reinterpret_cast<float4*>(p.ddecay) + at * 128 + l.lane;
        float *const skips = p.dskip + at * S::kChannels + l.channel, *const biases = p.dbias + at * S::kChannels + l.channel;
        if (FOLD && before) {
            States sofar;
            sofar.load(decays);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) ddecay.h[j][i] = add_pair(ddecay.h[j][i], sofar.h[j][i]);
            if (l.lane < APART)
#pragma unroll
                for (int k = 0; k < E; ++k) { dskip[k] += skips[k]; dbias[k] += biases[k]; }
        }
        if (l.lane < APART) {
            put(skips, dskip);
            put(biases, dbias);
        }
        ddecay.store(decays);
        if (FOLD) {
            ddecay.clear();
#pragma unroll
            for (int k = 0; k < E; ++k) dskip[k] = dbias[k] = 0.f;
            since = 0;
            before = true;
        }
    };
    fetch(worker, last_of(worker));                     // workers are no more than segments
    for (int64_t segment = worker; segment < p.segments; segment += p.workers) {
        const int64_t begin = segment * p.segment, end = end_of(segment);
        back.clear();
        if (!p.alone) back.load(reinterpret_cast<const float4*>(p.maps) + (segment * p.tiles + tile) * 128 + l.lane);
        for (int64_t k0 = last_of(segment); k0 >= 0; --k0) {
            const int64_t t0 = begin + k0 * S::kChunk;
            const int left = (int)min((int64_t)S::kChunk, end - t0), there = l.token < left ? l.own : 0;
            const uint32_t begins = __ballot_sync(~0u, links != -1), ends = __ballot_sync(~0u, tails >= 0);
            {
                float xs[E], us[E], ds[E], bias[E];
                x.get(xs);
                delta.get(us);
                take(m.bias + l.channel, bias);
#pragma unroll
                for (int k = 0; k < E; ++k) us[k] += bias[k];
                softplus_all(us, us, bias);
#pragma unroll
                for (int k = 0; k < E; ++k) xs[k] *= us[k];
                put(l.cell(m.dt), us);
                put(l.cell(m.slope), bias);
                put(l.cell(m.in), xs);
                dy.get(ds);
                if (p.gate != nullptr) {
                    float z[E];
                    gate.get(z);
#pragma unroll
                    for (int k = 0; k < E; ++k) us[k] = ds[k];
                    by_silu_slope<sizeof(T) == 4>(z, us, ds);
                    put(l.cell(m.gate), us);
                }
                put(l.cell(m.dy), ds);
            }
            l.put_narrow(m.narrow, 0, b);
            l.put_narrow(m.narrow, 1, c);
            __syncwarp();
            auto begin_at = [&](int t) {
                const int32_t row = __shfl_sync(~0u, links, t);
                if (row >= 0) l.each(p, p.initial, row, h); else h.clear();
            };
            auto forth = [&](int t) {
                h.store(m.before + t * 128 + l.lane);
                Pair dt[2], in[2], bs[4];
                l.order.two_pairs(m.dt + t * S::kRow + 4 * l.cl, dt);
                l.order.two_pairs(m.in + t * S::kRow + 4 * l.cl, in);
                m.narrow.get(0, l.order.upper_i / 2, t, l.nl, bs);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) h.h[j][i] = fma_pair(exp2_pair(mul_pair(dt[j], l.rate.h[j][i])), h.h[j][i], mul_pair(in[j], bs[i]));
            };
            auto end_at = [&](int t) {
                const int32_t row = __shfl_sync(~0u, tails, t);
                if (p.dstate == nullptr) return;
                States more;
                l.each(p, p.dstate, row, more);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) back.h[j][i] = add_pair(back.h[j][i], more.h[j][i]);
            };
            auto begun_at = [&](int t) {
                const int32_t row = __shfl_sync(~0u, links, t);
                if (row >= 0 && p.dinitial != nullptr) l.give(p, p.dinitial, row, back);
                back.clear();
            };
            // where a lane's sums over the channels go: B's gradient or C's
            constexpr int HALF = S::kChannelLanes / 2;
            using N = Kept<4, HALF>;
            const int which = N::first(l.cl % HALF);
            float* const narrow_to = p.db + (which < 2 ? 0 : p.dc_after) + (tile * p.plan.tokens + t0) * S::kStates + 4 * l.nl + l.order.upper_i + which % 2;
            auto back_through = [&](int t) {
                Pair dt[2], in[2], d[2], bs[4], cs[4];
                l.order.two_pairs(m.dt + t * S::kRow + 4 * l.cl, dt);
                l.order.two_pairs(m.in + t * S::kRow + 4 * l.cl, in);
                l.order.two_pairs(m.dy + t * S::kRow + 4 * l.cl, d);
                m.narrow.get(l.order.upper_i / 2, t, l.nl, bs, cs);
                States before;
                before.load(m.before + t * 128 + l.lane);
                Pair y[2], by_b[2], by_a[2], to_b[4], to_c[4];
                auto add = [](bool first, Pair a, Pair b, Pair& sum) { sum = first ? mul_pair(a, b) : fma_pair(a, b, sum); };
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Pair grad = fma_pair(d[j], cs[i], back.h[j][i]), a = exp2_pair(mul_pair(dt[j], l.rate.h[j][i]));
                        const Pair kept = mul_pair(a, before.h[j][i]), now = fma_pair(in[j], bs[i], kept), through = mul_pair(grad, kept);
                        add(i == 0, cs[i], now, y[j]);
                        add(j == 0, d[j], now, to_c[i]);
                        add(j == 0, in[j], grad, to_b[i]);
                        add(i == 0, grad, bs[i], by_b[j]);
                        add(i == 0, through, l.rate.h[j][i], by_a[j]);
                        ddecay.h[j][i] = fma_pair(through, dt[j], ddecay.h[j][i]);
                        back.h[j][i] = mul_pair(a, grad);
                    }
                float sums[3][2], narrow[4];
                sum_states<LN>(y[0], y[1], sums[0], l.lane);
                sum_states<LN>(by_b[0], by_b[1], sums[1], l.lane);
                sum_states<LN>(by_a[0], by_a[1], sums[2], l.lane);
                __syncwarp();                           // all have read the token's dt x, whose place is written
                using K = Kept<4, LN>;
                if (K::owner(l.nl))
#pragma unroll
                    for (int i = 0; i < K::kCount; ++i) {
                        const int at = t * S::kRow + 4 * l.cl + K::first(l.nl) + i;
                        m.out[at] = sums[0][i];
                        m.in[at] = sums[1][i];
                        m.by_a[at] = sums[2][i];
                    }
                // of the channels' two halves the states' upper or lower two, then B's or C's
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float u, v, x, z;
                    split(to_b[i], u, v);
                    split(to_b[i + 2], x, z);
                    narrow[i] = u + v + __shfl_xor_sync(~0u, x + z, 16);
                    split(to_c[i], u, v);
                    split(to_c[i + 2], x, z);
                    narrow[2 + i] = u + v + __shfl_xor_sync(~0u, x + z, 16);
                }
                sum_lanes<4, HALF, LN>(narrow, l.lane);
                if (N::owner(l.cl % HALF))
#pragma unroll
                    for (int i = 0; i < N::kCount; ++i) (i < 2 ? narrow_to : narrow_to + p.dc_after)[t * S::kStates + i % 2] = narrow[i];
            };
            // the states again, then back through the tokens. CHECKED: something may begin or end in the midst, or the chunk end early
            auto walk = [&](auto checked) {
                constexpr bool CHECKED = decltype(checked)::value != 0;
                const int to = CHECKED ? left : S::kChunk;
                if (!CHECKED && begins != 0u) begin_at(0);
#pragma unroll 4
                for (int t = 0; t < to; ++t) {
                    if (CHECKED && begins >> t & 1u) begin_at(t);
                    forth(t);
                }
                if (!CHECKED && ends != 0u) end_at(S::kChunk - 1);
#pragma unroll 2
                for (int t = to - 1; t >= 0; --t) {
                    if (CHECKED && ends >> t & 1u) end_at(t);
                    back_through(t);
                    if (CHECKED && begins >> t & 1u) begun_at(t);
                }
                if (!CHECKED && begins != 0u) begun_at(0);
            };
            // most chunks are whole, and nothing begins or ends but at their edges
            if (left == S::kChunk && (begins & ~1u) == 0u && (ends & ~(1u << (S::kChunk - 1))) == 0u) walk(Flag<0>{}); else walk(Flag<1>{});
            __syncwarp();
            {
                float xs[E], us[E], ds[E], dt[E], by_b[E], out[E], skip[E];
                x.get(xs);
                if (k0 > 0) fetch(segment, k0 - 1);
                else if (const int64_t next = segment + p.workers; next < p.segments) fetch(next, last_of(next));
                take(l.cell(m.in), by_b);
                take(l.cell(m.by_a), us);
                take(l.cell(m.slope), out);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    us[k] = fmaf(by_b[k], xs[k], us[k] * kFromBase2) * out[k];
                    if (there > 0) dbias[k] += us[k];
                }
                l.store(p, p.ddelta, t0, left, us);
                take(l.cell(m.dy), ds);
                take(l.cell(m.dt), dt);
                take(m.skip + l.channel, skip);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    dskip[k] = fmaf(ds[k], xs[k], dskip[k]);       // 0 where there is no token
                    out[k] = fmaf(by_b[k], dt[k], skip[k] * ds[k]);
                }
                l.store(p, p.dx, t0, left, out);
                if (p.gate != nullptr) {
                    take(l.cell(m.out), out);
                    take(l.cell(m.gate), us);
#pragma unroll
                    for (int k = 0; k < E; ++k) out[k] = us[k] * fmaf(skip[k], xs[k], out[k]);
                    l.store(p, p.dgate, t0, left, out);
                }
            }
            __syncwarp();
            if (FOLD && ((since += S::kChunk) >= kFold || (k0 == 0 && segment + p.workers >= p.segments))) leave();
        }
    }
    if (!FOLD) leave();
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
        int c, n;
        place_of<LN>(which * 32 + lane, c, n);
        if (const int64_t channel = tile * S::kChannels + c; channel < p.channels && n < p.states && ddecay != nullptr) ddecay[channel * p.states + n] = sum;
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
    for (uint32_t k = 0; k < p.tiles; ++k) { b += p.db[k * n + at]; c += p.db[p.dc_after + k * n + at]; }
    const int64_t to = at / width * p.states + at % width;
    db[to] = from_float<T>(b);
    dc[to] = from_float<T>(c);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static int scan_lanes(int64_t states) { return states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : 16; }
static int64_t scan_chunk(int lanes) { return lanes == 2 ? 4 : 8; }

struct ScanShape {
    int lanes;
    int64_t tiles, channels, states, chunk, segment, segments, chunks, workers;
    bool alone;
    ScanShape(const nuka_b200_episodes_t& plan, int64_t all_channels, int64_t all_states) {
        lanes = scan_lanes(all_states); states = 4 * lanes; channels = 128 / lanes; chunk = scan_chunk(lanes);
        tiles = (all_channels + channels - 1) / channels;
        // rows of one length where they give every SM sixteen warps, or are so short that a second walk would cost more than the first (64 rows of 24 x 64 14 us whole and 23 cut, 16 of 48 x 512 21 and 27,
        // 8 of 64 x 64 23 and 21), of less than a chunk several together; else equal shares for sixteen warps an SM, 16 tokens at least
        const int64_t wanted = 16 * 148;
        if (plan.length > 0 && (plan.length <= 64 || plan.rows * tiles >= wanted)) segment = plan.length < 8 ? (15 + plan.length) / plan.length * plan.length : plan.length;
        else segment = plan.tokens <= 16 ? plan.tokens : std::max<int64_t>(16, (plan.tokens * tiles / wanted + 7) / 8 * 8);
        segments = (plan.tokens + segment - 1) / segment;
        alone = plan.tokens <= segment || (plan.length > 0 && segment % plan.length == 0);
        chunks = (segment + chunk - 1) / chunk;
        workers = std::max<int64_t>(1, std::min<int64_t>(segments, 8 * 148 / tiles));
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
    // a lane's share of a chunk: eight values (four with 32 states, two with 64), and of B and C four (one, eight, sixteen with 8, 32 and 64 states)
    using S = ScanTile<LN>;
    auto lies = [](const void* at, uint64_t on) { return reinterpret_cast<uintptr_t>(at) % on == 0u; };
    constexpr uint64_t EACH = std::min<uint64_t>(16, S::kEach * sizeof(T)), NARROW = std::min<uint64_t>(16, S::kNarrow * sizeof(T));
    p.wide_narrow = d.states % S::kNarrow == 0 && d.b_stride % S::kNarrow == 0 && d.c_stride % S::kNarrow == 0 && lies(d.b, NARROW) && lies(d.c, NARROW);
    p.wide = d.channels % S::kEach == 0;
    for (int64_t stride : {d.x_stride, d.delta_stride, d.gate_stride}) p.wide = p.wide && stride % S::kEach == 0;
    for (const void* at : {d.x, d.delta, d.gate, static_cast<const void*>(d.y)}) p.wide = p.wide && lies(at, EACH);
    if (backward)
        for (const void* at : {d.dy, static_cast<const void*>(d.dx), static_cast<const void*>(d.ddelta), static_cast<const void*>(d.dgate)}) p.wide = p.wide && lies(at, EACH);
    p.wide_states = d.states % 2 == 0;
    for (const float* at : {d.decay, d.initial, static_cast<const float*>(d.state)}) p.wide_states = p.wide_states && lies(at, 8);
    if (backward)
        for (const float* at : {d.dstate, static_cast<const float*>(d.dinitial)}) p.wide_states = p.wide_states && lies(at, 8);
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
    p.db = work; p.dc_after = narrow; p.ddecay = work + 2 * narrow; p.dskip = p.ddecay + s.workers * s.tiles * 512; p.dbias = p.dskip + s.workers * s.tiles * s.channels;
    constexpr int SHARED = sizeof(ScanGradShared<T, LN>) * kScanWarps;
    const auto grad = (s.segments + s.workers - 1) / s.workers * s.segment > kLongSum ? scan_grad_kernel<T, LN, true> : scan_grad_kernel<T, LN, false>;
    const cudaError_t set = cudaFuncSetAttribute(grad, cudaFuncAttributeMaxDynamicSharedMemorySize, SHARED);
    if (set != cudaSuccess) return set;
    if (!s.alone) {
        scan_back_maps_kernel<T, LN><<<jobs, kScanWarps * 32, 0, stream>>>(p);
        scan_carries_kernel<LN, true><<<carries, 1024, 0, stream>>>(p);
    }
    grad<<<(unsigned)((s.workers * s.tiles + kScanWarps - 1) / kScanWarps), kScanWarps * 32, SHARED, stream>>>(p);
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
    const int64_t tokens = d.plan->tokens;
    if (tokens == 0 || d.channels == 0) {               // weights' gradients, and those of B and C, are sums of nothing; what has no values is left alone
        const size_t size = d.dtype == NUKA_B200_F32 ? 4 : 2;
        cudaError_t set = cudaSuccess;
        const struct { void* at; size_t bytes; } sums[] = {{d.ddecay, (size_t)(d.channels * d.states) * 4}, {d.dskip, (size_t)d.channels * 4}, {d.ddelta_bias, (size_t)d.channels * 4},
                                                           {d.db, (size_t)(tokens * d.states) * size}, {d.dc, (size_t)(tokens * d.states) * size}};
        for (const auto& s : sums)
            if (backward && s.at != nullptr && s.bytes != 0 && set == cudaSuccess) set = cudaMemsetAsync(s.at, 0, s.bytes, stream);
        return set;
    }
    return d.dtype == NUKA_B200_F32 ? run_scan<float>(d, backward, stream) : d.dtype == NUKA_B200_F16 ? run_scan<__half>(d, backward, stream) : run_scan<__nv_bfloat16>(d, backward, stream);
}

// ---- one token per env ---------------------------------------------------------------------------------------------
// The states' bytes bound it. A warp has an env and a tile of channels, its lanes four channels of four states each, as over rollouts; what a channel's states share is worked out by one lane.
template <typename T, int LN> __global__ void __launch_bounds__(kScanWarps * 32, 6) scan_step_kernel(int64_t jobs, uint32_t tiles, bool wide, const nuka_b200_scan_step_t d) {
    constexpr int CHANNELS = 128 / LN, OWN = (CHANNELS + 31) / 32;
    __shared__ __align__(16) float shared[kScanWarps][3][CHANNELS];
    const int lane = threadIdx.x % 32, nl = lane % LN, cl = lane / LN;
    const int64_t job = (int64_t)blockIdx.x * kScanWarps + threadIdx.x / 32, env = job / tiles, c0 = job % tiles * CHANNELS;
    if (job >= jobs) return;
    float(&m)[3][CHANNELS] = shared[threadIdx.x / 32];
    const int count = (int)min((int64_t)CHANNELS, d.channels - c0), states = (int)d.states, there = states - 4 * nl;
    const bool begins = d.fresh != nullptr && d.fresh[env] != 0;
    float* const state = d.state + (env * d.channels + c0 + 4 * cl) * states + 4 * nl;
    const float* const decay = d.decay + (c0 + 4 * cl) * states + 4 * nl;
    float h[4][4], rate[4][4], b[4], c[4], x[OWN], z[OWN];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (wide && 4 * cl + j < count && there >= 4) {
            if (begins) { h[j][0] = h[j][1] = h[j][2] = h[j][3] = 0.f; } else take(state + j * states, h[j]);
            take(decay + j * states, rate[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool is = 4 * cl + j < count && i < there;
                h[j][i] = is && !begins ? state[j * states + i] : 0.f;
                rate[j][i] = is ? decay[j * states + i] : 0.f;
            }
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        b[i] = i < there ? to_float<T>(static_cast<const T*>(d.b)[env * d.b_stride + 4 * nl + i]) : 0.f;
        c[i] = i < there ? to_float<T>(static_cast<const T*>(d.c)[env * d.c_stride + 4 * nl + i]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < OWN; ++k)
        if (const int ch = lane + 32 * k; ch < count) {
            x[k] = to_float<T>(static_cast<const T*>(d.x)[env * d.x_stride + c0 + ch]);
            if (d.gate != nullptr) z[k] = to_float<T>(static_cast<const T*>(d.gate)[env * d.gate_stride + c0 + ch]);
            const float u = to_float<T>(static_cast<const T*>(d.delta)[env * d.delta_stride + c0 + ch]) + (d.delta_bias != nullptr ? d.delta_bias[c0 + ch] : 0.f), dt = softplus(u, fading<true>(u));
            m[0][ch] = dt * kToBase2;
            m[1][ch] = dt * x[k];
        } else if (ch < CHANNELS) {
            m[0][ch] = m[1][ch] = 0.f;
        }
    __syncwarp();
    float dt[4], in[4], y[4];
    take(m[0] + 4 * cl, dt);
    take(m[1] + 4 * cl, in);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[j][i] = fmaf(exp2_fast(dt[j] * rate[j][i]), h[j][i], in[j] * b[i]);
            if (begins) h[j][i] = in[j] * b[i];
            y[j] = fmaf(c[i], h[j][i], y[j]);
        }
        if (wide && 4 * cl + j < count && there >= 4) {
            put(state + j * states, h[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * cl + j < count && i < there) state[j * states + i] = h[j][i];
        }
    }
    sum_lanes<4, LN, 1>(y, lane);
    using K = Kept<4, LN>;
    if (K::owner(nl))
#pragma unroll
        for (int i = 0; i < K::kCount; ++i) m[2][4 * cl + K::first(nl) + i] = y[i];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < OWN; ++k)
        if (const int ch = lane + 32 * k; ch < count) {
            float out = m[2][ch];
            if (d.skip != nullptr) out = fmaf(d.skip[c0 + ch], x[k], out);
            if (d.gate != nullptr) out *= silu<sizeof(T) == 4>(z[k]);
            static_cast<T*>(d.y)[env * d.channels + c0 + ch] = from_float<T>(out);
        }
}

template <typename T, int LN> static cudaError_t run_scan_step(const nuka_b200_scan_step_t& d, cudaStream_t stream) {
    const int64_t tiles = (d.channels + 128 / LN - 1) / (128 / LN), jobs = d.envs * tiles;
    const bool wide = d.states % 4 == 0 && reinterpret_cast<uintptr_t>(d.state) % 16 == 0 && reinterpret_cast<uintptr_t>(d.decay) % 16 == 0;
    scan_step_kernel<T, LN><<<(unsigned)((jobs + kScanWarps - 1) / kScanWarps), kScanWarps * 32, 0, stream>>>(jobs, (uint32_t)tiles, wide, d);
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
