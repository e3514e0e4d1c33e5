// Gradients of an episode's first keys and values (sinks) from far queries.
//
// The keys' kernel has a tile of 128 keys and streams the queries past it that see one of them. Sinks are seen to their episode's end, the few of them in a tile of 128: streaming all of those queries past the tile would
// make that job as long as the episode is. So they are left out there, and worked out here, by products of eight keys: P^T = exp2(K Q^T - lse), dP^T = V dO^T, then dV^T += dO^T P and dK^T += Q^T dS, the eight keys the
// columns of the second products. Operands come 16 bytes to a lane straight from memory as in the history's kernel: the order of an inner dimension is free.
// The queries' bytes bound it, q and dO once for each eight sinks; what it takes is the chain of loads, scores, exponentials and products of sixteen queries, so a slot's queries and heads are dealt out over blocks and
// their warps, as many as the slots leave places for, and the sums joined in a fixed order: a block's warps in shared memory, then the splits.
//
// Measured, bf16, 8 heads, 2 of keys: 20011 tokens in 40 episodes, dim 64, window 64, 4 sinks: 15 us, 3 each for the slots before and the join behind (keys' kernel 60; with all queries of its sinks 115);
// 16384 tokens, one episode, dim 128, window 1024, 16 sinks: 30, 4 and 4 (keys' 218; 543). The second products' operands are the first ones', turned over by 8 x 8 in registers; loaded again in the other order they took 40 in place of 30.
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sinks.cuh"
#include "nkb_tcgen.cuh"

namespace nkb {

constexpr int kFarWarps = 4;

constexpr int far_blocks(int64_t dim) { return dim <= 64 ? 4 : 2; }          // of an SM

struct FarParams {
    const int32_t *first, *end;
    int64_t tokens, pitch, q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride;
    int heads_q, dim, window, sinks, span, tiles;
    float scale2;
    const void *q, *k, *v, *dout;
    const float *lse, *delta;
    FarSinks far;
};

struct FarRange { int first, count, from, past; };      // the tile's sinks, and their far queries
__device__ __forceinline__ FarRange far_range(const FarParams& p, int tile) {
    const int j0 = tile * p.span, last = (int)min((int64_t)j0 + p.span, p.tokens) - 1, first = p.first[last], end = p.end[last], begin = max(first, j0);
    return {begin, min(p.sinks - (begin - first), last - begin + 1), (int)min((int64_t)end, (int64_t)last + p.window), end};
}

// Which tiles have far queries: slots in the tiles' order. One block.
__global__ void __launch_bounds__(1024) far_plan_kernel(const FarParams p) {
    __shared__ int part[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int base = 0;
    for (int at = 0; at < p.tiles; at += 1024) {
        const int tile = at + threadIdx.x;
        bool is = false;
        if (tile < p.tiles) {
            const FarRange r = far_range(p, tile);
            is = r.count > 0 && r.past - r.from >= p.far.least;
        }
        const uint32_t which = __ballot_sync(~0u, is);
        if (lane == 0) part[warp] = __popc(which);
        __syncthreads();
        int before = base, all = base;
        for (int w = 0; w < 32; ++w) { if (w < warp) before += part[w]; all += part[w]; }
        const int slot = before + __popc(which & ((1u << lane) - 1u));
        if (tile < p.tiles) p.far.slot_of[tile] = is && slot < p.far.slots ? slot : -1;
        if (is && slot < p.far.slots) p.far.tile_of[slot] = tile;
        base = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const int count = min(base, p.far.slots);
        p.far.count[0] = count;
        p.far.count[1] = (int)max((int64_t)1, p.far.jobs / max((int64_t)1, (int64_t)count * p.far.groups * p.far.heads_k));
    }
}

// Sixteen queries of a head, numbers g and g + 8 to a lane, 16 bytes of 8 columns at 32 c + 8 t; what is not there is 0. Statistics of queries 2 t, 2 t + 1 and 8 further.
template <typename T, int CHUNKS> struct FarQueries {
    uint4 q[2][CHUNKS], dout[2][CHUNKS];
    float lse[2][2], delta[2][2];
    __device__ __forceinline__ void load(const FarParams& p, int head, int i0, int past, int g, int t) {
        const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = i0 + 8 * half + g;
            const T *const from = static_cast<const T*>(p.q) + i * p.q_stride + head * p.q_head_stride + 8 * t, *const by = static_cast<const T*>(p.dout) + ((int64_t)i * p.heads_q + head) * p.dim + 8 * t;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const bool there = i < past && 32 * c + 8 * t < p.dim;
                q[half][c] = there ? load_raw<T, 8>(from + 32 * c) : none;
                dout[half][c] = there ? load_raw<T, 8>(by + 32 * c) : none;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int64_t own = head * p.pitch + min(i0 + 8 * half + 2 * t + s, past - 1);
                lse[half][s] = p.lse[own];
                delta[half][s] = p.delta[own];
            }
        }
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kFarWarps * 32, far_blocks(DP)) far_sinks_kernel(const FarParams p) {
    constexpr int CHUNKS = DP / 32;
    __shared__ float sums[kFarWarps / 2][2][kSinkRows][DP];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const FarSinks& far = p.far;
    const int group = p.heads_q / far.heads_k, splits = far.count[1];
    const int64_t jobs = (int64_t)far.count[0] * far.groups * far.heads_k * splits;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int split = (int)(job % splits), head_k = (int)(job / splits % far.heads_k), part = (int)(job / splits / far.heads_k % far.groups), slot = (int)(job / splits / far.heads_k / far.groups);
        const FarRange r = far_range(p, far.tile_of[slot]);
        const int sinks = min(kSinkRows, r.count - part * kSinkRows), first = r.first + part * kSinkRows;           // of this job; none or fewer where the tile has fewer
        // queries of the split, a multiple of 16; each warp takes its share of (head, 16 queries) in turn
        const int each = ((r.past - r.from) / splits + 16) / 16 * 16, from = (int)min((int64_t)r.past, r.from + (int64_t)split * each), past = (int)min((int64_t)r.past, (int64_t)from + each);
        const int steps = sinks > 0 ? (past - from + 15) / 16 : 0;
        // keys and values of sink g, 16 bytes of 8 columns: products of rows 8 to 15 are not used
        uint4 k[CHUNKS], v[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const bool there = g < sinks && 32 * c + 8 * t < p.dim;
            k[c] = there ? load_raw<T, 8>(static_cast<const T*>(p.k) + (int64_t)(first + g) * p.k_stride + head_k * p.k_head_stride + 32 * c + 8 * t) : none;
            v[c] = there ? load_raw<T, 8>(static_cast<const T*>(p.v) + (int64_t)(first + g) * p.v_stride + head_k * p.v_head_stride + 32 * c + 8 * t) : none;
        }
        // [c][u][0, 1] and [2, 3]: of column 32 c + 4 u + 8 (g / 2) + g % 2 and of the one two further, sinks 2 t and 2 t + 1
        float dk[CHUNKS][2][4] = {}, dv[CHUNKS][2][4] = {};
        for (int x = warp; x < steps * group; x += kFarWarps) {
            const int i0 = from + x % steps * 16;
            FarQueries<T, CHUNKS> now;
            now.load(p, head_k * group + x / steps, i0, past, g, t);
            // what is not there are zeros, and so are its probabilities: whatever lies behind the episode meets no product
            uint32_t probs[2], grads[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float score[4] = {}, prob[4] = {};      // sink g: queries 2 t and 2 t + 1
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    mma16816<T>(score, k[c].x, 0u, k[c].y, 0u, now.q[half][c].x, now.q[half][c].y);
                    mma16816<T>(score, k[c].z, 0u, k[c].w, 0u, now.q[half][c].z, now.q[half][c].w);
                    mma16816<T>(prob, v[c].x, 0u, v[c].y, 0u, now.dout[half][c].x, now.dout[half][c].y);
                    mma16816<T>(prob, v[c].z, 0u, v[c].w, 0u, now.dout[half][c].z, now.dout[half][c].w);
                }
                float a[2], b[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bool there = g < sinks && i0 + 8 * half + 2 * t + s < past;
                    a[s] = exp2_fast(fmaf(score[s], p.scale2, -now.lse[half][s]));
                    b[s] = there ? a[s] * (prob[s] - now.delta[half][s]) : 0.f;
                    a[s] = there ? a[s] : 0.f;
                }
                probs[half] = pack<T>(a[0], a[1]);
                grads[half] = pack<T>(b[0], b[1]);
            }
            // queries down, columns across -> columns down, queries 2 t and 2 t + 1 across, as the products' first operand
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                mma16816<T>(dv[c][0], transpose8(now.dout[0][c].x), transpose8(now.dout[0][c].y), transpose8(now.dout[1][c].x), transpose8(now.dout[1][c].y), probs[0], probs[1]);
                mma16816<T>(dv[c][1], transpose8(now.dout[0][c].z), transpose8(now.dout[0][c].w), transpose8(now.dout[1][c].z), transpose8(now.dout[1][c].w), probs[0], probs[1]);
                mma16816<T>(dk[c][0], transpose8(now.q[0][c].x), transpose8(now.q[0][c].y), transpose8(now.q[1][c].x), transpose8(now.q[1][c].y), grads[0], grads[1]);
                mma16816<T>(dk[c][1], transpose8(now.q[0][c].z), transpose8(now.q[0][c].w), transpose8(now.q[1][c].z), transpose8(now.q[1][c].w), grads[0], grads[1]);
            }
        }
        // the block's warps into one, half of them at a time
        auto each_sum = [&](auto use) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int column = 32 * c + 4 * u + 8 * (g / 2) + g % 2 + e / 2 * 2, sink = 2 * t + e % 2;
                        use(0, sink, column, dk[c][u][e]);
                        use(1, sink, column, dv[c][u][e]);
                    }
        };
#pragma unroll
        for (int half = kFarWarps / 2; half > 0; half /= 2) {
            if (warp >= half && warp < 2 * half) each_sum([&](int which, int sink, int column, float& x) { sums[warp - half][which][sink][column] = x; });
            __syncthreads();
            if (warp < half) each_sum([&](int which, int sink, int column, float& x) { x += sums[warp][which][sink][column]; });
            __syncthreads();
        }
        if (warp == 0) {
            float* const to = far.sums + job * (2 * kSinkRows * DP);
            each_sum([&](int which, int sink, int column, float& x) { to[(which * kSinkRows + sink) * DP + column] = x; });
        }
    }
}

// The splits' sums into the first one's, always in the same order: a lane has four of a job's sums, the block's warps a share of the splits each. `width`: floats of a job.
__global__ void __launch_bounds__(256) far_join_kernel(const FarSinks far, int width) {
    __shared__ float4 part[8][32];
    const int splits = far.count[1], lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t at = ((int64_t)blockIdx.x * 32 + lane) * 4, which = at / width;           // a block's are of one job: its width is a multiple of 128
    if (splits == 1 || which >= (int64_t)far.count[0] * far.groups * far.heads_k) return;
    float* const to = far.sums + which * splits * width + at % width;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = warp; s < splits; s += 8) {
        const float4 v = *reinterpret_cast<const float4*>(to + (int64_t)s * width);
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) { sum.x += part[w][lane].x; sum.y += part[w][lane].y; sum.z += part[w][lane].z; sum.w += part[w][lane].w; }
    *reinterpret_cast<float4*>(to) = sum;
}

// Far queries that a tile must have for its sinks to be worked out here, else the keys' kernel has all queries of its sinks: there a job is as long as the longest of them, here each eight sinks read all far queries once
// more. Up to 16 sinks a step of that kernel is enough, with more only those of long rows are worth it. Whole training steps in us, 8 heads, 2 of keys, dim 64, with 16, 32 and 64 sinks, here and there: one episode of 16384,
// window 256, 165, 175 and 196, and 1600; the same among twenty of 50 tokens 174, 188 and 220, and 1770; 8 of 4000, window 128, 214, 231 and 301, and 570; 40 of 500, window 64, 149 here, 169 and 174 there; 4096 of 24, window 8, 4 sinks, 390 here and 370 there; dim 128, 16384, window 1024, 473, 493 and 532, and 790. With more than 64 sinks always there.
constexpr int64_t kMostSinks = 64, kFewSinks = 16, kFewFar = 64, kManyFar = 1024;
static int64_t far_least(int64_t sinks) { return sinks <= kFewSinks ? kFewFar : kManyFar; }

// Slots at most: tiles whose last key's episode is so much longer than the window and has sinks in the tile.
static int64_t far_slots(const nuka_b200_attention_t& d, int64_t sinks, int span, int tiles) {
    const nuka_b200_episodes_t& e = *d.plan;
    const int64_t reach = std::min(d.window, e.tokens) + far_least(sinks);      // tokens of such an episode, at least
    if (sinks > kMostSinks || (e.length > 0 && (span % e.length == 0 || reach > e.length))) return 0;         // a tile's rows are whole, or too short
    const int64_t episodes = std::min(e.tokens / reach, e.length == 0 ? e.rows : e.tokens);
    return std::min<int64_t>(tiles, episodes * 2);      // fewer sinks than a tile has keys lie in two tiles at most
}
// As many jobs as there may be slots for, and room to split them where the GPU has more places.
static int64_t far_jobs(const nuka_b200_attention_t& d, int64_t slots, int groups) { return std::max<int64_t>(slots * groups * d.heads_k, 148 * far_blocks(d.dim)); }
static int64_t far_width(const nuka_b200_attention_t& d) { return 2 * kSinkRows * (d.dim <= 64 ? 64 : 128); }
static int64_t far_indexes(int64_t slots, int tiles) { return (tiles + slots + 2 + 3) / 4 * 4; }

uint64_t far_sinks_bytes(const nuka_b200_attention_t& d, int64_t sinks, int span, int tiles) {
    const int64_t slots = far_slots(d, sinks, span, tiles);
    return slots == 0 ? 0u : (uint64_t)(far_jobs(d, slots, (int)((sinks + kSinkRows - 1) / kSinkRows)) * far_width(d) + far_indexes(slots, tiles)) * 4u;
}

FarSinks far_sinks(const nuka_b200_attention_t& d, int64_t sinks, int span, int tiles, void* workspace) {
    FarSinks f;
    f.slots = (int)far_slots(d, sinks, span, tiles);
    f.least = (int)far_least(sinks);
    if (f.slots == 0) return f;
    f.groups = (int)((sinks + kSinkRows - 1) / kSinkRows);
    f.heads_k = (int)d.heads_k;
    f.jobs = far_jobs(d, f.slots, f.groups);
    f.slot_of = static_cast<int32_t*>(workspace);
    f.tile_of = f.slot_of + tiles;
    f.count = f.tile_of + f.slots;
    f.sums = reinterpret_cast<float*>(f.slot_of + far_indexes(f.slots, tiles));
    return f;
}

cudaError_t launch_far_sinks(const nuka_b200_attention_t& d, int window, int sinks, int span, int tiles, int64_t pitch, const FarSinks& far, cudaStream_t stream) {
    FarParams p{};
    p.first = d.plan->first; p.end = d.plan->end; p.tokens = d.plan->tokens; p.pitch = pitch;
    p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride; p.v_stride = d.v_stride; p.v_head_stride = d.v_head_stride;
    p.heads_q = (int)d.heads_q; p.dim = (int)d.dim; p.window = window; p.sinks = sinks; p.span = span; p.tiles = tiles; p.scale2 = d.scale * 1.4426950408889634f;
    p.q = d.q; p.k = d.k; p.v = d.v; p.dout = d.dout; p.lse = d.lse; p.delta = d.delta; p.far = far;
    far_plan_kernel<<<1, 1024, 0, stream>>>(p);
    const unsigned blocks = 148 * far_blocks(d.dim);
    if (d.dtype == NUKA_B200_F16) d.dim <= 64 ? far_sinks_kernel<__half, 64><<<blocks, kFarWarps * 32, 0, stream>>>(p) : far_sinks_kernel<__half, 128><<<blocks, kFarWarps * 32, 0, stream>>>(p);
    else d.dim <= 64 ? far_sinks_kernel<__nv_bfloat16, 64><<<blocks, kFarWarps * 32, 0, stream>>>(p) : far_sinks_kernel<__nv_bfloat16, 128><<<blocks, kFarWarps * 32, 0, stream>>>(p);
    const int64_t sums = (int64_t)far.slots * far.groups * far.heads_k * far_width(d);
    far_join_kernel<<<(unsigned)(sums / 128), 256, 0, stream>>>(far, (int)far_width(d));
    return cudaGetLastError();
}

}  // namespace nkb
