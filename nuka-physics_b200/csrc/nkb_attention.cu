// Causal attention over packed episodes, forwards and backwards, on the tensor cores.
//
// Rows of the products are 128 tokens that lie one behind the other, whatever episodes they belong to: a token i sees the keys max(first_i, i - window + 1)
// to i, both ends grow with i, so a tile of queries sees one range of keys, from the first one's first to the last one's own, and only
// the tiles at that range's ends need a mask.  Short episodes share a tile; no length is known to the host.
//
//   forwards    S = Q K^T, P = exp2(scale log2(e) S - m), O += P V, m the running maximum, at last O / sum P
//   queries     S, dP = dO V^T, dS = P (dP - D) with D = dO . O, dQ += dS K
//   keys        S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q over all heads of the key's group
//
// The backward pass works the scores out twice, once for the queries' gradients and once for the keys': 7 products in place of 5, and in return no gradient is summed
// through atomics, so that the same call gives the same bits, and the shared heads' sum stays in tensor memory.
// Warps have roles: one or two load tiles by TMA, one or two issue products, four for each tile turn scores into probabilities, a row to a thread;
// P and dS go back to tensor memory as the next product's operand in the inputs' type (their one rounding more; sums and statistics are in 32 bits).
// One tile's products run under the other's exponentials: forwards the two are one block's, backwards those of two blocks on an SM, and with wide heads, of which one block fills an SM,
// the next step's scores run under the present one's exponentials.
// A block stays for several jobs, its loads and products a step ahead of its rows.
//
// Measured, bf16, causal (8 heads, 2 of keys):
//                                                           forwards    queries     keys
//   98304 tokens in rows of 24, dim 64                         73 us      106        100        252 MB of inputs and outputs forwards: 3.4 TB/s
//   20011 tokens in 40 episodes, dim 64                        61          71        115
//   16384 tokens, one episode, dim 128                        435          --         --        550 GFLOP of visible pairs: 1.26 PFLOP/s
//   40000 tokens in 4 episodes, dim 128                       790        1200       2315        1.04, 1.02 and 0.71 PFLOP/s of visible pairs
// Long episodes are bound by the chain of a step, scores to exponentials to product, that each tile walks through: the tensor cores are busy for half of it.
// Short rows are bound by the same chain once a tile, with its loads and its rows' way out around it: 128 rows see 24 keys each, and a tile's product is
// mostly mask, so there neither the bytes nor the products are near their limits.
#include <cuda_runtime.h>
#include <algorithm>
#include "nkb_sequence.cuh"
#include "nkb_sequence.h"
#include "nkb_tcgen.cuh"

namespace nkb {

constexpr int kRows = 128;                              // tokens of a block's tile, a thread and a tensor-memory lane each
constexpr int kStream = 64;                             // tokens of a streamed tile of the backward pass
constexpr int kBlock = 192;                             // four warps of rows, one that loads, one that multiplies
constexpr float kLog2e = 1.4426950408889634f;

struct AttentionParams {
    const int32_t *first, *end;
    int64_t tokens, pitch;                              // pitch: floats between the heads' rows of lse and delta
    int heads_q, heads_k, dim, window;                  // window 0: all of the episode
    int span, tiles;                                    // tokens of a tile, at most 128, and how many tiles
    int split;                                          // blocks of a key job, a cluster, each with an equal share of the group's heads
    int by_heads, across, along;                        // of the forward kernel's jobs: tiles of two heads or of two stretches of tokens; jobs side by side, and behind one another
    float scale, scale2;                                // scale2: times log2(e)
    const void *q, *k, *v;
    int64_t q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride;
    void *out, *dq, *dk, *dv;
    const void* dout;
    float *lse, *delta;
};

__device__ __forceinline__ float nan_value() { return __uint_as_float(0x7fffffffu); }

// A tile of queries and a head; the longest of one long row first.  What it reads of the plan is looked at only when it is used, a job after it was asked for.
struct QueryJob {
    int i0, last, head, first;                          // queries i0 to last; first: the plan's, of the first
    __device__ __forceinline__ QueryJob(const AttentionParams& p, int job) {
        const int tile = job / p.heads_q;
        head = job - tile * p.heads_q;
        i0 = (p.tiles - 1 - tile) * p.span;
        last = (int)min((int64_t)i0 + p.span, p.tokens) - 1;
        first = p.first[i0];
    }
    __device__ __forceinline__ int begin(const AttentionParams& p) const { return p.window > 0 ? max(first, i0 - p.window + 1) : first; }             // of its keys
    __device__ __forceinline__ int steps(const AttentionParams& p) const { return (last - begin(p)) / kStream + 1; }
};

// One thread's row of 32-bit accumulators, times `by`, into DP or fewer values of T; whether all are finite.
template <typename T, int DP> __device__ __forceinline__ bool store_row(uint32_t at, float by, int dim, T* to) {
    float probe = 0.f;                                  // becomes NaN where a value is not finite
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
        uint32_t r[32];
        __syncwarp();
        tensor_load(at + c, r);
        wait_loads();
#pragma unroll
        for (int k = 0; k < 32; k += 8)
            if (to != nullptr && c + k < dim) {
#pragma unroll
                for (int e = 0; e < 8; ++e) probe = fmaf(__uint_as_float(r[k + e]), 0.f, probe);
                uint4 v;
                v.x = pack<T>(__uint_as_float(r[k]) * by, __uint_as_float(r[k + 1]) * by);
                v.y = pack<T>(__uint_as_float(r[k + 2]) * by, __uint_as_float(r[k + 3]) * by);
                v.z = pack<T>(__uint_as_float(r[k + 4]) * by, __uint_as_float(r[k + 5]) * by);
                v.w = pack<T>(__uint_as_float(r[k + 6]) * by, __uint_as_float(r[k + 7]) * by);
                *reinterpret_cast<uint4*>(to + c + k) = v;
            }
    }
    return probe == 0.f;
}

// ROWS x DP of one head: panels of 64 columns, each ROWS x 128 bytes
template <int ROWS, int DP> __device__ __forceinline__ void load_panels(unsigned char* to, const CUtensorMap* map, uint64_t* bar, int head, int token) {
#pragma unroll
    for (int c = 0; c < DP; c += 64) load_tile(to + c / 64 * ROWS * 128, map, bar, c, head, token);
}
// d = A B^T over DP inner columns: A 128 rows, B N rows, both as loaded
template <typename T, int N, int DP> __device__ __forceinline__ void multiply_rows(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int k = 0; k < DP; k += 16)
        multiply(d, inner_rows(a + k / 64 * kRows * 128 + k % 64 * 2), inner_rows(b + k / 64 * N * 128 + k % 64 * 2), product_of<T>(N, false), k != 0);
}
// d (+)= A B over N rows of B, A in tensor memory, `EACH` of its columns in a row, two values to a column, and those of the next ones twice as far
template <typename T, int N, int DP, int EACH = N> __device__ __forceinline__ void multiply_columns(uint32_t d, uint32_t a, uint32_t b, bool add) {
#pragma unroll
    for (int k = 0; k < N; k += 16) multiply_tensor(d, a + k / EACH * EACH + k % EACH / 2, outer_rows(b + k * 128, N * 128), product_of<T>(DP, true), add || k != 0);
}

// All lanes of a warp wait, and go on together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* lost) { return __all_sync(~0u, barrier_wait(bar, parity, lost)) != 0; }

// Which of the columns 0 to 31 lie between `from` and `to`.
__device__ __forceinline__ uint32_t columns_between(int from, int to) {
    const uint32_t above = from <= 0 ? ~0u : from > 31 ? 0u : ~0u << from, below = to < 0 ? 0u : to >= 31 ? ~0u : (2u << to) - 1u;
    return above & below;
}

// A row of 64-column panels of 128 rows, swizzled as TMA takes it: 16 bytes number `k` of row `row`.
__device__ __forceinline__ unsigned char* staged(unsigned char* tile, int row, int k) { return tile + k / 8 * kRows * 128 + row * 128 + ((k % 8) ^ (row % 8)) * 16; }
// A thread's row of 32-bit accumulators, times `by`, into a staged tile of T; whether all are finite.
template <typename T, int DP> __device__ __forceinline__ bool stage_row(uint32_t at, float by, unsigned char* tile, int row) {
    float probe = 0.f;                                  // becomes NaN where a value is not finite
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
        uint32_t r[32];
        tensor_load(at + c, r);
        wait_loads();
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) probe = fmaf(__uint_as_float(r[k + e]), 0.f, probe);
            uint4 v;
            v.x = pack<T>(__uint_as_float(r[k]) * by, __uint_as_float(r[k + 1]) * by);
            v.y = pack<T>(__uint_as_float(r[k + 2]) * by, __uint_as_float(r[k + 3]) * by);
            v.z = pack<T>(__uint_as_float(r[k + 4]) * by, __uint_as_float(r[k + 5]) * by);
            v.w = pack<T>(__uint_as_float(r[k + 6]) * by, __uint_as_float(r[k + 7]) * by);
            *reinterpret_cast<uint4*>(staged(tile, row, (c + k) / 8)) = v;
        }
    }
    return probe == 0.f;
}

// ---- rows that are not finite -----------------------------------------------------------------------------------------
// A product over a tile multiplies what a row does not see by 0, and 0 times an infinity or NaN is NaN: an episode that is not finite would reach the others of its tiles. And in f16 a dS above
// 65504 becomes an infinity. So a block remembers that a row came out not finite though its own statistics are, and when all its jobs are done, its pipeline at rest and no wait under way
// that could give up meanwhile, its warps go over its rows once more: of a row that is not finite the columns in question are worked out in 32 bits, from what the row sees and nothing else.
// A column that is not finite by its definition is left as it is, whichever of infinity and NaN it became; what shows that is read without a product: a visible value for the
// outputs; for the gradients a query's lse or D, which are not finite wherever its row of q or dO is not.
// A lane has four columns of the row's result, and of each 32 keys or queries one weight.
// 30000 finite tokens, 20000 of which some are infinite, and 700 (8 heads, 2 of keys, dim 64, bf16; 2.0 and 7.9 ms where all are finite): 2.0 to 133 ms forwards, 7.8 to 173 back, by what is
// infinite and where; 16384 tokens in f16 with most of dS beyond its range 95 ms back (1.6).
template <typename T> __device__ __forceinline__ float dot(const T* a, const T* b, int dim) {
    float s = 0.f;
    for (int c = 0; c < dim; c += 8) {
        float u[8], v[8];
        unpack<T, 8>(load_raw<T, 8>(a + c), u);
        unpack<T, 8>(load_raw<T, 8>(b + c), v);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fmaf(u[k], v[k], s);
    }
    return s;
}
template <typename T> __device__ __forceinline__ const T* query_row(const AttentionParams& p, int i, int head) { return static_cast<const T*>(p.q) + i * p.q_stride + head * p.q_head_stride; }
template <typename T> __device__ __forceinline__ const T* key_row(const AttentionParams& p, int j, int head) { return static_cast<const T*>(p.k) + j * p.k_stride + head * p.k_head_stride; }
template <typename T> __device__ __forceinline__ const T* value_row(const AttentionParams& p, int j, int head) { return static_cast<const T*>(p.v) + j * p.v_stride + head * p.v_head_stride; }
template <typename T> __device__ __forceinline__ const T* dout_row(const AttentionParams& p, int i, int head) { return static_cast<const T*>(p.dout) + ((int64_t)i * p.heads_q + head) * p.dim; }
__device__ __forceinline__ int first_key(const AttentionParams& p, int i) { return p.window > 0 ? max(p.first[i], i - p.window + 1) : p.first[i]; }
__device__ __forceinline__ int past_query(const AttentionParams& p, int j) { return p.window > 0 ? (int)min((int64_t)p.end[j], (int64_t)j + p.window) : p.end[j]; }

// Which of a lane's four values are not finite.
template <typename T> __device__ __forceinline__ uint32_t spoilt_of(uint2 v) {
    constexpr uint32_t E = __is_same(T, __nv_bfloat16) ? 0x7f80u : 0x7c00u;
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) m |= ((k < 2 ? v.x : v.y) >> (k % 2 * 16) & E) == E ? 1u << k : 0u;
    return m;
}
// The lane's four columns of a row of a result that this kernel wrote; none behind dim.
template <typename T> __device__ __forceinline__ uint2 result_of(const T* row, int dim, int lane) { return 4 * lane < dim ? __ldcg(reinterpret_cast<const uint2*>(row + 4 * lane)) : make_uint2(0u, 0u); }
template <typename T> __device__ __forceinline__ void give_columns(T* row, uint32_t which, const float (&sum)[4], float by, int lane) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (which >> k & 1u) row[4 * lane + k] = from_float<T>(sum[k] * by);
}
// sum += the weights of the lanes below `count` times their rows
template <typename T, typename Row> __device__ __forceinline__ void add_rows(float (&sum)[4], float weight, int count, int dim, int lane, Row row) {
#pragma unroll 4
    for (int k = 0; k < count; ++k) {
        const float by = __shfl_sync(~0u, weight, k);
        if (4 * lane < dim) {
            float v[4];
            unpack<T, 4>(load_raw<T, 4>(row(k) + 4 * lane), v);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(by, v[e], sum[e]);
        }
    }
}
constexpr uint32_t kFinal = 0xffffu;                    // first value of an output row whose lse is not finite: NaN as no conversion gives it

template <typename T> __device__ __noinline__ void mend_out(const AttentionParams& p, int i, int head, int lane) {
    T* const out = static_cast<T*>(p.out) + ((int64_t)i * p.heads_q + head) * p.dim;
    const uint2 is = result_of(out, p.dim, lane);
    uint32_t which = spoilt_of<T>(is);
    if (!__any_sync(~0u, which != 0u) || (__shfl_sync(~0u, is.x, 0) & 0xffffu) == kFinal) return;
    const int key_head = head / (p.heads_q / p.heads_k), low = first_key(p, i);
    for (int j = low; j <= i && __any_sync(~0u, which != 0u); j += 8)
#pragma unroll
        for (int k = 0; k < 8; ++k) which &= ~spoilt_of<T>(result_of(value_row<T>(p, min(j + k, i), key_head), p.dim, lane));
    if (!__any_sync(~0u, which != 0u)) return;
    float top = -INFINITY, total = 0.f, sum[4] = {};
    for (int j = low; j <= i; j += 32) {
        const int count = min(32, i - j + 1);
        const float score = lane < count ? dot(query_row<T>(p, i, head), key_row<T>(p, j + lane, key_head), p.dim) * p.scale2 : -INFINITY;
        float best = score;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, d));
        best = fmaxf(best, top);
        const float shift = best == -INFINITY ? 0.f : best, by = exp2f(top - shift), weight = exp2f(score - shift);
        total = fmaf(total, by, weight);                // the lane's own part
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] *= by;
        add_rows<T>(sum, weight, count, p.dim, lane, [&](int k) { return value_row<T>(p, j + k, key_head); });
        top = best;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
    give_columns(out, which, sum, 1.f / total, lane);
}

template <typename T> __device__ __noinline__ void mend_query_grad(const AttentionParams& p, int i, int head, int lane) {
    const float lse = p.lse[head * p.pitch + i], delta = __ldcg(p.delta + head * p.pitch + i);
    if (!isfinite(lse) || !isfinite(delta)) return;
    T* const dq = static_cast<T*>(p.dq) + ((int64_t)i * p.heads_q + head) * p.dim;
    const uint32_t which = spoilt_of<T>(result_of(dq, p.dim, lane));
    if (!__any_sync(~0u, which != 0u)) return;
    const int key_head = head / (p.heads_q / p.heads_k);
    float sum[4] = {};
    for (int j = first_key(p, i); j <= i; j += 32) {
        const int count = min(32, i - j + 1), own = min(j + lane, i);
        const float prob = exp2f(fmaf(dot(query_row<T>(p, i, head), key_row<T>(p, own, key_head), p.dim), p.scale2, -lse));
        const float weight = prob * (dot(dout_row<T>(p, i, head), value_row<T>(p, own, key_head), p.dim) - delta);
        add_rows<T>(sum, weight, count, p.dim, lane, [&](int k) { return key_row<T>(p, j + k, key_head); });
    }
    give_columns(dq, which, sum, p.scale, lane);
}

// values: the value's gradient, else the key's
template <typename T> __device__ __noinline__ void mend_key_grad(const AttentionParams& p, int j, int key_head, bool values, int lane) {
    T* const to = static_cast<T*>(values ? p.dv : p.dk) + ((int64_t)j * p.heads_k + key_head) * p.dim;
    uint32_t which = spoilt_of<T>(result_of(to, p.dim, lane));
    if (!__any_sync(~0u, which != 0u)) return;
    const int group = p.heads_q / p.heads_k, past = past_query(p, j);
    for (int head = key_head * group; head < (key_head + 1) * group; ++head)
        for (int i = j; i < past; i += 32) {
            const int64_t at = head * p.pitch + min(i + lane, past - 1);
            const bool unset = !isfinite(p.delta[at]);
            if (__any_sync(~0u, !isfinite(p.lse[at]) || (unset && !values))) return;
            for (uint32_t left = __ballot_sync(~0u, unset); left != 0u; left &= left - 1u) {
                which &= ~spoilt_of<T>(result_of(dout_row<T>(p, min(i + __ffs(left) - 1, past - 1), head), p.dim, lane));
                if (!__any_sync(~0u, which != 0u)) return;
            }
        }
    float sum[4] = {};
    for (int head = key_head * group; head < (key_head + 1) * group; ++head)
        for (int i = j; i < past; i += 32) {
            const int count = min(32, past - i), own = min(i + lane, past - 1);
            float weight = exp2f(fmaf(dot(query_row<T>(p, own, head), key_row<T>(p, j, key_head), p.dim), p.scale2, -p.lse[head * p.pitch + own]));
            if (!values) weight *= dot(dout_row<T>(p, own, head), value_row<T>(p, j, key_head), p.dim) - p.delta[head * p.pitch + own];
            add_rows<T>(sum, weight, count, p.dim, lane, [&](int k) { return values ? dout_row<T>(p, i + k, head) : query_row<T>(p, i + k, head); });
        }
    give_columns(to, which, sum, values ? 1.f : p.scale, lane);
}

// A block that gave up waits, again for a bounded time, for the loads that it still has under way; what they bring is not used.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const long long began = clock64();
    while (!barrier_try(bar, parity) && clock64() - began < kBarrierCycles) {}
}

// The last loads into a ring of `stages` buffers of which `used` were begun.
__device__ __forceinline__ void drain_ring(uint64_t* bars, int stages, int used) {
    for (int n = max(0, used - stages); n < used; ++n) drain(&bars[n % stages], n / stages & 1);
}

extern __shared__ unsigned char dynamic_shared[];
__device__ __forceinline__ unsigned char* aligned_shared() { return dynamic_shared + ((1024u - (shared_address(dynamic_shared) & 1023u)) & 1023u); }

// ---- forwards ---------------------------------------------------------------------------------------------------------
// A block takes jobs in turn: two tiles of queries, of two heads that share a key head or else of two neighbouring stretches of tokens, that meet the same keys, so that a tile of
// keys and values is loaded once for 256 rows.  While one tile's rows are at their exponentials the tensor cores work for the other's. Loads run ahead
// into the next job while the rows of the present one end. A row's scores of a step are taken into registers at once, so that the next step's are multiplied while its
// exponentials go on.
constexpr int kForward = 384;                           // two times four warps of rows, two that multiply, two that load
template <int N> struct Number { static constexpr int value = N; };

template <int DP> struct Forward {
    // keys of a step: as many as leave tensor memory room for the scores, P beside them and O, twice
    static constexpr int kStep = DP == 64 ? 128 : 80;
    static constexpr int kQueries = DP == 64 ? 2 : 1, kStages = DP == 64 ? 3 : 2;              // buffers
    static constexpr int kTile = kRows * DP * 2, kPart = kStep * DP * 2;
    static constexpr int kKeys = 2 * kQueries * kTile, kStaged = kKeys + 2 * kStages * kPart, kShared = kStaged + 2 * kTile + 1024;
    static constexpr int kProb = kStep, kOut = kStep + kStep / 2, kSet = 256;                  // columns; the scores are at 0
    // Rows leave under the next job's exponentials, for which P is held back; wide heads, whose P goes out as it comes, have not the registers (their jobs are longer, too).
    static constexpr bool kLate = DP == 64;
};

// What it reads of the plan is looked at only when it is used, a job after it was asked for.
struct ForwardJob {
    int i0[2], last[2], head[2], first;                 // queries i0 to last (none if below i0)
    __device__ __forceinline__ ForwardJob(const AttentionParams& p, int job) {
        const int row = job / p.across, place = job - row * p.across, at = p.along - 1 - row;      // the longest first
        for (int s = 0; s < 2; ++s) {
            head[s] = p.by_heads ? place * 2 + s : place;
            i0[s] = (p.by_heads ? at : at * 2 + s) * p.span;
            last[s] = (int)min((int64_t)i0[s] + p.span, p.tokens) - 1;
        }
        first = p.first[i0[0]];
    }
    __device__ __forceinline__ int begin(const AttentionParams& p) const { return p.window > 0 ? max(first, i0[0] - p.window + 1) : first; }          // of its keys
    __device__ __forceinline__ int steps(const AttentionParams& p, int step) const { return (max(last[0], last[1]) - begin(p)) / step + 1; }
    // Every other round backwards, so that the longest of one round goes with the shortest of the next.
    static __device__ __forceinline__ int of_turn(int turn) { return turn * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kForward, 1) attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                const __grid_constant__ CUtensorMap map_o, const __grid_constant__ AttentionParams p) {
    using F = Forward<DP>;
    __shared__ uint64_t q_full[F::kQueries], q_empty[F::kQueries], k_full[F::kStages], k_empty[F::kStages], v_full[F::kStages], v_empty[F::kStages];
    __shared__ uint64_t s_full[2], s_empty[2], p_full[2], o_done[2], ended[2];
    __shared__ uint32_t tensor;
    __shared__ int lost, spoilt[2];
    unsigned char* const shared = aligned_shared();
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        lost = spoilt[0] = spoilt[1] = 0;
        for (int s = 0; s < F::kQueries; ++s) { barrier_init(&q_full[s], 1); barrier_init(&q_empty[s], 2); }
        for (int s = 0; s < F::kStages; ++s) { barrier_init(&k_full[s], 1); barrier_init(&k_empty[s], 2); barrier_init(&v_full[s], 1); barrier_init(&v_empty[s], 2); }
        for (int s = 0; s < 2; ++s) {
            barrier_init(&s_full[s], 1);
            barrier_init(&s_empty[s], kRows);
            barrier_init(&p_full[s], kRows);
            barrier_init(&o_done[s], 1);
            barrier_init(&ended[s], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 10) tensor_alloc<512>(&tensor);
    fence_before();
    __syncthreads();
    fence_after();
    // what the multiplying warp's loops depend on comes by shuffles from one lane: the compiler then knows it to be the same for all and keeps it in uniform registers
    const uint32_t base = __shfl_sync(~0u, tensor, 0), q_at = shared_address(shared), k_at = q_at + F::kKeys, v_at = k_at + F::kStages * F::kPart;
    const int jobs = p.across * p.along;
    // registers: 128 x (2 x 200 + 104) of the 384 x 168 that the block has

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 10) {
        if (lane == 0) {
            // queries and keys; values are another warp's, so that keys do not wait for the room that values wait for
            int queries = 0, keys = 0;                  // loads begun so far
            bool fine = true;
            ForwardJob next(p, blockIdx.x);
            for (int turn = 0, job = blockIdx.x; fine && job < jobs; job = ForwardJob::of_turn(++turn)) {
                const ForwardJob now = next;
                const int after = ForwardJob::of_turn(turn + 1);
                if (after < jobs) next = ForwardJob(p, after);
                const int b = queries % F::kQueries, key_head = now.head[0] / (p.heads_q / p.heads_k), j0 = now.begin(p), count = now.steps(p, F::kStep);
                if (queries >= F::kQueries && !(fine = barrier_wait(&q_empty[b], (queries / F::kQueries - 1) & 1, &lost))) break;
                barrier_expect(&q_full[b], 2 * F::kTile);
                for (int s = 0; s < 2; ++s) load_panels<kRows, DP>(shared + (2 * b + s) * F::kTile, &map_q, &q_full[b], now.head[s], now.i0[s]);
                ++queries;
                for (int j = 0; j < count; ++j, ++keys) {
                    const int s = keys % F::kStages, round = keys / F::kStages;
                    if (round > 0 && !(fine = barrier_wait(&k_empty[s], (round - 1) & 1, &lost))) break;
                    barrier_expect(&k_full[s], F::kPart);
                    load_panels<F::kStep, DP>(shared + F::kKeys + s * F::kPart, &map_k, &k_full[s], key_head, j0 + j * F::kStep);
                }
            }
            drain_ring(q_full, F::kQueries, queries);
            drain_ring(k_full, F::kStages, keys);
        }
    } else if (warp == 11) {
        if (lane == 0) {
            int values = 0;
            bool fine = true;
            ForwardJob next(p, blockIdx.x);
            for (int turn = 0, job = blockIdx.x; fine && job < jobs; job = ForwardJob::of_turn(++turn)) {
                const ForwardJob now = next;
                const int after = ForwardJob::of_turn(turn + 1);
                if (after < jobs) next = ForwardJob(p, after);
                const int key_head = now.head[0] / (p.heads_q / p.heads_k), j0 = now.begin(p), count = now.steps(p, F::kStep);
                for (int j = 0; j < count; ++j, ++values) {
                    const int s = values % F::kStages, round = values / F::kStages;
                    if (round > 0 && !(fine = barrier_wait(&v_empty[s], (round - 1) & 1, &lost))) break;
                    barrier_expect(&v_full[s], F::kPart);
                    load_panels<F::kStep, DP>(shared + F::kKeys + (F::kStages + s) * F::kPart, &map_v, &v_full[s], key_head, j0 + j * F::kStep);
                }
            }
            drain_ring(v_full, F::kStages, values);
        }
    } else if (warp < 10) {
        const int set = warp - 8;
        const uint32_t columns = base + set * F::kSet, q_set = q_at + set * F::kTile;
        constexpr bool ACROSS = F::kQueries > 1;        // whether the scores run ahead over a job's end, too
        int job = blockIdx.x, turn = 0, j = 0, count = 0, ahead = 0;                               // of the scores, one step ahead of P V
        ForwardJob next(p, job);
        int k_stage = 0, k_phase = 0, v_stage = 0, v_phase = 0, q_buffer = 0, q_phase = 0;
        auto scores = [&]() {
            if (j == 0) {
                count = __shfl_sync(~0u, next.steps(p, F::kStep), 0);
                const int after = ForwardJob::of_turn(turn + 1);
                if (after < jobs) next = ForwardJob(p, after);
                if (!warp_wait(&q_full[q_buffer], q_phase, &lost)) return false;
            }
            if (!warp_wait(&k_full[k_stage], k_phase, &lost)) return false;
            if (ahead > 0 && !warp_wait(&s_empty[set], (ahead - 1) & 1, &lost)) return false;
            fence_after();
            multiply_rows<T, F::kStep, DP>(columns, q_set + 2 * q_buffer * F::kTile, k_at + k_stage * F::kPart);
            commit(&s_full[set]);
            commit(&k_empty[k_stage]);
            ++ahead;
            if (++k_stage == F::kStages) { k_stage = 0; k_phase ^= 1; }
            if (++j == count) {
                commit(&q_empty[q_buffer]);
                j = 0;
                if (++q_buffer == F::kQueries) { q_buffer = 0; q_phase ^= 1; }
                job = ForwardJob::of_turn(++turn);
            }
            return true;
        };
        int n = 0, done = 0;
        bool fine = scores();
        for (int own = blockIdx.x; fine && own < jobs; own = ForwardJob::of_turn(++done)) {
            const int steps = count;                    // of the job that the scores have just begun
            for (int i = 0; i < steps; ++i, ++n) {
                if ((i + 1 < steps || (ACROSS && job < jobs)) && !(fine = scores())) break;
                if (!(fine = warp_wait(&p_full[set], n & 1, &lost))) break;
                if (!(fine = warp_wait(&v_full[v_stage], v_phase, &lost))) break;
                fence_after();
                multiply_columns<T, F::kStep, DP>(columns + F::kOut, columns + F::kProb, v_at + v_stage * F::kPart, i != 0);
                commit(&v_empty[v_stage]);
                commit(&o_done[set]);
                if (++v_stage == F::kStages) { v_stage = 0; v_phase ^= 1; }
            }
            // where queries have one buffer, only when the job's last product is under way: the next one's may still be on their way
            if (!ACROSS && fine && job < jobs) fine = scores();
        }
        commit(&ended[set]);
        drain(&ended[set], 0);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int set = warp / 4, row = threadIdx.x % kRows;
        const uint32_t mine = base + set * F::kSet + ((uint32_t)(warp % 4 * 32) << 16);
        const Pair scale2 = pair_of(p.scale2, p.scale2);
        bool fine = true;
        int n = 0;
        // The rows of a job leave when the next one's first probabilities are worked out: P V of its last step is under way meanwhile.
        struct Leaving { int first, last, head; float top, sum; } leaving{0, -1, 0, 0.f, 0.f};
        unsigned char* const tile = shared + F::kStaged + set * F::kTile;
        auto leave = [&]() {
            // through shared memory, so that rows go in whole lines and nobody waits for them
            const int i = leaving.first + row;
            if (row == 0) wait_stores_read();
            meet(1 + set, kRows);
            const bool finite = stage_row<T, DP>(mine + F::kOut, fine ? 1.f / leaving.sum : nan_value(), tile, row);
            const float lse = fine ? fmaf(leaving.top, p.scale2, log2f(leaving.sum)) : nan_value();
            if (fine && i <= leaving.last) {
                if (!isfinite(lse)) *reinterpret_cast<unsigned short*>(staged(tile, row, 0)) = (unsigned short)kFinal;
                else if (!finite) spoilt[set] = 1;
            }
            fence_shared();
            meet(1 + set, kRows);
            if (row == 0 && leaving.first <= leaving.last) {
#pragma unroll
                for (int c = 0; c < DP; c += 64)
                    if (c < p.dim) store_tile(&map_o, tile + c / 64 * kRows * 128, c, leaving.head, leaving.first);
                stores_end();
            }
            if (i <= leaving.last && p.lse != nullptr) p.lse[leaving.head * p.pitch + i] = lse;
        };
        ForwardJob next(p, blockIdx.x);
        auto first_of = [&](const ForwardJob& job) { return p.first[min(job.i0[set] + row, job.last[set] >= job.i0[set] ? job.last[set] : 0)]; };
        int next_first = first_of(next);
        for (int turn = 0, job = blockIdx.x; job < jobs; job = ForwardJob::of_turn(++turn)) {
            const int first = next.i0[set], last = next.last[set], i = first + row, head = next.head[set], j0 = next.begin(p), count = next.steps(p, F::kStep);
            const bool live = i <= last;
            const int high = live ? i : -1, low = !live ? 0 : p.window > 0 ? max(next_first, i - p.window + 1) : next_first;
            const int after = ForwardJob::of_turn(turn + 1);
            if (after < jobs) { next = ForwardJob(p, after); next_first = first_of(next); }
            // keys that any and that all of the warp's rows see; a row that is not there sees none
            const int any_low = __reduce_min_sync(~0u, live ? low : 0x7fffffff), any_high = __reduce_max_sync(~0u, high);
            const int all_low = __reduce_max_sync(~0u, live ? low : 0x7fffffff), all_high = __reduce_min_sync(~0u, high);
            float top = -INFINITY, sum = 0.f;           // of the scores as they are; the sum of exp2(scale2 (S - top))
            bool left = false;
            for (int j = 0; j < count; ++j, ++n) {
                const int k0 = j0 + j * F::kStep;
                fine = fine && warp_wait(&s_full[set], n & 1, &lost);
                if (!fine) break;
                fence_after();
                uint32_t r[F::kStep], packed[F::kStep / 2];
#pragma unroll
                for (int c = 0; c < F::kStep; c += 16) tensor_load16(mine + c, r + c);
                wait_loads();
                fence_before();
                barrier_arrive(&s_empty[set]);
                Pair part[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
                float by = 1.f;
                bool any = false;
                auto rescale = [&]() {
#pragma unroll
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t o[32];
                        tensor_load(mine + F::kOut + c, o);
                        wait_loads();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
                        tensor_store(mine + F::kOut + c, o);
                    }
                };
                // all: every row of the warp sees every key; else CHUNK keys at a time may be hidden from all, or from some
                auto rows = [&](auto all) {
                    constexpr bool ALL = decltype(all)::value != 0;
                    constexpr int CHUNK = DP == 64 ? 32 : 16;
                    auto hidden = [&](int c) { return !ALL && (k0 + c > any_high || k0 + c + CHUNK - 1 < any_low); };
                    float best[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < F::kStep; c += CHUNK) {
                        if (hidden(c)) continue;
                        if (!ALL && (k0 + c < all_low || k0 + c + CHUNK - 1 > all_high)) {
                            const uint32_t seen = columns_between(low - k0 - c, high - k0 - c);
#pragma unroll
                            for (int k = 0; k < CHUNK; ++k) r[c + k] = seen >> k & 1u ? r[c + k] : 0xff800000u;
                        }
#pragma unroll
                        for (int k = 0; k < CHUNK / 2; ++k) best[k % 4] = max3(best[k % 4], __uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1]));
                    }
                    const float now_top = fmaxf(max3(best[0], best[1], best[2]), best[3]);
                    // the maximum in use follows only where the new one is more than 2^8 above: P stays below 2^8, and O is seldom rescaled
                    const bool up = now_top != top && ((now_top - top) * p.scale2 > 8.f || top == -INFINITY);
                    any = __any_sync(~0u, up);
                    by = up ? exp2_fast((top - now_top) * p.scale2) : 1.f;
                    if (up) top = now_top;
                    sum *= by;
                    const float shift = top == -INFINITY ? 0.f : -top * p.scale2;
                    const Pair shifts = pair_of(shift, shift);
                    if (!F::kLate && n > 0) {
                        if (!warp_wait(&o_done[set], (n - 1) & 1, &lost)) return false;
                        fence_after();
                        if (any && j > 0) rescale();
                    }
#pragma unroll
                    for (int c = 0; c < F::kStep; c += CHUNK) {
                        if (hidden(c)) {
#pragma unroll
                            for (int k = 0; k < CHUNK / 2; ++k) packed[c / 2 + k] = 0u;
                        } else {
#pragma unroll
                            for (int k = 0; k < CHUNK; k += 2) {
                                float a, b;
                                split(fma_pair(pair_of(__uint_as_float(r[c + k]), __uint_as_float(r[c + k + 1])), scale2, shifts), a, b);
                                a = exp2_fast(a);
                                b = exp2_fast(b);
                                part[k / 2 % 2] = add_pair(part[k / 2 % 2], pair_of(a, b));
                                packed[(c + k) / 2] = pack<T>(a, b);
                            }
                        }
                        if (!F::kLate)
#pragma unroll
                            for (int k = 0; k < CHUNK / 2; k += 8) tensor_store8(mine + F::kProb + c / 2 + k, packed + c / 2 + k);
                    }
                    return true;
                };
                if (!(fine = k0 >= all_low && k0 + F::kStep - 1 <= all_high ? rows(Number<1>{}) : rows(Number<0>{}))) break;
                float x, y;
                split(add_pair(part[0], part[1]), x, y);
                sum += x + y;
                if (F::kLate) {
                    // P V of the step before has ended: P and O may be written, and the rows of a job that it ended may leave
                    if (n > 0) {
                        fine = warp_wait(&o_done[set], (n - 1) & 1, &lost);
                        if (!fine) break;
                        fence_after();
                        if (j == 0) { leave(); left = true; }
                        if (any && j > 0) rescale();
                    }
#pragma unroll
                    for (int c = 0; c < F::kStep / 2; c += 8) tensor_store8(mine + F::kProb + c, packed + c);
                }
                wait_stores();
                fence_before();
                barrier_arrive(&p_full[set]);
            }
            if (F::kLate && turn > 0 && !left) leave(); // a block that gave up: NaN for this job's, and below for what is left
            leaving = Leaving{first, last, head, top, sum};
            if (!F::kLate) {
                fine = fine && warp_wait(&o_done[set], (n - 1) & 1, &lost);
                fence_after();
                leave();
            }
        }
        if (F::kLate) {
            fine = fine && warp_wait(&o_done[set], (n - 1) & 1, &lost);
            fence_after();
            leave();
        }
        if (row == 0) wait_stores_done();
        meet(1 + set, kRows);
        if (spoilt[set] != 0 && lost == 0)
            for (int turn = 0, job = blockIdx.x; job < jobs; job = ForwardJob::of_turn(++turn)) {
                const ForwardJob done(p, job);
                for (int i = done.i0[set] + warp % 4; i <= done.last[set]; i += 4) mend_out<T>(p, i, done.head[set], lane);
            }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 10) tensor_free<512>(tensor);
}

// ---- backwards: gradients of the queries -------------------------------------------------------------------------------
// Two blocks to an SM, or one of wide heads, each of which takes (tile of queries, head) jobs in turn; loads and products run ahead as forwards, and rows leave under the next job's first exponentials.
template <int DP> struct Queries {
    // one block to an SM has columns for two steps' scores, the next ones multiplied while the present ones are worked on; where two share the SM, the other block's work goes on meanwhile
    static constexpr int kBlocks = DP == 64 ? 2 : 1, kBuffers = DP == 64 ? 1 : 2, kColumns = 512 / kBlocks;
    static constexpr int kStages = DP == 64 ? 2 : 3;
    // threads of a row, with one block to an SM two, each with half of a step's columns (40000 tokens in 4 episodes, 8 heads, 2 of keys: 1309 us with one, 1220 with two; keys' 2751 and 2344)
    static constexpr int kHalves = DP == 64 ? 1 : 2, kWorkers = kHalves * kRows, kThreads = kBlock + kWorkers - kRows, kPer = kStream / kHalves;
    static constexpr int kTile = kRows * DP * 2, kPart = kStream * DP * 2;
    // queries, dO and, for D = dO . O, O; steps of keys and values; the rows that leave
    static constexpr int kKeys = 3 * kTile, kStaged = kKeys + 2 * kStages * kPart, kShared = kStaged + kTile + 1024;
    static constexpr int kGrad = kStream, kScores = 2 * kStream, kOut = kBuffers * kScores, kProb = kOut + DP;
};

template <typename T, int DP>
__global__ void __launch_bounds__(Queries<DP>::kThreads, Queries<DP>::kBlocks) query_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_o,
                                                               const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dq,
                                                               const AttentionParams p) {
    using F = Queries<DP>;
    __shared__ uint64_t q_full, q_empty, full[F::kStages], empty[F::kStages], s_full[F::kBuffers], s_empty[F::kBuffers], p_full, o_done, ended;
    __shared__ uint32_t tensor;
    __shared__ int lost, spoilt;
    __shared__ float offs[F::kHalves][kRows];
    unsigned char* const shared = aligned_shared();
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        lost = spoilt = 0;
        barrier_init(&q_full, 1);
        barrier_init(&q_empty, 1 + F::kWorkers);      // the scores' products, and the rows' reads of dO and O
        for (int s = 0; s < F::kStages; ++s) { barrier_init(&full[s], 1); barrier_init(&empty[s], 1); }
        for (int s = 0; s < F::kBuffers; ++s) { barrier_init(&s_full[s], 1); barrier_init(&s_empty[s], F::kWorkers); }
        barrier_init(&p_full, F::kWorkers);
        barrier_init(&o_done, 1);
        barrier_init(&ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 5) tensor_alloc<F::kColumns>(&tensor);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t base = __shfl_sync(~0u, tensor, 0), q_at = shared_address(shared), do_at = q_at + F::kTile, kv_at = q_at + F::kKeys;
    const int jobs = p.tiles * p.heads_q, stride = gridDim.x, group = p.heads_q / p.heads_k;

    if (warp == 4) {
        if (lane == 0) {
            int steps = 0, queries = 0;                 // loads begun so far
            bool fine = true;
            QueryJob next(p, blockIdx.x);
            for (int job = blockIdx.x; fine && job < jobs; job += stride) {
                const QueryJob now = next;
                if (job + stride < jobs) next = QueryJob(p, job + stride);
                if (queries > 0 && !(fine = barrier_wait(&q_empty, (queries - 1) & 1, &lost))) break;
                barrier_expect(&q_full, 3 * F::kTile);
                load_panels<kRows, DP>(shared, &map_q, &q_full, now.head, now.i0);
                load_panels<kRows, DP>(shared + F::kTile, &map_do, &q_full, now.head, now.i0);
                load_panels<kRows, DP>(shared + 2 * F::kTile, &map_o, &q_full, now.head, now.i0);
                ++queries;
                const int j0 = now.begin(p), count = now.steps(p), key_head = now.head / group;
                for (int j = 0; j < count; ++j, ++steps) {
                    const int s = steps % F::kStages, turn = steps / F::kStages;
                    if (turn > 0 && !(fine = barrier_wait(&empty[s], (turn - 1) & 1, &lost))) break;
                    barrier_expect(&full[s], 2 * F::kPart);
                    unsigned char* to = shared + F::kKeys + 2 * s * F::kPart;
                    load_panels<kStream, DP>(to, &map_k, &full[s], key_head, j0 + j * kStream);
                    load_panels<kStream, DP>(to + F::kPart, &map_v, &full[s], key_head, j0 + j * kStream);
                }
            }
            drain_ring(&q_full, 1, queries);
            drain_ring(full, F::kStages, steps);
        }
    } else if (warp == 5) {
        int job = blockIdx.x, j = 0, count = 0, ahead = 0, queries = 0, stage = 0, phase = 0;      // of the scores
        QueryJob next(p, job);
        auto scores = [&]() {
            if (j == 0) {
                count = __shfl_sync(~0u, next.steps(p), 0);
                if (job + stride < jobs) next = QueryJob(p, job + stride);
                if (!warp_wait(&q_full, queries & 1, &lost)) return false;
            }
            if (!warp_wait(&full[stage], phase, &lost)) return false;
            const int b = ahead % F::kBuffers;
            if (ahead >= F::kBuffers && !warp_wait(&s_empty[b], (ahead / F::kBuffers - 1) & 1, &lost)) return false;
            fence_after();
            multiply_rows<T, kStream, DP>(base + b * F::kScores, q_at, kv_at + 2 * stage * F::kPart);
            multiply_rows<T, kStream, DP>(base + b * F::kScores + F::kGrad, do_at, kv_at + (2 * stage + 1) * F::kPart);
            commit(&s_full[b]);
            ++ahead;
            if (++stage == F::kStages) { stage = 0; phase ^= 1; }
            if (++j == count) { commit(&q_empty); j = 0; ++queries; job += stride; }
            return true;
        };
        int n = 0, own_stage = 0;
        bool fine = scores();
        for (int own = blockIdx.x; fine && own < jobs; own += stride) {
            const int steps = count;                    // of the job that the scores have just begun
            for (int i = 0; i < steps; ++i, ++n) {
                if (i + 1 < steps && !(fine = scores())) break;
                if (!(fine = warp_wait(&p_full, n & 1, &lost))) break;
                fence_after();
                multiply_columns<T, kStream, DP>(base + F::kOut, base + F::kProb, kv_at + 2 * own_stage * F::kPart, i != 0);
                commit(&empty[own_stage]);
                commit(&o_done);
                if (++own_stage == F::kStages) own_stage = 0;
                // over a job's end only now: the next one's queries may still be on their way
                if (i + 1 == steps && job < jobs && !(fine = scores())) break;
            }
        }
        commit(&ended);
        drain(&ended, 0);
    } else {
        // a warp reaches the tensor memory's lanes 32 (warp % 4) and on
        const int row = warp % 4 * 32 + lane, half = warp / 4 == 0 ? 0 : 1;
        const uint32_t mine = base + ((uint32_t)(warp % 4 * 32) << 16);
        bool fine = true;
        int n = 0, queries = 0;
        struct Leaving { int first, last, head; float lse, delta; } leaving{0, -1, 0, 0.f, 0.f};
        // Every warp calls it once for each job, whether it gave up or not, and the named barrier in it is the only one: all meet there in the same order.
        auto leave = [&]() {
            const int i = leaving.first + row;
            const bool there = i <= leaving.last;
            unsigned char* const tile = shared + F::kStaged;
            if (threadIdx.x == 0) wait_stores_read();
            meet(1, F::kWorkers);
            // the row's other thread has its part of D, unless it gave up, which `lost` then says; the keys' gradients become NaN by D
            if (F::kHalves > 1) leaving.delta += offs[0][row] + offs[1 % F::kHalves][row];
            if (there && half == 0) p.delta[leaving.head * p.pitch + i] = fine && lost == 0 ? leaving.delta : nan_value();
            const bool finite = stage_row<T, DP / F::kHalves>(mine + F::kOut + half * (DP / 2), fine ? p.scale : nan_value(), tile + half * kRows * 128, row);
            if (!finite && there && isfinite(leaving.lse) && isfinite(leaving.delta)) spoilt = 1;
            fence_shared();
            meet(1, F::kWorkers);
            if (threadIdx.x == 0 && leaving.first <= leaving.last) {
                for (int c = 0; c < DP; c += 64)
                    if (c < p.dim) store_tile(&map_dq, tile + c / 64 * kRows * 128, c, leaving.head, leaving.first);
                stores_end();
            }
        };
        QueryJob next(p, blockIdx.x);
        auto first_of = [&](const QueryJob& job) { return p.first[min(job.i0 + row, job.last)]; };
        auto lse_of = [&](const QueryJob& job) { return p.lse[job.head * p.pitch + min(job.i0 + row, job.last)]; };
        int next_first = first_of(next);
        float next_lse = lse_of(next);
        for (int job = blockIdx.x; job < jobs; job += stride, ++queries) {
            const QueryJob now = next;
            const int i = now.i0 + row, j0 = now.begin(p), count = now.steps(p);
            const bool live = i <= now.last;
            const int high = live ? i : -1, low = !live ? 0 : p.window > 0 ? max(next_first, i - p.window + 1) : next_first;
            const float lse = next_lse;
            if (job + stride < jobs) { next = QueryJob(p, job + stride); next_first = first_of(next); next_lse = lse_of(next); }
            const int any_low = __reduce_min_sync(~0u, live ? low : 0x7fffffff), any_high = __reduce_max_sync(~0u, high);
            const int all_low = __reduce_max_sync(~0u, live ? low : 0x7fffffff), all_high = __reduce_min_sync(~0u, high);
            // D = dO . O of the thread's row.  O has the error of its own rounding and of P's, which the sum of dS over the row, 0 by definition, shows: the keys' kernel, which runs
            // after this one, gets D without it. Where a step holds all keys of a row D is summed from its own P and dP before dS, which matters where few keys share a row (dq of
            // 24-token episodes was off by 1.8 times its rounding; with many keys the error averages out).
            float delta = 0.f;
            fine = fine && warp_wait(&q_full, queries & 1, &lost);
            if (fine)
#pragma unroll
                for (int c = 0; c < DP / 8; ++c) {
                    float u[8], v[8];
                    unpack<T, 8>(*reinterpret_cast<const uint4*>(staged(shared + F::kTile, row, c)), u);
                    unpack<T, 8>(*reinterpret_cast<const uint4*>(staged(shared + 2 * F::kTile, row, c)), v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) delta = fmaf(u[k], v[k], delta);
                }
            barrier_arrive(&q_empty);
            const Pair scale2 = pair_of(p.scale2, p.scale2), shift = pair_of(-lse, -lse);
            Pair off = pair_of(0.f, 0.f);
            bool left = false;
            for (int j = 0; j < count; ++j, ++n) {
                const int k0 = j0 + j * kStream;
                const int b = n % F::kBuffers;
                const uint32_t here = mine + b * F::kScores;
                fine = fine && warp_wait(&s_full[b], n / F::kBuffers & 1, &lost);
                if (!fine) break;
                fence_after();
                uint32_t packed[F::kPer / 2];
                const bool all = k0 >= all_low && k0 + kStream - 1 <= all_high;
                auto hidden = [&](int c0) { return k0 + c0 > any_high || k0 + c0 + 31 < any_low; };          // from all of the warp's rows
                // P and P (dP - D) of 32 keys
                auto part = [&](int c0, Pair minus, auto use) {
                    uint32_t r[32], d[32];
                    tensor_load(here + c0, r);
                    tensor_load(here + F::kGrad + c0, d);
                    wait_loads();
                    const uint32_t seen = all ? ~0u : columns_between(low - k0 - c0, high - k0 - c0);
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float a, b, x, y;
                        split(fma_pair(pair_of(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, shift), a, b);
                        a = exp2_fast(a);
                        b = exp2_fast(b);
                        split(mul_pair(pair_of(a, b), add_pair(pair_of(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), minus)), x, y);
                        if (!all) {
                            x = seen >> c & 1u ? x : 0.f;
                            y = seen >> (c + 1) & 1u ? y : 0.f;
                        }
                        use(c, x, y);
                    }
                };
                const bool whole = live && low >= k0 && high < k0 + kStream;
                if (__any_sync(~0u, whole)) {
                    float own = 0.f;
#pragma unroll 1
                    for (int c0 = 0; c0 < kStream; c0 += 32)
                        if (!hidden(c0)) part(c0, pair_of(0.f, 0.f), [&](int, float x, float y) { own += x + y; });
                    if (whole) delta = own;
                }
                const Pair minus = pair_of(-delta, -delta);
#pragma unroll
                for (int own = 0; own < F::kPer; own += 32) {
                    const int c0 = half * F::kPer + own;
                    if (hidden(c0)) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) packed[own / 2 + c] = 0u;
                    } else {
                        part(c0, minus, [&](int c, float x, float y) {
                            off = add_pair(off, pair_of(x, y));
                            packed[(own + c) / 2] = pack<T>(x, y);
                        });
                    }
                }
                fence_before();
                barrier_arrive(&s_empty[b]);
                if (n > 0) fine = warp_wait(&o_done, (n - 1) & 1, &lost);
                if (!fine) break;
                if (n > 0) fence_after();
                if (j == 0 && n > 0) { leave(); left = true; }
                if constexpr (F::kHalves == 1) {
                    tensor_store(mine + F::kProb, packed);
                } else {
                    for (int c = 0; c < F::kPer / 2; c += 8) tensor_store8(mine + F::kProb + half * (F::kPer / 2) + c, packed + c);
                }
                wait_stores();
                fence_before();
                barrier_arrive(&p_full);
            }
            float x, y;
            split(off, x, y);
            if (queries > 0 && !left) leave();          // a block that gave up: NaN for this job's, and below for what is left
            if (F::kHalves == 1) delta += x + y;
            else offs[half][row] = x + y;               // read in leave(), between whose two meetings nobody writes it
            leaving = Leaving{now.i0, now.last, now.head, lse, delta};
        }
        fine = fine && warp_wait(&o_done, (n - 1) & 1, &lost);
        fence_after();
        leave();
        if (threadIdx.x == 0) wait_stores_done();
        meet(1, F::kWorkers);
        if (spoilt != 0 && lost == 0)
            for (int job = blockIdx.x; job < jobs; job += stride) {
                const QueryJob done(p, job);
                for (int i = done.i0 + half * 4 + warp % 4; i <= done.last; i += F::kWorkers / 32) mend_query_grad<T>(p, i, done.head, lane);
            }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 5) tensor_free<F::kColumns>(tensor);
}

// ---- backwards: gradients of keys and values ----------------------------------------------------------------------------
// The same with (tile of keys, key head) jobs: the queries of all heads of the group that see any of the keys pass by, 64 at a time, with their statistics.
// Where jobs are few, a cluster's blocks share the heads of a group, and add up their sums in 32 bits through each other's shared memory at the end, always in the order of the heads.
// That sum is worth about ten steps, so jobs are cut in two as long as that leaves one block for each place on the GPU, or, where rows are long, four.
// 8 heads, 2 of keys, dim 64, uncut and cut in 2 and 4: 3000 tokens in 10 episodes 44, 31 and 22 us; 6000 in 30: 35, 30 and 34; 20011 in 40: 92, 96 and 107; 20000 in 100: 62, 74 and 86;
// 6000 in 2: 270, 148 and 91; 12000 in 3: 360, 214 and 215.
template <int DP> struct Keys {
    // one block to an SM has columns for two steps' scores; P and dS take their scores' place
    static constexpr int kBlocks = DP == 64 ? 2 : 1, kBuffers = DP == 64 ? 1 : 2, kColumns = 512 / kBlocks;
    static constexpr int kStages = DP == 64 ? 2 : 4;
    // threads of a row, with one block to an SM two, each with half of a step's columns (40000 tokens in 4 episodes, 8 heads, 2 of keys: 1309 us with one, 1220 with two; keys' 2751 and 2344)
    static constexpr int kHalves = DP == 64 ? 1 : 2, kWorkers = kHalves * kRows, kThreads = kBlock + kWorkers - kRows, kPer = kStream / kHalves;
    static constexpr int kTile = kRows * DP * 2, kPart = kStream * DP * 2;
    static constexpr int kStaged = 2 * kTile + 2 * kStages * kPart, kShared = kStaged + (DP == 64 ? 2 * kTile : 0) + 1024;         // rows of wide heads leave without a staged tile
    static constexpr int kGrad = kStream, kScores = 2 * kStream, kValue = kBuffers * kScores, kKey = kValue + DP;
};

// A tile of keys and a key head; the longest of one long row are the first ones.
struct KeyJob {
    int j0, last, head, end;                            // keys j0 to last; end: the plan's, of the last
    __device__ __forceinline__ KeyJob(const AttentionParams& p, int job) {
        const int tile = job / p.heads_k;
        head = job - tile * p.heads_k;
        j0 = tile * p.span;
        last = (int)min((int64_t)j0 + p.span, p.tokens) - 1;
        end = p.end[last];
    }
    __device__ __forceinline__ int begin() const { return j0 & ~3; }               // of its queries: a multiple of 16 bytes of their statistics
    __device__ __forceinline__ int past(const AttentionParams& p) const { return p.window > 0 ? (int)min((int64_t)end, (int64_t)last + p.window) : end; }
    __device__ __forceinline__ int steps(const AttentionParams& p) const { return (past(p) - 1 - begin()) / kStream + 1; }            // for one head
};

// Queries of a step that are seen by none of the tile's keys, behind a long episode's end for instance: where they are not finite, which their lse or D is then not either, zeros take
// their place in the second products. (Else every key of the episode would have to be worked out again.)  The first products have read them by then.  With one block to an SM the rows'
// warps do it, else the one that multiplies: its check is ready before the probabilities, and the rows have no registers left; with two score buffers it is the chain itself (40000 tokens
// in 4 episodes, dim 128: 2396 us there, 2314 here; 12000 in 3, dim 64, one key head: 233 there, 241 here).
__device__ __forceinline__ bool hidden_spoilt(int x, int from, int past, const float* lse, const float* delta) { return (x < from || x >= past) && !(isfinite(lse[x]) && isfinite(delta[x])); }
// Query x of the streamed tiles of q and dO: panels first, first + step and so on of both.
template <int DP> __device__ __forceinline__ void clear_query(unsigned char* tiles, int x, int first, int step) {
    for (int c = first; c < 2 * DP / 64; c += step)
        for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(tiles + c * kStream * 128 + x * 128 + k * 16) = make_uint4(0u, 0u, 0u, 0u);
}
template <int DP, int THREADS> __device__ __noinline__ void clear_hidden(int from, int past, unsigned char* tiles, const float* lse, const float* delta, int thread) {
    const int x = thread % kStream;
    if (hidden_spoilt(x, from, past, lse, delta)) clear_query<DP>(tiles, x, thread / kStream, THREADS / kStream);
    fence_shared();
    __syncwarp();
}

template <typename T, int DP>
__global__ void __launch_bounds__(Keys<DP>::kThreads, Keys<DP>::kBlocks) key_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
                                                                            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dk,
                                                                            const __grid_constant__ CUtensorMap map_dv, const AttentionParams p) {
    using F = Keys<DP>;
    __shared__ uint64_t k_full, k_empty, full[F::kStages], empty[F::kStages], s_full[F::kBuffers], p_full, o_done, ended;
    __shared__ __align__(16) float lse[F::kStages][kStream], delta[F::kStages][kStream];
    __shared__ uint32_t tensor;
    __shared__ int lost, spoilt;
    unsigned char* const shared = aligned_shared();
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        lost = spoilt = 0;
        barrier_init(&k_full, 1);
        barrier_init(&k_empty, 1);
        for (int s = 0; s < F::kStages; ++s) { barrier_init(&full[s], 1); barrier_init(&empty[s], 1); }
        for (int s = 0; s < F::kBuffers; ++s) barrier_init(&s_full[s], 1);
        barrier_init(&p_full, F::kWorkers);
        barrier_init(&o_done, 1);
        barrier_init(&ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 5) tensor_alloc<F::kColumns>(&tensor);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t base = __shfl_sync(~0u, tensor, 0), k_at = shared_address(shared), v_at = k_at + F::kTile, part_at = v_at + F::kTile;
    const int rank = p.split > 1 ? (int)cluster_rank() : 0, job0 = blockIdx.x / p.split, stride = gridDim.x / p.split, jobs = p.tiles * p.heads_k;
    const int group = p.heads_q / p.heads_k / p.split;     // heads of a block, from number rank * group on

    if (warp == 4) {
        if (lane == 0) {
            int steps = 0, keys = 0;                    // loads begun so far
            bool fine = true;
            KeyJob next(p, job0);
            for (int job = job0; fine && job < jobs; job += stride) {
                const KeyJob now = next;
                if (job + stride < jobs) next = KeyJob(p, job + stride);
                if (keys > 0 && !(fine = barrier_wait(&k_empty, (keys - 1) & 1, &lost))) break;
                barrier_expect(&k_full, 2 * F::kTile);
                load_panels<kRows, DP>(shared, &map_k, &k_full, now.head, now.j0);
                load_panels<kRows, DP>(shared + F::kTile, &map_v, &k_full, now.head, now.j0);
                ++keys;
                const int each = now.steps(p);
                for (int h = 0; fine && h < group; ++h)
                    for (int m = 0; m < each; ++m, ++steps) {
                        const int s = steps % F::kStages, turn = steps / F::kStages, head = now.head * (p.heads_q / p.heads_k) + rank * group + h, i = now.begin() + m * kStream;
                        if (turn > 0 && !(fine = barrier_wait(&empty[s], (turn - 1) & 1, &lost))) break;
                        barrier_expect(&full[s], 2 * F::kPart + 2 * kStream * 4);
                        unsigned char* to = shared + 2 * F::kTile + 2 * s * F::kPart;
                        load_panels<kStream, DP>(to, &map_q, &full[s], head, i);
                        load_panels<kStream, DP>(to + F::kPart, &map_do, &full[s], head, i);
                        load_bytes(lse[s], p.lse + head * p.pitch + i, kStream * 4, &full[s]);
                        load_bytes(delta[s], p.delta + head * p.pitch + i, kStream * 4, &full[s]);
                    }
            }
            drain_ring(&k_full, 1, keys);
            drain_ring(full, F::kStages, steps);
        }
    } else if (warp == 5) {
        int job = job0, j = 0, count = 0, ahead = 0, keys = 0, stage = 0, phase = 0;         // of the scores
        KeyJob next(p, job);
        auto scores = [&]() {
            if (j == 0) {
                count = __shfl_sync(~0u, next.steps(p) * group, 0);
                if (job + stride < jobs) next = KeyJob(p, job + stride);
                if (!warp_wait(&k_full, keys & 1, &lost)) return false;
            }
            if (!warp_wait(&full[stage], phase, &lost)) return false;
            const int b = ahead % F::kBuffers;
            if (F::kBuffers == 1 && ahead > 0 && !warp_wait(&o_done, (ahead - 1) & 1, &lost)) return false;     // P and dS, which lie there, are free then
            fence_after();
            multiply_rows<T, kStream, DP>(base + b * F::kScores, k_at, part_at + 2 * stage * F::kPart);
            multiply_rows<T, kStream, DP>(base + b * F::kScores + F::kGrad, v_at, part_at + (2 * stage + 1) * F::kPart);
            commit(&s_full[b]);
            ++ahead;
            if (++stage == F::kStages) { stage = 0; phase ^= 1; }
            if (++j == count) { commit(&k_empty); j = 0; ++keys; job += stride; }
            return true;
        };
        int n = 0, own_stage = 0;
        bool fine = scores();
        for (int own = job0; fine && own < jobs; own += stride) {
            const int steps = count;                    // of the job that the scores have just begun
            const KeyJob now(p, own);
            const int each = steps / group;
            for (int i = 0, m = 0; i < steps; ++i, ++n) {
                // the other buffer's P and dS are free when the products before have ended
                if (F::kBuffers > 1 && n > 0 && !(fine = warp_wait(&o_done, (n - 1) & 1, &lost))) break;
                if (F::kBuffers > 1 && i + 1 < steps && !(fine = scores())) break;
                const int i0 = now.begin() + m * kStream;
                uint32_t clear = 0u;
                if (F::kBuffers == 1 && (m == 0 || m + 1 == each))
                    for (int x = lane; x < kStream; x += 32)
                        if (hidden_spoilt(x, now.j0 - i0, now.past(p) - i0, lse[own_stage], delta[own_stage])) clear |= 1u << x / 32;
                if (++m == each) m = 0;
                if (!(fine = warp_wait(&p_full, n & 1, &lost))) break;
                if (F::kBuffers == 1 && __any_sync(~0u, clear != 0u)) {
                    for (int x = lane; x < kStream; x += 32)
                        if (clear >> x / 32 & 1u) clear_query<DP>(shared + 2 * F::kTile + 2 * own_stage * F::kPart, x, 0, 1);
                    fence_shared();
                    __syncwarp();
                }
                fence_after();
                const uint32_t probs = base + n % F::kBuffers * F::kScores;
                multiply_columns<T, kStream, DP, F::kPer>(base + F::kValue, probs, part_at + (2 * own_stage + 1) * F::kPart, i != 0);
                multiply_columns<T, kStream, DP, F::kPer>(base + F::kKey, probs + F::kGrad, part_at + 2 * own_stage * F::kPart, i != 0);
                commit(&empty[own_stage]);
                commit(&o_done);
                if (++own_stage == F::kStages) own_stage = 0;
                if ((F::kBuffers == 1 || i + 1 == steps) && job < jobs && !(fine = scores())) break;
            }
        }
        commit(&ended);
        drain(&ended, 0);
    } else {
        // a warp reaches the tensor memory's lanes 32 (warp % 4) and on
        const int row = warp % 4 * 32 + lane, half = warp / 4 == 0 ? 0 : 1;
        const uint32_t mine = base + ((uint32_t)(warp % 4 * 32) << 16);
        bool fine = true;
        int n = 0, keys = 0, stage = 0, phase = 0;
        struct Leaving { int first, last, head; } leaving{0, -1, 0};
        auto leave = [&]() {
            const int j = leaving.first + row;
            const bool there = j <= leaving.last;
            if (p.split > 1) {
                // in 32 bits where the operands were, 16 bytes at a time, rows turned against each other so that lanes meet different banks
#pragma unroll
                for (int which = half; which < 2; which += F::kHalves)
#pragma unroll
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t r[32];
                        tensor_load(mine + (which ? F::kValue : F::kKey) + c, r);
                        wait_loads();
                        const float by = !fine ? nan_value() : which ? 1.f : p.scale;
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<float4*>(shared + which * kRows * DP * 4 + row * DP * 4 + (((c + k) / 4) ^ (row % 8)) * 16) =
                                make_float4(__uint_as_float(r[k]) * by, __uint_as_float(r[k + 1]) * by, __uint_as_float(r[k + 2]) * by, __uint_as_float(r[k + 3]) * by);
                    }
            } else if (DP == 64) {
                unsigned char *const dv = shared + F::kStaged, *const dk = dv + F::kTile;
                if (row == 0) wait_stores_read();
                meet(1, kRows);
                const bool keys_finite = stage_row<T, DP>(mine + F::kKey, fine ? p.scale : nan_value(), dk, row), values_finite = stage_row<T, DP>(mine + F::kValue, fine ? 1.f : nan_value(), dv, row);
                if (there && !(keys_finite && values_finite)) spoilt = 1;
                fence_shared();
                meet(1, kRows);
                if (row == 0 && leaving.first <= leaving.last) {
                    store_tile(&map_dv, dv, 0, leaving.head, leaving.first);
                    store_tile(&map_dk, dk, 0, leaving.head, leaving.first);
                    stores_end();
                }
            } else {
                T* const to[2] = {static_cast<T*>(p.dk) + ((int64_t)j * p.heads_k + leaving.head) * p.dim, static_cast<T*>(p.dv) + ((int64_t)j * p.heads_k + leaving.head) * p.dim};
                const bool finite = store_row<T, DP>(mine + (half ? F::kValue : F::kKey), !fine ? nan_value() : half ? 1.f : p.scale, p.dim, there ? to[half] : nullptr);
                if (there && !finite) spoilt = 1;
            }
        };
        KeyJob next(p, job0);
        auto end_of = [&](const KeyJob& job) { return p.end[min(job.j0 + row, job.last)]; };
        int next_end = end_of(next);
        const Pair scale2 = pair_of(p.scale2, p.scale2), minus_one = pair_of(-1.f, -1.f);
        for (int job = job0; job < jobs; job += stride, ++keys) {
            const KeyJob now = next;
            const int j = now.j0 + row, each = now.steps(p);
            const bool live = j <= now.last;
            // the queries that see the key
            const int low = live ? j : 0, high = !live ? -1 : (p.window > 0 ? (int)min((int64_t)next_end, (int64_t)j + p.window) : next_end) - 1;
            if (job + stride < jobs) { next = KeyJob(p, job + stride); next_end = end_of(next); }
            const int any_low = __reduce_min_sync(~0u, live ? low : 0x7fffffff), any_high = __reduce_max_sync(~0u, high);
            const int all_low = __reduce_max_sync(~0u, live ? low : 0x7fffffff), all_high = __reduce_min_sync(~0u, high);
            bool first = true, left = false;
            for (int h = 0; fine && h < group; ++h)
                for (int m = 0; m < each; ++m, ++n) {
                    const int i = now.begin() + m * kStream;
                    // the statistics came with the tile that the scores waited for; this wait makes them visible here, too
                    const int b = n % F::kBuffers;
                    const uint32_t here = mine + b * F::kScores;
                    fine = fine && warp_wait(&full[stage], phase, &lost) && warp_wait(&s_full[b], n / F::kBuffers & 1, &lost);
                    if (!fine) break;
                    fence_after();
                    if (F::kBuffers > 1 && (i < now.j0 || i + kStream > now.past(p))) clear_hidden<DP, F::kWorkers>(now.j0 - i, now.past(p) - i, shared + 2 * F::kTile + 2 * stage * F::kPart, lse[stage], delta[stage], half * kRows + row);
                    uint32_t probs[F::kPer / 2], grads[F::kPer / 2];
                    const float4 *l4 = reinterpret_cast<const float4*>(lse[stage]), *d4 = reinterpret_cast<const float4*>(delta[stage]);
                    const bool all = i >= all_low && i + kStream - 1 <= all_high;
#pragma unroll
                    for (int own = 0; own < F::kPer; own += 32) {
                        const int c0 = half * F::kPer + own;
                        uint32_t r[32], d[32];
                        tensor_load(here + c0, r);
                        tensor_load(here + F::kGrad + c0, d);
                        wait_loads();
                        if (i + c0 > any_high || i + c0 + 31 < any_low) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) probs[own / 2 + c] = grads[own / 2 + c] = 0u;
                            continue;
                        }
                        const uint32_t seen = all ? ~0u : columns_between(low - i - c0, high - i - c0);
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const float4 l = l4[(c0 + c) / 4], e = d4[(c0 + c) / 4];
                            const Pair ls[2] = {pair_of(l.x, l.y), pair_of(l.z, l.w)}, es[2] = {pair_of(e.x, e.y), pair_of(e.z, e.w)};
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int at = c + 2 * k;
                                float a, b, x, y;
                                split(fma_pair(ls[k], minus_one, mul_pair(pair_of(__uint_as_float(r[at]), __uint_as_float(r[at + 1])), scale2)), a, b);
                                a = exp2_fast(a);
                                b = exp2_fast(b);
                                split(mul_pair(pair_of(a, b), fma_pair(es[k], minus_one, pair_of(__uint_as_float(d[at]), __uint_as_float(d[at + 1])))), x, y);
                                if (!all) {
                                    const bool u = seen >> at & 1u, v = seen >> (at + 1) & 1u;
                                    a = u ? a : 0.f; x = u ? x : 0.f;
                                    b = v ? b : 0.f; y = v ? y : 0.f;
                                }
                                probs[(own + at) / 2] = pack<T>(a, b);
                                grads[(own + at) / 2] = pack<T>(x, y);
                            }
                        }
                    }
                    // each one in turn where there are two buffers, whose scores say nothing of the products before: a wait tells a phase from the one before it only
                    if (n > 0 && (F::kBuffers > 1 || first)) fine = warp_wait(&o_done, (n - 1) & 1, &lost);
                    if (!fine) break;
                    if (n > 0 && first) fence_after();
                    if (first && n > 0) { leave(); left = true; }
                    first = false;
                    if constexpr (F::kHalves == 1) {
                        tensor_store(here, probs);
                        tensor_store(here + F::kGrad, grads);
                    } else {
                        // where the thread's own scores were, since the row's other thread may still have to read its own
                        for (int c = 0; c < F::kPer / 2; c += 8) {
                            tensor_store8(here + half * F::kPer + c, probs + c);
                            tensor_store8(here + F::kGrad + half * F::kPer + c, grads + c);
                        }
                    }
                    wait_stores();
                    fence_before();
                    barrier_arrive(&p_full);
                    if (++stage == F::kStages) { stage = 0; phase ^= 1; }
                }
            if (keys > 0 && !left) leave();             // a block that gave up: NaN for this job's, and below for what is left
            leaving = {now.j0, now.last, now.head};
        }
        fine = fine && warp_wait(&o_done, (n - 1) & 1, &lost);
        fence_after();
        leave();
        if (row == 0) wait_stores_done();
        meet(1, F::kWorkers);
        if (p.split == 1 && spoilt != 0 && lost == 0)
            for (int job = job0; job < jobs; job += stride) {
                const KeyJob done(p, job);
                for (int j = done.j0 + half * 4 + warp % 4; j <= done.last; j += F::kWorkers / 32)
                    for (int which = 0; which < 2; ++which) mend_key_grad<T>(p, j, done.head, which, lane);
            }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 5) tensor_free<F::kColumns>(tensor);
    if (p.split > 1) {
        __syncwarp();
        cluster_meet();
        // each block takes its share of the rows of the cluster's one job
        const KeyJob job(p, job0);
        const int rows = kRows / p.split;
        for (int x = threadIdx.x; x < 2 * rows * (DP / 4); x += F::kThreads) {
            const int which = x / (rows * (DP / 4)), row = rank * rows + x / (DP / 4) % rows, c = x % (DP / 4) * 4, j = job.j0 + row;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int b = 0; b < p.split; ++b) {
                const float4 v = load_of_block(shared_address(shared) + which * kRows * DP * 4 + row * DP * 4 + ((c / 4) ^ (row % 8)) * 16, b);
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            if (j > job.last || c >= p.dim) continue;
            const float out[4] = {sum.x, sum.y, sum.z, sum.w};
            if (!(fmaf(sum.x, 0.f, fmaf(sum.y, 0.f, fmaf(sum.z, 0.f, sum.w * 0.f))) == 0.f)) spoilt = 1;
            store<T, 4>(static_cast<T*>(which ? p.dv : p.dk) + ((int64_t)j * p.heads_k + job.head) * p.dim + c, out);
        }
        __syncwarp();
        cluster_meet();                                 // nobody leaves while others read its shared memory
        __syncthreads();
        if (spoilt != 0 && lost == 0)
            for (int x = warp; x < 2 * rows; x += F::kThreads / 32)
                if (const int j = job.j0 + rank * rows + x % rows; j <= job.last) mend_key_grad<T>(p, j, job.head, x >= rows, lane);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult how;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &how) == cudaSuccess && how == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(f) : nullptr;
    }();
    return found;
}

// tokens x heads x dim; what lies outside is read as 0, columns behind dim among it
static bool map_of(CUtensorMap* map, uint32_t dtype, const void* p, int64_t dim, int64_t heads, int64_t tokens, int64_t head_stride, int64_t stride, int rows) {
    const cuuint64_t sizes[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head_stride * 2 : dim * 2), (cuuint64_t)(tokens > 1 ? stride * 2 : dim * heads * 2)};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, steps[3] = {1, 1, 1};
    return encoder()(map, dtype == NUKA_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), sizes, strides, box, steps,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A multiple of 16 bytes, and a streamed tile that begins at the last token ends within it.
int64_t attention_pitch(int64_t tokens) { return (tokens + kStream + 3) / 4 * 4; }

// Whole rows to a tile where rows of one length fill three quarters of it: queries then meet their keys within their own tile.
static int tile_span(const nuka_b200_episodes_t& plan) {
    const int64_t whole = plan.length > 0 && plan.length <= kRows ? kRows / plan.length * plan.length : 0;
    return 4 * whole >= 3 * kRows ? (int)whole : kRows;
}

template <typename K> static cudaError_t with_shared(K kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }

template <typename T, int DP> static cudaError_t run_attention(const nuka_b200_attention_t& d, bool backward, cudaStream_t stream) {
    AttentionParams p{};
    const nuka_b200_episodes_t& e = *d.plan;
    p.first = e.first; p.end = e.end; p.tokens = e.tokens; p.pitch = attention_pitch(e.tokens);
    p.heads_q = (int)d.heads_q; p.heads_k = (int)d.heads_k; p.dim = (int)d.dim; p.window = (int)std::min(d.window, e.tokens);
    p.span = tile_span(e); p.tiles = (int)((e.tokens + p.span - 1) / p.span);
    p.by_heads = p.heads_q / p.heads_k % 2 == 0;
    p.across = p.by_heads ? p.heads_q / 2 : p.heads_q; p.along = p.by_heads ? p.tiles : (p.tiles + 1) / 2;
    p.scale = d.scale; p.scale2 = d.scale * kLog2e;
    p.q = d.q; p.k = d.k; p.v = d.v; p.q_stride = d.q_stride; p.q_head_stride = d.q_head_stride; p.k_stride = d.k_stride; p.k_head_stride = d.k_head_stride;
    p.v_stride = d.v_stride; p.v_head_stride = d.v_head_stride;
    p.out = d.out; p.lse = d.lse; p.dout = d.dout; p.delta = d.delta; p.dq = d.dq; p.dk = d.dk; p.dv = d.dv;
    if (encoder() == nullptr) return cudaErrorNotSupported;
    CUtensorMap q, k, v, g, o;
    if (!backward) {
        // first, because it makes the device's context the thread's own: maps cannot be encoded without one
        cudaError_t set = with_shared(attention_kernel<T, DP>, Forward<DP>::kShared);
        if (set != cudaSuccess) return set;
        if (!map_of(&q, d.dtype, d.q, d.dim, d.heads_q, e.tokens, d.q_head_stride, d.q_stride, kRows) || !map_of(&k, d.dtype, d.k, d.dim, d.heads_k, e.tokens, d.k_head_stride, d.k_stride, Forward<DP>::kStep) ||
            !map_of(&v, d.dtype, d.v, d.dim, d.heads_k, e.tokens, d.v_head_stride, d.v_stride, Forward<DP>::kStep) || !map_of(&o, d.dtype, d.out, d.dim, d.heads_q, e.tokens, d.dim, d.dim * d.heads_q, p.span))
            return cudaErrorInvalidValue;
        attention_kernel<T, DP><<<(unsigned)std::min(p.across * p.along, 148), kForward, Forward<DP>::kShared, stream>>>(q, k, v, o, p);
        return cudaGetLastError();
    }
    CUtensorMap dq, dk, dv;
    for (int keys = 0; keys < 2; ++keys) {
        const int own = keys ? kStream : kRows, other = keys ? kRows : kStream;
        cudaError_t set = keys ? with_shared(key_grad_kernel<T, DP>, Keys<DP>::kShared) : with_shared(query_grad_kernel<T, DP>, Queries<DP>::kShared);
        if (set != cudaSuccess) return set;
        const int64_t wide = d.dim * d.heads_q, narrow = d.dim * d.heads_k;
        if (!map_of(&q, d.dtype, d.q, d.dim, d.heads_q, e.tokens, d.q_head_stride, d.q_stride, own) || !map_of(&g, d.dtype, d.dout, d.dim, d.heads_q, e.tokens, d.dim, wide, own) ||
            !map_of(&k, d.dtype, d.k, d.dim, d.heads_k, e.tokens, d.k_head_stride, d.k_stride, other) || !map_of(&v, d.dtype, d.v, d.dim, d.heads_k, e.tokens, d.v_head_stride, d.v_stride, other) ||
            !map_of(&o, d.dtype, d.out, d.dim, d.heads_q, e.tokens, d.dim, wide, kRows) || !map_of(&dq, d.dtype, d.dq, d.dim, d.heads_q, e.tokens, d.dim, wide, p.span) ||
            !map_of(&dk, d.dtype, d.dk, d.dim, d.heads_k, e.tokens, d.dim, narrow, p.span) || !map_of(&dv, d.dtype, d.dv, d.dim, d.heads_k, e.tokens, d.dim, narrow, p.span))
            return cudaErrorInvalidValue;
        // few jobs, that is long ones, are better dealt out by the hardware as blocks end
        const int jobs = p.tiles * (keys ? p.heads_k : p.heads_q), slots = 148 * (keys ? Keys<DP>::kBlocks : Queries<DP>::kBlocks), blocks = jobs <= 4 * slots ? jobs : slots, group = p.heads_q / p.heads_k;
        const int64_t row = e.tokens / std::max<int64_t>(e.rows, 1), reach = d.window > 0 ? std::min<int64_t>(row, d.window) : row, places = reach >= 1024 ? 4 * slots : slots;
        p.split = 1;
        while (keys && p.split < 8 && group % (2 * p.split) == 0 && 2 * p.split * (int64_t)jobs <= places) p.split *= 2;
        if (!keys) {
            query_grad_kernel<T, DP><<<(unsigned)blocks, Queries<DP>::kThreads, Queries<DP>::kShared, stream>>>(q, g, o, k, v, dq, p);
        } else if (p.split == 1) {
            key_grad_kernel<T, DP><<<(unsigned)blocks, Keys<DP>::kThreads, Keys<DP>::kShared, stream>>>(q, g, k, v, dk, dv, p);
        } else {
            cudaLaunchAttribute cluster{};
            cluster.id = cudaLaunchAttributeClusterDimension;
            cluster.val.clusterDim.x = (unsigned)p.split; cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1u;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3((unsigned)(jobs * p.split)); config.blockDim = dim3(Keys<DP>::kThreads); config.dynamicSmemBytes = Keys<DP>::kShared; config.stream = stream;
            config.attrs = &cluster; config.numAttrs = 1u;
            set = cudaLaunchKernelEx(&config, key_grad_kernel<T, DP>, q, g, k, v, dk, dv, p);
            if (set != cudaSuccess) return set;
        }
        set = cudaGetLastError();
        if (set != cudaSuccess) return set;
    }
    return cudaSuccess;
}

cudaError_t launch_attention(const nuka_b200_attention_t& d, bool backward, cudaStream_t stream) {
    if (d.plan->tokens == 0) return cudaSuccess;
    if (d.dtype == NUKA_B200_F16) return d.dim <= 64 ? run_attention<__half, 64>(d, backward, stream) : run_attention<__half, 128>(d, backward, stream);
    return d.dim <= 64 ? run_attention<__nv_bfloat16, 64>(d, backward, stream) : run_attention<__nv_bfloat16, 128>(d, backward, stream);
}

}  // namespace nkb
