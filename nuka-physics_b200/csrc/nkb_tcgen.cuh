// Inline PTX of the tensor-core kernels: barriers in shared memory, TMA loads, 5th-generation tensor-core products with
// accumulators in tensor memory.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace nkb {

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- barriers -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(bar)), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(shared_address(bar)), "r"(parity) : "memory");
    return done != 0u;
}
// A wait gives up after about 2 s, or when another warp of the block gave up: the block then ends its work, and its outputs become NaN.
// The clock is read at each turn: sixteen tries between two readings go on a little later (queries' gradients of 98304 x 8 x 64 in rows of 24: 121 us, against 111 so).
constexpr long long kBarrierCycles = 4000000000ll;
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, uint32_t parity, volatile int* lost) {
    if (barrier_try(bar, parity)) return true;
    const long long began = clock64();
    for (;;) {
        if (barrier_try(bar, parity)) return true;
        if (*lost != 0) return false;
        if (clock64() - began > kBarrierCycles) { *lost = 1; return false; }
    }
}

// ---- clusters -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// all threads of all blocks; what was written to shared memory before is seen after
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.release.aligned; barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 load_of_block(uint32_t address, uint32_t rank) {
    float4 v;
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
    return v;
}

// ---- TMA --------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void load_tile(void* to, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(shared_address(to)),
                 "l"(map), "r"(shared_address(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
// both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void load_bytes(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(to)), "l"(from), "r"(bytes), "r"(shared_address(bar)) : "memory");
}
// a tile out of shared memory, which is written by the thread's group of stores; what lies outside the tensor is left out
__device__ __forceinline__ void store_tile(const CUtensorMap* map, const void* from, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(shared_address(from)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void stores_end() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }        // their shared memory may be written again
__device__ __forceinline__ void wait_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }              // ordinary stores before, TMA after
__device__ __forceinline__ void meet(int which, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(which), "r"(threads) : "memory"); }

// ---- tensor memory ------------------------------------------------------------------------------------------------------
template <int COLUMNS> __device__ __forceinline__ void tensor_alloc(uint32_t* to) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(to)), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLUMNS> __device__ __forceinline__ void tensor_free(uint32_t at) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(COLUMNS)); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes, a lane to a thread
__device__ __forceinline__ void tensor_load(uint32_t at, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tensor_store(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

// 16 columns; 8 columns
__device__ __forceinline__ void tensor_load16(uint32_t at, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tensor_store8(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

// ---- products -----------------------------------------------------------------------------------------------------------
// Operands in shared memory are rows of 128 bytes (64 values), swizzled by the TMA load's 128-byte mode, panels of 64 columns one behind the other.
// As rows x 64 columns of the product's inner dimension (K-major): 8 rows are 1024 bytes.  The step to the next 16 inner values is 32 bytes.
__device__ __forceinline__ uint64_t inner_rows(uint32_t address) {
    return (uint64_t)((address & 0x3ffffu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The same bytes with the rows as the inner dimension and the 64 columns as the outer one (MN-major): 8 rows are 1024 bytes, the next 64 columns a panel
// further.  The step to the next 16 rows is 2048 bytes.
__device__ __forceinline__ uint64_t outer_rows(uint32_t address, uint32_t panel) {
    return (uint64_t)((address & 0x3ffffu) >> 4) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 128 x N, accumulated in 32 bits; both operands bf16 or both f16; b_outer: B is MN-major
template <typename T> __host__ __device__ constexpr uint32_t product_of(int n, bool b_outer) {
    return 1u << 4 | (sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? (1u << 7 | 1u << 10) : 0u) | (b_outer ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
// The whole warp calls these, and one lane of it issues: inside a branch of one lane the compiler cannot keep the operands in uniform registers, and moving them there takes
// longer than the product (75 cycles an instruction in place of 30).
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{ .reg .pred e, p; elect.sync _|e, 0xffffffff; setp.ne.u32 p, %4, 0; @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(what),
                 "r"((uint32_t)add) : "memory");
}
// A from tensor memory, two values to a column
__device__ __forceinline__ void multiply_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{ .reg .pred e, p; elect.sync _|e, 0xffffffff; setp.ne.u32 p, %4, 0; @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(what),
                 "r"((uint32_t)add) : "memory");
}
// the barrier completes when the products that the warp issued so far have
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("{ .reg .pred e; elect.sync _|e, 0xffffffff; @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(shared_address(bar)) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two 32-bit values at a time
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float low, float high) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(low), "f"(high));
    return r;
}
__device__ __forceinline__ void split(Pair p, float& low, float& high) { asm("mov.b64 {%0, %1}, %2;" : "=f"(low), "=f"(high) : "l"(p)); }
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul_pair(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t pack(float low, float high);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float low, float high) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float low, float high) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}

}  // namespace nkb
