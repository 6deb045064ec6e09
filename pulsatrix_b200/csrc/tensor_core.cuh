// The fifth-generation tensor core as inline PTX for sm_100a: descriptors, tensor memory, matrix instructions of one CTA, and
// tiled copies into shared memory (no multicast).
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "psx_async.cuh"

namespace psx {

// A shared-memory operand with rows of 128 bytes, swizzled in 128-byte rows as the tiled copies write it (tiles start on 1024
// bytes).  Rows along the product's sum (K-major): `leading` is not used, `stride` is the distance of eight rows.  Rows along
// the other dimension (one row per summand): `leading` is the distance of the next 64 16-bit columns, `stride` that of eight rows.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address, uint32_t leading, uint32_t stride) {
    return (uint64_t)((address >> 4) & 0x3fff) | (uint64_t)((leading >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// 16-bit operands of one type, float accumulators; b_by_rows: B has one row per summand.
__host__ __device__ constexpr uint32_t product_descriptor(bool bfloat, bool b_by_rows, int m, int n) {
    return 1u << 4 | (bfloat ? 1u << 7 | 1u << 10 : 0u) | (b_by_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// d (tensor memory) = [d +] a b, both operands in shared memory / a in tensor memory.  One thread issues.
__device__ __forceinline__ void product_of_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :: "r"(d), "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void product_of_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :: "r"(d), "r"(a), "l"(b), "r"(kind), "r"((uint32_t)add) : "memory");
}
// One arrival on the barrier when everything that this thread has issued is done.
__device__ __forceinline__ void products_arrive(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar)) : "memory");
}

// One thread of a warp whose threads are all here.
__device__ __forceinline__ bool elected() {
    uint32_t mine;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(mine));
    return mine != 0;
}

__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_loads_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One warp; the first column's address lands in *address (shared memory).  columns: a power of two from 32 to 512.
__device__ __forceinline__ void tensor_allocate(uint32_t* address, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(address)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}

// 32 (16) columns of this thread's lane: x[i] is column i.  A warp reaches the 32 lanes that its number modulo 4 says.
__device__ __forceinline__ void tensor_load32(uint32_t address, float* x) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tensor_store32(uint32_t address, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
          "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
          "r"(address) : "memory");
}
__device__ __forceinline__ void tensor_store16(uint32_t address, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(address) : "memory");
}

// A box of a three-dimensional tensor into shared memory; its bytes complete on the barrier.  x times the element size is a
// multiple of 16 bytes; what lies outside the tensor arrives as zeros.
__device__ __forceinline__ void tiled_copy_to_shared(uint32_t to, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_address(bar)) : "memory");
}

// Writes to shared memory by this thread, ahead of what the asynchronous units (copies, matrix instructions) do next.
__device__ __forceinline__ void shared_writes_before_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace psx
