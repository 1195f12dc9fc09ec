// The 5th-generation tensor cores (tcgen05) and tiled asynchronous copies, as the matrix products in matmul.cuh use them.
//
// One thread issues the products: both operands lie in shared memory as tiles of 64 values x 64 rows (8 KB) in the 128-byte swizzle that
// the tiled copy writes, the 32-bit accumulator of 128 rows lies in tensor memory, one lane per row and one column per value.  A tile's
// contiguous direction is either the one that is summed over ("K-major") or the rows or columns of the result ("MN-major"); both are
// read in place, so that no operand is ever transposed in memory.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "tma.cuh"

namespace dl {

constexpr int kChunk = 64;                       // values in a tile's contiguous direction, and rows of a tile
constexpr int kChunkBytes = kChunk * kChunk * 2;  // one copied tile

#ifdef __CUDACC__
// PAIR: two CTAs of a cluster work on one tile.  The barrier is then the first one's: `bar` is its address in the cluster.
template <bool PAIR>
__device__ __forceinline__ void tile_load(void *dst, const CUtensorMap *map, int inner, int row, int plane, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         smem_addr(dst)),
                     "l"(map), "r"(inner), "r"(row), "r"(plane), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         smem_addr(dst)),
                     "l"(map), "r"(inner), "r"(row), "r"(plane), "r"(bar)
                     : "memory");
}
__device__ __forceinline__ void map_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address in the cluster of what lies at p in the shared memory of its CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void mbar_arrive_in_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Tensor memory: a whole warp (of both CTAs of a pair) takes `columns` (a power of two, 32 to 512) and gives them back.
template <bool PAIR>
__device__ __forceinline__ void tensor_alloc(uint32_t *where, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D (+)= A B^T over 16 values: 128 rows (256 of a pair, 128 in each CTA, which holds those of A and half of B), the instruction
// descriptor says how many columns.
template <bool PAIR>
__device__ __forceinline__ void tensor_multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
            : "memory");
}
// Arrives on `bar` (of both CTAs of a pair) once all products issued so far are done, and their reads of shared memory with them.
template <bool PAIR>
__device__ __forceinline__ void tensor_commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// 32 columns of the warp's 32 lanes of tensor memory: lane = row.
__device__ __forceinline__ void tensor_read32(uint32_t address, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(address));
}
__device__ __forceinline__ void tensor_read_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Descriptor of an operand in shared memory, 128-byte swizzle.  K-major: rows of 128 bytes, 8-row groups every 1024 bytes, 16 values
// further is 32 bytes further.  MN-major: 8 rows of the sum every 1024 bytes, the next 64 rows (columns) of the result a chunk
// further; 16 rows of the sum are 2048 bytes.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address) {
    return (uint64_t)((address >> 4) & 0x3FFF) | (uint64_t)(kChunkBytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
#endif

// 32-bit accumulation of fp16 (bf16: bfloat) operands, rows x columns.
static inline uint32_t instruction_descriptor(bool bfloat, bool a_mn, bool b_mn, int rows, int columns) {
    return 1u << 4 | (uint32_t)bfloat << 7 | (uint32_t)bfloat << 10 | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 |
           (uint32_t)(columns / 8) << 17 | (uint32_t)(rows / 16) << 24;
}

// Map of `planes` matrices of rows x inner 16-bit values, copied in tiles of tile_rows x 64; what lies outside reads as zero.  False where the
// driver does not take it (base and pitches must be multiples of 16 bytes).
bool make_tile_map(CUtensorMap *map, const void *base, bool bfloat, int64_t inner, int64_t rows, int64_t planes, int64_t row_bytes,
                   int64_t plane_bytes, int tile_rows);

}  // namespace dl
