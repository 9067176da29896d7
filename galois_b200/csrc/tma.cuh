// Tiled bulk copies (TMA): the host side's tensor maps and the device side's loads.  None of them is multicast.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "ptx.cuh"

// Fills *map for a tensor of `rank` dimensions (sizes in elements, strides of dimensions 1.. in bytes, multiples of
// 16) that is copied in boxes of `box` elements; rows of a box are 64 or 128 bytes, swizzled over as many.  Places
// outside the tensor read as zeros.  0, or a failure recorded on the context.
int gb_tensor_map(galois_b200_ctx* ctx, CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* size,
                  const uint64_t* stride, const uint32_t* box, int row_bytes);

#ifdef __CUDACC__
// One box to shared memory (its address a multiple of 1024), completing on an mbarrier.  Coordinate x0 is always a
// multiple of the box's row.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x0, int x1, int x2, int x3, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map),
                 "r"(smem_u32(bar)), "r"(x0), "r"(x1), "r"(x2), "r"(x3)
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x0, int x1, int x2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
                 "r"(smem_u32(bar)), "r"(x0), "r"(x1), "r"(x2)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
#endif
