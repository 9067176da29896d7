// Tensor maps for the kernels that copy tiles with TMA.
#include "tma.cuh"

#include <atomic>

int gb_tensor_map(galois_b200_ctx* ctx, CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* size,
                  const uint64_t* stride, const uint32_t* box, int row_bytes) {
    // the driver's function, looked up once (the library links the runtime only); contexts may do so in several threads
    typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<encode_fn> found_before{nullptr};
    encode_fn encode = found_before.load(std::memory_order_acquire);
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        GB_CUDA(ctx, cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !fn) return gb_fail(ctx, GALOIS_B200_E_STATE, "the driver has no cuTensorMapEncodeTiled");
        encode = (encode_fn)fn;
        found_before.store(encode, std::memory_order_release);
    }
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(map, type, (cuuint32_t)rank, const_cast<void*>(base), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return gb_fail(ctx, GALOIS_B200_E_LAYOUT, "cuTensorMapEncodeTiled refuses the layout (status %d)", (int)r);
    return 0;
}
