// Maps for tiled copies, encoded by the driver.
#include "tensor_core.cuh"

namespace dl {

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

bool make_tile_map(CUtensorMap *map, const void *base, bool bfloat, int64_t inner, int64_t rows, int64_t planes, int64_t row_bytes,
                   int64_t plane_bytes, int tile_rows) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    if (planes == 1) plane_bytes = row_bytes * rows;   // not used, but looked at
    const cuuint64_t sizes[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t pitches[2] = {(cuuint64_t)row_bytes, (cuuint64_t)plane_bytes};
    const cuuint32_t box[3] = {kChunk, (cuuint32_t)tile_rows, 1}, steps[3] = {1, 1, 1};
    return encode(map, bfloat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), sizes,
                  pitches, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace dl
