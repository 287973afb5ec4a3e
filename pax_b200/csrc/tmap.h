// tmap.h -- the driver's tensor-map encoder, looked up once per translation
// unit, and the map of a plain matrix.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <mutex>

namespace pax {

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// Map of a row-major matrix, rows x cols elements of `elem` bytes, ld elements
// between rows; box of box_cols x box_rows (x 1: the maps have a third
// dimension of one), 128B swizzle.
inline bool matrix_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int elem, long long rows,
                       long long cols, long long ld, uint32_t box_cols, uint32_t box_rows) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const uint64_t pitch = (uint64_t)ld * elem;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
    cuuint64_t strides[2] = {pitch, (pitch * (uint64_t)rows + 15) & ~uint64_t(15)};
    cuuint32_t box[3] = {box_cols, box_rows, 1}, estr[3] = {1, 1, 1};
    return enc(m, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Element types of the feed-forward products' maps.
constexpr CUtensorMapDataType kF16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kF32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                              kU8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;

}  // namespace pax
