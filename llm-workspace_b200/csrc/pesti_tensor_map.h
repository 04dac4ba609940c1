// Tensor maps of row-major matrices for bulk tensor copies in 128-byte swizzled boxes.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/pesti_sampler.h"
#include "pesti_error.h"

static inline CUtensorMapDataType pesti_map_type(pesti_dtype dtype) {
  return dtype == PESTI_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : dtype == PESTI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// `rows` rows of `columns` elements, row_bytes apart (a multiple of 16); boxes of box_columns x box_rows, whose rows are
// 128 bytes.  Elements outside the matrix are read as 0 and not written.
static inline int pesti_tensor_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long columns,
                                   long long rows, long long row_bytes, int box_columns, int box_rows) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> found_encode{nullptr};  // the same value whoever writes it
  Encode encode = found_encode.load(std::memory_order_relaxed);
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return pesti_set_cuda_error(e, "cuTensorMapEncodeTiled");
    if (found != cudaDriverEntryPointSuccess || !f)
      return pesti_set_error(PESTI_E_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
    encode = (Encode)f;
    found_encode.store(encode, std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult rc = encode(map, type, 2, (void*)base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? PESTI_OK : pesti_set_error(PESTI_E_CUDA, "cuTensorMapEncodeTiled failed");
}
