// Host encoding of the TMA descriptors the kernels of this library use.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace bmoe {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled is resolved through the runtime so the library has no
// link-time dependency on libcuda.
inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult query = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault,
                                &query) != cudaSuccess ||
        query != cudaDriverEntryPointSuccess) {
      return nullptr;
    }
    return reinterpret_cast<EncodeTiledFn>(sym);
  }();
  return fn;
}

// Element type of a matrix a tensor map describes.
enum class Elem : uint32_t { kBf16, kF32, kByte };

// Row-major matrix [rows, cols] viewed as a 2-D tensor {cols, rows} with a SWIZZLE_128B
// box of 128 bytes (64 BF16 / 32 FP32 / 128 one-byte columns) x box_rows rows.
inline bool encode_matrix(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols,
                   uint32_t box_rows, Elem type) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  const uint32_t elem = type == Elem::kF32 ? 4u : (type == Elem::kBf16 ? 2u : 1u);
  const CUtensorMapDataType kind =
      type == Elem::kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : (type == Elem::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8);
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {cols * elem};
  const cuuint32_t box[2] = {128u / elem, box_rows};
  const cuuint32_t elem_strides[2] = {1, 1};
  const CUresult rc = encode(
      map, kind, 2, const_cast<void*>(base), dims, strides,
      box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS;
}

}  // namespace bmoe
