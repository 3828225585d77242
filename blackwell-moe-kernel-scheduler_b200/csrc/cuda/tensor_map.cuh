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

// Box of a tensor of `rank` dimensions, innermost first: box[0] elements are 128 bytes of
// contiguous memory (SWIZZLE_128B), strides[i] the bytes between neighbours of dimension i + 1,
// each a multiple of the one before.
inline bool encode_box(CUtensorMap* map, const void* base, Elem type, uint32_t rank,
                       const uint64_t* dims, const uint64_t* strides, const uint32_t* box) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr || rank > 5) return false;
  const CUtensorMapDataType kind =
      type == Elem::kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : (type == Elem::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8);
  cuuint64_t size[5], stride[4];
  cuuint32_t extent[5];
  const cuuint32_t elem_strides[5] = {1, 1, 1, 1, 1};
  for (uint32_t i = 0; i < rank; ++i) {
    size[i] = dims[i];
    extent[i] = box[i];
    if (i + 1 < rank) stride[i] = strides[i];
  }
  return encode(map, kind, rank, const_cast<void*>(base), size, stride, extent, elem_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace bmoe
