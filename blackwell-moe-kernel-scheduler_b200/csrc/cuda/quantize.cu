// Token rows -> 8-bit integers with one scale per row (the A operand of an INT8 product),
// gathered by index on the way: the dispatch permutation of bmoe_gather_rows with half the
// bytes written. Per row, FP32, one rounding per operation:
//   largest = max(max |x|, 2^-100), scale = largest / 127, q = rint(x * (127 * (1 / largest)))
// The floor keeps 1 / largest finite and makes a row of zeros quantise to zeros.
#include <cuda_runtime.h>

#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"

namespace bmoe {
namespace {

constexpr uint32_t kQuantThreads = 256;

struct QuantizeArgs {
  const void* src;
  const int64_t* index;
  int8_t* dst;
  float* scale;
  uint64_t rows;
  uint64_t src_rows;
  uint64_t src_stride;
  uint32_t cols;
};

// max of |values| that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const uint16_t* p) {
  return __uint_as_float(static_cast<uint32_t>(*p) << 16);
}

// Nearest integer, ties to even; what is not a number becomes -127 (the row's scale then
// says NaN or inf).
__device__ __forceinline__ int8_t to_int8(float v) {
  const int q = __float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f));
  return static_cast<int8_t>(q);
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(QuantizeArgs a) {
  __shared__ float partial[kQuantThreads / 32];
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t from = a.index != nullptr ? a.index[r] : static_cast<int64_t>(r);
    if (from < 0 || static_cast<uint64_t>(from) >= a.src_rows) continue;
    const T* const row = static_cast<const T*>(a.src) + static_cast<uint64_t>(from) * a.src_stride;
    float largest = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kQuantThreads) {
      largest = max_nan(largest, fabsf(load_value(row + c)));
    }
    for (uint32_t d = 16; d > 0; d >>= 1) {
      largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, d));
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) partial[threadIdx.x >> 5] = largest;
    __syncthreads();
    for (uint32_t w = 0; w < kQuantThreads / 32; ++w) largest = max_nan(largest, partial[w]);
    largest = max_nan(largest, 0x1p-100f);
    const float inverse = 127.0f * (1.0f / largest);
    for (uint32_t c = threadIdx.x; c < a.cols; c += kQuantThreads) {
      a.dst[r * a.cols + c] = to_int8(load_value(row + c) * inverse);
    }
    if (threadIdx.x == 0) a.scale[r] = largest / 127.0f;
  }
}

}  // namespace

cudaError_t preload_quantize_kernels() {
  cudaError_t rc = preload_one(quantize_rows_kernel<uint16_t>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<float>);
  return rc;
}

}  // namespace bmoe

extern "C" int bmoe_quantize_rows(const bmoe_quantize_rows_args* args) {
  if (args == nullptr) return BMOE_INVALID_ARGUMENT;
  const bmoe_quantize_rows_args& a = *args;
  if (a.src_type != BMOE_TYPE_BF16 && a.src_type != BMOE_TYPE_FP32) {
    return BMOE_UNSUPPORTED_DATA_TYPE;
  }
  const uint32_t elem = a.src_type == BMOE_TYPE_BF16 ? 2u : 4u;
  if (a.cols == 0 || a.cols % 16 != 0 ||
      (a.src_stride != 0 && (a.src_stride < a.cols || a.src_stride % (16 / elem) != 0))) {
    return BMOE_INVALID_ARGUMENT;
  }
  if (a.rows == 0) return BMOE_OK;
  if (a.src_dev == nullptr || a.dst_dev == nullptr || a.scale_dev == nullptr ||
      (reinterpret_cast<uintptr_t>(a.src_dev) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(a.dst_dev) & 15u) != 0 ||
      (a.index_dev == nullptr && a.rows > a.src_rows)) {
    return BMOE_INVALID_ARGUMENT;
  }
  bmoe::QuantizeArgs k;
  k.src = a.src_dev;
  k.index = a.index_dev;
  k.dst = a.dst_dev;
  k.scale = a.scale_dev;
  k.rows = a.rows;
  k.src_rows = a.src_rows;
  k.src_stride = a.src_stride != 0 ? a.src_stride : a.cols;
  k.cols = a.cols;
  const uint64_t resident = 8ull * bmoe::device_sm_count();
  const uint32_t grid = static_cast<uint32_t>(a.rows < resident ? a.rows : resident);
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  if (elem == 2) {
    bmoe::quantize_rows_kernel<uint16_t><<<grid, bmoe::kQuantThreads, 0, stream>>>(k);
  } else {
    bmoe::quantize_rows_kernel<float><<<grid, bmoe::kQuantThreads, 0, stream>>>(k);
  }
  return cudaPeekAtLastError() == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
