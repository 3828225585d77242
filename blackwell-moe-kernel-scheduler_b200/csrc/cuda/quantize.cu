// Token rows -> 8-bit integers with one scale per row (the A operand of an INT8 product),
// gathered by index on the way: the dispatch permutation of bmoe_gather_rows with half the
// bytes written. Per row, FP32, one rounding per operation:
//   largest = max(max |x|, 2^-100), scale = largest / 127, q = rint(x * (127 * (1 / largest)))
// The floor keeps 1 / largest finite and makes a row of zeros quantise to zeros.
//
// Bound: HBM, 3 bytes per BF16 value, and close behind it the ALU (two integer operations a
// pair for the maximum, a shift or mask, a product, a sum and three quarters of a permutation
// per value). Measured on B200: 16384 rows of 2048 in 17 us (5.9 TB/s, 0.90 of a copy), 8192
// rows of 4096 gathered from 4096 in 15.9 us (10.3 for the bytes alone, the second reads
// come from L2), 512 rows of 7168 in 3.4 us. Two passes over the row, one value a thread, took
// 36.9 us for the gathered case; clamping before the conversion and FP32 maxima 18.2.
#include <cuda_runtime.h>

#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"

namespace bmoe {
namespace {

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

constexpr uint32_t kUnit = 16;            // values a thread takes at a time: one 16-byte store

// Without their sign, floats have the order of their bits, NaN above infinity: the largest
// |value| of a row is an integer maximum, two BF16 values at a time.
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// One unit in its own type.
template <typename T>
struct Unit {
  static constexpr uint32_t kVectors = kUnit * sizeof(T) / 16;
  uint4 v[kVectors];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // Running maximum of |values|, as bits: of pairs for BF16.
  __device__ __forceinline__ uint32_t raise(uint32_t most) const {
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i) {
      const uint32_t words[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 4) {
          most = max(most, words[w] & 0x7fffffffu);
        } else {
          most = max_pair(most, words[w] & 0x7fff7fffu);
        }
      }
    }
    return most;
  }
  __device__ __forceinline__ float at(uint32_t i) const {
    const uint32_t word = i * sizeof(T) / 4;
    const uint4& four = v[word / 4];
    const uint32_t bits =
        word % 4 == 0 ? four.x : (word % 4 == 1 ? four.y : (word % 4 == 2 ? four.z : four.w));
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(bits);
    } else {
      return __uint_as_float(i % 2 == 0 ? bits << 16 : bits & 0xffff0000u);
    }
  }
};

// Nearest integer, ties to even, as the low byte of the result: 1.5 * 2^23 + v has it there (an
// FP32 addition rounds to nearest even at that magnitude). |v| is at most 127 and a few
// roundings, so the integer is at most 127. What is not a number becomes -1; the row's scale
// then says NaN or inf. The product is rounded by itself (no fused multiply-add).
__device__ __forceinline__ uint32_t to_int8_bits(float v, float inverse) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inverse), 12582912.0f));
}

template <typename T>
__device__ __forceinline__ void store_unit(int8_t* to, const Unit<T>& unit, float inverse) {
  uint32_t word[4];
#pragma unroll
  for (uint32_t w = 0; w < 4; ++w) {
    const uint32_t b0 = to_int8_bits(unit.at(4 * w), inverse);
    const uint32_t b1 = to_int8_bits(unit.at(4 * w + 1), inverse);
    const uint32_t b2 = to_int8_bits(unit.at(4 * w + 2), inverse);
    const uint32_t b3 = to_int8_bits(unit.at(4 * w + 3), inverse);
    word[w] = __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
  }
  *reinterpret_cast<uint4*>(to) = make_uint4(word[0], word[1], word[2], word[3]);
}

// WARPS warps share a row; a CTA of one-warp rows holds four of them. A thread keeps HELD units
// in registers between the maximum and the conversion, so a row is read once; what is
// beyond (rows of more than 65536 values) is read again.
template <typename T, uint32_t WARPS, uint32_t HELD>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS)
quantize_rows_kernel(QuantizeArgs a) {
  __shared__ uint32_t partial[WARPS];
  constexpr uint32_t kThreads = 32 * WARPS;
  const uint64_t r =
      WARPS == 1 ? static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (r >= a.rows) return;
  const uint32_t thread = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t from = a.index != nullptr ? a.index[r] : static_cast<int64_t>(r);
  if (from < 0 || static_cast<uint64_t>(from) >= a.src_rows) return;
  const T* const row = static_cast<const T*>(a.src) + static_cast<uint64_t>(from) * a.src_stride;
  int8_t* const to = a.dst + r * a.cols;
  const uint32_t units = a.cols / kUnit;

  Unit<T> held[HELD];
#pragma unroll
  for (uint32_t i = 0; i < HELD; ++i) {
    const uint32_t u = i * kThreads + thread;
    if (u < units) {
      held[i].load(row + u * kUnit);
    } else {
      held[i].clear();
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (uint32_t i = 0; i < HELD; ++i) most = held[i].raise(most);
  for (uint32_t u = HELD * kThreads + thread; u < units; u += kThreads) {
    Unit<T> unit;
    unit.load(row + u * kUnit);
    most = unit.raise(most);
  }
  if constexpr (sizeof(T) == 2) most = max(most << 16, most & 0xffff0000u);
  most = __reduce_max_sync(0xffffffffu, most);
  if constexpr (WARPS > 1) {
    if ((thread & 31) == 0) partial[thread >> 5] = most;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) most = max(most, partial[w]);
  }
  // the floor 2^-100; NaN stays (its bits are above)
  const float largest = __uint_as_float(max(most, __float_as_uint(0x1p-100f)));
  const float inverse = __fmul_rn(127.0f, __fdiv_rn(1.0f, largest));
#pragma unroll
  for (uint32_t i = 0; i < HELD; ++i) {
    const uint32_t u = i * kThreads + thread;
    if (u < units) store_unit(to + u * kUnit, held[i], inverse);
  }
  for (uint32_t u = HELD * kThreads + thread; u < units; u += kThreads) {
    Unit<T> unit;
    unit.load(row + u * kUnit);
    store_unit(to + u * kUnit, unit, inverse);
  }
  if (thread == 0) a.scale[r] = largest / 127.0f;
}

template <typename T, uint32_t WARPS, uint32_t HELD>
cudaError_t launch_quantize(const QuantizeArgs& a, cudaStream_t stream) {
  const uint64_t grid = WARPS == 1 ? (a.rows + 3) / 4 : a.rows;
  quantize_rows_kernel<T, WARPS, HELD>
      <<<static_cast<uint32_t>(grid), WARPS == 1 ? 128 : 32 * WARPS, 0, stream>>>(a);
  return cudaPeekAtLastError();
}

// Threads by the length of a row: about four units (64 values) each.
template <typename T>
cudaError_t dispatch_quantize(const QuantizeArgs& a, cudaStream_t stream) {
  if (a.cols <= 512) return launch_quantize<T, 1, 1>(a, stream);
  if (a.cols <= 2048) return launch_quantize<T, 1, 4>(a, stream);
  if (a.cols <= 4096) return launch_quantize<T, 4, 2>(a, stream);
  if (a.cols <= 8192) return launch_quantize<T, 4, 4>(a, stream);
  if (a.cols <= 16384) return launch_quantize<T, 8, 4>(a, stream);
  return launch_quantize<T, 32, 4>(a, stream);
}

template <typename T>
cudaError_t preload_quantize() {
  cudaError_t rc = preload_one(quantize_rows_kernel<T, 1, 1>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<T, 1, 4>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<T, 4, 2>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<T, 4, 4>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<T, 8, 4>);
  if (rc == cudaSuccess) rc = preload_one(quantize_rows_kernel<T, 32, 4>);
  return rc;
}

}  // namespace

cudaError_t preload_quantize_kernels() {
  const cudaError_t rc = preload_quantize<uint16_t>();
  return rc == cudaSuccess ? preload_quantize<float>() : rc;
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
      a.rows > 0x7fffffffull ||
      (a.src_stride != 0 && (a.src_stride < a.cols || a.src_stride % (16 / elem) != 0))) {
    return BMOE_INVALID_ARGUMENT;
  }
  if (a.rows == 0) return BMOE_OK;
  if (a.src_dev == nullptr || a.dst_dev == nullptr || a.scale_dev == nullptr ||
      bmoe::off_grid(a.src_dev, 16) || bmoe::off_grid(a.dst_dev, 16) ||
      bmoe::off_grid(a.index_dev, 8) || bmoe::off_grid(a.scale_dev, 4) ||
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
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const cudaError_t rc = elem == 2 ? bmoe::dispatch_quantize<uint16_t>(k, stream)
                                   : bmoe::dispatch_quantize<float>(k, stream);
  return rc == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
