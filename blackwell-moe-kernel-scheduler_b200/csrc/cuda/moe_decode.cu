// A whole expert layer for a few tokens (a decode step), in two launches:
//   h[t, j] = silu(x[t] Wgate_e^T) * (x[t] Wup_e^T)      e = expert_ids[t, j]
//   out[t]  = bf16( sum_j weights[t, j] * (h[t, j] Wdown_e^T) )
// Simple form: one warp per (assignment, channel), h in FP32 in the workspace.
#include <cuda_runtime.h>

#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"

namespace bmoe {
namespace {

constexpr uint32_t kDecodeThreads = 256;

struct DecodeArgs {
  const uint16_t* x;
  const void* w1;
  const void* w2;
  const float* s1;
  const float* s2;
  const int64_t* ids;
  const float* coef;
  uint16_t* out;
  float* h;
  uint32_t tokens, top_k, experts, hidden, inter;
};

__device__ __forceinline__ float bf16(uint16_t v) {
  return __uint_as_float(static_cast<uint32_t>(v) << 16);
}
__device__ __forceinline__ float weight_of(const uint16_t* p) { return bf16(*p); }
__device__ __forceinline__ float weight_of(const int8_t* p) { return static_cast<float>(*p); }

__device__ __forceinline__ float warp_sum(float v) {
  for (uint32_t d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

template <typename W>
__global__ void __launch_bounds__(kDecodeThreads) decode_up_kernel(DecodeArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t i = blockIdx.x * (kDecodeThreads / 32) + (threadIdx.x >> 5);
  const uint32_t r = blockIdx.y;
  const int64_t e = a.ids[r];
  if (i >= a.inter || e < 0 || e >= a.experts) return;
  const uint16_t* const x = a.x + static_cast<size_t>(r / a.top_k) * a.hidden;
  const size_t row = static_cast<size_t>(e) * 2 * a.inter + i;
  const W* const gate = static_cast<const W*>(a.w1) + row * a.hidden;
  const W* const up = gate + static_cast<size_t>(a.inter) * a.hidden;
  float g = 0.0f, u = 0.0f;
  for (uint32_t k = lane; k < a.hidden; k += 32) {
    const float v = bf16(x[k]);
    g = fmaf(weight_of(gate + k), v, g);
    u = fmaf(weight_of(up + k), v, u);
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (a.s1 != nullptr) {
    g *= a.s1[row];
    u *= a.s1[row + a.inter];
  }
  if (lane == 0) a.h[static_cast<size_t>(r) * a.inter + i] = g / (1.0f + expf(-g)) * u;
}

template <typename W>
__global__ void __launch_bounds__(kDecodeThreads) decode_down_kernel(DecodeArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t n = blockIdx.x * (kDecodeThreads / 32) + (threadIdx.x >> 5);
  const uint32_t t = blockIdx.y;
  if (n >= a.hidden) return;
  float sum = 0.0f;
  for (uint32_t j = 0; j < a.top_k; ++j) {
    const uint32_t r = t * a.top_k + j;
    const int64_t e = a.ids[r];
    if (e < 0 || e >= a.experts) continue;
    const size_t row = static_cast<size_t>(e) * a.hidden + n;
    const W* const w = static_cast<const W*>(a.w2) + row * a.inter;
    const float* const h = a.h + static_cast<size_t>(r) * a.inter;
    float part = 0.0f;
    for (uint32_t k = lane; k < a.inter; k += 32) part = fmaf(weight_of(w + k), h[k], part);
    part = warp_sum(part);
    if (a.s2 != nullptr) part *= a.s2[row];
    sum = fmaf(a.coef[r], part, sum);
  }
  if (lane == 0) {
    uint16_t b;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(sum));
    a.out[static_cast<size_t>(t) * a.hidden + n] = b;
  }
}

template <typename W>
cudaError_t launch_decode(const DecodeArgs& a, cudaStream_t stream) {
  const uint32_t warps = kDecodeThreads / 32;
  decode_up_kernel<W><<<dim3((a.inter + warps - 1) / warps, a.tokens * a.top_k), kDecodeThreads,
                        0, stream>>>(a);
  decode_down_kernel<W><<<dim3((a.hidden + warps - 1) / warps, a.tokens), kDecodeThreads, 0,
                          stream>>>(a);
  return cudaPeekAtLastError();
}

bool unaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

cudaError_t preload_decode_kernels() {
  cudaError_t rc = preload_one(decode_up_kernel<uint16_t>);
  if (rc == cudaSuccess) rc = preload_one(decode_up_kernel<int8_t>);
  if (rc == cudaSuccess) rc = preload_one(decode_down_kernel<uint16_t>);
  if (rc == cudaSuccess) rc = preload_one(decode_down_kernel<int8_t>);
  return rc;
}

}  // namespace bmoe

extern "C" uint64_t bmoe_moe_decode_workspace(uint32_t tokens, uint32_t top_k, uint32_t inter) {
  return (static_cast<uint64_t>(tokens) * top_k * inter * sizeof(float) + 255) / 256 * 256;
}

extern "C" int bmoe_moe_decode(const bmoe_moe_decode_args* args) {
  if (args == nullptr) return BMOE_INVALID_ARGUMENT;
  const bmoe_moe_decode_args& a = *args;
  if (a.data_type != BMOE_TYPE_BF16 && a.data_type != BMOE_TYPE_INT8) {
    return BMOE_UNSUPPORTED_DATA_TYPE;
  }
  const bool int8 = a.data_type == BMOE_TYPE_INT8;
  const uint32_t step = int8 ? 16u : 8u;
  if (a.tokens > BMOE_MOE_DECODE_MAX_TOKENS || a.top_k == 0 ||
      a.top_k > BMOE_MOE_DECODE_MAX_TOP_K || a.experts == 0 ||
      a.experts > BMOE_MOE_DECODE_MAX_EXPERTS || a.hidden == 0 || a.hidden % step != 0 ||
      a.inter == 0 || a.inter % step != 0 || a.hidden > (1u << 24) || a.inter > (1u << 24)) {
    return BMOE_INVALID_ARGUMENT;
  }
  if (a.tokens == 0) return BMOE_OK;
  if (a.x_dev == nullptr || a.w_gate_up_dev == nullptr || a.w_down_dev == nullptr ||
      a.expert_ids_dev == nullptr || a.weights_dev == nullptr || a.out_dev == nullptr ||
      a.workspace_dev == nullptr || bmoe::unaligned(a.x_dev) || bmoe::unaligned(a.w_gate_up_dev) ||
      bmoe::unaligned(a.w_down_dev) || bmoe::unaligned(a.out_dev) ||
      (reinterpret_cast<uintptr_t>(a.workspace_dev) & 255u) != 0 ||
      a.workspace_bytes < bmoe_moe_decode_workspace(a.tokens, a.top_k, a.inter) ||
      (int8 && (a.gate_up_scale_dev == nullptr || a.down_scale_dev == nullptr))) {
    return BMOE_INVALID_ARGUMENT;
  }
  bmoe::DecodeArgs k;
  k.x = static_cast<const uint16_t*>(a.x_dev);
  k.w1 = a.w_gate_up_dev;
  k.w2 = a.w_down_dev;
  k.s1 = int8 ? a.gate_up_scale_dev : nullptr;
  k.s2 = int8 ? a.down_scale_dev : nullptr;
  k.ids = a.expert_ids_dev;
  k.coef = a.weights_dev;
  k.out = static_cast<uint16_t*>(a.out_dev);
  k.h = static_cast<float*>(a.workspace_dev);
  k.tokens = a.tokens;
  k.top_k = a.top_k;
  k.experts = a.experts;
  k.hidden = a.hidden;
  k.inter = a.inter;
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const cudaError_t rc = int8 ? bmoe::launch_decode<int8_t>(k, stream)
                              : bmoe::launch_decode<uint16_t>(k, stream);
  return rc == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
