// The router's choice: logits [tokens, experts] -> the top-k experts of every token and
// their weights, the inputs of the expert-parallel count / route kernels, of the top-k
// combine and of the few-token layer. The reference has no router: routed token counts are
// its input (agent/search_space.yaml:10-13).
//
//   softmax:  key = logit                    score = exp(logit - max) / sum
//   sigmoid:  key = sigmoid(logit) + bias    score = sigmoid(logit)   (key = logit if no bias)
// The k largest keys are chosen, largest first, the lower id first among equals.
//
// One warp per token. Keys live in registers as unsigned integers whose order is the
// order of the floats; a choice is one warp maximum over the keys and one warp minimum
// over the ids that hold it.
//
// Bound: latency (loads, top_k dependent rounds) for few tokens, instruction issue for many (77 %
// of the slots; the bytes alone would take 0.9 us). Measured on B200: 16384 x 128 BF16, top-8,
// softmax 9.0 us; 4 x 256 FP32, top-8, sigmoid with bias 4.9 us. Scanning all keys of a lane in
// every round instead of sorting them once took 11.0 us; one packed 32-bit key and id for
// BF16, which saves the second warp operation, measured no faster (9.0).
#include <cuda_runtime.h>

#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"

namespace bmoe {
namespace {

constexpr uint32_t kRouteTopkThreads = 128;
constexpr uint32_t kFull = 0xffffffffu;

struct RouteTopkArgs {
  const void* logits;
  const float* bias;
  int64_t* ids;
  float* weights;
  uint64_t tokens;
  uint64_t row_stride;
  uint32_t experts;
  uint32_t top_k;
  float scale;
};

// Unsigned keys in the order of the floats, 0 for what cannot be chosen (NaN, -inf).
// Both zeros are equal, so the lower id goes first.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t bits = __float_as_uint(v + 0.0f);
  return (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ unsigned long long order_key(double v) {
  if (!(v > -static_cast<double>(INFINITY))) return 0ull;
  const unsigned long long bits =
      static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (bits >> 63) != 0 ? ~bits : bits | 0x8000000000000000ull;
}

// The float of a 32-bit key.
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) != 0 ? key & 0x7fffffffu : ~key);
}

// Distance below which sums sigmoid + bias computed in 32 bits may be in another order than
// their exact values: the sigmoid is off by at most 2^-22 (exponential one step, sum and
// quotient half a step each), the sum by half a step of itself, both keys count: 2^-21 + 2^-23
// for sums up to 1, doubled.
constexpr float kCloseSums = 0x1p-20f;

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kFull, v); }

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(kFull, static_cast<uint32_t>(v >> 32));
  const uint32_t mine = static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u;
  return static_cast<unsigned long long>(hi) << 32 | __reduce_max_sync(kFull, mine);
}

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const uint16_t* p) {
  return __uint_as_float(static_cast<uint32_t>(*p) << 16);
}

// top_k rounds of "largest key, lowest id" over the lane's V keys (key i belongs to
// expert i * 32 + lane). Lane j returns the id of the j-th choice (or -1). Up to 8 keys are
// sorted first (odd-even transposition, equal keys stay in the order of their ids), so that
// a round only looks at the front one: two warp operations and one shift.
// With CLOSE, *close tells whether two neighbours among the chosen, or the last one and the next
// in line, are so close that 32-bit keys do not decide their order.
template <bool CLOSE, typename Key, uint32_t V>
__device__ __forceinline__ int choose(Key (&key)[V], uint32_t top_k, uint32_t lane,
                                      bool* close) {
  int mine = -1;
  float above = INFINITY;
  auto check = [&](Key top) {
    if constexpr (CLOSE) {
      const float v = top != 0 ? key_value(top) : -INFINITY;
      if (above - v <= kCloseSums * fmaxf(1.0f, fabsf(v))) *close = true;
      above = v;
    }
  };
  if constexpr (V <= 8) {
    uint32_t id[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) id[i] = i * 32 + lane;
#pragma unroll
    for (uint32_t round = 0; round < V; ++round) {
#pragma unroll
      for (uint32_t i = round & 1; i + 1 < V; i += 2) {
        if (key[i + 1] > key[i]) {
          const Key k = key[i];
          key[i] = key[i + 1];
          key[i + 1] = k;
          const uint32_t e = id[i];
          id[i] = id[i + 1];
          id[i + 1] = e;
        }
      }
    }
    for (uint32_t j = 0; j < top_k + (CLOSE ? 1 : 0); ++j) {
      const Key top = warp_max(key[0]);
      if (top == 0) break;   // nothing left that can be chosen
      check(top);
      if (CLOSE && j == top_k) break;
      const uint32_t chosen = __reduce_min_sync(kFull, key[0] == top ? id[0] : kFull);
      if (lane == j) mine = static_cast<int>(chosen);
      if (id[0] == chosen) {
#pragma unroll
        for (uint32_t i = 0; i + 1 < V; ++i) {
          key[i] = key[i + 1];
          id[i] = id[i + 1];
        }
        key[V - 1] = 0;
      }
    }
    return mine;
  }
  for (uint32_t j = 0; j < top_k + (CLOSE ? 1 : 0); ++j) {
    Key best = 0;
    uint32_t at = 0;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    }
    const Key top = warp_max(best);
    if (top == 0) break;   // nothing left that can be chosen
    check(top);
    if (CLOSE && j == top_k) break;
    const uint32_t id = __reduce_min_sync(kFull, best == top ? at * 32 + lane : kFull);
    if (lane == j) mine = static_cast<int>(id);
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
      if (i * 32 + lane == id) key[i] = 0;
    }
  }
  return mine;
}

// V keys per lane; SIGMOID with BIAS chooses by the sum, in 64 bits where 32 do not decide.
template <typename T, uint32_t V, bool SIGMOID, bool BIAS>
__global__ void __launch_bounds__(kRouteTopkThreads)
route_topk_kernel(RouteTopkArgs a, uint32_t renormalize) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t token =
      static_cast<uint64_t>(blockIdx.x) * (kRouteTopkThreads / 32) + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  const T* const row = static_cast<const T*>(a.logits) + token * a.row_stride;
  float logit[V];
#pragma unroll
  for (uint32_t i = 0; i < V; ++i) {
    const uint32_t e = i * 32 + lane;
    logit[i] = e < a.experts ? load_logit(row + e) : -INFINITY;
  }

  int id;
  bool close = false;
  if constexpr (SIGMOID && BIAS) {
    uint32_t key[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
      const uint32_t e = i * 32 + lane;
      const float b = e < a.experts ? a.bias[e] : 0.0f;
      key[i] = logit[i] > -INFINITY ? order_key(1.0f / (1.0f + expf(-logit[i])) + b) : 0u;
    }
    id = choose<true>(key, a.top_k, lane, &close);
  } else {
    uint32_t key[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) key[i] = order_key(logit[i]);
    id = choose<false>(key, a.top_k, lane, &close);
  }
  if (SIGMOID && BIAS && close) {
    // (the whole warp) once in some thousand tokens: decided by the sums in 64 bits
    unsigned long long key[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
      const uint32_t e = i * 32 + lane;
      const double b = e < a.experts ? static_cast<double>(a.bias[e]) : 0.0;
      const double sum = 1.0 / (1.0 + exp(-static_cast<double>(logit[i]))) + b;
      key[i] = logit[i] > -INFINITY ? order_key(sum) : 0ull;
    }
    id = choose<false>(key, a.top_k, lane, &close);
  }

  // The chosen logit, from the row again (it is in L1).
  const float mine = id >= 0 ? load_logit(row + id) : -INFINITY;
  float score;
  if constexpr (SIGMOID) {
    score = id >= 0 ? 1.0f / (1.0f + expf(-mine)) : 0.0f;
  } else {
    float largest = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) largest = fmaxf(largest, logit[i]);
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
      largest = fmaxf(largest, __shfl_xor_sync(kFull, largest, d));
    }
    // the largest logits count 1 each, also when they are infinite
    auto part = [&](float v) {
      return v == largest ? 1.0f : (v > -INFINITY ? expf(v - largest) : 0.0f);
    };
    score = id >= 0 ? part(mine) : 0.0f;
    if (renormalize == 0) {
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) {
        if (logit[i] > -INFINITY) sum += part(logit[i]);
      }
#pragma unroll
      for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
      score = id >= 0 ? score / sum : 0.0f;
    }
  }
  if (renormalize != 0) {
    float sum = score;
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
    score = sum > 0.0f ? score / sum : 0.0f;
  }
  if (lane < a.top_k) {
    a.ids[token * a.top_k + lane] = id;
    a.weights[token * a.top_k + lane] = score * a.scale;
  }
}

template <typename T, uint32_t V>
cudaError_t launch_route_topk(const RouteTopkArgs& a, bool sigmoid, uint32_t renormalize,
                              cudaStream_t stream) {
  const uint32_t per_cta = kRouteTopkThreads / 32;
  const uint32_t grid = static_cast<uint32_t>((a.tokens + per_cta - 1) / per_cta);
  if (sigmoid && a.bias != nullptr) {
    route_topk_kernel<T, V, true, true><<<grid, kRouteTopkThreads, 0, stream>>>(a, renormalize);
  } else if (sigmoid) {
    route_topk_kernel<T, V, true, false><<<grid, kRouteTopkThreads, 0, stream>>>(a, renormalize);
  } else {
    route_topk_kernel<T, V, false, false><<<grid, kRouteTopkThreads, 0, stream>>>(a, renormalize);
  }
  return cudaPeekAtLastError();
}

template <typename T>
cudaError_t dispatch_route_topk(const RouteTopkArgs& a, bool sigmoid, uint32_t renormalize,
                                cudaStream_t stream) {
  // as many keys per lane as the experts need
  if (a.experts <= 64) return launch_route_topk<T, 2>(a, sigmoid, renormalize, stream);
  if (a.experts <= 128) return launch_route_topk<T, 4>(a, sigmoid, renormalize, stream);
  if (a.experts <= 256) return launch_route_topk<T, 8>(a, sigmoid, renormalize, stream);
  return launch_route_topk<T, 32>(a, sigmoid, renormalize, stream);
}

template <typename T, uint32_t V>
cudaError_t preload_route_topk() {
  cudaError_t rc = preload_one(route_topk_kernel<T, V, false, false>);
  if (rc == cudaSuccess) rc = preload_one(route_topk_kernel<T, V, true, false>);
  if (rc == cudaSuccess) rc = preload_one(route_topk_kernel<T, V, true, true>);
  return rc;
}

template <typename T>
cudaError_t preload_route_topk_all() {
  cudaError_t rc = preload_route_topk<T, 2>();
  if (rc == cudaSuccess) rc = preload_route_topk<T, 4>();
  if (rc == cudaSuccess) rc = preload_route_topk<T, 8>();
  if (rc == cudaSuccess) rc = preload_route_topk<T, 32>();
  return rc;
}

}  // namespace

cudaError_t preload_router_kernels() {
  cudaError_t rc = preload_route_topk_all<float>();
  if (rc == cudaSuccess) rc = preload_route_topk_all<uint16_t>();
  return rc;
}

}  // namespace bmoe

extern "C" int bmoe_route_topk(const bmoe_route_topk_args* args) {
  if (args == nullptr) return BMOE_INVALID_ARGUMENT;
  const bmoe_route_topk_args& a = *args;
  const uint32_t elem = a.logits_type == BMOE_TYPE_BF16 ? 2u : 4u;
  if (a.logits_type != BMOE_TYPE_BF16 && a.logits_type != BMOE_TYPE_FP32) {
    return BMOE_UNSUPPORTED_DATA_TYPE;
  }
  if (a.experts == 0 || a.experts > BMOE_ROUTE_MAX_EXPERTS || a.top_k == 0 ||
      a.top_k > a.experts || a.top_k > BMOE_ROUTE_MAX_TOP_K ||
      a.scoring > BMOE_SCORE_SIGMOID ||
      (a.bias_dev != nullptr && a.scoring != BMOE_SCORE_SIGMOID) ||
      (a.row_stride != 0 && a.row_stride < a.experts && a.tokens > 1) ||
      a.tokens > 0x7fffffffull) {
    return BMOE_INVALID_ARGUMENT;
  }
  if (a.tokens == 0) return BMOE_OK;
  if (a.logits_dev == nullptr || a.expert_ids_dev == nullptr || a.weights_dev == nullptr ||
      bmoe::off_grid(a.logits_dev, elem) || bmoe::off_grid(a.expert_ids_dev, 8) ||
      bmoe::off_grid(a.weights_dev, 4) || bmoe::off_grid(a.bias_dev, 4)) {
    return BMOE_INVALID_ARGUMENT;
  }
  bmoe::RouteTopkArgs k;
  k.logits = a.logits_dev;
  k.bias = a.bias_dev;
  k.ids = a.expert_ids_dev;
  k.weights = a.weights_dev;
  k.tokens = a.tokens;
  k.row_stride = a.row_stride != 0 ? a.row_stride : a.experts;
  k.experts = a.experts;
  k.top_k = a.top_k;
  k.scale = a.scale;
  const bool sigmoid = a.scoring == BMOE_SCORE_SIGMOID;
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const cudaError_t rc =
      elem == 2 ? bmoe::dispatch_route_topk<uint16_t>(k, sigmoid, a.renormalize, stream)
                : bmoe::dispatch_route_topk<float>(k, sigmoid, a.renormalize, stream);
  return rc == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
