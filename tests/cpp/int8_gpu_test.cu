// Int8GroupedGemmPlan through the C++ headers: known answers with exact sums, the refusals, and
// the C entry points of the layer operators from the same program.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "blackwell_moe/kernels/grouped_gemm.cuh"
#include "bmoe_b200.h"

namespace {

int failures = 0;

void expect(bool ok, const char* what) {
  std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
  if (!ok) ++failures;
}

template <typename T>
T* to_device(const std::vector<T>& host) {
  T* p = nullptr;
  cudaMalloc(&p, host.size() * sizeof(T));
  cudaMemcpy(p, host.data(), host.size() * sizeof(T), cudaMemcpyHostToDevice);
  return p;
}

float bf16_value(uint16_t bits) {
  const uint32_t wide = static_cast<uint32_t>(bits) << 16;
  float f;
  static_assert(sizeof(f) == sizeof(wide), "float");
  __builtin_memcpy(&f, &wide, 4);
  return f;
}

}  // namespace

int main() {
  using namespace blackwell_moe;
  const std::uint32_t experts = 3, n = 72, k = 48;
  const std::vector<std::uint32_t> counts = {5, 0, 130};

  std::vector<std::int8_t*> a(experts, nullptr), b(experts, nullptr);
  std::vector<std::uint16_t*> d(experts, nullptr);
  std::vector<float*> row(experts, nullptr), col(experts, nullptr);
  std::vector<std::vector<std::int8_t>> ha(experts), hb(experts);
  for (std::uint32_t e = 0; e < experts; ++e) {
    if (counts[e] == 0) continue;
    ha[e].resize(counts[e] * k);
    hb[e].resize(n * k);
    for (std::size_t i = 0; i < ha[e].size(); ++i) ha[e][i] = static_cast<std::int8_t>(i * 37 % 255 - 127);
    for (std::size_t i = 0; i < hb[e].size(); ++i) hb[e][i] = static_cast<std::int8_t>(i * 91 % 256 - 128);
    a[e] = to_device(ha[e]);
    b[e] = to_device(hb[e]);
    row[e] = to_device(std::vector<float>(counts[e], 0.5f));
    std::vector<float> c(n);
    for (std::uint32_t j = 0; j < n; ++j) c[j] = j % 2 == 0 ? 0.25f : 4.0f;
    col[e] = to_device(c);
    cudaMalloc(&d[e], counts[e] * n * 2);
  }
  GroupedGemmArguments args;
  args.a = reinterpret_cast<const void* const*>(a.data());
  args.b = reinterpret_cast<const void* const*>(b.data());
  args.d = reinterpret_cast<void* const*>(d.data());
  args.tokens_per_expert = counts.data();
  args.experts = experts;
  args.n = n;
  args.k = k;
  args.data_type = DataType::kInt8;

  Int8GroupedGemmPlan plan;
  expect(plan.initialize(args) == KernelStatus::kInvalidArgument, "scales are required");
  args.row_scale = row.data();
  args.col_scale = col.data();
  GroupedGemmArguments other = args;
  other.data_type = DataType::kBf16;
  expect(plan.initialize(other) == KernelStatus::kUnsupportedDataType, "INT8 plan takes INT8 only");
  Bf16GroupedGemmPlan bf16_plan;
  expect(bf16_plan.initialize(args) == KernelStatus::kUnsupportedDataType, "BF16 plan refuses INT8");
  Fp8E4m3GroupedGemmPlan fp8_plan;
  expect(fp8_plan.initialize(args) == KernelStatus::kUnsupportedDataType, "FP8 plan refuses INT8");
  expect(plan.initialize(args) == KernelStatus::kSuccess, "initialize");
  expect(plan.run() == KernelStatus::kSuccess, "run");
  expect(plan.poll() == KernelStatus::kSuccess, "poll");
  expect(plan.stats().active_experts == 2, "two active experts");

  // sums are exact and the scales powers of two: one BF16 rounding, at most half a step (2^-8)
  double worst = 0.0;
  for (std::uint32_t e = 0; e < experts; ++e) {
    if (counts[e] == 0) continue;
    std::vector<std::uint16_t> got(counts[e] * n);
    cudaMemcpy(got.data(), d[e], got.size() * 2, cudaMemcpyDeviceToHost);
    for (std::uint32_t m = 0; m < counts[e]; ++m) {
      for (std::uint32_t j = 0; j < n; ++j) {
        long sum = 0;
        for (std::uint32_t i = 0; i < k; ++i) sum += long(ha[e][m * k + i]) * hb[e][j * k + i];
        const double want = sum * 0.5 * (j % 2 == 0 ? 0.25 : 4.0);
        const double off = std::fabs(bf16_value(got[m * n + j]) - want);
        worst = std::fmax(worst, want == 0.0 ? off : off / std::fabs(want));
      }
    }
  }
  expect(worst <= 1.0 / 256.0, "known answers within half a BF16 step");

  // router and quantiser through the C interface
  std::vector<float> logits = {1.f, 3.f, 2.f, 3.f};
  float* logits_dev = to_device(logits);
  std::int64_t* ids_dev = nullptr;
  float* weights_dev = nullptr;
  cudaMalloc(&ids_dev, 2 * sizeof(std::int64_t));
  cudaMalloc(&weights_dev, 2 * sizeof(float));
  bmoe_route_topk_args route = {};
  route.logits_dev = logits_dev;
  route.expert_ids_dev = ids_dev;
  route.weights_dev = weights_dev;
  route.tokens = 1;
  route.experts = 4;
  route.top_k = 2;
  route.logits_type = BMOE_TYPE_FP32;
  route.renormalize = 1;
  route.scale = 1.0f;
  expect(bmoe_route_topk(&route) == BMOE_OK, "bmoe_route_topk");
  std::int64_t ids[2] = {};
  float weights[2] = {};
  cudaMemcpy(ids, ids_dev, sizeof(ids), cudaMemcpyDeviceToHost);
  cudaMemcpy(weights, weights_dev, sizeof(weights), cudaMemcpyDeviceToHost);
  expect(ids[0] == 1 && ids[1] == 3 && weights[0] == 0.5f && weights[1] == 0.5f,
         "ties go to the lower id and share the weight");
  expect(cudaDeviceSynchronize() == cudaSuccess, "device");
  std::printf("%s\n", failures == 0 ? "all passed" : "failed");
  return failures == 0 ? 0 : 1;
}
