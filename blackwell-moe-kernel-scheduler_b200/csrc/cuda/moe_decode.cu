// A whole expert layer for a few tokens (a decode step), in two launches:
//   h[t, j] = silu(x[t] Wgate_e^T) * (x[t] Wup_e^T)      e = expert_ids[t, j]
//   out[t]  = bf16( sum_j weights[t, j] * (h[t, j] Wdown_e^T) )
//
// What bounds it is the stream of the chosen experts' weights from HBM: an expert has one
// to a few rows, so a weight is used a few times at most. Both kernels therefore read every
// weight once, straight into registers in the operand layout of mma.sync m16n8k16 with the
// WEIGHTS as the 16-row operand and up to 8 tokens as the columns: no shared-memory round
// trip and no 128-row tile that a handful of rows would leave empty (the tile of
// tcgen05.mma), and the tensor work stays far below the pipe's rate at these row counts.
//
// Operand layout. A lane (g = lane / 4, t = lane % 4) reads 16 bytes of rows g and g + 8 at
// byte 16 t of a 64-byte step, i.e. 8 BF16 or 16 INT8 values of k, and the 8 or 16 values of
// x (or h) at the same k for column g. The k order inside a step is permuted the same way on
// both sides, which a sum over k does not see.
#include <cuda_runtime.h>

#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"

namespace bmoe {
namespace {

constexpr uint32_t kFullWarp = 0xffffffffu;
constexpr uint32_t kMaxTokens = BMOE_MOE_DECODE_MAX_TOKENS;
constexpr uint32_t kStepBytes = 64;   // bytes of a weight row per step
constexpr uint32_t kUnroll = 4;       // steps whose weights are in flight together ("block")

struct DecodeArgs {
  const uint16_t* x;        // [tokens, hidden]
  const uint8_t* w1;        // [experts, 2 * inter, hidden]
  const uint8_t* w2;        // [experts, hidden, inter]
  const float* s1;          // INT8: [experts, 2 * inter]
  const float* s2;          // INT8: [experts, hidden]
  const int64_t* ids;       // [tokens, top_k]
  const float* coef;        // [tokens, top_k]
  uint16_t* out;            // [tokens, hidden]
  uint16_t* h_hi;           // [tokens * top_k, inter], upper and
  uint16_t* h_lo;           // lower half of weights * h
  uint32_t tokens, top_k, experts, hidden, inter;
  uint32_t by_expert;       // grid.y of the first kernel: expert ids, or assignments
};

// ------------------------------------------------------------- fragments --

// Weights are read once: keep them out of L1, where the activations live.
__device__ __forceinline__ uint4 load_weights(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two signed bytes of `word` (selector 0x4140: bytes 0, 1; 0x4342: bytes 2, 3) -> BF16 pair,
// exact. With v = 128 + (b & 127) as the bits 0x4300 | (b & 0x7f), and 128 or 256 as the bits
// 0x4300 | (b & 0x80), the signed value is their difference.
__device__ __forceinline__ uint32_t int8_pair(uint32_t word, uint32_t selector) {
  const uint32_t both = __byte_perm(word, 0x43434343u, selector);
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(both & 0xff7fff7fu), "r"(both & 0xff80ff80u));
  return r;
}

// One step of one 16-row tile against one 8-column tile: 32 (BF16) or 64 (INT8) of k.
// lo, hi: this lane's 16 bytes of rows g and g + 8; b: its 8 or 16 activations.
template <bool INT8>
struct Step {
  static constexpr uint32_t kActs = INT8 ? 2 : 1;   // 16-byte loads of activations per lane
  uint4 lo, hi;

  __device__ __forceinline__ void multiply(float (&acc)[4], const uint4 (&b)[kActs]) const {
    if constexpr (!INT8) {
      mma_bf16(acc, lo.x, hi.x, lo.y, hi.y, b[0].x, b[0].y);
      mma_bf16(acc, lo.z, hi.z, lo.w, hi.w, b[0].z, b[0].w);
    } else {
      mma_bf16(acc, int8_pair(lo.x, 0x4140), int8_pair(hi.x, 0x4140), int8_pair(lo.x, 0x4342),
               int8_pair(hi.x, 0x4342), b[0].x, b[0].y);
      mma_bf16(acc, int8_pair(lo.y, 0x4140), int8_pair(hi.y, 0x4140), int8_pair(lo.y, 0x4342),
               int8_pair(hi.y, 0x4342), b[0].z, b[0].w);
      mma_bf16(acc, int8_pair(lo.z, 0x4140), int8_pair(hi.z, 0x4140), int8_pair(lo.z, 0x4342),
               int8_pair(hi.z, 0x4342), b[1].x, b[1].y);
      mma_bf16(acc, int8_pair(lo.w, 0x4140), int8_pair(hi.w, 0x4140), int8_pair(lo.w, 0x4342),
               int8_pair(hi.w, 0x4342), b[1].z, b[1].w);
    }
  }
};

// This lane's activations of one step: k = step * K + lane's share, zeros beyond `k_total`
// (a multiple of the 8 or 16 values of a lane) and for a column without a row. Plain loads:
// h is written by the first kernel while the second is already resident, so a load through the
// read-only path, which the compiler may move above the wait between them, would be wrong.
template <bool INT8>
__device__ __forceinline__ void load_acts(uint4 (&b)[Step<INT8>::kActs], const uint16_t* row,
                                          uint32_t k, uint32_t k_total) {
  const bool live = row != nullptr && k < k_total;
#pragma unroll
  for (uint32_t i = 0; i < Step<INT8>::kActs; ++i) {
    b[i] = live ? *reinterpret_cast<const uint4*>(row + k + 8 * i) : zero4();
  }
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

__device__ __forceinline__ uint16_t to_bf16(float v) {
  uint16_t b;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(v));
  return b;
}

__device__ __forceinline__ float from_bf16(uint16_t v) {
  return __uint_as_float(static_cast<uint32_t>(v) << 16);
}

// --------------------------------------------------- gate and up products --

// One CTA computes 16 * WR channels of one expert for all of its tokens: WR warps side by side
// (16 gate and 16 up rows each), times WK warps that share the k range block by block.
template <bool INT8, uint32_t NT, uint32_t WR, uint32_t WK>
__global__ void __launch_bounds__(32 * WR * WK) decode_up_kernel(DecodeArgs a) {
  using S = Step<INT8>;
  constexpr uint32_t kStep = INT8 ? 64 : 32;         // k values per step
  constexpr uint32_t kLane = INT8 ? 16 : 8;          // of which a lane holds these
  extern __shared__ float4 partial[];                // [WK][WR][2][NT][32]
  __shared__ uint16_t list_row[kMaxTokens];          // assignment of column p
  __shared__ uint8_t list_token[kMaxTokens];
  __shared__ float list_coef[kMaxTokens];
  __shared__ uint32_t list_count, list_expert;

  // let the second kernel's CTAs take their places as this grid's last CTAs run
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {
    // Tokens of this CTA's expert. By assignment: the expert's first one does the work.
    const int64_t e = a.by_expert != 0 ? static_cast<int64_t>(blockIdx.y) : a.ids[blockIdx.y];
    uint32_t count = 0, owner = 0;
    if (e >= 0 && e < a.experts) {
      for (uint32_t t0 = 0; t0 < a.tokens; t0 += 32) {
        const uint32_t t = t0 + lane;
        int first = -1;
        float coef = 0.0f;
        if (t < a.tokens) {
          for (uint32_t j = 0; j < a.top_k; ++j) {
            if (a.ids[t * a.top_k + j] == e) {   // twice: the sum of both weights
              if (first < 0) first = static_cast<int>(t * a.top_k + j);
              coef += a.coef[t * a.top_k + j];
            }
          }
        }
        const uint32_t mask = __ballot_sync(kFullWarp, first >= 0);
        if (count == 0 && mask != 0) {
          owner = static_cast<uint32_t>(__shfl_sync(kFullWarp, first, __ffs(mask) - 1));
        }
        if (first >= 0) {
          const uint32_t p = count + __popc(mask & ((1u << lane) - 1));
          list_row[p] = static_cast<uint16_t>(first);
          list_token[p] = static_cast<uint8_t>(t);
          list_coef[p] = coef;
        }
        count += __popc(mask);
      }
      if (a.by_expert == 0 && owner != blockIdx.y) count = 0;
    }
    if (lane == 0) {
      list_count = count;
      list_expert = static_cast<uint32_t>(e);
    }
  }
  __syncthreads();
  const uint32_t count = list_count;
  if (count == 0) return;
  const uint32_t expert = list_expert;
  const uint32_t tiles = (count + 7) / 8;

  const uint32_t g = lane >> 2, t = lane & 3;
  const uint32_t wr = warp % WR, wk = warp / WR;
  const uint32_t row0 = (blockIdx.x * WR + wr) * 16;
  const size_t row_bytes = static_cast<size_t>(a.hidden) * (INT8 ? 1 : 2);
  // rows beyond inter read the last one and are not stored
  const uint32_t r_lo = min(row0 + g, a.inter - 1), r_hi = min(row0 + g + 8, a.inter - 1);
  const size_t first_row = static_cast<size_t>(expert) * 2 * a.inter;
  const uint8_t* const gate_lo = a.w1 + (first_row + r_lo) * row_bytes + 16 * t;
  const uint8_t* const gate_hi = a.w1 + (first_row + r_hi) * row_bytes + 16 * t;
  const size_t up_bytes = static_cast<size_t>(a.inter) * row_bytes;
  const uint16_t* x_row[NT];
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n) {
    const uint32_t p = n * 8 + g;
    x_row[n] = p < count ? a.x + static_cast<size_t>(list_token[p]) * a.hidden : nullptr;
  }

  float acc[2][NT][4];
#pragma unroll
  for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
    }
  }
  const uint32_t steps = (a.hidden + kStep - 1) / kStep;
  for (uint32_t s0 = wk * kUnroll; s0 < steps; s0 += WK * kUnroll) {
    S w[kUnroll][2];
#pragma unroll
    for (uint32_t u = 0; u < kUnroll; ++u) {
      const uint32_t k = (s0 + u) * kStep + t * kLane;
      const size_t at = static_cast<size_t>(s0 + u) * kStepBytes;
      const bool live = k < a.hidden;
      w[u][0].lo = live ? load_weights(gate_lo + at) : zero4();
      w[u][0].hi = live ? load_weights(gate_hi + at) : zero4();
      w[u][1].lo = live ? load_weights(gate_lo + up_bytes + at) : zero4();
      w[u][1].hi = live ? load_weights(gate_hi + up_bytes + at) : zero4();
    }
#pragma unroll
    for (uint32_t u = 0; u < kUnroll; ++u) {
      const uint32_t k = (s0 + u) * kStep + t * kLane;
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n) {
        if (n == 0 || n < tiles) {
          uint4 b[S::kActs];
          load_acts<INT8>(b, x_row[n], k, a.hidden);
          w[u][0].multiply(acc[0][n], b);
          w[u][1].multiply(acc[1][n], b);
        }
      }
    }
  }

  // Join the k shares in a fixed order and write weights * silu(gate) * up.
  auto slot = [&](uint32_t k_share, uint32_t row_warp, uint32_t m, uint32_t n) {
    return (((k_share * WR + row_warp) * 2 + m) * NT + n) * 32;
  };
#pragma unroll
  for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
      partial[slot(wk, wr, m, n) + lane] =
          make_float4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
    }
  }
  __syncthreads();
  const float* const sums = reinterpret_cast<const float*>(partial);
  for (uint32_t i = threadIdx.x; i < WR * tiles * 128; i += 32 * WR * WK) {
    // element i: channel c of row group q, column p; rows run fastest
    const uint32_t c = i % 16, p = (i / 16) % (tiles * 8), q = i / (16 * tiles * 8);
    const uint32_t channel = (blockIdx.x * WR + q) * 16 + c;
    if (p >= count || channel >= a.inter) continue;
    // accumulator layout: lane (c % 8) * 4 + (p % 8) / 2, register 2 * (c / 8) + p % 2
    const uint32_t in_tile = ((c % 8) * 4 + (p % 8) / 2) * 4 + 2 * (c / 8) + p % 2;
    float gate = 0.0f, up = 0.0f;
#pragma unroll
    for (uint32_t s = 0; s < WK; ++s) {
      gate += sums[slot(s, q, 0, p / 8) * 4 + in_tile];
      up += sums[slot(s, q, 1, p / 8) * 4 + in_tile];
    }
    if constexpr (INT8) {
      const float* const scale = a.s1 + first_row + channel;
      gate *= scale[0];
      up *= scale[a.inter];
    }
    const float v = silu(gate) * up * list_coef[p];
    // 16 significant bits in two BF16 numbers; an infinity has no remainder
    const uint16_t hi = to_bf16(v);
    const float rest = v - from_bf16(hi);
    const size_t at = static_cast<size_t>(list_row[p]) * a.inter + channel;
    a.h_hi[at] = hi;
    a.h_lo[at] = to_bf16(isfinite(v) ? rest : 0.0f);
  }
}

// ------------------------------------------------------------ down product --

// A cluster computes 16 * MT * WR output channels for all tokens: WR warps side by side (MT
// tiles of 16 rows each), and the chosen experts' k ranges, laid end to end, shared among
// the cluster's CTAs x WK warps. Every warp sums into its own shared-memory tile [tokens][rows];
// the tiles are joined in a fixed order, across the cluster through distributed shared memory.
template <bool INT8, uint32_t NT, uint32_t MT, uint32_t WR, uint32_t WK>
__global__ void __launch_bounds__(32 * WR * WK) decode_down_kernel(DecodeArgs a) {
  using S = Step<INT8>;
  constexpr uint32_t kStep = INT8 ? 64 : 32;
  constexpr uint32_t kLane = INT8 ? 16 : 8;
  constexpr uint32_t kRows = 16 * MT;                // rows of a warp
  constexpr uint32_t kPitch = kRows + 8;             // floats between tokens of a tile
  constexpr uint32_t kWarps = WR * WK;
  extern __shared__ float4 dynamic[];
  __shared__ uint32_t active_bits[BMOE_MOE_DECODE_MAX_EXPERTS / 32];
  __shared__ uint16_t active[BMOE_MOE_DECODE_MAX_EXPERTS];
  __shared__ uint32_t active_count;
  __shared__ uint16_t list_row[kWarps][kMaxTokens];
  __shared__ uint8_t list_token[kWarps][kMaxTokens];
  float* const tile_all = reinterpret_cast<float*>(dynamic);      // [kWarps][tokens][kPitch]
  int16_t* const ids = reinterpret_cast<int16_t*>(tile_all + kWarps * a.tokens * kPitch);

  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t assignments = a.tokens * a.top_k;

  // The chosen experts in ascending order.
  if (threadIdx.x < BMOE_MOE_DECODE_MAX_EXPERTS / 32) active_bits[threadIdx.x] = 0;
  for (uint32_t i = threadIdx.x; i < kWarps * a.tokens * kPitch; i += 32 * kWarps) {
    tile_all[i] = 0.0f;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < assignments; i += 32 * kWarps) {
    const int64_t e = a.ids[i];
    const bool live = e >= 0 && e < a.experts;
    ids[i] = live ? static_cast<int16_t>(e) : static_cast<int16_t>(-1);
    if (live) atomicOr(&active_bits[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t bits = active_bits[lane];
    uint32_t before = __popc(bits);
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(kFullWarp, before, d);
      if (lane >= d) before += v;
    }
    if (lane == 31) active_count = before;
    before -= __popc(bits);
    while (bits != 0) {
      active[before++] = static_cast<uint16_t>(lane * 32 + __ffs(bits) - 1);
      bits &= bits - 1;
    }
  }
  __syncthreads();

  uint32_t cta_rank, cta_count;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta_rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cta_count));
  const uint32_t g = lane >> 2, t = lane & 3;
  const uint32_t wr = warp % WR, wk = warp / WR;
  const uint32_t group = blockIdx.x / cta_count;                  // of 16 * MT * WR rows
  const uint32_t row0 = (group * WR + wr) * kRows;
  const size_t row_bytes = static_cast<size_t>(a.inter) * (INT8 ? 1 : 2);
  float* const tile = tile_all + warp * a.tokens * kPitch;

  // This warp's share of the experts' k blocks, laid end to end.
  const uint32_t steps = (a.inter + kStep - 1) / kStep;
  const uint32_t blocks = (steps + kUnroll - 1) / kUnroll;        // of one expert
  const uint32_t total = active_count * blocks;
  const uint32_t workers = cta_count * WK, worker = cta_rank * WK + wk;
  const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(total) * worker / workers);
  const uint32_t end =
      static_cast<uint32_t>(static_cast<uint64_t>(total) * (worker + 1) / workers);

  uint32_t row_of[MT][2];
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m) {
    row_of[m][0] = min(row0 + m * 16 + g, a.hidden - 1);
    row_of[m][1] = min(row0 + m * 16 + g + 8, a.hidden - 1);
  }

  bool waited = false;
  uint32_t block = begin;
  while (block < end) {
    const uint32_t slot = block / blocks;
    const uint32_t expert = active[slot];
    const uint32_t stop = min(end, (slot + 1) * blocks);
    // tokens of this expert, in ascending order (the first of two equal ids counts)
    uint32_t count = 0;
    __syncwarp();
    for (uint32_t t0 = 0; t0 < a.tokens; t0 += 32) {
      const uint32_t token = t0 + lane;
      int first = -1;
      if (token < a.tokens) {
        for (uint32_t j = 0; j < a.top_k; ++j) {
          if (first < 0 && ids[token * a.top_k + j] == static_cast<int>(expert)) {
            first = static_cast<int>(token * a.top_k + j);
          }
        }
      }
      const uint32_t mask = __ballot_sync(kFullWarp, first >= 0);
      if (first >= 0) {
        const uint32_t p = count + __popc(mask & ((1u << lane) - 1));
        list_row[warp][p] = static_cast<uint16_t>(first);
        list_token[warp][p] = static_cast<uint8_t>(token);
      }
      count += __popc(mask);
    }
    __syncwarp();
    const uint32_t tiles = (count + 7) / 8;
    size_t h_at[NT];
    bool h_live[NT];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
      const uint32_t p = n * 8 + g;
      h_live[n] = p < count;
      h_at[n] = h_live[n] ? static_cast<size_t>(list_row[warp][p]) * a.inter : 0;
    }
    const uint8_t* w_at[MT][2];
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m) {
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        w_at[m][i] = a.w2 + (static_cast<size_t>(expert) * a.hidden + row_of[m][i]) * row_bytes +
                     16 * t;
      }
    }
    float acc[MT][NT][4];
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m) {
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
      }
    }
    for (; block < stop; ++block) {
      const uint32_t s0 = (block - slot * blocks) * kUnroll;
      S w[kUnroll][MT];
#pragma unroll
      for (uint32_t u = 0; u < kUnroll; ++u) {
        const uint32_t k = (s0 + u) * kStep + t * kLane;
        const size_t at = static_cast<size_t>(s0 + u) * kStepBytes;
#pragma unroll
        for (uint32_t m = 0; m < MT; ++m) {
          w[u][m].lo = k < a.inter ? load_weights(w_at[m][0] + at) : zero4();
          w[u][m].hi = k < a.inter ? load_weights(w_at[m][1] + at) : zero4();
        }
      }
      if (!waited) {
        // h comes from the first kernel; the weights above do not
        asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
      }
#pragma unroll
      for (uint32_t u = 0; u < kUnroll; ++u) {
        const uint32_t k = (s0 + u) * kStep + t * kLane;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) {
          if (n == 0 || n < tiles) {
            uint4 b[S::kActs], rest[S::kActs];
            load_acts<INT8>(b, h_live[n] ? a.h_hi + h_at[n] : nullptr, k, a.inter);
            load_acts<INT8>(rest, h_live[n] ? a.h_lo + h_at[n] : nullptr, k, a.inter);
#pragma unroll
            for (uint32_t m = 0; m < MT; ++m) {
              w[u][m].multiply(acc[m][n], b);
              w[u][m].multiply(acc[m][n], rest);
            }
          }
        }
      }
    }
    // into the warp's tile: columns p of this expert are tokens list_token[p]
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m) {
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n) {
        if (n == 0 || n < tiles) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t p = n * 8 + 2 * t + (i & 1), half = i >> 1;
            if (p < count) {
              float v = acc[m][n][i];
              if constexpr (INT8) {
                v *= a.s2[static_cast<size_t>(expert) * a.hidden + row_of[m][half]];
              }
              tile[list_token[warp][p] * kPitch + m * 16 + g + 8 * half] += v;
            }
          }
        }
      }
    }
  }

  // A warp without a share waits as well: this grid must not end before the first one.
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");

  // Join the WK warps of this CTA, then the cluster's CTAs, each in ascending order.
  __syncthreads();
  constexpr uint32_t kCtaRows = kRows * WR;
  const uint32_t cells = a.tokens * kCtaRows;
  if constexpr (WK > 1) {
    for (uint32_t i = threadIdx.x; i < cells; i += 32 * kWarps) {
      const uint32_t token = i / kCtaRows, row = i % kCtaRows;
      const uint32_t at = token * kPitch + row % kRows;
      float sum = 0.0f;
#pragma unroll
      for (uint32_t s = 0; s < WK; ++s) {
        sum += tile_all[(s * WR + row / kRows) * a.tokens * kPitch + at];
      }
      tile_all[row / kRows * a.tokens * kPitch + at] = sum;
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t tile_smem = static_cast<uint32_t>(__cvta_generic_to_shared(tile_all));
  for (uint32_t i = cta_rank * 32 * kWarps + threadIdx.x; i < cells;
       i += cta_count * 32 * kWarps) {
    const uint32_t token = i / kCtaRows, row = i % kCtaRows;
    const uint32_t channel = group * kCtaRows + row;
    const uint32_t at =
        tile_smem + 4 * ((row / kRows * a.tokens + token) * kPitch + row % kRows);
    float sum = 0.0f;
    for (uint32_t c = 0; c < cta_count; ++c) {
      uint32_t remote;
      float v;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(c));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
      sum += v;
    }
    if (channel < a.hidden) a.out[static_cast<size_t>(token) * a.hidden + channel] = to_bf16(sum);
  }
  // nobody leaves while a neighbour still reads its tile
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------ launch --

template <bool INT8, uint32_t NT, uint32_t WR, uint32_t WK>
constexpr uint32_t up_smem() {
  return WK * WR * 2 * NT * 32 * sizeof(float4);
}

template <uint32_t MT, uint32_t WR, uint32_t WK>
uint32_t down_smem(uint32_t tokens, uint32_t top_k) {
  return WR * WK * tokens * (16 * MT + 8) * 4 + (tokens * top_k * 2 + 15) / 16 * 16;
}

// Opt-in shared memory is an attribute of a function on a device; setting it is cheap and
// the same value every time, so every launch does it and nothing is cached.
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, uint32_t bytes) {
  return bytes <= 48u * 1024u - 8192u
             ? cudaSuccess
             : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(bytes));
}

template <bool INT8, uint32_t NT, uint32_t MT, uint32_t WR, uint32_t WK>
cudaError_t launch_decode(const DecodeArgs& a, cudaStream_t stream) {
  const uint32_t sms = device_sm_count();
  {
    constexpr uint32_t smem = up_smem<INT8, NT, WR, WK>();
    const auto kernel = decode_up_kernel<INT8, NT, WR, WK>;
    cudaError_t rc = allow_smem(kernel, smem);
    if (rc != cudaSuccess) return rc;
    const uint32_t slots = a.by_expert != 0 ? a.experts : a.tokens * a.top_k;
    kernel<<<dim3((a.inter + 16 * WR - 1) / (16 * WR), slots), 32 * WR * WK, smem, stream>>>(a);
    rc = cudaPeekAtLastError();
    if (rc != cudaSuccess) return rc;
  }
  const uint32_t smem = down_smem<MT, WR, WK>(a.tokens, a.top_k);
  const auto kernel = decode_down_kernel<INT8, NT, MT, WR, WK>;
  cudaError_t rc = allow_smem(kernel, smem);
  if (rc != cudaSuccess) return rc;
  // enough CTAs for two per SM, in clusters of at most 8
  const uint32_t groups = (a.hidden + 16 * MT * WR - 1) / (16 * MT * WR);
  uint32_t cluster = 1;
  while (cluster < 8 && groups * cluster < 2 * sms) cluster *= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(groups * cluster);
  config.blockDim = dim3(32 * WR * WK);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = cluster;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  rc = cudaLaunchKernelEx(&config, kernel, a);
  return rc != cudaSuccess ? rc : cudaPeekAtLastError();
}

template <bool INT8>
cudaError_t dispatch_decode(const DecodeArgs& a, cudaStream_t stream) {
  if (a.tokens <= 8) return launch_decode<INT8, 1, 2, 1, 8>(a, stream);
  if (a.tokens <= 32) return launch_decode<INT8, 4, 2, 2, 4>(a, stream);
  return launch_decode<INT8, 8, 2, 4, 2>(a, stream);
}

template <bool INT8, uint32_t NT, uint32_t MT, uint32_t WR, uint32_t WK>
cudaError_t preload_decode() {
  const cudaError_t rc = preload_one(decode_up_kernel<INT8, NT, WR, WK>);
  return rc == cudaSuccess ? preload_one(decode_down_kernel<INT8, NT, MT, WR, WK>) : rc;
}

template <bool INT8>
cudaError_t preload_decode_type() {
  cudaError_t rc = preload_decode<INT8, 1, 2, 1, 8>();
  if (rc == cudaSuccess) rc = preload_decode<INT8, 4, 2, 2, 4>();
  if (rc == cudaSuccess) rc = preload_decode<INT8, 8, 2, 4, 2>();
  return rc;
}

bool unaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// Bytes of one BF16 plane of h.
uint64_t plane_bytes(uint32_t tokens, uint32_t top_k, uint32_t inter) {
  return (static_cast<uint64_t>(tokens) * top_k * inter * 2 + 255) / 256 * 256;
}

}  // namespace

cudaError_t preload_decode_kernels() {
  const cudaError_t rc = preload_decode_type<false>();
  return rc == cudaSuccess ? preload_decode_type<true>() : rc;
}

}  // namespace bmoe

extern "C" uint64_t bmoe_moe_decode_workspace(uint32_t tokens, uint32_t top_k, uint32_t inter) {
  return 2 * bmoe::plane_bytes(tokens, top_k, inter);
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
      a.inter == 0 || a.inter % step != 0 || a.hidden > BMOE_MOE_DECODE_MAX_WIDTH ||
      a.inter > BMOE_MOE_DECODE_MAX_WIDTH) {
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
  k.w1 = static_cast<const uint8_t*>(a.w_gate_up_dev);
  k.w2 = static_cast<const uint8_t*>(a.w_down_dev);
  k.s1 = a.gate_up_scale_dev;
  k.s2 = a.down_scale_dev;
  k.ids = a.expert_ids_dev;
  k.coef = a.weights_dev;
  k.out = static_cast<uint16_t*>(a.out_dev);
  k.h_hi = static_cast<uint16_t*>(a.workspace_dev);
  k.h_lo = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(a.workspace_dev) +
                                       bmoe::plane_bytes(a.tokens, a.top_k, a.inter));
  k.tokens = a.tokens;
  k.top_k = a.top_k;
  k.experts = a.experts;
  k.hidden = a.hidden;
  k.inter = a.inter;
  k.by_expert = a.experts <= a.tokens * a.top_k ? 1u : 0u;
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const cudaError_t rc = int8 ? bmoe::dispatch_decode<true>(k, stream)
                              : bmoe::dispatch_decode<false>(k, stream);
  return rc == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
