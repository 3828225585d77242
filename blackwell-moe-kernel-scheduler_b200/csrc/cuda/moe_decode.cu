// A whole expert layer for a few tokens (a decode step), in two launches or four:
//   h[t, j] = silu(x[t] Wgate_e^T) * (x[t] Wup_e^T)      e = expert_ids[t, j]
//   out[t]  = bf16( sum_j weights[t, j] * (h[t, j] Wdown_e^T) )
//
// What bounds it is the stream of the chosen experts' weights from HBM: an expert has one to a
// few tokens, so a weight is used a few times at most. Both products read every weight once,
// 128 rows at a time through a ring of TMA boxes, with the WEIGHTS as the 128-row operand of
// tcgen05.mma and the expert's tokens as its 16 to 192 columns: the rows are full however
// few tokens there are, and the ring (about 100 KB per CTA, two CTAs per SM where they fit)
// keeps enough bytes in flight to hold HBM busy while CTAs come and go.
//   warp 0     TMA producer
//   warp 1     MMA issuer (one elected lane), Tensor Memory
//   warps 4-7  epilogue
// BF16 weights: h keeps 16 significant bits as two BF16 numbers whose products are added: the
// upper and the lower halves of the tokens are separate columns of the same MMA. What that leaves
// out (2.5e-6 of the result in norm) is about what the MMA's own FP32 sums do (2.1e-6 over 2048
// products, 4.4e-6 over 4096, 1.6e-5 over 14336 in one accumulator; a BF16 result's half
// step is 3.9e-3): a third BF16 number would cost half as many activation bytes again for less
// than that.
// INT8 weights are multiplied in one of two ways (use_digits has the rule and what it measured):
//   as they are, against activations written as fixed-point numbers of three signed bytes. The
//   digits of a token are three columns of the same MMA, its sums are exact 32-bit integers.
//   Two more launches make the digits of x and, once the largest value of its rows is known, of h.
//   converted to BF16 between shared and Tensor Memory (a signed byte is a BF16 value, so this is
//   exact) by warps 4-11, as the MMA's A operand. The first kernel's warps 4-7 are its epilogue
//   afterwards, the second has warps 12-15. It needs no more launches, but integer instructions
//   for every weight: 50 % of the ALU at 70 % of HBM's rate, and the power to run them (with 64
//   tokens and 1.4 GB of weights, 285 us in a short run and 322 at the 1000 W limit).
// Few tiles are split along k over the CTAs of a cluster, joined in a fixed order through
// distributed shared memory. The only atomics are maxima of rows of h: the same bits on every run.
//
// Measured on B200 (us of device time in a CUDA graph, inputs past L2; share of the 6.55 TB/s a
// copy reaches): hidden 4096, inter 14336, two of 8 experts, T=1: 112 BF16 (96 %), 65 INT8 (83 %);
// all 8 hit, T=16: 444-456 BF16 (94-97 %), 226 INT8 (95 %), T=64: 448 BF16 (96 %), 254 INT8 (85 %).
// 128 experts of 2048 x 768, top-8: T=1 22.6 BF16 (51 %), T=32 143 (90 %). INT8 that is converted,
// 64 tokens on one expert of (4096, 14336): 65 (41 %), on each of two: 111 (48 %). (Of one GPU;
// others of the same kind, and long runs at the 1000 W limit, take up to 8 % longer.) hidden 512, inter 1024, T=1: 9.7 (latency
// of two dependent launches). Fragments loaded straight into registers for mma.sync, the first
// version, took 178 us for T=1, 848 for T=32 and 1227 for T=64 in INT8.
// One grid that fills the GPU once with an equal share of blocks per CTA was tried for the
// first kernel and is 0-25 % slower: SMs do not get equal shares of HBM, and a grid of more
// CTAs than places evens that out.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "bmoe_b200.h"
#include "preload.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace bmoe {
namespace {

constexpr uint32_t kFullWarp = 0xffffffffu;
constexpr uint32_t kMaxTokens = BMOE_MOE_DECODE_MAX_TOKENS;
constexpr uint32_t kRows = 128;                  // weight rows of a tile
constexpr uint32_t kABytes = kRows * 128;        // one k-block of weights: 128 bytes of a row
constexpr uint32_t kGroup = 8;                   // tokens of one activation box
constexpr uint32_t kMostQuads = 6;               // gathers of four tokens per piece
constexpr uint32_t kTwoPerSm = 110u * 1024u;     // dynamic shared memory of a CTA that shares
constexpr uint32_t kOnePerSm = 222u * 1024u;     // its SM, and of one that does not
constexpr uint32_t kMaxStages = 12;
constexpr uint32_t kTmemA = 128;                 // columns of the INT8 A operand, in front
constexpr uint32_t kDigits = 3;                  // signed bytes of a fixed-point activation
constexpr uint64_t kWaitBudgetNs = 1000000000ull;

// BF16 weights; INT8 weights turned into BF16 on their way to the MMA; or INT8 weights as they
// are, against activations as fixed-point numbers of three signed bytes.
enum class Kind : uint32_t { kBf16, kConvert, kDigits };

struct DecodeArgs {
  const float* s1;          // INT8: [experts, 2 * inter]
  const float* s2;          // INT8: [experts, hidden]
  const int64_t* ids;       // [tokens, top_k]
  const float* coef;        // [tokens, top_k]
  uint16_t* out;            // [tokens, hidden]
  uint16_t* h;              // [2][tokens * top_k, inter]: upper and lower half of weights * h
  const uint16_t* x;        // Kind::kDigits: [tokens, hidden]
  float* h32;               // weights * h, [tokens * top_k, inter]
  uint8_t* digits;          // [3][tokens, hidden] of x, later [3][tokens * top_k, inter] of h
  uint32_t* x_most;         // and the bits of the largest magnitude of every row of x
  uint32_t* h_most;         // [tokens] and of weights * h [tokens * top_k]
  uint32_t* status;         // optional: where a bounded wait gave up
  uint32_t tokens, top_k, experts, hidden, inter;
  uint32_t by_expert;       // grid.y of the first kernel: expert ids, or assignments
};

struct DecodeParams {
  CUtensorMap weights;      // w_gate_up as {hidden, inter, 2 * experts}, box 128 B x 64 x 2, or
                            // w_down as {inter, hidden, experts}, box 128 B x 128
  CUtensorMap acts[kMaxTokens / kGroup];   // boxes of 8, 16, ... rows: x as {hidden, tokens},
                                           // h as {inter, rows, 2}, both halves in one box;
                                           // of digits {.., rows, 3}, all three in one box
  CUtensorMap rows;         // x again, box of one row (gathered by four); of digits as
                            // {hidden, 3 * tokens}
  DecodeArgs a;
};

// A k-block is 128 bytes of every weight row: 64 BF16 or 128 INT8 values, against one 128-byte
// wide piece of the activations, or two of BF16 values.
template <Kind KIND>
struct Block {
  static constexpr uint32_t kPieces = KIND == Kind::kConvert ? 2 : 1;
  static constexpr uint32_t kK = KIND == Kind::kBf16 ? 64 : 128;
};

// Stages of one CTA: the columns that its experts really need decide how many fit.
template <Kind KIND>
struct Ring {
  uint32_t base, piece_bytes, stage_bytes, stages;
  // columns: a multiple of 16, at least as many as any MMA of the CTA has
  __device__ __forceinline__ Ring(uint32_t at, uint32_t bytes, uint32_t columns)
      : base(at),
        piece_bytes(columns * 128),
        stage_bytes(kABytes + Block<KIND>::kPieces * columns * 128),
        stages(min(bytes / stage_bytes, kMaxStages)) {}
  __device__ __forceinline__ uint32_t at(uint32_t slot) const { return base + slot * stage_bytes; }
};

// Barriers of a CTA (static shared memory).
struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];   // stage: bytes landed / MMAs done with it
  uint64_t a_full[2], a_empty[2]; // INT8: converted weights in Tensor Memory / read by the MMAs
  uint64_t d_full[2], d_empty[2]; // accumulator: complete / drained
};

struct Wait {
  volatile uint32_t* abort_word;
  __device__ __forceinline__ bool operator()(uint64_t& bar, uint32_t parity) const {
    return ptx::mbar_wait(ptx::smem_addr(&bar), parity, abort_word, kWaitBudgetNs);
  }
};

// Position in a ring of slots: slot and the parity of its current use.
struct Cursor {
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void next(uint32_t slots) {
    if (++slot == slots) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

__device__ __forceinline__ void report(const DecodeArgs& a, uint32_t site) {
  if (a.status != nullptr) atomicCAS(a.status, 0u, 0x50000000u | site);
}

// A wait of this call, or of one before it that shares the status word, ran out: the result
// is NaN rather than plausible. An epilogue whose own waits succeeded has all of its sums, so it
// is the one that knows.
__device__ __forceinline__ bool failed_before(const DecodeArgs& a) {
  return a.status != nullptr && *a.status != 0;
}
__device__ __forceinline__ float not_a_number() { return __uint_as_float(0x7fc00000u); }

// The signed bytes of `word` as BF16 pairs (bytes 0 and 1, 2 and 3), exact. With 128 + (b & 127)
// as the bits 0x4300 | (b & 0x7f), and 128 or 256 as the bits 0x4300 | (b & 0x80), the signed value
// is their difference: two masks, four byte permutations, two subtractions. (Masking the
// permuted pairs is as many instructions and 1.5 % slower over a layer; arithmetic without
// masks - f = bits 0x43 u of u = b + 128, q = f / 2 - 128, value q - max(0, -q) or
// min(q, f - 256) - is no faster.)
__device__ __forceinline__ void int8_pairs(uint32_t word, uint32_t& low, uint32_t& high) {
  const uint32_t bits = word & 0x7f7f7f7fu, signs = word & 0x80808080u;
  asm("sub.rn.bf16x2 %0, %1, %2;"
      : "=r"(low)
      : "r"(__byte_perm(bits, 0x43434343u, 0x4140)), "r"(__byte_perm(signs, 0x43434343u, 0x4140)));
  asm("sub.rn.bf16x2 %0, %1, %2;"
      : "=r"(high)
      : "r"(__byte_perm(bits, 0x43434343u, 0x4342)), "r"(__byte_perm(signs, 0x43434343u, 0x4342)));
}

__device__ __forceinline__ uint16_t to_bf16(float v) {
  uint16_t b;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(v));
  return b;
}

__device__ __forceinline__ float from_bf16(uint16_t v) {
  return __uint_as_float(static_cast<uint32_t>(v) << 16);
}

// ------------------------------------------------------------------- roles --

// MMA issuer: `blocks` k-blocks into the accumulator at `d_tmem` (n columns). Returns false
// when a wait gave up. The warp is converged; one elected lane issues.
template <Kind KIND>
__device__ __forceinline__ bool issue_blocks(const Wait& wait, Barriers& bars,
                                             const Ring<KIND>& ring, Cursor& stage, Cursor& a_buf,
                                             uint32_t tmem, uint32_t d_tmem, uint32_t n,
                                             uint32_t blocks, uint64_t& done) {
  constexpr bool CONVERT = KIND == Kind::kConvert;
  const uint32_t idesc = KIND == Kind::kDigits ? ptx::make_s8_idesc(kRows, n)
                                               : ptx::make_bf16_idesc(kRows, n);
  for (uint32_t b = 0; b < blocks; ++b) {
    if (!wait(bars.full[stage.slot], stage.parity)) return false;
    if (CONVERT && !wait(bars.a_full[a_buf.slot], a_buf.parity)) return false;
    ptx::tc_fence_after_sync();
    const uint32_t at = ring.at(stage.slot);
    const uint64_t a_desc = ptx::make_kmajor_sw128_desc(at);
    const uint32_t a_tmem = tmem + a_buf.slot * (kTmemA / 2);
    if (ptx::elect_one()) {
#pragma unroll
      for (uint32_t piece = 0; piece < Block<KIND>::kPieces; ++piece) {
        const uint64_t b_desc =
            ptx::make_kmajor_sw128_desc(at + kABytes + piece * ring.piece_bytes);
#pragma unroll
        for (uint32_t ks = 0; ks < 4; ++ks) {
          const uint32_t acc = (b | piece | ks) != 0 ? 1u : 0u;
          if constexpr (KIND == Kind::kDigits) {
            ptx::umma_s8_ss(d_tmem, a_desc + 2 * ks, b_desc + 2 * ks, idesc, acc);
          } else if constexpr (CONVERT) {
            ptx::umma_bf16_ts(d_tmem, a_tmem + (piece * 4 + ks) * 8, b_desc + 2 * ks, idesc, acc);
          } else {
            ptx::umma_bf16_ss(d_tmem, a_desc + 2 * ks, b_desc + 2 * ks, idesc, acc);
          }
        }
      }
      ptx::umma_commit(ptx::smem_addr(&bars.empty[stage.slot]));
      if (CONVERT) ptx::umma_commit(ptx::smem_addr(&bars.a_empty[a_buf.slot]));
      if (b + 1 == blocks) ptx::umma_commit(ptx::smem_addr(&done));
    }
    __syncwarp();
    stage.next(ring.stages);
    a_buf.next(2);
  }
  return true;
}

// INT8: one warp's 32 rows of every second of `blocks` k-blocks (`turn` 0 or 1, and that buffer)
// from shared memory to Tensor Memory as BF16. Two groups of four warps take turns, since most
// of a block's time in a warp is latency. The conversion costs a large layer of few tokens 72-76
// instead of 85-87 % of the copy bandwidth (hence the digits, which leave it the small layers and
// the crowded experts): the integer pipe is busy 56 % of the time at 4.5 TB/s and the issue
// slots 49 % (one token). Fewer integer operations (see int8_pairs), four groups instead of two
// and converting ahead of the free buffer all measured within 1 %.
//
// The buffer is waited for before the stage. With an odd number of stages the two groups use a
// slot in turn, so a group has not seen the slot's use before its own, and a wait by parity
// takes that use, if its load is still under way, for the one it waits for: the block of one
// ring earlier would be converted. Buffer b % 2 is free when the MMAs of block b - 2 are
// through, so block b - 2 and all before it have landed, and with two stages or more the
// slot's use before is one of them.
__device__ __forceinline__ bool convert_blocks(const Wait& wait, Barriers& bars,
                                               const Ring<Kind::kConvert>& ring, uint32_t tmem,
                                               uint32_t quad, uint32_t turn, uint32_t lane,
                                               uint32_t blocks) {
  Cursor stage;
  uint32_t a_parity = 0;
  if (turn != 0) stage.next(ring.stages);
  const uint32_t to = tmem + turn * (kTmemA / 2) + ((quad * 32) << 16);
  for (uint32_t b = turn; b < blocks; b += 2) {
    if (!wait(bars.a_empty[turn], a_parity ^ 1u)) return false;
    if (!wait(bars.full[stage.slot], stage.parity)) return false;
    ptx::tc_fence_after_sync();
    const uint32_t row = ring.at(stage.slot) + (quad * 32 + lane) * 128;
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {
      uint32_t v[32];
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) {
        // 16-byte pieces of a 128-byte row are swizzled by the row's place in its group of 8
        const uint4 w = ptx::ld_shared_v4(row + (((half * 4 + c) ^ (lane & 7)) << 4));
        int8_pairs(w.x, v[8 * c + 0], v[8 * c + 1]);
        int8_pairs(w.y, v[8 * c + 2], v[8 * c + 3]);
        int8_pairs(w.z, v[8 * c + 4], v[8 * c + 5]);
        int8_pairs(w.w, v[8 * c + 6], v[8 * c + 7]);
      }
      ptx::tmem_store_32x32(to + half * 32, v);
    }
    ptx::tmem_store_wait();
    ptx::tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&bars.a_full[turn]));
    stage.next(ring.stages);
    stage.next(ring.stages);
    a_parity ^= 1u;
  }
  return true;
}

__device__ __forceinline__ void init_barriers(Barriers& bars) {
  for (uint32_t s = 0; s < kMaxStages; ++s) {
    ptx::mbar_init(ptx::smem_addr(&bars.full[s]), 1);
    ptx::mbar_init(ptx::smem_addr(&bars.empty[s]), 1);
  }
  for (uint32_t b = 0; b < 2; ++b) {
    ptx::mbar_init(ptx::smem_addr(&bars.a_full[b]), 4);    // converting warps
    ptx::mbar_init(ptx::smem_addr(&bars.a_empty[b]), 1);
    ptx::mbar_init(ptx::smem_addr(&bars.d_full[b]), 1);
    ptx::mbar_init(ptx::smem_addr(&bars.d_empty[b]), 4);   // epilogue warps
  }
  ptx::fence_barrier_init();
}

// Copies and MMAs that an expired wait left behind land before their memory goes away.
__device__ __forceinline__ void settle(volatile uint32_t* abort_word) {
  if (*abort_word == 0) return;
  const uint64_t start = ptx::global_timer_ns();
  while (ptx::global_timer_ns() - start < 200000) __nanosleep(1000);
}

// The word at the same shared-memory address of every CTA of the cluster, summed in the order
// of their ranks; all loads are in flight together. The sum has to be used before the cluster's
// last barrier: a load that nobody waits for could still be under way when its CTA is gone.
__device__ __forceinline__ float sum_over_cluster(uint32_t address, uint32_t ranks) {
  float part[8];
  if (ranks == 1) {
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(part[0]) : "r"(address) : "memory");
    return part[0];
  }
#pragma unroll
  for (uint32_t s = 0; s < 8; ++s) {
    part[s] = s < ranks ? ptx::ld_cluster_f32(ptx::map_to_cta(address, s)) : 0.0f;
  }
  float sum = part[0];
#pragma unroll
  for (uint32_t s = 1; s < 8; ++s) {
    if (s < ranks) sum += part[s];
  }
  return sum;
}

// Sums of 8 tokens from the integer sums of their digits, `plane` columns apart, most
// significant first: FP32 holds the largest within 2^-24 of itself.
__device__ __forceinline__ void digits_to_float(uint32_t tmem, uint32_t plane, float (&v)[kGroup]) {
  uint32_t d[kDigits][kGroup];
#pragma unroll
  for (uint32_t i = 0; i < kDigits; ++i) ptx::tmem_load_32x8(tmem + i * plane, d[i]);
  ptx::tmem_load_wait();
#pragma unroll
  for (uint32_t c = 0; c < kGroup; ++c) {
    v[c] = 0.0f;
#pragma unroll
    for (uint32_t i = kDigits; i-- > 0;) {
      v[c] = fmaf(static_cast<float>(static_cast<int32_t>(d[i][c])),
                  static_cast<float>(1u << (8 * (kDigits - 1 - i))), v[c]);
    }
  }
}

// ----------------------------------------------------- activations to digits --

constexpr uint32_t kDigitThreads = 512;

__device__ __forceinline__ void load16(const uint16_t* from, float (&v)[16]) {
#pragma unroll
  for (uint32_t half = 0; half < 2; ++half) {
    const uint4 w = *reinterpret_cast<const uint4*>(from + 8 * half);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      v[8 * half + 2 * i] = __uint_as_float(words[i] << 16);
      v[8 * half + 2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void load16(const float* from, float (&v)[16]) {
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const float4 w = *reinterpret_cast<const float4*>(from + 4 * i);
    v[4 * i] = w.x;
    v[4 * i + 1] = w.y;
    v[4 * i + 2] = w.z;
    v[4 * i + 3] = w.w;
  }
}

// Rows as fixed-point numbers of three signed bytes:
//   v = unit * (d0 * 65536 + d1 * 256 + d2),  unit = 2^(e - 21),  2^e <= max |v| < 2^(e + 1)
// The unit is a power of two, so BF16 values down to 2^-14 of the row's largest are exact and
// smaller ones are off by half a unit at most, 2^-22 of the largest. Three digits because two
// (2^-14) would be coarser than BF16 itself and four cost the MMA, the ring and the SM's intake
// a third more. A row with a NaN or an infinity has the unit NaN; e >= -100 keeps the factor
// 1 / unit finite, and a row of zeros zero (rows whose largest is below 2^-100 have the unit 2^-121).
__device__ __forceinline__ uint32_t digit_exponent(uint32_t most) {   // e + 127
  return min(max(most >> 23, 27u), 254u);
}

__device__ __forceinline__ float digit_unit(uint32_t most) {
  return __uint_as_float(most < 0x7f800000u ? (digit_exponent(most) - 21u) << 23 : 0x7fc00000u);
}

// Planes [digit][rows][cols] from rows [rows, cols]. Of x (BF16) a CTA takes a whole row, finds
// its largest magnitude (bits, as unsigned integers: NaN last) and clears those of the row's h.
// Of h (FP32) the first kernel has found it, so a row is shared among the CTAs of grid.y (2 us
// less at 14336 values than one CTA with two passes).
template <typename T>
__global__ void __launch_bounds__(kDigitThreads, 2)
decode_digits_kernel(const T* src, uint8_t* planes, uint32_t cols, uint32_t* x_most,
                     uint32_t* h_most, uint32_t top_k) {
  constexpr bool kOfX = sizeof(T) == 2;
  __shared__ uint32_t warp_most[kDigitThreads / 32];
  ptx::launch_dependents();
  ptx::wait_for_previous_grid();
  const T* const row = src + static_cast<size_t>(blockIdx.x) * cols;
  const uint32_t from = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
  const uint32_t step = gridDim.y * blockDim.x * 16;
  uint32_t most = 0;
  if constexpr (kOfX) {
    for (uint32_t c = from; c < cols; c += step) {
      float v[16];
      load16(row + c, v);
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    most = __reduce_max_sync(kFullWarp, most);
    if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
    __syncthreads();
    const uint32_t warps = blockDim.x / 32;
    most = (threadIdx.x & 31) < warps ? warp_most[threadIdx.x & 31] : 0u;
    most = __reduce_max_sync(kFullWarp, most);
    if (threadIdx.x == 0) x_most[blockIdx.x] = most;
    if (threadIdx.x < top_k) h_most[blockIdx.x * top_k + threadIdx.x] = 0;
  } else {
    most = h_most[blockIdx.x];
  }
  const bool finite = most < 0x7f800000u;
  const float factor = __uint_as_float((127u + 21u + 127u - digit_exponent(most)) << 23);
  const size_t plane = static_cast<size_t>(gridDim.x) * cols;
  uint8_t* const to = planes + static_cast<size_t>(blockIdx.x) * cols;
  for (uint32_t c = from; c < cols; c += step) {
    float v[16];
    load16(row + c, v);
    uint32_t word[kDigits][4] = {};
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      int32_t rest = finite ? __float2int_rn(v[i] * factor) : 0;
#pragma unroll
      for (uint32_t d = kDigits; d-- > 0;) {
        word[d][i / 4] |= (static_cast<uint32_t>(rest) & 0xffu) << (8 * (i % 4));
        rest = (rest + 128) >> 8;
      }
    }
#pragma unroll
    for (uint32_t d = 0; d < kDigits; ++d) {
      *reinterpret_cast<uint4*>(to + d * plane + c) =
          make_uint4(word[d][0], word[d][1], word[d][2], word[d][3]);
    }
  }
}

// --------------------------------------------------- gate and up products --

template <Kind KIND>
constexpr uint32_t kUpThreads = KIND == Kind::kConvert ? 384 : 256;

template <Kind KIND, uint32_t COLS>
constexpr uint32_t kUpTmem = KIND == Kind::kConvert  ? 256
                             : KIND == Kind::kDigits ? 4 * COLS
                                                     : (COLS < 32 ? 32 : COLS);

// A cluster computes 64 channels of one expert for all of its tokens: the tile's rows 0-63
// are the channels' gate rows, 64-127 their up rows. The activations of a k-block are one box per
// piece (every load takes the producer some 60 cycles to issue): the groups of 8 tokens from
// the expert's first to its last. Where its tokens are few and far between that would
// be more bytes than the weights, and an SM takes in some 30 bytes a cycle: then only the
// tokens themselves are gathered, four per load, if that is half the rows or less.
template <Kind KIND, uint32_t COLS>
__global__ void __launch_bounds__(kUpThreads<KIND>, 2)
decode_up_kernel(const __grid_constant__ DecodeParams p, uint32_t ring_bytes) {
  constexpr bool INT8 = KIND != Kind::kBf16, DIGITS = KIND == Kind::kDigits;
  constexpr uint32_t kPieces = Block<KIND>::kPieces, kBlockK = Block<KIND>::kK;
  constexpr uint32_t kPlanes = DIGITS ? kDigits : 1;   // columns per token
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers bars;
  __shared__ uint32_t tmem_slot, abort_slot, spoiled_slot;
  __shared__ uint32_t list_mask[2], list_base, list_expert;   // tokens of the expert
  __shared__ float list_coef[kMaxTokens], channel_scale[2][64];
  __shared__ uint8_t list_token[kMaxTokens];
  const DecodeArgs& a = p.a;
  const uint32_t base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Wait wait{&abort_slot};

  if (warp == 0) {
    if (lane == 0) {
      ptx::tensormap_prefetch(&p.weights);
      ptx::tensormap_prefetch(&p.acts[0]);
    }
    // Tokens of this cluster's expert; rows of h in front of it (one per assignment to a
    // lower id). By assignment: the expert's first one does the work.
    const int64_t e = a.by_expert != 0 ? static_cast<int64_t>(blockIdx.y) : a.ids[blockIdx.y];
    uint32_t mask[2] = {0, 0}, before = 0, owner = kFullWarp;
    if (e >= 0 && e < a.experts) {
#pragma unroll 4
      for (uint32_t r = lane; r < a.tokens * a.top_k; r += 32) {
        const int64_t id = a.ids[r];
        if (id == e) {
          const uint32_t t = r / a.top_k;
          mask[0] |= t < 32 ? 1u << t : 0u;
          mask[1] |= t < 32 ? 0u : 1u << (t - 32);
          owner = min(owner, r);
        }
        before += id >= 0 && id < e ? 1u : 0u;
      }
      mask[0] = __reduce_or_sync(kFullWarp, mask[0]);
      mask[1] = __reduce_or_sync(kFullWarp, mask[1]);
      before = __reduce_add_sync(kFullWarp, before);
      owner = __reduce_min_sync(kFullWarp, owner);
      if (a.by_expert == 0 && owner != blockIdx.y) mask[0] = mask[1] = 0;
    }
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {
      if ((mask[half] >> lane) & 1u) {
        const uint32_t t = half * 32 + lane;
        const uint32_t at =
            (half != 0 ? __popc(mask[0]) : 0) + __popc(mask[half] & ((1u << lane) - 1));
        list_token[at] = static_cast<uint8_t>(t);
      }
    }
    if (lane == 0) {
      list_mask[0] = mask[0];
      list_mask[1] = mask[1];
      list_base = before;
      list_expert = static_cast<uint32_t>(e);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      abort_slot = 0;
      spoiled_slot = failed_before(a) ? 1u : 0u;
      init_barriers(bars);
    }
    __syncwarp();
    ptx::tmem_alloc(ptx::smem_addr(&tmem_slot), (kUpTmem<KIND, COLS>));
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  // Let the second kernel's CTAs take their places as this grid's last CTAs run; not before
  // this CTA has its Tensor Memory, which a waiting CTA of the second kernel would hold.
  ptx::launch_dependents();
  const uint32_t tmem = tmem_slot;
  const uint32_t mask[2] = {list_mask[0], list_mask[1]};
  const uint32_t count = __popc(mask[0]) + __popc(mask[1]);
  if (count == 0) {                        // the whole cluster: its CTAs share the expert
    if constexpr (DIGITS) ptx::wait_for_previous_grid();   // nor may this grid end first
    if (warp == 1) ptx::tmem_dealloc(tmem, (kUpTmem<KIND, COLS>));
    return;
  }
  const uint32_t expert = list_expert;
  const uint32_t d_tmem = tmem + (KIND == Kind::kConvert ? kTmemA : 0);
  const uint32_t token0 = list_token[0] / kGroup * kGroup;
  const uint32_t boxes = list_token[count - 1] / kGroup - token0 / kGroup + 1;
  const uint32_t quads = (count + 3) / 4;
  const bool gather = COLS > 16 && quads <= boxes && quads <= kMostQuads;
  const uint32_t plane = gather ? 4 * quads : kGroup * boxes;   // columns of a plane of digits
  const uint32_t columns = plane * kPlanes;
  const uint32_t n = (columns + 15) / 16 * 16;     // columns of the MMA
  const Ring<KIND> ring(base, ring_bytes, n);

  const uint32_t rank = ptx::cluster_cta_rank(), ranks = ptx::cluster_cta_count();
  const uint32_t channel0 = blockIdx.x / ranks * 64;
  const uint32_t all_blocks = (a.hidden + kBlockK - 1) / kBlockK;
  const uint32_t begin = all_blocks * rank / ranks, end = all_blocks * (rank + 1) / ranks;

  if (warp == 0) {
    Cursor stage;
    const uint32_t bytes = kABytes + columns * kPieces * 128;
    // token indices of the gathers, a byte each; the rows behind the last are outside x
    uint32_t quad_tokens[kMostQuads];
#pragma unroll
    for (uint32_t q = 0; q < kMostQuads; ++q) {
      quad_tokens[q] = 0;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t t = 4 * q + i < count ? list_token[4 * q + i] : kMaxTokens;
        quad_tokens[q] |= t << (8 * i);
      }
    }
    auto load_weights = [&](uint32_t b, uint32_t s) {
      const uint32_t bar = ptx::smem_addr(&bars.full[s]);
      ptx::mbar_arrive_expect_tx(bar, bytes);
      ptx::tma_load_3d(ring.at(s), &p.weights, bar, static_cast<int32_t>(b * kBlockK),
                       static_cast<int32_t>(channel0), static_cast<int32_t>(2 * expert));
    };
    auto load_acts = [&](uint32_t b, uint32_t s) {
      const uint32_t bar = ptx::smem_addr(&bars.full[s]);
#pragma unroll
      for (uint32_t piece = 0; piece < kPieces; ++piece) {
        const uint32_t to = ring.at(s) + kABytes + piece * ring.piece_bytes;
        const int32_t k = static_cast<int32_t>(b * kBlockK + 64 * piece);
        if (!gather) {
          if constexpr (DIGITS) {
            ptx::tma_load_3d(to, &p.acts[boxes - 1], bar, k, static_cast<int32_t>(token0), 0);
          } else {
            ptx::tma_load_2d(to, &p.acts[boxes - 1], bar, k, static_cast<int32_t>(token0));
          }
        } else if constexpr (COLS > 16) {
#pragma unroll
          for (uint32_t q = 0; q < kMostQuads; ++q) {
            const uint32_t t = quad_tokens[q];
            if (q >= quads) break;
#pragma unroll
            for (uint32_t d = 0; d < kPlanes; ++d) {
              const int32_t first = static_cast<int32_t>(d * a.tokens);
              ptx::tma_gather4(to + (d * quads + q) * 512, &p.rows, bar, k, first + (t & 0xff),
                               first + ((t >> 8) & 0xff), first + ((t >> 16) & 0xff),
                               first + (t >> 24));
            }
          }
        }
      }
    };
    uint32_t ahead = begin;
    if constexpr (DIGITS) {
      // the first stages' weights do not wait for the digits of x
      ahead = min(begin + ring.stages, end);
      if (ptx::elect_one()) {
        for (uint32_t b = begin; b < ahead; ++b) load_weights(b, b - begin);
      }
      __syncwarp();
      ptx::wait_for_previous_grid();
      ptx::fence_proxy_async_all();
      if (ptx::elect_one()) {
        for (uint32_t b = begin; b < ahead; ++b) load_acts(b, b - begin);
      }
      __syncwarp();
      stage.parity = 1;                    // second use of every stage
    }
    for (uint32_t b = ahead; b < end; ++b) {
      if (!wait(bars.empty[stage.slot], stage.parity ^ 1u)) {
        if (lane == 0) report(a, 1);
        break;
      }
      if (ptx::elect_one()) {
        load_weights(b, stage.slot);
        load_acts(b, stage.slot);
      }
      __syncwarp();
      stage.next(ring.stages);
    }
  } else if (warp == 1) {
    Cursor stage, a_buf;
    if (!issue_blocks<KIND>(wait, bars, ring, stage, a_buf, tmem, d_tmem, n, end - begin,
                            bars.d_full[0])) {
      if (lane == 0) report(a, 2);
    }
  } else if (warp == 2) {
    // weight of every listed token: the sum where it names the expert twice
    for (uint32_t at = lane; at < count; at += 32) {
      const uint32_t t = list_token[at];
      float coef = 0.0f;
      for (uint32_t j = 0; j < a.top_k; ++j) {
        if (a.ids[t * a.top_k + j] == static_cast<int64_t>(expert)) coef += a.coef[t * a.top_k + j];
      }
      list_coef[at] = coef;
    }
  } else if (warp == 3) {
    if constexpr (INT8) {
      for (uint32_t c = lane; c < 64 && channel0 + c < a.inter; c += 32) {
        const float* const scale = a.s1 + static_cast<size_t>(expert) * 2 * a.inter + channel0 + c;
        channel_scale[0][c] = scale[0];
        channel_scale[1][c] = scale[a.inter];
      }
    }
  } else if (warp >= 4) {
    const uint32_t quad = warp & 3;
    bool ok = true;
    if constexpr (KIND == Kind::kConvert) {
      ok = convert_blocks(wait, bars, ring, tmem, quad, (warp - 4) / 4, lane, end - begin);
      if (!ok && lane == 0) report(a, 3);
    }
    // Accumulator -> shared memory [column][row], over the ring: all of its bytes are used.
    if (warp < 8 && ok && wait(bars.d_full[0], 0)) {
      ptx::tc_fence_after_sync();
      const uint32_t to = base + (quad * 32 + lane) * 4;
      if constexpr (DIGITS) {
        for (uint32_t c = 0; c < plane; c += kGroup) {
          float v[kGroup];
          digits_to_float(d_tmem + ((quad * 32) << 16) + c, plane, v);
#pragma unroll
          for (uint32_t i = 0; i < kGroup; ++i) {
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + (c + i) * kRows * 4), "f"(v[i])
                         : "memory");
          }
        }
      }
#pragma unroll
      for (uint32_t c = 0; c < (DIGITS ? 0 : COLS); c += 16) {
        if (c < n) {
          uint32_t v[16];
          ptx::tmem_load_32x16(d_tmem + ((quad * 32) << 16) + c, v);
          ptx::tmem_load_wait();
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + (c + i) * kRows * 4), "r"(v[i])
                         : "memory");
          }
        }
      }
      ptx::tc_fence_before_sync();
    } else if (warp < 8 && lane == 0) {
      spoiled_slot = 1;
      report(a, 4);
    }
  }
  __syncwarp();
  if constexpr (DIGITS) ptx::wait_for_previous_grid();   // x_most; and see above
  settle(&abort_slot);
  if (warp >= 4 && warp < 8 && spoiled_slot != 0) {
    // NaN in h, and from there in every output channel of the expert's tokens
    for (uint32_t c = 0; c < plane; ++c) {
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + (c * kRows + (warp & 3) * 32 + lane) * 4),
                   "f"(not_a_number())
                   : "memory");
    }
  }
  if (ranks > 1) {
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }

  // Join the k shares in a fixed order; weights * silu(gate) * up in FP32 (its digits are made
  // from the whole row) or in two BF16 halves.
  for (uint32_t i = rank * kUpThreads<KIND> + threadIdx.x; i < 64 * count;
       i += ranks * kUpThreads<KIND>) {
    const uint32_t c = i % 64, at = i / 64;
    const uint32_t channel = channel0 + c;
    const bool inside = channel < a.inter;
    if (!DIGITS && !inside) continue;
    const uint32_t cell = base + ((gather ? at : list_token[at] - token0) * kRows + c) * 4;
    float gate = 0.0f, up = 0.0f;
    if (inside) {
      gate = sum_over_cluster(cell, ranks);
      up = sum_over_cluster(cell + 64 * 4, ranks);
    }
    if constexpr (INT8) {
      const float unit = DIGITS ? digit_unit(a.x_most[list_token[at]]) : 1.0f;
      gate *= channel_scale[0][c] * unit;
      up *= channel_scale[1][c] * unit;
    }
    const float v = gate / (1.0f + expf(-gate)) * up * list_coef[at];
    if constexpr (DIGITS) {
      // a warp has 32 channels of one token
      const uint32_t most = __reduce_max_sync(kFullWarp, inside ? __float_as_uint(fabsf(v)) : 0u);
      if (lane == 0) atomicMax(a.h_most + list_base + at, most);
      if (inside) a.h32[static_cast<size_t>(list_base + at) * a.inter + channel] = v;
      continue;
    }
    // 16 significant bits in two BF16 numbers; an infinity has no remainder
    const uint16_t hi = to_bf16(v);
    const float rest = v - from_bf16(hi);
    uint16_t* const to = a.h + static_cast<size_t>(list_base + at) * a.inter + channel;
    to[0] = hi;
    to[static_cast<size_t>(a.tokens) * a.top_k * a.inter] = to_bf16(isfinite(rest) ? rest : 0.0f);
  }
  if (ranks > 1) ptx::cluster_sync_relaxed();   // a neighbour may still read this CTA's tile
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, (kUpTmem<KIND, COLS>));
  }
}

// ------------------------------------------------------------ down product --

template <Kind KIND>
constexpr uint32_t kDownThreads = KIND == Kind::kConvert ? 512 : 256;

template <Kind KIND, uint32_t COLS>
constexpr uint32_t kDownTmem = KIND == Kind::kConvert  ? (COLS == 64 ? 512 : 256)
                               : KIND == Kind::kDigits ? 8 * COLS
                                                       : 4 * COLS;

// Lists in dynamic shared memory, per expert: token mask (8 bytes), assignments (4), and for
// the chosen ones in ascending order id and first row of h (2 + 2).
constexpr uint32_t kListBytes = 16;

// A cluster computes 128 output channels for all tokens: the chosen experts' k ranges, laid
// end to end, are shared among its CTAs. A thread of the epilogue owns one channel and adds
// every expert's accumulator columns to its tokens' sums in shared memory.
template <Kind KIND, uint32_t COLS>
__global__ void __launch_bounds__(kDownThreads<KIND>, 2)
decode_down_kernel(const __grid_constant__ DecodeParams p, uint32_t ring_bytes) {
  constexpr bool INT8 = KIND != Kind::kBf16, CONVERT = KIND == Kind::kConvert;
  constexpr bool DIGITS = KIND == Kind::kDigits;
  constexpr uint32_t kPieces = Block<KIND>::kPieces, kBlockK = Block<KIND>::kK;
  constexpr uint32_t kThreads = kDownThreads<KIND>;
  constexpr uint32_t kPlanes = DIGITS ? kDigits : 2;        // columns per row of h
  constexpr uint32_t kColumns = DIGITS ? 4 * COLS : 2 * COLS;   // of an accumulator
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers bars;
  __shared__ uint32_t tmem_slot, abort_slot, spoiled_slot, active_count;
  const DecodeArgs& a = p.a;
  const uint32_t raw = ptx::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const behind = smem_raw + (base - raw) + ring_bytes;
  float* const sums = reinterpret_cast<float*>(behind);                  // [tokens][128]
  uint32_t* const masks = reinterpret_cast<uint32_t*>(behind + a.tokens * kRows * 4);
  uint32_t* const assigned = masks + 2 * a.experts;
  uint16_t* const active = reinterpret_cast<uint16_t*>(assigned + a.experts);
  uint16_t* const first_row = active + a.experts;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Wait wait{&abort_slot};

  // Lists of the chosen experts; nothing here depends on the first kernel.
  for (uint32_t i = threadIdx.x; i < 3 * a.experts; i += kThreads) masks[i] = 0;
  for (uint32_t i = threadIdx.x; i < a.tokens * kRows; i += kThreads) sums[i] = 0.0f;
  if (warp == 1) {
    if (lane == 0) {
      abort_slot = 0;
      spoiled_slot = failed_before(a) ? 1u : 0u;
      init_barriers(bars);
    }
    __syncwarp();
    ptx::tmem_alloc(ptx::smem_addr(&tmem_slot), (kDownTmem<KIND, COLS>));
    ptx::tmem_relinquish();
  } else if (warp == 0 && lane == 0) {
    ptx::tensormap_prefetch(&p.weights);
    ptx::tensormap_prefetch(&p.acts[0]);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  for (uint32_t i = threadIdx.x; i < a.tokens * a.top_k; i += kThreads) {
    const int64_t e = a.ids[i];
    if (e >= 0 && e < a.experts) {
      const uint32_t t = i / a.top_k;
      atomicOr(&masks[2 * e + t / 32], 1u << (t % 32));
      atomicAdd(&assigned[e], 1u);
    }
  }
  __syncthreads();
  if (warp == 0) {
    // experts lane * per ... of this lane: counts, then ids and rows behind a warp scan
    const uint32_t per = (a.experts + 31) / 32;
    const uint32_t from = min(lane * per, a.experts), to = min(from + per, a.experts);
    uint32_t chosen = 0, rows = 0;
    for (uint32_t e = from; e < to; ++e) {
      chosen += assigned[e] != 0 ? 1u : 0u;
      rows += assigned[e];
    }
    uint32_t chosen_end = chosen, rows_end = rows;
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(kFullWarp, chosen_end, d);
      const uint32_t v = __shfl_up_sync(kFullWarp, rows_end, d);
      if (lane >= d) {
        chosen_end += u;
        rows_end += v;
      }
    }
    if (lane == 31) active_count = chosen_end;
    uint32_t at = chosen_end - chosen, row = rows_end - rows;
    for (uint32_t e = from; e < to; ++e) {
      if (assigned[e] != 0) {
        active[at] = static_cast<uint16_t>(e);
        first_row[at] = static_cast<uint16_t>(row);
        ++at;
        row += assigned[e];
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = tmem_slot;
  const uint32_t rank = ptx::cluster_cta_rank(), ranks = ptx::cluster_cta_count();
  const uint32_t channel0 = blockIdx.x / ranks * kRows;
  const uint32_t d_tmem = tmem + (CONVERT ? kTmemA : 0);
  const uint32_t blocks = (a.inter + kBlockK - 1) / kBlockK;             // of one expert
  const uint32_t total = active_count * blocks;
  const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(total) * rank / ranks);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(total) * (rank + 1) / ranks);

  // Columns of the expert at position `slot`, and how many of its blocks from `at` on are ours.
  auto tokens_of = [&](uint32_t slot) {
    const uint32_t e = active[slot];
    return __popc(masks[2 * e]) + __popc(masks[2 * e + 1]);
  };
  auto run_of = [&](uint32_t at) { return min(end, (at / blocks + 1) * blocks) - at; };
  // rows of h that are loaded for the expert, in groups of 8
  auto boxes_of = [&](uint32_t slot) { return (tokens_of(slot) + kGroup - 1) / kGroup; };
  uint32_t most = 1;
  for (uint32_t at = begin; at < end; at += run_of(at)) most = max(most, boxes_of(at / blocks));
  // columns of the MMA: a multiple of 16
  auto columns_of = [&](uint32_t groups) { return (groups * kPlanes * kGroup + 15) / 16 * 16; };
  const Ring<KIND> ring(base, ring_bytes, columns_of(most));

  if (warp == 0) {
    auto load_weights = [&](uint32_t at, uint32_t s) {
      const uint32_t slot = at / blocks;
      ptx::tma_load_3d(ring.at(s), &p.weights, ptx::smem_addr(&bars.full[s]),
                       static_cast<int32_t>((at - slot * blocks) * kBlockK),
                       static_cast<int32_t>(channel0), active[slot]);
    };
    auto expect = [&](uint32_t at, uint32_t s) {
      ptx::mbar_arrive_expect_tx(ptx::smem_addr(&bars.full[s]),
                                 kABytes + boxes_of(at / blocks) * kPlanes * kPieces * kGroup * 128);
    };
    auto load_acts = [&](uint32_t at, uint32_t s) {
      const uint32_t slot = at / blocks;
      const uint32_t boxes = boxes_of(slot);
      const int32_t k = static_cast<int32_t>((at - slot * blocks) * kBlockK);
#pragma unroll
      for (uint32_t piece = 0; piece < kPieces; ++piece) {
        // rows beyond the expert's are other rows of h: columns that nobody reads
        ptx::tma_load_3d(ring.at(s) + kABytes + piece * ring.piece_bytes, &p.acts[boxes - 1],
                         ptx::smem_addr(&bars.full[s]), k + static_cast<int32_t>(64 * piece),
                         first_row[slot], 0);
      }
    };
    // The first stages' weights do not wait for the first kernel, their activations do.
    const uint32_t ahead = min(begin + ring.stages, end);
    if (ptx::elect_one()) {
      for (uint32_t at = begin; at < ahead; ++at) {
        expect(at, at - begin);
        load_weights(at, at - begin);
      }
    }
    __syncwarp();
    ptx::wait_for_previous_grid();
    ptx::fence_proxy_async_all();
    if (ptx::elect_one()) {
      for (uint32_t at = begin; at < ahead; ++at) load_acts(at, at - begin);
    }
    __syncwarp();
    Cursor stage;
    stage.parity = 1;                      // second use of every stage
    for (uint32_t at = ahead; at < end; ++at) {
      if (!wait(bars.empty[stage.slot], stage.parity ^ 1u)) {
        if (lane == 0) report(a, 5);
        break;
      }
      if (ptx::elect_one()) {
        expect(at, stage.slot);
        load_weights(at, stage.slot);
        load_acts(at, stage.slot);
      }
      __syncwarp();
      stage.next(ring.stages);
    }
  } else if (warp == 1) {
    Cursor stage, a_buf, d_buf;
    for (uint32_t at = begin; at < end;) {
      const uint32_t run = run_of(at);
      const uint32_t n = columns_of(boxes_of(at / blocks));
      if (!wait(bars.d_empty[d_buf.slot], d_buf.parity ^ 1u)) {
        if (lane == 0) report(a, 6);
        break;
      }
      ptx::tc_fence_after_sync();
      if (!issue_blocks<KIND>(wait, bars, ring, stage, a_buf, tmem,
                              d_tmem + d_buf.slot * kColumns, n, run,
                              bars.d_full[d_buf.slot])) {
        if (lane == 0) report(a, 7);
        break;
      }
      d_buf.next(2);
      at += run;
    }
  } else if (CONVERT && warp >= 4 && warp < 12) {
    if constexpr (CONVERT) {
      if (!convert_blocks(wait, bars, ring, tmem, warp & 3, (warp - 4) / 4, lane, end - begin)) {
        if (lane == 0) report(a, 8);
      }
    }
  } else if (warp >= (CONVERT ? 12 : 4)) {
    const uint32_t quad = warp & 3;
    const uint32_t row = quad * 32 + lane;
    float* const mine = sums + row;
    Cursor d_buf;
    if constexpr (DIGITS) ptx::wait_for_previous_grid();   // h_most
    for (uint32_t at = begin; at < end;) {
      const uint32_t run = run_of(at);
      const uint32_t e = active[at / blocks];
      const uint32_t count = tokens_of(at / blocks);
      unsigned long long left = static_cast<unsigned long long>(masks[2 * e + 1]) << 32 | masks[2 * e];
      float scale = 1.0f;
      if constexpr (INT8) {
        if (channel0 + row < a.hidden) {
          scale = a.s2[static_cast<size_t>(e) * a.hidden + channel0 + row];
        }
      }
      if (!wait(bars.d_full[d_buf.slot], d_buf.parity)) {
        if (lane == 0) {
          spoiled_slot = 1;
          report(a, 9);
        }
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t from = d_tmem + ((quad * 32) << 16) + d_buf.slot * kColumns;
      const uint32_t boxes = boxes_of(at / blocks);
      for (uint32_t c = 0; c < boxes * kGroup; c += kGroup) {
        float v[kGroup];
        if constexpr (DIGITS) {
          digits_to_float(from + c, boxes * kGroup, v);
        } else {
          uint32_t upper[kGroup], lower[kGroup];
          ptx::tmem_load_32x8(from + c, upper);
          ptx::tmem_load_32x8(from + boxes * kGroup + c, lower);
          ptx::tmem_load_wait();
#pragma unroll
          for (uint32_t i = 0; i < kGroup; ++i) {
            v[i] = __uint_as_float(upper[i]) + __uint_as_float(lower[i]);
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < kGroup; ++i) {
          if (c + i < count) {
            const uint32_t token = __ffsll(static_cast<long long>(left)) - 1;
            left &= left - 1;
            const float unit = DIGITS ? digit_unit(a.h_most[first_row[at / blocks] + c + i]) : 1.0f;
            mine[token * kRows] = fmaf(v[i], scale * unit, mine[token * kRows]);
          }
        }
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&bars.d_empty[d_buf.slot]));
      d_buf.next(2);
      at += run;
    }
    __syncwarp();
    if (spoiled_slot != 0) {
      for (uint32_t t = 0; t < a.tokens; ++t) mine[t * kRows] = not_a_number();
    }
  }
  __syncwarp();
  // No thread goes on before the first kernel has ended: out may be x, and this grid must
  // not end first.
  ptx::wait_for_previous_grid();
  settle(&abort_slot);
  if (ranks > 1) {
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }

  // Join the cluster's CTAs in a fixed order.
  const uint32_t sums_smem = ptx::smem_addr(sums);
  for (uint32_t i = rank * kThreads + threadIdx.x; i < a.tokens * kRows; i += ranks * kThreads) {
    const uint32_t channel = channel0 + i % kRows;
    if (channel < a.hidden) {
      const float sum = sum_over_cluster(sums_smem + i * 4, ranks);
      a.out[static_cast<size_t>(i / kRows) * a.hidden + channel] = to_bf16(sum);
    }
  }
  if (ranks > 1) ptx::cluster_sync_relaxed();   // a neighbour may still read this CTA's sums
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, (kDownTmem<KIND, COLS>));
  }
}

// ------------------------------------------------------------------ launch --

using DecodeKernel = void (*)(const DecodeParams, uint32_t);

struct Launch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attribute[2];

  Launch(uint32_t threads, uint32_t smem, uint32_t cluster, bool after_previous,
         cudaStream_t stream) {
    config.blockDim = dim3(threads);
    config.gridDim = dim3(cluster);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = cluster;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = after_previous ? 2 : 1;
  }
};

// The opt-in shared-memory size is an attribute of a kernel on a device; set once.
template <DecodeKernel kernel>
cudaError_t opt_in(int device) {
  static std::atomic<bool> done[64];
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t rc =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOnePerSm);
  if (rc == cudaSuccess) done[device].store(true, std::memory_order_release);
  return rc;
}

// Clusters of every size that the current device runs at once (SMs of a cluster share a
// processing cluster of the GPU): a property of the device and the kernel, asked for once, for
// one CTA per SM. Two CTAs of half the shared memory fit where one does; the runtime's count
// does not take that into account, so a cluster of them counts as one of half its size.
template <DecodeKernel kernel>
cudaError_t places_of(int device, uint32_t threads, uint32_t smem, uint32_t (&at_once)[9]) {
  static std::atomic<uint32_t> known[64][9];   // 0: not asked yet
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  uint32_t one[9] = {};
  for (uint32_t size = 1; size <= 8; ++size) {
    one[size] = known[device][size].load(std::memory_order_acquire);
    if (one[size] != 0) continue;
    cudaError_t rc = opt_in<kernel>(device);
    if (rc != cudaSuccess) return rc;
    const Launch launch(threads, kOnePerSm, size, false, nullptr);
    int clusters = 0;
    rc = cudaOccupancyMaxActiveClusters(&clusters, kernel, &launch.config);
    if (rc != cudaSuccess) return rc;
    one[size] = clusters > 0 ? static_cast<uint32_t>(clusters) : 1u;
    known[device][size].store(one[size], std::memory_order_release);
  }
  at_once[1] = smem == kTwoPerSm ? 2 * one[1] : one[1];
  for (uint32_t size = 2; size <= 8; ++size) {
    at_once[size] = smem == kTwoPerSm ? one[(size + 1) / 2] : one[size];
  }
  return cudaSuccess;
}

// Cluster size (up to 8, the portable limit) that finishes first: rounds of tiles per
// cluster times the blocks of a tile per CTA; a CTA keeps two blocks of a tile at least.
uint32_t cluster_size(const uint32_t (&at_once)[9], uint64_t tiles, uint64_t blocks) {
  uint32_t best = 1;
  double least = 0.0;
  for (uint32_t size = 1; size <= 8 && (size == 1 || 2ull * size <= blocks); ++size) {
    const uint64_t rounds = (tiles + at_once[size] - 1) / at_once[size];
    const double time = static_cast<double>(rounds) * static_cast<double>(blocks) / size;
    if (size == 1 || time < 0.97 * least) {   // a larger cluster has to be worth its join
      best = size;
      least = time;
    }
  }
  return best;
}

template <DecodeKernel kernel>
cudaError_t run_kernel(Launch& launch, uint64_t clusters, uint32_t gridy, uint32_t ring_bytes,
                       const DecodeParams& params) {
  const uint32_t size = launch.attribute[0].val.clusterDim.x;
  launch.config.gridDim = dim3(static_cast<uint32_t>(clusters * size), gridy);
  const cudaError_t rc = cudaLaunchKernelEx(&launch.config, kernel, params, ring_bytes);
  return rc != cudaSuccess ? rc : cudaPeekAtLastError();
}

// The kernels that make digits run between and beside those that fill an SM's shared memory. By
// default an SM would be set up with little of it for them, which it can only be when idle,
// and the neighbours' CTAs would have to wait (12 us of 77 for INT8 T=1, hidden 4096, inter 14336).
template <auto kernel>
cudaError_t share_sm() {
  static std::atomic<bool> done[64];
  int device = 0;
  cudaError_t rc = cudaGetDevice(&device);
  if (rc != cudaSuccess) return rc;
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
  rc = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                            cudaSharedmemCarveoutMaxShared);
  if (rc == cudaSuccess) done[device].store(true, std::memory_order_release);
  return rc;
}

// Rows of x or h to digits.
template <typename T>
cudaError_t launch_digits(const T* src, const DecodeArgs& a, uint32_t rows, uint32_t cols,
                          cudaStream_t stream) {
  constexpr bool kOfX = sizeof(T) == 2;
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(kOfX ? kDigitThreads : 128u);
  config.gridDim = dim3(rows, kOfX ? 1u : (cols + 2047u) / 2048u);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = kOfX ? 0 : 1;        // that of h starts while the first kernel ends
  cudaError_t rc = share_sm<decode_digits_kernel<T>>();
  if (rc != cudaSuccess) return rc;
  rc = cudaLaunchKernelEx(&config, decode_digits_kernel<T>, src, a.digits,
                                            cols, a.x_most, a.h_most, a.top_k);
  return rc != cudaSuccess ? rc : cudaPeekAtLastError();
}

template <Kind KIND, uint32_t COLS>
cudaError_t launch_decode(const DecodeParams& up, const DecodeParams& down, cudaStream_t stream) {
  constexpr bool DIGITS = KIND == Kind::kDigits;
  constexpr uint32_t kPieces = Block<KIND>::kPieces, kBlockK = Block<KIND>::kK;
  constexpr DecodeKernel kUp = decode_up_kernel<KIND, COLS>;
  constexpr DecodeKernel kDown = decode_down_kernel<KIND, COLS>;
  // Rings of two stages at least, whatever the experts' columns: loads overlap MMAs, and
  // convert_blocks counts on it. The second kernel's ring shares its place with the sums of the
  // tokens and the lists of the experts.
  constexpr auto stage_most = [](uint32_t columns) {
    return kABytes + kPieces * ((columns + 15) / 16 * 16) * 128;
  };
  constexpr uint32_t kUpPlanes = DIGITS ? kDigits : 1, kDownPlanes = DIGITS ? kDigits : 2;
  static_assert(kTwoPerSm - 1024 >= 2 * stage_most(COLS * kUpPlanes));
  static_assert(kOnePerSm - 1024 >= COLS * kRows * 4 + BMOE_MOE_DECODE_MAX_EXPERTS * kListBytes +
                                        2 * stage_most(COLS * kDownPlanes));
  const DecodeArgs& a = up.a;
  const uint32_t assignments = a.tokens * a.top_k;
  const uint32_t slots = a.by_expert != 0 ? a.experts : assignments;
  int device = 0;
  cudaError_t rc = cudaGetDevice(&device);
  if (rc != cudaSuccess) return rc;
  if constexpr (DIGITS) {
    rc = launch_digits(a.x, a, a.tokens, a.hidden, stream);
    if (rc != cudaSuccess) return rc;
  }

  // First kernel: a cluster per tile, two CTAs per SM (one streams while the other starts or
  // ends). Tiles that leave SMs idle are split along k, up to 8 ways (the portable cluster
  // size), as long as every CTA keeps two k-blocks. Splitting further, so that both places of
  // every SM are taken, costs more in starts and joins than it spreads (96 tiles, T=1:
  // 23.6 us in one piece, 24.1 in two, 26.1 in four).
  const uint64_t tiles = (a.inter + 63) / 64;
  const uint64_t blocks = (a.hidden + kBlockK - 1) / kBlockK;
  uint32_t split = 1;
  while (split < 8 && tiles * slots * split * 2 <= device_sm_count() && 4 * split <= blocks) {
    split *= 2;
  }
  rc = opt_in<kUp>(device);
  if (rc != cudaSuccess) return rc;
  Launch first(kUpThreads<KIND>, kTwoPerSm, split, DIGITS, stream);
  rc = run_kernel<kUp>(first, tiles, slots, kTwoPerSm - 1024, up);
  if (rc != cudaSuccess) return rc;
  if constexpr (DIGITS) {
    rc = launch_digits<float>(a.h32, a, assignments, a.inter, stream);
    if (rc != cudaSuccess) return rc;
  }

  // Second kernel: a cluster per 128 channels, all at once. The sums of many tokens leave less
  // for the ring: two CTAs per SM if three stages fit at twice the average number of an
  // expert's tokens and two if one expert has them all, else one.
  const uint32_t reserved = (a.tokens * kRows * 4 + a.experts * kListBytes + 15) / 16 * 16;
  const uint32_t twice = 2 * assignments / a.experts + kGroup;
  const uint32_t columns =
      (twice < a.tokens ? twice : a.tokens) / kGroup * (DIGITS ? 4 : 2) * kGroup;
  const uint32_t crowd = (a.tokens + kGroup - 1) / kGroup * kGroup;
  const bool two = kDownTmem<KIND, COLS> <= 256 &&
                   kTwoPerSm - 1024 >= reserved + 3 * (kABytes + kPieces * columns * 128) &&
                   kTwoPerSm - 1024 >= reserved + 2 * stage_most(crowd * kDownPlanes);
  const uint32_t smem = two ? kTwoPerSm : kOnePerSm;
  uint32_t at_once[9];
  rc = places_of<kDown>(device, kDownThreads<KIND>, smem, at_once);
  if (rc != cudaSuccess) return rc;
  const uint64_t groups = (a.hidden + kRows - 1) / kRows;
  const uint32_t size = cluster_size(
      at_once, groups, static_cast<uint64_t>((a.inter + kBlockK - 1) / kBlockK) * slots);
  Launch second(kDownThreads<KIND>, smem, size, true, stream);
  return run_kernel<kDown>(second, groups, 1, smem - 1024 - reserved, down);
}

// columns that a stage has room for: what the tokens need
template <Kind KIND>
cudaError_t dispatch_decode(const DecodeParams& up, const DecodeParams& down,
                            cudaStream_t stream) {
  if (up.a.tokens <= 16) return launch_decode<KIND, 16>(up, down, stream);
  if (up.a.tokens <= 32) return launch_decode<KIND, 32>(up, down, stream);
  return launch_decode<KIND, 64>(up, down, stream);
}

template <Kind KIND, uint32_t COLS>
cudaError_t preload_decode() {
  const cudaError_t rc = preload_one(decode_up_kernel<KIND, COLS>);
  return rc == cudaSuccess ? preload_one(decode_down_kernel<KIND, COLS>) : rc;
}

template <Kind KIND>
cudaError_t preload_decode_type() {
  cudaError_t rc = preload_decode<KIND, 16>();
  if (rc == cudaSuccess) rc = preload_decode<KIND, 32>();
  if (rc == cudaSuccess) rc = preload_decode<KIND, 64>();
  return rc;
}

// The workspace: h in 4 bytes a value (two BF16 halves, or FP32), and for few tokens digits
// of x, later of h, and the largest magnitudes of their rows.
struct Workspace {
  uint64_t digits, most, bytes;
  Workspace(uint64_t tokens, uint64_t top_k, uint64_t inter) {
    const auto align = [](uint64_t v) { return (v + 255) / 256 * 256; };
    const uint64_t rows = tokens * top_k;
    digits = align(4 * rows * inter);
    most = digits + align(kDigits * rows * inter);
    bytes = most + align(4 * (tokens + rows));
  }
};

// INT8 weights against digits of the activations instead of being converted, where that is
// faster: with enough weights that the stream outweighs two more launches, and not so many
// tokens per expert that three columns a token are more bytes than an SM takes in beside them.
// Measured (us, digits against conversion): 25 MB of weights 16.1 to 15.5, 33 MB 17.0 to 16.7, 38 MB
// 18.6 to 19.9, 50 MB 17.7 to 20.0, 1.4 GB 221 to 245; per expert 16 tokens 158 to 166 and 256 to 284,
// 24 tokens 174 to 188, 32 tokens 114 to 110 and 36.8 to 33.9, 64 tokens 72 to 68. The digits of x
// go where those of h will be, so they have to fit there.
constexpr uint64_t kDigitWeightBytes = 36u * 1000u * 1000u;
constexpr uint64_t kDigitTokensPerExpert = 24;

bool use_digits(const bmoe_moe_decode_args& a) {
  const uint64_t assignments = static_cast<uint64_t>(a.tokens) * a.top_k;
  const uint64_t experts = assignments < a.experts ? assignments : a.experts;
  return a.hidden <= static_cast<uint64_t>(a.top_k) * a.inter &&
         3 * experts * a.hidden * a.inter >= kDigitWeightBytes &&
         assignments <= kDigitTokensPerExpert * a.experts;
}

bool encode_maps(DecodeParams& up, DecodeParams& down, const bmoe_moe_decode_args& a,
                 Kind kind) {
  const uint8_t* const digits = up.a.digits;
  const Elem weight = kind == Kind::kBf16 ? Elem::kBf16 : Elem::kByte;
  const uint64_t elem = kind == Kind::kBf16 ? 2 : 1;
  const uint32_t line = kind == Kind::kBf16 ? 64 : 128;
  const uint64_t hidden = a.hidden, inter = a.inter;
  const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.top_k;
  {
    const uint64_t dims[3] = {hidden, inter, 2ull * a.experts};
    const uint64_t strides[2] = {hidden * elem, inter * hidden * elem};
    const uint32_t box[3] = {line, 64, 2};
    if (!encode_box(&up.weights, a.w_gate_up_dev, weight, 3, dims, strides, box)) return false;
  }
  {
    const uint64_t dims[3] = {inter, hidden, a.experts};
    const uint64_t strides[2] = {inter * elem, hidden * inter * elem};
    const uint32_t box[3] = {line, kRows, 1};
    if (!encode_box(&down.weights, a.w_down_dev, weight, 3, dims, strides, box)) return false;
  }
  if (kind == Kind::kDigits) {
    const uint64_t x_dims[3] = {hidden, a.tokens, kDigits};
    const uint64_t x_strides[2] = {hidden, a.tokens * hidden};
    const uint64_t h_dims[3] = {inter, rows, kDigits}, h_strides[2] = {inter, rows * inter};
    const uint64_t row_dims[2] = {hidden, kDigits * a.tokens}, row_strides[1] = {hidden};
    const uint32_t row_box[2] = {128, 1};
    if (a.tokens > 16 &&
        !encode_box(&up.rows, digits, Elem::kByte, 2, row_dims, row_strides, row_box)) {
      return false;
    }
    for (uint32_t g = 0; g * kGroup < a.tokens; ++g) {
      const uint32_t box[3] = {128, (g + 1) * kGroup, kDigits};
      if (!encode_box(&up.acts[g], digits, Elem::kByte, 3, x_dims, x_strides, box) ||
          !encode_box(&down.acts[g], digits, Elem::kByte, 3, h_dims, h_strides, box)) {
        return false;
      }
    }
    return true;
  }
  const uint64_t x_dims[2] = {hidden, a.tokens}, x_strides[1] = {hidden * 2};
  const uint64_t h_dims[3] = {inter, rows, 2}, h_strides[2] = {inter * 2, rows * inter * 2};
  const uint32_t row_box[2] = {64, 1};   // gathered rows: more than 16 tokens only
  if (a.tokens > 16 &&
      !encode_box(&up.rows, a.x_dev, Elem::kBf16, 2, x_dims, x_strides, row_box)) {
    return false;
  }
  for (uint32_t g = 0; g * kGroup < a.tokens; ++g) {
    const uint32_t box[3] = {64, (g + 1) * kGroup, 2};
    if (!encode_box(&up.acts[g], a.x_dev, Elem::kBf16, 2, x_dims, x_strides, box) ||
        !encode_box(&down.acts[g], a.workspace_dev, Elem::kBf16, 3, h_dims, h_strides, box)) {
      return false;
    }
  }
  return true;
}

}  // namespace

cudaError_t preload_decode_kernels() {
  cudaError_t rc = preload_decode_type<Kind::kBf16>();
  if (rc == cudaSuccess) rc = preload_decode_type<Kind::kConvert>();
  if (rc == cudaSuccess) rc = preload_decode_type<Kind::kDigits>();
  if (rc == cudaSuccess) rc = preload_one(decode_digits_kernel<uint16_t>);
  if (rc == cudaSuccess) rc = preload_one(decode_digits_kernel<float>);
  return rc;
}

}  // namespace bmoe

extern "C" uint64_t bmoe_moe_decode_workspace(uint32_t tokens, uint32_t top_k, uint32_t inter) {
  return bmoe::Workspace(tokens, top_k, inter).bytes;
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
      a.workspace_dev == nullptr || bmoe::off_grid(a.x_dev, 16) ||
      bmoe::off_grid(a.w_gate_up_dev, 16) || bmoe::off_grid(a.w_down_dev, 16) ||
      bmoe::off_grid(a.out_dev, 16) || bmoe::off_grid(a.workspace_dev, 256) ||
      bmoe::off_grid(a.expert_ids_dev, 8) || bmoe::off_grid(a.weights_dev, 4) ||
      bmoe::off_grid(a.gate_up_scale_dev, 4) || bmoe::off_grid(a.down_scale_dev, 4) ||
      bmoe::off_grid(a.status_dev, 4) ||
      a.workspace_bytes < bmoe_moe_decode_workspace(a.tokens, a.top_k, a.inter) ||
      (int8 && (a.gate_up_scale_dev == nullptr || a.down_scale_dev == nullptr))) {
    return BMOE_INVALID_ARGUMENT;
  }
  bmoe::DecodeParams up;
  bmoe::DecodeArgs& k = up.a;
  k.s1 = a.gate_up_scale_dev;
  k.s2 = a.down_scale_dev;
  k.ids = a.expert_ids_dev;
  k.coef = a.weights_dev;
  k.out = static_cast<uint16_t*>(a.out_dev);
  const bmoe::Workspace places(a.tokens, a.top_k, a.inter);
  uint8_t* const workspace = static_cast<uint8_t*>(a.workspace_dev);
  k.h = static_cast<uint16_t*>(a.workspace_dev);
  k.h32 = static_cast<float*>(a.workspace_dev);
  k.x = static_cast<const uint16_t*>(a.x_dev);
  k.digits = workspace + places.digits;
  k.x_most = reinterpret_cast<uint32_t*>(workspace + places.most);
  k.h_most = k.x_most + a.tokens;
  k.status = a.status_dev;
  k.tokens = a.tokens;
  k.top_k = a.top_k;
  k.experts = a.experts;
  k.hidden = a.hidden;
  k.inter = a.inter;
  k.by_expert = a.experts <= a.tokens * a.top_k ? 1u : 0u;
  bmoe::DecodeParams down;
  down.a = k;
  const bmoe::Kind kind = !int8                 ? bmoe::Kind::kBf16
                          : bmoe::use_digits(a) ? bmoe::Kind::kDigits
                                                : bmoe::Kind::kConvert;
  if (!bmoe::encode_maps(up, down, a, kind)) return BMOE_CUDA_ERROR;
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  cudaError_t rc;
  switch (kind) {
    case bmoe::Kind::kBf16:
      rc = bmoe::dispatch_decode<bmoe::Kind::kBf16>(up, down, stream);
      break;
    case bmoe::Kind::kConvert:
      rc = bmoe::dispatch_decode<bmoe::Kind::kConvert>(up, down, stream);
      break;
    default:
      rc = bmoe::dispatch_decode<bmoe::Kind::kDigits>(up, down, stream);
  }
  return rc == cudaSuccess ? BMOE_OK : BMOE_CUDA_ERROR;
}
