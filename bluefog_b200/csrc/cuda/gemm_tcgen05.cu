// bf16 GEMM on Blackwell's 5th-generation tensor cores:  C[M,N] = act(A[M,K] * B[N,K]^T + bias).
//
// One CTA computes one 128 x 128 output tile.  Warp 0 is the TMA producer: it streams
// 128x64 tiles of A and B (K-major, 128-byte swizzle) into a 6-stage shared-memory ring with
// `cp.async.bulk.tensor.2d` (no cluster multicast).  Warp 1 allocates 128 columns of tensor
// memory and issues `tcgen05.mma.cta_group::1.kind::f16` (M=128, N=128, K=16) from one
// elected lane, accumulating in fp32 in TMEM, and releases ring stages with
// `tcgen05.commit`.  Warps 2-5 are the epilogue: once the accumulator is complete they read
// it back with `tcgen05.ld.32x32b.x32`, add the bias, apply the activation, convert to bf16
// and store.  Producer, MMA issuer and epilogue run concurrently and synchronise only
// through mbarriers.  Every mbarrier wait has a time limit: on expiry the kernel records an
// error code, stops issuing work, waits (bounded) for its TMA copies in flight, frees its TMEM
// and returns.
//
// That is the one-tile-per-CTA kernel (gemm_bf16_nt_kernel).  The default is the persistent kernel further
// down: one CTA per SM walks 128 x 128/256 tiles in groups of eight tile rows, the accumulator is
// double-buffered in TMEM so that the epilogue of one tile overlaps the MMAs of the next, the output leaves
// through swizzled staging boxes and TMA stores, and operands may be K-major or MN-major (NT, NN, TN
// products).  Its epilogue mode is a template parameter: bias + activation; pre-activation and GELU in one
// pass; product times GELU'(saved pre-activation); column sums and sums of squares of the output for a
// following BatchNorm.
//
// The reference has no GEMM of its own (its models call cuBLAS through PyTorch,
// examples/pytorch_benchmark.py:76-100); this kernel is what the models of this library use for
// their linear layers and 1x1 convolutions.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <climits>
#include <cstdlib>
#include <string>
#include <type_traits>

#include "gemm_tcgen05.h"
#include "tcgen05_common.cuh"
#include "comm_kernels.h"

namespace bfb {
namespace {

using namespace t5;

constexpr int BM = 128, BN = 128, BK = 64;
constexpr int kStages = 6;
constexpr int kUmmaK = 16;
constexpr int kThreads = 192;
constexpr uint32_t kStageBytesA = BM * BK * 2;
constexpr uint32_t kStageBytesB = BN * BK * 2;
constexpr uint32_t kStageBytes = kStageBytesA + kStageBytesB;
constexpr uint32_t kTmemCols = 128;
constexpr size_t kSmemBytes = 1024 /*alignment slack*/ + size_t(kStages) * kStageBytes + 256 /*barriers*/;

// Instruction descriptor: D=f32, A=B=bf16, both K-major, N=128, M=128.
constexpr uint32_t kInstrDesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(BM >> 4) << 24);

__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(kInstrDesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float act_fn(float x, int act) {
  if (act == kActRelu) return fmaxf(x, 0.f);
  if (act == kActGeluTanh) {
    const float c = 0.7978845608028654f;
    return 0.5f * x * (1.f + tanhf(c * (x + 0.044715f * x * x * x)));
  }
  return x;
}

// Order in which the persistent kernel walks the output tiles: groups of eight tile rows, inside a group the
// row index runs fastest.  The CTAs that are resident together then share 8 A panels and about tiles/8 B panels
// instead of one or two A panels and every B panel, so a B matrix larger than L2 (a 50 304-column classifier)
// is streamed from DRAM once per group of eight tile rows rather than once per tile row.
__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int kGroup = 8;
  const int per_group = kGroup * tiles_n;
  const int gid = tile / per_group;
  const int first = gid * kGroup;
  const int rows = min(tiles_m - first, kGroup);
  const int r = tile - gid * per_group;
  tm = first + r % rows;
  tn = r / rows;
}

// two floats in one 64-bit register, the operand form of the packed f32x2 instructions
__device__ __forceinline__ unsigned long long pack_f32x2(uint32_t lo_bits, uint32_t hi_bits) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo_bits), "r"(hi_bits));
  return v;
}
__device__ __forceinline__ void unpack_f32x2(unsigned long long v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}

// d/dx of the tanh-approximated GELU of act_fn
__device__ __forceinline__ float gelu_tanh_grad(float x) {
  const float c = 0.7978845608028654f;
  const float u = c * (x + 0.044715f * x * x * x);
  const float t = tanhf(u);
  return 0.5f * (1.f + t) + 0.5f * x * (1.f - t * t) * c * (1.f + 3.f * 0.044715f * x * x);
}

// Gates of a gated feed-forward block, act(x) = x * sigmoid(w(x)): w = x (kActSilu), or w = 2 sqrt(2/pi) (x + 0.044715 x^3)
// (kActGeluTanh: (1 + tanh z) / 2 = sigmoid(2 z), which keeps its relative accuracy where tanh is near -1).
// Returns act(x); grad receives act'(x) = s + x s (1 - s) w'(x).
__device__ __forceinline__ float gate_fn(float x, int act, float* grad) {
  float w = x, dw = 1.f;
  if (act == kActGeluTanh) {
    const float c = 1.5957691216057308f;
    w = c * (x + 0.044715f * x * x * x);
    dw = c * (1.f + 0.134145f * x * x);
  }
  const float s = __fdividef(1.f, 1.f + __expf(-w));
  const float y = x * s;
  if (grad != nullptr) *grad = s + y * (1.f - s) * dw;
  return y;
}
// What a gated block keeps for its backward pass, 16 bits each: act(g) and u act'(g), the factors of dH in dU and dG.  Their format
// has a sign, six bits of exponent (2^-36 to 2^27; smaller values become zero, what is larger, infinite or not a number becomes
// the largest code, which reads as NaN) and nine of mantissa: each is off by at most 2^-10 of itself.  Kept in bf16, their
// rounding, that of dG and dU and that of the gradients themselves made the gradients of the input and of the gate and up
// weights 1.8 times as far from exact ones as the last rounding alone does; now it is 1.4 times.  Scaled by 2^-90 the exponent
// of an fp32 number in this range has two leading zeros.
constexpr float kFactorScale = 8.077935669463161e-28f;                         // 2^-90
__device__ __forceinline__ uint32_t pack_factors(float lo, float hi) {
  const uint32_t a = __float_as_uint(lo * kFactorScale), b = __float_as_uint(hi * kFactorScale);
  const uint32_t ma = min((a & 0x7fffffffu) + 0x2000u, 0x1fffffffu) >> 14, mb = min((b & 0x7fffffffu) + 0x2000u, 0x1fffffffu) >> 14;
  return ((a >> 16) & 0x8000u) | ma | (b & 0x80000000u) | (mb << 16);
}
// The factors in a word.  Their scale is taken off here and not with dH, which it would make infinite from 2^38 on.
constexpr float kFactorUnscale = 1.2379400392853803e27f;                       // 2^90
__device__ __forceinline__ float2 unpack_factors(uint32_t w) {
  return make_float2(__uint_as_float(((w << 16) & 0x80000000u) | ((w << 14) & 0x1fffc000u)) * kFactorUnscale,
                     __uint_as_float((w & 0x80000000u) | ((w >> 2) & 0x1fffc000u)) * kFactorUnscale);
}
constexpr uint32_t kFactorNan = 0x7fffu;

// eight floats as bf16, 16 bytes
__device__ __forceinline__ uint4 pack8(const float* v) {
  uint4 pk;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  return pk;
}

__global__ void __launch_bounds__(kThreads, 1)
gemm_bf16_nt_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ bias, int M, int N, int K,
                    int act, unsigned int* __restrict__ status) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_a = smem;
  unsigned char* stage_b = smem + size_t(kStages) * kStageBytesA;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + size_t(kStages) * kStageBytes);
  // bars[0..S): full, bars[S..2S): empty, bars[2S]: accumulator complete
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * BM;
  const int n0 = blockIdx.x * BN;
  const int num_kb = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    failed_s = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bars[s]), 1);
      mbar_init(smem_u32(&bars[kStages + s]), 1);
    }
    mbar_init(smem_u32(&bars[2 * kStages]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_s;

  int armed = 0;  // producer: stages whose TMA copies were issued (for the failure path)
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < num_kb; ++kb) {
        const int s = kb % kStages;
        const uint32_t parity = ((kb / kStages) & 1) ^ 1;
        if (!mbar_wait(smem_u32(&bars[kStages + s]), parity, failed)) break;
        const uint32_t full = smem_u32(&bars[s]);
        mbar_expect_tx(full, kStageBytes);
        tma_load_2d(smem_u32(stage_a + size_t(s) * kStageBytesA), &map_a, full, kb * BK, m0);
        tma_load_2d(smem_u32(stage_b + size_t(s) * kStageBytesB), &map_b, full, kb * BK, n0);
        armed = kb + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int kb = 0; kb < num_kb; ++kb) {
        const int s = kb % kStages;
        const uint32_t parity = (kb / kStages) & 1;
        if (!mbar_wait(smem_u32(&bars[s]), parity, failed)) break;
        // (no tcgen05 fence here: the data arrived through the async proxy and its mbarrier; a fence after every
        // stage wait makes the issuing thread wait out the MMAs in flight: 150 instead of 48 cycles per 128x64x16 MMA)
        const uint64_t adesc = make_desc(smem_u32(stage_a + size_t(s) * kStageBytesA));
        const uint64_t bdesc = make_desc(smem_u32(stage_b + size_t(s) * kStageBytesB));
#pragma unroll
        for (int k = 0; k < BK / kUmmaK; ++k) {
          // advancing by 16 bf16 = 32 bytes inside the swizzle atom = +2 in the 16-byte address field
          umma_bf16(tmem_base, adesc + uint64_t(2 * k), bdesc + uint64_t(2 * k), (kb | k) != 0 ? 1u : 0u);
        }
        umma_commit(smem_u32(&bars[kStages + s]));   // frees the stage when these MMAs have read it
      }
      if (!*failed) umma_commit(smem_u32(&bars[2 * kStages]));  // accumulator complete
    }
  } else {
    // Epilogue warps 2..5: TMEM lane group = warp % 4.
    const int q = warp & 3;
    const bool ok = mbar_wait(smem_u32(&bars[2 * kStages]), 0, failed);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (ok) {
      const int m = m0 + q * 32 + lane;
      const bool vec_ok = (N % 8) == 0;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tmem_base + (uint32_t(q * 32) << 16) + uint32_t(c * 32), r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        const int nbase = n0 + c * 32;
        if (m < M && nbase < N) {
          __nv_bfloat16* dst = out + size_t(m) * N + nbase;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = nbase + j * 8;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float x = __uint_as_float(r[j * 8 + i]);
              if (bias != nullptr && n + i < N) x += __bfloat162float(bias[n + i]);
              v[i] = act_fn(x, act);
            }
            if (vec_ok && n + 8 <= N) {
              uint4 pk;
              __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
              for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
              *reinterpret_cast<uint4*>(dst + j * 8) = pk;
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (n + i < N) dst[j * 8 + i] = __float2bfloat16_rn(v[i]);
            }
          }
        }
      }
    }
  }
  // Tear-down. On the failure path the producer first waits (bounded) for the copies it issued.
  if (warp == 0 && lane == 0 && *failed) {
    const int first = armed > kStages ? armed - kStages : 0;
    for (int kb = first; kb < armed; ++kb) {
      const unsigned long long t0 = now_ns();
      while (!mbar_try(smem_u32(&bars[kb % kStages]), (kb / kStages) & 1) && now_ns() - t0 < kWaitLimitNs) {}
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
  if (threadIdx.x == 0 && failed_s && status != nullptr) atomicExch(status, 1u);
}


// ------------------------------------------------------------------------------------------ //
// Two-SM variant (tcgen05 cta_group::2): a cluster of two CTAs owns a 256 x 256 output tile.  Each CTA loads its
// own 128 rows of A and HALF of B (128 of the 256 columns) per ring stage; one thread of the leader CTA issues
// 256 x 256 x 16 MMAs that read A from each CTA's own shared memory and both halves of B, and leave 128 rows of
// the accumulator in each CTA's tensor memory.  Per SM and MMA that is 4 KB of A and 4 KB of B out of shared
// memory instead of 4 + 8: a 128 x 256 tile on one SM reads (and TMA writes) more than the 128 bytes per clock an
// SM's shared memory has, which is what held the one-SM kernel at 0.84 of the library on large products.
//   loads     : cp.async.bulk.tensor with .cta_group::2 (no multicast): data lands in the issuing CTA, the byte
//               count is signalled on the LEADER's full barrier, which expects both CTAs' bytes;
//   empty/acc : tcgen05.commit.cta_group::2 ... multicast::cluster arrives on the barrier at the same offset in
//               both CTAs (ring slots free, accumulator complete);
//   acc_empty : the eight epilogue warps of both CTAs arrive on the leader's barrier (count 16, remote arrive).
// Every wait is bounded.  It is the PAIR mode of the persistent kernel below, so every operand mode and epilogue has it.
// ------------------------------------------------------------------------------------------ //
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(leader_bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"((unsigned short)3)
      : "memory");
}

// ------------------------------------------------------------------------------------------ //
// Persistent variant: one CTA per SM walks over output tiles of 128 x BN_; the accumulator is
// double-buffered in tensor memory (2 x BN_ columns) so that the epilogue of tile i runs while
// the MMAs of tile i+1 are issued.  Ring-stage and accumulator hand-over use four kinds of
// mbarriers: full/empty per smem stage, acc_full/acc_empty per accumulator buffer.
// The epilogue leaves through shared memory: every epilogue warp converts [32 rows x 64 columns]
// of its accumulator quarter to bf16, writes them in the 128-byte-swizzle layout and hands the box
// to a TMA store (two boxes per warp in flight), so global memory sees full 128-byte rows and the
// tile edges are clipped by the tensor map.  Row pitches that TMA cannot address (N % 8 != 0)
// take the direct-store epilogue.
// ------------------------------------------------------------------------------------------ //
template <int BN_, int EPI = 0, int PAIR = 0>
struct PersistentCfg {
  // PAIR: two CTAs of a cluster share a (2 * BM) x BN_ tile (tcgen05 cta_group::2); each holds its 128 rows of A and
  // half of B, so a stage is smaller and the ring deeper.
  // the column-statistics epilogue gives one ring stage up for its per-warp partial sums
  // PAIR runs eight epilogue warps, two per 32-lane quarter of tensor memory, each on half of the tile's columns:
  // with a reduction of 1024 the main loop of a 256 x 256 tile takes 4.3 us, and four warps that convert, activate
  // and store 256 columns each (and wait for their own TMA stores and auxiliary loads in turn) took three times
  // that on the GELU epilogues.  Their staging boxes cost one of the six ring stages.
  static constexpr int kEpiWarps = PAIR ? 8 : 4;
  static constexpr int kThreadsP = 64 + 32 * kEpiWarps;
  // the gate's gradient gives one up for a third pair of boxes per epilogue warp, so that two chunks of kept factors are on their
  // way (dH of 8192 x 1024 x 2752 61 -> 55 us; with a reduction of 2048, which would rather have the stage, 16384 rows and 5504
  // columns 308 -> 317 us); tiles of 128 columns on pairs have room for both
  static constexpr int kStagesP =
      (PAIR ? 5 : ((BN_ == 256) ? 4 : 6)) - (EPI == kEpiColumnStats || (EPI == kEpiGatedGrad && !(PAIR && BN_ == 128)) ? 1 : 0);
  static constexpr int kPre = EPI == kEpiGatedGrad ? 3 : 2;    // pairs of boxes
  // per epilogue warp: BN_ column sums and BN_ sums of squares
  static constexpr uint32_t kStatBytes = EPI == kEpiColumnStats ? kEpiWarps * 2 * BN_ * 4 : 0;
  static constexpr int kRowsB = PAIR ? BN_ / 2 : BN_;          // rows (output columns) of B one CTA loads
  // kEpiGated: the accumulator holds BN_ / 2 columns of the gate product and the same columns of the up product beside
  // them, and BN_ / 2 output columns leave
  static constexpr int kTileN = EPI == kEpiGated ? BN_ / 2 : BN_;
  static constexpr int kTileM = PAIR ? 2 * BM : BM;
  static constexpr uint32_t kBytesA = BM * BK * 2;
  static constexpr uint32_t kBytesB = kRowsB * BK * 2;
  static constexpr uint32_t kBytesStage = kBytesA + kBytesB;
  static constexpr uint32_t kCols = 2 * BN_;
  // output staging: per epilogue warp two [32 rows x 64 columns] bf16 boxes (4 KiB each, 1024-byte aligned)
  static constexpr uint32_t kBytesOutBox = 32 * 64 * 2;
  static constexpr uint32_t kBytesOutWarp = kPre * kBytesOutBox;
  static constexpr uint32_t kBytesOut = kEpiWarps * kBytesOutWarp;
  static constexpr uint32_t kBytesBars = EPI == kEpiGatedGrad ? 512 : 256;
  static constexpr size_t kSmem = 1024 + size_t(kStagesP) * kBytesStage + kBytesOut + kBytesBars + kStatBytes;
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN_ >> 3) << 17) | (uint32_t(kTileM >> 4) << 24);
};

// BMODE 0: B is [N, K] row-major (K-major operand).  BMODE 1: B is [K, N] row-major and is consumed as an
// MN-major operand: every ring stage holds BN_/64 boxes of [64 K-rows x 64 N-columns] (8 KiB each, 128-byte
// swizzle); the descriptor's leading-dimension stride is the distance between boxes, its stride-dimension
// stride the 1024 bytes between groups of eight K-rows, and one MMA step advances 16 rows = 2048 bytes.
// AMODE 1: A is given as [K, M] row-major (the transposed product dY^T * X of a weight gradient) and is
// consumed MN-major in the same way: two boxes of [64 K-rows x 64 M-columns] per stage, bit 15 of the
// instruction descriptor.
// EPI (GemmEpi) is a template parameter so that the plain epilogue keeps its small register footprint.
// PAIR 1: launched as clusters of two CTAs (see the two-SM notes above): loads signal the
// leader's full barrier, commits are multicast to both CTAs, the leader's MMA thread issues cta_group::2 MMAs and
// waits for the epilogue warps of both CTAs.
template <int BN_, int BMODE = 0, int AMODE = 0, int EPI = 0, int PAIR = 0>
__global__ void __launch_bounds__((PersistentCfg<BN_, EPI, PAIR>::kThreadsP), 1)
gemm_bf16_nt_persistent_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                               const __grid_constant__ CUtensorMap map_c, __nv_bfloat16* __restrict__ out,
                               const __nv_bfloat16* __restrict__ bias, int M, int N, int K, int act, int tma_out,
                               unsigned int* __restrict__ status, const __grid_constant__ CUtensorMap map_aux,
                               const __nv_bfloat16* __restrict__ aux_in, float* __restrict__ col_stats,
                               const __grid_constant__ CUtensorMap map_b2, const __grid_constant__ CUtensorMap map_aux2) {
  using Cfg = PersistentCfg<BN_, EPI, PAIR>;
  constexpr int S = Cfg::kStagesP;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_a = smem;
  unsigned char* stage_b = smem + size_t(S) * Cfg::kBytesA;
  unsigned char* stage_out = smem + size_t(S) * Cfg::kBytesStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_out + Cfg::kBytesOut);
  // bars[0..S): full, [S..2S): empty, [2S..2S+2): acc_full, [2S+2..2S+4): acc_empty
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int tiles_n = (N + Cfg::kTileN - 1) / Cfg::kTileN;
  const int tiles_m = (M + Cfg::kTileM - 1) / Cfg::kTileM;
  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (K + BK - 1) / BK;
  const int first_tile = PAIR ? int(blockIdx.x >> 1) : int(blockIdx.x);
  const int tile_step = PAIR ? int(gridDim.x >> 1) : int(gridDim.x);

  if (threadIdx.x == 0) {
    failed_s = 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&bars[s]), 1);
      mbar_init(smem_u32(&bars[S + s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bars[2 * S + a]), 1);        // one tcgen05.commit
      mbar_init(smem_u32(&bars[2 * S + 2 + a]), (PAIR ? 2 : 1) * Cfg::kEpiWarps);    // one arrive per epilogue warp (of both CTAs)
    }
    if (EPI == kEpiGatedGrad)
      for (int a = 0; a < Cfg::kPre * Cfg::kEpiWarps; ++a) mbar_init(smem_u32(&bars[2 * S + 4 + a]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (PAIR) {
    // nobody signals a peer's barrier before the peer has initialised it
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (EPI == kEpiGatedGrad) let_next_kernel_start();
  const uint32_t tmem_base = tmem_base_s;

  int armed = 0;
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
        int tm, tn;
        tile_coords(tile, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * Cfg::kTileM + int(rank) * BM;
        // PAIR: this CTA's half of the tile's columns; with two B matrices the leader loads the gate's, the other the up's
        const int n0 = tn * Cfg::kTileN + (EPI == kEpiGated ? 0 : int(rank) * Cfg::kRowsB);
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % S;
          if (!mbar_wait(smem_u32(&bars[S + s]), ((it / S) & 1) ^ 1, failed)) { ok = false; break; }
          // PAIR: the leader's barrier counts the bytes of both CTAs; the leader arms it
          if (leader) mbar_expect_tx(smem_u32(&bars[s]), (PAIR ? 2u : 1u) * Cfg::kBytesStage);
          const uint32_t full = PAIR ? mapa_u32(smem_u32(&bars[s]), 0u) : smem_u32(&bars[s]);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if (PAIR) tma_load_2d_pair(dst, map, full, x, y);
            else tma_load_2d(dst, map, full, x, y);
          };
          if (AMODE == 0) {
            load(smem_u32(stage_a + size_t(s) * Cfg::kBytesA), &map_a, kb * BK, m0);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j)
              load(smem_u32(stage_a + size_t(s) * Cfg::kBytesA + size_t(j) * 8192), &map_a, m0 + j * 64, kb * BK);
          }
          if (EPI == kEpiGated) {
            const uint32_t dst = smem_u32(stage_b + size_t(s) * Cfg::kBytesB);
            if (PAIR) {
              load(dst, leader ? &map_b : &map_b2, kb * BK, n0);
            } else {
              load(dst, &map_b, kb * BK, n0);
              load(dst + (BN_ / 2) * BK * 2, &map_b2, kb * BK, n0);
            }
          } else if (BMODE == 0) {
            load(smem_u32(stage_b + size_t(s) * Cfg::kBytesB), &map_b, kb * BK, n0);
          } else {
#pragma unroll
            for (int j = 0; j < Cfg::kRowsB / 64; ++j)
              load(smem_u32(stage_b + size_t(s) * Cfg::kBytesB + size_t(j) * 8192), &map_b, n0 + j * 64, kb * BK);
          }
          armed = it + 1;
        }
      }
    }
  } else if (warp == 1) {
    // the whole warp walks along, one elected lane issues: its descriptors then stay in uniform registers (see elect_one)
    if (leader) {
      int it = 0, local = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++local) {
        const int acc = local & 1;
        // the epilogue (of both CTAs) must have drained this accumulator buffer (tile local-2)
        if (!(PAIR ? mbar_wait_cluster(smem_u32(&bars[2 * S + 2 + acc]), ((local >> 1) & 1) ^ 1, failed)
                   : mbar_wait(smem_u32(&bars[2 * S + 2 + acc]), ((local >> 1) & 1) ^ 1, failed))) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tmem_d = tmem_base + uint32_t(acc * BN_);
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % S;
          if (!mbar_wait(smem_u32(&bars[s]), (it / S) & 1, failed)) { ok = false; break; }
          // (no tcgen05 fence here: the data arrived through the async proxy and its mbarrier; a fence after every
          // stage wait makes the issuing thread wait out the MMAs in flight: 150 instead of 48 cycles per 128x64x16 MMA)
          const uint32_t a_addr = smem_u32(stage_a + size_t(s) * Cfg::kBytesA);
          const uint64_t adesc = AMODE == 0 ? make_desc(a_addr) : make_desc_mn(a_addr, 8192, 1024);
          const uint32_t b_addr = smem_u32(stage_b + size_t(s) * Cfg::kBytesB);
          const uint64_t bdesc = BMODE == 0 ? make_desc(b_addr) : make_desc_mn(b_addr, 8192, 1024);
          // MN-major operands: bits 15 (A) and 16 (B) of the instruction descriptor; 16 K-rows of 128 bytes per MMA step
          constexpr uint32_t idesc = Cfg::kIdesc | (AMODE != 0 ? (1u << 15) : 0u) | (BMODE != 0 ? (1u << 16) : 0u);
          constexpr uint64_t a_step = AMODE == 0 ? 2 : (16 * 128) >> 4;
          constexpr uint64_t b_step = BMODE == 0 ? 2 : (16 * 128) >> 4;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / kUmmaK; ++k) {
              if (PAIR) {
                asm volatile(
                    "{\n\t.reg .pred p;\n\t"
                    "setp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
                    ::"r"(tmem_d), "l"(adesc + a_step * uint64_t(k)), "l"(bdesc + b_step * uint64_t(k)), "r"(idesc),
                      "r"((kb | k) != 0 ? 1u : 0u), "r"(0u)
                    : "memory");
              } else {
                asm volatile(
                    "{\n\t.reg .pred p;\n\t"
                    "setp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                    ::"r"(tmem_d), "l"(adesc + a_step * uint64_t(k)), "l"(bdesc + b_step * uint64_t(k)), "r"(idesc),
                      "r"((kb | k) != 0 ? 1u : 0u)
                    : "memory");
              }
            }
            if (PAIR) umma_commit_pair(smem_u32(&bars[S + s]));
            else umma_commit(smem_u32(&bars[S + s]));
          }
          __syncwarp();
        }
        if (ok && elect_one()) {
          if (PAIR) umma_commit_pair(smem_u32(&bars[2 * S + acc]));
          else umma_commit(smem_u32(&bars[2 * S + acc]));
        }
        __syncwarp();
      }
    }
  } else {
    const int q = warp & 3;                // the quarter of tensor memory (32 lanes = 32 rows) this warp can read
    const int ew = warp - 2;               // epilogue warp index
    // eight warps: warps 2-5 take the first half of the columns, warps 6-9 the second
    constexpr int kChunks = Cfg::kTileN / 64;
    constexpr int kChunksW = Cfg::kEpiWarps == 8 ? kChunks / 2 : kChunks;
    const int c_first = Cfg::kEpiWarps == 8 ? (ew >> 2) * kChunksW : 0;
    const bool vec_ok = (N % 8) == 0;
    unsigned char* my_out = stage_out + size_t(ew) * Cfg::kBytesOutWarp;
    int local = 0;
    int boxes = 0;                       // TMA stores issued by this warp
    // kEpiColumnStats: this warp's partial column sums [BN_] and sums of squares [BN_] of the current column
    // block live in shared memory (lanes 0-7 each own eight columns of every 64-column chunk, so no atomics)
    // and go to col_stats with vector reductions when the column block changes and at the end: adding every
    // box to global memory directly serialises thousands of reductions per address.
    float* wstat = reinterpret_cast<float*>(stage_out + Cfg::kBytesOut + Cfg::kBytesBars) + (EPI == kEpiColumnStats ? ew * 2 * BN_ : 0);
    int stat_n0 = -1;
    auto flush_stats = [&]() {
      if (stat_n0 >= 0 && lane < 8) {
#pragma unroll 1
        for (int c = c_first; c < c_first + kChunksW; ++c) {
          const int col = c * 64 + lane * 8;
          const int n = stat_n0 + col;
          float4* ws = reinterpret_cast<float4*>(wstat + col);
          float4* wq = reinterpret_cast<float4*>(wstat + BN_ + col);
          if (n < N) {                   // N is a multiple of 8 in this mode: the whole group is inside
            atomicAdd(reinterpret_cast<float4*>(col_stats + n), ws[0]);
            atomicAdd(reinterpret_cast<float4*>(col_stats + n) + 1, ws[1]);
            atomicAdd(reinterpret_cast<float4*>(col_stats + N + n), wq[0]);
            atomicAdd(reinterpret_cast<float4*>(col_stats + N + n) + 1, wq[1]);
          }
          ws[0] = ws[1] = wq[0] = wq[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    };
    if constexpr (EPI == kEpiColumnStats) {
      for (int i = lane; i < 2 * BN_; i += 32) wstat[i] = 0.f;
      __syncwarp();
    }
    // kEpiGatedGrad: the kept factors come through TMA boxes of 32 rows x 32 columns, two chunks ahead, into three sets of a box for
    // each per warp; dU and dG replace them there and leave from there.  (Read by the threads row by row, 32 sectors per load,
    // the epilogue took four times as long as the main loop of a reduction of 1024.)
    constexpr int kParts = Cfg::kTileN / 32 / (Cfg::kEpiWarps == 8 ? 2 : 1);
    const int part_first = Cfg::kEpiWarps == 8 ? (ew >> 2) * kParts : 0;
    int pre_tile = first_tile, pre_part = part_first, loaded = 0, used = 0;
    auto pre_bar = [&](int set) { return smem_u32(&bars[2 * S + 4 + ew * Cfg::kPre + set]); };
    auto prefetch = [&]() {
      for (; pre_tile < num_tiles; pre_tile += tile_step, pre_part = part_first) {
        int tm, tn;
        tile_coords(pre_tile, tiles_m, tiles_n, tm, tn);
        const int row = tm * Cfg::kTileM + int(rank) * BM + q * 32, col = tn * Cfg::kTileN + pre_part * 32;
        if (pre_part == part_first + kParts || row >= M || col >= N) continue;
        if (lane == 0) {
          const uint32_t bar = pre_bar(loaded % Cfg::kPre), dst = smem_u32(my_out) + (loaded % Cfg::kPre) * 4096u;
          mbar_expect_tx(bar, 4096);
          tma_load_2d(dst, &map_b2, bar, col, row);
          tma_load_2d(dst + 2048, &map_aux2, bar, col, row);
        }
        ++loaded;
        ++pre_part;
        return;
      }
    };
    if constexpr (EPI == kEpiGatedGrad) {
#pragma unroll 1
      for (int i = 1; i < Cfg::kPre; ++i) prefetch();
    }
    for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++local) {
      const int acc = local & 1;
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, tm, tn);
      const int m0 = tm * Cfg::kTileM + int(rank) * BM;         // this CTA's 128 rows, all BN_ columns
      const int n0 = tn * Cfg::kTileN;
      if (!mbar_wait(smem_u32(&bars[2 * S + acc]), (local >> 1) & 1, failed)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int m = m0 + q * 32 + lane;
      if constexpr (EPI == kEpiColumnStats) {
        if (n0 != stat_n0) {
          flush_stats();
          stat_n0 = n0;
        }
      }
      if constexpr (EPI == kEpiGated) {
        // h = act(g) u from the fp32 accumulators; act(g) and u act'(g) leave too when tma_out is 2.  Boxes of 32 rows x 32 columns,
        // one for each of the three per warp: they are written when the chunk is computed, so their last stores had that long
        // to be read (boxes of 64 columns in turn in two buffers: 93 instead of 80 us for 8192 x 1024 x 2752).
#pragma unroll 1
        for (int c = part_first; c < part_first + kParts; ++c) {
          const int nbase = n0 + c * 32;
          if (nbase >= N || m0 + q * 32 >= M) break;           // warp-uniform
          const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * BN_ + c * 32);
          uint32_t g[32], u[32], f[16], d[16];
          tmem_ld32(taddr, g);
          tmem_ld32(taddr + BN_ / 2, u);
          tmem_wait_ld();
          tie32(g);
          tie32(u);
          auto put = [&](int box, const uint32_t* v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              int off = lane * 64 + j * 16;
              off ^= ((off >> 7) & 3) << 4;                    // 64-byte swizzle
              *reinterpret_cast<uint4*>(my_out + box * 2048 + off) = make_uint4(v[j * 4], v[j * 4 + 1], v[j * 4 + 2], v[j * 4 + 3]);
            }
          };
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float s0, s1;
            const float a0 = gate_fn(__uint_as_float(g[2 * i]), act, &s0), a1 = gate_fn(__uint_as_float(g[2 * i + 1]), act, &s1);
            const float u0 = __uint_as_float(u[2 * i]), u1 = __uint_as_float(u[2 * i + 1]);
            const __nv_bfloat162 p = __floats2bfloat162_rn(a0 * u0, a1 * u1);
            if (tma_out == 2) {
              f[i] = pack_factors(a0, a1);
              d[i] = pack_factors(u0 * s0, u1 * s1);
            }
            g[i] = reinterpret_cast<const uint32_t&>(p);
          }
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
          put(0, g);
          if (tma_out == 2) {
            put(1, f);
            put(2, d);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_c, smem_u32(my_out), nbase, m0 + q * 32);
            if (tma_out == 2) {
              tma_store_2d(&map_aux, smem_u32(my_out + 2048), nbase, m0 + q * 32);
              tma_store_2d(&map_aux2, smem_u32(my_out + 4096), nbase, m0 + q * 32);
            }
            tma_store_commit();
          }
        }
      } else if constexpr (EPI == kEpiGatedGrad) {
        // accumulator = dH, times the kept factors:  dG = dH (u act'(g)) through map_c, dU = dH act(g) through map_aux
#pragma unroll 1
        for (int c = part_first; c < part_first + kParts; ++c) {
          const int nbase = n0 + c * 32;
          if (nbase >= N || m0 + q * 32 >= M) break;           // warp-uniform; prefetch() walks the same chunks
          uint32_t r[32];
          tmem_ld32(tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * BN_ + c * 32), r);
          unsigned char* box = my_out + (used % Cfg::kPre) * 4096;
          if (!mbar_wait(pre_bar(used % Cfg::kPre), (used / Cfg::kPre) & 1, failed)) {
            tmem_wait_ld();
            break;
          }
          tmem_wait_ld();
          tie32(r);
          uint4 dg[4], du[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            int off = lane * 64 + j * 16;
            off ^= ((off >> 7) & 3) << 4;                      // 64-byte swizzle
            const uint4 fv = *reinterpret_cast<const uint4*>(box + off), dv = *reinterpret_cast<const uint4*>(box + 2048 + off);
            const uint32_t f[4] = {fv.x, fv.y, fv.z, fv.w}, d[4] = {dv.x, dv.y, dv.z, dv.w};
            float a[8], b[8];
            uint32_t top = 0u;                                 // largest codes of the upper and lower halves
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              top = __vmaxu2(top, __vmaxu2(f[i] & 0x7fff7fffu, d[i] & 0x7fff7fffu));
              const float h0 = __uint_as_float(r[j * 8 + 2 * i]), h1 = __uint_as_float(r[j * 8 + 2 * i + 1]);
              const float2 x = unpack_factors(f[i]), y = unpack_factors(d[i]);
              b[2 * i] = h0 * x.x;
              b[2 * i + 1] = h1 * x.y;
              a[2 * i] = h0 * y.x;
              a[2 * i + 1] = h1 * y.y;
            }
            if ((top & 0xffffu) == kFactorNan || top >> 16 == kFactorNan) {       // rare
              const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if ((f[i] & 0x7fffu) == kFactorNan) b[2 * i] = nan;
                if ((f[i] >> 16 & 0x7fffu) == kFactorNan) b[2 * i + 1] = nan;
                if ((d[i] & 0x7fffu) == kFactorNan) a[2 * i] = nan;
                if ((d[i] >> 16 & 0x7fffu) == kFactorNan) a[2 * i + 1] = nan;
              }
            }
            dg[j] = pack8(a);
            du[j] = pack8(b);
          }
          if (lane == 0) tma_store_wait_read<0>();             // the other set has left: the next chunk may come in
          __syncwarp();
          prefetch();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            int off = lane * 64 + j * 16;
            off ^= ((off >> 7) & 3) << 4;
            *reinterpret_cast<uint4*>(box + off) = dg[j];
            *reinterpret_cast<uint4*>(box + 2048 + off) = du[j];
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_c, smem_u32(box), nbase, m0 + q * 32);
            tma_store_2d(&map_aux, smem_u32(box + 2048), nbase, m0 + q * 32);
            tma_store_commit();
          }
          ++used;
        }
      } else if (tma_out) {
#pragma unroll 1
        for (int c = c_first; c < c_first + kChunksW; ++c) {
          const int nbase = n0 + c * 64;
          if (nbase >= N || m0 + q * 32 >= M) break;           // warp-uniform
          uint32_t r[64];
          const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * BN_ + c * 64);
          tmem_ld32(taddr, r);
          tmem_ld32(taddr + 32, r + 32);
          // the box written two stores ago must have been read out of shared memory
          if (lane == 0) tma_store_wait_read<1>();
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          __syncwarp();
          if constexpr (EPI == kEpiNone || EPI == kEpiColumnStats) {
            unsigned char* box = my_out + size_t(boxes & 1) * Cfg::kBytesOutBox;
            unsigned char* row = box + lane * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float x = __uint_as_float(r[j * 8 + i]);
                if (bias != nullptr) {
                  const int n = nbase + j * 8 + i;
                  x += n < N ? __bfloat162float(bias[n]) : 0.f;
                }
                v[i] = act_fn(x, act);
              }
              uint4 pk;
              __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
              for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
              *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) << 4)) = pk;      // 128-byte swizzle
            }
            if constexpr (EPI == kEpiColumnStats) {
              // Statistics of the staged (rounded) box: lane l reads the eight columns (l & 7)*8.. of rows
              // (l >> 3) + 4i back with 16-byte loads that follow the swizzle, sums them as packed float pairs, the
              // four row groups are folded with shuffles and eight lanes add the result to this warp's partial sums.
              // Rows past M hold exact zeros (zero-filled A rows, no bias, no activation).  The chunk loop stays
              // rolled: as straight-line code the epilogue ran out of the instruction cache.
              __syncwarp();
              unsigned long long s2[4] = {0ull, 0ull, 0ull, 0ull}, q2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int rr = (lane >> 3) + 4 * i;
                const uint4 wv = *reinterpret_cast<const uint4*>(box + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                const uint32_t w4[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const unsigned long long f = pack_f32x2(w4[k] << 16, w4[k] & 0xffff0000u);   // two bf16 -> two floats
                  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s2[k]) : "l"(f));
                  asm("fma.rn.f32x2 %0, %1, %1, %0;" : "+l"(q2[k]) : "l"(f));
                }
              }
              float v[16];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                unpack_f32x2(s2[k], v[2 * k], v[2 * k + 1]);
                unpack_f32x2(q2[k], v[8 + 2 * k], v[8 + 2 * k + 1]);
              }
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                v[k] += __shfl_xor_sync(0xffffffffu, v[k], 8);
                v[k] += __shfl_xor_sync(0xffffffffu, v[k], 16);
              }
              if (lane < 8) {
                float4* ws = reinterpret_cast<float4*>(wstat + c * 64 + lane * 8);
                float4* wq = reinterpret_cast<float4*>(wstat + BN_ + c * 64 + lane * 8);
                float4 t;
                t = ws[0]; t.x += v[0]; t.y += v[1]; t.z += v[2]; t.w += v[3]; ws[0] = t;
                t = ws[1]; t.x += v[4]; t.y += v[5]; t.z += v[6]; t.w += v[7]; ws[1] = t;
                t = wq[0]; t.x += v[8]; t.y += v[9]; t.z += v[10]; t.w += v[11]; wq[0] = t;
                t = wq[1]; t.x += v[12]; t.y += v[13]; t.z += v[14]; t.w += v[15]; wq[1] = t;
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&map_c, smem_u32(box), nbase, m0 + q * 32);
              tma_store_commit();
            }
            ++boxes;
          } else if constexpr (EPI == kEpiMulGeluGrad || EPI == kEpiAddAux) {
            // kEpiMulGeluGrad: out = accumulator * GELU'(aux), the backward of a fused Linear+GELU (aux = the saved
            // pre-activation).  kEpiAddAux: out = accumulator + aux (aux = a gradient that joins this one).
            unsigned char* box = my_out + size_t(boxes & 1) * Cfg::kBytesOutBox;
            unsigned char* row = box + lane * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint4 av = make_uint4(0u, 0u, 0u, 0u);
              if (m < M && nbase + j * 8 < N) av = __ldg(reinterpret_cast<const uint4*>(aux_in + size_t(m) * N + nbase + j * 8));
              const __nv_bfloat162* ah = reinterpret_cast<const __nv_bfloat162*>(&av);
              float v[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 t2 = __bfloat1622float2(ah[i]);
                if constexpr (EPI == kEpiAddAux) {
                  float b0 = 0.f, b1 = 0.f;
                  if (bias != nullptr) {                       // out = accumulator + bias + aux (a layer with a residual)
                    const int n = nbase + j * 8 + 2 * i;
                    b0 = n < N ? __bfloat162float(bias[n]) : 0.f;
                    b1 = n + 1 < N ? __bfloat162float(bias[n + 1]) : 0.f;
                  }
                  v[2 * i] = __uint_as_float(r[j * 8 + 2 * i]) + b0 + t2.x;
                  v[2 * i + 1] = __uint_as_float(r[j * 8 + 2 * i + 1]) + b1 + t2.y;
                } else {
                  v[2 * i] = __uint_as_float(r[j * 8 + 2 * i]) * gelu_tanh_grad(t2.x);
                  v[2 * i + 1] = __uint_as_float(r[j * 8 + 2 * i + 1]) * gelu_tanh_grad(t2.y);
                }
              }
              uint4 pk;
              __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
              for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
              *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) << 4)) = pk;      // 128-byte swizzle
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&map_c, smem_u32(box), nbase, m0 + q * 32);
              tma_store_commit();
            }
            ++boxes;
          } else {
            // kEpiStorePreact: two boxes leave per chunk, x = accumulator + bias through map_aux and act(x)
            // through map_c; both staging boxes are in use, so every earlier store must have been read
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            unsigned char* row_raw = my_out + lane * 128;
            unsigned char* row_act = my_out + Cfg::kBytesOutBox + lane * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                x[i] = __uint_as_float(r[j * 8 + i]);
                if (bias != nullptr) {
                  const int n = nbase + j * 8 + i;
                  x[i] += n < N ? __bfloat162float(bias[n]) : 0.f;
                }
              }
              uint4 pk_raw, pk_act;
              __nv_bfloat162* hr = reinterpret_cast<__nv_bfloat162*>(&pk_raw);
              __nv_bfloat162* ha = reinterpret_cast<__nv_bfloat162*>(&pk_act);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                hr[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                // the activation sees the rounded pre-activation, as a separate activation kernel would
                const float2 xr = __bfloat1622float2(hr[i]);
                ha[i] = __floats2bfloat162_rn(act_fn(xr.x, act), act_fn(xr.y, act));
              }
              const int off = (j ^ (lane & 7)) << 4;                                // 128-byte swizzle
              *reinterpret_cast<uint4*>(row_raw + off) = pk_raw;
              *reinterpret_cast<uint4*>(row_act + off) = pk_act;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&map_aux, smem_u32(my_out), nbase, m0 + q * 32);
              tma_store_2d(&map_c, smem_u32(my_out + Cfg::kBytesOutBox), nbase, m0 + q * 32);
              tma_store_commit();
            }
            boxes += 2;
          }
        }
      } else {
#pragma unroll 1
        for (int c = 2 * c_first; c < 2 * (c_first + kChunksW); ++c) {
          uint32_t r[32];
          tmem_ld32(tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * BN_ + c * 32), r);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const int nbase = n0 + c * 32;
          if (m < M && nbase < N) {
            __nv_bfloat16* dst = out + size_t(m) * N + nbase;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int n = nbase + j * 8;
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float x = __uint_as_float(r[j * 8 + i]);
                if (bias != nullptr && n + i < N) x += __bfloat162float(bias[n + i]);
                v[i] = act_fn(x, act);
              }
              if (vec_ok && n + 8 <= N) {
                uint4 pk;
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                *reinterpret_cast<uint4*>(dst + j * 8) = pk;
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (n + i < N) dst[j * 8 + i] = __float2bfloat16_rn(v[i]);
              }
            }
          }
        }
      }
      // hand the accumulator buffer back to the MMA warp
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(mapa_u32(smem_u32(&bars[2 * S + 2 + acc]), 0u));
        else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bars[2 * S + 2 + acc])) : "memory");
      }
    }
    if constexpr (EPI == kEpiColumnStats) flush_stats();
    // the stores of this warp must be complete before its shared memory goes away, and after a failure its loads too
    if (lane == 0) tma_store_wait_all();
    if constexpr (EPI == kEpiGatedGrad) {
      for (; used < loaded; ++used) {
        const unsigned long long t0 = now_ns();
        while (!mbar_try(pre_bar(used % Cfg::kPre), (used / Cfg::kPre) & 1) && now_ns() - t0 < kWaitLimitNs) {}
      }
    }
  }
  if (warp == 0 && lane == 0 && *failed && leader) {
    const int first = armed > S ? armed - S : 0;
    for (int it = first; it < armed; ++it) {
      const unsigned long long t0 = now_ns();
      while (!mbar_try(smem_u32(&bars[it % S]), (it / S) & 1) && now_ns() - t0 < kWaitLimitNs) {}
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (PAIR) {
    // neither CTA leaves (or frees tensor memory) while the other may still read its shared memory or signal it
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Cfg::kCols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Cfg::kCols) : "memory");
  }
  if (threadIdx.x == 0 && failed_s && status != nullptr) atomicExch(status, 1u);
}

// ------------------------------------------------------------------------------------------ //
// Up to three products in one launch of the two-SM kernel (256 x 256 tiles): the input gradient and both weight gradients of a
// gated block do not depend on one another, and as launches of their own each ends in a wave that leaves SM pairs idle (8192 x
// 1024 x 2752: 128, 88 and 44 tiles on 74 pairs, two, two and one wave, 68 + 91 + 50 us; together 161 us).  The tiles with the
// longest reductions come first, but for those that need nothing of the kernel before (the down projection's weight gradient
// does not need the gradient of the gate): they fill the SMs that its last wave leaves idle (1537 x 776 x 2056,
// whose dH has 63 tiles: 101 -> 99 us for the block).  B is [reduction, N] row-major in all of them; A is [M, reduction] or, for a
// weight gradient, [reduction, M].  The tile is the same for all sizes: a width of 776 takes four of 256, and the last one holds
// eight columns; narrower ones have not been tried in this launch.
// ------------------------------------------------------------------------------------------ //
constexpr int kMaxGroup = 3;
struct GroupProblem {
  int M, N, num_kb, tiles_m, tiles_n, first_item, a_mn, early;
};
struct GroupArgs {
  CUtensorMap a[kMaxGroup], b[kMaxGroup], c[kMaxGroup];
  GroupProblem p[kMaxGroup];
  int items;
};

__global__ void __launch_bounds__((PersistentCfg<256, kEpiNone, 1>::kThreadsP), 1)
gemm_bf16_group_kernel(const __grid_constant__ GroupArgs args, unsigned int* __restrict__ status) {
  using Cfg = PersistentCfg<256, kEpiNone, 1>;
  constexpr int S = Cfg::kStagesP;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_a = smem;
  unsigned char* stage_b = smem + size_t(S) * Cfg::kBytesA;
  unsigned char* stage_out = smem + size_t(S) * Cfg::kBytesStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_out + Cfg::kBytesOut);
  // bars[0..S): full, [S..2S): empty, [2S..2S+2): acc_full, [2S+2..2S+4): acc_empty
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int first = int(blockIdx.x >> 1), step = int(gridDim.x >> 1);
  // problem of an item and its tile
  auto locate = [&](int item, int& tm, int& tn) {
    int i = 0;
    while (i + 1 < kMaxGroup && item >= args.p[i + 1].first_item) ++i;
    tile_coords(item - args.p[i].first_item, args.p[i].tiles_m, args.p[i].tiles_n, tm, tn);
    return i;
  };

  if (threadIdx.x == 0) {
    failed_s = 0;
    for (int s = 0; s < 2 * S + 2; ++s) mbar_init(smem_u32(&bars[s]), 1);
    for (int a = 0; a < 2; ++a) mbar_init(smem_u32(&bars[2 * S + 2 + a]), 2 * Cfg::kEpiWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  // nobody signals a peer's barrier before the peer has initialised it
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;

  int armed = 0;
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true, waited = false;
      for (int item = first; item < args.items && ok; item += step) {
        int tm, tn;
        const int i = locate(item, tm, tn);
        if (!waited && args.p[i].early == 0) {
          wait_for_kernel_before();
          waited = true;
        }
        const int m0 = tm * Cfg::kTileM + int(rank) * BM, n0 = tn * 256 + int(rank) * Cfg::kRowsB;
        const bool a_mn = args.p[i].a_mn != 0;
        const int num_kb = args.p[i].num_kb;
        for (int kb = 0; kb < num_kb; ++kb, ++armed) {
          const int s = armed % S;
          ok = mbar_wait(smem_u32(&bars[S + s]), ((armed / S) & 1) ^ 1, failed);
          if (!ok) break;
          // the leader's barrier counts the bytes of both CTAs; the leader arms it
          if (leader) mbar_expect_tx(smem_u32(&bars[s]), 2u * Cfg::kBytesStage);
          const uint32_t full = mapa_u32(smem_u32(&bars[s]), 0u);
          const uint32_t a = smem_u32(stage_a + size_t(s) * Cfg::kBytesA), b = smem_u32(stage_b + size_t(s) * Cfg::kBytesB);
          if (a_mn) {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d_pair(a + j * 8192, &args.a[i], full, m0 + j * 64, kb * BK);
          } else {
            tma_load_2d_pair(a, &args.a[i], full, kb * BK, m0);
          }
#pragma unroll
          for (int j = 0; j < Cfg::kRowsB / 64; ++j) tma_load_2d_pair(b + j * 8192, &args.b[i], full, n0 + j * 64, kb * BK);
        }
      }
      if (!waited) wait_for_kernel_before();           // the end of this launch is the end of those before it
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      int it = 0, local = 0;
      bool ok = true;
      for (int item = first; item < args.items && ok; item += step, ++local) {
        int tm, tn;
        const int i = locate(item, tm, tn);
        const int acc = local & 1, num_kb = args.p[i].num_kb;
        const bool a_mn = args.p[i].a_mn != 0;
        // the epilogue of both CTAs must have drained this accumulator buffer
        ok = mbar_wait_cluster(smem_u32(&bars[2 * S + 2 + acc]), ((local >> 1) & 1) ^ 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint32_t tmem_d = tmem_base + uint32_t(acc * 256);
        // with the operand's layout known to the compiler: read from a table, it would leave the descriptors out of uniform registers
        auto reduce = [&](auto layout) {
          constexpr bool A_MN = decltype(layout)::value;
          constexpr uint32_t idesc = Cfg::kIdesc | (A_MN ? 1u << 15 : 0u) | (1u << 16);
          constexpr uint64_t a_step = A_MN ? (16 * 128) >> 4 : 2;
          for (int kb = 0; kb < num_kb; ++kb, ++it) {
            const int s = it % S;
            ok = mbar_wait(smem_u32(&bars[s]), (it / S) & 1, failed);
            if (!ok) break;
            const uint32_t a_addr = smem_u32(stage_a + size_t(s) * Cfg::kBytesA);
            const uint64_t adesc = A_MN ? make_desc_mn(a_addr, 8192, 1024) : make_desc(a_addr);
            const uint64_t bdesc = make_desc_mn(smem_u32(stage_b + size_t(s) * Cfg::kBytesB), 8192, 1024);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < BK / kUmmaK; ++k)
                asm volatile(
                    "{\n\t.reg .pred p;\n\t"
                    "setp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
                    ::"r"(tmem_d), "l"(adesc + a_step * uint64_t(k)), "l"(bdesc + uint64_t(128 * k)), "r"(idesc),
                      "r"((kb | k) != 0 ? 1u : 0u), "r"(0u)
                    : "memory");
              umma_commit_pair(smem_u32(&bars[S + s]));
              if (kb == num_kb - 1) umma_commit_pair(smem_u32(&bars[2 * S + acc]));
            }
            __syncwarp();
          }
        };
        if (a_mn) reduce(std::true_type());
        else reduce(std::false_type());
      }
    }
  } else {
    const int q = warp & 3, ew = warp - 2;             // quarter of tensor memory; two warps per quarter, half of the columns each
    unsigned char* my_out = stage_out + size_t(ew) * 2 * Cfg::kBytesOutBox;
    int local = 0, boxes = 0;
    for (int item = first; item < args.items; item += step, ++local) {
      int tm, tn;
      const int i = locate(item, tm, tn);
      const int acc = local & 1, M = args.p[i].M, N = args.p[i].N;
      const int m = tm * Cfg::kTileM + int(rank) * BM + q * 32, n0 = tn * 256 + (ew >> 2) * 128;
      if (!mbar_wait(smem_u32(&bars[2 * S + acc]), (local >> 1) & 1, failed)) break;
      fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        const int n = n0 + c * 64;
        if (n >= N || m >= M) break;                   // warp-uniform
        uint32_t r[64];
        const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(acc * 256 + (ew >> 2) * 128 + c * 64);
        tmem_ld32(taddr, r);
        tmem_ld32(taddr + 32, r + 32);
        if (lane == 0) tma_store_wait_read<1>();       // the box written two stores ago has been read
        tmem_wait_ld();
        tie32(r);
        tie32(r + 32);
        __syncwarp();
        unsigned char* box = my_out + size_t(boxes & 1) * Cfg::kBytesOutBox;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = pack8(reinterpret_cast<const float*>(r + j * 8));      // 128-byte swizzle
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&args.c[i], smem_u32(box), n, m);
          tma_store_commit();
        }
        ++boxes;
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&bars[2 * S + 2 + acc]), 0u));
    }
    if (lane == 0) tma_store_wait_all();               // before this shared memory goes away
    __syncwarp();
  }
  if (warp == 0 && lane == 0 && *failed && leader) {
    for (int it = armed > S ? armed - S : 0; it < armed; ++it) {
      const unsigned long long t0 = now_ns();
      while (!mbar_try(smem_u32(&bars[it % S]), (it / S) & 1) && now_ns() - t0 < kWaitLimitNs) {}
    }
  }
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  // neither CTA leaves (or frees tensor memory) while the other may still read its shared memory or signal it
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Cfg::kCols) : "memory");
  }
  if (threadIdx.x == 0 && failed_s && status != nullptr) atomicExch(status, 1u);
}

// ------------------------------------------------------------------------------------------ //
// Few rows: out[M, N] = x[M, K] w[N, K]^T with M <= 64, where the weights are what is read (8 x 1024 x 2752: 17 MB, 2.6 us from
// memory).  The roles are swapped - 128 weight rows are the M side of the MMA, NB >= M tokens its N side - so that a CTA reads
// weights only once, and a cluster of `split` CTAs shares a tile's reduction so that all SMs read: with 128 x 256 tiles of
// the kernel above the two products of that block kept 22 and 4 SMs busy and took 13 and 28 us.  The partial tiles meet in
// distributed shared memory; every CTA adds up the cluster's sums for its share of the tokens, in the order of the slices.
// GATED: 64 gate and 64 up rows make a tile, and act(g) u leaves (the factors for the backward pass too when `pre` is given).
// ------------------------------------------------------------------------------------------ //
template <int NB>
struct SkinnyCfg {
  static constexpr int kStagesS = 4;
  static constexpr uint32_t kBytesA = 128 * BK * 2;
  static constexpr uint32_t kBytesB = NB * BK * 2;
  static constexpr uint32_t kColsT = NB < 32 ? 32 : NB;
  static constexpr size_t kSmem = 1024 + kStagesS * (kBytesA + kBytesB) + NB * 128 * 4;
};

template <int NB, bool GATED>
__global__ void __launch_bounds__(192)
gemm_bf16_skinny_kernel(const __grid_constant__ CUtensorMap map_lo, const __grid_constant__ CUtensorMap map_hi,
                        const __grid_constant__ CUtensorMap map_x, __nv_bfloat16* __restrict__ out, unsigned short* __restrict__ pre,
                        const __nv_bfloat16* __restrict__ residual, const int M, const int N, const int num_kb, const int split, const int act,
                        unsigned int* __restrict__ status) {
  using Cfg = SkinnyCfg<NB>;
  constexpr int S = Cfg::kStagesS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_b = smem + S * Cfg::kBytesA;
  float* sums = reinterpret_cast<float*>(stage_b + S * Cfg::kBytesB);          // [token][weight row of the tile]
  __shared__ uint64_t bars[2 * S + 1];
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % split, n0 = (blockIdx.x / split) * (GATED ? 64 : 128);
  const int kb0 = rank * num_kb / split, kb1 = (rank + 1) * num_kb / split;

  if (threadIdx.x == 0) {
    failed_s = 0;
    for (int i = 0; i < 2 * S + 1; ++i) mbar_init(smem_u32(&bars[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kColsT) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_base_s;
  bool ok = true;
  if (GATED) let_next_kernel_start();
  if (warp == 0) {
    if (lane == 0) {
      int armed = 0;
      auto weights = [&](int i) {
        const int s = i % S, kb = kb0 + i;
        const uint32_t full = smem_u32(&bars[s]), a = smem_u32(smem + s * Cfg::kBytesA);
        mbar_expect_tx(full, Cfg::kBytesA + Cfg::kBytesB);
        tma_load_2d(a, &map_lo, full, kb * BK, n0);
        tma_load_2d(a + Cfg::kBytesA / 2, &map_hi, full, kb * BK, GATED ? n0 : n0 + 64);
      };
      // The down projection starts beside the product before it: what it reads of the weights at first does not depend on that,
      // everything else comes after the rows.
      const int early = GATED ? 0 : min(S, kb1 - kb0);
      for (int i = 0; i < early; ++i) weights(i);
      if (!GATED) wait_for_kernel_before();
      for (; armed < kb1 - kb0; ++armed) {
        const int s = armed % S;
        ok = mbar_wait(smem_u32(&bars[S + s]), ((armed / S) & 1) ^ 1, failed);
        if (!ok) break;
        if (armed >= early) weights(armed);
        tma_load_2d(smem_u32(stage_b + s * Cfg::kBytesB), &map_x, smem_u32(&bars[s]), (kb0 + armed) * BK, 0);
      }
      if (!ok || *failed) {
        for (int f = armed > S ? armed - S : 0; f < armed; ++f) {
          const unsigned long long t0 = now_ns();
          while (!mbar_try(smem_u32(&bars[f % S]), (f / S) & 1) && now_ns() - t0 < kWaitLimitNs) {}
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(NB >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    for (int i = 0; i < kb1 - kb0 && ok; ++i) {
      const int s = i % S;
      ok = mbar_wait(smem_u32(&bars[s]), (i / S) & 1, failed);
      if (!ok) break;
      if (elect_one()) {
        const uint64_t a = make_desc(smem_u32(smem + s * Cfg::kBytesA)), b = make_desc(smem_u32(stage_b + s * Cfg::kBytesB));
#pragma unroll
        for (int k = 0; k < BK / kUmmaK; ++k) umma_f16(tmem, a + uint64_t(2 * k), b + uint64_t(2 * k), idesc, (i | k) != 0 ? 1u : 0u);
        umma_commit(smem_u32(&bars[S + s]));
      }
      __syncwarp();
    }
    // also after a failure, so that tensor memory is not freed under a product
    if (elect_one()) umma_commit(smem_u32(&bars[2 * S]));
    __syncwarp();
    if (!ok) {
      const unsigned long long t0 = now_ns();
      while (!mbar_try(smem_u32(&bars[2 * S]), 0) && now_ns() - t0 < kWaitLimitNs) {}
    }
  } else {
    const int row = (warp & 3) * 32 + lane;
    ok = mbar_wait(smem_u32(&bars[2 * S]), 0, failed);
    fence_after_sync();
    const uint32_t t = tmem + (uint32_t((warp & 3) * 32) << 16);
#pragma unroll
    for (int c = 0; c < NB; c += 16) {
      uint32_t r[16];
      tmem_ld16(t + c, r);
      tmem_wait_ld();
      tie16(r);
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[(c + i) * 128 + row] = kb1 > kb0 ? __uint_as_float(r[i]) : 0.f;
    }
  }
  __syncwarp();
  if (split > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (warp >= 2 && ok) {
    const int e = threadIdx.x - 64;
    auto total = [&](int at) {
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = 0.f;
        if (c < split) {
          const uint32_t addr = mapa_u32(smem_u32(sums + at), c);
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[c]) : "r"(addr) : "memory");
        }
      }
#pragma unroll
      for (int c = 1; c < 8; ++c) v[0] += v[c];
      return v[0];
    };
    const int first = rank * (NB / split), last = min(first + NB / split, M);
    if (GATED) {
      const int f = n0 + (e & 63);
      for (int t = first + (e >> 6); t < last; t += 2) {
        const float g = total(t * 128 + (e & 63)), u = total(t * 128 + 64 + (e & 63));
        if (f < N) {
          float slope;
          const float a = gate_fn(g, act, &slope);
          out[size_t(t) * N + f] = __float2bfloat16_rn(a * u);
          if (pre != nullptr) {
            const uint32_t w = pack_factors(a, u * slope);
            pre[size_t(t) * (2 * N) + f] = static_cast<unsigned short>(w);
            pre[size_t(t) * (2 * N) + N + f] = static_cast<unsigned short>(w >> 16);
          }
        }
      }
    } else {
      const int n = n0 + e;
      for (int t = first; t < last; ++t) {
        const float v = total(t * 128 + e);
        if (n < N) out[size_t(t) * N + n] = __float2bfloat16_rn(v + (residual != nullptr ? __bfloat162float(residual[size_t(t) * N + n]) : 0.f));
      }
    }
  }
  __syncwarp();
  if (split > 1) {
    // nobody leaves while another may still read its shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kColsT) : "memory");
  }
  if (threadIdx.x == 0 && failed_s && status != nullptr) atomicExch(status, 1u);
}

// pitch: elements from row to row (0: the rows follow one another); boxes of 64 columns in the 128-byte swizzle, of 32 in the 64-byte one
bool MakeMap(CUtensorMap* map, const void* base, int rows, int cols /*K*/, int box_rows, long long pitch = 0, int box_cols = BK) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch != 0 ? pitch : cols) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  return EncodeTiled(map, 2, base, dims, strides, box, nullptr, box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

// Launches one instantiation of the persistent kernel on min(tiles, SMs) CTAs; PAIR: on clusters of two CTAs, one
// cluster per (2 * BM) x BN_ tile at a time.
template <int BN_, int BMODE, int AMODE, int EPI, int PAIR = 0>
cudaError_t LaunchPersistent(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_c,
                             const CUtensorMap& map_aux, __nv_bfloat16* out, const __nv_bfloat16* bias,
                             const __nv_bfloat16* aux_in, int M, int N, int K, int act, int tma_out, int sm_count,
                             unsigned int* status, cudaStream_t stream, float* col_stats = nullptr,
                             const CUtensorMap* map_b2 = nullptr, const CUtensorMap* map_aux2 = nullptr) {
  using Cfg = PersistentCfg<BN_, EPI, PAIR>;
  auto kernel = gemm_bf16_nt_persistent_kernel<BN_, BMODE, AMODE, EPI, PAIR>;
  // the permission for this much shared memory belongs to a device
  constexpr int kMaxDevices = 64;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr_set[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg::kSmem));
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr_set[dev] = true;
  }
  const int tiles = ((M + Cfg::kTileM - 1) / Cfg::kTileM) * ((N + Cfg::kTileN - 1) / Cfg::kTileN);
  const CUtensorMap& b2 = map_b2 != nullptr ? *map_b2 : map_b;
  const CUtensorMap& aux2 = map_aux2 != nullptr ? *map_aux2 : map_aux;
  if (!PAIR) {
    kernel<<<tiles < sm_count ? tiles : sm_count, Cfg::kThreadsP, Cfg::kSmem, stream>>>(map_a, map_b, map_c, out, bias, M, N, K, act,
                                                                               tma_out, status, map_aux, aux_in, col_stats, b2, aux2);
    return cudaSuccess;
  }
  const int pairs = tiles < sm_count / 2 ? tiles : sm_count / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(Cfg::kThreadsP);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_c, out, bias, M, N, K, act, tma_out, status, map_aux, aux_in, col_stats, b2,
                            aux2);
}

// Whether a plain product goes to the two-SM kernel: TMA-storable output, at least one full pair tile in each
// direction, enough tiles to occupy the pairs, and a reduction long enough for the main loop to matter (measured:
// +8 % at 8192^3, +11 % on 8192 x 50304 x 1024, +4-5 % on GPT-2's 8192 x {1024, 3072, 4096} x {1024, 4096}; with
// K <= 256 the product is bound by its epilogue and the larger tile is 20-30 % slower).
// BLUEFOG_B200_GEMM_PAIR=0 keeps everything on the one-SM kernel, =1 sends every eligible shape to the pair.
bool UsePair(int M, int N, int K, int sm_count) {
  static const int mode = [] {
    const char* v = std::getenv("BLUEFOG_B200_GEMM_PAIR");
    return v == nullptr ? -1 : std::atoi(v);
  }();
  if (mode == 0) return false;
  if ((N % 8) != 0 || N < 256 || M < 256) return false;
  if (mode > 0) return true;
  const long long tiles = (long long)((M + 255) / 256) * ((N + 255) / 256);
  return K >= 1024 && tiles >= sm_count / 4;
}

// Tiles for the products of a gated block, which come in every size: pairs of SMs with 256 columns per tile, or with 128, or single
// SMs.  A CTA's time for 64 elements of the reduction is that of its loads, 32 KB and 24 KB at about 50 bytes a cycle (the MMAs
// need 512 and 256 cycles); a tile more costs a whole wave.  The block of 1537 x 776 x 2056, three launches for its last three
// gradients: 154 us with UsePair's rule, 127 us with 256-column pairs throughout, 124 us with this one.
enum GemmTiles { kTilesSingle, kTilesPair256, kTilesPair128 };
GemmTiles PlanTiles(int M, int N, int K, int sm_count) {
  if (M <= 128 || N <= 128 || sm_count < 2) return kTilesSingle;
  const long long kb = (K + BK - 1) / BK, pairs = sm_count / 2, rows = (M + 255) / 256;
  auto cost = [&](long long columns, long long cycles) {
    const long long tiles = rows * ((N + columns - 1) / columns);
    return (tiles + pairs - 1) / pairs * (kb * cycles + 2000);
  };
  return cost(128, 490) < cost(256, 655) ? kTilesPair128 : kTilesPair256;
}

int SmCount() {
  static int sm_count = 0;
  if (sm_count == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (sm_count <= 0) sm_count = 148;
  }
  return sm_count;
}

template <int NB, bool GATED>
cudaError_t LaunchSkinny(const CUtensorMap& lo, const CUtensorMap& hi, const CUtensorMap& x, __nv_bfloat16* out, unsigned short* pre,
                         const __nv_bfloat16* residual, int M, int N, int K, int act, unsigned int* status, cudaStream_t stream) {
  using Cfg = SkinnyCfg<NB>;
  auto kernel = gemm_bf16_skinny_kernel<NB, GATED>;
  constexpr int kMaxDevices = 64;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr_set[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg::kSmem));
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr_set[dev] = true;
  }
  // as many slices of the reduction as give most SMs a CTA, of one 64-column block at least
  const int width = GATED ? 64 : 128, tiles = (N + width - 1) / width, num_kb = (K + BK - 1) / BK;
  int split = 1;
  while (split < 8 && 2 * split <= num_kb && 2 * tiles * split <= 2 * SmCount()) split *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * split);
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = GATED ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, kernel, lo, hi, x, out, pre, residual, M, N, num_kb, split, act, status);
}

// N: output columns (GATED: of the gated product, w holds 2 N rows)
template <bool GATED>
cudaError_t Skinny(const void* x, const void* w, void* out, void* pre, const void* residual, int M, int N, int K, int act, unsigned int* status,
                   cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out) |
                        reinterpret_cast<uintptr_t>(pre) | reinterpret_cast<uintptr_t>(residual);
  if (M <= 0 || M > kSkinnyRows || N <= 0 || K <= 0 || (K % 8) != 0 || (N % 8) != 0 || (all & 15) != 0 || x == nullptr || w == nullptr || out == nullptr)
    return cudaErrorInvalidValue;
  const int nb = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  CUtensorMap lo, hi, mx;
  if (!MakeMap(&lo, w, N, K, 64) || !MakeMap(&mx, x, M, K, nb)) return cudaErrorInvalidValue;
  hi = lo;
  if (GATED && !MakeMap(&hi, static_cast<const __nv_bfloat16*>(w) + size_t(N) * K, N, K, 64)) return cudaErrorInvalidValue;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  unsigned short* p = static_cast<unsigned short*>(pre);
  const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(residual);
  const cudaError_t e = nb == 16   ? LaunchSkinny<16, GATED>(lo, hi, mx, o, p, r, M, N, K, act, status, stream)
                        : nb == 32 ? LaunchSkinny<32, GATED>(lo, hi, mx, o, p, r, M, N, K, act, status, stream)
                                   : LaunchSkinny<64, GATED>(lo, hi, mx, o, p, r, M, N, K, act, status, stream);
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

}  // namespace

bool GemmSupported() { return GetEncodeFn() != nullptr; }

cudaError_t LaunchGemmGatedDown(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status, cudaStream_t stream,
                                const void* addend) {
  if (M <= kSkinnyRows) return Skinny<false>(a, b, out, nullptr, addend, M, N, K, kActNone, status, stream);
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(addend);
  if (M <= 0 || N <= 0 || K <= 0 || (N % 8) != 0 || (K % 8) != 0 || (all & 15) != 0 || a == nullptr || b == nullptr || out == nullptr)
    return cudaErrorInvalidValue;
  const int sm_count = SmCount();
  const GemmTiles tiles = PlanTiles(M, N, K, sm_count);
  const int bn = tiles == kTilesPair128 || (tiles == kTilesSingle && N <= 128) ? 128 : 256;
  CUtensorMap map_a, map_b, map_c;
  if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, tiles == kTilesSingle ? bn : bn / 2) || !MakeMap(&map_c, out, M, N, 32))
    return cudaErrorInvalidValue;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  const __nv_bfloat16* add = static_cast<const __nv_bfloat16*>(addend);
  auto go = [&](auto epi) {
    constexpr int EPI = decltype(epi)::value;
    if (tiles == kTilesPair256)
      return LaunchPersistent<256, 0, 0, EPI, 1>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count, status, stream);
    if (tiles == kTilesPair128)
      return LaunchPersistent<128, 0, 0, EPI, 1>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count, status, stream);
    if (bn == 256) return LaunchPersistent<256, 0, 0, EPI>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count, status, stream);
    return LaunchPersistent<128, 0, 0, EPI>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count, status, stream);
  };
  const cudaError_t e = add != nullptr ? go(std::integral_constant<int, kEpiAddAux>()) : go(std::integral_constant<int, kEpiNone>());
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

cudaError_t LaunchGemmGroup(const GemmGroupItem* list, int count, unsigned int* status, cudaStream_t stream) {
  (void)cudaGetLastError();
  if (count < 1 || count > kMaxGroup) return cudaErrorInvalidValue;
  // what can start early, then the longest reductions
  const GemmGroupItem* by_length[kMaxGroup];
  for (int i = 0; i < count; ++i) by_length[i] = list + i;
  std::stable_sort(by_length, by_length + count, [](const GemmGroupItem* x, const GemmGroupItem* y) {
    return x->early != y->early ? x->early : x->K > y->K;
  });
  GroupArgs args;
  args.items = 0;
  for (int i = 0; i < kMaxGroup; ++i) {
    if (i >= count) {
      args.p[i] = {0, 0, 0, 1, 1, INT_MAX, 0, 0};
      continue;
    }
    const GemmGroupItem& g = *by_length[i];
    const uintptr_t all = reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.b) | reinterpret_cast<uintptr_t>(g.out);
    if (g.M <= 0 || g.N <= 0 || g.K <= 0 || g.N % 8 != 0 || (g.a_transposed ? g.M : g.K) % 8 != 0 || (all & 15) != 0 || g.a == nullptr || g.b == nullptr || g.out == nullptr)
      return cudaErrorInvalidValue;
    if (!(g.a_transposed ? MakeMap(&args.a[i], g.a, g.K, g.M, 64) : MakeMap(&args.a[i], g.a, g.M, g.K, BM)) ||
        !MakeMap(&args.b[i], g.b, g.K, g.N, 64) || !MakeMap(&args.c[i], g.out, g.M, g.N, 32))
      return cudaErrorInvalidValue;
    args.p[i] = {g.M, g.N, (g.K + BK - 1) / BK, (g.M + 255) / 256, (g.N + 255) / 256, args.items, g.a_transposed ? 1 : 0, g.early ? 1 : 0};
    args.items += args.p[i].tiles_m * args.p[i].tiles_n;
  }
  for (int i = count; i < kMaxGroup; ++i) args.a[i] = args.b[i] = args.c[i] = args.a[0];
  using Cfg = PersistentCfg<256, kEpiNone, 1>;
  constexpr int kMaxDevices = 64;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr_set[dev]) {
    e = cudaFuncSetAttribute(gemm_bf16_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg::kSmem));
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr_set[dev] = true;
  }
  const int pairs = std::min(args.items, SmCount() / 2);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(Cfg::kThreadsP);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = by_length[0]->early ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, gemm_bf16_group_kernel, args, status);
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

cudaError_t LaunchGemmBf16NT(const void* a, const void* b, void* out, const void* bias, int M, int N, int K, int act,
                             unsigned int* status, cudaStream_t stream, void* preact_out, float* col_stats,
                             const void* addend) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (M <= 0 || N <= 0 || K <= 0) return cudaErrorInvalidValue;
  // TMA needs 16-byte aligned bases and row pitches: K must be a multiple of 8 bf16 elements.
  if ((K % 8) != 0 || (reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 15))
    return cudaErrorInvalidValue;
  static const int variant = [] {
    const char* v = std::getenv("BLUEFOG_B200_GEMM_VARIANT");   // "tile" = one tile per CTA, default persistent
    return (v != nullptr && std::string(v) == "tile") ? 0 : 1;
  }();
  const int sm_count = SmCount();
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  const __nv_bfloat16* bp = static_cast<const __nv_bfloat16*>(bias);
  CUtensorMap map_a, map_b, map_c;
  const int tma_out = (N % 8) == 0 ? 1 : 0;        // TMA needs a 16-byte row pitch
  if (variant != 0) {
    // output boxes of [32 rows x 64 columns]; without a usable pitch the map is a valid dummy over A
    if (!(tma_out ? MakeMap(&map_c, out, M, N, 32) : MakeMap(&map_c, a, M, K, 32))) return cudaErrorInvalidValue;
  }
  CUtensorMap map_aux = map_c;
  const bool preact = preact_out != nullptr;
  if (preact) {
    if (variant == 0 || !tma_out || (reinterpret_cast<uintptr_t>(preact_out) & 15)) return cudaErrorInvalidValue;
    if (!MakeMap(&map_aux, preact_out, M, N, 32)) return cudaErrorInvalidValue;
  }
  cudaError_t e = cudaSuccess;
  if (addend != nullptr) {
    // out = a b^T + bias + addend (a layer whose output joins a residual stream): the addend is read in the epilogue
    if (variant == 0 || !tma_out || preact || col_stats != nullptr || act != 0 || (reinterpret_cast<uintptr_t>(addend) & 15))
      return cudaErrorInvalidValue;
    const __nv_bfloat16* add = static_cast<const __nv_bfloat16*>(addend);
    if (UsePair(M, N, K, sm_count)) {
      if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 128)) return cudaErrorInvalidValue;
      e = LaunchPersistent<256, 0, 0, kEpiAddAux, 1>(map_a, map_b, map_c, map_c, o, bp, add, M, N, K, 0, 1, sm_count, status, stream);
    } else if (N > 128) {
      if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 256)) return cudaErrorInvalidValue;
      e = LaunchPersistent<256, 0, 0, kEpiAddAux>(map_a, map_b, map_c, map_c, o, bp, add, M, N, K, 0, 1, sm_count, status, stream);
    } else {
      if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 128)) return cudaErrorInvalidValue;
      e = LaunchPersistent<128, 0, 0, kEpiAddAux>(map_a, map_b, map_c, map_c, o, bp, add, M, N, K, 0, 1, sm_count, status, stream);
    }
  } else if (col_stats != nullptr) {
    // column statistics of the plain product only: the kernel relies on rows past M being exact zeros
    if (variant == 0 || !tma_out || preact || bias != nullptr || act != 0) return cudaErrorInvalidValue;
    const int bn = N > 128 ? 256 : 128;
    if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, bn)) return cudaErrorInvalidValue;
    e = N > 128 ? LaunchPersistent<256, 0, 0, kEpiColumnStats>(map_a, map_b, map_c, map_aux, o, nullptr, nullptr, M, N, K, 0, 1,
                                                               sm_count, status, stream, col_stats)
                : LaunchPersistent<128, 0, 0, kEpiColumnStats>(map_a, map_b, map_c, map_aux, o, nullptr, nullptr, M, N, K, 0, 1,
                                                               sm_count, status, stream, col_stats);
  } else if (variant == 0) {
    if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, BN)) return cudaErrorInvalidValue;
    static bool attr_set = false;
    if (!attr_set) {
      e = cudaFuncSetAttribute(gemm_bf16_nt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes));
      if (e != cudaSuccess) return e;
      attr_set = true;
    }
    dim3 grid((N + BN - 1) / BN, (M + BM - 1) / BM);
    gemm_bf16_nt_kernel<<<grid, kThreads, kSmemBytes, stream>>>(map_a, map_b, o, bp, M, N, K, act, status);
  } else if (tma_out && UsePair(M, N, K, sm_count)) {
    if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 128)) return cudaErrorInvalidValue;
    e = preact ? LaunchPersistent<256, 0, 0, kEpiStorePreact, 1>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, 1,
                                                                 sm_count, status, stream)
               : LaunchPersistent<256, 0, 0, kEpiNone, 1>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, 1, sm_count,
                                                          status, stream);
  } else if (N > 128) {
    if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 256)) return cudaErrorInvalidValue;
    e = preact ? LaunchPersistent<256, 0, 0, kEpiStorePreact>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, tma_out,
                                                              sm_count, status, stream)
               : LaunchPersistent<256, 0, 0, kEpiNone>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, tma_out,
                                                       sm_count, status, stream);
  } else {
    if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, N, K, 128)) return cudaErrorInvalidValue;
    e = preact ? LaunchPersistent<128, 0, 0, kEpiStorePreact>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, tma_out,
                                                              sm_count, status, stream)
               : LaunchPersistent<128, 0, 0, kEpiNone>(map_a, map_b, map_c, map_aux, o, bp, nullptr, M, N, K, act, tma_out,
                                                       sm_count, status, stream);
  }
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

// out[M,N] = a[M,K] * b[K,N]: the B operand is consumed MN-major straight from its row-major memory, so a
// product with a transposed weight (an input gradient) needs no transposed copy.  With gelu_preact the result
// is multiplied elementwise by GELU'(gelu_preact[M,N]) in the epilogue (the backward of a fused Linear+GELU).
cudaError_t LaunchGemmBf16NN(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status,
                             cudaStream_t stream, const void* gelu_preact, const void* addend) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (M <= 0 || N <= 0 || K <= 0 || (K % 8) != 0 || (N % 8) != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (reinterpret_cast<uintptr_t>(gelu_preact) & 15) || (reinterpret_cast<uintptr_t>(addend) & 15) ||
      (gelu_preact != nullptr && addend != nullptr))
    return cudaErrorInvalidValue;
  const int sm_count = SmCount();
  CUtensorMap map_a, map_b, map_c;
  // B: [K rows, N columns]; boxes of 64 columns (128 bytes) x 64 rows
  if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, K, N, 64) || !MakeMap(&map_c, out, M, N, 32))
    return cudaErrorInvalidValue;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  const __nv_bfloat16* aux = static_cast<const __nv_bfloat16*>(gelu_preact);
  cudaError_t e;
  if (UsePair(M, N, K, sm_count)) {
    const __nv_bfloat16* add = static_cast<const __nv_bfloat16*>(addend);
    if (add != nullptr)
      e = LaunchPersistent<256, 1, 0, kEpiAddAux, 1>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count, status, stream);
    else if (aux != nullptr)
      e = LaunchPersistent<256, 1, 0, kEpiMulGeluGrad, 1>(map_a, map_b, map_c, map_c, o, nullptr, aux, M, N, K, 0, 1, sm_count, status,
                                                          stream);
    else
      e = LaunchPersistent<256, 1, 0, kEpiNone, 1>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1, sm_count, status,
                                                   stream);
  } else if (addend != nullptr) {
    const __nv_bfloat16* add = static_cast<const __nv_bfloat16*>(addend);
    e = N > 128 ? LaunchPersistent<256, 1, 0, kEpiAddAux>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count,
                                                          status, stream)
                : LaunchPersistent<128, 1, 0, kEpiAddAux>(map_a, map_b, map_c, map_c, o, nullptr, add, M, N, K, 0, 1, sm_count,
                                                          status, stream);
  } else if (N > 128) {
    e = aux != nullptr ? LaunchPersistent<256, 1, 0, kEpiMulGeluGrad>(map_a, map_b, map_c, map_c, o, nullptr, aux, M, N, K, 0, 1,
                                                                      sm_count, status, stream)
                       : LaunchPersistent<256, 1, 0, kEpiNone>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1,
                                                               sm_count, status, stream);
  } else {
    e = aux != nullptr ? LaunchPersistent<128, 1, 0, kEpiMulGeluGrad>(map_a, map_b, map_c, map_c, o, nullptr, aux, M, N, K, 0, 1,
                                                                      sm_count, status, stream)
                       : LaunchPersistent<128, 1, 0, kEpiNone>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1,
                                                               sm_count, status, stream);
  }
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

// h[M,F] = act(a Wg^T) * (a Wu^T) with [Wg; Wu] = w [2F, K]: one tile of the accumulator holds the same columns of both
// products, so the activation and the product with the gate are part of the epilogue.
cudaError_t LaunchGemmBf16Gated(const void* a, const void* w, void* h, void* factors, int M, int F, int K, int act,
                                unsigned int* status, cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (M <= 0 || F <= 0 || K <= 0 || (K % 8) != 0 || (F % 8) != 0 || (act != kActSilu && act != kActGeluTanh) || a == nullptr || w == nullptr || h == nullptr)
    return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) || (reinterpret_cast<uintptr_t>(h) & 15) ||
      (reinterpret_cast<uintptr_t>(factors) & 15))
    return cudaErrorInvalidValue;
  if (M <= kSkinnyRows) return Skinny<true>(a, w, h, factors, nullptr, M, F, K, act, status, stream);
  const int sm_count = SmCount();
  const __nv_bfloat16* wu = static_cast<const __nv_bfloat16*>(w) + size_t(F) * K;
  unsigned short* kept = static_cast<unsigned short*>(factors);
  CUtensorMap map_a, map_g, map_u, map_h, map_f, map_d;
  // the weights' boxes: half of the accumulator's columns each
  const bool pair = M > 128 && F > 64 && sm_count >= 2;       // pairs as in PlanTiles; their 256 columns are 128 of the result
  const int box_w = pair || F > 64 ? 128 : 64;
  if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_g, w, F, K, box_w) || !MakeMap(&map_u, wu, F, K, box_w) || !MakeMap(&map_h, h, M, F, 32, 0, 32))
    return cudaErrorInvalidValue;
  map_f = map_d = map_h;
  if (kept != nullptr && (!MakeMap(&map_f, kept, M, F, 32, 2ll * F, 32) || !MakeMap(&map_d, kept + F, M, F, 32, 2ll * F, 32))) return cudaErrorInvalidValue;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(h);
  const int mode = kept != nullptr ? 2 : 1;
  const cudaError_t e =
      pair      ? LaunchPersistent<256, 0, 0, kEpiGated, 1>(map_a, map_g, map_h, map_f, o, nullptr, nullptr, M, F, K, act, mode, sm_count,
                                                            status, stream, nullptr, &map_u, &map_d)
      : F > 64 ? LaunchPersistent<256, 0, 0, kEpiGated>(map_a, map_g, map_h, map_f, o, nullptr, nullptr, M, F, K, act, mode, sm_count, status,
                                                        stream, nullptr, &map_u, &map_d)
               : LaunchPersistent<128, 0, 0, kEpiGated>(map_a, map_g, map_h, map_f, o, nullptr, nullptr, M, F, K, act, mode, sm_count, status,
                                                        stream, nullptr, &map_u, &map_d);
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

// dpre[M,2F] = [dG dU] from dH = a[M,K] * b[K,F] and the kept factors[M,2F] = [act(G), U act'(G)].
cudaError_t LaunchGemmBf16NNGatedGrad(const void* a, const void* b, const void* factors, void* dpre, int M, int F, int K,
                                      unsigned int* status, cudaStream_t stream) {
  (void)cudaGetLastError();
  if (M <= 0 || F <= 0 || K <= 0 || (K % 8) != 0 || (F % 8) != 0 || a == nullptr || b == nullptr || factors == nullptr || dpre == nullptr)
    return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15) || (reinterpret_cast<uintptr_t>(factors) & 15) ||
      (reinterpret_cast<uintptr_t>(dpre) & 15))
    return cudaErrorInvalidValue;
  const int sm_count = SmCount();
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(dpre);
  const unsigned short* kept = static_cast<const unsigned short*>(factors);
  const GemmTiles tiles = PlanTiles(M, F, K, sm_count);
  CUtensorMap map_a, map_b, map_dg, map_du, map_f, map_d;
  if (!MakeMap(&map_a, a, M, K, BM) || !MakeMap(&map_b, b, K, F, 64) || !MakeMap(&map_dg, o, M, F, 32, 2ll * F, 32) ||
      !MakeMap(&map_du, o + F, M, F, 32, 2ll * F, 32) || !MakeMap(&map_f, kept, M, F, 32, 2ll * F, 32) ||
      !MakeMap(&map_d, kept + F, M, F, 32, 2ll * F, 32))
    return cudaErrorInvalidValue;
  const cudaError_t e =
      tiles == kTilesPair256   ? LaunchPersistent<256, 1, 0, kEpiGatedGrad, 1>(map_a, map_b, map_dg, map_du, o, nullptr, nullptr, M, F, K, 0, 1,
                                                                               sm_count, status, stream, nullptr, &map_f, &map_d)
      : tiles == kTilesPair128 ? LaunchPersistent<128, 1, 0, kEpiGatedGrad, 1>(map_a, map_b, map_dg, map_du, o, nullptr, nullptr, M, F, K, 0, 1,
                                                                               sm_count, status, stream, nullptr, &map_f, &map_d)
      : F > 128 ? LaunchPersistent<256, 1, 0, kEpiGatedGrad>(map_a, map_b, map_dg, map_du, o, nullptr, nullptr, M, F, K, 0, 1, sm_count, status,
                                                             stream, nullptr, &map_f, &map_d)
                : LaunchPersistent<128, 1, 0, kEpiGatedGrad>(map_a, map_b, map_dg, map_du, o, nullptr, nullptr, M, F, K, 0, 1, sm_count, status,
                                                             stream, nullptr, &map_f, &map_d);
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

// out[M,N] = a[K,M]^T * b[K,N]: both operands row-major with the reduction dimension outermost (the weight
// gradient dW = dY^T X of a linear layer: a = dY [rows, N_out], b = X [rows, K_in]); both are consumed MN-major.
cudaError_t LaunchGemmBf16TN(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status,
                             cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (M <= 0 || N <= 0 || K <= 0 || (M % 8) != 0 || (N % 8) != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15) || (reinterpret_cast<uintptr_t>(out) & 15))
    return cudaErrorInvalidValue;
  const int sm_count = SmCount();
  CUtensorMap map_a, map_b, map_c;
  // A: [K rows, M columns], B: [K rows, N columns]; boxes of 64 columns (128 bytes) x 64 rows
  if (!MakeMap(&map_a, a, K, M, 64) || !MakeMap(&map_b, b, K, N, 64) || !MakeMap(&map_c, out, M, N, 32))
    return cudaErrorInvalidValue;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  const cudaError_t e =
      UsePair(M, N, K, sm_count)
          ? LaunchPersistent<256, 1, 1, kEpiNone, 1>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1, sm_count, status,
                                                     stream)
      : N > 128 ? LaunchPersistent<256, 1, 1, kEpiNone>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1, sm_count,
                                                      status, stream)
              : LaunchPersistent<128, 1, 1, kEpiNone>(map_a, map_b, map_c, map_c, o, nullptr, nullptr, M, N, K, 0, 1, sm_count,
                                                      status, stream);
  if (e != cudaSuccess) return e;
  CountKernelLaunch();
  return cudaGetLastError();
}

}  // namespace bfb
