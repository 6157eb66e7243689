// Causal attention over packed sequences with grouped heads, forward and backward, on tcgen05 tensor cores.
//
//   forward   S = scale q k^T (key <= query, same sequence),  P = softmax(S),  out = P v
//   backward  delta = rowsum(dout * out),  dP = dout v^T,  dS = P (dP - delta)
//             dv = P^T dout (summed over the query heads of a group),  dk = scale dS^T q (ditto),  dq = scale dS k
//
// Every kernel works on tiles of 128 queries x 128 keys, one row of the score tile per thread, and never writes a score
// to memory.  The backward pass is two kernels, one that owns a key tile (dk, dv) and one that owns a query tile (dq):
// seven products per tile instead of five, but no atomics, so gradients do not depend on the order in which CTAs run, and
// no fp32 copy of dq.
//
// Numbers: scores, row maxima, row sums, all accumulators and the statistics kept for the backward pass are fp32.  P and
// dS are rounded to bf16 because they are operands of the next product (each rounding is off by at most 2^-9 of the
// value, the size of the rounding of the result itself).  A row's sum is taken over the unrounded values.
//
// Sequences: a tile never crosses a sequence boundary.  Tile slot cu[b] / 128 + b + i belongs to rows [128 i, 128 i + 128)
// of sequence b; slots of different sequences cannot collide because ceil(len / 128) <= cu[b+1]/128 - cu[b]/128 + 1.  So a
// CTA finds its rows from its slot with a search over cu and the host never needs to know the lengths.  Slots that hold
// no tile end at once.  TMA boxes do reach over the end of a sequence: score columns of such rows are masked, and rows
// that take part in a reduction are overwritten with zeros in shared memory first, so that nothing that another sequence
// or the padding holds (infinities and NaN included) reaches a result.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_tcgen05.h"
#include "comm_kernels.h"
#include "tcgen05_common.cuh"

namespace bfb {
namespace {

using namespace t5;

constexpr int kTile = 128;                       // rows of a query tile and of a key tile
constexpr uint32_t kBoxBytes = kTile * 128;      // 128 rows of 64 bf16 values, 128-byte swizzle
constexpr float kLog2e = 1.4426950408889634f;

// x / d for 0 <= x < 2^31 without a division (a 64-bit product; m = ceil(2^(31 + s) / d), 2^(s - 1) < d <= 2^s)
struct Divisor {
  unsigned int d, m;
  int s;
};
Divisor MakeDivisor(int d) {
  Divisor v{static_cast<unsigned int>(d), 0, 0};
  while ((1ll << v.s) < d) ++v.s;
  v.m = static_cast<unsigned int>(((1ull << (31 + v.s)) + d - 1) / d);
  return v;
}
__device__ __forceinline__ int divide(int x, const Divisor& v) {
  return int((static_cast<unsigned long long>(static_cast<unsigned int>(x)) * v.m) >> (31 + v.s));
}

struct Geo {
  const int* cu;
  int batch;
  int seq;              // tokens per sequence, or of all sequences together when cu is given
  int tiles_per_seq;    // without cu
  int tiles;
  int heads;
  int group;            // query heads per key head
  int dim;
  Divisor by_heads, by_kv_heads, by_batch, by_group;
};

struct Tile {
  int start;            // first token of the sequence
  int len;              // its length
  int index;            // tile within the sequence
  int slot;             // where the tile's row statistics lie
  int batch;            // sequence, or `batch` for the tokens behind the last one
};

__device__ __forceinline__ int cu_at(const Geo& g, int b) { return b <= 0 ? 0 : min(max(__ldg(g.cu + b), 0), g.seq); }

// The tile that comes `order`-th: tiles with much work first (queries at the end of a sequence, keys at its start).
// Called by whole warps.  False when the slot holds no tile.
__device__ __forceinline__ bool find_tile(const Geo& g, int order, bool late_first, Tile& t) {
  if (g.cu == nullptr) {
    const int i = divide(order, g.by_batch);
    t.batch = order - i * g.batch;
    t.index = late_first ? g.tiles_per_seq - 1 - i : i;
    t.slot = t.batch * g.tiles_per_seq + t.index;
    t.start = t.batch * g.seq;
    t.len = g.seq;
    return true;
  }
  t.slot = late_first ? g.tiles - 1 - order : order;
  // last b in [0, batch] with cu[b] / 128 + b <= slot; 32 probes at a time
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = g.batch + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int b = lo + lane * step;
    const bool below = b < hi && (cu_at(g, b) >> 7) + b <= t.slot;
    const int n = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  t.batch = lo;
  t.start = cu_at(g, lo);
  const int end = lo >= g.batch ? g.seq : cu_at(g, lo + 1);
  t.len = max(end - t.start, 0);
  t.index = t.slot - ((t.start >> 7) + lo);
  return t.index >= 0 && t.index * kTile < t.len;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// maximum that keeps a NaN: a row that holds one is NaN throughout, as in a softmax written out
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

// instruction descriptors: fp32 accumulator, bf16 operands, M = 128, N as given; B K-major or MN-major (bit 16)
constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
}

// scores[128 x 128] = A B^T over DP columns; A, B: DP / 64 boxes of [128 rows x 64 columns]
template <int DP>
__device__ __forceinline__ void mma_scores(uint32_t tmem_d, uint32_t a, uint32_t b) {
  const uint64_t da = make_desc(a), db = make_desc(b);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint64_t off = uint64_t(k >> 2) * (kBoxBytes >> 4) + uint64_t(k & 3) * 2;
    umma_f16(tmem_d, da + off, db + off, idesc(kTile, false), k != 0 ? 1u : 0u);
  }
}
// acc[128 x DP] += A B: A 128 x 128 bf16 in tensor memory (K elements 0-63 at `a`, 64-127 at `a` + a_half columns), B =
// DP / 64 boxes of [128 K-rows x 64 columns], read as an MN-major operand
template <int DP>
__device__ __forceinline__ void mma_accumulate(uint32_t tmem_d, uint32_t a, uint32_t a_half, uint32_t b, bool first) {
  const uint64_t db = make_desc_mn(b, kBoxBytes, 1024);
#pragma unroll
  for (int k = 0; k < kTile / 16; ++k)
    umma_f16_ts(tmem_d, a + uint32_t(k >> 2) * a_half + uint32_t(k & 3) * 8, db + uint64_t(k) * (2048 >> 4), idesc(DP, true),
                (first && k == 0) ? 0u : 1u);
}

// Zeros in rows [first, 128) of DP / 64 boxes; called by a whole warp, visible to the tensor cores afterwards.
template <int DP>
__device__ __forceinline__ void zero_rows(unsigned char* boxes, int first) {
  const int lane = threadIdx.x & 31;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  for (int b = 0; b < DP / 64; ++b)
    for (int c = first * 8 + lane; c < kTile * 8; c += 32) *reinterpret_cast<uint4*>(boxes + size_t(b) * kBoxBytes + size_t(c) * 16) = z;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// rows [row0, row0 + 128) of a [tokens, heads, dim] result set to zero where row < end
__device__ __forceinline__ void zero_result(const AttnTensor& t, int head, int row0, int end, int dim) {
  const int chunks = dim / 8;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  const int rows = min(kTile, end - row0);
  for (int i = threadIdx.x; i < rows * chunks; i += blockDim.x) {
    const int r = i / chunks, c = i - r * chunks;
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(t.ptr) + (long long)(row0 + r) * t.token_stride + (long long)head * t.head_stride;
    *reinterpret_cast<uint4*>(p + c * 8) = z;
  }
}

// One warp's 32 accumulator rows: columns [col0, col0 + 32 NC) of tensor memory are scaled per row, rounded and written to the
// warp's rows of a staging box (64 columns per box, starting with 16-byte chunk chunk0).
template <int NC>
__device__ __forceinline__ void stage_rows(uint32_t taddr, float factor, unsigned char* box, int row, int chunk0) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t r[32];
    tmem_ld32(taddr + uint32_t(c * 32), r);
    tmem_wait_ld();
    tie32(r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 v;
      v.x = pack_bf16(__uint_as_float(r[j * 8 + 0]) * factor, __uint_as_float(r[j * 8 + 1]) * factor);
      v.y = pack_bf16(__uint_as_float(r[j * 8 + 2]) * factor, __uint_as_float(r[j * 8 + 3]) * factor);
      v.z = pack_bf16(__uint_as_float(r[j * 8 + 4]) * factor, __uint_as_float(r[j * 8 + 5]) * factor);
      v.w = pack_bf16(__uint_as_float(r[j * 8 + 6]) * factor, __uint_as_float(r[j * 8 + 7]) * factor);
      const int chunk = chunk0 + c * 4 + j;
      *reinterpret_cast<uint4*>(box + size_t(chunk >> 3) * kBoxBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = v;
    }
  }
}
// Chunks [chunk0, chunk0 + CHUNKS) of the warp's 32 staged rows to memory; consecutive lanes write consecutive 16 bytes.
template <int CHUNKS>
__device__ __forceinline__ void store_rows(const AttnTensor& t, int head, int token0, int rows_left, int dim, const unsigned char* box,
                                           int row0, int chunk0) {
  const int lane = threadIdx.x & 31;
  const int last = min(chunk0 + CHUNKS, dim / 8) - chunk0;
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int r = (k * 32 + lane) / CHUNKS, c = (k * 32 + lane) % CHUNKS;
    if (r >= rows_left || c >= last) continue;
    const int row = row0 + r, chunk = chunk0 + c;
    const uint4 v = *reinterpret_cast<const uint4*>(box + size_t(chunk >> 3) * kBoxBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(t.ptr) + (long long)(token0 + r) * t.token_stride + (long long)head * t.head_stride;
    *reinterpret_cast<uint4*>(p + chunk * 8) = v;
  }
}

// ---------------------------------------------------------------------------------------------------------------- //
// Forward.  One CTA per query tile and head, two CTAs per SM: while the softmax warps of one wait for a product, those of
// the other keep the exponential unit busy.  Eight softmax warps: two threads share a row, 64 columns each, and exchange
// their maxima through shared memory (with one thread per row the 128 scores in its registers spilled and one warp per
// scheduler and CTA could not hide the latency of its own exponentials: 12 cycles per element against the 8 that the unit
// needs).  Key tiles are taken from the diagonal downwards, so only the first one needs a mask.  Tensor memory (256 of 512
// columns per CTA): scores 128, output DP, and P in a place of its own where there is room (DP = 64: the next scores are
// computed while this tile's exponentials are taken), over the scores otherwise.  The output is rescaled only when a row's
// maximum grew by more than 2^8 (the sums stay far inside fp32).
// ---------------------------------------------------------------------------------------------------------------- //
template <int DP>
struct FwdCfg {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kSlots = DP == 64 ? 5 : 2;       // ring of key / value tiles
  static constexpr uint32_t kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kThreads = 320;
  static constexpr uint32_t kColO = 128;
  static constexpr bool kOwnP = DP == 64;
  static constexpr uint32_t kColP = kOwnP ? 192 : 0;
  static constexpr size_t kSmem = 1024 + size_t(kSlots + 1) * kTileBytes;
};

template <int DP>
__global__ void __launch_bounds__(FwdCfg<DP>::kThreads, 2)
attn_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const Geo g, const AttnTensor out, float* __restrict__ stats,
                const float scale_log2, unsigned int* __restrict__ status) {
  using Cfg = FwdCfg<DP>;
  constexpr int NS = Cfg::kSlots;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem_q = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem_q + Cfg::kTileBytes;
  __shared__ uint64_t bars[2 * NS + 6];
  __shared__ float maxima[2][2][kTile];
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_q = bar0 + 8u * (2 * NS), bar_s = bar_q + 8u, bar_sfree = bar_q + 16u, bar_p = bar_q + 24u,
                 bar_pv = bar_q + 32u, bar_end = bar_q + 40u;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (NS + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int order = divide(blockIdx.x, g.by_heads);
  const int head = blockIdx.x - order * g.heads;
  if (g.cu != nullptr && blockIdx.x == 0) {
    bool bad = false;
    for (int b = threadIdx.x; b < g.batch; b += blockDim.x) {
      const int c = __ldg(g.cu + b + 1);
      bad |= c < (b == 0 ? 0 : __ldg(g.cu + b)) || c > g.seq;
    }
    if (bad) atomicOr(status, kAttnBadSequences);
  }
  Tile t;
  if (!find_tile(g, order, true, t)) return;
  const int row0 = t.index * kTile;                    // first query of the tile within its sequence
  if (g.cu != nullptr && t.batch == g.batch) {
    zero_result(out, head, t.start + row0, t.start + t.len, g.dim);
    return;
  }
  const int n = t.index + 1;                           // key tiles
  const int kv_head = divide(head, g.by_group);

  if (warp == 8 && lane == 0) {
    failed_s = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(bar_q, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_sfree, 8);
    mbar_init(bar_p, 8);
    mbar_init(bar_pv, 1);
    mbar_init(bar_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // the first tiles travel while tensor memory is allocated
    mbar_expect_tx(bar_q, Cfg::kTileBytes);
    for (int b = 0; b < Cfg::kBoxes; ++b) tma_load_3d(smem_u32(smem_q) + b * kBoxBytes, &map_q, bar_q, b * 64, head, t.start + row0);
    mbar_expect_tx(full(0), Cfg::kTileBytes);
    for (int b = 0; b < Cfg::kBoxes; ++b)
      tma_load_3d(smem_u32(ring) + b * kBoxBytes, &map_k, full(0), b * 64, kv_head, t.start + (n - 1) * kTile);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_base_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_base_s;

  if (warp == 8) {
    if (lane == 0) {
      // in the order of use: K0 K1 V0 K2 V1 ... where scores run ahead, else K0 V0 K1 V1 ...; K0 is under way
      int armed = 1;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int it) {
        const int s = armed % NS;
        if (!mbar_wait(empty(s), ((armed / NS) & 1) ^ 1, failed)) return false;
        mbar_expect_tx(full(s), Cfg::kTileBytes);
        for (int b = 0; b < Cfg::kBoxes; ++b)
          tma_load_3d(smem_u32(ring + size_t(s) * Cfg::kTileBytes) + b * kBoxBytes, map, full(s), b * 64, kv_head,
                      t.start + (n - 1 - it) * kTile);
        ++armed;
        return true;
      };
      if (Cfg::kOwnP) {
        for (int it = 0; it < n && ok; ++it) {
          if (it + 1 < n) ok = load(&map_k, it + 1);
          if (ok) ok = load(&map_v, it);
        }
      } else {
        for (int it = 0; it < n && ok; ++it) ok = (it == 0 || load(&map_k, it)) && load(&map_v, it);
      }
      if (!ok || *failed) {
        // copies in flight have to land before this shared memory goes away
        for (int f = armed > NS ? armed - NS : 0; f < armed; ++f) {
          const long long t0 = clock64();
          while (!mbar_try(full(f % NS), (f / NS) & 1) && clock64() - t0 < kWaitLimitCycles) {}
        }
        const long long t0 = clock64();
        while (!mbar_try(bar_q, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
    }
  } else if (warp == 9) {
    // the whole warp walks along, lane 0 issues; `used` counts ring slots in the order of the loads
    int used = 0;
    bool ok = mbar_wait(bar_q, 0, failed);
    auto scores = [&]() {
      const int s = used % NS;
      if (!mbar_wait(full(s), (used / NS) & 1, failed)) return false;
      ++used;
      if (lane == 0) {
        mma_scores<DP>(tmem, smem_u32(smem_q), smem_u32(ring + size_t(s) * Cfg::kTileBytes));
        umma_commit(empty(s));
        umma_commit(bar_s);
      }
      __syncwarp();
      return true;
    };
    ok = ok && scores();
    for (int it = 0; it < n && ok; ++it) {
      if (Cfg::kOwnP && it + 1 < n) {
        ok = mbar_wait(bar_sfree, it & 1, failed);     // this tile's scores are in registers
        fence_after_sync();
        ok = ok && scores();
        if (!ok) break;
      }
      const int s = used % NS;
      ok = mbar_wait(full(s), (used / NS) & 1, failed);
      if (!ok) break;
      ++used;
      unsigned char* v = ring + size_t(s) * Cfg::kTileBytes;
      // P is zero behind the end of the sequence, which is not enough when the rows there hold infinities or NaN
      if (it == 0 && t.len - row0 < kTile) zero_rows<DP>(v, t.len - row0);
      ok = mbar_wait(bar_p, it & 1, failed);
      if (!ok) break;
      fence_after_sync();
      if (lane == 0) {
        mma_accumulate<DP>(tmem + Cfg::kColO, tmem + Cfg::kColP, 32, smem_u32(v), it == 0);
        umma_commit(empty(s));
        umma_commit(bar_pv);
      }
      __syncwarp();
      if (!Cfg::kOwnP && it + 1 < n) ok = scores();    // over P: products run in the order of issue
    }
    if (!ok || *failed) {
      if (lane == 0) {
        umma_commit(bar_end);                          // tensor memory is not freed under a product
        const long long t0 = clock64();
        while (!mbar_try(bar_end, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
      __syncwarp();
    }
  } else {
    const int half = warp >> 2;                        // columns 64 half .. 64 half + 63
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + half * 64, tO = tmem + lanes + Cfg::kColO + half * (DP / 2), tP = tmem + lanes + Cfg::kColP + half * 32;
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };   // the two warps of 32 rows
    float m = 0.f, l = 0.f;
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      // no way out of this loop: after a wait that failed the others fail at once, and the two warps of a pair meet in
      // every iteration
      ok = mbar_wait(bar_s, it & 1, failed) && ok;
      fence_after_sync();
      uint32_t r[64];
      tmem_ld32(tS, r);
      tmem_ld32(tS + 32, r + 32);
      tmem_wait_ld();
      tie32(r);
      tie32(r + 32);
      if (Cfg::kOwnP) {
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_sfree);
      }
      if (it == 0) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (half * 64 + c > row) r[c] = 0xff800000u;             // -inf
      }
      float mx[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) mx[k] = max_nan(__uint_as_float(r[k]), __uint_as_float(r[k + 4]));
#pragma unroll
      for (int c = 8; c < 64; c += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = max3_nan(mx[k], __uint_as_float(r[c + k]), __uint_as_float(r[c + k + 4]));
      float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
      // two sets of cells in turn: a thread is at most one tile ahead of its partner
      maxima[it & 1][half][row] = top;
      pair_sync();
      top = max_nan(top, maxima[it & 1][half ^ 1][row]);
      if (it == 0) {
        m = top;
      } else {
        const bool grown = !((top - m) * scale_log2 <= 8.f);
        if (__any_sync(0xffffffffu, grown)) {
          // rare; the product before has to be complete.  A row that did not grow keeps its reference, so that its bits do
          // not depend on what the warp's other rows hold.
          ok = mbar_wait(bar_pv, (it - 1) & 1, failed) && ok;
          const float next = grown ? max_nan(m, top) : m;
          const float f = ex2((m - (next == -INFINITY ? 0.f : next)) * scale_log2);
          m = next;
          l *= f;
          fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < DP / 2; c += 16) {
            uint32_t o[16];
            tmem_ld16(tO + c, o);
            tmem_wait_ld();
            tie16(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st16(tO + c, o);
          }
        }
      }
      // a row whose scores are all -inf so far takes 0 as its reference: exp(-inf - 0) = 0 instead of NaN
      const float shift = m == -INFINITY ? 0.f : -m * scale_log2;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t p[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const float a = ex2(fmaf(__uint_as_float(r[2 * c]), scale_log2, shift));
        const float b = ex2(fmaf(__uint_as_float(r[2 * c + 1]), scale_log2, shift));
        sum[(2 * c) & 3] += a;
        sum[(2 * c + 1) & 3] += b;
        p[c] = pack_bf16(a, b);
      }
      if (Cfg::kOwnP && it > 0) ok = mbar_wait(bar_pv, (it - 1) & 1, failed) && ok;   // P has been read
      tmem_st32(tP, p);
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p);
    }
    // the row's sum is in two places
    maxima[n & 1][half][row] = l;
    pair_sync();
    l += maxima[n & 1][half ^ 1][row];
    if (ok && mbar_wait(bar_pv, (n - 1) & 1, failed)) {
      fence_after_sync();
      stage_rows<DP / 64>(tO, 1.f / l, smem_q, row, half * (DP / 16));
      __syncwarp();
      const int left = t.len - row0 - (row & ~31);
      store_rows<DP / 16>(out, head, t.start + row0 + (row & ~31), left, g.dim, smem_q, row & ~31, half * (DP / 16));
      if (stats != nullptr && half == 0)
        stats[((long long)head * g.tiles + t.slot) * kTile + row] = lane < left ? fmaf(m, scale_log2, log2f(l)) : INFINITY;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
  }
  if (threadIdx.x == 0 && failed_s) atomicOr(status, kAttnTimeout);
}

// ---------------------------------------------------------------------------------------------------------------- //
// delta[head, row] = sum_d dout * out, one tile and head per block; rows that belong to no token get 0.
// ---------------------------------------------------------------------------------------------------------------- //
__global__ void __launch_bounds__(256) attn_delta_kernel(const Geo g, const AttnTensor out, const AttnTensor dout, float* __restrict__ delta) {
  const int order = divide(blockIdx.x, g.by_heads);
  const int head = blockIdx.x - order * g.heads;
  Tile t;
  if (!find_tile(g, order, true, t) || (g.cu != nullptr && t.batch == g.batch)) return;
  const int sub = threadIdx.x & 15;                    // sixteen threads per row, eight values each
  for (int r = threadIdx.x >> 4; r < kTile; r += 16) {
    float s = 0.f;
    const int row = t.index * kTile + r;
    if (row < t.len && sub * 8 < g.dim) {
      const long long tok = t.start + row;
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(out.ptr) + tok * out.token_stride +
                                                      (long long)head * out.head_stride + sub * 8);
      const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(dout.ptr) + tok * dout.token_stride +
                                                      (long long)head * dout.head_stride + sub * 8);
      const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&a);
      const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 u = __bfloat1622float2(x[i]), v = __bfloat1622float2(y[i]);
        s = fmaf(u.x, v.x, fmaf(u.y, v.y, s));
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (sub == 0) delta[((long long)head * g.tiles + t.slot) * kTile + r] = s;
  }
}

// ---------------------------------------------------------------------------------------------------------------- //
// Backward.  KV: a CTA owns a key tile of one key head and walks over the query tiles at and after it, for every query
// head of the group; scores are held transposed (rows = keys), so P^T and dS^T are the tensor-memory operands of
// dv += P^T dout and dk += dS^T q, and the row statistics are per column.  Otherwise a CTA owns a query tile of one head
// and walks over the key tiles from the diagonal downwards: dq += dS k.  One CTA per SM; eight warps take the
// exponentials, two per quarter of tensor memory, each with one half of the columns.
// Tensor memory: scores (two buffers where 512 columns allow it, so that the next scores are ready when a tile's work
// ends), dP, accumulators.  The bf16 operands replace the fp32 values they come from: elements 0-63 at the start of the
// region, 64-127 at its middle, so each half of the warps writes where it alone has read.
// ---------------------------------------------------------------------------------------------------------------- //
template <int DP, bool KV>
struct BwdCfg {
  static constexpr int kBoxes = DP / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kStages = DP == 64 ? 4 : 2;
  static constexpr bool kTwoScores = !(KV && DP == 128);
  static constexpr int kThreads = 320;
  static constexpr uint32_t kColDP = 128, kColS1 = 256;
  static constexpr uint32_t kCol1 = 512 - DP, kCol0 = kCol1 - DP;      // accumulators of dk / dq and of dv
  static constexpr uint32_t kStatBytes = KV ? 2 * kTile * 4 : 0;
  static constexpr size_t kSmem = 1024 + 2 * size_t(kTileBytes) + size_t(kStages) * (2 * kTileBytes + kStatBytes);
};

template <int DP, bool KV>
__global__ void __launch_bounds__((BwdCfg<DP, KV>::kThreads), 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Geo g,
                const float* __restrict__ stats, const float* __restrict__ delta, const AttnTensor d0, const AttnTensor d1,
                const float scale, const float scale_log2, unsigned int* __restrict__ status) {
  using Cfg = BwdCfg<DP, KV>;
  constexpr int NS = Cfg::kStages;
  constexpr bool kTwo = Cfg::kTwoScores;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem_x = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem_x + 2 * Cfg::kTileBytes;
  float* ring_stats = reinterpret_cast<float*>(ring + size_t(NS) * 2 * Cfg::kTileBytes);      // KV: per stage lse[128], delta[128]
  __shared__ uint64_t bars[2 * NS + 10];
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_x = bar0 + 8u * (2 * NS), bar_s = bar_x + 8u /* two */, bar_dp = bar_x + 24u, bar_dpfree = bar_x + 32u,
                 bar_p = bar_x + 40u /* two */, bar_ds = bar_x + 56u /* two */, bar_end = bar_x + 72u;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (NS + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int own_heads = KV ? g.heads / g.group : g.heads;
  const int order = divide(blockIdx.x, KV ? g.by_kv_heads : g.by_heads);
  const int own_head = blockIdx.x - order * own_heads;
  Tile t;
  if (!find_tile(g, order, !KV, t)) return;
  const int row0 = t.index * kTile;
  if (g.cu != nullptr && t.batch == g.batch) {
    if (KV) zero_result(d0, own_head, t.start + row0, t.start + t.len, g.dim);
    zero_result(d1, own_head, t.start + row0, t.start + t.len, g.dim);
    return;
  }
  const int seq_tiles = (t.len + kTile - 1) / kTile;
  const int per_head = KV ? seq_tiles - t.index : t.index + 1;
  const int n = KV ? per_head * g.group : per_head;
  const int first_slot = t.slot - t.index;
  // tile of the other side (query tile for KV, key tile otherwise) in iteration `it`
  auto other_tile = [&](int it) { return KV ? t.index + it % per_head : t.index - it; };

  if (threadIdx.x == 0) {
    failed_s = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(bar_x, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_s + 8u, 1);
    mbar_init(bar_dp, 1);
    mbar_init(bar_dpfree, 8);
    // two each, for even and odd iterations: a warp may be one iteration ahead of another, and its arrival must not
    // count for the other's
    for (int k = 0; k < 2; ++k) {
      mbar_init(bar_p + 8u * k, 8);
      mbar_init(bar_ds + 8u * k, 8);
    }
    mbar_init(bar_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_base_s;

  if (warp == 8) {
    if (lane == 0) {
      mbar_expect_tx(bar_x, 2 * Cfg::kTileBytes);
      for (int b = 0; b < Cfg::kBoxes; ++b) {
        tma_load_3d(smem_u32(smem_x) + b * kBoxBytes, KV ? &map_k : &map_q, bar_x, b * 64, own_head, t.start + row0);
        tma_load_3d(smem_u32(smem_x) + Cfg::kTileBytes + b * kBoxBytes, KV ? &map_v : &map_do, bar_x, b * 64, own_head, t.start + row0);
      }
      int armed = 0;
      bool ok = true;
      for (int it = 0; it < n; ++it) {
        const int s = it % NS;
        ok = mbar_wait(empty(s), ((it / NS) & 1) ^ 1, failed);
        if (!ok) break;
        const int j = other_tile(it);
        const int head = KV ? own_head * g.group + it / per_head : divide(own_head, g.by_group);
        const uint32_t dst = smem_u32(ring + size_t(s) * 2 * Cfg::kTileBytes);
        mbar_expect_tx(full(s), 2 * Cfg::kTileBytes + Cfg::kStatBytes);
        for (int b = 0; b < Cfg::kBoxes; ++b) {
          tma_load_3d(dst + b * kBoxBytes, KV ? &map_q : &map_k, full(s), b * 64, head, t.start + j * kTile);
          tma_load_3d(dst + Cfg::kTileBytes + b * kBoxBytes, KV ? &map_do : &map_v, full(s), b * 64, head, t.start + j * kTile);
        }
        if (KV) {
          const long long at = ((long long)head * g.tiles + first_slot + j) * kTile;
          bulk_load(smem_u32(ring_stats + s * 2 * kTile), stats + at, full(s), kTile * 4);
          bulk_load(smem_u32(ring_stats + s * 2 * kTile + kTile), delta + at, full(s), kTile * 4);
        }
        armed = it + 1;
      }
      if (!ok || *failed) {
        for (int f = armed > NS ? armed - NS : 0; f < armed; ++f) {
          const long long t0 = clock64();
          while (!mbar_try(full(f % NS), (f / NS) & 1) && clock64() - t0 < kWaitLimitCycles) {}
        }
        const long long t0 = clock64();
        while (!mbar_try(bar_x, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
    }
  } else if (warp == 9) {
    const uint32_t x0 = smem_u32(smem_x), x1 = x0 + Cfg::kTileBytes;
    auto stage = [&](int it) { return ring + size_t(it % NS) * 2 * Cfg::kTileBytes; };
    auto s_col = [&](int it) { return tmem + ((kTwo && (it & 1)) ? Cfg::kColS1 : 0u); };
    bool ok = mbar_wait(bar_x, 0, failed);
    // waits for the tiles of an iteration and issues its scores
    auto scores = [&](int it) {
      if (!mbar_wait(full(it % NS), (it / NS) & 1, failed)) return false;
      const int j = other_tile(it);
      if (t.len - j * kTile < kTile) {                 // rows behind the end of the sequence take part in the reductions
        zero_rows<DP>(stage(it), t.len - j * kTile);
        zero_rows<DP>(stage(it) + Cfg::kTileBytes, t.len - j * kTile);
      }
      if (lane == 0) {
        mma_scores<DP>(s_col(it), x0, smem_u32(stage(it)));
        umma_commit(bar_s + (kTwo ? 8u * (it & 1) : 0u));
      }
      __syncwarp();
      return true;
    };
    auto grad_scores = [&](int it) {
      if (lane == 0) {
        mma_scores<DP>(tmem + Cfg::kColDP, x1, smem_u32(stage(it)) + Cfg::kTileBytes);
        umma_commit(bar_dp);
      }
      __syncwarp();
    };
    ok = ok && scores(0);
    if (ok) grad_scores(0);
    for (int it = 0; it < n && ok; ++it) {
      const bool more = it + 1 < n;
      if (kTwo && more) {
        // the other score buffer: its operand was read by a product issued before these
        ok = scores(it + 1);
        if (!ok) break;
      }
      if (KV) {
        ok = mbar_wait(bar_p + 8u * (it & 1), (it >> 1) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        if (lane == 0) mma_accumulate<DP>(tmem + Cfg::kCol0, s_col(it), 64, smem_u32(stage(it)) + Cfg::kTileBytes, it == 0);
        __syncwarp();
        if (!kTwo && more) {
          ok = scores(it + 1);                         // over P: products run in the order of issue
          if (!ok) break;
        }
      } else if (more) {
        ok = mbar_wait(bar_dpfree, it & 1, failed);
        if (!ok) break;
        fence_after_sync();
        grad_scores(it + 1);
      }
      ok = mbar_wait(bar_ds + 8u * (it & 1), (it >> 1) & 1, failed);
      if (!ok) break;
      fence_after_sync();
      if (lane == 0) {
        mma_accumulate<DP>(tmem + Cfg::kCol1, KV ? tmem + Cfg::kColDP : s_col(it), 64, smem_u32(stage(it)), it == 0);
        umma_commit(empty(it % NS));
      }
      __syncwarp();
      if (KV && more) grad_scores(it + 1);             // over dS
    }
    if (lane == 0) {
      umma_commit(bar_end);
      if (!ok || *failed) {
        const long long t0 = clock64();
        while (!mbar_try(bar_end, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
    }
    __syncwarp();
  } else {
    const int half = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    float lse = 0.f, dlt = 0.f;
    if (!KV) {
      const long long at = ((long long)own_head * g.tiles + t.slot) * kTile + row;
      lse = stats[at];
      dlt = delta[at];
    }
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const bool diagonal = other_tile(it) == t.index;
      const float* st = ring_stats + (it % NS) * 2 * kTile + half * 64;
      const uint32_t tS = tmem + lanes + ((kTwo && (it & 1)) ? Cfg::kColS1 : 0u) + half * 64;
      const uint32_t tD = tmem + lanes + Cfg::kColDP + half * 64;
      ok = kTwo ? mbar_wait(bar_s + 8u * (it & 1), (it >> 1) & 1, failed) : mbar_wait(bar_s, it & 1, failed);
      if (!ok) break;
      if (KV) {
        // the statistics came with the tiles of this stage: acquire their barrier too
        ok = mbar_wait(full(it % NS), (it / NS) & 1, failed);
        if (!ok) break;
      }
      fence_after_sync();
      uint32_t r[64];
      tmem_ld32(tS, r);
      tmem_ld32(tS + 32, r + 32);
      tmem_wait_ld();
      tie32(r);
      tie32(r + 32);
      float p[64];
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        float4 s4 = make_float4(lse, lse, lse, lse);
        if (KV) s4 = *reinterpret_cast<const float4*>(st + c);
        p[c + 0] = ex2(fmaf(__uint_as_float(r[c + 0]), scale_log2, -s4.x));
        p[c + 1] = ex2(fmaf(__uint_as_float(r[c + 1]), scale_log2, -s4.y));
        p[c + 2] = ex2(fmaf(__uint_as_float(r[c + 2]), scale_log2, -s4.z));
        p[c + 3] = ex2(fmaf(__uint_as_float(r[c + 3]), scale_log2, -s4.w));
      }
      if (diagonal) {
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          const int col = half * 64 + c;
          if (KV ? col < row : col > row) p[c] = 0.f;
        }
      }
      if (KV) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) pk[c] = pack_bf16(p[2 * c], p[2 * c + 1]);
        tmem_st32(tS, pk);
        tmem_wait_st();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8u * (it & 1));
      }
      ok = mbar_wait(bar_dp, it & 1, failed);
      if (!ok) break;
      fence_after_sync();
      tmem_ld32(tD, r);
      tmem_ld32(tD + 32, r + 32);
      tmem_wait_ld();
      tie32(r);
      tie32(r + 32);
      if (!KV) {
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_dpfree);
      }
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        float4 d4 = make_float4(dlt, dlt, dlt, dlt);
        if (KV) d4 = *reinterpret_cast<const float4*>(st + kTile + c);
        pk[c / 2] = pack_bf16(p[c] * (__uint_as_float(r[c]) - d4.x), p[c + 1] * (__uint_as_float(r[c + 1]) - d4.y));
        pk[c / 2 + 1] = pack_bf16(p[c + 2] * (__uint_as_float(r[c + 2]) - d4.z), p[c + 3] * (__uint_as_float(r[c + 3]) - d4.w));
      }
      tmem_st32(KV ? tD : tS, pk);
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_ds + 8u * (it & 1));
    }
    if (ok && mbar_wait(bar_end, 0, failed) && !*failed) {
      fence_after_sync();
      // the ring is at rest: staging boxes for the results
      const int left = t.len - row0 - (warp & 3) * 32;
      const int token0 = t.start + row0 + (warp & 3) * 32;
      if (KV) {
        unsigned char* box = ring + size_t(half) * Cfg::kTileBytes;
        stage_rows<DP / 32>(tmem + lanes + (half ? Cfg::kCol1 : Cfg::kCol0), half ? scale : 1.f, box, row, 0);
        __syncwarp();
        store_rows<DP / 8>(half ? d1 : d0, own_head, token0, left, g.dim, box, row & ~31, 0);
      } else {
        stage_rows<DP / 64>(tmem + lanes + Cfg::kCol1 + half * (DP / 2), scale, ring, row, half * (DP / 16));
        __syncwarp();
        store_rows<DP / 16>(d1, own_head, token0, left, g.dim, ring, row & ~31, half * (DP / 16));
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  if (threadIdx.x == 0 && failed_s) atomicOr(status, kAttnTimeout);
}

// ---- host side ---------------------------------------------------------------------------------------------------

bool MakeMap(CUtensorMap* map, const AttnTensor& t, int heads, int dim, long long tokens) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(t.head_stride) * 2, static_cast<cuuint64_t>(t.token_stride) * 2};
  const cuuint32_t box[3] = {64, 1, kTile};
  return EncodeTiled(map, 3, t.ptr, dims, strides, box);
}

bool Addressable(const AttnTensor& t) {
  return t.ptr != nullptr && (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 && t.token_stride > 0 && t.head_stride > 0 &&
         t.token_stride % 8 == 0 && t.head_stride % 8 == 0;
}

Geo MakeGeo(const AttnShape& s) {
  Geo g;
  g.cu = s.cu;
  g.batch = s.batch;
  g.seq = static_cast<int>(s.seq);
  g.tiles_per_seq = static_cast<int>((s.seq + kTile - 1) / kTile);
  g.tiles = static_cast<int>(AttnTiles(s));
  g.heads = s.heads;
  g.group = s.heads / s.kv_heads;
  g.dim = s.dim;
  g.by_heads = MakeDivisor(s.heads);
  g.by_kv_heads = MakeDivisor(s.kv_heads);
  g.by_batch = MakeDivisor(s.batch);
  g.by_group = MakeDivisor(g.group);
  return g;
}

// Shared memory above 48 KB has to be allowed per device; a call costs about a microsecond, so it is made once for each.
template <auto kernel>
cudaError_t AllowSmem(size_t bytes) {
  constexpr int kMaxDevices = 64;
  static bool done[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kMaxDevices && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < kMaxDevices) done[dev] = true;
  return e;
}

template <int DP>
cudaError_t Forward(const AttnShape& s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnTensor& out,
                    float* stats, unsigned int* status, cudaStream_t stream) {
  constexpr auto kernel = attn_fwd_kernel<DP>;
  using Cfg = FwdCfg<DP>;
  const cudaError_t e = AllowSmem<kernel>(Cfg::kSmem);
  if (e != cudaSuccess) return e;
  const Geo g = MakeGeo(s);
  kernel<<<static_cast<unsigned>(g.tiles) * g.heads, Cfg::kThreads, Cfg::kSmem, stream>>>(mq, mk, mv, g, out, stats, s.scale * kLog2e, status);
  CountKernelLaunch();
  return cudaGetLastError();
}

template <int DP, bool KV>
cudaError_t Backward(const AttnShape& s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& md,
                     const float* stats, const float* delta, const AttnTensor& d0, const AttnTensor& d1, unsigned int* status,
                     cudaStream_t stream) {
  constexpr auto kernel = attn_bwd_kernel<DP, KV>;
  using Cfg = BwdCfg<DP, KV>;
  const cudaError_t e = AllowSmem<kernel>(Cfg::kSmem);
  if (e != cudaSuccess) return e;
  const Geo g = MakeGeo(s);
  kernel<<<static_cast<unsigned>(g.tiles) * (KV ? s.kv_heads : s.heads), Cfg::kThreads, Cfg::kSmem, stream>>>(
      mq, mk, mv, md, g, stats, delta, d0, d1, s.scale, s.scale * kLog2e, status);
  CountKernelLaunch();
  return cudaGetLastError();
}

}  // namespace

long long AttnTiles(const AttnShape& s) {
  return s.cu == nullptr ? s.batch * ((s.seq + kTile - 1) / kTile) : s.seq / kTile + s.batch + 1;
}

bool AttnSupported(const AttnShape& s) {
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  return GetEncodeFn() != nullptr && s.batch > 0 && s.seq > 0 && s.heads > 0 && s.kv_heads > 0 && s.heads % s.kv_heads == 0 &&
         s.dim >= 8 && s.dim <= 128 && s.dim % 8 == 0 && s.scale > 0.f && tokens < (1ll << 31) - 2 * kTile &&
         AttnTiles(s) * s.heads < (1ll << 31);
}

cudaError_t LaunchAttnForward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                              const AttnTensor& out, float* stats, unsigned int* status, cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (!AttnSupported(s) || !Addressable(q) || !Addressable(k) || !Addressable(v) || !Addressable(out) || status == nullptr)
    return cudaErrorInvalidValue;
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  CUtensorMap mq, mk, mv;
  if (!MakeMap(&mq, q, s.heads, s.dim, tokens) || !MakeMap(&mk, k, s.kv_heads, s.dim, tokens) ||
      !MakeMap(&mv, v, s.kv_heads, s.dim, tokens))
    return cudaErrorInvalidValue;
  return s.dim <= 64 ? Forward<64>(s, mq, mk, mv, out, stats, status, stream) : Forward<128>(s, mq, mk, mv, out, stats, status, stream);
}

cudaError_t LaunchAttnBackward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                               const AttnTensor& out, const AttnTensor& dout, const float* stats, float* delta,
                               const AttnTensor& dq, const AttnTensor& dk, const AttnTensor& dv, unsigned int* status,
                               cudaStream_t stream) {
  (void)cudaGetLastError();
  const AttnTensor* all[8] = {&q, &k, &v, &out, &dout, &dq, &dk, &dv};
  for (const AttnTensor* t : all)
    if (!Addressable(*t)) return cudaErrorInvalidValue;
  if (!AttnSupported(s) || stats == nullptr || delta == nullptr || status == nullptr) return cudaErrorInvalidValue;
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  CUtensorMap mq, mk, mv, md;
  if (!MakeMap(&mq, q, s.heads, s.dim, tokens) || !MakeMap(&mk, k, s.kv_heads, s.dim, tokens) ||
      !MakeMap(&mv, v, s.kv_heads, s.dim, tokens) || !MakeMap(&md, dout, s.heads, s.dim, tokens))
    return cudaErrorInvalidValue;
  const Geo g = MakeGeo(s);
  attn_delta_kernel<<<static_cast<unsigned>(g.tiles) * g.heads, 256, 0, stream>>>(g, out, dout, delta);
  CountKernelLaunch();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  e = s.dim <= 64 ? Backward<64, true>(s, mq, mk, mv, md, stats, delta, dv, dk, status, stream)
                  : Backward<128, true>(s, mq, mk, mv, md, stats, delta, dv, dk, status, stream);
  if (e != cudaSuccess) return e;
  return s.dim <= 64 ? Backward<64, false>(s, mq, mk, mv, md, stats, delta, dq, dq, status, stream)
                     : Backward<128, false>(s, mq, mk, mv, md, stats, delta, dq, dq, status, stream);
}

}  // namespace bfb
