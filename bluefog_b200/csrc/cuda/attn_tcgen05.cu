// Causal attention over packed sequences with grouped heads, forward and backward, on tcgen05 tensor cores.
//
//   forward   S = scale q k^T (key <= query, same sequence),  P = softmax(S),  out = P v
//   backward  delta = rowsum(dout * out),  dP = dout v^T,  dS = P (dP - delta)
//             dv = P^T dout (summed over the query heads of a group),  dk = scale dS^T q (ditto),  dq = scale dS k
//
// Head widths are padded to 64 or 128 columns: TMA fills the boxes up with zeros, and all MMA steps run over them (80 columns: eight
// steps in the scores where five hold data).  Two widths are compiled, not sixteen; for heads up to 64 the products are not what the
// time goes to (8 x 1024 tokens, 16 heads: 35 of 40 us without any), and what steps by the width would gain has not been measured.
//
// No kernel writes a score to memory: a CTA keeps 128 queries (or keys) and walks over the others 64 or 128 at a time.  The backward
// pass has two kinds of CTAs: those that own a key tile (dk, dv) and those that own a query tile (dq), seven products per tile
// instead of five, but no atomics, so gradients do not depend on the order in which CTAs run, and no fp32 copy of dq.
//
// Numbers: scores, row maxima, row sums, all accumulators and the statistics kept for the backward pass are fp32.  P and
// dS are rounded to bf16 because they are operands of the next product (each rounding is off by at most 2^-8 of the
// value, as the rounding of the result itself is).  So that delta does not suffer from the rounding of out - it is small against
// the dP that it is subtracted from only where many keys share the weight -, a forward pass with a backward pass to come
// also keeps the next eight bits of out (see low_bytes): without them dq and dk of 136 tokens are 1.6 times as far off as their
// own rounding alone, of 8 tokens 2.2 times, with them 1.45 and 1.5, for 4 of the 152 us of a GPT-2 medium layer.  A row's sum
// is taken over the unrounded values.
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
  int heads, kv_heads;
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

// Values that the kernel before may still be writing when this one starts (programmatic launch): an access in its place of the
// program, behind the wait, and past the L1 cache.  A const __restrict__ pointer would promise the compiler that they never change.
__device__ __forceinline__ float load_late(const float* p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
// Hand-over of what a thread has seen, in whichever kernel it was written, to a kernel that runs beside this one.
__device__ __forceinline__ void hand_over(unsigned int* word) { asm volatile("st.release.gpu.global.u32 [%0], 1;" ::"l"(word) : "memory"); }
__device__ __forceinline__ bool handed_over(const unsigned int* word) {
  unsigned int v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(word) : "memory");
  return v != 0u;
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

// Of four fp32 values, times factor, the eight bits that follow those of a bf16 number.  As a signed byte they are to be added to the
// rounded number in that place: rounding up added the carry that their sign takes back (with_low).  A tie that was rounded
// down, one value in 2^17, comes out an ulp too small.
__device__ __forceinline__ uint32_t low_bytes(const uint32_t* v, float factor) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
  return __byte_perm(__byte_perm(b[0], b[1], 0x0051), __byte_perm(b[2], b[3], 0x0051), 0x5410);
}
// byte i of `low` added to a bf16 number in the upper half of its word
__device__ __forceinline__ float with_low(uint32_t bf16, uint32_t low, int i) {
  return __uint_as_float(bf16 + static_cast<uint32_t>(static_cast<int>(low << (24 - 8 * i)) >> 16 & ~0xff));
}
// where eight of them lie in a box of [128 rows x 64 bytes]
__device__ __forceinline__ int low_at(int row, int chunk) { return (chunk >> 3) * (kTile * 64) + row * 64 + (((chunk & 7) ^ (row >> 1 & 7)) << 3); }

// two floats in one 64-bit register, and the packed instructions on them
typedef unsigned long long float2_t;
__device__ __forceinline__ float2_t pair(float lo, float hi) {
  float2_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(float2_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ float2_t fma2(float2_t a, float2_t b, float2_t c) {
  float2_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float2_t add2(float2_t a, float2_t b) {
  float2_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float2_t mul2(float2_t a, float2_t b) {
  float2_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// instruction descriptors: fp32 accumulator, bf16 operands, M = 128, N as given; B K-major or MN-major (bit 16)
constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
}

// scores[128 x N] = A B^T over DP columns; A: DP / 64 boxes of [128 rows x 64 columns] in shared memory, or 128 rows of DP bf16
// values in tensor memory; B: DP / 64 boxes of [N rows x 64 columns]
template <int DP, int N>
__device__ __forceinline__ void mma_scores(uint32_t tmem_d, uint32_t a, uint32_t b) {
  const uint64_t da = make_desc(a), db = make_desc(b);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    umma_f16(tmem_d, da + uint64_t(k >> 2) * (kBoxBytes >> 4) + uint64_t(k & 3) * 2, db + uint64_t(k >> 2) * (N * 128 >> 4) + uint64_t(k & 3) * 2,
             idesc(N, false), k != 0 ? 1u : 0u);
}
template <int DP, int N>
__device__ __forceinline__ void mma_scores_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b) {
  const uint64_t db = make_desc(b);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    umma_f16_ts(tmem_d, tmem_a + k * 8, db + uint64_t(k >> 2) * (N * 128 >> 4) + uint64_t(k & 3) * 2, idesc(N, false), k != 0 ? 1u : 0u);
}
// acc[128 x DP] += A B: A 128 x K bf16 in tensor memory, 32 elements (16 columns) every `a_step` columns; B = DP / 64 boxes of
// [K rows x 64 columns], read as an MN-major operand
template <int DP, int K>
__device__ __forceinline__ void mma_accumulate(uint32_t tmem_d, uint32_t a, uint32_t a_step, uint32_t b, bool first) {
  const uint64_t db = make_desc_mn(b, K * 128, 1024);
#pragma unroll
  for (int k = 0; k < K / 16; ++k)
    umma_f16_ts(tmem_d, a + uint32_t(k >> 1) * a_step + uint32_t(k & 1) * 8, db + uint64_t(k) * (2048 >> 4), idesc(DP, true),
                (first && k == 0) ? 0u : 1u);
}

// All warps of a block learn that its barriers and its tensor memory are there; the producer, which made the barriers and has no
// use for tensor memory, only says so and goes on loading.
template <int THREADS>
__device__ __forceinline__ void set_up_done(bool producer) {
  fence_before_sync();
  __syncwarp();
  if (producer) asm volatile("barrier.cta.arrive 15, %0;" ::"n"(THREADS) : "memory");
  else asm volatile("barrier.cta.sync 15, %0;" ::"n"(THREADS) : "memory");
  fence_after_sync();
}

// Zeros in rows [first, N) of DP / 64 boxes of N rows; called by a whole warp, visible to the tensor cores afterwards.
template <int DP, int N>
__device__ __forceinline__ void zero_rows(unsigned char* boxes, int first) {
  const int lane = threadIdx.x & 31;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  for (int b = 0; b < DP / 64; ++b)
    for (int c = first * 8 + lane; c < N * 8; c += 32) *reinterpret_cast<uint4*>(boxes + size_t(b) * (N * 128) + size_t(c) * 16) = z;
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
// warp's rows of a staging box (64 columns per box, starting with 16-byte chunk chunk0); their next bits go to `low`, boxes of
// 128 rows of 64 bytes, where that is given.
template <int NC>
__device__ __forceinline__ void stage_rows(uint32_t taddr, float factor, unsigned char* box, int row, int chunk0, unsigned char* low = nullptr) {
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
      if (low != nullptr) *reinterpret_cast<uint2*>(low + low_at(row, chunk)) = make_uint2(low_bytes(r + j * 8, factor), low_bytes(r + j * 8 + 4, factor));
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

// The same for the bytes of `low`, eight at a time.
template <int CHUNKS>
__device__ __forceinline__ void store_low(const AttnTensor& t, int head, int token0, int rows_left, int dim, const unsigned char* box,
                                          int row0, int chunk0) {
  const int lane = threadIdx.x & 31;
  const int last = min(chunk0 + CHUNKS, dim / 8) - chunk0;
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int r = (k * 32 + lane) / CHUNKS, c = (k * 32 + lane) % CHUNKS;
    if (r >= rows_left || c >= last) continue;
    *reinterpret_cast<uint2*>(static_cast<unsigned char*>(t.ptr) + (long long)(token0 + r) * t.token_stride + (long long)head * t.head_stride + (chunk0 + c) * 8) =
        *reinterpret_cast<const uint2*>(box + low_at(row0 + r, chunk0 + c));
  }
}

// ---------------------------------------------------------------------------------------------------------------- //
// Forward.  One CTA per tile of 128 queries and head, kN keys at a time.  The exponentials are what there is most of: 16 a cycle
// and SM, 1024 cycles per 128 x 128 scores against 512 (DP = 64) or 1024 of products.  One tile's chain - scores, maximum,
// exponentials, product - leaves that unit idle most of the time, so three CTAs (DP = 64: 64 keys, 128 tensor-memory columns each)
// or two (DP = 128: 128 keys, 256 columns) run on an SM and fill each other's waits, their beginnings and ends included.  Every
// softmax thread has 64 scores: a whole row of 64, or half a row of 128, the two threads of a row then exchanging maxima
// through shared memory.  P replaces the scores.  The output is rescaled only when a row's maximum grew by more than 2^8
// (the sums stay far inside fp32).  Keys are taken from the diagonal downwards, so that only the first tiles need a mask.
// ---------------------------------------------------------------------------------------------------------------- //
template <int DP>
struct FwdCfg {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kN = DP == 64 ? 64 : 128;        // keys of a tile
  static constexpr int kHalves = kN / 64;               // threads per row
  static constexpr int kWarps = 4 * kHalves;            // those that take exponentials
  static constexpr int kThreads = 32 * (kWarps + 2);
  static constexpr int kCtasPerSm = DP == 64 ? 3 : 2;
  static constexpr int kSlots = DP == 64 ? 4 : 2;       // ring of key / value tiles
  static constexpr uint32_t kQBytes = kBoxes * kBoxBytes;
  static constexpr uint32_t kYBytes = kBoxes * kN * 128;
  static constexpr uint32_t kCols = DP == 64 ? 128 : 256;
  static constexpr uint32_t kColO = kN;
  static constexpr size_t kSmem = 1024 + size_t(kQBytes) + size_t(kSlots) * kYBytes;
};

template <int DP>
__global__ void __launch_bounds__(FwdCfg<DP>::kThreads, FwdCfg<DP>::kCtasPerSm)
attn_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const Geo g, const AttnTensor out, const AttnTensor low,
                float* __restrict__ stats, const float scale_log2, unsigned int* __restrict__ status) {
  using Cfg = FwdCfg<DP>;
  constexpr int NS = Cfg::kSlots, N = Cfg::kN, H = Cfg::kHalves;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem_q = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem_q + Cfg::kQBytes;
  __shared__ uint64_t bars[2 * NS + 5];
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  __shared__ float maxima[2][H][kTile];
  volatile int* failed = &failed_s;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_q = bar0 + 8u * (2 * NS), bar_s = bar_q + 8u, bar_p = bar_q + 16u, bar_pv = bar_q + 24u, bar_end = bar_q + 32u;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (NS + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int order = divide(blockIdx.x, g.by_heads);
  const int head = blockIdx.x - order * g.heads;
  if (g.cu != nullptr && blockIdx.x == 0) {
    bool bad = threadIdx.x == 0 && __ldg(g.cu) != 0;   // taken as 0 all the same
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
  const int kv_head = divide(head, g.by_group);
  // key tiles: those that overlap the query tile in ascending order, so that every row sees a key in the first one, then downwards
  const int first = t.index * (kTile / N);
  const int diagonal = min((t.len - row0 + N - 1) / N, kTile / N);
  const int n = first + diagonal;
  auto key_tile = [&](int it) { return it < diagonal ? first + it : n - 1 - it; };

  int armed = 0;                                       // the producer's place: K0 V0 K1 V1 ...
  auto load = [&] {
    const int s = armed % NS;
    mbar_expect_tx(full(s), Cfg::kYBytes);
    for (int b = 0; b < Cfg::kBoxes; ++b)
      tma_load_3d(smem_u32(ring + size_t(s) * Cfg::kYBytes) + b * (N * 128), (armed & 1) ? &map_v : &map_k, full(s), b * 64, kv_head,
                  t.start + key_tile(armed >> 1) * N);
    ++armed;
  };
  if (warp == Cfg::kWarps && lane == 0) {
    failed_s = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(bar_q, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_p, Cfg::kWarps);
    mbar_init(bar_pv, 1);
    mbar_init(bar_end, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // the first two tiles travel while tensor memory is allocated
    mbar_expect_tx(bar_q, Cfg::kQBytes);
    for (int b = 0; b < Cfg::kBoxes; ++b) tma_load_3d(smem_u32(smem_q) + b * kBoxBytes, &map_q, bar_q, b * 64, head, t.start + row0);
    load();
  }
  if (warp == Cfg::kWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  set_up_done<Cfg::kThreads>(warp == Cfg::kWarps);

  if (warp == Cfg::kWarps) {
    if (lane == 0) {
      bool ok = true;
      while (armed < 2 * n) {
        ok = mbar_wait(empty(armed % NS), ((armed / NS) & 1) ^ 1, failed);
        if (!ok) break;
        load();
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
  } else if (warp == Cfg::kWarps + 1) {
    const uint32_t tmem = tmem_base_s;
    // the whole warp walks along, one lane issues; load 2 it is a key tile, 2 it + 1 a value tile
    auto slot = [&](int load) { return ring + size_t(load % NS) * Cfg::kYBytes; };
    auto arrived = [&](int load) { return mbar_wait(full(load % NS), (load / NS) & 1, failed); };
    auto scores = [&](int it) {
      mma_scores<DP, N>(tmem, smem_u32(smem_q), smem_u32(slot(2 * it)));
      umma_commit(empty((2 * it) % NS));
      umma_commit(bar_s);
    };
    bool ok = mbar_wait(bar_q, 0, failed) && arrived(0);
    if (ok && elect_one()) scores(0);
    __syncwarp();
    for (int it = 0; it < n && ok; ++it) {
      const bool more = it + 1 < n;
      ok = arrived(2 * it + 1);
      if (!ok) break;
      // P is zero behind the end of the sequence, which is not enough when the rows there hold infinities or NaN
      const int left = t.len - key_tile(it) * N;
      if (left < N) zero_rows<DP, N>(slot(2 * it + 1), left);
      // the next keys have arrived long ago; looked at here, their barrier is not between P and the products
      ok = (!more || NS == 2 || arrived(2 * it + 2)) && mbar_wait(bar_p, it & 1, failed);
      if (!ok) break;
      fence_after_sync();
      if (elect_one()) {
        mma_accumulate<DP, N>(tmem + Cfg::kColO, tmem, 16, smem_u32(slot(2 * it + 1)), it == 0);
        umma_commit(empty((2 * it + 1) % NS));
        umma_commit(bar_pv);
        if (more && NS > 2) scores(it + 1);            // over P: products run in the order of issue
      }
      __syncwarp();
      if (more && NS == 2) {                           // two slots: these keys could only be loaded after the scores before
        ok = arrived(2 * it + 2);
        if (ok && elect_one()) scores(it + 1);
        __syncwarp();
      }
    }
    if (!ok || *failed) {
      if (elect_one()) {
        umma_commit(bar_end);                          // tensor memory is not freed under a product
        const long long t0 = clock64();
        while (!mbar_try(bar_end, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
      __syncwarp();
    }
  } else {
    const uint32_t tmem = tmem_base_s;
    const int half = warp >> 2;                        // columns 64 half .. 64 half + 63
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + half * 64, tO = tmem + lanes + Cfg::kColO + half * (DP / H), tP = tmem + lanes + half * 32;
    // the two warps of 32 rows
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
    const float2_t scale2 = pair(scale_log2, scale_log2);
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
      if (it < diagonal) {
        const int last = row - it * N - half * 64;     // last column that this row sees
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c > last) r[c] = 0xff800000u;            // -inf
      }
      float mx[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) mx[k] = max_nan(__uint_as_float(r[k]), __uint_as_float(r[k + 4]));
#pragma unroll
      for (int c = 8; c < 64; c += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = max3_nan(mx[k], __uint_as_float(r[c + k]), __uint_as_float(r[c + k + 4]));
      float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
      if (H == 2) {
        // two sets of cells in turn: a thread is at most one tile ahead of its partner.  P may replace the scores afterwards.
        maxima[it & 1][half][row] = top;
        pair_sync();
        top = max_nan(top, maxima[it & 1][half ^ (H - 1)][row]);
      }
      if (it == 0) {
        m = top;
      } else {
        const bool grown = !((top - m) * scale_log2 <= 8.f);
        if (__any_sync(0xffffffffu, grown)) {
          // rare.  The product before these scores is complete.  A row that did not grow keeps its reference, so that its
          // bits do not depend on what the warp's other rows hold.
          const float next = grown ? max_nan(m, top) : m;
          const float f = ex2((m - (next == -INFINITY ? 0.f : next)) * scale_log2);
          m = next;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < DP / H; c += 16) {
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
      const float2_t shift2 = pair(shift, shift);
      float2_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float a, b;
          unpair(fma2(pair(__uint_as_float(r[h * 32 + 2 * c]), __uint_as_float(r[h * 32 + 2 * c + 1])), scale2, shift2), a, b);
          a = ex2(a);
          b = ex2(b);
          sum[c & 1] = add2(sum[c & 1], pair(a, b));
          p[c] = pack_bf16(a, b);
        }
        tmem_st16(tP + h * 16, p);
      }
      float lo, hi;
      unpair(add2(sum[0], sum[1]), lo, hi);
      l += lo + hi;
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p);
    }
    if (H == 2) {
      // the row's sum is in two places
      maxima[n & 1][half][row] = l;
      pair_sync();
      l += maxima[n & 1][half ^ (H - 1)][row];
    }
    if (ok && mbar_wait(bar_pv, (n - 1) & 1, failed)) {
      fence_after_sync();
      // all tiles have been used: the ring has room for the low bits
      stage_rows<DP / H / 32>(tO, 1.f / l, smem_q, row, half * (DP / H / 8), low.ptr != nullptr ? ring : nullptr);
      __syncwarp();
      const int left = t.len - row0 - (row & ~31);
      store_rows<DP / H / 8>(out, head, t.start + row0 + (row & ~31), left, g.dim, smem_q, row & ~31, half * (DP / H / 8));
      if (low.ptr != nullptr) store_low<DP / H / 8>(low, head, t.start + row0 + (row & ~31), left, g.dim, ring, row & ~31, half * (DP / H / 8));
      if (stats != nullptr && half == 0)
        stats[((long long)head * g.tiles + t.slot) * kTile + row] = lane < left ? -fmaf(m, scale_log2, log2f(l)) : -INFINITY;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == Cfg::kWarps + 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_s), "r"(Cfg::kCols) : "memory");
  }
  if (threadIdx.x == 0 && failed_s) atomicOr(status, kAttnTimeout);
}

// ---------------------------------------------------------------------------------------------------------------- //
// delta[head, row] = - sum_d dout * out, out with its low bits, one tile and head per block; rows that belong to no token get 0.  LANES threads per row,
// eight values each.  Clears the word by which the key tiles tell the query tiles that all this has ended.
// ---------------------------------------------------------------------------------------------------------------- //
template <int LANES>
__global__ void __launch_bounds__(256) attn_delta_kernel(const Geo g, const AttnTensor out, const AttnTensor low, const AttnTensor dout, float* __restrict__ delta,
                                                         unsigned int* __restrict__ delta_ready) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *delta_ready = 0u;
  const int order = divide(blockIdx.x, g.by_heads);
  const int head = blockIdx.x - order * g.heads;
  Tile t;
  if (!find_tile(g, order, true, t) || (g.cu != nullptr && t.batch == g.batch)) return;
  let_next_kernel_start();
  constexpr int kRows = 256 / LANES, kFlight = 4;      // rows of a pass, and passes whose loads are in flight together
  const int sub = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
  auto place = [&](const AttnTensor& x, int row) { return (long long)(t.start + row) * x.token_stride + (long long)head * x.head_stride + sub * 8; };
#pragma unroll 1
  for (int first = 0; first < kTile; first += kFlight * kRows) {
    uint4 a[kFlight], c[kFlight];
    uint2 b[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int row = t.index * kTile + first + r0 + k * kRows;
      a[k] = c[k] = make_uint4(0u, 0u, 0u, 0u);
      b[k] = make_uint2(0u, 0u);
      if (row < t.len && sub * 8 < g.dim) {
        a[k] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(out.ptr) + place(out, row));
        b[k] = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(low.ptr) + place(low, row));
        c[k] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(dout.ptr) + place(dout, row));
      }
    }
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const uint32_t x[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, z[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t y = i < 2 ? b[k].x : b[k].y;
        s = fmaf(with_low(x[i] << 16, y, 2 * (i & 1)), __uint_as_float(z[i] << 16),
                 fmaf(with_low(x[i] & 0xffff0000u, y, 2 * (i & 1) + 1), __uint_as_float(z[i] & 0xffff0000u), s));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (sub == 0) delta[((long long)head * g.tiles + t.slot) * kTile + first + r0 + k * kRows] = -s;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- //
// Backward.  KV: a CTA owns a tile of 128 keys of one key head and walks over the queries at and after it, 64 at a time, for every
// query head of the group; scores are held transposed (rows = keys), so P^T and dS^T are the tensor-memory operands of
// dv += P^T dout and dk += dS^T q, and the row statistics are per column.  Otherwise a CTA owns a tile of 128 queries of one
// head and walks over the keys from the diagonal downwards, 64 at a time: dq += dS k.  Both kinds are blocks of one launch.
// What limits this is the chain products -> exponentials -> products of one tile, so two chains run side by side on an SM: two CTAs
// of 256 tensor-memory columns for DP = 64, two sets of eight warps with score buffers of their own in one CTA for DP = 128
// (with 128 columns at a time and one chain the layer of GPT-2 medium took 93 + 71 us, 3100 and 2270 cycles per 128 x 128 tile,
// against the 1024 that its exponentials need).  Eight warps take one 128 x 64 tile, two per quarter of tensor memory with 32
// columns of it.  Their bf16 operands replace the fp32 values that the same warp has read.  Products with 64 columns whose first
// operand comes from shared memory are bound by the reads of that operand (48 cycles instead of 32 per 16 elements), so the
// query kind keeps q and dout in tensor memory; the key kind has no room for that.
// ---------------------------------------------------------------------------------------------------------------- //
template <int DP>
struct BwdCfg {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kN = 64;                                        // rows of a streamed tile
  static constexpr uint32_t kXBytes = kBoxes * kBoxBytes;              // each of the two resident tiles
  static constexpr uint32_t kYBytes = kBoxes * kN * 128;               // each of the two streamed tiles of a stage
  static constexpr int kStages = 4;
  static constexpr int kSets = DP == 64 ? 1 : 2;
  static constexpr bool kEarly = kSets == 1;                           // see the products
  static constexpr int kWarps = 8 * kSets;                             // those that take exponentials
  static constexpr int kThreads = 32 * (kWarps + 2);
  static constexpr int kCtasPerSm = DP == 64 ? 2 : 1;
  static constexpr uint32_t kCols = DP == 64 ? 256 : 512;
  static constexpr uint32_t kCol1 = kCols - DP, kCol0 = kCol1 - DP;    // accumulators of dk / dq and of dv
  static constexpr uint32_t kColX = 128 * kSets;                       // queries: q and dout as operands, DP / 2 columns each
  static constexpr size_t kSmem = 1024 + 2 * size_t(kXBytes) + size_t(kStages) * (2 * kYBytes + 2 * kN * 4);
};

// dv and dk of a key tile from the fp32 sums of the SPLIT CTAs of the cluster ([2][128][DP] at `sums` in each, 16-byte chunks swizzled
// within 128 bytes): this CTA's 128 / SPLIT rows, the CTAs in the order of their heads.  All loads of a chunk are in flight
// together, since each takes about a microsecond.
template <int DP, int SPLIT>
__device__ __forceinline__ void add_up(const uint32_t sums, const int rank, const int head, const int token0, const int rows_left, const int dim,
                                       const float scale, const AttnTensor& dv, const AttnTensor& dk, const int threads) {
  constexpr int kRows = kTile / SPLIT, kChunks = DP / 8;
  for (int i = threadIdx.x; i < 2 * kRows * kChunks; i += threads) {
    const int chunk = i % kChunks, rest = i / kChunks;
    const bool second = rest >= kRows;
    const int row = rank * kRows + rest % kRows;
    const uint32_t at = sums + (second ? kTile * DP * 4 : 0) + row * (DP * 4) + (chunk >> 2) * 128;
    const uint32_t lo = at + ((((chunk & 3) * 2) ^ (row & 7)) << 4), hi = at + ((((chunk & 3) * 2 + 1) ^ (row & 7)) << 4);
    float4 a[SPLIT], b[SPLIT];
#pragma unroll
    for (int c = 0; c < SPLIT; ++c) {
      a[c] = ld_cluster_v4(mapa_u32(lo, c));
      b[c] = ld_cluster_v4(mapa_u32(hi, c));
    }
#pragma unroll
    for (int c = 1; c < SPLIT; ++c) {
      a[0].x += a[c].x, a[0].y += a[c].y, a[0].z += a[c].z, a[0].w += a[c].w;
      b[0].x += b[c].x, b[0].y += b[c].y, b[0].z += b[c].z, b[0].w += b[c].w;
    }
    if (row < rows_left && chunk * 8 < dim) {
      const float f = second ? scale : 1.f;
      const AttnTensor& d = second ? dk : dv;
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(d.ptr) + (long long)(token0 + row) * d.token_stride + (long long)head * d.head_stride + chunk * 8) =
          make_uint4(pack_bf16(a[0].x * f, a[0].y * f), pack_bf16(a[0].z * f, a[0].w * f), pack_bf16(b[0].x * f, b[0].y * f), pack_bf16(b[0].z * f, b[0].w * f));
    }
  }
}

template <int DP, bool KV>
__device__ __forceinline__ void attn_bwd_body(const CUtensorMap* map_q, const CUtensorMap* map_k, const CUtensorMap* map_v, const CUtensorMap* map_do,
                                              const Geo& g, const int block, const int split, unsigned int* const delta_ready, const float* stats, const float* delta,
                                              const AttnTensor& d0, const AttnTensor& d1, const float scale, const float scale_log2,
                                              unsigned int* __restrict__ status) {
  using Cfg = BwdCfg<DP>;
  constexpr int NS = Cfg::kStages, SETS = Cfg::kSets, N = Cfg::kN;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem_x = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem_x + 2 * Cfg::kXBytes;
  float* ring_stats = reinterpret_cast<float*>(ring + size_t(NS) * 2 * Cfg::kYBytes);      // KV: per stage -lse[64], -delta[64]
  __shared__ uint64_t bars[2 * NS + 3 + 4 * SETS];
  __shared__ uint32_t tmem_base_s;
  __shared__ int failed_s;
  volatile int* failed = &failed_s;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_x = bar0 + 8u * (2 * NS), bar_xa = bar_x + 8u, bar_end = bar_x + 16u;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (NS + s); };
  // bar_p: the scores' place may be used, KV: as the operand P that replaced them, otherwise for the next scores
  auto bar_s = [&](int set) { return bar_x + 24u + 32u * set; };
  auto bar_dp = [&](int set) { return bar_x + 32u + 32u * set; };
  auto bar_p = [&](int set) { return bar_x + 40u + 32u * set; };
  auto bar_ds = [&](int set) { return bar_x + 48u + 32u * set; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // KV: `split` CTAs of a cluster (a power of two) share a tile, each with its part of the group's query heads
  const int part_of_group = KV ? block & (split - 1) : 0;
  const int item = KV ? block >> (__ffs(split) - 1) : block;
  const int own_heads = KV ? g.kv_heads : g.heads;
  const int order = divide(item, KV ? g.by_kv_heads : g.by_heads);
  const int own_head = item - order * own_heads;
  const int first_head = KV ? own_head * g.group + part_of_group * (g.group >> (__ffs(split) - 1)) : divide(own_head, g.by_group);
  Tile t;
  if (!find_tile(g, order, !KV, t)) return;
  const int row0 = t.index * kTile;
  if (g.cu != nullptr && t.batch == g.batch) {
    if (part_of_group != 0) return;
    if (KV) zero_result(d0, own_head, t.start + row0, t.start + t.len, g.dim);
    zero_result(d1, own_head, t.start + row0, t.start + t.len, g.dim);
    return;
  }
  const int seq_parts = (t.len + N - 1) / N;           // streamed tiles of the sequence
  const int first_part = KV ? 2 * t.index : min(2 * t.index + 1, seq_parts - 1);
  const int per_head = KV ? seq_parts - first_part : first_part + 1;
  const int n = KV ? per_head * (g.group >> (__ffs(split) - 1)) : per_head;
  const int first_slot = t.slot - t.index;

  // the producer's place: tiles loaded so far, the next one and its head
  int armed = 0, next_part = first_part, next_head = first_head;
  auto load = [&] {
    const int s = armed % NS;
    const uint32_t dst = smem_u32(ring + size_t(s) * 2 * Cfg::kYBytes);
    mbar_expect_tx(full(s), 2 * Cfg::kYBytes + (KV ? 2 * N * 4 : 0));
    for (int b = 0; b < Cfg::kBoxes; ++b) {
      tma_load_3d(dst + b * (N * 128), KV ? map_q : map_k, full(s), b * 64, next_head, t.start + next_part * N);
      tma_load_3d(dst + Cfg::kYBytes + b * (N * 128), KV ? map_do : map_v, full(s), b * 64, next_head, t.start + next_part * N);
    }
    if (KV) {
      const long long at = ((long long)next_head * g.tiles + first_slot) * kTile + next_part * N;
      bulk_load(smem_u32(ring_stats + s * 2 * N), stats + at, full(s), N * 4);
      bulk_load(smem_u32(ring_stats + s * 2 * N + N), delta + at, full(s), N * 4);
      if (++next_part == seq_parts) {
        next_part = first_part;
        ++next_head;
      }
    } else {
      --next_part;
    }
    ++armed;
  };
  if (warp == Cfg::kWarps && lane == 0) {
    failed_s = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(bar_x, 1);
    mbar_init(bar_xa, 8);
    mbar_init(bar_end, 1);
    for (int k = 0; k < SETS; ++k) {
      mbar_init(bar_s(k), 1);
      mbar_init(bar_dp(k), 1);
      mbar_init(bar_p(k), 8);
      mbar_init(bar_ds(k), 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // the resident tiles and the first streamed ones travel while tensor memory is allocated; every box holds 64 rows
    mbar_expect_tx(bar_x, 2 * Cfg::kXBytes);
    const CUtensorMap* m0 = KV ? map_k : map_q;
    const CUtensorMap* m1 = KV ? map_v : map_do;
    for (int b = 0; b < Cfg::kBoxes; ++b)
      for (int h = 0; h < 2; ++h) {
        const uint32_t dst = smem_u32(smem_x) + b * kBoxBytes + h * (kBoxBytes / 2);
        tma_load_3d(dst, m0, bar_x, b * 64, own_head, t.start + row0 + h * 64);
        tma_load_3d(dst + Cfg::kXBytes, m1, bar_x, b * 64, own_head, t.start + row0 + h * 64);
      }
    if (KV) {
      wait_for_kernel_before();                        // delta
      if (split > 1) hand_over(delta_ready);           // the query tiles are a launch of their own
      let_next_kernel_start();
    }
    load();
  }
  if (warp == Cfg::kWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(Cfg::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  set_up_done<Cfg::kThreads>(warp == Cfg::kWarps);

  if (warp == Cfg::kWarps) {
    if (lane == 0) {
      bool ok = true;
      while (armed < n) {
        ok = mbar_wait(empty(armed % NS), ((armed / NS) & 1) ^ 1, failed);
        if (!ok) break;
        load();
      }
      if (!ok || *failed) {
        // copies in flight have to land before this shared memory goes away
        for (int f = armed > NS ? armed - NS : 0; f < armed; ++f) {
          const long long t0 = clock64();
          while (!mbar_try(full(f % NS), (f / NS) & 1) && clock64() - t0 < kWaitLimitCycles) {}
        }
        const long long t0 = clock64();
        while (!mbar_try(bar_x, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
    }
  } else if (warp == Cfg::kWarps + 1) {
    const uint32_t tmem = tmem_base_s;
    const uint32_t x0 = smem_u32(smem_x), x1 = x0 + Cfg::kXBytes;
    auto stage = [&](int it) { return ring + size_t(it % NS) * 2 * Cfg::kYBytes; };
    auto s_col = [&](int it) { return tmem + uint32_t(it % SETS) * 128u; };
    bool ok = mbar_wait(KV ? bar_x : bar_xa, 0, failed);
    fence_after_sync();
    int part = first_part;
    // waits for the tiles of an iteration
    auto tiles = [&](int it) {
      if (!mbar_wait(full(it % NS), (it / NS) & 1, failed)) return false;
      if (t.len - part * N < N) {                      // rows behind the end of the sequence take part in the reductions
        zero_rows<DP, N>(stage(it), t.len - part * N);
        zero_rows<DP, N>(stage(it) + Cfg::kYBytes, t.len - part * N);
      }
      if (KV) {
        if (++part == seq_parts) part = first_part;
      } else {
        --part;
      }
      return true;
    };
    // Scores and dP of an iteration replace the operands of the set's tile before; products run in the order of issue.  With one
    // set the next scores are issued as soon as their place is free (kEarly), so that the set finds them ready when it has
    // written dS, and its exponentials cover the way of dS through the products and of the next dP (8192 tokens, heads of 64: 572
    // -> 519 us).  With two sets, whose products fill that time, the additional hand-over costs (heads of 128: 829 -> 898 us).
    auto scores = [&](int it) {
      const uint32_t y = smem_u32(stage(it));
      if (KV) mma_scores<DP, N>(s_col(it), x0, y);
      else mma_scores_ts<DP, N>(s_col(it), tmem + Cfg::kColX, y);
      umma_commit(bar_s(it % SETS));
    };
    auto grad_scores = [&](int it) {
      const uint32_t y = smem_u32(stage(it)) + Cfg::kYBytes;
      if (KV) mma_scores<DP, N>(s_col(it) + N, x1, y);
      else mma_scores_ts<DP, N>(s_col(it) + N, tmem + Cfg::kColX + DP / 2, y);
      umma_commit(bar_dp(it % SETS));
    };
    for (int it = 0; it < SETS && it < n && ok; ++it) {
      ok = tiles(it);
      if (ok && elect_one()) {
        scores(it);
        grad_scores(it);
      }
      __syncwarp();
    }
    for (int it = 0; it < n && ok; ++it) {
      const bool more = it + SETS < n;
      const uint32_t phase = (it / SETS) & 1;
      // the next tiles have arrived long ago; looked at here, their barrier is not between the operands and the products
      ok = !more || tiles(it + SETS);
      if (Cfg::kEarly) {
        ok = ok && mbar_wait(bar_p(it % SETS), phase, failed);
        if (!ok) break;
        fence_after_sync();
        if (elect_one()) {
          if (KV) mma_accumulate<DP, N>(tmem + Cfg::kCol0, s_col(it), 32, smem_u32(stage(it)) + Cfg::kYBytes, it == 0);
          if (more) scores(it + SETS);
        }
        __syncwarp();
      }
      ok = ok && mbar_wait(bar_ds(it % SETS), phase, failed);
      if (!ok) break;
      fence_after_sync();
      if (elect_one()) {
        if (KV && !Cfg::kEarly) mma_accumulate<DP, N>(tmem + Cfg::kCol0, s_col(it), 32, smem_u32(stage(it)) + Cfg::kYBytes, it == 0);
        mma_accumulate<DP, N>(tmem + Cfg::kCol1, s_col(it) + N, 32, smem_u32(stage(it)), it == 0);
        umma_commit(empty(it % NS));
        if (!Cfg::kEarly && more) scores(it + SETS);
        if (more) grad_scores(it + SETS);
      }
      __syncwarp();
    }
    if (elect_one()) {
      umma_commit(bar_end);
      if (!ok || *failed) {                            // tensor memory is not freed under a product
        const long long t0 = clock64();
        while (!mbar_try(bar_end, 0) && clock64() - t0 < kWaitLimitCycles) {}
      }
    }
    __syncwarp();
  } else {
    const uint32_t tmem = tmem_base_s;
    const int set = warp >> 3, half = (warp >> 2) & 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    bool ok = true;
    // A thread holds eight columns of four rows: with a row per thread every thread would read the statistics of all its columns,
    // and the shared memory that the products read from was what the exponentials of the key kind waited for.
    const int sub_row = (warp & 3) * 32 + (lane >> 2), sub_col = half * 32 + (lane & 3) * 2;
    float2_t lse2[4], dlt2[4];                         // KV: column pairs 8 g + sub_col; otherwise rows sub_row + 8 k, twice
    if (!KV) {
      // delta.  As a launch of their own the query tiles run beside the key tiles, all of which have waited for it and said so before
      // these blocks can start; to wait for the launch of the key tiles itself is right as well, but lets nothing run beside it.
      if (delta_ready == nullptr || !handed_over(delta_ready)) wait_for_kernel_before();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long at = ((long long)own_head * g.tiles + t.slot) * kTile + sub_row + 8 * k;
        const float lse = load_late(stats + at), dlt = load_late(delta + at);
        lse2[k] = pair(lse, lse);
        dlt2[k] = pair(dlt, dlt);
      }
      if (set == 0) {
        // q (first half of the warps) or dout (second) from shared to tensor memory, a row per thread
        ok = mbar_wait(bar_x, 0, failed);
#pragma unroll
        for (int b = 0; b < Cfg::kBoxes; ++b) {
          uint32_t r[32];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(smem_x + half * Cfg::kXBytes + b * kBoxBytes + row * 128 + ((c ^ (row & 7)) << 4));
            r[c * 4] = v.x;
            r[c * 4 + 1] = v.y;
            r[c * 4 + 2] = v.z;
            r[c * 4 + 3] = v.w;
          }
          tmem_st32(tmem + lanes + Cfg::kColX + half * (DP / 2) + b * 32, r);
        }
        tmem_wait_st();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_xa);
      }
    }
    const float2_t scale2 = pair(scale_log2, scale_log2);
    const uint32_t tS = tmem + lanes + set * 128u + half * 32u, tD = tS + N, kUpper = 16u << 16;
    int part = 0;                                      // streamed tile, counted from the first one of a head
    for (int it = set; it < n; it += SETS) {
      if (it == set) part = set;
      else part += SETS;
      while (part >= per_head) part -= per_head;
      // columns from here on belong to rows of the tile (KV: queries at and after the first key), so a mask is needed
      const bool diagonal = KV ? part < 2 : it < first_part - 2 * t.index + 1;
      const uint32_t phase = (it / SETS) & 1;
      if (KV) {
        const float* st = ring_stats + (it % NS) * 2 * N + sub_col;
        ok = ok && mbar_wait(full(it % NS), (it / NS) & 1, failed);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lse2[k] = *reinterpret_cast<const float2_t*>(st + 8 * k);
          dlt2[k] = *reinterpret_cast<const float2_t*>(st + N + 8 * k);
        }
      }
      ok = ok && mbar_wait(bar_s(set), phase, failed);
      if (!ok) break;
      fence_after_sync();
      uint32_t r[32];                                  // 16 u + 4 g + 2 b + e: row sub_row + 16 u + 8 b, column sub_col + 8 g + e
      tmem_ld_16x256b_x4(tS, r);
      tmem_ld_16x256b_x4(tS + kUpper, r + 16);
      tmem_wait_ld();
      tie32(r);
      if (Cfg::kEarly && !KV) {
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(set));
      }
      float p[32];
#pragma unroll
      for (int i = 0; i < 32; i += 2)
        unpair(fma2(pair(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), scale2, lse2[KV ? (i >> 2) & 3 : i >> 4 << 1 | ((i >> 1) & 1)]),
               p[i], p[i + 1]);
#pragma unroll
      for (int i = 0; i < 32; ++i) p[i] = ex2(p[i]);
      if (diagonal) {
        const int over = sub_col + (KV ? part * N : (first_part - it - 2 * t.index) * N) - sub_row;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int d = over + ((i >> 2) & 3) * 8 + (i & 1) - (i >> 4) * 16 - ((i >> 1) & 1) * 8;       // column - row
          if (KV ? d < 0 : d > 0) p[i] = 0.f;
        }
      }
      uint32_t pk[16];
      if (KV) {
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16(p[2 * i], p[2 * i + 1]);
        tmem_st_16x128b_x4(tS, pk);
        tmem_st_16x128b_x4(tS + kUpper, pk + 8);
        if (Cfg::kEarly) {
          tmem_wait_st();
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p(set));
        }
      }
      ok = mbar_wait(bar_dp(set), phase, failed);
      if (!ok) break;
      fence_after_sync();
      tmem_ld_16x256b_x4(tD, r);
      tmem_ld_16x256b_x4(tD + kUpper, r + 16);
      tmem_wait_ld();
      tie32(r);
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float x, y;
        unpair(mul2(pair(p[i], p[i + 1]), add2(pair(__uint_as_float(r[i]), __uint_as_float(r[i + 1])),
                                               dlt2[KV ? (i >> 2) & 3 : i >> 4 << 1 | ((i >> 1) & 1)])), x, y);
        pk[i / 2] = pack_bf16(x, y);
      }
      tmem_st_16x128b_x4(tD, pk);
      tmem_st_16x128b_x4(tD + kUpper, pk + 8);
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_ds(set));
    }
    if (ok && mbar_wait(bar_end, 0, failed) && !*failed) {
      fence_after_sync();
      // the ring is at rest: staging boxes for the results
      const int left = t.len - row0 - (row & ~31);
      const int token0 = t.start + row0 + (row & ~31);
      if (KV && split > 1) {
        // fp32 sums of this CTA's query heads for the cluster: rows of DP values, 16-byte chunks swizzled within 128 bytes
        const bool second = SETS == 1 ? half == 1 : set == 1;
        const int col = SETS == 1 ? 0 : half * 64;
        unsigned char* sums = ring + (second ? kTile * DP * 4 : 0) + row * (DP * 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t r[32];
          tmem_ld32(tmem + lanes + (second ? Cfg::kCol1 : Cfg::kCol0) + col + c * 32, r);
          tmem_wait_ld();
          tie32(r);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(sums + (col / 32 + c) * 128 + ((j ^ (row & 7)) << 4)) = make_uint4(r[j * 4], r[j * 4 + 1], r[j * 4 + 2], r[j * 4 + 3]);
        }
      } else if (KV) {
        // dv by the first half of the warps, dk by the second; 64 columns per thread
        const bool second = SETS == 1 ? half == 1 : set == 1;
        const int col = SETS == 1 ? 0 : half * 64;
        unsigned char* box = ring + (second ? Cfg::kXBytes : 0);
        stage_rows<2>(tmem + lanes + (second ? Cfg::kCol1 : Cfg::kCol0) + col, second ? scale : 1.f, box, row, col / 8);
        __syncwarp();
        store_rows<8>(second ? d1 : d0, own_head, token0, left, g.dim, box, row & ~31, col / 8);
      } else {
        const int col = (set * 2 + half) * 32;
        stage_rows<1>(tmem + lanes + Cfg::kCol1 + col, scale, ring, row, col / 8);
        __syncwarp();
        store_rows<4>(d1, own_head, token0, left, g.dim, ring, row & ~31, col / 8);
      }
    }
  }
  if (KV && split > 1) {
    // every CTA of the cluster adds up 128 / split rows of all of them, in the order of the heads
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp < Cfg::kWarps) {
      if (split == 2) add_up<DP, 2>(smem_u32(ring), part_of_group, own_head, t.start + row0, t.len - row0, g.dim, scale, d0, d1, 32 * Cfg::kWarps);
      else if (split == 4) add_up<DP, 4>(smem_u32(ring), part_of_group, own_head, t.start + row0, t.len - row0, g.dim, scale, d0, d1, 32 * Cfg::kWarps);
      else add_up<DP, 8>(smem_u32(ring), part_of_group, own_head, t.start + row0, t.len - row0, g.dim, scale, d0, d1, 32 * Cfg::kWarps);
    }
    // nobody leaves while another may still read its shared memory
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  if (warp == Cfg::kWarps + 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_s), "r"(Cfg::kCols) : "memory");
  }
  if (threadIdx.x == 0 && failed_s) atomicOr(status, kAttnTimeout);
}

// The first kv_blocks blocks own key tiles (`split` of a cluster share one), the others query tiles.  The kernel starts while the one
// that computes delta still runs, and waits for it where it reads that.  Query tiles alone (no kv_blocks) start beside the launch of the
// key tiles, whose blocks let them in only after they have waited for delta.  That alone orders no memory accesses, so they also
// hand over what they have seen (delta_ready).
template <int DP>
__global__ void __launch_bounds__(BwdCfg<DP>::kThreads, BwdCfg<DP>::kCtasPerSm)
attn_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Geo g, const int kv_blocks, const int split,
                const float* stats, const float* delta, unsigned int* const delta_ready, const AttnTensor dq, const AttnTensor dk,
                const AttnTensor dv, const float scale, const float scale_log2, unsigned int* __restrict__ status) {
  if (int(blockIdx.x) < kv_blocks)
    attn_bwd_body<DP, true>(&map_q, &map_k, &map_v, &map_do, g, blockIdx.x, split, delta_ready, stats, delta, dv, dk, scale, scale_log2, status);
  else
    attn_bwd_body<DP, false>(&map_q, &map_k, &map_v, &map_do, g, blockIdx.x - kv_blocks, 1, kv_blocks == 0 ? delta_ready : nullptr, stats, delta, dq, dq, scale,
                             scale_log2, status);
  wait_for_kernel_before();                            // the end of this launch is the end of those before it
}

__global__ void take_status_kernel(unsigned int* status, unsigned int* value) { *value = atomicExch(status, 0u); }

// ---- host side ---------------------------------------------------------------------------------------------------

bool MakeMap(CUtensorMap* map, const AttnTensor& t, int heads, int dim, long long tokens, int rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(t.head_stride) * 2, static_cast<cuuint64_t>(t.token_stride) * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
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
  g.kv_heads = s.kv_heads;
  g.group = s.heads / s.kv_heads;
  g.dim = s.dim;
  g.by_heads = MakeDivisor(s.heads);
  g.by_kv_heads = MakeDivisor(s.kv_heads);
  g.by_batch = MakeDivisor(s.batch);
  g.by_group = MakeDivisor(g.group);
  return g;
}

int SmCount() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  return n;
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
                    const AttnTensor& low, float* stats, unsigned int* status, cudaStream_t stream) {
  constexpr auto kernel = attn_fwd_kernel<DP>;
  using Cfg = FwdCfg<DP>;
  const cudaError_t e = AllowSmem<kernel>(Cfg::kSmem);
  if (e != cudaSuccess) return e;
  const Geo g = MakeGeo(s);
  kernel<<<static_cast<unsigned>(g.tiles) * g.heads, Cfg::kThreads, Cfg::kSmem, stream>>>(mq, mk, mv, g, out, low, stats, s.scale * kLog2e, status);
  CountKernelLaunch();
  return cudaGetLastError();
}

template <int DP>
cudaError_t Backward(const AttnShape& s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& md,
                     const float* stats, const float* delta, unsigned int* delta_ready, const AttnTensor& dq, const AttnTensor& dk, const AttnTensor& dv,
                     unsigned int* status, cudaStream_t stream) {
  constexpr auto kernel = attn_bwd_kernel<DP>;
  using Cfg = BwdCfg<DP>;
  const cudaError_t e = AllowSmem<kernel>(Cfg::kSmem);
  if (e != cudaSuccess) return e;
  const Geo g = MakeGeo(s);
  // The query heads of a group add to the same key tile.  Up to eight CTAs of a cluster (the portable size) share them and add up
  // their sums through distributed shared memory: without it one CTA walked over all of them, and few key heads left SMs idle
  // (packed documents, four query heads to a key head: 380 against 330 us, forward included).  Three times as many blocks as run
  // together even out what they differ by; more only add sums.  The query kind then has a launch of its own, since blocks that
  // need no cluster would still be started as one.
  int split = 1;
  while (split < 8 && g.group % (2 * split) == 0 && g.tiles * s.kv_heads * split < 3 * SmCount() * Cfg::kCtasPerSm) split *= 2;
  const int kv_blocks = g.tiles * s.kv_heads * split, q_blocks = g.tiles * s.heads;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(split > 1 ? kv_blocks : kv_blocks + q_blocks));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  const float scale_log2 = s.scale * kLog2e;
  cudaError_t r = cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, md, g, kv_blocks, split, stats, delta, delta_ready, dq, dk, dv, s.scale, scale_log2, status);
  if (r != cudaSuccess) return r;
  CountKernelLaunch();
  if (split > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(q_blocks));
    cfg.numAttrs = 1;
    r = cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, md, g, 0, 1, stats, delta, delta_ready, dq, dk, dv, s.scale, scale_log2, status);
    if (r != cudaSuccess) return r;
    CountKernelLaunch();
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t LaunchTakeStatus(unsigned int* status, unsigned int* value, cudaStream_t stream) {
  (void)cudaGetLastError();
  if (status == nullptr || value == nullptr) return cudaErrorInvalidValue;
  take_status_kernel<<<1, 1, 0, stream>>>(status, value);
  CountKernelLaunch();
  return cudaGetLastError();
}

long long AttnTiles(const AttnShape& s) {
  return s.cu == nullptr ? s.batch * ((s.seq + kTile - 1) / kTile) : s.seq / kTile + s.batch + 1;
}

bool AttnSupported(const AttnShape& s) {
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  return GetEncodeFn() != nullptr && s.batch > 0 && s.seq > 0 && s.heads > 0 && s.kv_heads > 0 && s.heads % s.kv_heads == 0 &&
         s.dim >= 8 && s.dim <= 128 && s.dim % 8 == 0 && s.scale > 0.f && tokens < (1ll << 31) - 2 * kTile &&
         AttnTiles(s) * s.heads * 2 < (1ll << 31);
}

cudaError_t LaunchAttnForward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                              const AttnTensor& out, const AttnTensor& low, float* stats, unsigned int* status, cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  if (!AttnSupported(s) || !Addressable(q) || !Addressable(k) || !Addressable(v) || !Addressable(out) || status == nullptr ||
      (low.ptr != nullptr && !Addressable(low)))
    return cudaErrorInvalidValue;
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  const int keys = s.dim <= 64 ? FwdCfg<64>::kN : FwdCfg<128>::kN;
  CUtensorMap mq, mk, mv;
  if (!MakeMap(&mq, q, s.heads, s.dim, tokens, kTile) || !MakeMap(&mk, k, s.kv_heads, s.dim, tokens, keys) ||
      !MakeMap(&mv, v, s.kv_heads, s.dim, tokens, keys))
    return cudaErrorInvalidValue;
  return s.dim <= 64 ? Forward<64>(s, mq, mk, mv, out, low, stats, status, stream) : Forward<128>(s, mq, mk, mv, out, low, stats, status, stream);
}

cudaError_t LaunchAttnBackward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                               const AttnTensor& out, const AttnTensor& low, const AttnTensor& dout, const float* stats, float* delta,
                               const AttnTensor& dq, const AttnTensor& dk, const AttnTensor& dv, unsigned int* status,
                               cudaStream_t stream) {
  (void)cudaGetLastError();
  const AttnTensor* all[9] = {&q, &k, &v, &out, &low, &dout, &dq, &dk, &dv};
  for (const AttnTensor* t : all)
    if (!Addressable(*t)) return cudaErrorInvalidValue;
  if (!AttnSupported(s) || stats == nullptr || delta == nullptr || status == nullptr) return cudaErrorInvalidValue;
  const long long tokens = s.cu == nullptr ? s.batch * s.seq : s.seq;
  CUtensorMap mq, mk, mv, md;
  if (!MakeMap(&mq, q, s.heads, s.dim, tokens, 64) || !MakeMap(&mk, k, s.kv_heads, s.dim, tokens, 64) ||
      !MakeMap(&mv, v, s.kv_heads, s.dim, tokens, 64) || !MakeMap(&md, dout, s.heads, s.dim, tokens, 64))
    return cudaErrorInvalidValue;
  const Geo g = MakeGeo(s);
  const unsigned blocks = static_cast<unsigned>(g.tiles) * g.heads;
  unsigned int* ready = reinterpret_cast<unsigned int*>(delta + (long long)g.heads * g.tiles * kTile);
  if (s.dim <= 64) attn_delta_kernel<8><<<blocks, 256, 0, stream>>>(g, out, low, dout, delta, ready);
  else attn_delta_kernel<16><<<blocks, 256, 0, stream>>>(g, out, low, dout, delta, ready);
  CountKernelLaunch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return s.dim <= 64 ? Backward<64>(s, mq, mk, mv, md, stats, delta, ready, dq, dk, dv, status, stream)
                     : Backward<128>(s, mq, mk, mv, md, stats, delta, ready, dq, dk, dv, status, stream);
}

}  // namespace bfb
