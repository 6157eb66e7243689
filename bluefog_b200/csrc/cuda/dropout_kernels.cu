// Dropout joined with the residual stream:  out = residual + keep * x / (1 - p),  and its backward pass  dx = keep * dy / (1 - p).
//
// The mask is never stored: keep(i) is a function of (seed, step, site, i), computed where it is needed by Philox4x32-10
// (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  One block
// of 128 bits serves eight elements, sixteen bits each: p is a multiple of 2^-16, and the factor is the inverse of the
// probability that is really used, so the expectation is exact.  A dropped element contributes zero whatever x holds.
//
// Bound by memory: x and residual are read and out is written once (6 bytes per bf16 element forward, 4 backward), which on 65536 x
// 2048 takes 121 and 95 us (6.6 and 5.7 TB/s).  Next to it stands the integer pipe: a block of Philox and eight tests take
// about 50 of its instructions, some 55 us on that tensor.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "comm_kernels.h"
#include "dropout_kernels.h"

namespace bfb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c.x) * 0xD2511F53u, b = uint64_t(c.z) * 0xCD9E8D57u;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ k0, uint32_t(b), uint32_t(a >> 32) ^ c.w ^ k1, uint32_t(a));
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// eight elements, the unit of a Philox block
template <typename T>
struct alignas(16) Eight {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> e;
  const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < int(sizeof(Eight<T>) / 16); ++i) reinterpret_cast<uint4*>(&e)[i] = s[i];
  return e;
}

// x becomes res + (keep ? factor * x : 0), in fp32 with one rounding to T.  A 16-bit word is compared where it stands, shifted to
// the upper half of its 32 bits (limit: threshold there), and the multiplication is predicated: what bounds the instruction count
// is the integer pipe.
template <typename T, bool RES>
__device__ __forceinline__ void apply(Eight<T>& x, const Eight<T>& res, const uint4 bits, const uint32_t limit, const bool none, float factor) {
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = (i & 1) ? w[i >> 1] : w[i >> 1] << 16;
    const float v = to_f(x.v[i]);
    float y = RES ? to_f(res.v[i]) : 0.f;
    if (u >= limit && !none) y = RES ? fmaf(v, factor, y) : v * factor;
    x.v[i] = from_f<T>(y);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < int(sizeof(Eight<T>) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&e)[i];
}

template <typename T, bool RES, int UNROLL>
__global__ void __launch_bounds__(kThreads)
dropout_add_kernel(const T* x, const T* residual, T* out, const long long n, const uint32_t threshold, const float factor,
                   const long long* __restrict__ key, const uint32_t site) {
  const unsigned long long seed = key[0], step = key[1];
  const uint32_t limit = threshold << 16;              // 65536 does not fit: then nothing is kept
  const bool none = threshold > 65535u;
  const long long groups = n / 8;
  auto bits = [&](long long g) {
    return philox(make_uint4(uint32_t(g), uint32_t(g >> 32) | site << 16, uint32_t(step), uint32_t(step >> 32)), uint32_t(seed), uint32_t(seed >> 32));
  };
  const long long stride = (long long)gridDim.x * (kThreads * UNROLL);
  long long g = (long long)blockIdx.x * (kThreads * UNROLL) + threadIdx.x;
  for (; g + (UNROLL - 1) * kThreads < groups; g += stride) {
    Eight<T> a[UNROLL], r[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      a[k] = load8(x + (g + k * kThreads) * 8);
      if (RES) r[k] = load8(residual + (g + k * kThreads) * 8);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      apply<T, RES>(a[k], r[k], bits(g + k * kThreads), limit, none, factor);
      store8(out + (g + k * kThreads) * 8, a[k]);
    }
  }
  for (; g <= groups; g += kThreads) {                 // what is left of the last round, and up to seven elements at the end
    if (g >= groups && groups * 8 == n) break;
    const int count = g < groups ? 8 : int(n - groups * 8);
    Eight<T> a = {}, r = {};
    for (int i = 0; i < 8; ++i)
      if (i < count) {
        a.v[i] = x[g * 8 + i];
        if (RES) r.v[i] = residual[g * 8 + i];
      }
    apply<T, RES>(a, r, bits(g), limit, none, factor);
    for (int i = 0; i < 8; ++i)
      if (i < count) out[g * 8 + i] = a.v[i];
    if (UNROLL == 1) break;
  }
}

template <typename T>
cudaError_t Launch(const void* x, const void* residual, void* out, long long n, unsigned int threshold, float factor,
                   const long long* key, unsigned int site, cudaStream_t stream) {
  int dev = 0, sms = 148;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const T* a = static_cast<const T*>(x);
  const T* r = static_cast<const T*>(residual);
  T* o = static_cast<T*>(out);
  // Loads in flight: two groups per stream and thread with a residual, four without (fp32: two of 32 bytes), where that leaves every
  // SM two blocks; with one, 65536 x 2048 bf16 takes 135 instead of 121 us with a residual and 102 instead of 95 us without.
  constexpr int kAlone = sizeof(T) == 4 ? 2 : 4;
  const int unroll = r != nullptr ? 2 : kAlone;
  const long long blocks = (n / 8 + kThreads) / kThreads;
  const bool wide = blocks >= 2ll * sms * unroll;
  const long long need = wide ? (blocks + unroll - 1) / unroll : blocks, most = (long long)sms * 32;
  const unsigned grid = static_cast<unsigned>(need < most ? need : most);
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(a, r, o, n, threshold, factor, key, site); };
  if (wide) r != nullptr ? go(dropout_add_kernel<T, true, 2>) : go(dropout_add_kernel<T, false, kAlone>);
  else r != nullptr ? go(dropout_add_kernel<T, true, 1>) : go(dropout_add_kernel<T, false, 1>);
  CountKernelLaunch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t LaunchDropoutAdd(const void* x, const void* residual, void* out, long long n, int type, unsigned int threshold,
                             float factor, const long long* key, unsigned int site, cudaStream_t stream) {
  (void)cudaGetLastError();   // the value returned below must be this launch's own, not an older error of the calling thread
  const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(out);
  if (n <= 0 || (n >> 51) != 0 || x == nullptr || out == nullptr || key == nullptr || (all & 15) != 0 || threshold > 65536u ||
      site > 65535u)
    return cudaErrorInvalidValue;
  switch (type) {
    case kDropF32: return Launch<float>(x, residual, out, n, threshold, factor, key, site, stream);
    case kDropF16: return Launch<__half>(x, residual, out, n, threshold, factor, key, site, stream);
    case kDropBF16: return Launch<__nv_bfloat16>(x, residual, out, n, threshold, factor, key, site, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace bfb
