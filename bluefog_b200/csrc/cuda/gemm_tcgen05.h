// bf16 GEMM on tcgen05 tensor cores (see gemm_tcgen05.cu).
#pragma once
#include <cuda_runtime.h>

namespace bfb {

enum GemmAct : int { kActNone = 0, kActRelu = 1, kActGeluTanh = 2, kActSilu = 3 };
// Extra work of the epilogue: store the pre-activation value (accumulator + bias) to a second matrix besides
// act(...) of it; or multiply the result by GELU'(aux[m, n]) (the input gradient through a GELU whose
// pre-activation was kept); or one half of a gated feed-forward block (two products in one accumulator, their gated
// product or its gradients out).
enum GemmEpi : int { kEpiNone = 0, kEpiStorePreact = 1, kEpiMulGeluGrad = 2, kEpiColumnStats = 3, kEpiAddAux = 4, kEpiGated = 5,
                     kEpiGatedGrad = 6 };

// True when the driver exposes cuTensorMapEncodeTiled (needed to build TMA descriptors).
bool GemmSupported();

// out[M,N] (bf16, row-major) = act(a[M,K] * b[N,K]^T + bias[N]); a, b bf16 row-major, K % 8 == 0,
// all base pointers 16-byte aligned. bias may be null. status: device word set to 1 when a
// bounded wait inside the kernel expired (may be null).
// preact_out (optional, [M,N] bf16, needs N % 8 == 0): receives a*b^T + bias before the activation.
// col_stats (optional, 2*N floats, needs N % 8 == 0, no bias, no activation): col_stats[n] += sum_m out[m,n] and
// col_stats[N + n] += sum_m out[m,n]^2 over the rounded bf16 output (the batch statistics of a following
// normalisation layer, taken while the tile is still on chip).
cudaError_t LaunchGemmBf16NT(const void* a, const void* b, void* out, const void* bias, int M, int N, int K, int act,
                             unsigned int* status, cudaStream_t stream, void* preact_out = nullptr,
                             float* col_stats = nullptr, const void* addend = nullptr);
// addend: bf16 [M, N] added to the product (and the bias) in the epilogue, e.g. the residual stream a layer's output
// joins; needs act == 0, N % 8 == 0, no preact_out and no col_stats.

// out[M,N] = a[M,K] * b[K,N] with b row-major (consumed as an MN-major operand); K % 8 == 0, N % 8 == 0.
// gelu_preact (optional, [M,N] bf16): the result is multiplied elementwise by GELU'(gelu_preact).
// addend (optional, [M,N] bf16, not together with gelu_preact): added to the product in fp32 before rounding (the
// gradient that reaches a block's input through its shortcut, so that no separate addition pass is needed).
cudaError_t LaunchGemmBf16NN(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status,
                             cudaStream_t stream, const void* gelu_preact = nullptr, const void* addend = nullptr);

// out[M,N] = a[K,M]^T * b[K,N], a and b row-major (both consumed MN-major); M % 8 == 0, N % 8 == 0.
cudaError_t LaunchGemmBf16TN(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status,
                             cudaStream_t stream);

// The down projection of a gated feed-forward block, out[M,N] = a[M,K] * b[N,K]^T (+ addend[M,N]), on tiles chosen for its size;
// up to kSkinnyRows rows its reduction (and that of LaunchGemmBf16Gated) is shared between clusters of CTAs, and it may start before the launch in
// front of it on the stream has ended: that one may write a, nothing else that is read here.  K, N % 8 == 0.
// kSkinnyRows is the widest token tile that the kernel with shared reductions was written for, and it is the faster one up to there;
// both products, forward, in a captured graph, against the tiles for more rows: 64 rows of 1024 x 2752 23 us (41), of 776 x 2056 25
// (44), of 2048 x 5504 49 (63); 32 rows 14 (41), 12 (42), 24 (63); 8 rows 12 (39), 11 (41), 21 (63).
constexpr int kSkinnyRows = 64;
cudaError_t LaunchGemmGatedDown(const void* a, const void* b, void* out, int M, int N, int K, unsigned int* status, cudaStream_t stream,
                                const void* addend = nullptr);

// One to three independent products in one launch: out[M,N] = A * b[K,N] with A = a[M,K], or a[K,M]^T when a_transposed.  N % 8
// == 0, and K % 8 == 0 (M % 8 == 0 when a_transposed).
struct GemmGroupItem {
  const void* a;
  const void* b;
  void* out;
  int M, N, K;
  bool a_transposed;
  bool early;            // neither operand comes from the launch in front of this one on the stream, nor anything that it reads goes to out
};
cudaError_t LaunchGemmGroup(const GemmGroupItem* list, int count, unsigned int* status, cudaStream_t stream);

// h[M,F] = act(a[M,K] * w[0:F,K]^T) * (a * w[F:2F,K]^T), act kActSilu or kActGeluTanh; K % 8 == 0, F % 8 == 0.  factors
// (optional, [M,2F] 16-bit words): receives act(G) and U act'(G) in a format of their own, for the gradient.
cudaError_t LaunchGemmBf16Gated(const void* a, const void* w, void* h, void* factors, int M, int F, int K, int act,
                                unsigned int* status, cudaStream_t stream);
// Its gradient: with dH[M,F] = a[M,K] * b[K,F], dpre[M,2F] = [dH U act'(G), dH act(G)].
cudaError_t LaunchGemmBf16NNGatedGrad(const void* a, const void* b, const void* factors, void* dpre, int M, int F, int K,
                                      unsigned int* status, cudaStream_t stream);

}  // namespace bfb
