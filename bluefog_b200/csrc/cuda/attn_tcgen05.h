// Causal attention over packed sequences with grouped heads, forward and backward (see attn_tcgen05.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace bfb {

// A bf16 operand [tokens, heads, D]: element (t, h, d) lies at ptr + t * token_stride + h * head_stride + d (in
// elements).  Strides are multiples of 8 and the pointer is 16-byte aligned.
struct AttnTensor {
  void* ptr = nullptr;
  long long token_stride = 0;
  long long head_stride = 0;
};

// cu == nullptr: `batch` sequences of `seq` tokens each.  Otherwise the tokens [0, seq) hold `batch` sequences one after
// the other, sequence b being [cu[b], cu[b + 1]) (int32 on the device, cu[0] is taken as 0); the tokens behind the last
// one belong to no sequence, and results and gradients are zero there.
struct AttnShape {
  const int* cu = nullptr;
  int batch = 0;
  long long seq = 0;
  int heads = 0;
  int kv_heads = 0;
  int dim = 0;           // D: a multiple of 8, at most 128
  float scale = 0.f;     // > 0
};

// Bits of the status word.
enum AttnStatus : unsigned int { kAttnTimeout = 1u, kAttnBadSequences = 2u };

// *value = *status, and *status = 0, in one step.
cudaError_t LaunchTakeStatus(unsigned int* status, unsigned int* value, cudaStream_t stream);

// 128-row tiles that the launches below cover; the row statistics hold 128 floats per head and tile.
long long AttnTiles(const AttnShape& s);
bool AttnSupported(const AttnShape& s);

// out = softmax(scale q k^T, causal within each sequence) v.  stats (optional, heads * AttnTiles * 128 floats): minus
// the base-2 logarithm of the row sums of exp, for the backward pass; -inf in rows that belong to no token.  low (optional, no
// pointer without): a byte per element of out, its next bits, for the backward pass.
cudaError_t LaunchAttnForward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                              const AttnTensor& out, const AttnTensor& low, float* stats, unsigned int* status, cudaStream_t stream);

// dq, dk, dv from dout; delta: workspace of the same size as stats and kAttnDeltaExtra floats more.
constexpr int kAttnDeltaExtra = 4;
cudaError_t LaunchAttnBackward(const AttnShape& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v,
                               const AttnTensor& out, const AttnTensor& low, const AttnTensor& dout, const float* stats, float* delta,
                               const AttnTensor& dq, const AttnTensor& dk, const AttnTensor& dv, unsigned int* status,
                               cudaStream_t stream);

}  // namespace bfb
