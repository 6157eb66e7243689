// Transformer-block operators with their backward passes: attention, dropout with the residual stream, gated feed-forward.
#pragma once
#include <ATen/ATen.h>

#include <map>
#include <mutex>
#include <vector>

namespace bfb {

// Arguments are checked by the callers in bluefog_b200/ops; what the kernels rely on is checked again here.  All take CUDA
// tensors on one device and launch on its current stream; results of inputs that need gradients carry them.

// q [.., T, heads, D], k and v [.., T, kv_heads, D], bf16; cu: int32 boundaries or none.
at::Tensor CausalAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& cu, double scale);
// The three side by side in the columns of qkv [.., T, (heads + 2 kv_heads) D].
at::Tensor CausalSelfAttention(const at::Tensor& qkv, int64_t heads, int64_t kv_heads, const c10::optional<at::Tensor>& cu, double scale);
// How the attention kernels walk over the memory of t [.., T, heads, D], {elements from token to token, from head to head}, or of t
// [.., T, columns] when side_by_side, {elements from token to token}; nothing where they work on a copy.  On any device.
c10::optional<std::vector<int64_t>> AttentionSpacing(const at::Tensor& t, bool side_by_side);
// residual + keep * factor * x; threshold of 65536 is the dropped share, key int64 [seed, step].
at::Tensor DropoutAdd(const at::Tensor& x, const c10::optional<at::Tensor>& residual, int64_t threshold, double factor,
                      const at::Tensor& key, int64_t site);
// (act(a Wg^T) * (a Wu^T)) Wd^T + residual, a [.., K], w_gate_up = [Wg; Wu] [2F, K], w_down [N, F], bf16; act: GemmAct.
// Nothing where the kernels do not take the arguments, whatever the reason: the caller finds out.
c10::optional<at::Tensor> GatedMlp(const at::Tensor& a, const at::Tensor& w_gate_up, const at::Tensor& w_down, int64_t act,
                                   const c10::optional<at::Tensor>& residual);

// A word of status bits on every device that was asked for, zero at first.
struct StatusWords {
  std::mutex mu;
  std::map<int, at::Tensor> of_device;
};
at::Tensor& StatusTensor(StatusWords& words, int device);

// That of the attention kernels (bits: AttnStatus), and the one that the GEMM kernels share.
unsigned int* AttnStatusWord(int device);
// The bits of the attention kernels of all streams since they were last taken; waits for the device.
unsigned int TakeAttnStatus(int device);
at::Tensor& GemmStatusWord(const at::Tensor& like);

}  // namespace bfb
