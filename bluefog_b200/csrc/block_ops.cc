// Autograd nodes of the transformer-block operators.  They are C++ nodes because a training step calls them once per layer
// and direction: with Python functions around the same launches an operator of 10 us cost 70 us of host time.
#include "block_ops.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "cuda/attn_tcgen05.h"
#include "cuda/dropout_kernels.h"
#include "cuda/gemm_tcgen05.h"

namespace bfb {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t StreamOf(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void Check(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e)); }

bool Aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// t itself where its memory is dense and 16-byte aligned, else a copy
at::Tensor Dense(const at::Tensor& t) {
  return t.is_contiguous() && Aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

at::Tensor OrUndefined(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }

bool NeedsGrad(std::initializer_list<at::Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// The kernels know nothing of tangents: an input that carries one (of any of the three operators or of their backward passes) is an
// error, or the result would pass for a constant.
template <typename... Tensors>
void NoTangents(const char* what, const Tensors&... tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  const bool any = ((tensors.defined() && tensors._fw_grad(/*level=*/0).defined()) || ...);
  TORCH_CHECK_NOT_IMPLEMENTED(!any, what, ": forward-mode differentiation is not supported");
}

// Tensors that stand for others (fake ones, which have no memory, and other subclasses that catch operators) do not reach a launch.
template <typename... Tensors>
bool AnyStandIn(const Tensors&... tensors) {
  return ((tensors.defined() && tensors.unsafeGetTensorImpl()->is_python_dispatch()) || ...);
}
template <typename... Tensors>
void NoStandIns(const char* what, const Tensors&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!AnyStandIn(tensors...), what, ": the kernels take plain tensors, not fake ones or other subclasses");
}

// Gradients of these operators are not differentiable; asking for theirs is an error, at the time they are asked for.
variable_list Once(const char* what, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (at::Tensor& g : grads)
    if (g.defined()) g.requires_grad_(true);                           // or they would pass for constants
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated only once",
                                                             static_cast<int64_t>(grads.size()));
  return (*node)(std::move(grads));
}

// ---- attention -----------------------------------------------------------------------------------------------------

// Spacing of the rows of t [.., tokens, columns...] (`inner` trailing dimensions belong to a row); 0 when they are not evenly spaced,
// as the rows of a broadcast dimension are not: they all lie in one place (the gradient of a sum over the tokens).  Extents of
// one have no spacing of their own.
int64_t RowStride(const at::Tensor& t, int64_t inner, int64_t row_size) {
  int64_t stride = -1, span = 0;                       // none met so far
  for (int64_t i = t.dim() - inner - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (t.stride(i) <= 0 || (stride >= 0 && t.stride(i) != span)) return 0;
    if (stride < 0) stride = t.stride(i);
    span = t.stride(i) * t.size(i);
  }
  return stride < 0 ? (row_size + 7) / 8 * 8 : stride;
}

// A [.., tokens, heads, D] operand, or false where the kernels cannot address it.
bool Describe(const at::Tensor& t, AttnTensor* a) {
  const int64_t n = t.dim(), heads = t.size(n - 2), d = t.size(n - 1);
  a->ptr = t.data_ptr();
  a->head_stride = heads > 1 ? t.stride(n - 2) : (d + 7) / 8 * 8;
  a->token_stride = RowStride(t, 2, heads * a->head_stride);
  return t.stride(n - 1) == 1 && Aligned(t) && a->head_stride % 8 == 0 && a->head_stride >= d && a->token_stride % 8 == 0 &&
         a->token_stride >= heads * a->head_stride;
}
at::Tensor Rows(const at::Tensor& t) {
  AttnTensor a;
  return Describe(t, &a) ? t : t.clone(at::MemoryFormat::Contiguous);
}
AttnTensor Described(const at::Tensor& t) {
  AttnTensor a;
  TORCH_CHECK(Describe(t, &a), "attention: rows have to be contiguous, 16-byte aligned and evenly spaced");
  return a;
}
bool QkvAddressable(const at::Tensor& t) {
  const int64_t cols = t.size(-1), stride = RowStride(t, 1, cols);
  return t.stride(-1) == 1 && Aligned(t) && stride % 8 == 0 && stride >= cols;
}
// qkv with rows that the kernels can address
at::Tensor QkvRows(const at::Tensor& t) { return QkvAddressable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
// the columns of `heads` heads of width d that start with head `first`
AttnTensor QkvPart(const at::Tensor& t, int64_t first, int64_t d) {
  AttnTensor a;
  a.ptr = static_cast<char*>(t.data_ptr()) + first * d * 2;
  a.head_stride = d;
  a.token_stride = RowStride(t, 1, t.size(-1));
  return a;
}

// lead: the dimensions in front of (heads, D)
AttnShape ShapeOf(at::IntArrayRef lead, int64_t heads, int64_t kv_heads, int64_t d, const at::Tensor& cu, double scale, const at::Tensor& like) {
  TORCH_CHECK(like.is_cuda() && like.scalar_type() == at::kBFloat16, "attention expects bf16 CUDA tensors");
  int64_t tokens = 1;
  for (int64_t n : lead) tokens *= n;
  AttnShape s;
  if (cu.defined()) {
    TORCH_CHECK(cu.is_cuda() && cu.get_device() == like.get_device() && cu.scalar_type() == at::kInt && cu.dim() == 1 &&
                cu.numel() >= 2 && cu.is_contiguous(), "attention: cu_seqlens has to be contiguous int32 on the device of q");
    s.cu = cu.data_ptr<int>();
    s.batch = static_cast<int>(cu.numel() - 1);
    s.seq = tokens;
  } else {
    s.seq = lead.back();
    s.batch = static_cast<int>(tokens / s.seq);
  }
  s.heads = static_cast<int>(heads);
  s.kv_heads = static_cast<int>(kv_heads);
  s.dim = static_cast<int>(d);
  s.scale = static_cast<float>(scale);
  TORCH_CHECK(AttnSupported(s), "attention: unsupported shape");
  return s;
}
AttnShape ShapeOf(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cu, double scale) {
  const int64_t n = q.dim();
  TORCH_CHECK(n >= 3 && k.dim() == n && q.numel() > 0 && k.sizes().slice(0, n - 2) == q.sizes().slice(0, n - 2) && k.size(n - 1) == q.size(n - 1),
              "attention: q and k do not match");
  return ShapeOf(q.sizes().slice(0, n - 2), q.size(n - 2), k.size(n - 2), q.size(n - 1), cu, scale, q);
}
AttnShape QkvShape(const at::Tensor& qkv, int64_t heads, int64_t kv_heads, const at::Tensor& cu, double scale) {
  TORCH_CHECK(qkv.dim() >= 2 && qkv.numel() > 0 && heads > 0 && kv_heads > 0 && qkv.size(-1) % (heads + 2 * kv_heads) == 0,
              "attention: columns do not match the heads");
  return ShapeOf(qkv.sizes().slice(0, qkv.dim() - 1), heads, kv_heads, qkv.size(-1) / (heads + 2 * kv_heads), cu, scale, qkv);
}
at::Tensor StatsFor(const AttnShape& s, const at::Tensor& like) {
  return at::empty({s.heads, AttnTiles(s), 128}, like.options().dtype(at::kFloat));
}
at::Tensor DeltaFor(const at::Tensor& stats) { return at::empty({stats.numel() + kAttnDeltaExtra}, stats.options()); }
// What the forward pass leaves for the backward pass besides the result.
struct Kept {
  at::Tensor stats, low;
  void Make(const AttnShape& s, const at::Tensor& out) {
    stats = StatsFor(s, out);
    low = at::empty(out.sizes(), out.options().dtype(at::kByte));
  }
};
float* StatsPtr(const at::Tensor& t) { return t.data_ptr<float>(); }

at::Tensor SeparateForward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, double scale, Kept* kept) {
  TORCH_CHECK(v.sizes() == k.sizes() && k.get_device() == q.get_device() && v.get_device() == q.get_device() &&
              k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "attention: q, k and v do not match");
  const AttnShape s = ShapeOf(q, k, cu, scale);
  at::Tensor out = at::empty(q.sizes(), q.options());
  if (kept != nullptr) kept->Make(s, out);
  Check(LaunchAttnForward(s, Described(q), Described(k), Described(v), Described(out), kept != nullptr ? Described(kept->low) : AttnTensor(),
                          kept != nullptr ? StatsPtr(kept->stats) : nullptr, AttnStatusWord(q.get_device()), StreamOf(q)), "attention forward launch");
  return out;
}

struct AttentionNode : public torch::autograd::Function<AttentionNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q0, const at::Tensor& k0, const at::Tensor& v0,
                            const c10::optional<at::Tensor>& boundaries, double scale) {
    const at::Tensor cu = OrUndefined(boundaries);
    const at::Tensor q = Rows(q0), k = Rows(k0), v = Rows(v0);
    Kept kept;
    at::Tensor out = SeparateForward(q, k, v, cu, scale, &kept);
    ctx->save_for_backward({q, k, v, cu, out, kept.stats, kept.low});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[4], &stats = saved[5];
    const c10::cuda::CUDAGuard guard(q.get_device());
    const AttnShape s = ShapeOf(q, k, saved[3], ctx->saved_data["scale"].toDouble());
    NoTangents("attention", grads[0]);
    const at::Tensor dout = Rows(grads[0]);
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
    at::Tensor delta = DeltaFor(stats);
    Check(LaunchAttnBackward(s, Described(q), Described(k), Described(v), Described(out), Described(saved[6]), Described(dout), StatsPtr(stats), StatsPtr(delta),
                             Described(dq), Described(dk), Described(dv), AttnStatusWord(q.get_device()), StreamOf(q)), "attention backward launch");
    variable_list g = Once("attention", {dq, dk, dv});
    return {g[0], g[1], g[2], at::Tensor(), at::Tensor()};
  }
};

at::Tensor QkvForward(const at::Tensor& qkv, int64_t h, int64_t hkv, const at::Tensor& cu, double scale, Kept* kept) {
  const AttnShape s = QkvShape(qkv, h, hkv, cu, scale);
  std::vector<int64_t> sizes(qkv.sizes().begin(), qkv.sizes().end() - 1);
  sizes.push_back(h);
  sizes.push_back(s.dim);
  at::Tensor out = at::empty(sizes, qkv.options());
  if (kept != nullptr) kept->Make(s, out);
  Check(LaunchAttnForward(s, QkvPart(qkv, 0, s.dim), QkvPart(qkv, h, s.dim), QkvPart(qkv, h + hkv, s.dim), Described(out),
                          kept != nullptr ? Described(kept->low) : AttnTensor(), kept != nullptr ? StatsPtr(kept->stats) : nullptr, AttnStatusWord(qkv.get_device()), StreamOf(qkv)),
        "attention forward launch");
  return out;
}

struct SelfAttentionNode : public torch::autograd::Function<SelfAttentionNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& qkv0, int64_t h, int64_t hkv, const c10::optional<at::Tensor>& boundaries,
                            double scale) {
    const at::Tensor cu = OrUndefined(boundaries);
    const at::Tensor qkv = QkvRows(qkv0);
    Kept kept;
    at::Tensor out = QkvForward(qkv, h, hkv, cu, scale, &kept);
    ctx->save_for_backward({qkv, cu, out, kept.stats, kept.low});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["h"] = h;
    ctx->saved_data["hkv"] = hkv;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &qkv = saved[0], &out = saved[2], &stats = saved[3];
    const c10::cuda::CUDAGuard guard(qkv.get_device());
    const int64_t h = ctx->saved_data["h"].toInt(), hkv = ctx->saved_data["hkv"].toInt();
    const AttnShape s = QkvShape(qkv, h, hkv, saved[1], ctx->saved_data["scale"].toDouble());
    NoTangents("attention", grads[0]);
    const at::Tensor dout = Rows(grads[0]);
    at::Tensor dqkv = at::empty(qkv.sizes(), qkv.options()), delta = DeltaFor(stats);
    Check(LaunchAttnBackward(s, QkvPart(qkv, 0, s.dim), QkvPart(qkv, h, s.dim), QkvPart(qkv, h + hkv, s.dim), Described(out), Described(saved[4]), Described(dout),
                             StatsPtr(stats), StatsPtr(delta), QkvPart(dqkv, 0, s.dim), QkvPart(dqkv, h, s.dim), QkvPart(dqkv, h + hkv, s.dim),
                             AttnStatusWord(qkv.get_device()), StreamOf(qkv)), "attention backward launch");
    return {Once("attention", {dqkv})[0], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---- dropout -------------------------------------------------------------------------------------------------------

at::Tensor DropoutLaunch(const at::Tensor& x, const at::Tensor& residual, int64_t threshold, double factor, const at::Tensor& key, int64_t site) {
  int type = -1;
  switch (x.scalar_type()) {
    case at::kFloat: type = kDropF32; break;
    case at::kHalf: type = kDropF16; break;
    case at::kBFloat16: type = kDropBF16; break;
    default: TORCH_CHECK(false, "dropout_add: fp32, fp16 or bf16");
  }
  TORCH_CHECK(x.is_cuda() && x.numel() > 0 && key.is_cuda() && key.get_device() == x.get_device() && key.scalar_type() == at::kLong &&
              key.numel() == 2 && threshold >= 0 && threshold <= 65536 && site >= 0 && site <= 65535, "dropout_add: bad arguments");
  if (residual.defined())
    TORCH_CHECK(residual.get_device() == x.get_device() && residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(),
                "dropout_add: residual does not match x");
  const at::Tensor a = Dense(x), r = residual.defined() ? Dense(residual) : residual, k = key.contiguous();
  at::Tensor out = at::empty(x.sizes(), x.options());
  Check(LaunchDropoutAdd(a.data_ptr(), r.defined() ? r.data_ptr() : nullptr, out.data_ptr(), a.numel(), type, static_cast<unsigned int>(threshold),
                         static_cast<float>(factor), reinterpret_cast<const long long*>(k.data_ptr<int64_t>()),
                         static_cast<unsigned int>(site), StreamOf(x)), "dropout_add launch");
  return out;
}

struct DropoutNode : public torch::autograd::Function<DropoutNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& residual, int64_t threshold,
                            double factor, const at::Tensor& key, int64_t site) {
    ctx->save_for_backward({key});
    ctx->saved_data["threshold"] = threshold;
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["site"] = site;
    ctx->saved_data["residual"] = residual.has_value();
    return DropoutLaunch(x, OrUndefined(residual), threshold, factor, key, site);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::Tensor dx;
    const at::Tensor dy = grads[0];
    if (ctx->needs_input_grad(0))                       // the operator itself without a residual: differentiable again
      dx = DropoutAdd(dy, c10::nullopt, ctx->saved_data["threshold"].toInt(), ctx->saved_data["factor"].toDouble(),
                      ctx->get_saved_variables()[0], ctx->saved_data["site"].toInt());
    // needs_input_grad counts the tensors that were given
    return {dx, ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1) ? dy : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---- gated feed-forward block --------------------------------------------------------------------------------------

unsigned int* GemmStatus(const at::Tensor& like) { return reinterpret_cast<unsigned int*>(GemmStatusWord(like).data_ptr()); }

at::Tensor GatedProduct(const at::Tensor& a, const at::Tensor& w_gate_up, int64_t act, at::Tensor* factors) {
  const int64_t m = a.size(0), f = w_gate_up.size(0) / 2;
  at::Tensor h = at::empty({m, f}, a.options());
  if (factors != nullptr) *factors = at::empty({m, 2 * f}, a.options().dtype(at::kShort));
  Check(LaunchGemmBf16Gated(a.data_ptr(), w_gate_up.data_ptr(), h.data_ptr(), factors != nullptr ? factors->data_ptr() : nullptr, static_cast<int>(m),
                            static_cast<int>(f), static_cast<int>(a.size(1)), static_cast<int>(act), GemmStatus(a), StreamOf(a)),
        "gated_mlp launch");
  return h;
}
// y has the given shape from the start: autograd would refuse to change a view made in a node's forward pass in place.
at::Tensor DownProduct(const at::Tensor& h, const at::Tensor& w_down, const at::Tensor& residual, at::IntArrayRef shape) {
  at::Tensor y = at::empty(shape, h.options());
  Check(LaunchGemmGatedDown(h.data_ptr(), w_down.data_ptr(), y.data_ptr(), static_cast<int>(h.size(0)), static_cast<int>(w_down.size(0)),
                            static_cast<int>(h.size(1)), GemmStatus(h), StreamOf(h), residual.defined() ? residual.data_ptr() : nullptr),
        "gated_mlp launch");
  return y;
}
at::Tensor Rows2d(const at::Tensor& t) { return Dense(t.reshape({-1, t.size(-1)})); }
std::vector<int64_t> WithColumns(const at::Tensor& a, int64_t columns) {
  std::vector<int64_t> s(a.sizes().begin(), a.sizes().end());
  s.back() = columns;
  return s;
}

// Kept for the backward pass: the gated product in bf16 like every activation, and the two factors of its gradient in 16 bits each.
struct GatedMlpNode : public torch::autograd::Function<GatedMlpNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a0, const at::Tensor& wgu0, const at::Tensor& wd0, int64_t act,
                            const c10::optional<at::Tensor>& residual) {
    const at::Tensor a = Rows2d(a0), wgu = Dense(wgu0), wd = Dense(wd0);
    const at::Tensor res = residual.has_value() ? Rows2d(*residual) : at::Tensor();
    at::Tensor factors;
    const at::Tensor h = GatedProduct(a, wgu, act, &factors);
    at::Tensor y = DownProduct(h, wd, res, WithColumns(a0, wd.size(0)));
    ctx->save_for_backward({a, wgu, wd, factors, h});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["sizes"] = a0.sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &a = saved[0], &wgu = saved[1], &wd = saved[2], &factors = saved[3], &h = saved[4];
    const c10::cuda::CUDAGuard guard(a.get_device());
    NoTangents("gated_mlp", grads[0]);
    const at::Tensor dy = Rows2d(grads[0]);
    const int m = static_cast<int>(a.size(0)), f = static_cast<int>(h.size(1)), k = static_cast<int>(a.size(1));
    const int n = static_cast<int>(wd.size(0));
    at::Tensor da, dwgu, dwd, dpre;
    GemmGroupItem list[3];
    int count = 0;
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1)) {
      // [dG dU] straight from the epilogue of dH = dy Wd
      dpre = at::empty(factors.sizes(), a.options());
      Check(LaunchGemmBf16NNGatedGrad(dy.data_ptr(), wd.data_ptr(), factors.data_ptr(), dpre.data_ptr(), m, f, n, GemmStatus(a), StreamOf(a)),
            "gated_mlp backward launch");
      if (ctx->needs_input_grad(0)) {
        da = at::empty(a.sizes(), a.options());
        list[count++] = {dpre.data_ptr(), wgu.data_ptr(), da.data_ptr(), m, k, 2 * f, false, false};
      }
      if (ctx->needs_input_grad(1)) {
        dwgu = at::empty(wgu.sizes(), a.options());
        list[count++] = {dpre.data_ptr(), a.data_ptr(), dwgu.data_ptr(), 2 * f, k, m, true, false};
      }
    }
    if (ctx->needs_input_grad(2)) {
      dwd = at::empty(wd.sizes(), a.options());
      list[count++] = {dy.data_ptr(), h.data_ptr(), dwd.data_ptr(), n, f, m, true, dpre.defined()};             // beside the last wave of dH
    }
    if (count > 0) Check(LaunchGemmGroup(list, count, GemmStatus(a), StreamOf(a)), "gated_mlp backward launch");
    if (da.defined()) da = da.view(ctx->saved_data["sizes"].toIntVector());
    variable_list g = Once("gated_mlp", {da, dwgu, dwd});
    return {g[0], g[1], g[2], at::Tensor(), ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(3) ? grads[0] : at::Tensor()};
  }
};

}  // namespace

c10::optional<std::vector<int64_t>> AttentionSpacing(const at::Tensor& t, bool side_by_side) {
  if (side_by_side) return QkvAddressable(t) ? c10::make_optional(std::vector<int64_t>{RowStride(t, 1, t.size(-1))}) : c10::nullopt;
  AttnTensor a;
  return Describe(t, &a) ? c10::make_optional(std::vector<int64_t>{a.token_stride, a.head_stride}) : c10::nullopt;
}

at::Tensor& StatusTensor(StatusWords& words, int device) {
  std::lock_guard<std::mutex> lock(words.mu);
  at::Tensor& w = words.of_device[device];
  if (!w.defined()) {
    // Real memory also where a mode that catches operators is active.
    const c10::impl::ExcludeDispatchKeyGuard no_modes(c10::python_ks);
    // Cleared on a stream of its own and waited for, so that no stream's first kernel is overtaken by it.  In a capture that also
    // keeps the word out of the graph's memory and its clearing out of the replays.
    c10::cuda::CUDAStreamCaptureModeGuard mode(cudaStreamCaptureModeRelaxed);
    c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, device);
    // streams of the pool are handed out in turn, so this one may be part of the capture itself
    auto captured = [&] {
      cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
      Check(cudaStreamIsCapturing(side.stream(), &status), "status word");
      return status != cudaStreamCaptureStatusNone;
    };
    for (int i = 0; i < 64 && captured(); ++i) side = c10::cuda::getStreamFromPool(false, device);
    const c10::cuda::CUDAStreamGuard on(side);
    w = at::zeros({1}, at::TensorOptions().device(at::kCUDA, device).dtype(at::kInt));
    side.synchronize();
  }
  return w;
}

unsigned int* AttnStatusWord(int device) {
  static StatusWords words;
  return reinterpret_cast<unsigned int*>(StatusTensor(words, device).data_ptr<int>());
}

unsigned int TakeAttnStatus(int device) {
  const c10::cuda::CUDAGuard guard(device);
  const c10::impl::ExcludeDispatchKeyGuard no_modes(c10::python_ks);
  unsigned int* word = AttnStatusWord(device);
  at::Tensor value = at::empty({1}, at::TensorOptions().device(at::kCUDA, device).dtype(at::kInt));
  // every stream's calls up to now; one of another thread that ends meanwhile is reported now or next time
  Check(cudaDeviceSynchronize(), "waiting for the device");
  Check(LaunchTakeStatus(word, reinterpret_cast<unsigned int*>(value.data_ptr<int>()), StreamOf(value)), "attention status");
  return static_cast<unsigned int>(value.item<int>());
}

at::Tensor CausalAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& cu, double scale) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "attention expects CUDA tensors");
  NoStandIns("attention", q, k, v, OrUndefined(cu));
  const c10::cuda::CUDAGuard guard(q.get_device());
  NoTangents("attention", q, k, v);
  if (NeedsGrad({q, k, v})) return AttentionNode::apply(q, k, v, cu, scale);
  return SeparateForward(Rows(q), Rows(k), Rows(v), OrUndefined(cu), scale, nullptr);
}

at::Tensor CausalSelfAttention(const at::Tensor& qkv, int64_t heads, int64_t kv_heads, const c10::optional<at::Tensor>& cu, double scale) {
  TORCH_CHECK(qkv.is_cuda(), "attention expects CUDA tensors");
  NoStandIns("attention", qkv, OrUndefined(cu));
  const c10::cuda::CUDAGuard guard(qkv.get_device());
  NoTangents("attention", qkv);
  if (NeedsGrad({qkv})) return SelfAttentionNode::apply(qkv, heads, kv_heads, cu, scale);
  return QkvForward(QkvRows(qkv), heads, kv_heads, OrUndefined(cu), scale, nullptr);
}

at::Tensor DropoutAdd(const at::Tensor& x, const c10::optional<at::Tensor>& residual, int64_t threshold, double factor,
                      const at::Tensor& key, int64_t site) {
  TORCH_CHECK(x.is_cuda(), "dropout_add expects a CUDA tensor");
  const at::Tensor r = OrUndefined(residual);
  NoStandIns("dropout_add", x, r, key);
  const c10::cuda::CUDAGuard guard(x.get_device());
  NoTangents("dropout_add", x, r);
  if (NeedsGrad({x, r})) return DropoutNode::apply(x, residual, threshold, factor, key, site);
  return DropoutLaunch(x, r, threshold, factor, key, site);
}

c10::optional<at::Tensor> GatedMlp(const at::Tensor& a, const at::Tensor& w_gate_up, const at::Tensor& w_down, int64_t act,
                                   const c10::optional<at::Tensor>& residual) {
  const at::Tensor r = OrUndefined(residual);
  auto usable = [&](const at::Tensor& t) { return t.is_cuda() && t.get_device() == a.get_device() && t.scalar_type() == at::kBFloat16; };
  if (!usable(a) || !usable(w_gate_up) || !usable(w_down) || (r.defined() && !usable(r)) || !GemmSupported()) return c10::nullopt;
  if (a.dim() < 1 || w_gate_up.dim() != 2 || w_down.dim() != 2 || a.numel() == 0 || w_gate_up.numel() == 0 || w_down.numel() == 0 ||
      w_gate_up.size(1) != a.size(-1) || w_gate_up.size(0) != 2 * w_down.size(1) || a.size(-1) % 8 != 0 || w_down.size(0) % 8 != 0 ||
      w_down.size(1) % 8 != 0 || a.numel() / a.size(-1) >= (1ll << 31) - 256)
    return c10::nullopt;
  if (r.defined() && r.sizes() != at::IntArrayRef(WithColumns(a, w_down.size(0)))) return c10::nullopt;
  if (AnyStandIn(a, w_gate_up, w_down, r)) return c10::nullopt;
  const c10::cuda::CUDAGuard guard(a.get_device());
  NoTangents("gated_mlp", a, w_gate_up, w_down, r);
  if (NeedsGrad({a, w_gate_up, w_down, r})) return GatedMlpNode::apply(a, w_gate_up, w_down, act, residual);
  // nothing is launched between the two products: the second one reads its other operands before the kernel in front of it ends
  const at::Tensor x = Rows2d(a), wgu = Dense(w_gate_up), wd = Dense(w_down), res = r.defined() ? Rows2d(r) : r;
  return DownProduct(GatedProduct(x, wgu, act, nullptr), wd, res, WithColumns(a, w_down.size(0)));
}

}  // namespace bfb
