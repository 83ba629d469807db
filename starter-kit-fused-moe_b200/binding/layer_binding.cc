// Python binding of the layer operators (dense products, 8-bit activation
// checkpoints, gradients, balance loss): argument checks, outputs and workspaces
// from torch's allocator, and the calls of the C ABI (include/moe_fp8.h).
//
// A native binding because these calls are short: through ctypes a call cost
// 16-30 us of host time (six allocations, a structure, the device and stream
// lookups in Python), three to six times the device time of the gate product of
// one token. Every tensor is checked before its pointer is used; nothing is kept
// between calls.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <utility>

#include "moe_fp8.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  throw py::value_error(c10::str(parts...));
}

void status(int rc, const char* what) {
  if (rc == MOE_OK) return;
  const std::string msg = c10::str(what, ": ", moe_fp8_last_error(), " (status ", rc, ")");
  if (rc == MOE_ERR_INVALID_ARGUMENT) throw py::value_error(msg);
  throw std::runtime_error(msg);
}

const char* name_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    case at::kFloat8_e8m0fnu: return "torch.float8_e8m0fnu";
    default: return c10::toString(t);
  }
}

void check(const Tensor& t, const char* name, int64_t dims, std::initializer_list<at::ScalarType> types) {
  if (t.dim() != dims || std::find(types.begin(), types.end(), t.scalar_type()) == types.end()) {
    std::string want;
    for (auto k : types) want += (want.empty() ? "" : " or ") + std::string(name_of(k));
    refuse(name, " must be a ", dims, "-d tensor of ", want, ", got ", name_of(t.scalar_type()), " ", t.sizes());
  }
  if (!t.is_cuda()) refuse(name, " must be a CUDA tensor");
}
void check(const Tensor& t, const char* name, int64_t dims, std::initializer_list<at::ScalarType> types, at::Device dev) {
  check(t, name, dims, types);
  if (t.device() != dev) refuse(name, " must be on ", dev, ", got ", t.device());
}
void shape(const Tensor& t, const char* name, at::IntArrayRef want) {
  if (t.sizes() != want) refuse(name, " must have shape ", want, ", got ", t.sizes());
}

// A matrix whose rows the kernels can read in place (copied if they cannot), and its row stride.
bool rows_readable(const Tensor& t) {
  const int64_t m = t.size(0), n = t.size(1);
  return (t.stride(1) == 1 || n == 1) && (t.stride(0) >= n || m == 1);
}
Tensor rows(const Tensor& t, int64_t& ld) {
  if (!rows_readable(t)) {
    ld = t.size(1);
    return t.contiguous();
  }
  ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
  return t;
}

std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {a, a};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {a, a + (last + 1) * t.element_size()};
}
bool overlap(const Tensor& a, const Tensor& b) {
  const auto x = span(a), y = span(b);
  if (x.first >= y.second || y.first >= x.second) return false;
  // column slices of the same rows lie side by side
  if (a.dim() == 2 && b.dim() == 2 && a.stride(1) == 1 && b.stride(1) == 1) {
    const int64_t pitch = a.stride(0) * a.element_size();
    const int64_t wa = a.size(1) * a.element_size(), wb = b.size(1) * b.element_size();
    if (pitch > 0 && pitch == b.stride(0) * b.element_size() && wa <= pitch) {
      const int64_t d = (int64_t)(y.first - x.first) % pitch, at = d < 0 ? d + pitch : d;
      return !(at >= wa && at + wb <= pitch);
    }
  }
  return true;
}

int activation_code(const std::string& s) {
  static const char* names[] = {"none", "relu", "gelu", "silu", "swiglu"};
  for (int i = 0; i < 5; ++i)
    if (s == names[i]) return i;
  refuse("activation must be one of none, relu, gelu, silu, swiglu, got '", s, "'");
}
int scoring_code(const std::string& s) {
  if (s == "sigmoid") return 0;
  if (s == "softmax") return 1;
  refuse("scoring must be one of sigmoid, softmax, got '", s, "'");
}

Tensor make(at::IntArrayRef sizes, at::ScalarType t, at::Device dev) {
  return at::detail::empty_cuda(sizes, t, dev, std::nullopt);   // torch's caching allocator, without the dispatcher
}
// The tensors of a call that live and die together, from one allocation (an
// allocation costs 0.7 us, several of them as much as the kernels of a short call).
struct Together {
  at::Device dev;
  int64_t bytes = 0;
  c10::Storage storage;
  int64_t add(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) & ~int64_t(255);
    return at;
  }
  void allocate() { storage = make({bytes}, at::kByte, dev).storage(); }
  Tensor view(int64_t at, at::IntArrayRef sizes, at::ScalarType t) const {
    Tensor r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                        c10::scalarTypeToTypeMeta(t));
    r.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    r.unsafeGetTensorImpl()->set_storage_offset(at / c10::elementSize(t));
    return r;
  }
};

void* stream_of(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

std::pair<Tensor, Tensor> checkpoint(const Tensor& x) {
  check(x, "x", 2, {at::kBFloat16, at::kFloat});
  at::NoGradGuard no_grad;
  const auto dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t T = x.size(0), K = x.size(1);
  Together out{dev};
  const int64_t at_q = out.add(T * K), at_s = out.add(blocks_of(K) * T);
  out.allocate();
  Tensor q = out.view(at_q, {T, K}, at::kFloat8_e4m3fn), s = out.view(at_s, {blocks_of(K), T}, at::kFloat8_e8m0fnu);
  if (x.numel()) {
    int64_t ld;
    const Tensor xr = rows(x, ld);
    status(moe_checkpoint_activations(xr.data_ptr(), x.scalar_type() == at::kBFloat16, T, K, ld, q.data_ptr(),
                                      s.data_ptr(), stream_of(dev)),
           "moe_checkpoint_activations");
  }
  return {q, s};
}

Tensor restore(const Tensor& q, const Tensor& scale, at::ScalarType dtype) {
  if (q.dim() != 2 && q.dim() != 3) refuse("q must be a tensor of 2 or 3 dimensions");
  check(q, "q", q.dim(), {at::kFloat8_e4m3fn});
  const auto dev = q.device();
  check(scale, "scale", q.dim(), {at::kFloat8_e8m0fnu}, dev);
  const int64_t T = q.size(-2), K = q.size(-1), batch = q.dim() == 3 ? q.size(0) : 1;
  if (q.dim() == 3) shape(scale, "scale", {batch, blocks_of(K), T});
  else shape(scale, "scale", {blocks_of(K), T});
  if (dtype != at::kBFloat16 && dtype != at::kFloat) refuse("dtype must be bfloat16 or float32");
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = make(q.sizes(), dtype, dev);
  if (q.numel()) {
    const Tensor qc = q.contiguous(), sc = scale.contiguous();
    status(moe_restore_activations(qc.data_ptr(), sc.data_ptr(), batch, T, K, out.data_ptr(), dtype == at::kFloat,
                                   stream_of(dev)),
           "moe_restore_activations");
  }
  return out;
}

std::tuple<Tensor, OptTensor, OptTensor> linear(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                                const OptTensor& residual, const std::string& activation,
                                                at::ScalarType out_dtype, const OptTensor& output, bool keep) {
  const int act = activation_code(activation);
  check(x, "x", 2, {at::kBFloat16});
  const auto dev = x.device();
  check(weight, "weight", 2, {at::kBFloat16}, dev);
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  if (K < 1 || N < 1 || weight.size(1) != K)
    refuse("weight must be [N, ", K, "] with N and K at least 1, got ", weight.sizes());
  if (act == MOE_ACT_SWIGLU && N % 2) refuse("swiglu needs an even number of weight rows, got ", N);
  if (M > (1 << 30) || K > (1 << 23) || N > (1 << 23)) refuse("a dimension is too large: x ", x.sizes(), ", weight ", weight.sizes());
  const int64_t O = act == MOE_ACT_SWIGLU ? N / 2 : N;
  if (out_dtype != at::kBFloat16 && out_dtype != at::kFloat)
    refuse("out_dtype must be bfloat16 or float32, got ", name_of(out_dtype));
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(dev);
  MoeLinearArgs a{};
  Tensor b, r, y;
  if (bias) {
    check(*bias, "bias", 1, {at::kBFloat16}, dev);
    shape(*bias, "bias", {N});
    b = bias->contiguous();
    a.bias = b.data_ptr();
  }
  if (residual) {
    check(*residual, "residual", 2, {at::kBFloat16}, dev);
    shape(*residual, "residual", {M, O});
  }
  const Tensor xr = rows(x, a.ldx), wr = rows(weight, a.ldw);
  if (output) {
    check(*output, "output", 2, {out_dtype}, dev);
    shape(*output, "output", {M, O});
    if (overlap(*output, x)) refuse("output overlaps x");
    if (overlap(*output, weight)) refuse("output overlaps weight");
    if (bias && overlap(*output, *bias)) refuse("output overlaps bias");
    if (residual && overlap(*output, *residual) &&
        !(out_dtype == at::kBFloat16 && output->data_ptr() == residual->data_ptr() && output->strides() == residual->strides()))
      refuse("output may be the residual itself but not overlap it otherwise");
    if (rows_readable(*output)) y = *output;
  }
  if (!y.defined()) y = make({M, O}, out_dtype, dev);
  if (residual) {
    r = rows(*residual, a.ldr);
    a.residual = r.data_ptr();
  }
  a.x = xr.data_ptr();
  a.weight = wr.data_ptr();
  a.y = y.data_ptr();
  a.ldy = M > 1 ? y.stride(0) : O;
  a.m = (int32_t)M;
  a.k = (int32_t)K;
  a.n = (int32_t)N;
  a.activation = act;
  a.y_f32 = out_dtype == at::kFloat;
  OptTensor z, zs;
  if (keep && act) {
    const int64_t halves = act == MOE_ACT_SWIGLU ? 2 : 1;
    Together kept{dev};
    const int64_t at_z = kept.add(halves * M * O), at_s = kept.add(halves * blocks_of(O) * M);
    kept.allocate();
    if (halves == 2) {
      z = kept.view(at_z, {2, M, O}, at::kFloat8_e4m3fn);
      zs = kept.view(at_s, {2, blocks_of(O), M}, at::kFloat8_e8m0fnu);
    } else {
      z = kept.view(at_z, {M, O}, at::kFloat8_e4m3fn);
      zs = kept.view(at_s, {blocks_of(O), M}, at::kFloat8_e8m0fnu);
    }
    a.z8 = z->data_ptr();
    a.z_scale = zs->data_ptr();
  }
  if (M > 0) {
    Tensor ws;
    if (const size_t need = moe_linear_workspace_bytes(&a)) {
      ws = make({(int64_t)need}, at::kByte, dev);
      a.workspace = ws.data_ptr();
      a.workspace_bytes = need;
    }
    status(moe_linear_run(&a, stream_of(dev)), "moe_linear_run");
  }
  if (output && !y.is_same(*output)) {
    output->copy_(y);
    y = *output;
  }
  return {y, z, zs};
}

std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> linear_checkpointed(
    const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, const std::string& activation,
    at::ScalarType out_dtype, const OptTensor& output) {
  auto [y, z, z_scale] = linear(x, weight, bias, residual, activation, out_dtype, output, true);
  auto [q, scale] = checkpoint(x);
  return {y, q, scale, z, z_scale};
}

std::tuple<OptTensor, OptTensor, OptTensor> linear_backward(const Tensor& grad_output, const Tensor& x8,
                                                            const Tensor& x_scale, const OptTensor& z8,
                                                            const OptTensor& z_scale, const std::string& activation,
                                                            const Tensor& weight, bool need_x, bool need_weight,
                                                            bool need_bias, at::ScalarType grad_dtype) {
  const int act = activation_code(activation);
  check(weight, "weight", 2, {at::kBFloat16});
  const auto dev = weight.device();
  const int64_t N = weight.size(0), K = weight.size(1);
  if (K < 1 || N < 1 || (act == MOE_ACT_SWIGLU && N % 2))
    refuse("weight must be [N, K] with K and N at least 1 (N even for swiglu), got ", weight.sizes());
  const int64_t O = act == MOE_ACT_SWIGLU ? N / 2 : N;
  check(grad_output, "grad_output", 2, {at::kBFloat16, at::kFloat}, dev);
  const int64_t M = grad_output.size(0);
  if (M > (1 << 30) || K > (1 << 23) || N > (1 << 23)) refuse("a dimension is too large: weight ", weight.sizes());
  shape(grad_output, "grad_output", {M, O});
  if (grad_dtype != at::kBFloat16 && grad_dtype != at::kFloat)
    refuse("grad_dtype must be bfloat16 or float32, got ", name_of(grad_dtype));
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(dev);
  MoeLinearGradArgs a{};
  check(x8, "checkpoint.x", 2, {at::kFloat8_e4m3fn}, dev);
  shape(x8, "checkpoint.x", {M, K});
  check(x_scale, "checkpoint.x_scale", 2, {at::kFloat8_e8m0fnu}, dev);
  shape(x_scale, "checkpoint.x_scale", {blocks_of(K), M});
  const Tensor xc = x8.contiguous(), xsc = x_scale.contiguous();
  a.x8 = xc.data_ptr();
  a.x_scale = xsc.data_ptr();
  Tensor zc, zsc;
  if (act) {
    if (!z8 || !z_scale) refuse("checkpoint.z and checkpoint.z_scale must be tensors for activation '", activation, "'");
    const int64_t dims = act == MOE_ACT_SWIGLU ? 3 : 2;
    check(*z8, "checkpoint.z", dims, {at::kFloat8_e4m3fn}, dev);
    check(*z_scale, "checkpoint.z_scale", dims, {at::kFloat8_e8m0fnu}, dev);
    if (dims == 3) {
      shape(*z8, "checkpoint.z", {2, M, O});
      shape(*z_scale, "checkpoint.z_scale", {2, blocks_of(O), M});
    } else {
      shape(*z8, "checkpoint.z", {M, O});
      shape(*z_scale, "checkpoint.z_scale", {blocks_of(O), M});
    }
    zc = z8->contiguous();
    zsc = z_scale->contiguous();
    a.z8 = zc.data_ptr();
    a.z_scale = zsc.data_ptr();
  }
  const Tensor wr = rows(weight, a.ldw), gr = rows(grad_output, a.ldg);
  a.weight = wr.data_ptr();
  a.grad_y = gr.data_ptr();
  a.m = (int32_t)M;
  a.k = (int32_t)K;
  a.n = (int32_t)N;
  a.activation = act;
  a.grad_y_f32 = grad_output.scalar_type() == at::kFloat;
  a.grad_f32 = grad_dtype == at::kFloat;
  OptTensor gx, gw, gb;
  if (need_x) gx = make({M, K}, grad_dtype, dev);
  if (need_weight) gw = make({N, K}, grad_dtype, dev);
  if (need_bias) gb = make({N}, grad_dtype, dev);
  a.grad_x = gx && M ? gx->data_ptr() : nullptr;
  a.grad_weight = gw ? gw->data_ptr() : nullptr;
  a.grad_bias = gb ? gb->data_ptr() : nullptr;
  Tensor ws;
  if (const size_t need = moe_linear_grad_workspace_bytes(&a)) {
    ws = make({(int64_t)need}, at::kByte, dev);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  status(moe_linear_grad(&a, stream_of(dev)), "moe_linear_grad");
  return {gx, gw, gb};
}

// Checked and contiguous inputs of the balance entries.
struct Router {
  Tensor logits, idx, cu;
  int64_t T, E, k, S;
  int scoring;
};
Router router(const Tensor& logits, const Tensor& idx, const OptTensor& cu, const std::string& scoring) {
  Router r;
  check(logits, "routing_logits", 2, {at::kFloat});
  const auto dev = logits.device();
  check(idx, "topk_idx", 2, {at::kInt}, dev);
  r.T = logits.size(0);
  r.E = logits.size(1);
  r.k = idx.size(1);
  if (idx.size(0) != r.T || r.E < 1 || r.E > 1024 || r.k < 1 || r.k > 32 || r.T > (1 << 30))
    refuse("routing_logits must be [T, E] with E in [1, 1024] and topk_idx [T, k] with k in [1, 32], got ",
           logits.sizes(), " and ", idx.sizes());
  r.scoring = scoring_code(scoring);
  r.S = 1;
  if (cu) {
    check(*cu, "cu_seqlens", 1, {at::kInt}, dev);
    r.S = cu->size(0) - 1;
    if (r.S < 1 || r.S > 65535) refuse("cu_seqlens must hold 2 to 65536 boundaries, got ", r.S + 1);
    r.cu = cu->contiguous();
  }
  r.logits = logits.contiguous();
  r.idx = idx.contiguous();
  return r;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> balance_loss(const Tensor& logits, const Tensor& idx,
                                                                const OptTensor& cu, double alpha,
                                                                const std::string& scoring) {
  at::NoGradGuard no_grad;
  const Router r = router(logits, idx, cu, scoring);
  const auto dev = logits.device();
  const c10::cuda::CUDAGuard guard(dev);
  Together out{dev};
  const int64_t at_loss = out.add(4), at_counts = out.add(4 * r.S * r.E), at_tokens = out.add(4 * r.S);
  const int64_t at_mean = out.add(4 * r.S * r.E), at_live = out.add(4);
  out.allocate();
  Tensor loss = out.view(at_loss, {}, at::kFloat), counts = out.view(at_counts, {r.S, r.E}, at::kInt);
  Tensor tokens = out.view(at_tokens, {r.S}, at::kInt), mean = out.view(at_mean, {r.S, r.E}, at::kFloat);
  Tensor live = out.view(at_live, {}, at::kInt);
  const size_t need = moe_balance_workspace_bytes((int32_t)r.T, (int32_t)r.E, (int32_t)r.S);
  Tensor ws = make({(int64_t)need}, at::kByte, dev);
  MoeBalanceArgs a{};
  a.routing_logits = static_cast<const float*>(r.logits.data_ptr());
  a.topk_idx = static_cast<const int32_t*>(r.idx.data_ptr());
  a.cu_seqlens = r.cu.defined() ? static_cast<const int32_t*>(r.cu.data_ptr()) : nullptr;
  a.loss = static_cast<float*>(loss.data_ptr());
  a.counts = static_cast<int32_t*>(counts.data_ptr());
  a.tokens = static_cast<int32_t*>(tokens.data_ptr());
  a.mean_scores = static_cast<float*>(mean.data_ptr());
  a.sequences = static_cast<int32_t*>(live.data_ptr());
  a.workspace = ws.data_ptr();
  a.workspace_bytes = need;
  a.num_tokens = (int32_t)r.T;
  a.num_experts = (int32_t)r.E;
  a.top_k = (int32_t)r.k;
  a.num_sequences = (int32_t)r.S;
  a.scoring = r.scoring;
  a.alpha = (float)alpha;
  status(moe_balance_loss(&a, stream_of(dev)), "moe_balance_loss");
  return {loss, counts, tokens, mean, live};
}

Tensor balance_loss_backward(const Tensor& logits, const Tensor& idx, const OptTensor& counts, const OptTensor& tokens,
                             const OptTensor& live, const OptTensor& cu, const OptTensor& grad_loss, double alpha,
                             const std::string& scoring, const OptTensor& grad_weights, double route_scale) {
  at::NoGradGuard no_grad;
  const Router r = router(logits, idx, cu, scoring);
  const auto dev = logits.device();
  const c10::cuda::CUDAGuard guard(dev);
  MoeBalanceGradArgs a{};
  Tensor c, t, l, g, w;
  if (grad_loss) {
    if (grad_loss->numel() != 1 || grad_loss->scalar_type() != at::kFloat || grad_loss->device() != dev)
      refuse("grad_loss must be a number or one f32 value on the logits' device");
    if (!counts) refuse("grad_loss needs what balance_loss returned");
    g = grad_loss->contiguous();
    a.grad_loss = static_cast<const float*>(g.data_ptr());
  }
  if (counts) {
    if (!tokens || !live) refuse("balance must be what balance_loss returned");
    check(*counts, "balance.counts", 2, {at::kInt}, dev);
    shape(*counts, "balance.counts", {r.S, r.E});
    check(*tokens, "balance.tokens", 1, {at::kInt}, dev);
    shape(*tokens, "balance.tokens", {r.S});
    check(*live, "balance.sequences", 0, {at::kInt}, dev);
    c = counts->contiguous();
    t = tokens->contiguous();
    l = live->contiguous();
    a.counts = static_cast<const int32_t*>(c.data_ptr());
    a.tokens = static_cast<const int32_t*>(t.data_ptr());
    a.sequences = static_cast<const int32_t*>(l.data_ptr());
  }
  if (grad_weights) {
    check(*grad_weights, "grad_topk_weights", 2, {at::kFloat}, dev);
    shape(*grad_weights, "grad_topk_weights", {r.T, r.k});
    w = grad_weights->contiguous();
    a.grad_topk_weights = static_cast<const float*>(w.data_ptr());
  }
  Tensor out = make({r.T, r.E}, at::kFloat, dev);
  a.routing_logits = static_cast<const float*>(r.logits.data_ptr());
  a.topk_idx = static_cast<const int32_t*>(r.idx.data_ptr());
  a.cu_seqlens = r.cu.defined() ? static_cast<const int32_t*>(r.cu.data_ptr()) : nullptr;
  a.grad_logits = static_cast<float*>(out.data_ptr());
  a.num_tokens = (int32_t)r.T;
  a.num_experts = (int32_t)r.E;
  a.top_k = (int32_t)r.k;
  a.num_sequences = (int32_t)r.S;
  a.scoring = r.scoring;
  a.alpha = (float)alpha;
  a.routed_scaling_factor = (float)route_scale;
  if (r.T > 0) status(moe_balance_loss_grad(&a, stream_of(dev)), "moe_balance_loss_grad");
  return out;
}

}  // namespace

PYBIND11_MODULE(moe_b200_layer, m) {
  m.def("linear", &linear);
  m.def("linear_checkpointed", &linear_checkpointed);
  m.def("linear_backward", &linear_backward);
  m.def("checkpoint", &checkpoint);
  m.def("restore", &restore);
  m.def("balance_loss", &balance_loss);
  m.def("balance_loss_backward", &balance_loss_backward);
}
