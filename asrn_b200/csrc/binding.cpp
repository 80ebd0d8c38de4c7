// PyTorch side of the fine-tuning operators (module asrn_b200._finetune): argument checks, allocation from PyTorch's
// allocator on the current stream, and the autograd nodes, around the C entry points of libasrn_b200.so. In C++ because
// these calls last 10 to 100 us, much of it the host's: a small loss takes 8.4 us (15.5 with the same code in Python), a
// small head_logprobs with its backward pass, which PyTorch runs in a thread of its own, 77 us (117), mlp8 99 us (149).
//
// Errors are raised as the Python package raises them: ValueError, TypeError, NotImplementedError, and RuntimeError for
// tensors that are not on a GPU and for CUDA errors.
#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <cstring>
#include <sstream>

#include "asrn_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] void not_implemented(const std::string& s) {
  py::gil_scoped_acquire gil;
  PyErr_SetString(PyExc_NotImplementedError, s.c_str());
  throw py::error_already_set();
}

template <class... T> std::string text(const T&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}

void check(int status, const char* what) {
  if (status == ASRN_OK) return;
  const std::string s = text(what, ": ", asrn_status_string(status));
  if (status == ASRN_ERR_UNSUPPORTED) TORCH_CHECK_NOT_IMPLEMENTED(false, s);
  TORCH_CHECK_VALUE(status != ASRN_ERR_ARG && status != ASRN_ERR_WORKSPACE, s);
  TORCH_CHECK(false, s);
}

// The tensors' device; they all have to be on the same GPU.
c10::Device device_of(const char* what, std::initializer_list<const Tensor*> ts) {
  const c10::Device dev = (*ts.begin())->device();
  for (const Tensor* t : ts)
    if (t->defined() && t->device() != dev) {
      const std::string s = text("asrn_b200.", what, " runs on CUDA tensors of one device; got ", dev, " and ", t->device());
      if (!dev.is_cuda() || !t->is_cuda()) throw std::runtime_error(s);
      throw py::value_error(s);
    }
  if (!dev.is_cuda())
    throw std::runtime_error(text("asrn_b200.", what, " runs on CUDA tensors only (there is no CPU implementation)"));
  return dev;
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(dev));
}
Tensor scratch(size_t bytes, c10::Device dev) { return empty({(int64_t)(bytes ? bytes : 256)}, at::kByte, dev); }

// Contiguous and 16-byte aligned (a view into a larger buffer may be neither); read through its address only.
Tensor rows(const Tensor& t) {
  const Tensor c = t.is_contiguous() ? t : t.detach().contiguous();
  return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.detach().clone();
}
Tensor f32(const Tensor& t) {
  return t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.detach().to(at::kFloat).contiguous();
}
Tensor mask_of(const char* what, const Tensor& m, at::IntArrayRef sizes) {
  if (m.sizes() != sizes || (m.scalar_type() != at::kBool && m.scalar_type() != at::kByte))
    throw py::value_error(text(what, ": mask has to be bool or uint8 of shape ", sizes, "; got ", m.scalar_type(), " ",
                               m.sizes()));
  return m.contiguous();
}

// The devices' status words of the kernels' bounded waits, in page-locked host memory that the devices write: a call sees
// what an earlier one recorded without waiting for the GPU. Never freed: at the program's end CUDA may be gone before this
// module. (Allocated in the relaxed capture mode: that is no part of a graph that may be under capture.)
constexpr int kDevices = 64;

volatile int* words() {
  static int* const at = [] {
    void* p = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t e = cudaHostAlloc(&p, kDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    C10_CUDA_CHECK(e);
    memset(p, 0, kDevices * sizeof(int));
    return static_cast<int*>(p);
  }();
  return at;
}

// The device's word for the call `what`, which is refused while the word holds an error.
int* status_word(const char* what, c10::Device dev) {
  TORCH_CHECK(dev.index() < kDevices, "asrn_b200.", what, ": device index ", (int)dev.index());
  volatile int* w = words() + dev.index();
  const int v = *w;
  TORCH_CHECK(v == ASRN_OK, "asrn_b200.", what, ": a bounded wait of an earlier call on ", dev, " gave up (",
              asrn_status_string(v), "): results since then are void. asrn_b200.finetune.status(reset=True) allows new calls");
  return const_cast<int*>(w);
}

int64_t status_address(int64_t device) {
  if (device < 0 || device >= kDevices) throw py::value_error(text("status: device index ", device));
  return (int64_t)(words() + device);
}

int64_t status(int64_t device, bool reset) {
  volatile int* w = reinterpret_cast<volatile int*>(status_address(device));
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  C10_CUDA_CHECK(cudaDeviceSynchronize());
  const int64_t v = *w;
  if (reset) *w = ASRN_OK;
  return v;
}

// The operands in bf16: as they are, or cast as autocast casts a linear layer's operands.
void to_bf16(const char* what, std::initializer_list<Tensor*> ts) {
  bool all = true, known = true;
  for (const Tensor* t : ts) {
    all &= t->scalar_type() == at::kBFloat16;
    known &= t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat;
  }
  if (all) return;
  if (!at::autocast::is_autocast_enabled(at::kCUDA) || at::autocast::get_autocast_dtype(at::kCUDA) != at::kBFloat16)
    not_implemented(text(what, " computes in bfloat16: pass bfloat16 tensors or call it under torch.autocast('cuda', "
                               "dtype=torch.bfloat16)"));
  if (!known) throw py::type_error(text(what, " takes float32 or bfloat16 tensors"));
  for (Tensor* t : ts) *t = t->to(at::kBFloat16);
}

// The backward passes here are no differentiable functions themselves. Where one is recorded (create_graph), what it makes
// depends on the node's inputs and on `more` through a node that raises: a second derivative is refused, not left out. Gradients
// of outputs that have none are undefined in `more`.
std::shared_ptr<torch::autograd::Node> refusal(const char* what, const variable_list& more) {
  torch::autograd::edge_list edges = torch::autograd::get_current_node()->next_edges();
  for (const Tensor& t : more)
    if (t.defined()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  return std::make_shared<torch::autograd::Error>(text("asrn_b200.", what, ": the second derivative is not implemented"),
                                                  std::move(edges));
}
void once(const char* what, variable_list& made, const variable_list& grads) {
  if (!at::GradMode::is_enabled()) return;
  const auto node = refusal(what, grads);
  for (Tensor& t : made)
    if (t.defined()) torch::autograd::set_history(t, node);
}

// ---- head ---------------------------------------------------------------------------------------------------------------

struct HeadLogprobs : torch::autograd::Function<HeadLogprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& weight, const Tensor& tokens, double tau) {
    const c10::Device dev = h.device();
    const int64_t V = weight.size(0), d = weight.size(1), N = tokens.numel();
    const Tensor hr = rows(h), w = rows(weight), tok = tokens.contiguous();
    Tensor out = empty(tokens.sizes(), at::kFloat, dev);
    const size_t nb_saved = asrn_head_saved_bytes(N, d), nb = asrn_head_workspace_bytes(N, V, d, 0);
    Tensor saved = scratch(nb_saved, dev);
    const Tensor ws = scratch(nb, dev);
    check(asrn_head_forward(N, V, d, hr.data_ptr(), w.data_ptr(), tok.data_ptr<int64_t>(), (float)tau, out.data_ptr<float>(),
                            saved.data_ptr(), nb_saved, ws.data_ptr(), nb, status_word("head_logprobs", dev), stream_of(dev)),
          "asrn_head_forward");
    ctx->save_for_backward({w, saved});
    ctx->saved_data["sizes"] = h.sizes().vec();
    ctx->saved_data["tau"] = tau;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Tensor &w = kept[0], &saved = kept[1];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const c10::Device dev = w.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t V = w.size(0), d = w.size(1), N = grads[0].numel();
    const Tensor g = f32(grads[0]);
    Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = empty(sizes, at::kBFloat16, dev);
    if (ctx->needs_input_grad(1)) dw = empty({V, d}, at::kBFloat16, dev);
    const size_t nb = asrn_head_workspace_bytes(N, V, d, 1);
    const Tensor ws = scratch(nb, dev);
    check(asrn_head_backward(N, V, d, w.data_ptr(), saved.data_ptr(), saved.numel(), (float)ctx->saved_data["tau"].toDouble(),
                             g.data_ptr<float>(), dh.defined() ? dh.data_ptr() : nullptr,
                             dw.defined() ? dw.data_ptr() : nullptr, ws.data_ptr(), nb, status_word("head_logprobs", dev),
                             stream_of(dev)),
          "asrn_head_backward");
    variable_list out{dh, dw, Tensor(), Tensor()};
    once("head_logprobs", out, grads);
    return out;
  }
};

Tensor head_logprobs(Tensor h, Tensor weight, const Tensor& tokens, double tau) {
  if (h.dim() < 1 || weight.dim() != 2 || h.size(-1) != weight.size(1) ||
      tokens.sizes() != h.sizes().slice(0, h.dim() - 1))
    throw py::value_error(text("head_logprobs: h (..., d), weight (V, d) and tokens (...) do not fit: ", h.sizes(), ", ",
                               weight.sizes(), ", ", tokens.sizes()));
  if (tokens.scalar_type() != at::kLong) throw py::type_error("head_logprobs: tokens are int64");
  if (!(tau > 0 && tau <= 1e30)) throw py::value_error("head_logprobs: temperatura has to be positive");
  const c10::Device dev = device_of("head_logprobs", {&h, &weight, &tokens});
  c10::cuda::CUDAGuard guard(dev);
  to_bf16("head_logprobs", {&h, &weight});
  if (h.size(-1) % 8 || weight.numel() == 0)
    not_implemented(text("head_logprobs: the width (", h.size(-1), ") has to be a multiple of 8, and the vocabulary not empty"));
  return HeadLogprobs::apply(h, weight, tokens, tau);
}

// ---- losses -------------------------------------------------------------------------------------------------------------

using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

void no_tangent(const char* what, const Tensor& logp) {
  if (logp._fw_grad(0).defined()) not_implemented(text(what, ": forward-mode derivatives are not implemented"));
}

Four preference_loss(const Tensor& logp, const Tensor& ref, const Tensor& mask, int64_t kind, double beta, double smoothing) {
  if (logp.dim() != 3 || logp.size(0) != 2 || ref.sizes() != logp.sizes())
    throw py::value_error(text("preference_loss: logp and ref_logp are (2, P, L); got ", logp.sizes(), " and ", ref.sizes()));
  if (!(beta > 0) || !(smoothing >= 0 && smoothing < 0.5))
    throw py::value_error("preference_loss: beta > 0 and 0 <= smoothing < 0.5");
  const c10::Device dev = device_of("preference_loss", {&logp, &ref, &mask});
  no_tangent("preference_loss", logp);
  at::AutoDispatchBelowADInplaceOrView below;            // nothing here is differentiated
  c10::cuda::CUDAGuard guard(dev);
  const Tensor m = mask_of("preference_loss", mask, logp.sizes()), lp = f32(logp), rf = f32(ref);
  const int64_t P = logp.size(1), L = logp.size(2);
  const size_t nb = asrn_preference_workspace_bytes(P, L);
  Tensor loss = empty({}, at::kFloat, dev), rewards = empty({2, P}, at::kFloat, dev);
  Tensor grad = empty(logp.sizes(), at::kFloat, dev);
  const Tensor ws = nb ? scratch(nb, dev) : Tensor();
  check(asrn_preference_loss(P, L, lp.data_ptr<float>(), rf.data_ptr<float>(), (const uint8_t*)m.data_ptr(), kind, beta,
                             smoothing, loss.data_ptr<float>(), grad.data_ptr<float>(), rewards.data_ptr<float>(),
                             nb ? ws.data_ptr() : nullptr, nb, stream_of(dev)),
        "asrn_preference_loss");
  return {loss, grad, rewards.select(0, 0), rewards.select(0, 1)};
}

Four policy_loss(const Tensor& logp, const Tensor& old, const Tensor& adv, const Tensor& mask,
                 const std::optional<Tensor>& ref_or_none, double low, double high, double kl, int64_t per) {
  const Tensor ref = ref_or_none ? *ref_or_none : Tensor();
  if (logp.dim() != 2 || old.sizes() != logp.sizes() || (ref.defined() && ref.sizes() != logp.sizes()))
    throw py::value_error(text("policy_loss: logp, old_logp and ref_logp are (B, L); got ", logp.sizes(), ", ", old.sizes(),
                               ref.defined() ? text(", ", ref.sizes()) : ""));
  const int64_t B = logp.size(0), L = logp.size(1);
  const bool each = adv.dim() == 2;
  if (each ? adv.sizes() != logp.sizes() : adv.dim() != 1 || adv.size(0) != B)
    throw py::value_error(text("policy_loss: advantages are (B, L) or (B); got ", adv.sizes()));
  if (!(low >= 0 && low < 1) || !(high >= 0) || !(kl >= 0))
    throw py::value_error("policy_loss: 0 <= clip[0] < 1, clip[1] >= 0 and kl >= 0");
  if (kl > 0 && !ref.defined()) throw py::value_error("policy_loss: a KL term needs ref_logp");
  const c10::Device dev = device_of("policy_loss", {&logp, &old, &adv, &mask, &ref});
  no_tangent("policy_loss", logp);
  at::AutoDispatchBelowADInplaceOrView below;            // nothing here is differentiated
  c10::cuda::CUDAGuard guard(dev);
  const Tensor m = mask_of("policy_loss", mask, logp.sizes()), lp = f32(logp), ol = f32(old), ad = f32(adv);
  const Tensor rf = ref.defined() ? f32(ref) : Tensor();
  const size_t nb = asrn_policy_workspace_bytes(B, L);
  Tensor out = empty({3}, at::kFloat, dev), grad = empty({B, L}, at::kFloat, dev);
  const Tensor ws = nb ? scratch(nb, dev) : Tensor();
  float* o = out.data_ptr<float>();
  check(asrn_policy_loss(B, L, lp.data_ptr<float>(), ol.data_ptr<float>(), rf.defined() ? rf.data_ptr<float>() : nullptr,
                         ad.data_ptr<float>(), each, (const uint8_t*)m.data_ptr(), low, high, kl, per, o,
                         grad.data_ptr<float>(), o + 1, nb ? ws.data_ptr() : nullptr, nb, stream_of(dev)),
        "asrn_policy_loss");
  return {out.select(0, 0), grad, out.select(0, 1), out.select(0, 2)};
}

// The loss as a function of logp whose gradient is known: the backward pass scales it.
struct KnownGradient : torch::autograd::Function<KnownGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logp, const Tensor& loss, const Tensor& grad) {
    ctx->save_for_backward({grad});
    ctx->saved_data["type"] = (int64_t)logp.scalar_type();
    return loss.clone();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor grad = ctx->get_saved_variables()[0];
    if (at::GradMode::is_enabled()) {                      // it depends on logp; the product with grads[0] is recorded
      grad = grad.detach();
      torch::autograd::set_history(grad, refusal("the losses", {}));
    }
    return {(grad * grads[0]).to((at::ScalarType)ctx->saved_data["type"].toInt()), Tensor(), Tensor()};
  }
};

Tensor known_gradient(const Tensor& logp, const Tensor& loss, const Tensor& grad) {
  return KnownGradient::apply(logp, loss, grad);
}

// ---- activations in 8 bits ------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  if (x.dim() < 1 || x.scalar_type() != at::kBFloat16) throw py::type_error("pack8 takes a bfloat16 tensor (..., f)");
  const c10::Device dev = device_of("pack8", {&x});
  c10::cuda::CUDAGuard guard(dev);
  const int64_t f = x.size(-1);
  if (f % 8 || f == 0) not_implemented(text("pack8: the last dimension (", f, ") has to be a multiple of 8"));
  const Tensor xr = rows(x.detach());
  const int64_t n = x.numel() / f;
  Tensor codes = empty({n, f}, at::kChar, dev), exps = empty({n, (f + 31) / 32}, at::kChar, dev);
  check(asrn_pack8(n, f, xr.data_ptr(), codes.data_ptr(), exps.data_ptr(), stream_of(dev)), "asrn_pack8");
  return {codes, exps};
}

Tensor unpack8(const Tensor& codes, const Tensor& exps, const std::vector<int64_t>& sizes) {
  const c10::Device dev = device_of("unpack8", {&codes, &exps});
  c10::cuda::CUDAGuard guard(dev);
  if (codes.dim() != 2 || exps.dim() != 2 || exps.size(0) != codes.size(0) ||
      exps.size(1) != (codes.size(1) + 31) / 32 || codes.scalar_type() != at::kChar || exps.scalar_type() != at::kChar)
    throw py::value_error("unpack8 takes what pack8 returned");
  Tensor x = empty(sizes, at::kBFloat16, dev);
  if (x.numel() != codes.numel()) throw py::value_error("unpack8 takes what pack8 returned");
  const Tensor c = rows(codes), e = exps.contiguous();
  check(asrn_unpack8(codes.size(0), codes.size(1), c.data_ptr(), e.data_ptr(), x.data_ptr(), stream_of(dev)),
        "asrn_unpack8");
  return x;
}

struct Mlp8 : torch::autograd::Function<Mlp8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w1, const Tensor& b1, const Tensor& w2,
                        const Tensor& b2, bool keep) {
    const c10::Device dev = x.device();
    const int64_t ff = w1.size(0), d = w1.size(1), dout = w2.size(0), N = x.numel() / d;
    const Tensor xr = rows(x), u1 = rows(w1), c1 = rows(b1), u2 = rows(w2), c2 = rows(b2);
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = dout;
    Tensor y = empty(sizes, at::kBFloat16, dev);
    const size_t nb_saved = keep ? asrn_mlp8_saved_bytes(N, d, ff) : 0, nb = asrn_mlp8_workspace_bytes(N, d, ff, dout, 0);
    Tensor saved = keep ? scratch(nb_saved, dev) : Tensor();
    const Tensor ws = scratch(nb, dev);
    check(asrn_mlp8_forward(N, d, ff, dout, xr.data_ptr(), u1.data_ptr(), c1.data_ptr(), u2.data_ptr(), c2.data_ptr(),
                            y.data_ptr(), keep ? saved.data_ptr() : nullptr, nb_saved, ws.data_ptr(), nb,
                            status_word("mlp8", dev), stream_of(dev)),
          "asrn_mlp8_forward");
    if (keep) {
      ctx->save_for_backward({u1, u2, saved});
      ctx->saved_data["sizes"] = x.sizes().vec();
    }
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Tensor &w1 = kept[0], &w2 = kept[1], &saved = kept[2];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const c10::Device dev = w1.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t ff = w1.size(0), d = w1.size(1), dout = w2.size(0), N = grads[0].numel() / dout;
    const Tensor dy = rows(grads[0]);
    const std::vector<int64_t> shapes[5] = {sizes, {ff, d}, {ff}, {dout, ff}, {dout}};
    variable_list out(6);
    void* at[5] = {};
    for (int i = 0; i < 5; ++i)
      if (ctx->needs_input_grad(i)) {
        out[i] = empty(shapes[i], at::kBFloat16, dev);
        at[i] = out[i].data_ptr();
      }
    const size_t nb = asrn_mlp8_workspace_bytes(N, d, ff, dout, 1);
    const Tensor ws = scratch(nb, dev);
    check(asrn_mlp8_backward(N, d, ff, dout, dy.data_ptr(), w1.data_ptr(), w2.data_ptr(), saved.data_ptr(), saved.numel(),
                             at[0], at[1], at[2], at[3], at[4], ws.data_ptr(), nb, status_word("mlp8", dev),
                             stream_of(dev)),
          "asrn_mlp8_backward");
    once("mlp8", out, grads);
    return out;
  }
};

Tensor mlp8(Tensor x, Tensor w1, Tensor b1, Tensor w2, Tensor b2) {
  if (x.dim() < 1 || w1.dim() != 2 || w2.dim() != 2 || w1.size(1) != x.size(-1) || b1.dim() != 1 ||
      b1.size(0) != w1.size(0) || w2.size(1) != w1.size(0) || b2.dim() != 1 || b2.size(0) != w2.size(0))
    throw py::value_error(text("mlp8: x (..., d), w1 (ff, d), b1 (ff), w2 (dout, ff), b2 (dout) do not fit: ", x.sizes(), ", ",
                               w1.sizes(), ", ", b1.sizes(), ", ", w2.sizes(), ", ", b2.sizes()));
  const c10::Device dev = device_of("mlp8", {&x, &w1, &b1, &w2, &b2});
  c10::cuda::CUDAGuard guard(dev);
  if (w1.size(0) % 8 || w1.size(1) % 8 || w2.size(0) % 8 || !w1.numel() || !w2.numel())
    not_implemented(text("mlp8: the widths (", w1.size(1), ", ", w1.size(0), ", ", w2.size(0),
                         ") have to be multiples of 8"));
  to_bf16("mlp8", {&x, &w1, &b1, &w2, &b2});
  bool keep = false;
  for (const Tensor* t : {&x, &w1, &b1, &w2, &b2}) keep |= t->requires_grad();
  return Mlp8::apply(x, w1, b1, w2, b2, keep && at::GradMode::is_enabled());
}

// Whether a call on these tensors is recorded (also where only a forward-mode derivative is: the recorded call refuses it).
bool recorded(std::initializer_list<const Tensor*> ts) {
  bool grad = false, tangent = false;
  for (const Tensor* t : ts)
    if (t->defined()) {
      grad |= t->requires_grad();
      tangent |= t->_fw_grad(0).defined();
    }
  return (grad && at::GradMode::is_enabled()) || tangent;
}
int type_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : 0; }
bool float_or_bf16(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
using MaybeTensor = std::optional<Tensor>;
Tensor or_none(const MaybeTensor& t) { return t ? *t : Tensor(); }
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
void* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- head: entropy and likeliest tokens -----------------------------------------------------------------------------------

struct StatsOut {
  Tensor logp, entropy, top_logp, top_tokens, saved, weight;
};

StatsOut stats_forward(const Tensor& h, const Tensor& weight, const Tensor& tokens, double tau, int64_t top, bool keep) {
  const c10::Device dev = h.device();
  const int64_t V = weight.size(0), d = weight.size(1), N = h.numel() / d;
  const Tensor hr = rows(h), tok = tokens.defined() ? tokens.contiguous() : tokens;
  const std::vector<int64_t> sizes(h.sizes().begin(), h.sizes().end() - 1);
  StatsOut o;
  o.weight = rows(weight);
  if (tok.defined()) o.logp = empty(sizes, at::kFloat, dev);
  o.entropy = empty(sizes, at::kFloat, dev);
  if (top) {
    std::vector<int64_t> wide = sizes;
    wide.push_back(top);
    o.top_logp = empty(wide, at::kFloat, dev);
    o.top_tokens = empty(wide, at::kLong, dev);
  }
  const bool saved = keep || tok.defined();                  // what is gathered needs the room
  const size_t nb_saved = saved ? asrn_head_stats_saved_bytes(N, d) : 0, nb = asrn_head_stats_workspace_bytes(N, V, d, top, 0);
  if (saved) o.saved = scratch(nb_saved, dev);
  const Tensor ws = scratch(nb, dev);
  check(asrn_head_stats_forward(N, V, d, hr.data_ptr(), o.weight.data_ptr(), (const int64_t*)data_or_null(tok), (float)tau, top,
                                (float*)data_or_null(o.logp), o.entropy.data_ptr<float>(), (float*)data_or_null(o.top_logp),
                                (int64_t*)data_or_null(o.top_tokens), data_or_null(o.saved), nb_saved, ws.data_ptr(), nb,
                                status_word("head_stats", dev), stream_of(dev)),
        "asrn_head_stats_forward");
  return o;
}

// Outputs: entropy, then logp where tokens were given, then the two of the likeliest tokens where they are wanted.
struct HeadStats : torch::autograd::Function<HeadStats> {
  static variable_list forward(AutogradContext* ctx, const Tensor& h, const Tensor& weight, const MaybeTensor& tokens,
                               double tau, int64_t top) {
    const StatsOut o = stats_forward(h, weight, or_none(tokens), tau, top, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({o.weight, o.saved});
    ctx->saved_data["sizes"] = h.sizes().vec();
    ctx->saved_data["tau"] = tau;
    variable_list out{o.entropy};
    if (o.logp.defined()) out.push_back(o.logp);
    if (top) {
      ctx->mark_non_differentiable({o.top_logp, o.top_tokens});
      out.push_back(o.top_logp);
      out.push_back(o.top_tokens);
    }
    ctx->saved_data["logp"] = o.logp.defined();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Tensor &w = kept[0], &saved = kept[1];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const c10::Device dev = w.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t V = w.size(0), d = w.size(1);
    int64_t N = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) N *= sizes[i];
    Tensor gh = grads[0], g;
    if (ctx->saved_data["logp"].toBool()) g = grads[1];
    if (gh.defined()) gh = f32(gh);
    if (g.defined()) g = f32(g);
    Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = empty(sizes, at::kBFloat16, dev);
    if (ctx->needs_input_grad(1)) dw = empty({V, d}, at::kBFloat16, dev);
    const size_t nb = asrn_head_stats_workspace_bytes(N, V, d, 0, 1);
    const Tensor ws = scratch(nb, dev);
    check(asrn_head_stats_backward(N, V, d, w.data_ptr(), saved.data_ptr(), saved.numel(),
                                   (float)ctx->saved_data["tau"].toDouble(), (const float*)data_or_null(g),
                                   (const float*)data_or_null(gh), data_or_null(dh), data_or_null(dw), ws.data_ptr(), nb,
                                   status_word("head_stats", dev), stream_of(dev)),
          "asrn_head_stats_backward");
    variable_list out{dh, dw, Tensor(), Tensor(), Tensor()};
    once("head_stats", out, grads);
    return out;
  }
};

std::tuple<MaybeTensor, Tensor, MaybeTensor, MaybeTensor> head_stats(Tensor h, Tensor weight, const MaybeTensor& tokens_or_none,
                                                                     double tau, int64_t top) {
  const Tensor tokens = or_none(tokens_or_none);
  if (h.dim() < 1 || weight.dim() != 2 || h.size(-1) != weight.size(1) ||
      (tokens.defined() && tokens.sizes() != h.sizes().slice(0, h.dim() - 1)))
    throw py::value_error(text("head_stats: h (..., d), weight (V, d) and tokens (...) do not fit: ", h.sizes(), ", ",
                               weight.sizes(), tokens.defined() ? text(", ", tokens.sizes()) : ""));
  if (tokens.defined() && tokens.scalar_type() != at::kLong) throw py::type_error("head_stats: tokens are int64");
  if (!(tau > 0 && tau <= 1e30)) throw py::value_error("head_stats: temperatura has to be positive");
  if (top < 0 || top > 32 || top > weight.size(0))
    throw py::value_error(text("head_stats: top is 0 to 32 and at most the vocabulary; got ", top));
  const c10::Device dev = device_of("head_stats", {&h, &weight, &tokens});
  c10::cuda::CUDAGuard guard(dev);
  to_bf16("head_stats", {&h, &weight});
  if (h.size(-1) % 8 || weight.numel() == 0)
    not_implemented(text("head_stats: the width (", h.size(-1), ") has to be a multiple of 8, and the vocabulary not empty"));
  MaybeTensor logp, top_logp, top_tokens;
  if (!recorded({&h, &weight})) {
    at::AutoDispatchBelowADInplaceOrView below;
    const StatsOut o = stats_forward(h, weight, tokens, tau, top, false);
    if (o.logp.defined()) logp = o.logp;
    if (top) {
      top_logp = o.top_logp;
      top_tokens = o.top_tokens;
    }
    return {logp, o.entropy, top_logp, top_tokens};
  }
  const variable_list out = HeadStats::apply(h, weight, tokens_or_none, tau, top);
  if (tokens.defined()) logp = out[1];
  if (top) {
    top_logp = out[out.size() - 2];
    top_tokens = out[out.size() - 1];
  }
  return {logp, out[0], top_logp, top_tokens};
}

// ---- layer norm -----------------------------------------------------------------------------------------------------------

struct NormOut {
  Tensor y, sum, read, weight, stats;          // read: x or the sum, what the backward pass reads; stats: where kept
};

NormOut norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps,
                     at::ScalarType type, bool keep) {
  const c10::Device dev = x.device();
  const int64_t d = weight.size(0), N = x.numel() / d;
  const Tensor xr = rows(x), b = bias.defined() ? rows(bias) : bias, r = residual.defined() ? rows(residual) : residual;
  NormOut o;
  o.weight = rows(weight);
  o.y = empty(x.sizes(), type, dev);
  if (r.defined()) o.sum = empty(x.sizes(), r.scalar_type(), dev);
  if (keep) o.stats = empty({N, 2}, at::kFloat, dev);
  check(asrn_layer_norm(N, d, xr.data_ptr(), type_code(xr), data_or_null(r), r.defined() ? type_code(r) : 0,
                        o.weight.data_ptr(), data_or_null(b), type_code(o.weight), (float)eps, data_or_null(o.sum),
                        o.y.data_ptr(), type_code(o.y), (float*)data_or_null(o.stats), stream_of(dev)),
        "asrn_layer_norm");
  o.read = r.defined() ? o.sum : xr;
  return o;
}

// Outputs: y, and the sum where there is a residual.
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias_or_none,
                               const MaybeTensor& residual_or_none, double eps, int64_t type) {
    const Tensor bias = or_none(bias_or_none), residual = or_none(residual_or_none);
    const NormOut o = norm_forward(x, weight, bias, residual, eps, (at::ScalarType)type, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({o.read, o.weight, o.stats});
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->saved_data["types"] = (int64_t)x.scalar_type();
    ctx->saved_data["y"] = type;
    ctx->saved_data["bias"] = bias.defined();
    if (!residual.defined()) return {o.y};
    return {o.y, o.sum};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Tensor &read = kept[0], &w = kept[1], &stats = kept[2];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const at::ScalarType x_type = (at::ScalarType)ctx->saved_data["types"].toInt();
    const c10::Device dev = read.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t d = w.size(0), N = stats.size(0);
    const bool both = grads.size() > 1, biased = ctx->saved_data["bias"].toBool();   // inputs left out are not counted
    const Tensor dy = grads[0].defined() ? rows(grads[0])
                                         : at::zeros(sizes, at::TensorOptions()
                                                                .dtype((at::ScalarType)ctx->saved_data["y"].toInt())
                                                                .device(dev));
    const Tensor ds = both && grads[1].defined() ? rows(grads[1]) : Tensor();
    const bool need_x = ctx->needs_input_grad(0), need_r = both && ctx->needs_input_grad(2 + biased),
               need_w = ctx->needs_input_grad(1), need_b = biased && ctx->needs_input_grad(2), same = read.scalar_type() == x_type;
    Tensor out, other, dw, db;                 // the gradient in the type of what was normalised, and in x's
    if (need_r || (need_x && same)) out = empty(sizes, read.scalar_type(), dev);
    if (need_x && !same) other = empty(sizes, x_type, dev);
    if (need_w) dw = empty({d}, w.scalar_type(), dev);
    if (need_b) db = empty({d}, w.scalar_type(), dev);
    const size_t nb = need_w || need_b ? asrn_layer_norm_workspace_bytes(N, d) : 0;
    const Tensor ws = nb ? scratch(nb, dev) : Tensor();
    check(asrn_layer_norm_backward(N, d, read.data_ptr(), type_code(read), stats.data_ptr<float>(), dy.data_ptr(), type_code(dy),
                                   data_or_null(ds), w.data_ptr(), type_code(w), data_or_null(out), data_or_null(other),
                                   data_or_null(dw), data_or_null(db), data_or_null(ws), nb, stream_of(dev)),
          "asrn_layer_norm_backward");
    variable_list made{need_x ? (same ? out : other) : Tensor(), dw, db, need_r ? out : Tensor(), Tensor(), Tensor()};
    once("layer_norm", made, grads);
    return made;
  }
};

std::tuple<Tensor, MaybeTensor> layer_norm(const Tensor& x, const Tensor& weight, const MaybeTensor& bias_or_none,
                                           const MaybeTensor& residual_or_none, double eps, const py::object& dtype) {
  const Tensor bias = or_none(bias_or_none), residual = or_none(residual_or_none);
  if (x.dim() < 1 || weight.dim() != 1 || x.size(-1) != weight.size(0) || (bias.defined() && bias.sizes() != weight.sizes()) ||
      (residual.defined() && residual.sizes() != x.sizes()))
    throw py::value_error(text("layer_norm: x (..., d), weight (d), bias (d) and residual (..., d) do not fit: ", x.sizes(),
                               ", ", weight.sizes(), bias.defined() ? text(", ", bias.sizes()) : "",
                               residual.defined() ? text(", ", residual.sizes()) : ""));
  if (!(eps >= 0 && eps < 1e30)) throw py::value_error("layer_norm: eps has to be 0 or more");
  for (const Tensor* t : {&x, &weight, &bias, &residual})
    if (t->defined() && !float_or_bf16(*t)) throw py::type_error("layer_norm takes float32 or bfloat16 tensors");
  if (bias.defined() && bias.scalar_type() != weight.scalar_type())
    throw py::type_error("layer_norm: weight and bias are of one type");
  at::ScalarType type = x.scalar_type();
  if (!dtype.is_none()) {
    if (!THPDtype_Check(dtype.ptr())) throw py::type_error("layer_norm: dtype is torch.float32 or torch.bfloat16");
    type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
    if (type != at::kFloat && type != at::kBFloat16) throw py::type_error("layer_norm: dtype is torch.float32 or torch.bfloat16");
  }
  const c10::Device dev = device_of("layer_norm", {&x, &weight, &bias, &residual});
  c10::cuda::CUDAGuard guard(dev);
  if (x.size(-1) == 0 || x.size(-1) > 16384)
    not_implemented(text("layer_norm: rows of 1 to 16384 values; got ", x.size(-1)));
  if (!recorded({&x, &weight, &bias, &residual})) {
    at::AutoDispatchBelowADInplaceOrView below;
    const NormOut o = norm_forward(x, weight, bias, residual, eps, type, false);
    return {o.y, maybe(o.sum)};
  }
  const variable_list out = LayerNorm::apply(x, weight, bias_or_none, residual_or_none, eps, (int64_t)type);
  return {out[0], residual.defined() ? MaybeTensor(out[1]) : MaybeTensor()};
}

// ---- product with bias, activation and residual ----------------------------------------------------------------------------

struct LinearOut {
  Tensor y, x, weight, slope;
};

LinearOut linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act,
                         bool keep) {
  const c10::Device dev = x.device();
  const int64_t n = weight.size(0), d = weight.size(1), N = x.numel() / d;
  LinearOut o;
  o.x = rows(x);
  o.weight = rows(weight);
  const Tensor b = bias.defined() ? rows(bias) : bias, r = residual.defined() ? rows(residual) : residual;
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = n;
  o.y = empty(sizes, r.defined() ? r.scalar_type() : at::kBFloat16, dev);
  if (keep && act) o.slope = empty({N, n}, at::kHalf, dev);
  check(asrn_linear_forward(N, d, n, o.x.data_ptr(), o.weight.data_ptr(), data_or_null(b), act, data_or_null(r),
                            r.defined() ? type_code(r) : 0, o.y.data_ptr(), data_or_null(o.slope), status_word("linear", dev),
                            stream_of(dev)),
        "asrn_linear_forward");
  return o;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias,
                        const MaybeTensor& residual, int64_t act) {
    const LinearOut o = linear_forward(x, weight, or_none(bias), or_none(residual), act, true);
    ctx->save_for_backward({o.x, o.weight, o.slope});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Tensor &x = kept[0], &w = kept[1], &slope = kept[2];
    const int64_t act = ctx->saved_data["act"].toInt();
    const c10::Device dev = x.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = w.size(0), d = w.size(1), N = x.numel() / d;
    const bool biased = ctx->saved_data["bias"].toBool();  // inputs left out are not counted
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = empty(x.sizes(), at::kBFloat16, dev);
    if (ctx->needs_input_grad(1)) dw = empty({n, d}, at::kBFloat16, dev);
    if (biased && ctx->needs_input_grad(2)) db = empty({n}, at::kBFloat16, dev);
    if (dx.defined() || dw.defined() || db.defined()) {
      const Tensor dy = rows(grads[0]);
      const size_t nb = asrn_linear_workspace_bytes(N, d, n, act, type_code(dy));
      const Tensor ws = scratch(nb, dev);
      check(asrn_linear_backward(N, d, n, dy.data_ptr(), type_code(dy), x.data_ptr(), w.data_ptr(), act, data_or_null(slope),
                                 data_or_null(dx), data_or_null(dw), data_or_null(db), ws.data_ptr(), nb,
                                 status_word("linear", dev), stream_of(dev)),
            "asrn_linear_backward");
    }
    variable_list out{dx, dw, db, Tensor(), Tensor()};
    once("linear", out, grads);
    // The residual's gradient is the result's.
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(2 + biased)) out[3] = grads[0];
    return out;
  }
};

Tensor linear(Tensor x, Tensor weight, const MaybeTensor& bias_or_none, int64_t act, const MaybeTensor& residual_or_none) {
  Tensor bias = or_none(bias_or_none);
  const Tensor residual = or_none(residual_or_none);
  bool fits = x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) &&
              (!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0)));
  if (fits && residual.defined())
    fits = residual.dim() == x.dim() && residual.size(-1) == weight.size(0) &&
           residual.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
  if (!fits)
    throw py::value_error(text("linear: x (..., d), weight (n, d), bias (n) and residual (..., n) do not fit: ", x.sizes(), ", ",
                               weight.sizes(), bias.defined() ? text(", ", bias.sizes()) : "",
                               residual.defined() ? text(", ", residual.sizes()) : ""));
  if (residual.defined() && !float_or_bf16(residual))
    throw py::type_error("linear: the residual is float32 or bfloat16");
  const c10::Device dev = device_of("linear", {&x, &weight, &bias, &residual});
  c10::cuda::CUDAGuard guard(dev);
  if (weight.size(0) % 8 || weight.size(1) % 8 || !weight.numel())
    not_implemented(text("linear: the widths (", weight.size(1), ", ", weight.size(0), ") have to be multiples of 8"));
  if (bias.defined())
    to_bf16("linear", {&x, &weight, &bias});
  else
    to_bf16("linear", {&x, &weight});
  if (!recorded({&x, &weight, &bias, &residual})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_forward(x, weight, bias, residual, act, false).y;
  }
  return Linear::apply(x, weight, maybe(bias), residual_or_none, act);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("head_logprobs", torch::wrap_pybind_function(&head_logprobs));
  m.def("preference_loss", torch::wrap_pybind_function(&preference_loss));
  m.def("policy_loss", torch::wrap_pybind_function(&policy_loss));
  m.def("known_gradient", torch::wrap_pybind_function(&known_gradient));
  m.def("pack8", torch::wrap_pybind_function(&pack8));
  m.def("unpack8", torch::wrap_pybind_function(&unpack8));
  m.def("mlp8", torch::wrap_pybind_function(&mlp8));
  m.def("head_stats", torch::wrap_pybind_function(&head_stats));
  m.def("layer_norm", torch::wrap_pybind_function(&layer_norm));
  m.def("linear", torch::wrap_pybind_function(&linear));
  m.def("status", torch::wrap_pybind_function(&status));
  m.def("status_address", torch::wrap_pybind_function(&status_address));
}
