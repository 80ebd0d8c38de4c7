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
// depends on the node's inputs and on `more` through a node that raises: a second derivative is refused, not left out.
std::shared_ptr<torch::autograd::Node> refusal(const char* what, const variable_list& more) {
  torch::autograd::edge_list edges = torch::autograd::get_current_node()->next_edges();
  for (const Tensor& t : more) edges.push_back(torch::autograd::impl::gradient_edge(t));
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

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("head_logprobs", torch::wrap_pybind_function(&head_logprobs));
  m.def("preference_loss", torch::wrap_pybind_function(&preference_loss));
  m.def("policy_loss", torch::wrap_pybind_function(&policy_loss));
  m.def("known_gradient", torch::wrap_pybind_function(&known_gradient));
  m.def("pack8", torch::wrap_pybind_function(&pack8));
  m.def("unpack8", torch::wrap_pybind_function(&unpack8));
  m.def("mlp8", torch::wrap_pybind_function(&mlp8));
  m.def("status", torch::wrap_pybind_function(&status));
  m.def("status_address", torch::wrap_pybind_function(&status_address));
}
