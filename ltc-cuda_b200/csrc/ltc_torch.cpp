// Torch binding of the sequence operators: output allocation, autograd and the calls into
// libltc_sm100.so without Python on the way.
//
// Measured: through ctypes and a Python autograd.Function a pass with a one-token step of 24 x 64 took
// 16.6 us and a training pass whose kernels take 55 us took 109 (the backward, on autograd's device
// thread, waits for the interpreter); here 8.4 and 74 us (the step by itself 5.9).  Argument checks stay
// in ltc_cuda.py, but for the step's.  The library is not linked: ltc_cuda.py passes the addresses of
// its entry points, so that LTC_SM100_LIB selects the library here too.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>

#include "../../include/ltc_sm100.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

#define LTC_ENTRY(name) decltype(&::name) name = nullptr
struct Entries {
  LTC_ENTRY(ltc_scan_plan);
  LTC_ENTRY(ltc_linear_scan_forward);
  LTC_ENTRY(ltc_linear_scan_backward);
  LTC_ENTRY(ltc_gated_scan_forward);
  LTC_ENTRY(ltc_gated_scan_backward);
  LTC_ENTRY(ltc_gated_scan_step);
  LTC_ENTRY(ltc_distill_forward);
  LTC_ENTRY(ltc_distill_backward);
  LTC_ENTRY(ltc_token_logprobs_forward);
  LTC_ENTRY(ltc_token_logprobs_backward);
  LTC_ENTRY(ltc_last_error);
} lib;
#undef LTC_ENTRY

void bind(const std::map<std::string, uintptr_t>& at) {
#define LTC_BIND(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at(#name))
  LTC_BIND(ltc_scan_plan);
  LTC_BIND(ltc_linear_scan_forward);
  LTC_BIND(ltc_linear_scan_backward);
  LTC_BIND(ltc_gated_scan_forward);
  LTC_BIND(ltc_gated_scan_backward);
  LTC_BIND(ltc_gated_scan_step);
  LTC_BIND(ltc_distill_forward);
  LTC_BIND(ltc_distill_backward);
  LTC_BIND(ltc_token_logprobs_forward);
  LTC_BIND(ltc_token_logprobs_backward);
  LTC_BIND(ltc_last_error);
#undef LTC_BIND
}

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, "ltc_cuda.", what, " failed: ", lib.ltc_last_error());
}

// ltc_cuda.set_check_waits: a Python function that raises if a bounded in-kernel wait has expired,
// called after every backward; null while the check is off
std::atomic<PyObject*> waits_check{nullptr};
void check_waits_after(const char* where) {
  if (!waits_check) return;
  const py::gil_scoped_acquire gil;
  PyObject* f = waits_check;
  if (!f) return;
  try {
    py::reinterpret_borrow<py::object>(f)(where);
  } catch (py::error_already_set& e) {
    TORCH_CHECK(false, py::str(e.value()).cast<std::string>());
  }
}

int32_t dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LTC_DTYPE_F32;
    case at::kBFloat16: return LTC_DTYPE_BF16;
    case at::kHalf: return LTC_DTYPE_F16;
    default: TORCH_CHECK(false, "ltc_cuda: unexpected type ", t.scalar_type());
  }
}
template <typename T = float>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor fresh(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor& like, size_t n) {
  return n ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)) : Tensor();
}
ltc_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// Forward-mode derivatives do not exist here, and a dropped tangent would read as a zero one.
void refuse_tangents(std::initializer_list<Tensor> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                                "ltc_cuda: the sequence operators have no forward-mode derivative");
}
// Saved tensors come back as a saved-tensor hook left them (offloaded, repacked): the values are the
// forward's, the layout need not be.  `t` as a contiguous array of the forward's type and length.
Tensor restored(const Tensor& t, at::ScalarType type, int64_t n, const at::Device& on) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.scalar_type() == type && t.numel() == n && t.device() == on,
              "ltc_cuda: a saved tensor came back as ", t.numel(), " x ", t.scalar_type(), " on ", t.device(),
              ", saved as ", n, " x ", type, " on ", on);
  const Tensor c = t.contiguous();
  TORCH_CHECK(reinterpret_cast<uintptr_t>(c.data_ptr()) % 4 == 0, "ltc_cuda: a saved tensor came back misaligned");
  return c;
}
// Gradients of a backward that is itself recorded: the first order stands, and the second raises.
// The raising node hangs on the operator's own inputs, so every path back to them meets it.
variable_list once(variable_list grads, variable_list inputs) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (const Tensor& g : grads)
    if (g.defined()) given.push_back(g);
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) given.push_back(t);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", given.size());
  given = (*error)(std::move(given));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = given[i++];
  return grads;
}

// ---- scans -------------------------------------------------------------------------
struct Scan {
  LtcScanDims dims;
  double scale;
  bool gated;
};

LtcScanInput input_of(const Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.dim() == 3 ? t.stride(1) : t.stride(0)};
}

// A saved scan input: the forward's type and shape, channels contiguous and time strides in range, as
// the forward's checks had them.
Tensor restored_rows(const Tensor& t, const LtcScanDims& d, const at::Device& on) {
  const bool packed = d.num_seqs > 0;
  TORCH_CHECK(t.defined() && t.is_cuda() && dtype_of(t) == d.dtype && t.device() == on && t.dim() == (packed ? 2 : 3) &&
                  t.size(-1) == d.H && t.size(-2) == d.T && (packed || t.size(0) == d.B),
              "ltc_cuda: a saved scan input came back with another type, shape or device");
  return (t.stride(-1) != 1 && d.H != 1) || t.stride(-2) > (1 << 28) ? t.contiguous() : t;
}

// (h, h_final, saved)
std::array<Tensor, 3> scan_forward(const Scan& s, const Tensor& decay, const Tensor& h0, const Tensor& starts,
                                   const Tensor* in, bool keep) {
  const LtcScanDims& d = s.dims;
  const Tensor& first = in[0];
  Tensor h = fresh(first), last = floats(first, {d.num_seqs ? d.num_seqs : d.B, d.H}), saved;
  if (first.numel() == 0) {
    if (h0.defined()) last.copy_(h0);
    else last.zero_();
    return {h, last, saved};
  }
  const c10::cuda::CUDAGuard guard(first.device());
  LtcScanPlan p;
  check(lib.ltc_scan_plan(&d, &p), "ltc_scan_plan");
  if (keep) saved = bytes(first, p.saved_bytes);
  const Tensor ws = bytes(first, p.fwd_workspace_bytes);
  const LtcScanInput a = input_of(in[0]), b = input_of(in[1]);
  if (s.gated) {
    const LtcScanInput c = input_of(in[2]);
    check(lib.ltc_gated_scan_forward(&d, &a, &b, &c, ptr(decay), static_cast<float>(s.scale), ptr(h0),
                                     ptr<int32_t>(starts), h.data_ptr(), ptr(last), ptr<void>(saved), ptr<void>(ws),
                                     p.fwd_workspace_bytes, stream_of(first)), "ltc_gated_scan");
  } else {
    check(lib.ltc_linear_scan_forward(&d, &a, &b, ptr(h0), ptr<int32_t>(starts), h.data_ptr(), ptr(last),
                                      ptr<void>(saved), ptr<void>(ws), p.fwd_workspace_bytes, stream_of(first)),
          "ltc_linear_scan");
  }
  return {h, last, saved};
}

struct ScanFunction : torch::autograd::Function<ScanFunction> {
  static variable_list forward(AutogradContext* ctx, const Scan& s, const OptTensor& decay_, const OptTensor& h0_,
                               const OptTensor& starts_, const Tensor& x0, const Tensor& x1, const OptTensor& x2_) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor decay = or_none(decay_), h0 = or_none(h0_), starts = or_none(starts_), x2 = or_none(x2_);
    const Tensor in[3] = {x0, x1, x2};
    auto [h, last, saved] = scan_forward(s, decay, h0, starts, in, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({decay, h0, starts, saved, x0, x1, x2});
    const LtcScanDims& d = s.dims;
    ctx->saved_data["dims"] = std::vector<int64_t>{d.B, d.T, d.H, d.dtype, d.num_seqs, s.gated};
    ctx->saved_data["scale"] = s.scale;
    return {h, last};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(7), inputs;
    {
      const at::NoGradGuard no_grad;
      const auto v = ctx->get_saved_variables();
      inputs = {v[0], v[1], v[4], v[5], v[6]};
      const auto n = ctx->saved_data["dims"].toIntVector();
      const LtcScanDims d{static_cast<int32_t>(n[0]), static_cast<int32_t>(n[1]), static_cast<int32_t>(n[2]),
                          static_cast<int32_t>(n[3]), static_cast<int32_t>(n[4])};
      const bool gated = n[5] != 0;
      Tensor in[3];
      for (int i = 0; i < (gated ? 3 : 2); ++i) in[i] = restored_rows(v[4 + i], d, v[4].device());
      const Tensor& first = in[0];
      const at::Device on = first.device();
      const Tensor decay = restored(v[0], at::kFloat, d.H, on);
      const Tensor h0 = restored(v[1], at::kFloat, static_cast<int64_t>(d.num_seqs ? d.num_seqs : d.B) * d.H, on);
      const Tensor starts = restored(v[2], at::kInt, d.num_seqs + 1, on);
      Tensor dh = g[0], dlast = g[1];
      Tensor ddecay = decay.defined() ? fresh(decay) : Tensor(), dh0 = h0.defined() ? fresh(h0) : Tensor();
      Tensor grads[3];
      for (int i = 0; i < (gated ? 3 : 2); ++i) grads[i] = fresh(in[i]);
      if (first.numel() == 0) {
        if (dh0.defined()) dlast.defined() ? dh0.copy_(dlast) : dh0.zero_();
        if (ddecay.defined()) ddecay.zero_();
      } else {
        const c10::cuda::CUDAGuard guard(first.device());
        if (dh.defined()) {
          dh = dh.to(first.scalar_type());
          if ((dh.stride(-1) != 1 && dh.size(-1) != 1) || dh.stride(-2) > (1 << 28)) dh = dh.contiguous();
        }
        if (dlast.defined()) dlast = dlast.to(at::kFloat).contiguous();
        LtcScanPlan p;
        check(lib.ltc_scan_plan(&d, &p), "ltc_scan_plan");
        const Tensor saved = restored(v[3], at::kByte, static_cast<int64_t>(p.saved_bytes), on);
        const Tensor ws = bytes(first, p.bwd_workspace_bytes);
        const LtcScanInput a = input_of(in[0]), b = input_of(in[1]);
        LtcScanInput gh{};
        if (dh.defined()) gh = input_of(dh);
        const LtcScanInput* pgh = dh.defined() ? &gh : nullptr;
        if (gated) {
          const LtcScanInput c = input_of(in[2]);
          check(lib.ltc_gated_scan_backward(&d, &a, &b, &c, ptr(decay),
                                            static_cast<float>(ctx->saved_data["scale"].toDouble()), ptr(h0),
                                            ptr<int32_t>(starts), ptr<void>(saved), pgh, ptr(dlast),
                                            grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(), ptr(ddecay),
                                            ptr(dh0), ptr<void>(ws), p.bwd_workspace_bytes, stream_of(first)),
                "ltc_gated_scan backward");
        } else {
          check(lib.ltc_linear_scan_backward(&d, &a, &b, ptr(h0), ptr<int32_t>(starts), ptr<void>(saved), pgh,
                                             ptr(dlast), grads[0].data_ptr(), grads[1].data_ptr(), ptr(dh0),
                                             ptr<void>(ws), p.bwd_workspace_bytes, stream_of(first)),
                "ltc_linear_scan backward");
        }
        check_waits_after("scan backward");
      }
      out[1] = ddecay;
      out[2] = dh0;
      for (int i = 0; i < 3; ++i) out[4 + i] = grads[i];
    }
    return once(std::move(out), std::move(inputs));
  }
};

// (h, h_final); dims = (B, T, H, S)
std::pair<Tensor, Tensor> scan(const OptTensor& decay_, const OptTensor& h0_, const OptTensor& starts_,
                               const std::array<int64_t, 4>& n, double scale, const std::vector<Tensor>& in) {
  const Tensor decay = or_none(decay_), h0 = or_none(h0_), starts = or_none(starts_);
  const OptTensor third = in.size() > 2 ? OptTensor(in[2]) : std::nullopt;
  const Tensor x2 = or_none(third);
  const Scan s{{static_cast<int32_t>(n[0]), static_cast<int32_t>(n[1]), static_cast<int32_t>(n[2]), dtype_of(in[0]),
                static_cast<int32_t>(n[3])}, scale, decay.defined()};
  refuse_tangents({in[0], in[1], x2, decay, h0});
  if (wants_grad({in[0], in[1], x2, decay, h0})) {
    auto r = ScanFunction::apply(s, decay_, h0_, starts_, in[0], in[1], third);
    return {r[0], r[1]};
  }
  const Tensor all[3] = {in[0], in[1], x2};
  auto r = scan_forward(s, decay, h0, starts, all, false);
  return {r[0], r[1]};
}

bool is_floats(const Tensor& t, const Tensor& like, at::IntArrayRef shape) {
  return t.scalar_type() == at::kFloat && t.device() == like.device() && t.sizes() == shape && t.is_contiguous();
}

// Whether a thread of the step could write into `out` (contiguous, fp32) what another has yet to read
// from `t`: they share memory and are not the same array, which a thread reads and writes in one place.
bool clashes(const Tensor& out, const Tensor& t) {
  if (out.numel() == 0) return false;
  const char *a = static_cast<const char*>(out.data_ptr()), *b = static_cast<const char*>(t.data_ptr());
  if (a == b && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == out.numel()) return false;
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return a < b + (last + 1) * t.element_size() && b < a + out.numel() * out.element_size();
}

// The one-token step: (h, new state), or None for operands that ltc_cuda.py has to look at (to
// copy them, or to name what is wrong).  In Python these checks took 4 us of a call, so they
// come first here, and only what fails them goes through Python's.
py::object gated_step(py::handle x_, py::handle rate_, py::handle gate_, py::handle decay_, py::handle state_,
                      py::handle out_, py::handle scale_) {
  for (const py::handle& o : {x_, rate_, gate_, decay_, state_})
    if (!THPVariable_Check(o.ptr())) return py::none();
  const bool given = !out_.is_none();
  if ((given && !THPVariable_Check(out_.ptr())) || !PyFloat_Check(scale_.ptr())) return py::none();
  const float scale = static_cast<float>(PyFloat_AS_DOUBLE(scale_.ptr()));
  if (!(scale > 0.f) || std::isinf(scale)) return py::none();
  const Tensor &x = THPVariable_Unpack(x_.ptr()), &rate = THPVariable_Unpack(rate_.ptr()),
               &gate = THPVariable_Unpack(gate_.ptr()), &decay = THPVariable_Unpack(decay_.ptr()),
               &state = THPVariable_Unpack(state_.ptr());
  const auto type = x.scalar_type();
  if (x.dim() != 2 || !x.is_cuda() || (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf))
    return py::none();
  const int64_t B = x.size(0), H = x.size(1);
  if (B > INT32_MAX || H > (1 << 28)) return py::none();
  for (const Tensor* t : {&x, &rate, &gate})
    if (t->scalar_type() != type || t->device() != x.device() || t->sizes() != x.sizes() ||
        (t->stride(1) != 1 && H != 1))
      return py::none();
  if (!is_floats(decay, x, {H}) || !is_floats(state, x, x.sizes())) return py::none();
  refuse_tangents({x, rate, gate, decay, state});
  if (wants_grad({x, rate, gate, decay, state})) return py::none();
  Tensor out;
  if (given) {
    out = THPVariable_Unpack(out_.ptr());
    if (!is_floats(out, x, x.sizes()) || wants_grad({out})) return py::none();
    for (const Tensor* t : {&x, &rate, &gate, &decay, &state})
      if (clashes(out, *t)) return py::none();
  }
  Tensor h;
  {
    const py::gil_scoped_release release;
    h = fresh(x);
    if (given) out.unsafeGetTensorImpl()->bump_version();  // an earlier graph that keeps it has to notice
    else out = floats(x, x.sizes());
    if (h.numel()) {
      const c10::cuda::CUDAGuard guard(x.device());
      const LtcScanDims d{static_cast<int32_t>(B), 1, static_cast<int32_t>(H), dtype_of(x), 0};
      const LtcScanInput a = input_of(x), b = input_of(rate), c = input_of(gate);
      check(lib.ltc_gated_scan_step(&d, &a, &b, &c, ptr(decay), scale, ptr(state), h.data_ptr(), ptr(out),
                                    stream_of(x)), "ltc_gated_scan_step");
    }
  }
  return py::make_tuple(h, out);
}

// ---- vocabulary --------------------------------------------------------------------
struct Rows {  // as _logits_operand describes them: rows, inner rows, strides
  std::array<int64_t, 4> n;
  double temperature;
};
LtcLogits logits_of(const Tensor& z, const Rows& r) {
  return {z.data_ptr(), r.n[0], r.n[1], r.n[2], r.n[3], static_cast<int32_t>(z.size(-1)), dtype_of(z),
          static_cast<float>(r.temperature)};
}
// rows, type, then the sizes and strides that the rows describe
void keep_rows(AutogradContext* ctx, const Tensor& z, const Rows& r) {
  std::vector<int64_t> v(r.n.begin(), r.n.end());
  v.push_back(dtype_of(z));
  v.insert(v.end(), z.sizes().begin(), z.sizes().end());
  v.insert(v.end(), z.strides().begin(), z.strides().end());
  ctx->saved_data["rows"] = std::move(v);
  ctx->saved_data["temperature"] = r.temperature;
}
// The saved logits and their rows: the recorded ones only for the layout that they were recorded for.
std::pair<Tensor, Rows> kept_rows(AutogradContext* ctx, const Tensor& z) {
  const auto v = ctx->saved_data["rows"].toIntVector();
  const size_t dims = (v.size() - 5) / 2;
  const at::IntArrayRef sizes(v.data() + 5, dims), strides(v.data() + 5 + dims, dims);
  TORCH_CHECK(z.defined() && z.is_cuda() && dtype_of(z) == v[4] && z.sizes() == sizes,
              "ltc_cuda: the saved logits came back with another type, shape or device");
  const Rows r{{v[0], v[1], v[2], v[3]}, ctx->saved_data["temperature"].toDouble()};
  if (z.strides() == strides) return {z, r};
  return {z.contiguous(), Rows{{v[0], std::max<int64_t>(v[0], 1), 0, sizes.back()}, r.temperature}};
}
// a per-row gradient; one that is the same for all rows stays a single value
std::pair<Tensor, int64_t> row_grad(const Tensor& g, int64_t rows) {
  if (!g.defined()) return {g, 0};
  Tensor f = g.to(at::kFloat);
  bool one = rows > 1;
  for (int64_t i = 0; i < f.dim(); ++i) one = one && (f.stride(i) == 0 || f.size(i) == 1);
  if (one) return {f, 0};
  return {f.contiguous(), 1};
}

// (loss, teacher probabilities, row statistics)
std::array<Tensor, 3> distill_forward(const Tensor& z, const Tensor& ids, const Tensor& teacher, const Rows& r,
                                      bool keep) {
  const int64_t rows = r.n[0], K = ids.size(-1);
  Tensor loss = floats(z, z.sizes().slice(0, z.dim() - 1)), probs, stats;
  if (keep) {
    probs = floats(z, {rows, K});
    stats = floats(z, {rows, 4});
  }
  if (rows) {
    const c10::cuda::CUDAGuard guard(z.device());
    const LtcLogits l = logits_of(z, r);
    check(lib.ltc_distill_forward(&l, ptr<int64_t>(ids), teacher.data_ptr(), dtype_of(teacher),
                                  static_cast<int32_t>(K), ptr(loss), ptr(probs), ptr(stats), stream_of(z)),
          "ltc_distill_loss");
  }
  return {loss, probs, stats};
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& ids, const Tensor& teacher,
                        const Rows& r) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, probs, stats] = distill_forward(z, ids, teacher, r, true);
    ctx->save_for_backward({z, ids, probs, stats});
    keep_rows(ctx, z, r);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(4), inputs;
    {
      const at::NoGradGuard no_grad;
      const auto v = ctx->get_saved_variables();
      inputs = {v[0]};
      const auto [z, r] = kept_rows(ctx, v[0]);
      const int64_t K = v[1].size(-1);
      const Tensor ids = restored(v[1], at::kLong, r.n[0] * K, z.device());
      const Tensor probs = restored(v[2], at::kFloat, r.n[0] * K, z.device());
      const Tensor stats = restored(v[3], at::kFloat, r.n[0] * 4, z.device());
      out[0] = fresh(z);
      if (r.n[0]) {
        const c10::cuda::CUDAGuard guard(z.device());
        const auto [gl, stride] = row_grad(g[0], r.n[0]);
        const LtcLogits l = logits_of(z, r);
        check(lib.ltc_distill_backward(&l, ptr<int64_t>(ids), static_cast<int32_t>(K), ptr(probs), ptr(stats), ptr(gl),
                                       stride, out[0].data_ptr(), stream_of(z)), "ltc_distill_loss backward");
      }
    }
    return once(std::move(out), std::move(inputs));
  }
};

Tensor distill(const Tensor& z, const Tensor& ids, const Tensor& teacher, const std::array<int64_t, 4>& rows,
               double temperature) {
  const Rows r{rows, temperature};
  refuse_tangents({z});
  if (wants_grad({z})) return DistillFunction::apply(z, ids, teacher, r);
  return distill_forward(z, ids, teacher, r, false)[0];
}

// (log probabilities, entropies, top ids, top log probabilities, row statistics)
std::array<Tensor, 5> scores_forward(const Tensor& z, const Tensor& tokens, const Rows& r, int64_t k, bool keep) {
  const auto lead = z.sizes().slice(0, z.dim() - 1);
  Tensor lp = floats(z, lead), ent = floats(z, lead), ids, best, stats;
  if (k) {
    std::vector<int64_t> shape(lead.begin(), lead.end());
    shape.push_back(k);
    ids = at::empty(shape, z.options().dtype(at::kLong));
    best = floats(z, shape);
  }
  if (keep) stats = floats(z, {r.n[0], 4});
  if (r.n[0]) {
    const c10::cuda::CUDAGuard guard(z.device());
    const LtcLogits l = logits_of(z, r);
    check(lib.ltc_token_logprobs_forward(&l, ptr<int64_t>(tokens), static_cast<int32_t>(k), ptr(lp), ptr(ent),
                                         ptr<int64_t>(ids), ptr(best), ptr(stats), stream_of(z)),
          "ltc_token_logprobs");
  }
  return {lp, ent, ids, best, stats};
}

struct ScoresFunction : torch::autograd::Function<ScoresFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& tokens, const Rows& r, int64_t k) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [lp, ent, ids, best, stats] = scores_forward(z, tokens, r, k, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({z, tokens, stats});
    keep_rows(ctx, z, r);
    if (!k) return {lp, ent};
    ctx->mark_non_differentiable({ids, best});
    return {lp, ent, ids, best};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(4), inputs;
    {
      const at::NoGradGuard no_grad;
      const auto v = ctx->get_saved_variables();
      inputs = {v[0]};
      const auto [z, r] = kept_rows(ctx, v[0]);
      const Tensor tokens = restored(v[1], at::kLong, r.n[0], z.device());
      const Tensor stats = restored(v[2], at::kFloat, r.n[0] * 4, z.device());
      out[0] = fresh(z);
      if (r.n[0]) {
        const c10::cuda::CUDAGuard guard(z.device());
        const auto [glp, slp] = row_grad(g[0], r.n[0]);
        const auto [gent, sent] = row_grad(g[1], r.n[0]);
        const LtcLogits l = logits_of(z, r);
        check(lib.ltc_token_logprobs_backward(&l, ptr<int64_t>(tokens), ptr(stats), ptr(glp), slp, ptr(gent), sent,
                                              out[0].data_ptr(), stream_of(z)), "ltc_token_logprobs backward");
      }
    }
    return once(std::move(out), std::move(inputs));
  }
};

std::tuple<Tensor, Tensor, OptTensor, OptTensor> scores(const Tensor& z, const Tensor& tokens,
                                                        const std::array<int64_t, 4>& rows, double temperature,
                                                        int64_t k) {
  const Rows r{rows, temperature};
  refuse_tangents({z});
  if (wants_grad({z})) {
    auto v = ScoresFunction::apply(z, tokens, r, k);
    if (!k) return {v[0], v[1], std::nullopt, std::nullopt};
    return {v[0], v[1], v[2], v[3]};
  }
  auto v = scores_forward(z, tokens, r, k, false);
  if (!k) return {v[0], v[1], std::nullopt, std::nullopt};
  return {v[0], v[1], v[2], v[3]};
}

}  // namespace

PYBIND11_MODULE(ltc_torch, m) {
  m.def("bind", &bind);
  m.def("set_check_waits", [](py::object f) {  // a module-level function, which outlives the module's use
    waits_check = f.is_none() ? nullptr : f.release().ptr();
  });
  // the interpreter is free while a call allocates and launches
  const auto release = py::call_guard<py::gil_scoped_release>();
  m.def("scan", &scan, release);
  m.def("gated_step", &gated_step);
  m.def("distill", &distill, release);
  m.def("scores", &scores, release);
}
