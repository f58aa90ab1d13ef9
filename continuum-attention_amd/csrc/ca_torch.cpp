// Autograd functions of the Python layer in native code.
//
// For the calls that small problems make often, an autograd Function written
// in Python costs more than the kernels: about 25 us of interpreter per
// direction on a warm core and about twice that in practice, since the
// autograd engine runs the backward on a thread of its own and both threads
// sleep in between ([1,2,64,16] fp32 forward and backward: 163 us of wall time
// around 26 us of kernels).  The functions here do what their Python
// counterparts (ops._CAExactTiled, decoder._RopeContinuumAttention,
// decoder._RMSNormFn, decoder._AddRMSNormFn, weights._CAWeights) do: the same
// allocations on the current stream, the same call into libca_hip.so, the same
// saved tensors (autograd's own, so saved-tensor hooks apply), the same errors.
//
// Every entry returns None when a call is not the plain case: tensor
// subclasses, tensors under functorch transforms, dispatch or function modes,
// tracing, forward-mode duals, views that need a copy, types and sizes the
// kernels do not take.  The caller then runs the Python function, which
// handles (or reports) all of them.
#include <torch/extension.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/continuum_attention_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject* ca_error = nullptr;  // _native.CAError (set at load, kept for good)

// The errors of _native.check, from any thread.
void check(int rc) {
  if (rc == CA_OK) return;
  const std::string msg = std::string("continuum-attention_amd: ") + ca_last_error();
  if (rc == CA_ERR_INVALID || rc == CA_ERR_UNSUPPORTED) TORCH_CHECK_VALUE(false, msg);
  py::gil_scoped_acquire gil;
  const py::object error = py::reinterpret_borrow<py::object>(ca_error)(rc, msg);
  PyErr_SetObject(ca_error, error.ptr());
  python_error e;  // autograd carries it from its threads to the caller
  e.persist();
  throw std::move(e);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return CA_DTYPE_F32;
    case at::kBFloat16: return CA_DTYPE_BF16;
    case at::kHalf: return CA_DTYPE_F16;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// Plain torch.Tensor / Parameter, dense, contiguous, 16-byte aligned, on a GPU.
bool plain(PyObject* o) { return THPVariable_CheckTypeExact(Py_TYPE(o)); }
bool usable(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && t.numel() > 0 && !t.is_neg() &&
         t.is_contiguous() && aligned(t) && !t._fw_grad(/*level=*/0).defined();
}
// No transform, mode or tracer that must see the call.
bool plain_context() {
  return !c10::impl::dispatch_mode_enabled() && !at::impl::torch_function_mode_enabled() &&
         !torch::jit::tracer::isTracing() &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool grads_needed(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// A tensor as the kernels read it (a saved or incoming one may be a view, of
// negated values too).
Tensor operand(Tensor t, at::ScalarType dtype) {
  t = t.detach().resolve_neg();
  if (t.scalar_type() != dtype) t = t.to(dtype);
  t = t.contiguous();
  return aligned(t) ? t : t.clone();
}

Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype).requires_grad(false));
}
Tensor workspace(size_t bytes, const Tensor& like) {
  return empty({(int64_t)std::max<size_t>(bytes, 1)}, like, at::kByte);
}

void first_order_only(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what);
}
// Saved tensors come back from saved-tensor hooks, from wherever those put them.
void on_one_gpu(const char* what, std::initializer_list<const Tensor*> ts) {
  const c10::Device device = (*ts.begin())->device();
  for (const Tensor* t : ts)
    TORCH_CHECK(t->is_cuda() && t->device() == device, what,
                ": all tensors must be on the same GPU");
}
constexpr const char* kOpFirstOrder = "CA Volta analytic kernel supports first-order gradients only";

// ---- the operator --------------------------------------------------------------

struct OpOut {
  Tensor out, y, stats;
};

OpOut op_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& gain, bool keep_y) {
  const c10::DeviceGuard guard(q.device());
  const int B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  const int code = dtype_code(q.scalar_type()), DP = ca_padded_head_dim(D);
  OpOut r;
  if (code != CA_DTYPE_F32 || DP != D) r.out = empty(q.sizes(), q, q.scalar_type());
  if (keep_y || !r.out.defined()) r.y = empty({B, H, T, DP}, q, at::kFloat);
  r.stats = empty({(int64_t)B * H * T, 2}, q, at::kFloat);
  const size_t bytes = ca_fwd_op_workspace_bytes(code, B, H, T, D);
  Tensor ws = workspace(bytes, q);
  check(ca_fwd_op(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), code,
                  gain.const_data_ptr<float>(), r.y.defined() ? r.y.data_ptr<float>() : nullptr,
                  r.out.defined() ? r.out.data_ptr() : nullptr, r.stats.data_ptr<float>(),
                  ws.data_ptr(), bytes, B, H, T, D, stream_of(q)));
  if (!r.out.defined()) r.out = r.y;
  return r;
}

struct OpFunction : torch::autograd::Function<OpFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& gain) {
    OpOut r = op_forward(q, k, v, gain, true);
    ctx->save_for_backward({q, k, v, gain, r.y, r.stats});
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kOpFirstOrder);
    const variable_list saved = ctx->get_saved_variables();
    const at::ScalarType dt = saved[0].scalar_type();
    const Tensor q = operand(saved[0], dt), k = operand(saved[1], dt), v = operand(saved[2], dt);
    const Tensor gain = operand(saved[3], at::kFloat), y = operand(saved[4], at::kFloat),
                 stats = operand(saved[5], at::kFloat), dy = operand(grads[0], dt);
    on_one_gpu("continuum_attention", {&q, &k, &v, &gain, &y, &stats, &dy});
    const c10::DeviceGuard guard(q.device());
    const int B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
    const int code = dtype_code(dt);
    Tensor dq = empty(q.sizes(), q, dt), dk = empty(q.sizes(), q, dt), dv = empty(q.sizes(), q, dt);
    Tensor dg = empty(saved[3].sizes(), q, at::kFloat);
    const size_t bytes = ca_bwd_op_workspace_bytes(code, B, H, T, D);
    Tensor ws = workspace(bytes, q);
    check(ca_bwd_op(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), code,
                    gain.const_data_ptr<float>(), y.const_data_ptr<float>(),
                    stats.const_data_ptr<float>(), dy.const_data_ptr(), dq.data_ptr(), dk.data_ptr(),
                    dv.data_ptr(), dg.data_ptr<float>(), ws.data_ptr(), bytes, B, H, T, D,
                    stream_of(q)));
    return {dq, dk, dv, dg};
  }
};

py::object op(py::handle qo, py::handle ko, py::handle vo, py::handle go) {
  for (const py::handle& o : {qo, ko, vo, go})
    if (!plain(o.ptr())) return py::none();
  const Tensor q = THPVariable_Unpack(qo.ptr()), k = THPVariable_Unpack(ko.ptr()),
               v = THPVariable_Unpack(vo.ptr()), gain = THPVariable_Unpack(go.ptr());
  if (!plain_context() || !usable(q) || !usable(k) || !usable(v) || !usable(gain)) return py::none();
  if (q.dim() != 4 || k.sizes() != q.sizes() || v.sizes() != q.sizes() ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      dtype_code(q.scalar_type()) < 0 || gain.scalar_type() != at::kFloat || gain.dim() != 1 ||
      gain.numel() != q.size(1))
    return py::none();
  for (const Tensor* t : {&k, &v, &gain})
    if (t->device() != q.device()) return py::none();
  // head dims below 8 run query tiles (ops._fused)
  const int64_t D = q.size(3), DP = D >= 8 && D <= 128 ? ca_padded_head_dim((int)D) : 0;
  if (!DP || q.size(2) > 65536 || q.numel() / D * DP > ((int64_t)1 << 31) - 1) return py::none();
  Tensor out;
  {
    py::gil_scoped_release release;
    if (grads_needed({&q, &k, &v, &gain}))
      out = OpFunction::apply(q, k, v, gain);
    else
      out = op_forward(q.detach(), k, v, gain, false).out;
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// ---- the decoder's attention on the qkv projection output ------------------------

struct RopeFunction : torch::autograd::Function<RopeFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& gain,
                        const std::optional<Tensor>& cs, int64_t heads) {
    const c10::DeviceGuard guard(qkv.device());
    const int B = qkv.size(0), T = qkv.size(1), C = qkv.size(2) / 3, H = heads, D = C / H;
    const int code = dtype_code(qkv.scalar_type());
    Tensor y = empty({B, H, T, D}, qkv, at::kFloat), out = empty({B, T, C}, qkv, qkv.scalar_type());
    Tensor stats = empty({(int64_t)B * H * T, 2}, qkv, at::kFloat);
    const size_t bytes = ca_fwd_qkv_workspace_bytes(B, H, T, D);
    Tensor ws = workspace(bytes, qkv);
    check(ca_fwd_qkv(qkv.const_data_ptr(), code, cs ? cs->const_data_ptr<float>() : nullptr,
                     gain.const_data_ptr<float>(), y.data_ptr<float>(), out.data_ptr(),
                     stats.data_ptr<float>(), ws.data_ptr(), bytes, B, T, H, D, stream_of(qkv)));
    ctx->save_for_backward({qkv, gain, y, stats});
    ctx->saved_data["heads"] = heads;
    if (cs) ctx->saved_data["cs"] = *cs;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kOpFirstOrder);
    const variable_list saved = ctx->get_saved_variables();
    const at::ScalarType dt = saved[0].scalar_type();
    const Tensor qkv = operand(saved[0], dt), gain = operand(saved[1], at::kFloat),
                 y = operand(saved[2], at::kFloat), stats = operand(saved[3], at::kFloat),
                 dy = operand(grads[0], dt);
    on_one_gpu("continuum attention", {&qkv, &gain, &y, &stats, &dy});
    const c10::DeviceGuard guard(qkv.device());
    const int H = ctx->saved_data["heads"].toInt();
    const int B = qkv.size(0), T = qkv.size(1), D = qkv.size(2) / 3 / H;
    const auto cs = ctx->saved_data.find("cs");
    const Tensor table = cs == ctx->saved_data.end() ? Tensor() : cs->second.toTensor();
    Tensor dqkv = empty(qkv.sizes(), qkv, dt), dg = empty(saved[1].sizes(), qkv, at::kFloat);
    const size_t bytes = ca_bwd_qkv_workspace_bytes(B, H, T, D);
    Tensor ws = workspace(bytes, qkv);
    check(ca_bwd_qkv(qkv.const_data_ptr(), dtype_code(dt),
                     table.defined() ? table.const_data_ptr<float>() : nullptr,
                     gain.const_data_ptr<float>(), y.const_data_ptr<float>(),
                     stats.const_data_ptr<float>(), dy.const_data_ptr(), dqkv.data_ptr(),
                     dg.data_ptr<float>(), ws.data_ptr(), bytes, B, T, H, D, stream_of(qkv)));
    return {dqkv, dg, Tensor(), Tensor()};
  }
};

// cs: None or the fp32 RoPE table (built by the caller for this shape)
py::object rope_attention(py::handle xo, py::handle go, py::handle co, int64_t heads) {
  if (!plain(xo.ptr()) || !plain(go.ptr()) || !(co.is_none() || plain(co.ptr()))) return py::none();
  const Tensor x = THPVariable_Unpack(xo.ptr()), gain = THPVariable_Unpack(go.ptr());
  std::optional<Tensor> cs;
  if (!co.is_none()) cs = THPVariable_Unpack(co.ptr());
  if (!plain_context() || !usable(x) || !usable(gain) || (cs && !usable(*cs))) return py::none();
  if (x.dim() != 3 || heads <= 0 || x.size(2) % (3 * heads) || dtype_code(x.scalar_type()) < 0 ||
      gain.scalar_type() != at::kFloat || gain.dim() != 1 || gain.numel() != heads ||
      gain.device() != x.device())
    return py::none();
  const int64_t D = x.size(2) / (3 * heads);
  if (D > 128 || ca_padded_head_dim((int)D) != D || x.numel() / 3 > ((int64_t)1 << 31) - 1 ||
      x.size(1) > 65536)
    return py::none();
  if (cs && (cs->scalar_type() != at::kFloat || cs->numel() != x.size(1) * D || cs->requires_grad() ||
             cs->device() != x.device()))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release release;
    out = RopeFunction::apply(x, gain, cs, heads);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// ---- RMSNorm and the residual add that feeds it ------------------------------------

constexpr const char* kNormFirstOrder = "the fused RMSNorm supports first-order gradients only";

Tensor norm_operand(const Tensor& t) {
  return operand(t, dtype_code(t.scalar_type()) < 0 ? at::kFloat : t.scalar_type());
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps,
                        int64_t out_dtype) {
    const c10::DeviceGuard guard(x.device());
    const int C = x.size(-1), N = x.numel() / C;
    const auto od = static_cast<at::ScalarType>(out_dtype);
    Tensor y = empty(x.sizes(), x, od), rstd = empty({N}, x, at::kFloat);
    check(ca_rmsnorm_fwd(x.const_data_ptr<float>(), w.const_data_ptr<float>(), y.data_ptr(),
                         dtype_code(od), rstd.data_ptr<float>(), N, C, (float)eps, stream_of(x)));
    ctx->save_for_backward({x, w, rstd});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kNormFirstOrder);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor x = operand(saved[0], at::kFloat), w = operand(saved[1], at::kFloat),
                 rstd = operand(saved[2], at::kFloat), g = norm_operand(grads[0]);
    on_one_gpu("RMSNorm", {&x, &w, &rstd, &g});
    const c10::DeviceGuard guard(x.device());
    const int C = x.size(-1), N = x.numel() / C;
    Tensor dx = empty(x.sizes(), x, at::kFloat), dw = empty(w.sizes(), x, at::kFloat);
    const size_t bytes = ca_rmsnorm_bwd_workspace_bytes(N, C);
    Tensor ws = workspace(bytes, x);
    check(ca_rmsnorm_bwd(g.const_data_ptr(), dtype_code(g.scalar_type()), x.const_data_ptr<float>(),
                         w.const_data_ptr<float>(), rstd.const_data_ptr<float>(),
                         dx.data_ptr<float>(), dw.data_ptr<float>(), ws.data_ptr(), bytes, N, C,
                         stream_of(x)));
    return {dx, dw, Tensor(), Tensor()};
  }
};

struct AddNormFunction : torch::autograd::Function<AddNormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& res,
                               const Tensor& w, double eps, int64_t out_dtype) {
    const c10::DeviceGuard guard(x.device());
    const int C = x.size(-1), N = x.numel() / C;
    const auto od = static_cast<at::ScalarType>(out_dtype);
    Tensor s = empty(x.sizes(), x, at::kFloat), y = empty(x.sizes(), x, od);
    Tensor rstd = empty({N}, x, at::kFloat);
    check(ca_add_rmsnorm_fwd(x.const_data_ptr<float>(), res.const_data_ptr(),
                             dtype_code(res.scalar_type()), s.data_ptr<float>(),
                             w.const_data_ptr<float>(), y.data_ptr(), dtype_code(od),
                             rstd.data_ptr<float>(), N, C, (float)eps, stream_of(x)));
    ctx->save_for_backward({s, w, rstd});
    ctx->saved_data["res_dtype"] = static_cast<int64_t>(res.scalar_type());
    ctx->set_materialize_grads(false);  // an unused s (after the last block) reads no zeros
    return {s, y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only("the fused add + RMSNorm supports first-order gradients only");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor s = operand(saved[0], at::kFloat), w = operand(saved[1], at::kFloat),
                 rstd = operand(saved[2], at::kFloat);
    const c10::DeviceGuard guard(s.device());
    const int C = s.size(-1), N = s.numel() / C;
    const auto rd = static_cast<at::ScalarType>(ctx->saved_data["res_dtype"].toInt());
    const Tensor g = grads[1].defined() ? norm_operand(grads[1]) : at::zeros_like(s);
    Tensor gs;
    if (grads[0].defined()) gs = operand(grads[0], at::kFloat);
    on_one_gpu("add + RMSNorm", {&s, &w, &rstd, &g, gs.defined() ? &gs : &g});
    Tensor dx = empty(s.sizes(), s, at::kFloat), dres = empty(s.sizes(), s, rd);
    Tensor dw = empty(w.sizes(), s, at::kFloat);
    const size_t bytes = ca_rmsnorm_bwd_workspace_bytes(N, C);
    Tensor ws = workspace(bytes, s);
    check(ca_add_rmsnorm_bwd(g.const_data_ptr(), dtype_code(g.scalar_type()),
                             gs.defined() ? gs.const_data_ptr<float>() : nullptr,
                             s.const_data_ptr<float>(), w.const_data_ptr<float>(),
                             rstd.const_data_ptr<float>(), dx.data_ptr<float>(), dres.data_ptr(),
                             dtype_code(rd), dw.data_ptr<float>(), ws.data_ptr(), bytes, N, C,
                             stream_of(s)));
    return {dx, dres, dw, Tensor(), Tensor()};
  }
};

bool norm_args(const Tensor& x, const Tensor& w, at::ScalarType od) {
  return usable(x) && usable(w) && x.dim() >= 1 && x.scalar_type() == at::kFloat &&
         w.scalar_type() == at::kFloat && w.dim() == 1 && w.numel() == x.size(-1) &&
         x.size(-1) <= 4096 && x.numel() <= ((int64_t)1 << 31) - 1 && w.device() == x.device() &&
         dtype_code(od) >= 0;
}

py::object rmsnorm(py::handle xo, py::handle wo, double eps, at::ScalarType od) {
  if (!plain(xo.ptr()) || !plain(wo.ptr())) return py::none();
  const Tensor x = THPVariable_Unpack(xo.ptr()), w = THPVariable_Unpack(wo.ptr());
  if (!plain_context() || !norm_args(x, w, od)) return py::none();
  Tensor y;
  {
    py::gil_scoped_release release;
    y = NormFunction::apply(x, w, eps, static_cast<int64_t>(od));
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(y));
}

py::object add_rmsnorm(py::handle xo, py::handle ro, py::handle wo, double eps, at::ScalarType od) {
  if (!plain(xo.ptr()) || !plain(ro.ptr()) || !plain(wo.ptr())) return py::none();
  const Tensor x = THPVariable_Unpack(xo.ptr()), res = THPVariable_Unpack(ro.ptr()),
               w = THPVariable_Unpack(wo.ptr());
  if (!plain_context() || !norm_args(x, w, od) || !usable(res) || res.sizes() != x.sizes() ||
      res.device() != x.device() || dtype_code(res.scalar_type()) < 0)
    return py::none();
  variable_list r;
  {
    py::gil_scoped_release release;
    r = AddNormFunction::apply(x, res, w, eps, static_cast<int64_t>(od));
  }
  return py::make_tuple(py::reinterpret_steal<py::object>(THPVariable_Wrap(r[0])),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(r[1])));
}

// ---- materialised weights ----------------------------------------------------------

struct WeightsFunction : torch::autograd::Function<WeightsFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits) {
    const c10::DeviceGuard guard(logits.device());
    const int T = logits.size(-1), N = logits.numel() / ((int64_t)T * T);
    Tensor w = empty(logits.sizes(), logits, at::kFloat);
    Tensor stats = empty({(int64_t)N * T, 2}, logits, at::kFloat);
    check(ca_weights_f32(logits.const_data_ptr<float>(), w.data_ptr<float>(),
                         stats.data_ptr<float>(), N, T, T, 0, stream_of(logits)));
    ctx->save_for_backward({logits});
    return w;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only("continuous_attention_weights on the GPU supports first-order gradients only");
    const Tensor s = operand(ctx->get_saved_variables()[0], at::kFloat),
                 g = operand(grads[0], at::kFloat);
    on_one_gpu("continuous_attention_weights", {&s, &g});
    TORCH_CHECK_VALUE(g.sizes() == s.sizes(), "grad_weights shape ", g.sizes(), " != scores shape ", s.sizes());
    const c10::DeviceGuard guard(s.device());
    const int T = s.size(-1), N = s.numel() / ((int64_t)T * T);
    Tensor ds = empty(s.sizes(), s, at::kFloat);
    check(ca_weights_bwd_f32(s.const_data_ptr<float>(), g.const_data_ptr<float>(), nullptr,
                             ds.data_ptr<float>(), N, T, T, 0, stream_of(s)));
    return {ds};
  }
};

py::object weights(py::handle so) {
  if (!plain(so.ptr())) return py::none();
  const Tensor s = THPVariable_Unpack(so.ptr());
  if (!plain_context() || !usable(s) || s.dim() < 2 || s.scalar_type() != at::kFloat ||
      s.size(-1) != s.size(-2) || s.size(-1) > (1 << 30) || s.numel() / s.size(-1) > ((int64_t)1 << 31) - 1)
    return py::none();
  Tensor w;
  {
    py::gil_scoped_release release;
    w = WeightsFunction::apply(s);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(w));
}

// ---- generation ----------------------------------------------------------------------
//
// The Python entry points of rotary.py, paged.py and int4.py call these first.
// A call these refuse (None) is checked, and carried out or reported, there.

// On a GPU, strided, not negated, no forward-mode dual.
bool readable(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t._fw_grad(/*level=*/0).defined();
}
// 32-bit integers [..] on `device`, contiguous.
bool counts(const Tensor& t, c10::Device device) {
  return t.scalar_type() == at::kInt && t.device() == device && t.is_contiguous();
}
// Rows of a token tensor: [tokens, heads, D] of any strides with contiguous
// rows, or more leading dims, contiguous.
struct HeadRows {
  int64_t tokens, heads, D, ts, hs;
  bool ok;
};
HeadRows head_rows(const Tensor& t) {
  HeadRows r{0, 0, 0, 0, 0, false};
  if (t.dim() < 3) return r;
  r.D = t.size(-1);
  r.heads = t.size(-2);
  if (r.D <= 0 || r.heads <= 0 || t.numel() == 0) return r;
  r.tokens = t.numel() / (r.D * r.heads);
  if (r.tokens > (1 << 30) || r.heads > (1 << 20)) return r;
  if (t.dim() == 3) {
    r.ok = t.stride(2) == 1;
    r.ts = t.stride(0);
    r.hs = t.stride(1);
  } else {
    r.ok = t.is_contiguous();
    r.hs = r.D;
    r.ts = r.heads * r.D;
  }
  return r;
}

// No two elements in one place (as far as nested strides show it).
bool disjoint(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;
  for (const auto& d : dims) {
    if (d.first < span) return false;
    span = d.first * (d.second - 1) + span;
  }
  return true;
}

struct RotaryPlan {
  double magnitude;
  int64_t half, rotary_dim, inverse;
};
// q (and k, if defined) turned; the arguments have been checked
variable_list turn(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& turns,
                   const RotaryPlan& p) {
  const c10::DeviceGuard guard(q.device());
  ca_rotary r{};
  auto rows = [](const Tensor& x, Tensor& held, int64_t& ts, int64_t& hs) {
    held = x.detach().resolve_neg();
    HeadRows h = head_rows(held);
    if (!h.ok) {
      held = held.contiguous();
      h = head_rows(held);
    }
    ts = h.ts;
    hs = h.hs;
    return h;
  };
  Tensor qh, kh;
  int64_t ts, hs;
  const HeadRows a = rows(q, qh, ts, hs);
  Tensor qo = empty(q.sizes(), q, q.scalar_type()), ko;
  r.q = qh.const_data_ptr();
  r.q_out = qo.data_ptr();
  r.q_token_stride = ts;
  r.q_head_stride = hs;
  r.q_out_token_stride = a.heads * a.D;
  r.q_out_head_stride = a.D;
  if (k.defined()) {
    const HeadRows b = rows(k, kh, ts, hs);
    ko = empty(k.sizes(), k, k.scalar_type());
    r.k = kh.const_data_ptr();
    r.k_out = ko.data_ptr();
    r.k_token_stride = ts;
    r.k_head_stride = hs;
    r.k_out_token_stride = b.heads * b.D;
    r.k_out_head_stride = b.D;
    r.k_heads = (int)b.heads;
  }
  r.positions = positions.const_data_ptr();
  r.positions64 = positions.scalar_type() == at::kLong;
  r.turns = turns.const_data_ptr<double>();
  r.magnitude = (float)p.magnitude;
  r.half = (int)p.half;
  r.inverse = (int)p.inverse;
  r.dtype = dtype_code(q.scalar_type());
  r.tokens = (int)a.tokens;
  r.q_heads = (int)a.heads;
  r.head_dim = (int)a.D;
  r.rotary_dim = (int)p.rotary_dim;
  check(ca_rotary_embedding(&r, stream_of(q)));
  return {qo, ko};
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k_or_none,
                               const Tensor& positions, const Tensor& turns, double magnitude, int64_t half, int64_t rotary_dim,
                               int64_t inverse) {
    ctx->save_for_backward({positions, turns});
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["plan"] = std::vector<int64_t>{half, rotary_dim, inverse};
    ctx->set_materialize_grads(false);
    const Tensor k = k_or_none ? *k_or_none : Tensor();
    variable_list y = turn(q, k, positions, turns, RotaryPlan{magnitude, half, rotary_dim, inverse});
    if (!k.defined()) y.pop_back();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> p = ctx->saved_data["plan"].toIntVector();
    const double magnitude = ctx->saved_data["magnitude"].toDouble();
    variable_list out(8);
    std::vector<int> which;
    for (int i = 0; i < (int)grads.size(); ++i)
      if (grads[i].defined()) which.push_back(i);
    if (which.empty()) return out;
    const Tensor a = grads[which[0]];
    std::optional<Tensor> b;
    if (which.size() > 1) b = grads[which[1]];
    on_one_gpu("rotary_embedding", {&a, &saved[0], &saved[1]});
    // the transpose is the rotation back; under create_graph it is recorded like it
    const variable_list y = apply(a, b, saved[0], saved[1], magnitude, p[0], p[1], 1 - p[2]);
    for (int i = 0; i < (int)which.size(); ++i) out[which[i]] = y[i];
    return out;
  }
};

py::object rotary(py::handle qo, py::handle ko, py::handle po, py::handle to, double magnitude, bool half,
                  int64_t rotary_dim) {
  if (!plain(qo.ptr()) || !plain(po.ptr()) || !plain(to.ptr()) || !(ko.is_none() || plain(ko.ptr())))
    return py::none();
  const Tensor q = THPVariable_Unpack(qo.ptr()), pos = THPVariable_Unpack(po.ptr()), turns = THPVariable_Unpack(to.ptr());
  const Tensor k = ko.is_none() ? Tensor() : THPVariable_Unpack(ko.ptr());
  if (!plain_context() || !readable(q) || (k.defined() && !readable(k))) return py::none();
  const HeadRows a = head_rows(q);
  if (!a.ok || dtype_code(q.scalar_type()) < 0 || turns.scalar_type() != at::kDouble || !turns.is_contiguous() ||
      turns.numel() * 2 != rotary_dim || turns.device() != q.device() || pos.device() != q.device() ||
      (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt) || !pos.is_contiguous() ||
      pos.numel() != a.tokens || pos.dim() != q.dim() - 2)
    return py::none();
  for (int64_t i = 0; i < pos.dim(); ++i)
    if (pos.size(i) != q.size(i)) return py::none();
  if (k.defined()) {
    const HeadRows b = head_rows(k);
    if (!b.ok || b.D != a.D || k.scalar_type() != q.scalar_type() || k.device() != q.device() || k.dim() != q.dim())
      return py::none();
    for (int64_t i = 0; i < pos.dim(); ++i)
      if (k.size(i) != q.size(i)) return py::none();
  }
  variable_list y;
  {
    py::gil_scoped_release release;
    if (grads_needed({&q}) || (k.defined() && grads_needed({&k})))
      y = RotaryFunction::apply(q, k.defined() ? std::optional<Tensor>(k) : std::nullopt, pos, turns, magnitude, (int64_t)half, rotary_dim, (int64_t)0);
    else
      y = turn(q, k, pos, turns, RotaryPlan{magnitude, half, rotary_dim, 0});
  }
  py::object yk = py::none();
  if (k.defined()) yk = py::reinterpret_steal<py::object>(THPVariable_Wrap(y[1]));
  return py::make_tuple(py::reinterpret_steal<py::object>(THPVariable_Wrap(y[0])), yk);
}

// The C description of a cache; false: Python checks it
bool describe(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, const Tensor* starts,
              int64_t tokens, ca_paged_cache& c) {
  if (!readable(k) || !readable(v) || k.dim() != 4 || v.sizes() != k.sizes() || v.strides() != k.strides() ||
      v.scalar_type() != k.scalar_type() || dtype_code(k.scalar_type()) < 0 || v.device() != k.device() ||
      k.numel() == 0 || k.stride(3) != 1)
    return false;
  for (int i = 0; i < 4; ++i)
    if (k.size(i) > (1 << 30)) return false;
  const c10::Device device = k.device();
  if (!counts(table, device) || table.dim() != 2 || table.numel() == 0 || !counts(lengths, device) ||
      lengths.dim() != 1 || lengths.size(0) != table.size(0) || table.size(0) > (1 << 24) || table.size(1) > (1 << 30))
    return false;
  if (starts && (!counts(*starts, device) || starts->dim() != 1 || starts->size(0) != table.size(0) + 1)) return false;
  c = ca_paged_cache{};
  c.k = const_cast<void*>(k.const_data_ptr());
  c.v = const_cast<void*>(v.const_data_ptr());
  c.table = table.const_data_ptr<int>();
  c.lengths = lengths.const_data_ptr<int>();
  c.starts = starts ? starts->const_data_ptr<int>() : nullptr;
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.row_stride = k.stride(2);
  c.table_stride = table.size(1);
  c.dtype = dtype_code(k.scalar_type());
  c.heads = (int)k.size(1);
  c.head_dim = (int)k.size(3);
  c.page_size = (int)k.size(2);
  c.num_pages = (int)k.size(0);
  c.pages_per_seq = (int)table.size(1);
  c.batch = (int)table.size(0);
  c.tokens = (int)tokens;
  return true;
}
bool shares_memory(const Tensor& a, const Tensor& b) {
  return a.storage().unsafeGetStorageImpl() == b.storage().unsafeGetStorageImpl() || a.const_data_ptr() == b.const_data_ptr() ||
         a.storage().data() == b.storage().data();
}
bool good_out(const Tensor& out, const Tensor& q) {
  return readable(out) && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() &&
         out.device() == q.device() && out.stride(2) == 1 && disjoint(out) && !shares_memory(out, q) && !grads_needed({&out});
}

py::object append(py::handle qo, py::handle ko, py::handle vo, py::handle po, py::handle to, double magnitude,
                  bool half, int64_t rotary_dim, py::handle kpo, py::handle vpo, py::handle table_o,
                  py::handle lengths_o, py::handle starts_o, py::handle oo) {
  for (const py::handle& o : {qo, ko, vo, po, to, kpo, vpo, table_o, lengths_o, starts_o})
    if (!plain(o.ptr())) return py::none();
  if (!oo.is_none() && !plain(oo.ptr())) return py::none();
  const Tensor q = THPVariable_Unpack(qo.ptr()), k = THPVariable_Unpack(ko.ptr()), v = THPVariable_Unpack(vo.ptr()),
               pos = THPVariable_Unpack(po.ptr()), turns = THPVariable_Unpack(to.ptr()), kp = THPVariable_Unpack(kpo.ptr()),
               vp = THPVariable_Unpack(vpo.ptr()), table = THPVariable_Unpack(table_o.ptr()),
               lengths = THPVariable_Unpack(lengths_o.ptr()), starts = THPVariable_Unpack(starts_o.ptr());
  if (!plain_context() || !readable(q) || !readable(k) || !readable(v) || q.dim() != 3 || k.dim() != 3 ||
      k.sizes() != v.sizes() || grads_needed({&q, &k, &v, &kp, &vp}))
    return py::none();
  const HeadRows a = head_rows(q), b = head_rows(k), w = head_rows(v);
  if (!a.ok || !b.ok || !w.ok || a.tokens != b.tokens || a.D != b.D || k.scalar_type() != q.scalar_type() ||
      v.scalar_type() != q.scalar_type() || kp.scalar_type() != q.scalar_type() || kp.device() != q.device() ||
      k.device() != q.device() || v.device() != q.device())
    return py::none();
  if (turns.scalar_type() != at::kDouble || !turns.is_contiguous() || turns.numel() * 2 != rotary_dim ||
      turns.device() != q.device() || pos.device() != q.device() || pos.dim() != 1 || pos.numel() != a.tokens ||
      (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt) || !pos.is_contiguous())
    return py::none();
  ca_paged_cache c;
  if (!describe(kp, vp, table, lengths, &starts, a.tokens, c) || c.heads != b.heads || c.head_dim != b.D ||
      !disjoint(kp) || c.k == c.v)
    return py::none();
  Tensor out;
  if (!oo.is_none()) {
    out = THPVariable_Unpack(oo.ptr());
    if (!good_out(out, q)) return py::none();
  }
  {
    py::gil_scoped_release release;
    const c10::DeviceGuard guard(q.device());
    if (!out.defined()) out = empty(q.sizes(), q, q.scalar_type());
    ca_rotary r{};
    r.q = q.const_data_ptr();
    r.k = k.const_data_ptr();
    r.q_out = out.data_ptr();
    r.positions = pos.const_data_ptr();
    r.turns = turns.const_data_ptr<double>();
    r.q_token_stride = a.ts;
    r.q_head_stride = a.hs;
    r.k_token_stride = b.ts;
    r.k_head_stride = b.hs;
    r.q_out_token_stride = out.stride(0);
    r.q_out_head_stride = out.stride(1);
    r.magnitude = (float)magnitude;
    r.positions64 = pos.scalar_type() == at::kLong;
    r.half = half;
    r.dtype = c.dtype;
    r.tokens = (int)a.tokens;
    r.q_heads = (int)a.heads;
    r.k_heads = (int)b.heads;
    r.head_dim = (int)a.D;
    r.rotary_dim = (int)rotary_dim;
    check(ca_rotary_append(&r, v.const_data_ptr(), w.ts, w.hs, &c, stream_of(q)));
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// max_new, max_length: -1 for the defaults
py::object attend(py::handle qo, py::handle kpo, py::handle vpo, py::handle table_o, py::handle lengths_o,
                  py::handle starts_o, py::handle go, int64_t max_new, int64_t max_length, py::handle so,
                  py::handle oo) {
  for (const py::handle& o : {qo, kpo, vpo, table_o, lengths_o, starts_o, go})
    if (!plain(o.ptr())) return py::none();
  for (const py::handle& o : {so, oo})
    if (!o.is_none() && !plain(o.ptr())) return py::none();
  const Tensor q = THPVariable_Unpack(qo.ptr()), kp = THPVariable_Unpack(kpo.ptr()), vp = THPVariable_Unpack(vpo.ptr()),
               table = THPVariable_Unpack(table_o.ptr()), lengths = THPVariable_Unpack(lengths_o.ptr()),
               starts = THPVariable_Unpack(starts_o.ptr()), gain = THPVariable_Unpack(go.ptr());
  if (!plain_context() || !readable(q) || q.dim() != 3 || !usable(gain) || gain.scalar_type() != at::kFloat ||
      grads_needed({&q, &kp, &vp, &gain}) || max_new < -1 || max_length < -1)
    return py::none();
  const HeadRows a = head_rows(q);
  const int64_t esize = q.element_size();
  ca_paged_cache c;
  if (!a.ok || !describe(kp, vp, table, lengths, &starts, a.tokens, c) || kp.device() != q.device() ||
      q.scalar_type() != kp.scalar_type() || c.head_dim != a.D || a.D % 8 || a.D > 128 || a.heads % c.heads ||
      gain.numel() != a.heads || gain.device() != q.device() || !aligned(q) || a.ts * esize % 16 || a.hs * esize % 16)
    return py::none();
  const int64_t capacity = (int64_t)c.pages_per_seq * c.page_size;
  if (capacity > (1 << 30)) return py::none();
  if (max_new < 0) max_new = a.tokens;
  if (max_length < 0 || max_length > capacity) max_length = capacity;
  max_new = std::min(max_new, a.tokens);
  Tensor sums, out;
  if (!so.is_none()) {
    sums = THPVariable_Unpack(so.ptr());
    if (!readable(sums) || sums.dim() != 3 || sums.scalar_type() != at::kFloat || sums.size(0) != c.batch ||
        sums.size(1) != c.heads || sums.numel() == 0 || sums.stride(2) != 1 || sums.device() != q.device() ||
        sums.size(2) > (1 << 30) || !disjoint(sums) || grads_needed({&sums}))
      return py::none();
  }
  if (!oo.is_none()) {
    out = THPVariable_Unpack(oo.ptr());
    if (!good_out(out, q) || !aligned(out) || out.stride(0) * esize % 16 || out.stride(1) * esize % 16) return py::none();
  }
  {
    py::gil_scoped_release release;
    const c10::DeviceGuard guard(q.device());
    if (!out.defined()) out = empty(q.sizes(), q, q.scalar_type());
    const size_t bytes = ca_paged_attention_workspace_bytes(c.dtype, c.batch, c.heads, (int)a.heads, c.head_dim,
                                                            c.tokens, (int)max_new, (int)max_length, sums.defined());
    Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    check(ca_paged_attention(&c, q.const_data_ptr(), a.ts, a.hs, (int)a.heads, gain.const_data_ptr<float>(),
                             out.data_ptr(), out.stride(0), out.stride(1),
                             sums.defined() ? sums.data_ptr<float>() : nullptr, sums.defined() ? sums.stride(0) : 0,
                             sums.defined() ? sums.stride(1) : 0, sums.defined() ? (int)sums.size(2) : 0, (int)max_new,
                             (int)max_length, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

py::object evict(py::handle kpo, py::handle vpo, py::handle table_o, py::handle lengths_o, py::handle so,
                 py::handle new_o, int64_t budget, int64_t sinks, int64_t recent) {
  for (const py::handle& o : {kpo, vpo, table_o, lengths_o, so, new_o})
    if (!plain(o.ptr())) return py::none();
  const Tensor kp = THPVariable_Unpack(kpo.ptr()), vp = THPVariable_Unpack(vpo.ptr()), table = THPVariable_Unpack(table_o.ptr()),
               lengths = THPVariable_Unpack(lengths_o.ptr()), sums = THPVariable_Unpack(so.ptr()),
               to = THPVariable_Unpack(new_o.ptr());
  ca_paged_cache c;
  if (!plain_context() || grads_needed({&kp, &vp, &sums}) || !describe(kp, vp, table, lengths, nullptr, 0, c) ||
      !readable(sums) || sums.dim() != 3 || sums.scalar_type() != at::kFloat || sums.size(0) != c.batch ||
      sums.size(1) != c.heads || sums.numel() == 0 || sums.stride(2) != 1 || sums.device() != kp.device() ||
      sums.size(2) > (1 << 30) || !disjoint(kp) || !counts(to, kp.device()) || to.dim() != 2 || to.size(0) != c.batch ||
      budget <= 0 || budget > (1 << 30) || sinks < 0 || recent < 0 || sinks + recent > budget ||
      to.size(1) * c.page_size < budget)
    return py::none();
  Tensor kept, lens, new_sums;
  {
    py::gil_scoped_release release;
    const c10::DeviceGuard guard(kp.device());
    kept = empty({c.batch, c.heads, budget}, kp, at::kInt);
    new_sums = empty({c.batch, c.heads, budget}, kp, at::kFloat);
    lens = empty({c.batch}, kp, at::kInt);
    check(ca_evict(&c, sums.const_data_ptr<float>(), sums.stride(0), sums.stride(1), (int)sums.size(2), (int)budget,
                   (int)sinks, (int)recent, to.const_data_ptr<int>(), to.size(1), kept.data_ptr<int>(),
                   new_sums.data_ptr<float>(), lens.data_ptr<int>(), stream_of(kp)));
  }
  return py::make_tuple(py::reinterpret_steal<py::object>(THPVariable_Wrap(kept)),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(lens)),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(new_sums)));
}

// weight: an Int4Weight's tensors, checked when it was made
py::object int4_product(py::handle xo, py::handle co, py::handle so, py::handle zo, int64_t N, int64_t K, int64_t group) {
  for (const py::handle& o : {xo, co, so})
    if (!plain(o.ptr())) return py::none();
  if (!zo.is_none() && !plain(zo.ptr())) return py::none();
  const Tensor x = THPVariable_Unpack(xo.ptr()), codes = THPVariable_Unpack(co.ptr()), scales = THPVariable_Unpack(so.ptr());
  const Tensor zeros = zo.is_none() ? Tensor() : THPVariable_Unpack(zo.ptr());
  if (!plain_context() || !readable(x) || x.dim() < 1 || x.numel() == 0 || x.size(-1) != K || grads_needed({&x}) ||
      dtype_code(x.scalar_type()) < 0 || scales.scalar_type() != x.scalar_type() || codes.device() != x.device() ||
      !usable(codes) || codes.scalar_type() != at::kInt || N <= 0 ||
      codes.numel() != (N + 15) / 16 * ((K + 127) / 128) * 256 || !usable(scales) || scales.device() != x.device() || group <= 0 ||
      scales.numel() != (K + group - 1) / group * ((N + 15) / 16 * 16) ||
      (zeros.defined() && (zeros.scalar_type() != x.scalar_type() || !usable(zeros) ||
                           zeros.numel() != scales.numel() || zeros.device() != x.device())))
    return py::none();
  const int64_t M = x.numel() / K;
  int64_t rs = K;
  if (x.dim() == 2 && x.stride(1) == 1 && (x.stride(0) >= K || M == 1))
    rs = std::max(x.stride(0), K);
  else if (!x.is_contiguous())
    return py::none();
  if (M > (1 << 19) || N > (1 << 26) || K > (1 << 30)) return py::none();
  Tensor y;
  {
    py::gil_scoped_release release;
    const c10::DeviceGuard guard(x.device());
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = N;
    y = empty(shape, x, x.scalar_type());
    check(ca_int4_linear(x.const_data_ptr(), rs, reinterpret_cast<const unsigned*>(codes.const_data_ptr<int>()),
                         scales.const_data_ptr(), zeros.defined() ? zeros.const_data_ptr() : nullptr, y.data_ptr(), N,
                         dtype_code(x.scalar_type()), (int)M, (int)N, (int)K, (int)group, stream_of(x)));
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(y));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_error", [](py::object cls) { ca_error = cls.release().ptr(); });
  m.def("check", &check, py::call_guard<py::gil_scoped_release>());
  m.def("op", &op);
  m.def("rope_attention", &rope_attention);
  m.def("rmsnorm", &rmsnorm);
  m.def("add_rmsnorm", &add_rmsnorm);
  m.def("weights", &weights);
  m.def("rotary", &rotary);
  m.def("append", &append);
  m.def("attend", &attend);
  m.def("evict", &evict);
  m.def("int4", &int4_product);
}
