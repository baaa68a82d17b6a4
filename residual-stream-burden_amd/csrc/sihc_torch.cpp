// Native dispatch of the eager `sihc::` ops.
//
// The Python custom ops (sihc_hip/sublayer_kernels.py, event_ops.py, indexed.py, kernels.py,
// conditioning.py, body.py) cost 50-150 us of interpreter and dispatcher time per forward and backward pair,
// more than the kernels of a small or ordinary call take. Each function here takes the arguments of one
// of those ops and, where the call is plain, allocates the outputs, enqueues the C-ABI call on
// the current stream and records one C++ autograd node whose backward does the same.
//
// Plain means: exactly the tensors and shapes that the op accepts, all packed (attention: with
// adjacent channels), dense, on one GPU and not empty, of type torch.Tensor or
// torch.nn.Parameter, and nothing in force that has to see the op: no dispatch or function mode (tracing, fake tensors, selective checkpointing),
// no functorch transform, no forward-mode tangent, and no kernel or autocast rule that the
// program registered for the op itself. Anything else returns NotImplemented and
// the caller runs the Python op, which validates, raises and composes as it always did. The
// same holds in a backward: under create_graph, or where a mode or a wrapped tensor shows up
// there, the node calls the registered ops through the dispatcher. Inputs are kept with
// save_for_backward, so saved-tensor hooks and version checks apply, and undefined output
// gradients are materialised as zeros, as for the Python ops. An unpack hook may return another
// type, shape, layout or device than was saved, so every backward repeats the forward's checks on
// what it got, and leaves operands that do not fit to the registered ops, which raise.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "sihc_hip.h"

namespace {

using at::Tensor;
using at::TensorList;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

PyObject* parameter_type = nullptr;  // torch.nn.Parameter

struct Failure {};  // a C-ABI call returned an error in a forward: the Python op repeats and reports it

// ------------------------------------------------------------------ what may run here
bool plain_mode() {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  if (!(tls.included_ - c10::default_included_set).empty()) return false;
  return !at::impl::torch_function_mode_enabled();
}
bool plain_strided(const Tensor& t) {
  static const c10::DispatchKeySet special({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                            c10::DispatchKey::FuncTorchBatched,
                                            c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                            c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                            c10::DispatchKey::ZeroTensor});
  return t.defined() && t.is_cuda() && t.layout() == c10::kStrided && !t.is_quantized() && !t.is_nested() &&
         !t.key_set().has_any(special) && !t._fw_grad(0).defined();
}
bool plain(const Tensor& t) { return plain_strided(t) && t.is_contiguous(); }
// The registered ops of a backward would drop a forward-mode tangent (a transform's tensor may hide one).
void refuse_tangents(const char* op, std::initializer_list<Tensor> grads) {
  for (const Tensor& t : grads)
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined() && !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper), op,
                                ": no forward-mode derivative");
}
bool below_autograd() {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  return tls.excluded_.has(c10::DispatchKey::AutogradCUDA);
}
int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return SIHC_DTYPE_F32;
  return t.scalar_type() == at::kBFloat16 ? SIHC_DTYPE_BF16 : -1;
}
bool unwrap(PyObject* o, Tensor& t) {
  PyObject* type = reinterpret_cast<PyObject*>(Py_TYPE(o));
  if (type != THPVariableClass && type != parameter_type) return false;
  t = THPVariable_Unpack(o);
  return true;
}
bool unwrap_list(PyObject* o, std::vector<Tensor>& out) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  out.resize(size_t(n));
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!unwrap(PySequence_Fast_GET_ITEM(o, i), out[size_t(i)])) return false;
  return true;
}

struct Shape {
  int64_t batch, grid, cell, channels, slots;
};
// A square NHWC carrier of whole cells and weights whose last dimensions are [channels, slots].
bool carrier_shape(const Tensor& x, const Tensor& w, Shape& s) {
  if (x.dim() != 4 || w.dim() < 2 || x.numel() == 0 || dtype_code(x) < 0) return false;
  s.slots = w.size(-1);
  if (s.slots != 4 && s.slots != 16) return false;
  s.cell = s.slots == 4 ? 2 : 4;
  s.batch = x.size(0);
  s.channels = x.size(3);
  s.grid = x.size(1) / s.cell;
  return x.size(1) == x.size(2) && x.size(1) % s.cell == 0 && w.size(-2) == s.channels &&
         w.scalar_type() == x.scalar_type() && w.device() == x.device() && s.channels < (int64_t(1) << 31) &&
         s.grid < (int64_t(1) << 15);
}
bool token_shape(const Tensor& z, const Tensor& x, const Shape& s) {
  return z.dim() == 3 && z.size(0) == s.batch && z.size(1) == s.grid * s.grid && z.size(2) == s.channels &&
         z.scalar_type() == x.scalar_type() && z.device() == x.device();
}
bool index_shape(const Tensor& index, const Tensor& x, const Shape& s) {
  return index.scalar_type() == at::kInt && index.dim() == 2 && index.size(0) == s.batch &&
         index.size(1) == s.grid * s.grid && index.device() == x.device();
}

// Everything the launches below take for granted about their operands: asked by the Python
// entries of the arguments and by the backward nodes of the gradients and unpacked tensors.
bool read_fits(const Tensor& x, const Tensor& alpha, const Tensor& index, Shape& s) {
  return plain(x) && plain(alpha) && alpha.dim() == 3 && alpha.size(0) >= 1 && alpha.size(0) <= SIHC_MAX_EVENTS &&
         carrier_shape(x, alpha, s) && (!index.defined() || (plain(index) && index_shape(index, x, s)));
}
// (also the adjoint of the read, whose gradients have the updates' shape)
bool write_fits(const Tensor& x, TensorList updates, const Tensor& beta, const Tensor& index, Shape& s) {
  if (!read_fits(x, beta, index, s) || beta.size(0) != int64_t(updates.size())) return false;
  for (const Tensor& u : updates)
    if (!plain(u) || !token_shape(u, x, s)) return false;
  return true;
}
bool triangular_fits(const Tensor& base, TensorList updates, const Tensor& gamma) {
  if (!plain(base) || !plain(gamma) || base.dim() < 1 || base.numel() == 0 || dtype_code(base) < 0 ||
      updates.empty() || updates.size() > SIHC_MAX_EVENTS || gamma.dim() != 2 ||
      gamma.size(0) != int64_t(updates.size()) || gamma.size(1) != base.size(-1) ||
      gamma.device() != base.device() ||
      (gamma.scalar_type() != base.scalar_type() && gamma.scalar_type() != at::kFloat))
    return false;
  for (const Tensor& u : updates)
    if (!plain(u) || !u.sizes().equals(base.sizes()) || u.scalar_type() != base.scalar_type() ||
        u.device() != base.device())
      return false;
  return true;
}
bool event_fits(const Tensor& x, const Tensor& dz, const Tensor& beta, const Tensor& alpha) {
  Shape s{};
  return plain(x) && plain(dz) && plain(beta) && plain(alpha) && beta.dim() == 2 && carrier_shape(x, beta, s) &&
         token_shape(dz, x, s) && alpha.sizes().equals(beta.sizes()) && alpha.scalar_type() == x.scalar_type() &&
         alpha.device() == x.device();
}
bool gather_fits(const Tensor& x, const Tensor& index, int64_t slots) {
  if (!plain(x) || !plain(index)) return false;
  const int64_t k = slots == 4 ? 2 : 4;
  if (x.dim() != 4 || x.numel() == 0 || dtype_code(x) < 0 || (slots != 4 && slots != 16) ||
      x.size(1) != x.size(2) || x.size(1) % k != 0 || x.size(3) >= (int64_t(1) << 31))
    return false;
  const Shape s{x.size(0), x.size(1) / k, k, x.size(3), slots};
  // (the adjoint holds a batch row of the index in LDS: 16384 cells)
  return index_shape(index, x, s) && s.grid <= 128;
}
bool scatter_fits(const Tensor& cells, const Tensor& index) {
  if (!plain(cells) || !plain(index) || cells.dim() != 4 || cells.numel() == 0 || dtype_code(cells) < 0 ||
      (cells.size(2) != 4 && cells.size(2) != 16) || cells.size(1) > 16384 || cells.size(3) >= (int64_t(1) << 31))
    return false;
  Shape s{cells.size(0), 1, cells.size(2) == 4 ? 2 : 4, cells.size(3), cells.size(2)};
  while (s.grid * s.grid < cells.size(1)) ++s.grid;
  return s.grid * s.grid == cells.size(1) && index_shape(index, cells, s);
}

bool embed_fits(const Tensor& table, const Tensor& ids) {
  return plain(table) && plain(ids) && table.dim() == 2 && table.numel() != 0 && ids.numel() != 0 &&
         dtype_code(table) >= 0 && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) &&
         ids.device() == table.device() && table.size(1) < (int64_t(1) << 31);
}
bool norm_fits(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups) {
  if (!plain(x) || !plain(weight) || !plain(bias) || x.dim() < 2 || x.numel() == 0 || dtype_code(x) < 0) return false;
  const int64_t c = x.size(-1);
  if (groups < 1 || c % groups || c > (int64_t(1) << 24)) return false;
  const int64_t width = c / groups;  // (wider groups: the registered op says what is taken)
  if (width > (x.scalar_type() == at::kBFloat16 && width % 8 == 0 ? 4096 : width % 2 == 0 ? 2048 : 1024)) return false;
  for (const Tensor* w : {&weight, &bias})
    if (w->dim() != 1 || w->size(0) != c || w->device() != x.device() || w->scalar_type() != weight.scalar_type())
      return false;
  return weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat;
}
bool attention_fits(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths) {
  for (const Tensor* t : {&q, &k, &v})
    if (!plain_strided(*t) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type() ||
        t->device() != q.device() || (t->size(3) > 1 && t->stride(3) != 1) || t->size(1) >= (int64_t(1) << 31) ||
        t->size(2) >= (int64_t(1) << 31))
      return false;
  if (dtype_code(q) < 0 || !k.sizes().equals(v.sizes()) || k.size(0) != q.size(0) || k.size(3) != q.size(3) ||
      q.size(3) > SIHC_MAX_HEAD_DIM || q.size(2) % k.size(2))
    return false;
  return !lengths.defined() || (plain(lengths) && lengths.scalar_type() == at::kInt && lengths.dim() == 1 &&
                                lengths.size(0) == q.size(0) && lengths.device() == q.device());
}
// Absent operands are undefined tensors here.
bool linear_fits(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& gate, const Tensor& residual,
                 int act) {
  if (!plain(x) || !plain(weight) || x.dim() < 2 || weight.dim() != 2 || x.numel() == 0 || weight.numel() == 0 ||
      dtype_code(x) < 0 || x.size(-1) != weight.size(1) || weight.size(0) > (1 << 24) || weight.size(1) > (1 << 24) ||
      x.numel() / x.size(-1) > (1 << 30) || (act == SIHC_ACT_SWIGLU && weight.size(0) % 2))
    return false;
  const int64_t outer = act == SIHC_ACT_SWIGLU ? weight.size(0) / 2 : weight.size(0);
  for (const Tensor* t : {&weight, &bias, &gate, &residual})
    if (t->defined() && (!plain_strided(*t) || t->scalar_type() != x.scalar_type() || t->device() != x.device()))
      return false;
  if (bias.defined() && (!bias.is_contiguous() || bias.dim() != 1 || bias.size(0) != weight.size(0))) return false;
  if (gate.defined() && (gate.dim() != 2 || gate.size(0) != x.size(0) || gate.size(1) != outer ||
                         (outer > 1 && gate.stride(1) != 1)))
    return false;
  return !residual.defined() ||
         (residual.is_contiguous() && residual.dim() == x.dim() && residual.size(-1) == outer &&
          residual.sizes().slice(0, size_t(x.dim()) - 1).equals(x.sizes().slice(0, size_t(x.dim()) - 1)));
}
// (k: undefined where x is turned alone)
bool heads_fit(const Tensor& q, const Tensor& k, const Tensor& positions, const std::vector<int64_t>& axes,
               double theta) {
  for (const Tensor* t : {&q, &k}) {
    if (t == &k && !k.defined()) continue;
    if (!plain_strided(*t) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type() ||
        t->device() != q.device() || t->size(0) != q.size(0) || t->size(1) != q.size(1) || t->size(3) != q.size(3) ||
        t->size(2) > (1 << 20) || (t->size(3) > 1 && t->stride(3) != 1))
      return false;
  }
  int64_t sum = 0;
  for (const int64_t w : axes) {
    if (w < 0 || w % 2 || w > SIHC_MAX_ROTARY_DIM) return false;
    sum += w;
  }
  if (dtype_code(q) < 0 || q.size(3) > SIHC_MAX_ROTARY_DIM || axes.size() > SIHC_MAX_AXES || sum > q.size(3) ||
      q.size(0) * q.size(1) > (int64_t(1) << 26) - 4 || !(theta > 0.0) || !std::isfinite(theta))
    return false;  // (of more tokens, the registered op knows whether a launch takes them)
  if (!plain(positions) || positions.device() != q.device() ||
      (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kFloat))
    return false;
  const int64_t n = positions.dim(), count = int64_t(axes.size());
  return (n == 2 && positions.size(0) == q.size(1) && positions.size(1) == count) ||
         (n == 3 && positions.size(0) == q.size(0) && positions.size(1) == q.size(1) && positions.size(2) == count);
}
bool qk_fits(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& positions,
             const std::vector<int64_t>& axes, double theta, double eps) {
  if (!k.defined() || !heads_fit(q, k, positions, axes, theta) || !(eps >= 0.0) || !std::isfinite(eps)) return false;
  for (const Tensor* w : {&qw, &kw})
    if (!plain(*w) || w->dim() != 1 || w->size(0) != q.size(3) || w->device() != q.device() ||
        w->scalar_type() != qw.scalar_type())
      return false;
  return qw.scalar_type() == q.scalar_type() || qw.scalar_type() == at::kFloat;
}
bool dropout_fits(const Tensor& x, double p, const Tensor& seed, int64_t stream, const Tensor& residual) {
  return plain(x) && x.numel() != 0 && dtype_code(x) >= 0 && p >= 0.0 && p < 1.0 && plain(seed) &&
         seed.scalar_type() == at::kLong && seed.numel() == 1 && seed.device() == x.device() && stream >= 0 &&
         (!residual.defined() || (plain(residual) && residual.sizes().equals(x.sizes()) &&
                                  residual.scalar_type() == x.scalar_type() && residual.device() == x.device()));
}
// `t` is a packed tensor like `like` (an output gradient, a saved output).
bool same(const Tensor& t, const Tensor& like) {
  return plain(t) && t.sizes().equals(like.sizes()) && t.scalar_type() == like.scalar_type() &&
         t.device() == like.device();
}
bool stats_fits(const Tensor& t, at::IntArrayRef sizes, const Tensor& like) {
  return plain(t) && t.sizes().equals(sizes) && t.scalar_type() == at::kFloat && t.device() == like.device();
}

// ----------------------------------------------------------------------- the C-ABI calls
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void check(int rc, bool forward) {
  if (rc == SIHC_OK) return;
  if (forward) throw Failure{};
  TORCH_CHECK(false, sihc_last_error());
}
struct Ptrs {
  void* p[SIHC_MAX_EVENTS] = {};
  explicit Ptrs(TensorList ts) {
    for (size_t i = 0; i < ts.size(); ++i) p[i] = ts[i].data_ptr();
  }
  const void* const* in() const { return const_cast<const void* const*>(p); }
};
const int32_t* index_ptr(const Tensor& index) { return index.defined() ? index.const_data_ptr<int32_t>() : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({int64_t((std::max<size_t>(bytes, 4) + 63) / 64 * 16)}, like.options().dtype(at::kFloat));
}
Shape shape_of(const Tensor& x, const Tensor& w) {
  Shape s{};
  s.slots = w.size(-1);
  s.cell = s.slots == 4 ? 2 : 4;
  s.batch = x.size(0);
  s.channels = x.size(3);
  s.grid = x.size(1) / s.cell;
  return s;
}

variable_list run_read(const Tensor& x, const Tensor& alpha, const Tensor& index) {
  const c10::DeviceGuard guard(x.device());
  const Shape s = shape_of(x, alpha);
  variable_list out;
  out.reserve(size_t(alpha.size(0)));
  for (int64_t e = 0; e < alpha.size(0); ++e)
    out.push_back(at::empty({s.batch, s.grid * s.grid, s.channels}, x.options()));
  check(sihc_read(x.const_data_ptr(), alpha.const_data_ptr(), Ptrs(out).p, int(out.size()), s.batch, int(s.grid),
                  int(s.cell), int(s.channels), index_ptr(index), dtype_code(x), stream_of(x)),
        true);
  return out;
}
Tensor run_write(const Tensor& x, TensorList updates, const Tensor& beta, const Tensor& index) {
  const c10::DeviceGuard guard(x.device());
  const Shape s = shape_of(x, beta);
  Tensor out = at::empty_like(x);
  check(sihc_write(x.const_data_ptr(), Ptrs(updates).in(), beta.const_data_ptr(), out.data_ptr(), int(updates.size()),
                   s.batch, int(s.grid), int(s.cell), int(s.channels), 1, index_ptr(index), dtype_code(x),
                   dtype_code(beta), stream_of(x)),
        true);
  return out;
}
std::tuple<Tensor, Tensor> run_read_backward(const Tensor& x, TensorList grads, const Tensor& alpha,
                                             const Tensor& index) {
  const c10::DeviceGuard guard(x.device());
  const Shape s = shape_of(x, alpha);
  Tensor dx = at::empty_like(x), da = at::empty_like(alpha);
  const int events = int(grads.size());
  Tensor ws = workspace(
      sihc_weight_grad_workspace_size(events, s.batch, int(s.grid), int(s.cell), int(s.channels)), x);
  check(sihc_read_backward(x.const_data_ptr(), Ptrs(grads).in(), alpha.const_data_ptr(), dx.data_ptr(), da.data_ptr(),
                           events, s.batch, int(s.grid), int(s.cell), int(s.channels), index_ptr(index),
                           dtype_code(x), dtype_code(da), ws.data_ptr(), size_t(ws.numel()) * 4, stream_of(x)),
        false);
  return {dx, da};
}
std::tuple<variable_list, Tensor> run_write_backward(const Tensor& grad, TensorList updates, const Tensor& beta,
                                                     const Tensor& index) {
  const c10::DeviceGuard guard(grad.device());
  const Shape s = shape_of(grad, beta);
  variable_list dz;
  for (const Tensor& u : updates) dz.push_back(at::empty_like(u));
  Tensor db = at::empty_like(beta);
  const int events = int(updates.size());
  Tensor ws = workspace(
      sihc_weight_grad_workspace_size(events, s.batch, int(s.grid), int(s.cell), int(s.channels)), grad);
  check(sihc_write_backward(grad.const_data_ptr(), Ptrs(updates).in(), beta.const_data_ptr(), Ptrs(dz).p,
                            db.data_ptr(), events, s.batch, int(s.grid), int(s.cell), int(s.channels),
                            index_ptr(index), dtype_code(grad), dtype_code(db), ws.data_ptr(),
                            size_t(ws.numel()) * 4, stream_of(grad)),
        false);
  return {dz, db};
}

// --------------------------------------------------------------------------- dispatcher
template <typename Sig>
auto registered(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}
// A backward may launch directly: nothing recorded or in force (its operands are asked apart).
bool direct() { return !at::GradMode::is_enabled() && plain_mode(); }

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// What a profiler sees of a call: the op's name and its arguments (made only if one looks).
using Args = std::vector<c10::IValue>;
Args listed(const Tensor& x, TensorList ts, const Tensor& w, const Tensor& index) {
  Args args{x, ts.vec(), w};
  if (index.defined()) args.emplace_back(index);
  return args;
}
// ------------------------------------------------------------------------ autograd nodes
struct ReadFn : torch::autograd::Function<ReadFn> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& alpha,
                               const std::optional<Tensor>& index) {
    const Tensor idx = index.value_or(Tensor());
    ctx->save_for_backward({x, alpha, idx});
    return run_read(x, alpha, idx);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &alpha = saved[1], &index = saved[2];
    for (Tensor& g : grads) g = g.contiguous();
    std::tuple<Tensor, Tensor> r;
    Shape s{};
    if (direct() && write_fits(x, grads, alpha, index, s)) {
      RECORD_FUNCTION(index.defined() ? "sihc::indexed_read_backward" : "sihc::sublayer_read_backward",
                      listed(x, grads, alpha, index));
      r = run_read_backward(x, grads, alpha, index);
    } else if (index.defined()) {
      static auto op = registered<std::tuple<Tensor, Tensor>(const Tensor&, TensorList, const Tensor&,
                                                             const Tensor&)>("sihc::indexed_read_backward");
      r = op.call(x, grads, alpha, index);
    } else {
      static auto op = registered<std::tuple<Tensor, Tensor>(const Tensor&, TensorList, const Tensor&)>(
          "sihc::sublayer_read_backward");
      r = op.call(x, grads, alpha);
    }
    return {std::get<0>(r), std::get<1>(r), Tensor()};
  }
};

struct WriteFn : torch::autograd::Function<WriteFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, TensorList updates, const Tensor& beta,
                        const std::optional<Tensor>& index) {
    const Tensor idx = index.value_or(Tensor());
    variable_list keep{beta, idx};
    keep.insert(keep.end(), updates.begin(), updates.end());
    ctx->save_for_backward(keep);
    return run_write(x, updates, beta, idx);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &beta = saved[0], &index = saved[1];
    const variable_list updates(saved.begin() + 2, saved.end());
    const Tensor grad = grads[0].contiguous();
    variable_list dz;
    Tensor db;
    Shape s{};
    if (direct() && write_fits(grad, updates, beta, index, s)) {
      RECORD_FUNCTION(index.defined() ? "sihc::indexed_write_backward" : "sihc::sublayer_write_backward",
                      listed(grad, updates, beta, index));
      std::tie(dz, db) = run_write_backward(grad, updates, beta, index);
    } else if (index.defined()) {
      static auto read =
          registered<std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&)>("sihc::indexed_read");
      static auto wgrad = registered<Tensor(const Tensor&, TensorList, const Tensor&, const Tensor&)>(
          "sihc::indexed_weight_grad");
      dz = read.call(grad, beta, index);
      db = wgrad.call(grad, updates, beta, index);
    } else {
      static auto read = registered<std::vector<Tensor>(const Tensor&, const Tensor&)>("sihc::sublayer_read");
      static auto wgrad =
          registered<Tensor(const Tensor&, TensorList, const Tensor&)>("sihc::sublayer_weight_grad");
      dz = read.call(grad, beta);
      db = wgrad.call(grad, updates, beta);
    }
    variable_list out{grad};
    out.insert(out.end(), dz.begin(), dz.end());
    out.push_back(db);
    out.emplace_back();
    return out;
  }
};

Tensor run_triangular(const Tensor& base, TensorList updates, const Tensor& gamma) {
  const c10::DeviceGuard guard(base.device());
  const int64_t c = base.size(-1);
  Tensor out = at::empty_like(base);
  check(sihc_triangular(base.const_data_ptr(), Ptrs(updates).in(), gamma.const_data_ptr(), out.data_ptr(),
                        int(updates.size()), base.numel() / c, int(c), dtype_code(base), dtype_code(gamma),
                        stream_of(base)),
        true);
  return out;
}
struct TriangularFn : torch::autograd::Function<TriangularFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& base, TensorList updates, const Tensor& gamma) {
    variable_list keep{gamma};
    keep.insert(keep.end(), updates.begin(), updates.end());
    ctx->save_for_backward(keep);
    return run_triangular(base, updates, gamma);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& gamma = saved[0];
    const variable_list updates(saved.begin() + 1, saved.end());
    const Tensor grad = grads[0].contiguous();
    variable_list out{grad};
    if (direct() && triangular_fits(grad, updates, gamma)) {
      RECORD_FUNCTION("sihc::sublayer_triangular_backward", listed(grad, updates, gamma, Tensor()));
      const c10::DeviceGuard device(grad.device());
      const int64_t c = grad.size(-1), rows = grad.numel() / c;
      const int active = int(updates.size());
      // one allocation, as the Python op's stacked result
      const Tensor stack = at::empty(
          [&] {
            std::vector<int64_t> sizes{active};
            sizes.insert(sizes.end(), grad.sizes().begin(), grad.sizes().end());
            return sizes;
          }(),
          grad.options());
      const variable_list dz = stack.unbind(0);
      const Tensor dg = at::empty_like(gamma);
      const Tensor ws = workspace(sihc_triangular_gamma_grad_workspace_size(active, rows, int(c)), grad);
      check(sihc_triangular_backward(grad.const_data_ptr(), Ptrs(updates).in(), gamma.const_data_ptr(), Ptrs(dz).p,
                                     dg.data_ptr(), active, rows, int(c), dtype_code(grad), dtype_code(gamma),
                                     dtype_code(dg), ws.data_ptr(), size_t(ws.numel()) * 4, stream_of(grad)),
            false);
      out.insert(out.end(), dz.begin(), dz.end());
      out.push_back(dg);
    } else {
      static auto op = registered<std::tuple<Tensor, Tensor>(const Tensor&, TensorList, const Tensor&)>(
          "sihc::sublayer_triangular_backward");
      const auto [stack, dg] = op.call(grad, updates, gamma);
      for (const Tensor& t : stack.unbind(0)) out.push_back(t);
      out.push_back(dg);
    }
    return out;
  }
};

variable_list run_event(const Tensor& x, const Tensor& dz, const Tensor& beta, const Tensor& alpha) {
  const c10::DeviceGuard guard(x.device());
  const Shape s = shape_of(x, beta);
  Tensor xo = at::empty_like(x), zo = at::empty_like(dz);
  check(sihc_event_forward(x.const_data_ptr(), dz.const_data_ptr(), beta.const_data_ptr(), alpha.const_data_ptr(),
                           xo.data_ptr(), zo.data_ptr(), s.batch, int(s.grid), int(s.cell), int(s.channels), nullptr,
                           dtype_code(x), stream_of(x)),
        true);
  return {xo, zo};
}
struct EventFn : torch::autograd::Function<EventFn> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dz, const Tensor& beta,
                               const Tensor& alpha) {
    variable_list out = run_event(x, dz, beta, alpha);
    ctx->save_for_backward({out[0], dz, beta, alpha});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &xo = saved[0], &dz = saved[1], &beta = saved[2], &alpha = saved[3];
    const Tensor gx = grads[0].contiguous(), gz = grads[1].contiguous();
    if (!direct() || !event_fits(xo, dz, beta, alpha) || !event_fits(gx, gz, beta, alpha) ||
        !gx.sizes().equals(xo.sizes()) || gx.scalar_type() != xo.scalar_type()) {
      static auto op = registered<std::tuple<Tensor, Tensor, Tensor, Tensor>(
          const std::optional<Tensor>&, const std::optional<Tensor>&, const Tensor&, const Tensor&, const Tensor&,
          const Tensor&)>("sihc::event_write_read_backward");
      const auto [a, b, c, d] = op.call(gx, gz, xo, dz, beta, alpha);
      return {a, b, c, d};
    }
    RECORD_FUNCTION("sihc::event_write_read_backward", (Args{gx, gz, xo, dz, beta, alpha}));
    const c10::DeviceGuard device(xo.device());
    const Shape s = shape_of(xo, beta);
    Tensor dx = at::empty_like(xo), ddz = at::empty_like(dz), db = at::empty_like(beta), da = at::empty_like(alpha);
    const Tensor ws = workspace(
        sihc_event_backward_workspace_size(s.batch, int(s.grid), int(s.cell), int(s.channels)), xo);
    check(sihc_event_backward(gx.const_data_ptr(), gz.const_data_ptr(), xo.const_data_ptr(), dz.const_data_ptr(),
                              beta.const_data_ptr(), alpha.const_data_ptr(), dx.data_ptr(), ddz.data_ptr(),
                              db.data_ptr(), da.data_ptr(), s.batch, int(s.grid), int(s.cell), int(s.channels),
                              nullptr, dtype_code(xo), dtype_code(beta), ws.data_ptr(), size_t(ws.numel()) * 4,
                              stream_of(xo)),
          false);
    return {dx, ddz, db, da};
  }
};

// The block-wise stage-end write: one weight tensor per block, stacked for the C ABI; their
// gradients are rows of one [E, C, S] result in the weights' type.
struct BlockWriteFn : torch::autograd::Function<BlockWriteFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, TensorList updates, TensorList betas,
                        const std::string& name) {
    ctx->saved_data["name"] = name;
    variable_list keep(updates.begin(), updates.end());
    keep.insert(keep.end(), betas.begin(), betas.end());
    ctx->save_for_backward(keep);
    return run_write(x, updates, at::stack(betas), Tensor());
  }
  // Updates and one [C, S] weight tensor each, of one type, for a carrier of 16 x 16 cells.
  static bool fits(const Tensor& x, const variable_list& updates, const variable_list& betas) {
    Shape s{};
    if (!plain(x)) return false;
    for (size_t i = 0; i < updates.size(); ++i) {
      const Tensor &u = updates[i], &w = betas[i];
      if (!plain(u) || !plain(w) || w.dim() != 2 || w.size(1) != betas[0].size(1) || !carrier_shape(x, w, s) ||
          s.grid != 16 || !token_shape(u, x, s))
        return false;
    }
    return true;
  }
  static variable_list finish(variable_list out) {
    out.emplace_back();  // the op's name
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const size_t n = saved.size() / 2;
    const variable_list updates(saved.begin(), saved.begin() + long(n)), betas(saved.begin() + long(n), saved.end());
    const Tensor grad = grads[0].contiguous();
    if (direct() && fits(grad, updates, betas)) {
      const Tensor beta = at::stack(betas);
      RECORD_FUNCTION("sihc::sublayer_write_backward", listed(grad, updates, beta, Tensor()));
      const auto [dz, db] = run_write_backward(grad, updates, beta, Tensor());
      variable_list out{grad};
      out.insert(out.end(), dz.begin(), dz.end());
      for (const Tensor& t : db.unbind(0)) out.push_back(t);
      return finish(std::move(out));
    }
    // the gradient ops of the legacy family, which widen bf16 updates and weights to fp32
    std::string name = ctx->saved_data["name"].toStringRef();  // sihc::final_accumulate_<tag>_traceable
    name.resize(name.rfind("_traceable"));
    auto gradient_op = [&](const char* which, const variable_list& rest) {
      const auto op = c10::Dispatcher::singleton().findSchemaOrThrow((name + which).c_str(), "");
      torch::jit::Stack stack{grad};
      for (const Tensor& t : rest) stack.emplace_back(t);
      op.callBoxed(stack);
      return stack.back().toTensor();
    };
    variable_list out{grad};
    for (const Tensor& t : gradient_op("_grad_dz_ptr", betas).unbind(0)) out.push_back(t);
    const variable_list db = gradient_op("_grad_beta_ptr", updates).unbind(0);
    for (size_t i = 0; i < n; ++i) out.push_back(db[i].to(betas[i].scalar_type()));
    return finish(std::move(out));
  }
};

Tensor run_gather(const Tensor& x, const Tensor& index, int64_t slots) {
  const c10::DeviceGuard guard(x.device());
  const int64_t k = slots == 4 ? 2 : 4, g = x.size(1) / k, c = x.size(3);
  Tensor cells = at::empty({x.size(0), g * g, slots, c}, x.options());
  check(sihc_gather_cells(x.const_data_ptr(), index_ptr(index), cells.data_ptr(), x.size(0), int(g), int(k), int(c),
                          dtype_code(x), stream_of(x)),
        true);
  return cells;
}
using CellsCall = int (*)(const void*, const int32_t*, void*, int64_t, int, int, int, int, void*);
Tensor run_scatter(CellsCall call, const Tensor& cells, const Tensor& index, bool forward) {
  const c10::DeviceGuard guard(cells.device());
  const int64_t k = cells.size(2) == 4 ? 2 : 4, c = cells.size(3), g = index.size(1);
  int64_t edge = 1;
  while (edge * edge < g) ++edge;
  Tensor x = at::empty({cells.size(0), edge * k, edge * k, c}, cells.options());
  check(call(cells.const_data_ptr(), index_ptr(index), x.data_ptr(), cells.size(0), int(edge), int(k), int(c),
             dtype_code(cells), stream_of(cells)),
        forward);
  return x;
}
struct GatherFn : torch::autograd::Function<GatherFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& index, int64_t slots) {
    ctx->save_for_backward({index});
    return run_gather(x, index, slots);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor index = ctx->get_saved_variables()[0], grad = grads[0].contiguous();
    if (direct() && scatter_fits(grad, index)) {
      RECORD_FUNCTION("sihc::scatter_add_cells", (Args{grad, index}));
      return {run_scatter(sihc_scatter_add_cells, grad, index, false), Tensor(), Tensor()};
    }
    static auto op = registered<Tensor(const Tensor&, const Tensor&)>("sihc::scatter_add_cells");
    return {op.call(grad, index), Tensor(), Tensor()};
  }
};
struct ScatterFn : torch::autograd::Function<ScatterFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& cells, const Tensor& index) {
    ctx->save_for_backward({index});
    ctx->saved_data["slots"] = cells.size(2);
    return run_scatter(sihc_scatter_cells, cells, index, true);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor index = ctx->get_saved_variables()[0], grad = grads[0].contiguous();
    const int64_t slots = ctx->saved_data["slots"].toInt();
    if (direct() && gather_fits(grad, index, slots)) {
      RECORD_FUNCTION("sihc::gather_cells", (Args{grad, index, slots}));
      return {run_gather(grad, index, slots), Tensor()};
    }
    static auto op = registered<Tensor(const Tensor&, const Tensor&, int64_t)>("sihc::gather_cells");
    return {op.call(grad, index, slots), Tensor()};
  }
};

// ------------------------------------------------------------------ conditioning operators
int id_bits(const Tensor& ids) { return ids.scalar_type() == at::kInt ? 32 : 64; }
Tensor run_embed(const Tensor& table, const Tensor& ids, double scale) {
  const c10::DeviceGuard guard(table.device());
  std::vector<int64_t> sizes(ids.sizes().begin(), ids.sizes().end());
  sizes.push_back(table.size(1));
  Tensor out = at::empty(sizes, table.options());
  check(sihc_embedding(table.const_data_ptr(), ids.const_data_ptr(), out.data_ptr(), ids.numel(), table.size(0),
                       int(table.size(1)), float(scale), id_bits(ids), dtype_code(table), stream_of(table)),
        true);
  return out;
}
struct EmbedFn : torch::autograd::Function<EmbedFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return run_embed(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0], grad = grads[0].contiguous();
    const int64_t rows = ctx->saved_data["rows"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor out;
    if (direct() && plain(ids) && plain(grad) && grad.dim() == ids.dim() + 1 && grad.numel() != 0 &&
        grad.sizes().slice(0, size_t(ids.dim())).equals(ids.sizes()) && dtype_code(grad) >= 0 &&
        (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) && ids.device() == grad.device()) {
      RECORD_FUNCTION("sihc::embedding_lookup_backward", (Args{grad, ids, rows, scale, padding}));
      const c10::DeviceGuard device(grad.device());
      const int c = int(grad.size(-1));
      out = at::empty({rows, c}, grad.options());
      const size_t bytes = sihc_embedding_backward_workspace_size(ids.numel(), rows, c);
      const Tensor ws = bytes ? workspace(bytes, grad) : Tensor();
      check(sihc_embedding_backward(grad.const_data_ptr(), ids.const_data_ptr(), out.data_ptr(), ids.numel(), rows, c,
                                    float(scale), padding, id_bits(ids), dtype_code(grad),
                                    bytes ? ws.data_ptr() : nullptr, bytes, stream_of(grad)),
            false);
    } else {
      static auto op = registered<Tensor(const Tensor&, const Tensor&, int64_t, double, int64_t)>(
          "sihc::embedding_lookup_backward");
      out = op.call(grad, ids, rows, scale, padding);
    }
    return {out, Tensor(), Tensor(), Tensor()};
  }
};

int64_t pixels_of(const Tensor& x) { return x.numel() / (x.size(0) * x.size(-1)); }
int act_code(const std::string& act) { return act == "silu" ? SIHC_ACT_SILU : SIHC_ACT_NONE; }
variable_list run_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, double eps,
                       const std::string& act) {
  const c10::DeviceGuard guard(x.device());
  const int64_t b = x.size(0), n = pixels_of(x);
  const int c = int(x.size(-1)), g = int(groups);
  Tensor y = at::empty_like(x), stats = at::empty({b, groups, 2}, x.options().dtype(at::kFloat)), ws;
  const size_t bytes = sihc_group_norm_workspace_size(b, n, c, g, dtype_code(x));
  if (bytes) ws = workspace(bytes, x);
  check(sihc_group_norm(x.const_data_ptr(), weight.const_data_ptr(), bias.const_data_ptr(), y.data_ptr(),
                        stats.data_ptr<float>(), b, n, c, g, float(eps), act_code(act), dtype_code(x),
                        dtype_code(weight), bytes ? ws.data_ptr() : nullptr, bytes, stream_of(x)),
        true);
  return {y, stats};
}
// What a backward needs beside the result leaves by a pointer: an output marked as not differentiable ends
// compiled autograd, which takes no such node.
struct NormFn : torch::autograd::Function<NormFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias,
                        int64_t groups, double eps, const std::string& act, Tensor* stats) {
    variable_list out = run_norm(x, weight, bias, groups, eps, act);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, bias, out[1]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    *stats = out[1];
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    if (!grads[0].defined()) return variable_list(7);
    const Tensor grad = grads[0].contiguous();
    const int64_t groups = ctx->saved_data["groups"].toInt();
    const std::string act = ctx->saved_data["act"].toStringRef();
    Tensor dx, dw, db;
    if (direct() && norm_fits(x, weight, bias, groups) && same(grad, x) &&
        stats_fits(stats, {x.size(0), groups, 2}, x)) {
      RECORD_FUNCTION("sihc::group_norm_act_backward", (Args{grad, x, weight, bias, stats, groups, act}));
      const c10::DeviceGuard device(x.device());
      const int64_t b = x.size(0), n = pixels_of(x);
      const int c = int(x.size(-1)), g = int(groups);
      dx = at::empty_like(x);
      dw = at::empty_like(weight);
      db = at::empty_like(bias);
      const Tensor ws = workspace(sihc_group_norm_backward_workspace_size(b, n, c, g, dtype_code(x)), x);
      check(sihc_group_norm_backward(grad.const_data_ptr(), x.const_data_ptr(), weight.const_data_ptr(),
                                     bias.const_data_ptr(), stats.const_data_ptr<float>(), dx.data_ptr(),
                                     dw.data_ptr(), db.data_ptr(), b, n, c, g, act_code(act), dtype_code(x),
                                     dtype_code(weight), ws.data_ptr(), size_t(ws.numel()) * 4, stream_of(x)),
            false);
    } else {
      static auto op = registered<std::tuple<Tensor, Tensor, Tensor>(
          const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, c10::string_view)>(
          "sihc::group_norm_act_backward");
      std::tie(dx, dw, db) = op.call(grad, x, weight, bias, stats, groups, act);
    }
    return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

sihc_attention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, double scale) {
  sihc_attention a{};
  a.batch = q.size(0);
  a.queries = int(q.size(1));
  a.keys = int(k.size(1));
  a.heads = int(q.size(2));
  a.kv_heads = int(k.size(2));
  a.dim = int(q.size(3));
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q.stride(i);
    a.k_stride[i] = k.stride(i);
    a.v_stride[i] = v.stride(i);
  }
  a.scale = float(scale);
  a.dtype = dtype_code(q);
  return a;
}
// (out, statistics, what out lost in rounding): the latter two empty unless `train`
variable_list run_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, double scale,
                            bool train) {
  const c10::DeviceGuard guard(q.device());
  const sihc_attention a = attention_of(q, k, v, scale);
  const bool rounded = train && q.scalar_type() == at::kBFloat16;
  Tensor out = at::empty(q.sizes(), q.options()), ws;
  Tensor stats = train ? at::empty({q.size(0), q.size(2), q.size(1), 2}, q.options().dtype(at::kFloat))
                       : at::empty({0}, q.options().dtype(at::kFloat));
  Tensor low = rounded ? at::empty(q.sizes(), q.options()) : at::empty({0}, q.options());
  const size_t bytes = sihc_cross_attention_workspace_size(&a);
  if (bytes) ws = workspace(bytes, q);
  check(sihc_cross_attention(&a, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), index_ptr(lengths),
                             out.data_ptr(), train ? stats.data_ptr<float>() : nullptr,
                             rounded ? low.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        true);
  return {out, stats, low};
}
struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static constexpr bool is_traceable = true;
  // rest: the statistics, what the result lost in rounding (NormFn's pointer)
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const std::optional<Tensor>& lengths, double scale, variable_list* rest) {
    const Tensor n = lengths.value_or(Tensor());
    variable_list out = run_attention(q, k, v, n, scale, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, n, out[0], out[1], out[2]});
    ctx->saved_data["scale"] = scale;
    *rest = {out[1], out[2]};
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &n = saved[3], &out = saved[4], &stats = saved[5],
                 &low = saved[6];
    if (!grads[0].defined()) return variable_list(6);
    const Tensor grad = grads[0].contiguous();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor dq, dk, dv;
    if (direct() && attention_fits(q, k, v, n) && same(grad, out) && grad.sizes().equals(q.sizes()) &&
        grad.scalar_type() == q.scalar_type() && grad.device() == q.device() &&
        (q.scalar_type() == at::kFloat || same(low, out)) &&
        stats_fits(stats, {q.size(0), q.size(2), q.size(1), 2}, q)) {
      RECORD_FUNCTION("sihc::cross_attention_backward", (Args{grad, q, k, v, maybe(n), out, stats, low, scale}));
      const c10::DeviceGuard device(q.device());
      const sihc_attention a = attention_of(q, k, v, scale);
      dq = at::empty(q.sizes(), q.options());
      dk = at::empty(k.sizes(), k.options());
      dv = at::empty(v.sizes(), v.options());
      const Tensor ws = workspace(sihc_cross_attention_backward_workspace_size(&a), q);
      check(sihc_cross_attention_backward(&a, grad.const_data_ptr(), q.const_data_ptr(), k.const_data_ptr(),
                                          v.const_data_ptr(), index_ptr(n), out.const_data_ptr(),
                                          stats.const_data_ptr<float>(),
                                          q.scalar_type() == at::kFloat ? nullptr : low.const_data_ptr(),
                                          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(),
                                          size_t(ws.numel()) * 4, stream_of(q)),
            false);
    } else {
      static auto op = registered<std::tuple<Tensor, Tensor, Tensor>(
          const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, const Tensor&,
          const Tensor&, const Tensor&, double)>("sihc::cross_attention_backward");
      std::tie(dq, dk, dv) = op.call(grad, q, k, v, maybe(n), out, stats, low, scale);
    }
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------- body operators
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const char* act_name(int act) {
  return act == SIHC_ACT_SWIGLU ? "swiglu" : act == SIHC_ACT_SILU ? "silu" : "none";
}
sihc_linear linear_of(const Tensor& x, const Tensor& weight, const Tensor& gate, int act) {
  sihc_linear l{};
  l.rows = x.numel() / x.size(-1);
  l.inner = int(x.size(-1));
  l.outer = int(act == SIHC_ACT_SWIGLU ? weight.size(0) / 2 : weight.size(0));
  l.act = act;
  l.dtype = dtype_code(x);
  l.rows_per_gate = gate.defined() ? l.rows / x.size(0) : l.rows;
  l.gate_stride = gate.defined() ? gate.stride(0) : 0;
  return l;
}
bool keeps(const Tensor& gate, int act) { return act != SIHC_ACT_NONE || gate.defined(); }
bool keeps_low(const Tensor& x, int act) { return act != SIHC_ACT_NONE && x.scalar_type() == at::kBFloat16; }
std::vector<int64_t> low_sizes(const Tensor& x, int64_t outer, int act) {
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end() - 1);
  sizes.push_back(act == SIHC_ACT_SWIGLU ? 2 : 1);
  sizes.push_back((outer + 7) / 8);
  return sizes;
}
uint32_t* words(const Tensor& t) { return static_cast<uint32_t*>(t.data_ptr()); }
// (result, h and more bits of it for the backward: undefined unless `train`, empty where it needs none)
variable_list run_linear(const Tensor& x, const Tensor& weight, const Tensor& bias, int act, const Tensor& gate,
                         const Tensor& residual, bool train) {
  const c10::DeviceGuard guard(x.device());
  const sihc_linear l = linear_of(x, weight, gate, act);
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = l.outer;
  Tensor y = at::empty(sizes, x.options()), ws;
  sizes.back() = weight.size(0);
  const bool h_kept = train && keeps(gate, act), low_kept = train && keeps_low(x, act);
  Tensor h, low;
  if (train) {
    const std::vector<int64_t> none{0};
    h = at::empty(h_kept ? sizes : none, x.options());
    low = at::empty(low_kept ? low_sizes(x, l.outer, act) : none, x.options().dtype(at::kInt));
  }
  const size_t bytes = sihc_linear_act_workspace_size(&l);
  if (bytes) ws = workspace(bytes, x);
  check(sihc_linear_act(&l, x.const_data_ptr(), weight.const_data_ptr(), ptr(bias), ptr(gate), ptr(residual),
                        y.data_ptr(), h_kept ? h.data_ptr() : nullptr, low_kept ? words(low) : nullptr,
                        bytes ? ws.data_ptr() : nullptr, bytes, stream_of(x)),
        true);
  return {y, h, low};
}
struct LinearFn : torch::autograd::Function<LinearFn> {
  static constexpr bool is_traceable = true;
  // rest: h and more bits of it (NormFn's pointer)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                        int64_t act, const std::optional<Tensor>& gate, const std::optional<Tensor>& residual,
                        variable_list* rest) {
    const Tensor g = gate.value_or(Tensor());
    variable_list out = run_linear(x, weight, bias.value_or(Tensor()), int(act), g, residual.value_or(Tensor()), true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, g, out[1], out[2]});
    ctx->saved_data["act"] = act;
    ctx->saved_data["given"] = int64_t(bias.has_value()) + 2 * int64_t(residual.has_value());
    *rest = {out[1], out[2]};
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &gate = saved[2], &h = saved[3], &low = saved[4];
    if (!grads[0].defined()) return variable_list(7);
    const int act = int(ctx->saved_data["act"].toInt());
    const int64_t given = ctx->saved_data["given"].toInt();
    size_t edge = 2;  // an edge for every tensor that was given
    const bool has_bias = given & 1, has_gate = gate.defined(), has_residual = given & 2;
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_b = has_bias && ctx->needs_input_grad(edge);
    edge += has_bias;
    const bool want_g = has_gate && ctx->needs_input_grad(edge);
    edge += has_gate;
    variable_list out(7);
    if (has_residual && ctx->needs_input_grad(edge)) out[5] = grads[0];
    if (!(want_x || want_w || want_b || want_g)) return out;
    const Tensor grad = grads[0].contiguous();
    Tensor dx, dw, db, dg;
    bool fits = direct() && linear_fits(x, weight, Tensor(), gate, Tensor(), act) && plain(grad) &&
                grad.scalar_type() == x.scalar_type() && grad.device() == x.device();
    if (fits) {
      std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
      sizes.back() = weight.size(0);
      fits = (!keeps(gate, act) || (plain(h) && h.sizes().equals(sizes) && h.scalar_type() == x.scalar_type() &&
                                    h.device() == x.device())) &&
             (!keeps_low(x, act) || (plain(low) && low.scalar_type() == at::kInt && low.device() == x.device() &&
                                     low.sizes().equals(low_sizes(x, linear_of(x, weight, gate, act).outer, act))));
      if (act == SIHC_ACT_SWIGLU) sizes.back() /= 2;
      fits = fits && grad.sizes().equals(sizes);
    }
    if (fits) {
      RECORD_FUNCTION("sihc::linear_act_backward", (Args{grad, x, weight, h, low, maybe(gate), act_name(act)}));
      const c10::DeviceGuard device(x.device());
      const sihc_linear l = linear_of(x, weight, gate, act);
      if (want_x) dx = at::empty_like(x);
      if (want_w) dw = at::empty_like(weight);
      if (want_b) db = at::empty({weight.size(0)}, weight.options());
      if (want_g) dg = at::empty({x.size(0), l.outer}, x.options());
      const Tensor ws = workspace(sihc_linear_act_backward_workspace_size(&l, has_gate), x);
      auto out_ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      check(sihc_linear_act_backward(&l, grad.const_data_ptr(), x.const_data_ptr(), weight.const_data_ptr(),
                                     keeps(gate, act) ? h.const_data_ptr() : nullptr,
                                     keeps_low(x, act) ? words(low) : nullptr, ptr(gate),
                                     out_ptr(dx), out_ptr(dw), out_ptr(db), out_ptr(dg), ws.data_ptr(),
                                     size_t(ws.numel()) * 4, stream_of(x)),
            false);
    } else {
      refuse_tangents("linear_act backward", {grad});
      static auto op = registered<std::tuple<Tensor, Tensor, Tensor, Tensor>(
          const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&,
          c10::string_view, bool, bool, bool, bool)>("sihc::linear_act_backward");
      std::tie(dx, dw, db, dg) =
          op.call(grad, x, weight, h, low, maybe(gate), act_name(act), want_x, want_w, want_b, want_g);
    }
    if (want_x) out[0] = dx;
    if (want_w) out[1] = dw;
    if (want_b) out[2] = db;
    if (want_g) out[4] = dg;
    return out;
  }
};

using Axes = std::vector<int64_t>;
sihc_heads heads_of(const Tensor& q, const Tensor& k, const Tensor& weight, const Tensor& positions, const Axes& axes,
                    double theta, double eps, bool inverse) {
  sihc_heads h{};
  h.batch = q.size(0);
  h.tokens = q.size(1);
  h.heads = int(q.size(2));
  h.kv_heads = k.defined() ? int(k.size(2)) : 0;
  h.dim = int(q.size(3));
  h.axes = int(axes.size());
  for (size_t i = 0; i < axes.size(); ++i) h.widths[i] = int(axes[i]);
  for (int i = 0; i < 3; ++i) {
    h.q_stride[i] = q.stride(i);
    h.k_stride[i] = k.defined() ? k.stride(i) : 0;
  }
  h.position_batch_stride = positions.dim() == 3 ? q.size(1) : 0;
  h.theta = theta;
  h.eps = float(eps);
  h.dtype = dtype_code(q);
  h.w_dtype = weight.defined() ? dtype_code(weight) : h.dtype;
  h.position_dtype = positions.scalar_type() == at::kFloat ? SIHC_POSITION_F32 : SIHC_POSITION_I32;
  h.inverse = inverse;
  return h;
}
variable_list run_qk(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& positions,
                     const Axes& axes, double theta, double eps) {
  const c10::DeviceGuard guard(q.device());
  const sihc_heads h = heads_of(q, k, qw, positions, axes, theta, eps, false);
  Tensor oq = at::empty(q.sizes(), q.options()), ok = at::empty(k.sizes(), k.options());
  check(sihc_qk_norm_rotary(&h, q.const_data_ptr(), k.const_data_ptr(), qw.const_data_ptr(), kw.const_data_ptr(),
                            positions.const_data_ptr(), oq.data_ptr(), ok.data_ptr(), stream_of(q)),
        true);
  return {oq, ok};
}
struct QkFn : torch::autograd::Function<QkFn> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& qw,
                               const Tensor& kw, const Tensor& positions, const Axes& axes, double theta, double eps) {
    ctx->save_for_backward({q, k, qw, kw, positions});
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["theta"] = theta;
    ctx->saved_data["eps"] = eps;
    return run_qk(q, k, qw, kw, positions, axes, theta, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &qw = saved[2], &kw = saved[3], &positions = saved[4];
    const Axes axes = ctx->saved_data["axes"].toIntVector();
    const double theta = ctx->saved_data["theta"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    const Tensor gq = grads[0].contiguous(), gk = grads[1].contiguous();
    auto fits = [](const Tensor& g, const Tensor& x) {
      return plain(g) && g.sizes().equals(x.sizes()) && g.scalar_type() == x.scalar_type() && g.device() == x.device();
    };
    Tensor dq, dk, dqw, dkw;
    if (direct() && qk_fits(q, k, qw, kw, positions, axes, theta, eps) && fits(gq, q) && fits(gk, k)) {
      RECORD_FUNCTION("sihc::qk_norm_rotary_backward", (Args{gq, gk, q, k, qw, kw, positions, axes, theta, eps}));
      const c10::DeviceGuard device(q.device());
      const sihc_heads h = heads_of(q, k, qw, positions, axes, theta, eps, false);
      dq = at::empty(q.sizes(), q.options());
      dk = at::empty(k.sizes(), k.options());
      dqw = at::empty_like(qw);
      dkw = at::empty_like(kw);
      const Tensor ws = workspace(sihc_qk_norm_rotary_backward_workspace_size(&h), q);
      check(sihc_qk_norm_rotary_backward(&h, gq.const_data_ptr(), gk.const_data_ptr(), q.const_data_ptr(),
                                         k.const_data_ptr(), qw.const_data_ptr(), kw.const_data_ptr(),
                                         positions.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(),
                                         dkw.data_ptr(), ws.data_ptr(), size_t(ws.numel()) * 4, stream_of(q)),
            false);
    } else {
      refuse_tangents("qk_norm_rotary backward", {gq, gk});
      static auto op = registered<std::tuple<Tensor, Tensor, Tensor, Tensor>(
          const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
          at::IntArrayRef, double, double)>("sihc::qk_norm_rotary_backward");
      std::tie(dq, dk, dqw, dkw) = op.call(gq, gk, q, k, qw, kw, positions, axes, theta, eps);
    }
    return {dq, dk, dqw, dkw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor run_rotary(const Tensor& x, const Tensor& positions, const Axes& axes, double theta, bool inverse,
                  bool forward) {
  const c10::DeviceGuard guard(x.device());
  const sihc_heads h = heads_of(x, Tensor(), Tensor(), positions, axes, theta, 0.0, inverse);
  Tensor y = at::empty(x.sizes(), x.options());
  check(sihc_qk_norm_rotary(&h, x.const_data_ptr(), nullptr, nullptr, nullptr, positions.const_data_ptr(),
                            y.data_ptr(), nullptr, stream_of(x)),
        forward);
  return y;
}
struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Axes& axes, double theta,
                        bool inverse) {
    ctx->save_for_backward({positions});
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["theta"] = theta;
    ctx->saved_data["inverse"] = inverse;
    return run_rotary(x, positions, axes, theta, inverse, true);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor positions = ctx->get_saved_variables()[0], grad = grads[0].contiguous();
    const Axes axes = ctx->saved_data["axes"].toIntVector();
    const double theta = ctx->saved_data["theta"].toDouble();
    const bool inverse = !ctx->saved_data["inverse"].toBool();
    Tensor dx;
    if (direct() && heads_fit(grad, Tensor(), positions, axes, theta)) {
      RECORD_FUNCTION("sihc::axis_rotary", (Args{grad, positions, axes, theta, inverse}));
      dx = run_rotary(grad, positions, axes, theta, inverse, false);
    } else {
      refuse_tangents("axis_rotary backward", {grad});
      static auto op = registered<Tensor(const Tensor&, const Tensor&, at::IntArrayRef, double, bool)>(
          "sihc::axis_rotary");
      dx = op.call(grad, positions, axes, theta, inverse);
    }
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor run_dropout(const Tensor& x, double p, const Tensor& seed, int64_t stream, const Tensor& residual,
                   bool forward) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty_like(x);
  check(sihc_dropout(x.const_data_ptr(), ptr(residual), y.data_ptr(), x.numel(), p, seed.const_data_ptr<int64_t>(),
                     stream, dtype_code(x), stream_of(x)),
        forward);
  return y;
}
struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, const Tensor& seed, int64_t stream,
                        const std::optional<Tensor>& residual) {
    ctx->save_for_backward({seed});
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["added"] = residual.has_value();
    return run_dropout(x, p, seed, stream, residual.value_or(Tensor()), true);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor seed = ctx->get_saved_variables()[0];
    const double p = ctx->saved_data["p"].toDouble();
    const int64_t stream = ctx->saved_data["stream"].toInt();
    variable_list out(5);
    // (edges: x, the seed, the residual)
    if (ctx->saved_data["added"].toBool() && ctx->needs_input_grad(2)) out[4] = grads[0];
    if (!ctx->needs_input_grad(0)) return out;
    const Tensor grad = grads[0].contiguous();
    if (direct() && dropout_fits(grad, p, seed, stream, Tensor())) {
      RECORD_FUNCTION("sihc::dropout", (Args{grad, p, seed, stream}));
      out[0] = run_dropout(grad, p, seed, stream, Tensor(), false);
    } else {
      refuse_tangents("dropout backward", {grad});
      static auto op = registered<Tensor(const Tensor&, double, const Tensor&, int64_t, const std::optional<Tensor>&)>(
          "sihc::dropout");
      out[0] = op.call(grad, p, seed, stream, std::nullopt);
    }
    return out;
  }
};

// ------------------------------------------------------------------------ Python entries
PyObject* to_list(const variable_list& ts) {
  PyObject* out = PyList_New(Py_ssize_t(ts.size()));
  for (size_t i = 0; out && i < ts.size(); ++i) PyList_SET_ITEM(out, Py_ssize_t(i), THPVariable_Wrap(ts[i]));
  return out;
}
PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

// One Python entry: the op that it stands for.
struct Entry {
  c10::OperatorHandle op;
  const char* name() const { return op.operator_name().name.c_str(); }
  // A custom op has kernels under alias keys only: one under these is the program's own.
  bool overridden() const {
    return op.hasKernelForDispatchKey(c10::DispatchKey::CUDA) ||
           op.hasKernelForDispatchKey(c10::DispatchKey::AutogradCUDA) ||
           op.hasKernelForDispatchKey(c10::DispatchKey::AutocastCUDA);
  }
};
constexpr const char* ENTRY = "sihc_entry";
const Entry& entry_of(PyObject* self) { return *static_cast<Entry*>(PyCapsule_GetPointer(self, ENTRY)); }

// Run `f`; a C-ABI error, or a C++ exception, hands the call to the Python op, which repeats
// the checks and raises what it always raised. A Python exception comes from the caller's own
// code (a saved-tensor hook) and goes on to the caller: checkpointing ends its recomputation
// by raising from such a hook, which must not run again for the same call.
template <typename F>
PyObject* guarded(PyObject* self, F&& f) {
  try {
    const Entry& entry = entry_of(self);
    if (!plain_mode() || entry.overridden()) return not_implemented();
    return f();
  } catch (const Failure&) {
    return not_implemented();
  } catch (python_error& e) {
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    PyErr_Clear();
    return not_implemented();
  }
}
// f() as a call of the op of `self`, with the GIL released: a launch waits where the queue is full,
// and an allocation may wait for the device. (The registered ops release it around every dispatch
// and launch.) Saved-tensor hooks take it again for their own calls.
template <typename A, typename F>
auto call(PyObject* self, A&& args, F&& f) {
  RECORD_FUNCTION(entry_of(self).name(), args());
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}
// Below autograd (a custom op's own body, inference mode) and under no_grad nothing is recorded.
bool unrecorded() { return !at::GradMode::is_enabled() || below_autograd(); }

PyObject* read_impl(PyObject* self, PyObject* const* args, bool indexed) {
  return guarded(self, [&]() -> PyObject* {
    Tensor x, alpha, index;
    Shape s{};
    if (!unwrap(args[0], x) || !unwrap(args[1], alpha) || (indexed && !unwrap(args[2], index))) return not_implemented();
    if ((indexed && !index.defined()) || !read_fits(x, alpha, index, s)) return not_implemented();
    return to_list(call(
        self, [&] { return index.defined() ? Args{x, alpha, index} : Args{x, alpha}; },
        [&] { return unrecorded() ? run_read(x, alpha, index) : ReadFn::apply(x, alpha, maybe(index)); }));
  });
}
PyObject* write_impl(PyObject* self, PyObject* const* args, bool indexed) {
  return guarded(self, [&]() -> PyObject* {
    Tensor x, beta, index;
    std::vector<Tensor> updates;
    Shape s{};
    if (!unwrap(args[0], x) || !unwrap_list(args[1], updates) || !unwrap(args[2], beta) ||
        (indexed && !unwrap(args[3], index)))
      return not_implemented();
    if ((indexed && !index.defined()) || !write_fits(x, updates, beta, index, s)) return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return listed(x, updates, beta, index); }, [&] {
      return unrecorded() ? run_write(x, updates, beta, index)
                          : WriteFn::apply(x, TensorList(updates), beta, maybe(index));
    }));
  });
}

PyObject* py_read(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  return n == 2 ? read_impl(self, args, false) : not_implemented();
}
PyObject* py_indexed_read(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  return n == 3 ? read_impl(self, args, true) : not_implemented();
}
PyObject* py_write(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  return n == 3 ? write_impl(self, args, false) : not_implemented();
}
PyObject* py_indexed_write(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  return n == 4 ? write_impl(self, args, true) : not_implemented();
}
PyObject* py_triangular(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor base, gamma;
    std::vector<Tensor> updates;
    if (!unwrap(args[0], base) || !unwrap_list(args[1], updates) || !unwrap(args[2], gamma)) return not_implemented();
    if (!triangular_fits(base, updates, gamma)) return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return listed(base, updates, gamma, Tensor()); }, [&] {
      return unrecorded() ? run_triangular(base, updates, gamma)
                          : TriangularFn::apply(base, TensorList(updates), gamma);
    }));
  });
}
PyObject* py_event(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor x, dz, beta, alpha;
    if (!unwrap(args[0], x) || !unwrap(args[1], dz) || !unwrap(args[2], beta) || !unwrap(args[3], alpha))
      return not_implemented();
    if (!event_fits(x, dz, beta, alpha)) return not_implemented();
    const variable_list out = call(
        self, [&] { return Args{x, dz, beta, alpha}; },
        [&] { return unrecorded() ? run_event(x, dz, beta, alpha) : EventFn::apply(x, dz, beta, alpha); });
    PyObject* pair = PyTuple_New(2);
    for (int i = 0; pair && i < 2; ++i) PyTuple_SET_ITEM(pair, i, THPVariable_Wrap(out[size_t(i)]));
    return pair;
  });
}

// (carrier edge, blocks, slots, x0, dz_0.., beta_0..)
PyObject* py_block_write(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n < 4) return not_implemented();
  const long edge = PyLong_AsLong(args[0]), blocks = PyLong_AsLong(args[1]), slots = PyLong_AsLong(args[2]);
  if (n != 4 + 2 * blocks) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor x;
    std::vector<Tensor> updates(static_cast<size_t>(blocks)), betas(static_cast<size_t>(blocks));
    if (!unwrap(args[3], x)) return not_implemented();
    for (long i = 0; i < blocks; ++i)
      if (!unwrap(args[4 + i], updates[size_t(i)]) || !unwrap(args[4 + blocks + i], betas[size_t(i)]))
        return not_implemented();
    if (!BlockWriteFn::fits(x, updates, betas) || x.size(1) != edge || betas[0].size(1) != slots)
      return not_implemented();
    auto listing = [&] {
      Args all{x};
      for (const auto* ts : {&updates, &betas})
        for (const Tensor& t : *ts) all.emplace_back(t);
      return all;
    };
    return THPVariable_Wrap(call(self, listing, [&] {
      return unrecorded() ? run_write(x, updates, at::stack(betas), Tensor())
                          : BlockWriteFn::apply(x, TensorList(updates), TensorList(betas),
                                                std::string(entry_of(self).name()));
    }));
  });
}
PyObject* py_gather(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 3 || !PyLong_CheckExact(args[2])) return not_implemented();
  const long slots = PyLong_AsLong(args[2]);
  return guarded(self, [&]() -> PyObject* {
    Tensor x, index;
    if (!unwrap(args[0], x) || !unwrap(args[1], index) || !gather_fits(x, index, slots)) return not_implemented();
    return THPVariable_Wrap(call(
        self, [&] { return Args{x, index, int64_t(slots)}; },
        [&] { return unrecorded() ? run_gather(x, index, slots) : GatherFn::apply(x, index, int64_t(slots)); }));
  });
}
PyObject* py_scatter(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor cells, index;
    if (!unwrap(args[0], cells) || !unwrap(args[1], index) || !scatter_fits(cells, index)) return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return Args{cells, index}; }, [&] {
      return unrecorded() ? run_scatter(sihc_scatter_cells, cells, index, true) : ScatterFn::apply(cells, index);
    }));
  });
}

bool unwrap_number(PyObject* o, double& v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  v = PyFloat_AsDouble(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
bool unwrap_integer(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
PyObject* tuple_of(const variable_list& ts) {
  PyObject* tuple = PyTuple_New(Py_ssize_t(ts.size()));
  for (size_t i = 0; tuple && i < ts.size(); ++i) PyTuple_SET_ITEM(tuple, Py_ssize_t(i), THPVariable_Wrap(ts[i]));
  return tuple;
}
PyObject* py_embed(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor table, ids;
    double scale;
    int64_t padding;
    if (!unwrap(args[0], table) || !unwrap(args[1], ids) || !unwrap_number(args[2], scale) ||
        !unwrap_integer(args[3], padding) || !embed_fits(table, ids))
      return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return Args{table, ids, scale, padding}; }, [&] {
      return unrecorded() ? run_embed(table, ids, scale) : EmbedFn::apply(table, ids, scale, padding);
    }));
  });
}
PyObject* py_norm(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 || !PyUnicode_CheckExact(args[5])) return not_implemented();
  const bool silu = PyUnicode_CompareWithASCIIString(args[5], "silu") == 0;
  if (!silu && PyUnicode_CompareWithASCIIString(args[5], "none") != 0) return not_implemented();
  const std::string act = silu ? "silu" : "none";
  return guarded(self, [&]() -> PyObject* {
    Tensor x, weight, bias;
    int64_t groups;
    double eps;
    if (!unwrap(args[0], x) || !unwrap(args[1], weight) || !unwrap(args[2], bias) ||
        !unwrap_integer(args[3], groups) || !unwrap_number(args[4], eps) || !norm_fits(x, weight, bias, groups))
      return not_implemented();
    return tuple_of(call(self, [&] { return Args{x, weight, bias, groups, eps, act}; }, [&] {
      if (unrecorded()) return run_norm(x, weight, bias, groups, eps, act);
      Tensor stats;
      const Tensor out = NormFn::apply(x, weight, bias, groups, eps, act, &stats);
      return variable_list{out, stats};
    }));
  });
}
PyObject* py_attention(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 || !PyBool_Check(args[5])) return not_implemented();
  const bool train = args[5] == Py_True;
  return guarded(self, [&]() -> PyObject* {
    Tensor q, k, v, lengths;
    double scale;
    if (!unwrap(args[0], q) || !unwrap(args[1], k) || !unwrap(args[2], v) ||
        (args[3] != Py_None && !unwrap(args[3], lengths)) || !unwrap_number(args[4], scale) ||
        !attention_fits(q, k, v, lengths))
      return not_implemented();
    return tuple_of(call(self, [&] { return Args{q, k, v, maybe(lengths), scale, train}; }, [&] {
      if (unrecorded() || !train) return run_attention(q, k, v, lengths, scale, train);
      variable_list rest;
      const Tensor out = AttentionFn::apply(q, k, v, maybe(lengths), scale, &rest);
      return variable_list{out, rest[0], rest[1]};
    }));
  });
}

bool unwrap_maybe(PyObject* o, Tensor& t) { return o == Py_None || unwrap(o, t); }
bool unwrap_axes(PyObject* o, Axes& axes) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  axes.resize(size_t(n));
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!unwrap_integer(PySequence_Fast_GET_ITEM(o, i), axes[size_t(i)])) return false;
  return true;
}
template <bool KEEPS>  // what the backward needs, with an autograd node; else the result alone
PyObject* py_linear(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 || !PyUnicode_CheckExact(args[3])) return not_implemented();
  int act = -1;
  for (const int a : {int(SIHC_ACT_NONE), int(SIHC_ACT_SILU), int(SIHC_ACT_SWIGLU)})
    if (PyUnicode_CompareWithASCIIString(args[3], act_name(a)) == 0) act = a;
  if (act < 0) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor x, weight, bias, gate, residual;
    if (!unwrap(args[0], x) || !unwrap(args[1], weight) || !unwrap_maybe(args[2], bias) ||
        !unwrap_maybe(args[4], gate) || !unwrap_maybe(args[5], residual) ||
        !linear_fits(x, weight, bias, gate, residual, act))
      return not_implemented();
    if (!KEEPS && !unrecorded())  // (an op without a rule: autograd says so)
      for (const Tensor* t : {&x, &weight, &bias, &gate, &residual})
        if (t->defined() && t->requires_grad()) return not_implemented();
    auto listing = [&] { return Args{x, weight, maybe(bias), act_name(act), maybe(gate), maybe(residual)}; };
    const variable_list out = call(self, listing, [&] {
      if (!KEEPS || unrecorded()) return run_linear(x, weight, bias, act, gate, residual, KEEPS);
      variable_list rest;
      const Tensor y = LinearFn::apply(x, weight, maybe(bias), int64_t(act), maybe(gate), maybe(residual), &rest);
      return variable_list{y, rest[0], rest[1]};
    });
    return KEEPS ? tuple_of(out) : THPVariable_Wrap(out[0]);
  });
}
PyObject* py_qk(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor q, k, qw, kw, positions;
    Axes axes;
    double theta, eps;
    if (!unwrap(args[0], q) || !unwrap(args[1], k) || !unwrap(args[2], qw) || !unwrap(args[3], kw) ||
        !unwrap(args[4], positions) || !unwrap_axes(args[5], axes) || !unwrap_number(args[6], theta) ||
        !unwrap_number(args[7], eps) || !qk_fits(q, k, qw, kw, positions, axes, theta, eps))
      return not_implemented();
    return tuple_of(call(self, [&] { return Args{q, k, qw, kw, positions, axes, theta, eps}; }, [&] {
      return unrecorded() ? run_qk(q, k, qw, kw, positions, axes, theta, eps)
                          : QkFn::apply(q, k, qw, kw, positions, axes, theta, eps);
    }));
  });
}
PyObject* py_rotary(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 5 || !PyBool_Check(args[4])) return not_implemented();
  const bool inverse = args[4] == Py_True;
  return guarded(self, [&]() -> PyObject* {
    Tensor x, positions;
    Axes axes;
    double theta;
    if (!unwrap(args[0], x) || !unwrap(args[1], positions) || !unwrap_axes(args[2], axes) ||
        !unwrap_number(args[3], theta) || !heads_fit(x, Tensor(), positions, axes, theta))
      return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return Args{x, positions, axes, theta, inverse}; }, [&] {
      return unrecorded() ? run_rotary(x, positions, axes, theta, inverse, true)
                          : RotaryFn::apply(x, positions, axes, theta, inverse);
    }));
  });
}
PyObject* py_dropout(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) return not_implemented();
  return guarded(self, [&]() -> PyObject* {
    Tensor x, seed, residual;
    double p;
    int64_t stream;
    if (!unwrap(args[0], x) || !unwrap_number(args[1], p) || !unwrap(args[2], seed) ||
        !unwrap_integer(args[3], stream) || !unwrap_maybe(args[4], residual) ||
        !dropout_fits(x, p, seed, stream, residual))
      return not_implemented();
    return THPVariable_Wrap(call(self, [&] { return Args{x, p, seed, stream, maybe(residual)}; }, [&] {
      return unrecorded() ? run_dropout(x, p, seed, stream, residual, true)
                          : DropoutFn::apply(x, p, seed, stream, maybe(residual));
    }));
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef define(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef entries[] = {
    define<py_read>("sublayer_read"),        define<py_write>("sublayer_write"),
    define<py_triangular>("sublayer_triangular"), define<py_event>("event_write_read"),
    define<py_indexed_read>("indexed_read"), define<py_indexed_write>("indexed_write"),
    define<py_block_write>("block_write"),   define<py_gather>("gather_cells"),
    define<py_scatter>("scatter_cells"),     define<py_embed>("embedding_lookup"),
    define<py_norm>("group_norm_act"),       define<py_attention>("cross_attention"),
    define<py_linear<true>>("linear_act"),   define<py_linear<false>>("linear_act_result"),
    define<py_qk>("qk_norm_rotary"),
    define<py_rotary>("axis_rotary"),        define<py_dropout>("dropout"),
};
// entry(name, op): the native entry `name` for the registered op `op` ("namespace::name")
PyObject* py_entry(PyObject*, PyObject* args) {
  const char *name, *op;
  if (!PyArg_ParseTuple(args, "ss", &name, &op)) return nullptr;
  for (PyMethodDef& def : entries) {
    if (std::strcmp(def.ml_name, name) != 0) continue;
    const auto handle = c10::Dispatcher::singleton().findSchema({op, ""});
    if (!handle) return PyErr_Format(PyExc_ValueError, "no registered op %s", op);
    PyObject* self = PyCapsule_New(new Entry{*handle}, ENTRY, [](PyObject* capsule) {
      delete static_cast<Entry*>(PyCapsule_GetPointer(capsule, ENTRY));
    });
    if (!self) return nullptr;
    PyObject* function = PyCFunction_New(&def, self);
    Py_DECREF(self);
    return function;
  }
  return PyErr_Format(PyExc_AttributeError, "no native entry %s", name);
}
// has_tangent(t): whether a tensor is a dual one, read without a dispatch, so that transforms do not answer for it
PyObject* py_has_tangent(PyObject*, PyObject* o) {
  if (THPVariable_Check(o) && THPVariable_Unpack(o)._fw_grad(0).defined()) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}
PyMethodDef methods[] = {{"entry", py_entry, METH_VARARGS, nullptr},
                         {"has_tangent", py_has_tangent, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sihc_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sihc_torch(void) {
  if (sihc_abi_version() != SIHC_ABI_VERSION)
    return PyErr_Format(PyExc_ImportError, "libsihc_hip.so has ABI %d, expected %d: rebuild it", sihc_abi_version(),
                        SIHC_ABI_VERSION);
  PyObject* nn = PyImport_ImportModule("torch.nn");
  if (!nn) return nullptr;
  parameter_type = PyObject_GetAttrString(nn, "Parameter");
  Py_DECREF(nn);
  if (!parameter_type) return nullptr;
  return PyModule_Create(&module);
}
