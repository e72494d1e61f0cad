// The host side of dense.py: the differentiable calls of the bf16 products, as native autograd functions.
//
// A training step of a small layer is bound by its host: forward and backward of one linear layer (five launches) took 190 us as an
// autograd function in Python and the loss of a small head 155, of which their kernels take a fifth.  Everything that a call does per
// launch is here; what cannot be read as it lies (odd pitches, misaligned rows) and every refusal with a message of its own is dense.py's:
// a call that it has to prepare first gets None back.
#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <ATen/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>

#include <string.h>

#include "../../include/metis_nvfp4.h"

namespace {

#define METIS_DENSE_ENTRIES(X)                                                                                             \
  X(metis_last_error_string) X(metis_linear) X(metis_linear_pointwise) X(metis_linear_pointwise_workspace_bytes)          \
  X(metis_bf16_product) X(metis_bf16_product_workspace_bytes) X(metis_head_loss_keep) X(metis_head_loss_workspace_bytes) X(metis_head_sum) X(metis_head_backward_kept) \
  X(metis_head_backward_workspace_bytes)
struct Entries {
#define X(name) decltype(&::name) name = nullptr;
  METIS_DENSE_ENTRIES(X)
#undef X
} lib;

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

void check(int32_t rc, const char* what) {
  if (rc == METIS_OK) return;
  if (rc == METIS_ERR_BAD_SHAPE) TORCH_CHECK_VALUE(false, what, ": ", lib.metis_last_error_string());
  TORCH_CHECK(false, what, ": status ", rc, ": ", lib.metis_last_error_string());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor empty_like_options(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}
Tensor scratch(const Tensor& like, int64_t bytes) { return empty_like_options(like, {bytes < 16 ? 16 : bytes}, at::kByte); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// A tensor as rows of its last dimension with one pitch, if it lies so.
struct Rows {
  int64_t rows = 0, cols = 0, ld = 0;
  bool ok = false;
  Rows() = default;
  explicit Rows(const Tensor& t) {
    if (t.dim() < 1) return;
    cols = t.size(-1);
    rows = cols ? t.numel() / cols : 0;
    if (t.is_contiguous() || rows <= 1) {
      ok = t.is_contiguous() || cols <= 1 || t.stride(-1) == 1;
      ld = cols;
    } else if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= cols) {
      ok = true;
      ld = t.stride(0);
    }
  }
};
// What the TMA unit reads: 16-byte aligned rows.  A single row's pitch is not read.
bool operand(const Tensor& t, Rows& r) {
  if (!r.ok || !aligned16(t)) return false;
  if (r.rows <= 1) r.ld = (r.cols + 7) / 8 * 8;
  return r.ld % 8 == 0;
}
bool plain(const Tensor& t, const Tensor& like, at::ScalarType type) {
  return t.is_cuda() && t.scalar_type() == type && t.device() == like.device() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj();
}
// t as rows that the TMA unit reads, copied if it has to be
Tensor as_operand(const Tensor& t, Rows& r) {
  r = Rows(t);
  if (operand(t, r)) return t;
  const Tensor c = t.clone(at::MemoryFormat::Contiguous);
  r = Rows(c);
  TORCH_CHECK(operand(c, r), "rows of ", r.cols, " elements cannot be read");
  return c;
}

// A tensor that was saved is what it was, but a hook of saved tensors may have laid it out otherwise, and has to be asked whether it gave back
// the same at all: the kernels read what they are pointed at.
const Tensor& given_back(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  TORCH_CHECK(plain(t, like, type) && t.sizes() == sizes, "a saved tensor came back as ", t.toString(), " of shape ", t.sizes(), " on ", t.device());
  return t;
}

// Gradients are formed by kernels that record nothing: one that is asked for with a graph of its own raises when it is differentiated.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list leaves;
  for (const Variable& g : grads) if (g.defined()) leaves.push_back(g.detach().requires_grad_(true));
  if (leaves.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>("the bf16 products are differentiable once", (int64_t)leaves.size());
  leaves = (*error)(std::move(leaves));
  size_t i = 0;
  for (Variable& g : grads) if (g.defined()) g = leaves[i++];
  return grads;
}

// The caller's status word, for the launches of the backward pass: no saved variable, so that the caller may set it back to 0 in between.
void keep_status(AutogradContext* ctx, const Tensor& status) {
  if (status.defined()) ctx->saved_data["status"] = status;
}
Tensor kept_status(AutogradContext* ctx) {
  const auto it = ctx->saved_data.find("status");
  return it == ctx->saved_data.end() ? Tensor() : it->second.toTensor();
}

// ---- linear -------------------------------------------------------------------------------------------------------

struct LinearResult { Tensor y, act, slope; };

LinearResult linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& gate, const Tensor& residual, int64_t act, bool keep_act, bool keep_slope, const Tensor& status) {
  c10::OptionalDeviceGuard guard(x.device());
  Rows rx(x), rw(w);
  operand(x, rx);
  operand(w, rw);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = rw.rows;
  // (what the gradients need is nobody else's: rows of whole 16-byte pieces)
  const int64_t pitch = (rw.rows + 7) / 8 * 8;
  LinearResult out{empty_like_options(x, shape, at::kBFloat16), keep_act ? empty_like_options(x, {rx.rows, pitch}, at::kBFloat16) : Tensor(),
                   keep_slope ? empty_like_options(x, {rx.rows, pitch}, at::kHalf) : Tensor()};
  if (rx.rows == 0) return out;
  metis_linear_args a = {};
  a.M = rx.rows; a.N = rw.rows; a.K = rx.cols;
  a.x = x.data_ptr(); a.ldx = rx.ld;
  a.w = w.data_ptr(); a.ldw = rw.ld;
  a.bias = ptr(bias); a.bias_dtype = bias.defined() && bias.scalar_type() == at::kFloat ? METIS_DTYPE_F32 : METIS_DTYPE_BF16;
  a.activation = (int32_t)act;
  if (gate.defined()) { a.gate = gate.data_ptr(); a.ldgate = Rows(gate).ld; }
  if (residual.defined()) { a.residual = residual.data_ptr(); a.ldr = Rows(residual).ld; }
  a.y = out.y.data_ptr(); a.ldy = a.N;
  a.act = ptr(out.act); a.ldact = pitch;
  a.slope = ptr(out.slope); a.ldslope = pitch;
  a.status = ptr<int32_t>(status);
  a.stream = stream_of(x);
  check(lib.metis_linear(&a), "metis_linear");
  return out;
}

// a b, or a^T b with `mn`, for matrices of 16-byte aligned rows
Tensor product(const Tensor& a, const Rows& ra, bool mn, int32_t half, const Tensor& b, const Rows& rb, const Tensor& status) {
  const int64_t M = mn ? ra.cols : ra.rows, K = mn ? ra.rows : ra.cols;
  const Tensor d = empty_like_options(b, {M, rb.cols}, at::kBFloat16);
  const int64_t bytes = lib.metis_bf16_product_workspace_bytes(M, rb.cols, K, mn, half);
  const Tensor ws = bytes > 0 ? scratch(b, bytes) : Tensor();
  check(lib.metis_bf16_product(a.data_ptr(), mn, ra.ld, b.data_ptr(), rb.ld, M, rb.cols, K, half, d.data_ptr(), rb.cols, ptr(ws), bytes, ptr<int32_t>(status), stream_of(b)), "metis_bf16_product");
  return d;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& gate,
                        const std::optional<Tensor>& residual, int64_t act, const Tensor* status) {
    const Tensor b = bias.value_or(Tensor()), g = gate.value_or(Tensor());
    const bool through = x.requires_grad() || weight.requires_grad() || (b.defined() && b.requires_grad());
    const bool gated = g.defined() && g.requires_grad();
    const LinearResult out = linear_forward(x, weight, b, g, residual.value_or(Tensor()), act, gated, act != METIS_ACT_NONE && through, *status);
    ctx->save_for_backward({weight.requires_grad() ? x : Tensor(), x.requires_grad() ? weight : Tensor(), through ? g : Tensor(), out.act, out.slope});
    ctx->saved_data["s"] = std::vector<int64_t>{act, bias.has_value(), gate.has_value(), residual.has_value(),
                                                b.defined() && b.scalar_type() == at::kFloat, weight.size(0), weight.size(1)};
    ctx->saved_data["x"] = x.sizes().vec();
    keep_status(ctx, *status);
    return out.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> o = ctx->saved_data["s"].toIntVector(), x_shape = ctx->saved_data["x"].toIntVector();
    const int64_t act = o[0], N = o[5], K = o[6];
    // (the edges are those of the tensors that were given)
    size_t edge = 2;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = o[1] && ctx->needs_input_grad(edge);
    edge += o[1];
    const bool need_gate = o[2] && ctx->needs_input_grad(edge);
    edge += o[2];
    const bool need_residual = o[3] && ctx->needs_input_grad(edge);
    {
      at::AutoGradMode off(false);
      const Tensor dy_shaped = grads[0];
      c10::OptionalDeviceGuard guard(dy_shaped.device());
      const at::ScalarType bias_type = o[4] ? at::kFloat : at::kBFloat16;
      if (need_residual) out[4] = dy_shaped;
      Tensor dy = dy_shaped.reshape({-1, N});
      const int64_t M = dy.size(0);
      if (M == 0) {
        const auto zeros = [&](at::IntArrayRef shape, at::ScalarType type) { return at::zeros(shape, at::TensorOptions().dtype(type).device(dy.device())); };
        if (need_x) out[0] = zeros(x_shape, at::kBFloat16);
        if (need_w) out[1] = zeros({N, K}, at::kBFloat16);
        if (need_b) out[2] = zeros({N}, bias_type);
        if (need_gate) out[3] = zeros(dy_shaped.sizes(), at::kBFloat16);
      } else {
        Rows rdy(dy);
        if (!rdy.ok) {
          dy = dy.contiguous();
          rdy = Rows(dy);
        }
        const int64_t kept_pitch = (N + 7) / 8 * 8;
        Rows rx, rw, rgate, ract, rslope;
        if (saved[0].defined()) saved[0] = as_operand(given_back(saved[0], dy, at::kBFloat16, x_shape), rx);
        if (saved[1].defined()) saved[1] = as_operand(given_back(saved[1], dy, at::kBFloat16, {N, K}), rw);
        if (saved[2].defined()) {
          rgate = Rows(given_back(saved[2], dy, at::kBFloat16, dy_shaped.sizes()));
          if (!rgate.ok) rgate = Rows(saved[2] = saved[2].contiguous());
        }
        if (saved[3].defined()) saved[3] = as_operand(given_back(saved[3], dy, at::kBFloat16, {M, kept_pitch}), ract);
        if (saved[4].defined()) saved[4] = as_operand(given_back(saved[4], dy, at::kHalf, {M, kept_pitch}), rslope);
        // dz is dy itself where nothing changes it and its rows can be read as they lie
        const bool product_wanted = need_x || need_w, epilogue = act != METIS_ACT_NONE || saved[2].defined();
        Rows rdz = rdy;
        const bool write_dz = product_wanted && (epilogue || !operand(dy, rdz));
        Tensor dz = dy;
        const Tensor status = kept_status(ctx);
        const int32_t half = product_wanted && epilogue && M <= METIS_TWO_PART_ROWS ? (int32_t)(M + 7) / 8 * 8 : 0;      // (dy as it is has one part)
        if (write_dz || need_b || need_gate) {
          metis_linear_pointwise_args a = {};
          a.M = M; a.N = N;
          a.dy = dy.data_ptr(); a.lddy = rdy.ld;
          if (saved[3].defined()) { a.act = saved[3].data_ptr(); a.ldact = ract.ld; }
          if (saved[4].defined()) { a.slope = saved[4].data_ptr(); a.ldslope = rslope.ld; }
          if (saved[2].defined()) { a.gate = saved[2].data_ptr(); a.ldgate = rgate.ld; }
          if (write_dz) {
            const int64_t pitch = (N + 7) / 8 * 8;
            dz = empty_like_options(dy, {half ? 2 * half : M, pitch}, at::kBFloat16);
            a.half = half;
            rdz.rows = M; rdz.cols = N; rdz.ld = pitch;
            a.dz = dz.data_ptr(); a.lddz = pitch;
          }
          if (need_gate) {
            out[3] = empty_like_options(dy, dy_shaped.sizes(), at::kBFloat16);
            a.dgate = out[3].data_ptr(); a.lddg = N;
          }
          Tensor ws;
          if (need_b) {
            out[2] = empty_like_options(dy, {N}, bias_type);
            ws = scratch(dy, lib.metis_linear_pointwise_workspace_bytes(M, N));
            a.dbias = out[2].data_ptr(); a.dbias_dtype = o[4] ? METIS_DTYPE_F32 : METIS_DTYPE_BF16;
            a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel();
          }
          a.stream = stream_of(dy);
          check(lib.metis_linear_pointwise(&a), "metis_linear_pointwise");
        }
        if (need_x) out[0] = product(dz, rdz, false, half, saved[1], rw, status).view(x_shape);
        if (need_w) out[1] = product(dz, rdz, true, half, saved[0], rx, status);
      }
    }
    return once(std::move(out));
  }
};

// ---- head -----------------------------------------------------------------------------------------------------------

enum HeadForm { kEach, kSum, kMean, kLogprobs };

struct HeadResult { Tensor out, lse, logp, entropy, inv_count; };

metis_head_args head_args(const Tensor& h, const Tensor& w, const Tensor& target, const Tensor& lse, int64_t ignore, double scale, int64_t form, const Tensor& status) {
  Rows rh(h), rw(w);
  operand(h, rh);
  operand(w, rw);
  metis_head_args a = {};
  a.M = rh.rows; a.V = rw.rows; a.K = rh.cols;
  a.h = h.data_ptr(); a.ldh = rh.ld;
  a.w = w.data_ptr(); a.ldw = rw.ld;
  a.target = static_cast<const int64_t*>(target.data_ptr());
  a.ignore_index = ignore;
  a.scale = (float)scale;
  a.negate = form == kLogprobs;
  a.lse = ptr<float>(lse);
  a.status = ptr<int32_t>(status);
  a.stream = stream_of(h);
  return a;
}

HeadResult head_forward(const Tensor& h, const Tensor& w, const Tensor& target, int64_t ignore, double scale, int64_t form, bool entropy, bool keep, const Tensor& status) {
  c10::OptionalDeviceGuard guard(h.device());
  const int64_t M = target.numel();
  HeadResult r;
  Tensor each = empty_like_options(h, target.sizes(), at::kFloat);
  r.lse = empty_like_options(h, {M}, at::kFloat);
  if (keep) r.logp = empty_like_options(h, {M}, at::kFloat);         // (the output is the caller's, who may change it)
  if (entropy) r.entropy = empty_like_options(h, target.sizes(), at::kFloat);
  metis_head_args a = head_args(h, w, target, r.lse, ignore, scale, form, status);
  const Tensor ws = scratch(h, lib.metis_head_loss_workspace_bytes(a.M, a.V, a.K, entropy));
  a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel();
  check(lib.metis_head_loss_keep(&a, ptr<float>(each), ptr<float>(r.entropy), ptr<float>(r.logp)), "metis_head_loss_keep");
  r.out = each;
  if (form == kSum || form == kMean) {
    r.out = empty_like_options(h, {}, at::kFloat);
    r.inv_count = empty_like_options(h, {1}, at::kFloat);
    check(lib.metis_head_sum(ptr<float>(each), a.target, ignore, M, form == kMean, ptr<float>(r.out), ptr<float>(r.inv_count), a.stream), "metis_head_sum");
  }
  return r;
}

struct HeadFunction : torch::autograd::Function<HeadFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& target, int64_t ignore, double scale, int64_t form, bool entropy,
                               const Tensor* status) {
    const HeadResult r = head_forward(h, w, target, ignore, scale, form, entropy, true, *status);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({h, w, target, r.lse, r.logp, r.inv_count});
    ctx->saved_data["o"] = std::vector<int64_t>{ignore, form, w.size(0), w.size(1)};
    ctx->saved_data["h"] = h.sizes().vec();
    ctx->saved_data["s"] = scale;
    keep_status(ctx, *status);
    if (!entropy) return {r.out};
    ctx->mark_non_differentiable({r.entropy});
    return {r.out, r.entropy};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> o = ctx->saved_data["o"].toIntVector();
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    if (!need_h && !need_w) return out;
    {
      at::AutoGradMode off(false);
      const std::vector<int64_t> h_shape = ctx->saved_data["h"].toIntVector();
      const Tensor& dout = grads[0];                        // (on the device of the forward pass: the engine sees to it)
      c10::OptionalDeviceGuard guard(dout.device());
      Rows rh, rw;
      const Tensor h = as_operand(given_back(saved[0], dout, at::kBFloat16, h_shape), rh), w = as_operand(given_back(saved[1], dout, at::kBFloat16, {o[2], o[3]}), rw);
      const Tensor target = given_back(saved[2], dout, at::kLong, at::IntArrayRef(h_shape).slice(0, h_shape.size() - 1)).contiguous();
      const Tensor lse = given_back(saved[3], dout, at::kFloat, {target.numel()}).contiguous(), logp = given_back(saved[4], dout, at::kFloat, {target.numel()}).contiguous();
      const Tensor inv_count = saved[5].defined() ? given_back(saved[5], dout, at::kFloat, {1}) : Tensor();
      metis_head_args a = head_args(h, w, target, lse, o[0], ctx->saved_data["s"].toDouble(), o[1], kept_status(ctx));
      Tensor g = grads[0].reshape({-1});
      const bool each = g.numel() > 1 && g.stride(0) != 0;         // else one value for all rows
      if (each) g = g.contiguous();
      if (need_h) out[0] = empty_like_options(h, h.sizes(), at::kBFloat16);
      if (need_w) out[1] = empty_like_options(h, w.sizes(), at::kBFloat16);
      const Tensor ws = scratch(h, lib.metis_head_backward_workspace_bytes(a.M, a.V, a.K));
      a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel();
      check(lib.metis_head_backward_kept(&a, ptr<float>(logp), ptr<float>(g), each, ptr<float>(inv_count), ptr(out[0]), a.K, ptr(out[1]), a.K), "metis_head_backward_kept");
    }
    return once(std::move(out));
  }
};

// ---- calls ------------------------------------------------------------------------------------------------------------

bool tensor_or_none(PyObject* o, Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}

bool status_word(const Tensor& status, const Tensor& like) {
  return !status.defined() || (plain(status, like, at::kInt) && status.numel() == 1);
}

// What torch records of its own operations and these calls do not show it: their answers would come without their derivative, or as constants
// of the trace, and nobody would know.  (Wrappers of function transforms have no data to read, and raise where it is read.)
void check_followed(std::initializer_list<const Tensor*> tensors) {
  using Mode = c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !(Modes::any_modes_set() && (Modes::get_mode(Mode::PROXY) || Modes::get_mode(Mode::FAKE) || Modes::get_mode(Mode::FUNCTIONAL))),
              "the bf16 products cannot be traced: they are no operations of torch");
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    TORCH_CHECK(!t->_fw_grad(0).defined(), "the bf16 products have no forward-mode derivative");
    TORCH_CHECK(!t->unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python), "the bf16 products take no tensor subclass that dispatches by itself");
  }
}

// x, weight, bias or None, gate or None, residual or None, activation, status or None -> the output, or None where dense.py has to look at the arguments first
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, w, bias, gate, residual, status;
  if (nargs != 7 || !PyLong_Check(args[5])) {
    PyErr_SetString(PyExc_TypeError, "linear: five tensors, an activation and a status word");
    return nullptr;
  }
  const int64_t act = PyLong_AsLongLong(args[5]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  if (!tensor_or_none(args[0], &x) || !tensor_or_none(args[1], &w) || !tensor_or_none(args[2], &bias) || !tensor_or_none(args[3], &gate) ||
      !tensor_or_none(args[4], &residual) || !tensor_or_none(args[6], &status) || !x.defined() || !w.defined())
    Py_RETURN_NONE;
  check_followed({&x, &w, &bias, &gate, &residual});
  if (!plain(x, x, at::kBFloat16) || !plain(w, x, at::kBFloat16) || w.dim() != 2 || x.dim() < 1) Py_RETURN_NONE;
  Rows rx(x), rw(w);
  if (!operand(x, rx) || !operand(w, rw) || rx.cols != rw.cols || rw.rows == 0 || rw.cols == 0 || rw.cols % 8 != 0) Py_RETURN_NONE;
  if (bias.defined() && !((bias.scalar_type() == at::kFloat && plain(bias, x, at::kFloat)) || plain(bias, x, at::kBFloat16))) Py_RETURN_NONE;
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != rw.rows || !bias.is_contiguous())) Py_RETURN_NONE;
  for (const Tensor* t : {&gate, &residual}) {
    if (!t->defined()) continue;
    if (!plain(*t, x, at::kBFloat16) || t->dim() != x.dim() || t->size(-1) != rw.rows || !Rows(*t).ok) Py_RETURN_NONE;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) if (t->size(i) != x.size(i)) Py_RETURN_NONE;
  }
  if (!status_word(status, x)) Py_RETURN_NONE;
  Tensor y;
  {
    NoGil free_;
    const auto records = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    if (c10::GradMode::is_enabled() && (records(x) || records(w) || records(bias) || records(gate) || records(residual))) {
      const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      y = LinearFunction::apply(x, w, given(bias), given(gate), given(residual), act, &status);
    } else {
      y = linear_forward(x, w, bias, gate, residual, act, false, false, status).y;
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// hidden, weight, target (int64), ignore_index, scale, form, entropy, status or None -> (output, entropies or None), or None as above
PyObject* head(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor h, w, target, status;
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "head: hidden, weight, target, ignore_index, scale, form, entropy, status");
    return nullptr;
  }
  const int64_t ignore = PyLong_AsLongLong(args[3]);
  if (ignore == -1 && PyErr_Occurred()) return nullptr;
  const double scale = PyFloat_AsDouble(args[4]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  const int64_t form = PyLong_AsLongLong(args[5]);
  if (form == -1 && PyErr_Occurred()) return nullptr;
  const int entropy = PyObject_IsTrue(args[6]);
  if (entropy < 0) return nullptr;
  if (!tensor_or_none(args[0], &h) || !tensor_or_none(args[1], &w) || !tensor_or_none(args[2], &target) || !tensor_or_none(args[7], &status) || !h.defined() || !w.defined() || !target.defined())
    Py_RETURN_NONE;
  check_followed({&h, &w, &target});
  if (!plain(h, h, at::kBFloat16) || !plain(w, h, at::kBFloat16) || !plain(target, h, at::kLong) || w.dim() != 2 || h.dim() < 1) Py_RETURN_NONE;
  Rows rh(h), rw(w);
  if (!operand(h, rh) || !operand(w, rw) || rh.cols != rw.cols || rw.rows == 0 || rw.cols == 0 || rw.cols % 8 != 0 || rh.rows == 0) Py_RETURN_NONE;
  if (!target.is_contiguous() || target.dim() != h.dim() - 1) Py_RETURN_NONE;
  for (int64_t i = 0; i < target.dim(); ++i) if (target.size(i) != h.size(i)) Py_RETURN_NONE;
  if (!status_word(status, h)) Py_RETURN_NONE;
  Tensor out, ent;
  {
    NoGil free_;
    if (c10::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad())) {
      const variable_list r = HeadFunction::apply(h, w, target, ignore, scale, form, entropy != 0, &status);
      out = r[0];
      if (entropy) ent = r[1];
    } else {
      const HeadResult r = head_forward(h, w, target, ignore, scale, form, entropy != 0, false, status);
      out = r.out;
      ent = r.entropy;
    }
  }
  PyObject* first = THPVariable_Wrap(out);
  if (!first) return nullptr;
  PyObject* second = ent.defined() ? THPVariable_Wrap(ent) : Py_NewRef(Py_None);
  if (!second) { Py_DECREF(first); return nullptr; }
  PyObject* pair = PyTuple_Pack(2, first, second);
  Py_DECREF(first);
  Py_DECREF(second);
  return pair;
  END_HANDLE_TH_ERRORS
}

// name, address: binds an entry point; returns whether this module has a use for it
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "bind: a name and an address");
    return nullptr;
  }
  const char* name = PyUnicode_AsUTF8(args[0]);
  if (!name) return nullptr;
  const unsigned long long address = PyLong_AsUnsignedLongLong(args[1]);
  if (address == (unsigned long long)-1 && PyErr_Occurred()) return nullptr;
#define X(entry) if (strcmp(name, #entry) == 0) { lib.entry = reinterpret_cast<decltype(lib.entry)>(static_cast<uintptr_t>(address)); Py_RETURN_TRUE; }
  METIS_DENSE_ENTRIES(X)
#undef X
  Py_RETURN_FALSE;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(linear), METHOD(head), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "metis_dense", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_metis_dense(void) { return PyModule_Create(&module); }
