// The host side of rollout.py: checks, allocations and calls of the kernels of a rollout, and the rotary positions as a native autograd function.
//
// A decode step makes two of these calls in every layer, for kernels of a few microseconds: from Python, with its checks and a foreign call of twenty
// arguments, each would cost several times that.  A cache is a capsule of its tensors: what they are is settled once, where their memory is at each call.
#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <ATen/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>

#include <string.h>

#include "../../include/metis_nvfp4.h"

namespace {

#define METIS_ROLLOUT_ENTRIES(X)                                                                                                   \
  X(metis_last_error_string) X(metis_rotary) X(metis_cache_check) X(metis_cache_append) X(metis_cache_attend) X(metis_cache_attend_workspace_bytes)     \
  X(metis_cache_workspace_bytes) X(metis_cache_reserve) X(metis_cache_fork) X(metis_cache_free) X(metis_cache_compact) X(metis_sample)
struct Entries {
#define X(name) decltype(&::name) name = nullptr;
  METIS_ROLLOUT_ENTRIES(X)
#undef X
} lib;

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- arguments ------------------------------------------------------------------------------------------------------

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

struct BadArguments {};

struct Args {
  PyObject* const* v;
  Py_ssize_t n, at = 0;
  PyObject* next() {
    if (at >= n) {
      PyErr_SetString(PyExc_TypeError, "too few arguments");
      throw BadArguments();
    }
    return v[at++];
  }
  Tensor tensor(const char* what) {
    PyObject* o = next();
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "%s must be a tensor, not %s", what, Py_TYPE(o)->tp_name);
      throw BadArguments();
    }
    return THPVariable_Unpack(o);
  }
  Tensor optional(const char* what) {
    if (at < n && v[at] == Py_None) { ++at; return Tensor(); }
    return tensor(what);
  }
  int64_t i64() {
    const long long x = PyLong_AsLongLong(next());
    if (x == -1 && PyErr_Occurred()) throw BadArguments();
    return x;
  }
  double f64() {
    const double x = PyFloat_AsDouble(next());
    if (x == -1.0 && PyErr_Occurred()) throw BadArguments();
    return x;
  }
  bool truth() {
    const int x = PyObject_IsTrue(next());
    if (x < 0) throw BadArguments();
    return x != 0;
  }
};

#define ROLLOUT_BEGIN(args, nargs) HANDLE_TH_ERRORS try { Args a{args, nargs};
#define ROLLOUT_END } catch (const BadArguments&) { return nullptr; } END_HANDLE_TH_ERRORS

void check(int32_t rc, const char* what) {
  if (rc == METIS_OK) return;
  if (rc == METIS_ERR_BAD_SHAPE) TORCH_CHECK_VALUE(false, what, ": ", lib.metis_last_error_string());
  TORCH_CHECK(false, what, ": status ", rc, ": ", lib.metis_last_error_string());
}

// What torch records of its own operations and these calls do not show it.
void check_followed(const Tensor& t, const char* what) {
  if (!t.defined()) return;
  TORCH_CHECK(!t._fw_grad(0).defined(), what, ": these calls have no forward-mode derivative");
  TORCH_CHECK(!t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python), what, ": these calls take no tensor subclass that dispatches by itself");
}
void check_untraced() {
  using Mode = c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !(Modes::any_modes_set() && (Modes::get_mode(Mode::PROXY) || Modes::get_mode(Mode::FAKE) || Modes::get_mode(Mode::FUNCTIONAL))),
              "the calls of a rollout cannot be traced: they are no operations of torch");
}
void check_constant(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !c10::GradMode::is_enabled() || !t.requires_grad(), what, " requires a gradient, which this call does not form: make it under torch.no_grad()");
}

void check_tensor(const Tensor& t, const char* what, at::ScalarType type, const char* type_name) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: there is no CPU fallback");
  TORCH_CHECK_TYPE(t.scalar_type() == type, what, " must be ", type_name, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, what, " must be a dense tensor");
  check_followed(t, what);
}
void check_device(const Tensor& t, const char* what, const c10::Device& device) { TORCH_CHECK_VALUE(t.device() == device, what, " is on ", t.device(), ", not on ", device); }

void* stream_of(const c10::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
Tensor empty_on(const c10::Device& device, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Indices: int32 or int64, contiguous, of `count` elements (any shape) where it is not negative.
Tensor indices(const Tensor& t, const char* what, const c10::Device& device, int64_t count) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: there is no CPU fallback");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what, " must be int32 or int64, got ", t.scalar_type());
  check_device(t, what, device);
  check_followed(t, what);
  TORCH_CHECK_VALUE(count < 0 || t.numel() == count, what, " has ", t.numel(), " elements, not ", count);
  return t.contiguous();
}
bool wide(const Tensor& t) { return t.defined() && t.scalar_type() == at::kLong; }

PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) { Py_DECREF(out); return nullptr; }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// ---- rotary positions -------------------------------------------------------------------------------------------------

struct Turn {
  Tensor turns;                    // int64 [rotary_dim / 2]: the bits of unsigned fractions of a turn
  double magnitude = 1.0;
  int64_t rotary_dim = 0;
  bool interleaved = false;
};

// Kernels read rotary_dim / 2 of them: Rotary's attributes are plain ones, which a program can set.
void check_turns(const Tensor& turns, int64_t rotary_dim) {
  TORCH_CHECK(turns.is_cuda(), "the rotary positions' frequencies must be a CUDA tensor: there is no CPU fallback");
  TORCH_CHECK_TYPE(turns.scalar_type() == at::kLong, "the rotary positions' frequencies must be int64, got ", turns.scalar_type());
  TORCH_CHECK_VALUE(rotary_dim > 0 && rotary_dim % 2 == 0 && turns.dim() == 1 && turns.size(0) == rotary_dim / 2 && turns.is_contiguous(),
                    "rotary positions of ", rotary_dim, " elements with frequencies ", turns.sizes(), " of strides ", turns.strides());
}

// x [..., heads, D] as tokens of two strides, the inner ones those of the third dimension from behind; copied where it has more
struct Tokens {
  Tensor t;
  int64_t outer = 1, inner = 1, s_outer = 0, s_inner = 0, s_head = 0;
  explicit Tokens(const Tensor& x) : t(x.resolve_neg()) {
    if (t.dim() > 4 || (t.size(-1) > 1 && t.stride(-1) != 1)) t = t.contiguous();
    if (t.dim() > 4) t = t.view({-1, t.size(-3), t.size(-2), t.size(-1)});
    const int64_t d = t.dim();
    s_head = t.stride(d - 2);
    if (d >= 3) { inner = t.size(d - 3); s_inner = t.stride(d - 3); }
    if (d >= 4) { outer = t.size(0); s_outer = t.stride(0); }
  }
};

variable_list turned(const Tensor& q, const Tensor& k, const Tensor& positions, const Turn& by, bool inverse) {
  c10::OptionalDeviceGuard guard(q.device());
  const Tensor q_out = empty_on(q.device(), q.sizes(), q.scalar_type());
  const Tensor k_out = k.defined() ? empty_on(q.device(), k.sizes(), q.scalar_type()) : Tensor();
  if (q.numel() == 0 || (k.defined() && k.numel() == 0)) {
    // (no tokens, or one of the two without heads)
    if (q.numel() > 0) return {turned(q, Tensor(), positions, by, inverse)[0], k_out};
    if (k.defined() && k.numel() > 0) return {q_out, turned(k, Tensor(), positions, by, inverse)[0]};
    return {q_out, k_out};
  }
  const Tokens tq(q);
  metis_rotary_args a = {};
  a.tokens = tq.outer * tq.inner; a.inner = tq.inner;
  a.heads_q = (int32_t)q.size(-2); a.head_dim = (int32_t)q.size(-1); a.rotary_dim = (int32_t)by.rotary_dim;
  a.interleaved = by.interleaved; a.inverse = inverse; a.dtype = q.scalar_type() == at::kFloat ? METIS_DTYPE_F32 : METIS_DTYPE_BF16;
  a.positions_64 = wide(positions);
  a.turns = reinterpret_cast<const uint64_t*>(by.turns.data_ptr()); a.magnitude = (float)by.magnitude;
  a.positions = ptr(positions);
  a.q = tq.t.data_ptr(); a.q_outer = tq.s_outer; a.q_token = tq.s_inner; a.q_head = tq.s_head; a.q_out = q_out.data_ptr();
  std::optional<Tokens> tk;
  if (k.defined()) {
    tk.emplace(k);
    a.heads_k = (int32_t)k.size(-2);
    a.k = tk->t.data_ptr(); a.k_outer = tk->s_outer; a.k_token = tk->s_inner; a.k_head = tk->s_head; a.k_out = k_out.data_ptr();
  }
  a.stream = stream_of(q.device());
  check(lib.metis_rotary(&a), "metis_rotary");
  return {q_out, k_out};
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const std::optional<Tensor>& positions, const Turn* by, bool inverse) {
    ctx->set_materialize_grads(false);
    const Tensor at_ = positions.value_or(Tensor());
    ctx->save_for_backward({at_, by->turns});
    ctx->saved_data["o"] = std::vector<int64_t>{by->rotary_dim, by->interleaved, inverse, k.has_value(), positions.has_value()};
    ctx->saved_data["m"] = by->magnitude;
    ctx->saved_data["q"] = q.sizes().vec();
    const variable_list out = turned(q, k.value_or(Tensor()), at_, *by, inverse);
    return k.has_value() ? out : variable_list{out[0]};
  }

  // The transposed map is the turn the other way, and is differentiated like this one where a graph of it is asked for.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> o = ctx->saved_data["o"].toIntVector();
    const Turn by{saved[1], ctx->saved_data["m"].toDouble(), o[0], o[1] != 0};
    const bool with_k = o[3] != 0;
    const Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), gk = with_k && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    variable_list out(5);
    if (!gq.defined() && !gk.defined()) return out;
    const Tensor& any = gq.defined() ? gq : gk;
    // saved tensors that a hook gave back are asked whether they are what was saved
    const std::vector<int64_t> q_shape = ctx->saved_data["q"].toIntVector();
    int64_t tokens = 1;
    for (size_t i = 0; i + 2 < q_shape.size(); ++i) tokens *= q_shape[i];
    TORCH_CHECK(by.turns.is_cuda() && by.turns.device() == any.device() && by.turns.scalar_type() == at::kLong && by.turns.numel() == o[0] / 2 && by.turns.is_contiguous(),
                "the saved frequencies came back as something else");
    Tensor positions;
    if (o[4]) {
      TORCH_CHECK(saved[0].defined() && saved[0].numel() == tokens, "the saved positions came back as something else");
      positions = indices(saved[0], "saved positions", any.device(), tokens);
    }
    const Tensor other = gq.defined() && gk.defined() ? gk : Tensor();
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    const variable_list r = c10::GradMode::is_enabled() ? RotaryFunction::apply(any, given(other), given(positions), &by, o[2] == 0) : turned(any, other, positions, by, o[2] == 0);
    out[0] = gq.defined() ? r[0] : Tensor();
    if (gk.defined()) out[1] = gq.defined() ? r[1] : r[0];
    return out;
  }
};

// q, k or None, positions or None, turns, magnitude, rotary_dim, interleaved -> q, k or None
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  const Tensor q = a.tensor("q"), k = a.optional("k");
  Tensor positions = a.optional("positions");
  Turn by;
  by.turns = a.tensor("turns");
  by.magnitude = a.f64();
  by.rotary_dim = a.i64();
  by.interleaved = a.truth();
  check_untraced();
  for (const auto& [t, name] : {std::make_pair(&q, "q"), std::make_pair(&k, "k")}) {
    if (!t->defined()) continue;
    check_tensor(*t, name, t->scalar_type() == at::kFloat ? at::kFloat : at::kBFloat16, "bfloat16 or float32");
    TORCH_CHECK_VALUE(t->dim() >= 2 && t->size(-1) >= by.rotary_dim && t->size(-1) % 8 == 0 && t->size(-1) <= 256,
                      name, " must be [..., heads, head_dim] with head_dim a multiple of 8 from ", by.rotary_dim, " to 256, not ", t->sizes());
    check_device(*t, name, by.turns.device());
  }
  check_turns(by.turns, by.rotary_dim);
  const at::IntArrayRef lead = q.sizes().slice(0, q.dim() - 2);
  if (k.defined()) {
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "q is ", q.scalar_type(), " and k ", k.scalar_type());
    TORCH_CHECK_VALUE(k.dim() == q.dim() && k.sizes().slice(0, k.dim() - 2) == lead && k.size(-1) == q.size(-1), "shapes do not fit: q ", q.sizes(), ", k ", k.sizes());
  }
  if (positions.defined()) {
    positions = indices(positions, "positions", q.device(), -1);
    if (positions.sizes() != lead) {
      TORCH_CHECK_VALUE(positions.dim() <= (int64_t)lead.size(), "positions ", positions.sizes(), " do not fit tokens ", lead);
      for (int64_t i = 1; i <= positions.dim(); ++i)
        TORCH_CHECK_VALUE(positions.size(-i) == lead[lead.size() - i] || positions.size(-i) == 1, "positions ", positions.sizes(), " do not fit tokens ", lead);
      positions = positions.expand(lead).contiguous();
    }
  }
  variable_list out;
  {
    NoGil free_;
    if (c10::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
      const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      out = RotaryFunction::apply(q, given(k), given(positions), &by, false);
      if (out.size() < 2) out.emplace_back();
    } else {
      out = turned(q, k, positions, by, false);
    }
  }
  return tuple_of({out[0], out[1]});
  ROLLOUT_END
}

// ---- the cache --------------------------------------------------------------------------------------------------------

// A tensor of a cache, as it was when the cache was made.
struct Held {
  const char* name;
  Tensor t;
  at::ScalarType type = at::kInt;
  std::vector<int64_t> shape;
  void keep(const Tensor& tensor) { t = tensor; type = t.scalar_type(); shape = t.sizes().vec(); }
  // Where its memory is now: a storage may be given back and taken again between two calls, or a tensor be set to another one's.
  void* address(const c10::Device& device) const {
    if (!t.defined()) return nullptr;
    TORCH_CHECK_VALUE(t.device() == device && t.scalar_type() == type && t.sizes() == shape && t.is_contiguous(),
                      "the cache's ", name, " has become another tensor: ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", it was ", type, " ", at::IntArrayRef(shape), " on ", device);
    const size_t has = t.storage().nbytes(), needs = (size_t)(t.storage_offset() + t.numel()) * t.element_size();
    TORCH_CHECK_VALUE(has >= needs, "the cache's ", name, " has no memory: a storage of ", has, " bytes for ", needs);
    return t.data_ptr();
  }
};
struct Cache {
  Held pool{"pool"}, tables{"tables"}, lengths{"lengths"}, refs{"refs"}, scales{"scales"}, status{"status"}, refused{"refused"};
  metis_cache c = {};                   // sizes; addresses are those of `now`
  c10::Device device = c10::Device(c10::kCPU);
  metis_cache now() const {
    metis_cache m = c;
    m.pool = pool.address(device);
    TORCH_CHECK_VALUE((reinterpret_cast<uintptr_t>(m.pool) & 15) == 0, "the cache's pool must be 16-byte aligned");
    m.tables = static_cast<int32_t*>(tables.address(device)); m.lengths = static_cast<int32_t*>(lengths.address(device));
    m.refs = static_cast<int32_t*>(refs.address(device)); m.scales = static_cast<const float*>(scales.address(device));
    m.status = static_cast<int32_t*>(status.address(device)); m.refused = static_cast<int32_t*>(refused.address(device));
    return m;
  }
  // Of a call that reads or writes elements.
  void check_constants() const {
    check_constant(pool.t, "pool");
    check_constant(scales.t, "scales");
  }
};
constexpr const char* kCapsule = "metis_cache";

void drop_cache(PyObject* o) { delete static_cast<Cache*>(PyCapsule_GetPointer(o, kCapsule)); }

Cache& cache_of(Args& a) {
  void* p = PyCapsule_GetPointer(a.next(), kCapsule);
  if (!p) throw BadArguments();
  return *static_cast<Cache*>(p);
}

// pool, tables, lengths, refs, scales or None, status, refused -> the cache
PyObject* cache(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  auto h = std::make_unique<Cache>();
  const Tensor pool = a.tensor("pool"), tables = a.tensor("tables"), lengths = a.tensor("lengths"), refs = a.tensor("refs"), scales = a.optional("scales"), status = a.tensor("status"), refused = a.tensor("refused");
  const bool e4m3 = pool.scalar_type() == at::kFloat8_e4m3fn;
  check_tensor(pool, "pool", e4m3 ? at::kFloat8_e4m3fn : at::kBFloat16, "bfloat16 or float8_e4m3fn");
  TORCH_CHECK_VALUE(pool.dim() == 6 && pool.size(2) == 2, "pool must be [pages, layers, 2, kv_heads, page_size, head_dim], not ", pool.sizes());
  h->device = pool.device();
  for (const auto& [t, name] : {std::make_pair(&tables, "tables"), std::make_pair(&lengths, "lengths"), std::make_pair(&refs, "refs"), std::make_pair(&status, "status"), std::make_pair(&refused, "refused")}) {
    check_tensor(*t, name, at::kInt, "int32");
    check_device(*t, name, h->device);
    TORCH_CHECK_VALUE(t->is_contiguous(), name, " must be contiguous");
  }
  TORCH_CHECK_VALUE(pool.is_contiguous() && aligned16(pool), "pool must be contiguous and 16-byte aligned");
  TORCH_CHECK_VALUE(tables.dim() == 2 && lengths.dim() == 1 && lengths.size(0) == tables.size(0), "tables ", tables.sizes(), " and lengths ", lengths.sizes(), " do not fit");
  TORCH_CHECK_VALUE(refs.dim() == 1 && refs.size(0) == pool.size(0), "refs ", refs.sizes(), " do not fit a pool of ", pool.size(0), " pages");
  TORCH_CHECK_VALUE(status.numel() == 1 && refused.dim() == 1 && refused.size(0) == tables.size(0), "status must have one element, refused one for each sequence");
  TORCH_CHECK_VALUE(e4m3 == scales.defined(), "scales go with float8_e4m3fn, and with nothing else");
  if (e4m3) {
    check_tensor(scales, "scales", at::kFloat, "float32");
    check_device(scales, "scales", h->device);
    TORCH_CHECK_VALUE(scales.is_contiguous() && scales.dim() == 3 && scales.size(0) == pool.size(1) && scales.size(1) == 2 && scales.size(2) == pool.size(3),
                      "scales must be contiguous [layers, 2, kv_heads], not ", scales.sizes());
    h->scales.keep(scales);
  }
  h->pool.keep(pool); h->tables.keep(tables); h->lengths.keep(lengths); h->refs.keep(refs); h->status.keep(status); h->refused.keep(refused);
  metis_cache& c = h->c;
  c.pages = pool.size(0); c.layers = (int32_t)pool.size(1); c.kv_heads = (int32_t)pool.size(3);
  c.page_size = (int32_t)pool.size(4); c.head_dim = (int32_t)pool.size(5); c.dtype = e4m3 ? METIS_DTYPE_E4M3 : METIS_DTYPE_BF16;
  c.sequences = tables.size(0); c.width = tables.size(1); c.flags = METIS_CACHE_HAS_REFUSED;
  const metis_cache m = h->now();
  check(lib.metis_cache_check(&m), "metis_cache_check");
  PyObject* o = PyCapsule_New(h.get(), kCapsule, drop_cache);
  if (o) h.release();
  return o;
  ROLLOUT_END
}

// x [tokens, heads, head_dim] as the kernels read it: rows of a head dense, strides that 16 bytes divide
Tensor heads_of(const Tensor& x, const char* what, const Cache& h, int64_t tokens, int64_t heads, int64_t step) {
  check_tensor(x, what, at::kBFloat16, "bfloat16");
  check_device(x, what, h.device);
  check_constant(x, what);
  TORCH_CHECK_VALUE(x.dim() == 3 && (tokens < 0 || x.size(0) == tokens) && (heads < 0 || x.size(1) == heads) && x.size(2) == h.c.head_dim,
                    what, " has shape ", x.sizes(), ", which does not fit ", tokens < 0 ? x.dim() == 3 ? x.size(0) : 0 : tokens, " tokens and a cache of ", h.c.kv_heads, " heads of ", h.c.head_dim);
  const bool fine = !x.is_neg() && x.stride(2) == 1 && (reinterpret_cast<uintptr_t>(x.data_ptr()) & (2 * step - 1)) == 0 && x.stride(0) % step == 0 && x.stride(1) % step == 0;
  return fine ? x : x.resolve_neg().clone(at::MemoryFormat::Contiguous);
}

// cache, layer, q or None, k, v, slots or None, positions or None, turns or None, magnitude, rotary_dim, interleaved -> q or None
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  const int64_t layer = a.i64();
  Tensor q = a.optional("q"), k = a.tensor("k"), v = a.tensor("v");
  Tensor slots = a.optional("slots"), positions = a.optional("positions");
  const Tensor turns = a.optional("turns");
  const double magnitude = a.f64();
  const int64_t rotary_dim = a.i64();
  const bool interleaved = a.truth();
  check_untraced();
  TORCH_CHECK_VALUE(layer >= 0 && layer < h.c.layers, "layer ", layer, " of a cache of ", h.c.layers);
  h.check_constants();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  k = heads_of(k, "k", h, -1, h.c.kv_heads, 8);
  const int64_t tokens = k.size(0);
  v = heads_of(v, "v", h, tokens, h.c.kv_heads, 8);
  if (q.defined()) q = heads_of(q, "q", h, tokens, -1, 8);
  slots = indices(slots, "slots", h.device, tokens);
  positions = indices(positions, "positions", h.device, tokens);
  if (turns.defined()) {
    check_turns(turns, rotary_dim);
    check_device(turns, "the rotary positions' frequencies", h.device);
    TORCH_CHECK_VALUE(rotary_dim <= h.c.head_dim, "rotary positions of ", rotary_dim, " elements on heads of ", h.c.head_dim);
  }
  Tensor out;
  {
    NoGil free_;
    if (q.defined()) out = empty_on(h.device, q.sizes(), at::kBFloat16);
    if (tokens > 0) {
      metis_append_args g = {};
      g.tokens = tokens; g.layer = (int32_t)layer; g.rotary_dim = (int32_t)rotary_dim; g.interleaved = interleaved;
      g.turns = turns.defined() ? reinterpret_cast<const uint64_t*>(turns.data_ptr()) : nullptr; g.magnitude = (float)magnitude;
      g.index_64 = (wide(slots) ? 1 : 0) | (wide(positions) ? 2 : 0);
      g.slots = ptr(slots); g.positions = ptr(positions);
      if (q.defined() && q.size(1) > 0) { g.heads_q = (int32_t)q.size(1); g.q = q.data_ptr(); g.q_token = q.stride(0); g.q_head = q.stride(1); g.q_out = out.data_ptr(); }
      g.k = k.data_ptr(); g.k_token = k.stride(0); g.k_head = k.stride(1);
      g.v = v.data_ptr(); g.v_token = v.stride(0); g.v_head = v.stride(1);
      g.stream = stream_of(h.device);
      check(lib.metis_cache_append(&m, &g), "metis_cache_append");
    }
  }
  return out.defined() ? THPVariable_Wrap(out) : Py_NewRef(Py_None);
  ROLLOUT_END
}

// cache, layer, q, slots or None, scale, whether lse -> out, lse or None
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  const int64_t layer = a.i64();
  Tensor q = a.tensor("q"), slots = a.optional("slots");
  const double scale = a.f64();
  const bool want_lse = a.truth();
  check_untraced();
  TORCH_CHECK_VALUE(layer >= 0 && layer < h.c.layers, "layer ", layer, " of a cache of ", h.c.layers);
  h.check_constants();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  q = heads_of(q, "q", h, -1, -1, 2);
  TORCH_CHECK_VALUE(q.size(1) > 0 && q.size(1) % h.c.kv_heads == 0, "q has ", q.size(1), " heads, which ", h.c.kv_heads, " key-value heads do not divide");
  slots = indices(slots, "slots", h.device, q.size(0));
  Tensor out, lse;
  {
    NoGil free_;
    out = empty_on(h.device, q.sizes(), at::kBFloat16);
    if (want_lse) lse = empty_on(h.device, q.sizes().slice(0, 2), at::kFloat);
    if (q.size(0) > 0) {
      metis_attend_args g = {};
      g.rows = q.size(0); g.layer = (int32_t)layer; g.heads_q = (int32_t)q.size(1);
      g.slots = ptr(slots); g.slots_64 = wide(slots); g.scale = (float)scale;
      g.q = q.data_ptr(); g.q_row = q.stride(0); g.q_head = q.stride(1);
      g.out = out.data_ptr(); g.lse = ptr<float>(lse);
      const int64_t bytes = lib.metis_cache_attend_workspace_bytes(&m, g.rows, g.heads_q);
      const Tensor ws = empty_on(h.device, {bytes < 16 ? 16 : bytes}, at::kByte);
      g.workspace = ws.data_ptr(); g.workspace_bytes = ws.numel();
      g.stream = stream_of(h.device);
      check(lib.metis_cache_attend(&m, &g), "metis_cache_attend");
    }
  }
  return tuple_of({out, lse});
  ROLLOUT_END
}

// cache, slots or None (all), counts or None, count
PyObject* reserve(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  Tensor slots = a.optional("slots"), counts = a.optional("counts");
  const int64_t count = a.i64();
  check_untraced();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  slots = indices(slots, "slots", h.device, -1);
  const int64_t n = slots.defined() ? slots.numel() : h.c.sequences;
  counts = indices(counts, "counts", h.device, n);
  // one width for both
  if (slots.defined() && counts.defined() && wide(slots) != wide(counts)) { slots = slots.to(at::kLong); counts = counts.to(at::kLong); }
  if (n > 0) {
    NoGil free_;
    const Tensor ws = empty_on(h.device, {lib.metis_cache_workspace_bytes(&m, n)}, at::kByte);
    check(lib.metis_cache_reserve(&m, ptr(slots), ptr(counts), count, wide(slots) || wide(counts), n, ws.data_ptr(), ws.numel(), stream_of(h.device)), "metis_cache_reserve");
  }
  Py_RETURN_NONE;
  ROLLOUT_END
}

// cache, src, dst, whether pages are shared
PyObject* fork(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  Tensor src = a.tensor("src"), dst = a.tensor("dst");
  const bool share = a.truth();
  check_untraced();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  src = indices(src, "src", h.device, -1);
  dst = indices(dst, "dst", h.device, src.numel());
  if (wide(src) != wide(dst)) { src = src.to(at::kLong); dst = dst.to(at::kLong); }
  const int64_t n = src.numel();
  if (n > 0) {
    NoGil free_;
    const Tensor ws = empty_on(h.device, {lib.metis_cache_workspace_bytes(&m, n)}, at::kByte);
    check(lib.metis_cache_fork(&m, src.data_ptr(), dst.data_ptr(), wide(src), n, share, ws.data_ptr(), ws.numel(), stream_of(h.device)), "metis_cache_fork");
  }
  Py_RETURN_NONE;
  ROLLOUT_END
}

// cache, slots or None (all)
PyObject* release(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  const Tensor slots = indices(a.optional("slots"), "slots", h.device, -1);
  check_untraced();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  const int64_t n = slots.defined() ? slots.numel() : h.c.sequences;
  if (n > 0) check(lib.metis_cache_free(&m, ptr(slots), wide(slots), n, stream_of(h.device)), "metis_cache_free");
  Py_RETURN_NONE;
  ROLLOUT_END
}

// cache -> pages that are held
PyObject* compact(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Cache& h = cache_of(a);
  check_untraced();
  const metis_cache m = h.now();
  c10::OptionalDeviceGuard guard(h.device);
  Tensor live;
  {
    NoGil free_;
    live = empty_on(h.device, {1}, at::kInt);
    const Tensor ws = empty_on(h.device, {lib.metis_cache_workspace_bytes(&m, 1)}, at::kByte);
    check(lib.metis_cache_compact(&m, ptr<int32_t>(live), ws.data_ptr(), ws.numel(), stream_of(h.device)), "metis_cache_compact");
  }
  return THPVariable_Wrap(live);
  ROLLOUT_END
}

// ---- sampling ---------------------------------------------------------------------------------------------------------

// A number, or one for each row on the device.
struct Parameter {
  Tensor rows;
  double one = 0.0;
  Parameter(Args& a, const char* what, const c10::Device& device, int64_t count, at::ScalarType type, const char* type_name) {
    if (!THPVariable_Check(a.v[a.at < a.n ? a.at : 0])) { one = a.f64(); return; }
    rows = a.tensor(what);
    check_tensor(rows, what, type, type_name);
    check_device(rows, what, device);
    check_constant(rows, what);
    TORCH_CHECK_VALUE(rows.dim() == 1 && rows.size(0) == count, what, " has shape ", rows.sizes(), ", not (", count, ",)");
    rows = rows.resolve_neg().contiguous();
  }
};

// logits, u, temperature, top_k, top_p, min_p (each a number or a tensor), whether log-probabilities -> tokens, log-probabilities or None
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  ROLLOUT_BEGIN(args, nargs)
  Tensor logits = a.tensor("logits"), u = a.tensor("u");
  check_untraced();
  const bool half = logits.scalar_type() == at::kBFloat16;
  check_tensor(logits, "logits", half ? at::kBFloat16 : at::kFloat, "bfloat16 or float32");
  check_constant(logits, "logits");
  TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) > 0, "logits must be [rows, vocab], not ", logits.sizes());
  const c10::Device device = logits.device();
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK_VALUE(vocab <= METIS_SAMPLE_MAX_VOCAB, "vocabularies have at most ", METIS_SAMPLE_MAX_VOCAB, " entries, not ", vocab);
  const bool u_64 = u.scalar_type() == at::kDouble;
  check_tensor(u, "u", u_64 ? at::kDouble : at::kFloat, "float32 or float64");
  check_device(u, "u", device);
  check_constant(u, "u");
  TORCH_CHECK_VALUE(u.dim() == 1 && u.size(0) == rows, "u has shape ", u.sizes(), ", not (", rows, ",)");
  c10::OptionalDeviceGuard guard(device);
  const Parameter temperature(a, "temperature", device, rows, at::kFloat, "a number or float32"), top_k(a, "top_k", device, rows, at::kInt, "a number or int32"),
      top_p(a, "top_p", device, rows, at::kFloat, "a number or float32"), min_p(a, "min_p", device, rows, at::kFloat, "a number or float32");
  const bool want = a.truth();
  TORCH_CHECK_VALUE(temperature.rows.defined() || temperature.one == 0.0 || (temperature.one >= 0x1p-126 && temperature.one <= 3e38), "temperature must be 0, or from 2^-126 to 3e38, not ", temperature.one);
  TORCH_CHECK_VALUE(top_k.rows.defined() || (top_k.one >= 0.0 && top_k.one <= 2147483647.0 && top_k.one == (double)(int64_t)top_k.one), "top_k must be a whole number, 0 for all, not ", top_k.one);
  TORCH_CHECK_VALUE(top_p.rows.defined() || (top_p.one >= 0.0 && top_p.one <= 1.0), "top_p must be from 0 to 1, not ", top_p.one);
  TORCH_CHECK_VALUE(min_p.rows.defined() || (min_p.one >= 0.0 && min_p.one <= 1.0), "min_p must be from 0 to 1, not ", min_p.one);
  Tensor token, logprob;
  {
    NoGil free_;
    if (logits.is_neg() || (vocab > 1 && logits.stride(1) != 1) || (rows > 1 && logits.stride(0) < vocab)) logits = logits.resolve_neg().clone(at::MemoryFormat::Contiguous);
    u = u.resolve_neg().contiguous();
    token = empty_on(device, {rows}, at::kLong);
    if (want) logprob = empty_on(device, {rows}, at::kFloat);
    if (rows > 0) {
      metis_sample_args g = {};
      g.rows = rows; g.vocab = vocab; g.logits = logits.data_ptr(); g.ld = rows > 1 ? logits.stride(0) : vocab; g.dtype = half ? METIS_DTYPE_BF16 : METIS_DTYPE_F32;
      g.u_64 = u_64; g.u = u.data_ptr();
      g.temperature = (float)temperature.one; g.top_k = (int32_t)top_k.one; g.top_p = top_p.one; g.min_p = (float)min_p.one;
      g.temperature_rows = ptr<float>(temperature.rows); g.top_k_rows = ptr<int32_t>(top_k.rows); g.top_p_rows = ptr<float>(top_p.rows); g.min_p_rows = ptr<float>(min_p.rows);
      g.token = ptr<int64_t>(token); g.logprob = ptr<float>(logprob);
      g.stream = stream_of(device);
      check(lib.metis_sample(&g), "metis_sample");
    }
  }
  return tuple_of({token, logprob});
  ROLLOUT_END
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
  METIS_ROLLOUT_ENTRIES(X)
#undef X
  Py_RETURN_FALSE;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rotary), METHOD(cache), METHOD(append), METHOD(attend), METHOD(reserve), METHOD(fork), METHOD(release), METHOD(compact), METHOD(sample),
                         METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "metis_rollout", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_metis_rollout(void) { return PyModule_Create(&module); }
