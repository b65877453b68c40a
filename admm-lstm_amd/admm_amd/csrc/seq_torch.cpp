// seq_torch.cpp -- the Python entry points of the sequence-layer operators: argument checks, result tensors, autograd, over the
// C ABI of libseqops.so (include/seq_ops.h).  Native because a call is often a few microseconds of kernel: the same work in
// Python with ctypes took 25 us for a call without gradients, and 80 us for one with.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/hip/HIPStream.h>

#include <cmath>
#include <optional>
#include <sstream>
#include <string>

#include "seq_ops.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// a libseqops.so call that returned an error code: AdmmError in Python
struct SeqError : std::runtime_error {
  int code;
  SeqError(const std::string& m, int c) : std::runtime_error(m), code(c) {}
};

template <class... A>
std::string say(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
std::string shape(at::IntArrayRef s) {   // as Python prints a tuple
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}
std::string type(at::ScalarType t) {
  return t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : t == at::kFloat ? "float32" : say(t);
}

#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) throw py::value_error(say(__VA_ARGS__)); \
  } while (0)

void check(int rc, const char* what) {
  if (rc) throw SeqError(say(what, " failed (code ", rc, "): ", seq_last_error()), rc);
}

// Derivatives in forward mode would be lost: the kernels read the values alone.
constexpr const char* kNoForwardMode = " carries a forward-mode derivative, which this operator does not propagate (use backward mode)";
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

Tensor tensor(const py::handle& h, const char* name) {
  if (!THPVariable_Check(h.ptr()))
    throw py::type_error(say(name, " must be a tensor (got ", Py_TYPE(h.ptr())->tp_name, ")"));
  const Tensor& t = THPVariable_Unpack(h.ptr());
  // (a trace would have the allocation of the result and not the kernel that writes it)
  if (torch::jit::tracer::isTracing()) throw std::runtime_error("the sequence-layer operators cannot be traced");
  // batched, sparse and fake tensors, and subclasses that run PyTorch's operators in a way of their own (distributed ones): the values
  // that a pointer leads to are none, or not what they stand for
  const at::TensorImpl* impl = t.unsafeGetTensorImpl();
  if (!impl->has_storage() || impl->is_python_dispatch() || t.layout() != at::kStrided)
    throw py::type_error(say(name, " must be a dense tensor with memory of its own (got ", Py_TYPE(h.ptr())->tp_name, ", ", t.layout(), ")"));
  if (has_tangent(t)) {
    PyErr_SetString(PyExc_NotImplementedError, say(name, kNoForwardMode).c_str());
    throw py::error_already_set();
  }
  return t.resolve_neg();   // (the imaginary part of a conjugate is negated as it is read)
}
// the gradients that a backward pass begins with
void check_given(const variable_list& d_out) {
  for (const Tensor& t : d_out) TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), "a gradient", kNoForwardMode);
}
Tensor maybe(const py::handle& h, const char* name) { return h.is_none() ? Tensor() : tensor(h, name); }

struct Named {
  const char* name;
  const Tensor& t;
};
// all of them HIP tensors on one device
void require_device(std::initializer_list<Named> all) {
  const Tensor* first = nullptr;
  for (const Named& n : all) {
    if (!n.t.defined()) continue;
    if (!n.t.is_cuda())
      throw std::runtime_error(say(n.name, " must be a HIP device tensor (got ", n.t.device().str(),
                                   "); admm-lstm_amd has no CPU execution path"));
    if (!first) first = &n.t;
    REQUIRE(n.t.device() == first->device(), n.name, " is on ", n.t.device().str(), ", the other tensors on ", first->device().str());
  }
}

int dtype_of(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 ? SEQ_BF16 : s == at::kHalf ? SEQ_FP16 : s == at::kFloat ? SEQ_FP32 : -1;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
// the tensor itself where its last axis is contiguous, else a contiguous copy
Tensor rows_last(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }
bool wants_grad(std::initializer_list<Tensor> all) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : all)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// autograd takes absent tensors as absent, not as undefined ones
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// What a backward returns: under create_graph the gradients carry a node that raises when they are differentiated again.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  for (Tensor& g : grads) marked.push_back(g.defined() ? g.detach().requires_grad_() : g);
  auto node = std::make_shared<torch::autograd::DelayedError>(say(what, " can be differentiated once only"), (int64_t)marked.size());
  return (*node)(std::move(marked));
}

// ----------------------------------------------------------------------------------------------- gated delta rule

void check_rows(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, int64_t lead, const char* lead_name) {
  REQUIRE(dtype_of(q) >= 0, "q must be bfloat16, float16 or float32 (got ", type(q.scalar_type()), ")");
  for (const Named& n : {Named{"k", k}, Named{"v", v}})
    REQUIRE(n.t.scalar_type() == q.scalar_type(), n.name, " must have the type of q, ", type(q.scalar_type()), " (got ", type(n.t.scalar_type()), ")");
  for (const Named& n : {Named{"g", g}, Named{"beta", beta}})
    REQUIRE(n.t.scalar_type() == at::kFloat, n.name, " must be float32 (got ", type(n.t.scalar_type()), ")");
  for (const Named& n : {Named{"q", q}, Named{"k", k}, Named{"v", v}})
    REQUIRE(n.t.dim() == lead + 2, n.name, " must be ", lead_name, " x heads x values (got shape ", shape(n.t.sizes()), ")");
  REQUIRE(q.sizes() == k.sizes(), "q and k differ in shape: ", shape(q.sizes()), " and ", shape(k.sizes()));
  REQUIRE(v.sizes().slice(0, lead) == q.sizes().slice(0, lead), "v has ", lead_name, " ", shape(v.sizes().slice(0, lead)), ", q ", shape(q.sizes().slice(0, lead)));
  for (const Named& n : {Named{"g", g}, Named{"beta", beta}})
    REQUIRE(n.t.sizes() == v.sizes().slice(0, lead + 1), n.name, " must have shape ", shape(v.sizes().slice(0, lead + 1)), " (got ", shape(n.t.sizes()), ")");
  const int64_t Hk = q.size(lead), Hv = v.size(lead);
  REQUIRE(Hk > 0 && Hv > 0 && Hv % Hk == 0, "the number of value heads (", Hv, ") must be a multiple of that of query/key heads (", Hk, ")");
  REQUIRE(q.size(-1) >= 1 && q.size(-1) <= SEQ_DELTA_MAX_K, "query/key rows must have 1 to ", SEQ_DELTA_MAX_K, " values (got ", q.size(-1), ")");
  REQUIRE(v.size(-1) >= 1 && v.size(-1) <= SEQ_DELTA_MAX_V, "value rows must not be empty, nor longer than ", SEQ_DELTA_MAX_V, " (got ", v.size(-1), ")");
}

// the C descriptor of one call and the tensors that it points into
struct RuleCall {
  Tensor q, k, v, g, beta, initial, offsets;
  SeqDelta d{};
  RuleCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const Tensor& beta_, const Tensor& initial_,
           const Tensor& offsets_, double scale)
      : q(rows_last(q_)), k(rows_last(k_)), v(rows_last(v_)), g(g_), beta(beta_), initial(initial_), offsets(offsets_) {
    d.batch = q.size(0), d.T = q.size(1);
    d.sequences = offsets.defined() ? offsets.numel() - 1 : d.batch;
    d.Hk = (int32_t)q.size(2), d.K = (int32_t)q.size(3), d.Hv = (int32_t)v.size(2), d.V = (int32_t)v.size(3);
    d.dtype = dtype_of(q);
    d.offsets_64 = offsets.defined() && offsets.scalar_type() == at::kLong;
    d.scale = (float)scale;
    d.device = q.device().index();
    d.q = data(q), d.k = data(k), d.v = data(v);
    d.g = static_cast<const float*>(data(g)), d.beta = static_cast<const float*>(data(beta));
    for (int i = 0; i < 3; ++i) {
      d.q_stride[i] = q.stride(i), d.k_stride[i] = k.stride(i), d.v_stride[i] = v.stride(i);
      d.g_stride[i] = g.stride(i), d.beta_stride[i] = beta.stride(i);
    }
    d.offsets = data(offsets);
    d.initial = static_cast<const float*>(data(initial));
  }
  std::tuple<Tensor, Tensor, Tensor> forward(bool saved) {
    int64_t need = 0;
    check(seq_delta_workspace(&d, saved, &need), "gated_delta_rule");
    Tensor work = bytes(need, q), o = at::empty(v.sizes(), v.options());
    Tensor final_state = at::empty({d.sequences, d.Hv, d.K, d.V}, q.options().dtype(at::kFloat));
    check(seq_delta_forward(&d, saved, work.data_ptr(), need, o.data_ptr(), final_state.data_ptr<float>(), stream_of(q)), "gated_delta_rule");
    return {o, final_state, work};
  }
};

struct RuleFunction : torch::autograd::Function<RuleFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                               const std::optional<Tensor>& initial_, const std::optional<Tensor>& offsets_, double scale) {
    const Tensor initial = initial_.value_or(Tensor()), offsets = offsets_.value_or(Tensor());
    auto [o, final_state, work] = RuleCall(q, k, v, g, beta, initial, offsets, scale).forward(true);
    ctx->save_for_backward({q, k, v, g, beta, initial, offsets, work});   // work too: freed with them after the backward pass
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {o, final_state};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d_out) {
    const variable_list in = ctx->get_saved_variables();
    check_given(d_out);
    RuleCall call(in[0], in[1], in[2], in[3], in[4], in[5], in[6], ctx->saved_data["scale"].toDouble());
    const Tensor work = in[7];
    Tensor d_o = d_out[0].defined() ? d_out[0].resolve_neg().contiguous() : at::zeros(call.v.sizes(), call.v.options());
    Tensor d_final = d_out[1].defined() ? d_out[1].resolve_neg().contiguous() : Tensor();
    int64_t need = 0;
    check(seq_delta_backward_scratch(&call.d, &need), "gated_delta_rule");
    Tensor scratch = bytes(need, call.q);
    variable_list grads(8);
    for (int i = 0; i < 5; ++i) grads[i] = at::empty(in[i].sizes(), in[i].options());
    if (in[5].defined() && ctx->needs_input_grad(5)) grads[5] = at::empty(in[5].sizes(), in[5].options());
    check(seq_delta_backward(&call.d, work.const_data_ptr(), work.numel(), scratch.data_ptr(), need, data(d_o),
                             static_cast<const float*>(data(d_final)), grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(),
                             grads[3].data_ptr<float>(), grads[4].data_ptr<float>(),
                             grads[5].defined() ? grads[5].data_ptr<float>() : nullptr, stream_of(call.q)),
          "gated_delta_rule backward");
    return once(std::move(grads), "gated_delta_rule");
  }
};

py::tuple gated_delta_rule(const py::handle& q_, const py::handle& k_, const py::handle& v_, const py::handle& g_, const py::handle& beta_,
                           std::optional<double> scale, const py::handle& initial_, const py::handle& offsets_) {
  const Tensor q = tensor(q_, "q"), k = tensor(k_, "k"), v = tensor(v_, "v"), g = tensor(g_, "g"), beta = tensor(beta_, "beta");
  Tensor initial = maybe(initial_, "initial_state"), offsets = maybe(offsets_, "offsets");
  check_rows(q, k, v, g, beta, 2, "batch x time");
  int64_t n = q.size(0);
  if (offsets.defined()) {
    REQUIRE(q.size(0) == 1, "packed sequences need a batch of 1 (got ", q.size(0), ")");
    REQUIRE(offsets.dim() == 1 && offsets.numel() >= 1 && (offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong),
            "offsets must be a vector of int32 or int64 (got ", type(offsets.scalar_type()), ", shape ", shape(offsets.sizes()), ")");
    offsets = offsets.contiguous();
    n = offsets.numel() - 1;
  }
  if (initial.defined()) {
    const std::vector<int64_t> want = {n, v.size(2), q.size(3), v.size(3)};
    REQUIRE(initial.scalar_type() == at::kFloat && initial.sizes() == at::IntArrayRef(want), "initial_state must be float32 of shape ",
            shape(want), " (got ", type(initial.scalar_type()), ", ", shape(initial.sizes()), ")");
    initial = initial.contiguous();
  }
  require_device({{"q", q}, {"k", k}, {"v", v}, {"g", g}, {"beta", beta}, {"initial_state", initial}, {"offsets", offsets}});
  const double s = scale.value_or(1 / std::sqrt((double)q.size(3)));
  if (wants_grad({q, k, v, g, beta, initial})) {
    const variable_list r = RuleFunction::apply(q, k, v, g, beta, given(initial), given(offsets), s);
    return py::make_tuple(r[0], r[1]);
  }
  auto [o, final_state, work] = RuleCall(q, k, v, g, beta, initial, offsets, s).forward(false);
  return py::make_tuple(o, final_state);
}

// whether the [K, V] states of a pool [P, Hv, K, V] are apart in memory
bool apart(const Tensor& s) {
  int64_t size = s.size(2) * s.size(3);
  const int a = s.stride(0) <= s.stride(1) ? 0 : 1;
  for (int i : {a, 1 - a}) {
    if (s.size(i) <= 1) continue;
    if (s.stride(i) < size) return false;
    size = s.stride(i) * s.size(i);
  }
  return true;
}

Tensor gated_delta_step(const py::handle& q_, const py::handle& k_, const py::handle& v_, const py::handle& g_, const py::handle& beta_,
                        const py::handle& state_, std::optional<double> scale, const py::handle& slots_) {
  const at::NoGradGuard no_grad;
  Tensor q = tensor(q_, "q"), k = tensor(k_, "k"), v = tensor(v_, "v");
  const Tensor g = tensor(g_, "g"), beta = tensor(beta_, "beta"), state = tensor(state_, "state");
  REQUIRE(!THPVariable_Unpack(state_.ptr()).is_neg(), "state must not be a view that is negated as it is read (it is updated in place)");
  Tensor slots = maybe(slots_, "slots");
  check_rows(q, k, v, g, beta, 1, "batch");
  const int64_t B = q.size(0), Hk = q.size(1), K = q.size(2), Hv = v.size(1), V = v.size(2);
  REQUIRE(state.scalar_type() == at::kFloat && state.dim() == 4 && state.size(1) == Hv && state.size(2) == K && state.size(3) == V,
          "state must be float32 of shape (states, ", Hv, ", ", K, ", ", V, ") (got ", type(state.scalar_type()), ", ", shape(state.sizes()), ")");
  REQUIRE(((V == 1 || state.stride(3) == 1) && (K == 1 || state.stride(2) == V)) || !state.numel(),
          "the last two axes of state must be contiguous (it is updated in place)");
  REQUIRE(apart(state), "the states overlap in memory (an expanded tensor?): they are updated in place");
  if (!slots.defined()) {
    REQUIRE(state.size(0) == B, B, " rows need ", B, " states (got ", state.size(0), "); pass slots for a pool");
  } else {
    REQUIRE((slots.scalar_type() == at::kInt || slots.scalar_type() == at::kLong) && slots.dim() == 1 && slots.size(0) == B,
            "slots must be int32 or int64 of shape (", B, ",) (got ", type(slots.scalar_type()), ", ", shape(slots.sizes()), ")");
    slots = slots.contiguous();
  }
  require_device({{"q", q}, {"k", k}, {"v", v}, {"g", g}, {"beta", beta}, {"state", state}, {"slots", slots}});
  REQUIRE(!state.requires_grad(), "state must not require gradients (it is updated in place, and carries none)");
  q = rows_last(q), k = rows_last(k), v = rows_last(v);
  Tensor o = at::empty({B, Hv, V}, v.options());
  SeqDeltaStep d{};
  d.batch = B, d.pool = state.size(0);
  d.Hk = (int32_t)Hk, d.Hv = (int32_t)Hv, d.K = (int32_t)K, d.V = (int32_t)V;
  d.dtype = dtype_of(q);
  d.slots_64 = slots.defined() && slots.scalar_type() == at::kLong;
  d.scale = (float)scale.value_or(1 / std::sqrt((double)K));
  d.device = q.device().index();
  d.q = data(q), d.k = data(k), d.v = data(v);
  d.g = static_cast<const float*>(data(g)), d.beta = static_cast<const float*>(data(beta));
  for (int i = 0; i < 2; ++i) {
    d.q_stride[i] = q.stride(i), d.k_stride[i] = k.stride(i), d.v_stride[i] = v.stride(i);
    d.g_stride[i] = g.stride(i), d.beta_stride[i] = beta.stride(i), d.state_stride[i] = state.stride(i);
  }
  d.slots = data(slots);
  d.state = state.data_ptr<float>();
  d.o = o.data_ptr();
  state.unsafeGetTensorImpl()->bump_version();   // autograd sees that saved views of it are stale (raises for an inference tensor
                                                 // outside of inference mode, before it is written)
  check(seq_delta_step(&d, stream_of(q)), "gated_delta_step");
  return o;
}

// ------------------------------------------------------------------------------------------------------ gated unit

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct UnitCall {
  Tensor x, wg, wu;
  SeqUnit u{};
  UnitCall(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, int act) : x(rows_last(x_)), wg(rows_last(wg_)), wu(rows_last(wu_)) {
    u.M = x.size(0);
    u.D = (int32_t)x.size(1), u.F = (int32_t)wg.size(1);
    u.act = act, u.dtype = dtype_of(x), u.device = x.device().index();
    u.x = data(x), u.wg = data(wg), u.wu = data(wu);
    u.x_ld = row_stride(x), u.wg_ld = row_stride(wg), u.wu_ld = row_stride(wu);
  }
  Tensor work(bool backward) {
    int64_t need = 0;
    check(seq_unit_workspace(&u, backward, &need), "gated_unit");
    return bytes(need, x);
  }
  std::pair<Tensor, Tensor> forward(bool keep) {
    Tensor y = at::empty({u.M, u.F}, x.options()), pre, w = work(false);
    if (keep) pre = at::empty({2, u.M, u.F}, x.options().dtype(at::kFloat));
    check(seq_unit_forward(&u, w.data_ptr(), w.numel(), y.data_ptr(), keep ? pre.data_ptr<float>() : nullptr, stream_of(x)), "gated_unit");
    return {y, pre};
  }
};

struct UnitFunction : torch::autograd::Function<UnitFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
    auto [y, pre] = UnitCall(x, wg, wu, (int)act).forward(true);
    ctx->save_for_backward({x, wg, wu, pre});
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d_out) {
    const variable_list in = ctx->get_saved_variables();
    check_given(d_out);
    UnitCall call(in[0], in[1], in[2], (int)ctx->saved_data["act"].toInt());
    const Tensor pre = in[3], dy = rows_last(d_out[0].resolve_neg()), w = call.work(true);
    variable_list grads(4);
    if (ctx->needs_input_grad(0)) grads[0] = at::empty(in[0].sizes(), in[0].options());
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2))
      for (int i : {1, 2}) grads[i] = at::empty(in[i].sizes(), in[i].options());
    auto out = [](Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(seq_unit_backward(&call.u, w.data_ptr(), w.numel(), pre.const_data_ptr<float>(), data(dy), row_stride(dy), out(grads[0]),
                            out(grads[1]), out(grads[2]), stream_of(call.x)),
          "gated_unit backward");
    return once(std::move(grads), "gated_unit");
  }
};

Tensor gated_unit(const py::handle& x_, const py::handle& wg_, const py::handle& wu_, const std::string& activation) {
  const Tensor x = tensor(x_, "x"), wg = tensor(wg_, "w_gate"), wu = tensor(wu_, "w_up");
  REQUIRE(dtype_of(x) >= 0, "x must be bfloat16, float16 or float32 (got ", type(x.scalar_type()), ")");
  const int act = activation == "silu" ? SEQ_SILU : activation == "gelu" ? SEQ_GELU : activation == "sigmoid" ? SEQ_SIGMOID : -1;
  REQUIRE(act >= 0, "activation must be one of silu, gelu, sigmoid (got '", activation, "')");
  REQUIRE(x.dim() >= 1, "x must have at least one axis");
  const int64_t D = x.size(-1);
  for (const Named& n : {Named{"w_gate", wg}, Named{"w_up", wu}}) {
    REQUIRE(n.t.scalar_type() == x.scalar_type(), n.name, " must have the type of x, ", type(x.scalar_type()), " (got ", type(n.t.scalar_type()), ")");
    REQUIRE(n.t.dim() == 2 && n.t.size(0) == D, n.name, " must be [", D, ", F] (got ", shape(n.t.sizes()), ")");
  }
  REQUIRE(wg.sizes() == wu.sizes(), "w_gate and w_up differ in shape: ", shape(wg.sizes()), ", ", shape(wu.sizes()));
  const int64_t F = wg.size(1);
  REQUIRE(D >= 1 && D <= SEQ_UNIT_MAX && F >= 1 && F <= SEQ_UNIT_MAX, "weights must be between 1 x 1 and ", SEQ_UNIT_MAX, " x ", SEQ_UNIT_MAX,
          " (got ", D, " x ", F, ")");
  require_device({{"x", x}, {"w_gate", wg}, {"w_up", wu}});
  const Tensor rows = x.dim() == 2 ? x : x.reshape({-1, D});
  Tensor y = wants_grad({x, wg, wu}) ? UnitFunction::apply(rows, wg, wu, (int64_t)act) : UnitCall(rows, wg, wu, act).forward(false).first;
  if (x.dim() == 2) return y;
  std::vector<int64_t> out = x.sizes().vec();
  out.back() = F;
  return y.view(out);
}

// --------------------------------------------------------------------------------------------------------- dropout

Tensor run_dropout(const Tensor& x, const Tensor& residual, int64_t below, int64_t seed, const Tensor& seed_device, int64_t offset) {
  Tensor y = at::empty(x.sizes(), x.options());
  check(seq_dropout(dtype_of(x), data(x), data(residual), y.data_ptr(), x.numel(), (int32_t)below, (uint64_t)seed, (uint64_t)offset,
                    static_cast<const int64_t*>(data(seed_device)), x.device().index(), stream_of(x)),
        "dropout");
  return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual_, int64_t below, int64_t seed,
                        const std::optional<Tensor>& seed_, int64_t offset) {
    const Tensor residual = residual_.value_or(Tensor()), seed_device = seed_.value_or(Tensor());
    ctx->save_for_backward({seed_device});   // an edit between the passes is an error, not another mask
    ctx->saved_data["residual"] = residual.defined();
    ctx->saved_data["below"] = below;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    return run_dropout(x, residual, below, seed, seed_device, offset);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d_out) {
    const variable_list in = ctx->get_saved_variables();
    check_given(d_out);
    variable_list grads(6);
    if (ctx->needs_input_grad(0))
      grads[0] = run_dropout(d_out[0].resolve_neg().contiguous(), Tensor(), ctx->saved_data["below"].toInt(), ctx->saved_data["seed"].toInt(), in[0],
                             ctx->saved_data["offset"].toInt());
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) grads[1] = d_out[0];
    return once(std::move(grads), "dropout");
  }
};

int64_t low64(const py::handle& h, const char* name) {
  py::object i = py::reinterpret_steal<py::object>(PyNumber_Index(h.ptr()));
  if (!i) {
    PyErr_Clear();
    throw py::type_error(say(name, " must be an integer"));
  }
  const unsigned long long v = PyLong_AsUnsignedLongLongMask(i.ptr());
  if (v == (unsigned long long)-1 && PyErr_Occurred()) throw py::error_already_set();
  return (int64_t)v;
}

Tensor dropout(const py::handle& x_, double p, const py::handle& seed_, const py::handle& offset, const py::handle& residual_) {
  Tensor x = tensor(x_, "x"), residual = maybe(residual_, "residual"), seed_device;
  REQUIRE(dtype_of(x) >= 0, "x must be bfloat16, float16 or float32 (got ", type(x.scalar_type()), ")");
  REQUIRE(p >= 0 && p <= 1, "p must be between 0 and 1 (got ", p, ")");
  if (residual.defined())
    REQUIRE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), "residual must be ", type(x.scalar_type()), " of shape ",
            shape(x.sizes()), " (got ", type(residual.scalar_type()), ", ", shape(residual.sizes()), ")");
  int64_t seed = 0;
  if (THPVariable_Check(seed_.ptr())) {
    seed_device = tensor(seed_, "seed");
    REQUIRE(seed_device.scalar_type() == at::kLong && seed_device.numel() == 1, "seed must be an integer or one int64 value (got ",
            type(seed_device.scalar_type()), ", shape ", shape(seed_device.sizes()), ")");
  } else {
    seed = low64(seed_, "seed");
  }
  require_device({{"x", x}, {"residual", residual}, {"seed", seed_device}});
  const int64_t off = low64(offset, "offset");
  x = x.contiguous();
  if (residual.defined()) residual = residual.contiguous();
  const int64_t below = std::lrint(p * 65536);
  if (wants_grad({x, residual})) return DropoutFunction::apply(x, given(residual), below, seed, given(seed_device), off);
  return run_dropout(x, residual, below, seed, seed_device, off);
}

}  // namespace

PYBIND11_MODULE(_seq_torch, m) {
  m.doc() = "Python entry points of libseqops.so";
  const py::object error = py::module_::import("admm_amd._native").attr("AdmmError");
  static PyObject* admm_error = error.inc_ref().ptr();   // for the life of the process
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const SeqError& e) {
      PyErr_SetObject(admm_error, py::reinterpret_borrow<py::object>(admm_error)(e.what(), e.code).ptr());
    }
  });
  m.def("abi_version", &seq_abi_version);
  m.def("gated_delta_rule", &gated_delta_rule);
  m.def("gated_delta_step", &gated_delta_step);
  m.def("gated_unit", &gated_unit);
  m.def("dropout", &dropout);
}
