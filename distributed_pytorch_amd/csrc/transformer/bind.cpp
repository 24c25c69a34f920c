// The transformer-block operators as torch sees them: allocation, launch and autograd nodes in C++.
//
// A training step of a small batch is bound by the host: as Python autograd functions a forward and backward call of one
// of these operators took 120 - 200 us of host time around 25 - 60 us of kernels.  So this module, unlike _C, is built
// against torch's headers.  Arguments are checked here (a few tenths of a microsecond; in Python 3 to 5 of the 7 that a small
// call takes): an operator returns None for what it does not take, and ops/functional.py then says what is wrong.
//
// Outputs and workspaces come from torch's allocator per call and launches go to torch's current stream of the tensors'
// device: nothing is shared between two calls or two graphs, and nothing synchronises with the host.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/TracerMode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "transformer.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace dpa {
namespace {

int code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kHalf: return kF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(), " for HIP kernels");
  }
}
hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
template <typename T> T* data(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }
// a parameter vector as the kernels read it
Tensor vec32(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.detach().to(at::kFloat).contiguous();
}
Tensor floats(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kFloat)); }
bool tracked(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// A tangent would be left out of the results without a word: these operators have no forward-mode derivative.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... Ts> void no_tangents(const char* op, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(ts) || ...), op, ": forward-mode derivatives are not implemented");
}

// Only the allocation of results goes through torch's dispatcher.  Who records a call there (torch.jit.trace, make_fx,
// fake tensors) would hold buffers that nothing fills, and a tensor subclass or wrapper has no memory that a kernel could read.
void not_recorded(const char* op) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK_NOT_IMPLEMENTED(!at::tracer::impl::is_dispatch_enabled(), op, ": cannot be traced");
  if (Modes::any_modes_set())
    TORCH_CHECK_NOT_IMPLEMENTED(!Modes::get_mode(Key::PROXY) && !Modes::get_mode(Key::FAKE) && !Modes::get_mode(Key::FUNCTIONAL),
                                op, ": cannot be traced");
}
bool is_plain(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                         DispatchKey::FuncTorchGradWrapper});
  return !t.defined() || !t.key_set().has_any(wrapped);
}
bool is_plain(const OptTensor& t) { return !t.has_value() || is_plain(*t); }
// in front of everything else that an operator does
template <typename... Ts> void check_call(const char* op, const Ts&... ts) {
  not_recorded(op);
  TORCH_CHECK_NOT_IMPLEMENTED((is_plain(ts) && ...), op, ": tensor subclasses and wrappers are not supported");
  no_tangents(op, ts...);
}

// ---- what ops/functional.py checks, argument by argument
bool float_type(const Tensor& t) {
  const auto d = t.scalar_type();
  return d == at::kFloat || d == at::kBFloat16 || d == at::kHalf;
}
bool rows_taken(const Tensor& x) {
  return float_type(x) && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) * (int64_t)x.element_size() <= 2048 * 16;
}
bool vector_taken(const Tensor& t, const Tensor& x) {
  return t.dim() == 1 && t.size(0) == x.size(-1) && t.device() == x.device();
}
bool norm_taken(const OptTensor& w, const OptTensor& b, int64_t kind, double eps, const Tensor& x) {
  if (!w.has_value()) return kind == kNormNone;
  return (kind == kNormLayer || (kind == kNormRms && !b.has_value())) && vector_taken(*w, x) &&
         (!b.has_value() || vector_taken(*b, x)) && eps >= 0.0;
}

// a gradient of a gradient would silently be missing
void once(const char* op) {
  not_recorded(op);
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the backward pass is not differentiable (create_graph)");
}

// Nodes of the graph are written out like torch's own, not as torch::autograd::Function: that class looks its inputs, outputs
// and saved values up in maps, 4 us a call.  `inputs`: one edge for each argument of the gradient, undefined ones too.
template <typename N, typename... Inputs> std::shared_ptr<N> make_node(const Inputs&... inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}
// A saved value comes back through the hooks that were set when it was saved (torch.autograd.graph.saved_tensors_hooks), which
// may return anything: what a kernel would read past the end of is refused.
void check_kept(const char* op, const Tensor& t, at::ScalarType type, at::IntArrayRef size, const at::Device& device) {
  TORCH_CHECK(t.defined() && is_plain(t) && t.scalar_type() == type && t.sizes() == size && t.device() == device, op,
              ": a saved tensor came back with another type, shape or device");
}
Tensor kept(const char* op, const Tensor& t, at::ScalarType type, at::IntArrayRef size, const at::Device& device) {
  check_kept(op, t, type, size, device);
  return t.contiguous();
}
// gradients of subclasses and wrappers have no memory to read either
template <typename... Ts> void check_grads(const char* op, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED((is_plain(ts) && ...), op, ": gradients that are tensor subclasses or wrappers are not supported");
}
SavedVariable saved(const Tensor& t, bool is_output = false) { return t.defined() ? SavedVariable(t, is_output) : SavedVariable(); }
void has_history(const Tensor& t, const std::shared_ptr<Node>& node) {
  if (t.defined()) torch::autograd::set_history(t, node);
}

// ------------------------------------------------------------------------------------------ residual norm
struct NormCfg {
  int64_t post, pre;                     // NormKind
  double post_eps, pre_eps;
  bool sinks;                            // parameters may have gradient sinks (ops/grad_sink.py)
};
struct RowShape {
  long rows, per_sample;
  int C;
};
RowShape row_shape(const Tensor& x) {
  RowShape r;
  r.C = (int)x.size(-1);
  r.rows = x.numel() / r.C;
  r.per_sample = x.dim() > 1 && x.size(0) > 0 && r.rows > 0 ? r.rows / x.size(0) : 1;      // (a vector is one row, no samples)
  return r;
}
// fp32 copies of post_w, post_b, pre_w, pre_b, gate, scale
using Vecs = std::array<Tensor, 6>;

struct RnOut {
  Tensor s, h, post_stat, pre_stat;
};
RnOut rn_forward(const Tensor& x, const Tensor& y, const Vecs& v, const NormCfg& c, bool want_stats) {
  const c10::DeviceGuard guard(x.device());
  const RowShape r = row_shape(x);
  RnOut o;
  if (y.defined()) o.s = at::empty_like(x);
  if (c.pre != kNormNone) o.h = at::empty_like(x);
  if (want_stats && c.post != kNormNone) o.post_stat = floats({2, r.rows}, x);
  if (want_stats && c.pre != kNormNone) o.pre_stat = floats({2, r.rows}, x);
  ResidualNormFwd p;
  p.x = data<void>(x); p.y = data<void>(y); p.s = data<void>(o.s); p.h = data<void>(o.h);
  p.post_w = data<float>(v[0]); p.post_b = data<float>(v[1]); p.pre_w = data<float>(v[2]); p.pre_b = data<float>(v[3]);
  p.gate = data<float>(v[4]); p.scale = data<float>(v[5]);
  p.post_stat = data<float>(o.post_stat); p.pre_stat = data<float>(o.pre_stat);
  p.rows = r.rows; p.per_sample = r.per_sample; p.C = r.C;
  p.post = (int)c.post; p.pre = (int)c.pre; p.gate_kind = v[4].defined() ? (int)v[4].dim() : kGateNone;
  p.post_eps = (float)c.post_eps; p.pre_eps = (float)c.pre_eps;
  residual_norm_fwd_launch(p, code(x), stream_of(x));
  return o;
}

// A parameter's gradient sink (ops/grad_sink.py), where it has one now: the kernel writes into its view.
struct Sink {
  py::object sink;           // set: the kernel writes here
  Tensor view;
  float beta = 0.f;
  bool late = false;         // the gradient goes through deliver() after the kernel
};
// The sinks of one backward pass, which runs without the GIL: an allocation or a launch that throws ends their life there, and
// only a holder of the GIL may drop what they refer to.
struct Sinks : std::array<Sink, 5> {
  Sinks() = default;
  Sinks(const Sinks&) = delete;
  Sinks& operator=(const Sinks&) = delete;
  ~Sinks() {
    bool held = false;
    for (const Sink& s : *this) held = held || s.sink;
    if (!held) return;
    const py::gil_scoped_acquire gil;
    for (Sink& s : *this) s.sink = py::object();
  }
};
// needs the GIL
void find_sink(const Tensor& param, Sink& out) {
  if (!param.is_leaf()) return;
  py::object p = py::reinterpret_steal<py::object>(THPVariable_Wrap(param));
  if (!py::hasattr(p, "_dpa_sink")) return;
  out.late = true;
  py::object s = py::module_::import("distributed_pytorch_amd.ops.grad_sink").attr("sink_of")(p);
  if (s.is_none()) return;
  out.view = s.attr("view").cast<Tensor>();
  if (!out.view.is_contiguous()) return;
  out.beta = s.attr("beta")().cast<float>();
  out.sink = std::move(s);
}
// through the framework's own delivery (accumulates into a sink, or hands the gradient to autograd); needs the GIL
Tensor deliver(const Tensor& param, const Tensor& grad) {
  py::object p = py::reinterpret_steal<py::object>(THPVariable_Wrap(param));
  py::object g = py::module_::import("distributed_pytorch_amd.ops.hip_ops").attr("_deliver")(p, grad);
  return g.is_none() ? Tensor() : g.cast<Tensor>();
}

struct ResidualNormBackward : Node {
  // y undefined: h = pre(x) alone
  SavedVariable x_, y_, post_stat_, pre_stat_, post_w_, post_b_, pre_w_, pre_b_, gate_, scale_;
  int64_t post = 0, pre = 0;
  bool has_y = false, may_sink = false;

  std::string name() const override { return "ResidualNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x_, &y_, &post_stat_, &pre_stat_, &post_w_, &post_b_, &pre_w_, &pre_b_, &gate_, &scale_}) v->reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    once("residual_norm");
    const std::lock_guard<std::mutex> lock(mutex_);
    std::array<Tensor, 10> sv{x_.unpack(), y_.unpack(), post_stat_.unpack(), pre_stat_.unpack(), post_w_.unpack(),
                                    post_b_.unpack(), pre_w_.unpack(), pre_b_.unpack(), gate_.unpack(), scale_.unpack()};
    const int64_t cfg[4] = {post, pre, has_y, may_sink};
    variable_list got(7);
    Tensor ds = has_y ? grads[0] : Tensor(), dh = has_y ? (grads.size() > 1 ? grads[1] : Tensor()) : grads[0];
    if (!ds.defined() && !dh.defined()) return got;
    check_grads("residual_norm", ds, dh);
    ds = dense(ds);
    dh = dense(dh);
    const Tensor& ref = ds.defined() ? ds : dh;
    const c10::DeviceGuard guard(ref.device());
    {
      const int64_t C = ref.size(-1), stat[2] = {2, ref.numel() / C};
      for (int i = 0; i < 2; ++i)
        if (sv[i].defined()) sv[i] = kept("residual_norm", sv[i], ref.scalar_type(), ref.sizes(), ref.device());
      for (int i = 2; i < 4; ++i)
        if (sv[i].defined()) sv[i] = kept("residual_norm", sv[i], at::kFloat, stat, ref.device());
      const int64_t gate[2] = {ref.size(0), C};
      for (int i = 4; i < 9; ++i) {                 // (vectors of any type, converted below; leaves stay themselves for their sinks)
        if (!sv[i].defined()) continue;
        const bool of_samples = i == 8 && sv[i].dim() == 2;
        check_kept("residual_norm", sv[i], sv[i].scalar_type(), of_samples ? at::IntArrayRef(gate) : at::IntArrayRef(C), ref.device());
      }
      if (sv[9].defined()) sv[9] = kept("residual_norm", sv[9], at::kFloat, ref.size(0), ref.device());
    }
    const Tensor &x = sv[0], &y = sv[1];
    // the caller's parameters in the order of the kernel's sums, and where their gradients go
    const std::array<Tensor, 5> params{sv[6], sv[7], sv[4], sv[5], sv[8]};
    constexpr int place[5] = {4, 5, 2, 3, 6};
    const Vecs v{vec32(sv[4]), vec32(sv[5]), vec32(sv[6]), vec32(sv[7]), vec32(sv[8]), sv[9]};
    const RowShape r = row_shape(ref);
    const int gate_kind = v[4].defined() ? (int)v[4].dim() : kGateNone;
    bool needs[7];
    for (int i = 0; i < 7; ++i) needs[i] = task_should_compute_output(i);
    const bool need_x = needs[0], need_y = needs[1];
    bool need[5], any_leaf = false;
    for (int i = 0; i < 5; ++i) {
      need[i] = needs[place[i]];
      any_leaf = any_leaf || (cfg[3] != 0 && need[i] && params[i].is_leaf());
    }
    // without a norm, gate or scale of its own the block's gradient is that of the sum
    const bool plain = cfg[0] == kNormNone && gate_kind == kGateNone && !v[5].defined();
    const bool branch = !plain && (need_y || need[2] || need[3] || need[4]);
    Tensor dx, dy;
    // without `pre` the sum's gradient is x's as it stands
    const bool same = cfg[1] == kNormNone && ds.defined();
    if (need_x || (need_y && plain)) dx = same ? ds : at::empty_like(ref);
    if (branch) dy = at::empty_like(ref);

    ResidualNormBwd p;
    Tensor own[5];
    Sinks sinks;
    if (any_leaf) {
      const py::gil_scoped_acquire gil;
      for (int i = 0; i < 5; ++i) {
        if (!need[i]) continue;
        find_sink(params[i], sinks[i]);
        if (i == 4 && gate_kind == kGateSample) sinks[i].sink = py::object();      // its sums have a buffer of their own
        for (int j = 0; j < i; ++j)             // a parameter used twice in this call: its second sum has a buffer of its own
          if (sinks[j].sink && sinks[i].sink && sinks[j].sink.is(sinks[i].sink)) sinks[i].sink = py::object();
      }
    }
    bool sums = false;
    for (int i = 0; i < 5; ++i) {
      if (!need[i] || (i == 4 && gate_kind == kGateSample)) continue;
      sums = true;
      if (sinks[i].sink) {
        p.out[i] = sinks[i].view.data_ptr<float>();
        p.beta[i] = sinks[i].beta;
      } else {
        own[i] = floats({r.C}, ref);
        p.out[i] = own[i].data_ptr<float>();
      }
    }
    Tensor partial, gate_partial, dgate;
    const bool gate_sums = gate_kind == kGateSample && need[4];
    if (gate_sums) dgate = floats({ref.size(0), r.C}, ref);
    if (r.rows > 0) {
      p.ds = data<void>(ds); p.dh = data<void>(dh); p.x = data<void>(x); p.y = data<void>(y);
      p.dx = same ? nullptr : data<void>(dx); p.dy = data<void>(dy);
      p.post_w = data<float>(v[0]); p.post_b = data<float>(v[1]); p.pre_w = data<float>(v[2]);
      p.gate = data<float>(v[4]); p.scale = data<float>(v[5]);
      p.post_stat = data<float>(sv[2]); p.pre_stat = data<float>(sv[3]); p.dgate_sample = data<float>(dgate);
      p.rows = r.rows; p.per_sample = r.per_sample; p.C = r.C;
      p.post = (int)cfg[0]; p.pre = (int)cfg[1]; p.gate_kind = gate_kind;
      if (sums || gate_sums) {
        long splits = 1;
        const long parts = residual_norm_parts(p, code(ref), &splits);
        if (sums) partial = floats({parts, 5, r.C}, ref);
        if (gate_sums) gate_partial = floats({ref.size(0) * splits, r.C}, ref);
        p.partial = data<float>(partial); p.gate_partial = data<float>(gate_partial);
      }
      if (p.dx != nullptr || p.dy != nullptr || sums || gate_sums) residual_norm_bwd_launch(p, code(ref), stream_of(ref));
    } else {                                    // no rows: every sum is zero
      for (int i = 0; i < 5; ++i) {
        if (own[i].defined()) own[i].zero_();
        if (sinks[i].sink && sinks[i].beta == 0.f) sinks[i].view.zero_();
      }
      if (dgate.defined()) dgate.zero_();
    }
    if (need_x) got[0] = dx;
    if (need_y) got[1] = plain ? dx : dy;
    for (int i = 0; i < 5; ++i) {
      if (!need[i] || sinks[i].sink) continue;
      const Tensor g = i == 4 && gate_kind == kGateSample ? dgate : own[i];
      got[place[i]] = g.scalar_type() == params[i].scalar_type() ? g : g.to(params[i].scalar_type());
    }
    if (any_leaf) {
      const py::gil_scoped_acquire gil;
      for (Sink& s : sinks)
        if (s.sink) {
          s.sink.attr("delivered")();
          s.sink = py::object();                // (dropped under the GIL)
        }
      for (int i = 0; i < 5; ++i)
        if (sinks[i].late && got[place[i]].defined()) got[place[i]] = deliver(params[i], got[place[i]]);
    }
    return got;
  }
};

// -> (s, h), None where there is none; None for arguments that it does not take
std::optional<std::pair<OptTensor, OptTensor>> residual_norm(const Tensor& x, const OptTensor& y, const OptTensor& post_w,
                                              const OptTensor& post_b, int64_t post, double post_eps, const OptTensor& pre_w,
                                              const OptTensor& pre_b, int64_t pre, double pre_eps, const OptTensor& gate,
                                              const OptTensor& scale, bool sinks) {
  check_call("residual_norm", x, y, post_w, post_b, pre_w, pre_b, gate, scale);
  if (!x.is_cuda() || !rows_taken(x) || !norm_taken(post_w, post_b, post, post_eps, x) || !norm_taken(pre_w, pre_b, pre, pre_eps, x))
    return std::nullopt;
  if (y.has_value()) {
    if (x.dim() < 2 || y->sizes() != x.sizes() || y->scalar_type() != x.scalar_type() || y->device() != x.device()) return std::nullopt;
    if (gate.has_value() &&
        !(vector_taken(*gate, x) || (gate->dim() == 2 && gate->size(0) == x.size(0) && gate->size(1) == x.size(-1) && gate->device() == x.device())))
      return std::nullopt;
    if (scale.has_value() &&
        (scale->dim() != 1 || scale->size(0) != x.size(0) || scale->device() != x.device() || scale->requires_grad()))
      return std::nullopt;
  }
  const Tensor Y = given(y), pw = given(post_w), pb = given(post_b), qw = given(pre_w), qb = given(pre_b), g = given(gate),
               sc = given(scale);
  const NormCfg c{post, pre, post_eps, pre_eps, sinks};
  const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  if (!tracked({x, Y, pw, pb, qw, qb, g})) {
    const RnOut o = rn_forward(x.contiguous(), dense(Y), {vec32(pw), vec32(pb), vec32(qw), vec32(qb), vec32(g), vec32(sc)}, c,
                               false);
    return std::make_pair(opt(o.s), opt(o.h));
  }
  const auto node = make_node<ResidualNormBackward>(x, Y, pw, pb, qw, qb, g);
  RnOut o;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor X = x.contiguous();
    const Tensor y0 = dense(Y);
    const Vecs v{vec32(pw), vec32(pb), vec32(qw), vec32(qb), vec32(g), vec32(sc)};
    o = rn_forward(X, y0, v, c, true);
    const bool has_pre = pre != kNormNone;
    if (has_pre) node->x_ = saved(X);
    if (has_pre || post != kNormNone || g.defined()) node->y_ = saved(y0);
    node->post_stat_ = saved(o.post_stat);
    node->pre_stat_ = saved(o.pre_stat);
    node->post_w_ = saved(pw);
    node->post_b_ = saved(pb);
    node->pre_w_ = saved(qw);
    node->pre_b_ = saved(qb);
    node->gate_ = saved(g);
    node->scale_ = saved(v[5]);
    node->post = post;
    node->pre = pre;
    node->has_y = Y.defined();
    node->may_sink = sinks;
  }
  has_history(o.s, node);
  has_history(o.h, node);
  return std::make_pair(opt(o.s), opt(o.h));
}

// ------------------------------------------------------------------------------------------ rotary
void rotary_run(const Tensor& src, const Tensor& out, const Tensor& pos, const Tensor& freqs, const Tensor& axis, int64_t heads,
                bool interleaved, bool negate) {
  const c10::DeviceGuard guard(src.device());
  RotaryParams p;
  p.in = src.data_ptr(); p.out = out.data_ptr(); p.pos = pos.data_ptr(); p.freq = freqs.data_ptr();
  p.axis = axis.data_ptr<int>();
  p.S = std::max<int64_t>(src.size(1), 1);
  p.tokens = src.size(0) * src.size(1);
  p.in_batch = src.stride(0); p.in_token = src.stride(1); p.out_batch = out.stride(0); p.out_token = out.stride(1);
  p.H = (int)heads; p.D = (int)(src.size(2) / (3 * heads)); p.pairs = (int)freqs.numel(); p.axes = (int)pos.size(-1);
  p.pos_kind = pos.scalar_type() == at::kLong ? kPosI64
               : pos.scalar_type() == at::kInt ? kPosI32 : pos.scalar_type() == at::kFloat ? kPosF32 : kPosF64;
  p.pos_batched = pos.dim() == 3; p.freq_f64 = freqs.scalar_type() == at::kDouble;
  p.interleaved = interleaved; p.negate = negate;
  rotary_launch(p, code(src), stream_of(src));
}
Tensor token_dense(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor rotary_new(const Tensor& t, const Tensor& pos, const Tensor& freqs, const Tensor& axis, int64_t heads, bool interleaved,
                  bool negate) {
  const Tensor src = token_dense(t);
  const Tensor out = at::empty(src.sizes(), src.options());
  rotary_run(src, out, pos, freqs, axis, heads, interleaved, negate);
  return out;
}

struct RotaryBackward : Node {
  SavedVariable pos_, freqs_, axis_;
  int64_t heads = 0, pairs = 0;
  bool interleaved = false;
  at::ScalarType pos_type = at::kLong, freqs_type = at::kDouble;
  c10::SmallVector<int64_t, 3> pos_size;

  std::string name() const override { return "RotaryBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&pos_, &freqs_, &axis_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    once("rotary");
    const std::lock_guard<std::mutex> lock(mutex_);
    variable_list got(1);
    if (!grads[0].defined()) return got;
    check_grads("rotary", grads[0]);
    Tensor pos = pos_.unpack(), freqs = freqs_.unpack(), axis = axis_.unpack();
    pos = kept("rotary", pos, pos_type, pos_size, grads[0].device());
    freqs = kept("rotary", freqs, freqs_type, pairs, grads[0].device());
    axis = kept("rotary", axis, at::kInt, pairs, grads[0].device());
    got[0] = rotary_new(grads[0], pos, freqs, axis, heads, interleaved, true);
    return got;
  }
};

bool rotary_taken(const Tensor& qkv, const Tensor& pos, const Tensor& freqs, const Tensor& axis, int64_t heads) {
  if (!qkv.is_cuda() || !float_type(qkv) || qkv.dim() != 3 || heads < 1 || qkv.size(2) == 0 || qkv.size(2) % (3 * heads) != 0)
    return false;
  const int64_t d = pos.dim();
  if ((d != 2 && d != 3) || pos.size(d - 2) != qkv.size(1) || (d == 3 && pos.size(0) != qkv.size(0)) || pos.size(d - 1) < 1)
    return false;
  const auto pt = pos.scalar_type(), ft = freqs.scalar_type(), at = axis.scalar_type();
  if ((pt != at::kLong && pt != at::kInt && pt != at::kFloat && pt != at::kDouble) || (ft != at::kFloat && ft != at::kDouble) ||
      (at != at::kInt && at != at::kLong))
    return false;
  return freqs.dim() == 1 && axis.sizes() == freqs.sizes() && 2 * freqs.numel() <= qkv.size(2) / (3 * heads) &&
         freqs.numel() <= 4096 && pos.device() == qkv.device() && freqs.device() == qkv.device() &&
         axis.device() == qkv.device() && !pos.requires_grad() && !freqs.requires_grad();
}
// (`inplace`: its strides have been checked)
OptTensor rotary(const Tensor& qkv, const Tensor& positions, const Tensor& freqs, const Tensor& axis, int64_t heads,
                 bool interleaved, bool inplace) {
  check_call("rotary", qkv, positions, freqs, axis);
  if (!rotary_taken(qkv, positions, freqs, axis, heads)) return std::nullopt;
  const Tensor pos = positions.contiguous(), f = freqs.contiguous();
  // (clamped first: an entry of 2^32 would become 0)
  const Tensor a = (axis.scalar_type() == at::kLong ? axis.clamp(-1, positions.size(-1)) : axis).to(at::kInt).contiguous();
  if (inplace) {
    qkv.unsafeGetTensorImpl()->bump_version();      // (raises for an inference tensor outside inference mode)
    rotary_run(qkv, qkv, pos, f, a, heads, interleaved, false);
    return qkv;
  }
  if (!tracked({qkv})) return rotary_new(qkv, pos, f, a, heads, interleaved, false);
  const auto node = make_node<RotaryBackward>(qkv);
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = rotary_new(qkv, pos, f, a, heads, interleaved, false);
    node->pos_ = saved(pos);
    node->freqs_ = saved(f);
    node->axis_ = saved(a);
    node->heads = heads;
    node->interleaved = interleaved;
    node->pairs = f.numel();
    node->pos_type = pos.scalar_type();
    node->freqs_type = f.scalar_type();
    node->pos_size.assign(pos.sizes().begin(), pos.sizes().end());
  }
  has_history(out, node);
  return out;
}

// ------------------------------------------------------------------------------------------ log probabilities
struct LpOut {
  Tensor lp, ent, top, idx, norm;
};
LpOut lp_forward(const Tensor& z, const Tensor& t, int64_t k) {
  const c10::DeviceGuard guard(z.device());
  const int64_t N = z.size(0), V = z.size(1);
  LpOut o{floats({N}, z), floats({N}, z), floats({N, k}, z), at::empty({N, k}, t.options()), floats({N, 2}, z)};
  TokenLogprobs p;
  p.logits = z.data_ptr(); p.target = t.data_ptr<int64_t>();
  p.N = N; p.C = V; p.ld = z.stride(0); p.k = (int)k;
  p.splits = token_logprobs_splits(N, V);
  Tensor stat, keys;
  if (p.splits > 1) {
    stat = floats({N, p.splits, 3}, z);
    keys = at::empty({N, p.splits, k}, t.options());
  }
  p.logprob = o.lp.data_ptr<float>(); p.entropy = o.ent.data_ptr<float>(); p.norm = o.norm.data_ptr<float>();
  p.top = o.top.data_ptr<float>(); p.index = o.idx.data_ptr<int64_t>();
  p.stat = data<float>(stat); p.keys = data<uint64_t>(keys);
  token_logprobs_launch(p, code(z), stream_of(z));
  return o;
}

struct TokenLogprobsBackward : Node {
  SavedVariable logits_, target_, norm_, entropy_, index_;
  int64_t k = 0, rows = 0, classes = 0;
  at::ScalarType type = at::kFloat;
  at::Device device = at::kCPU;

  std::string name() const override { return "TokenLogprobsBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&logits_, &target_, &norm_, &entropy_, &index_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    once("token_logprobs");
    const std::lock_guard<std::mutex> lock(mutex_);
    variable_list got(1);
    std::array<Tensor, 5> sv{logits_.unpack(), target_.unpack(), norm_.unpack(), entropy_.unpack(shared_from_this()),
                                   index_.unpack()};
    Tensor g[3];
    bool any = false;
    for (int i = 0; i < 3; ++i) {
      if (grads[i].defined()) g[i] = vec32(grads[i]);
      any = any || g[i].defined();
    }
    if (!any) return got;
    check_grads("token_logprobs", grads[0], grads[1], grads[2]);
    const c10::DeviceGuard guard(device);
    check_kept("token_logprobs", sv[0], type, {rows, classes}, device);
    if (sv[0].stride(1) != 1) sv[0] = sv[0].contiguous();
    sv[1] = kept("token_logprobs", sv[1], at::kLong, rows, device);
    sv[2] = kept("token_logprobs", sv[2], at::kFloat, {rows, 2}, device);
    sv[3] = kept("token_logprobs", sv[3], at::kFloat, rows, device);
    sv[4] = kept("token_logprobs", sv[4], at::kLong, {rows, k}, device);
    const Tensor& z = sv[0];
    const Tensor dz = at::empty(z.sizes(), z.options());
    TokenLogprobsBwd p;
    p.logits = z.data_ptr(); p.target = sv[1].data_ptr<int64_t>(); p.norm = sv[2].data_ptr<float>();
    p.entropy = sv[3].data_ptr<float>(); p.index = sv[4].data_ptr<int64_t>();
    p.d_logprob = data<float>(g[0]); p.d_entropy = data<float>(g[1]); p.d_top = data<float>(g[2]);
    p.dlogits = dz.data_ptr();
    p.N = z.size(0); p.C = z.size(1); p.ld = z.stride(0); p.k = (int)k;
    token_logprobs_bwd_launch(p, code(z), stream_of(z));
    got[0] = dz;
    return got;
  }
};

// logits [N, V]
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> token_logprobs(const Tensor& logits, const Tensor& target, int64_t k) {
  check_call("token_logprobs", logits, target);
  const auto type = target.scalar_type();
  if (!logits.is_cuda() || !float_type(logits) || logits.dim() != 2 || logits.size(1) < 1 || logits.size(1) > 1l << 30 ||
      target.dim() != 1 || target.size(0) != logits.size(0) || target.device() != logits.device() ||
      (type != at::kLong && type != at::kInt && type != at::kShort && type != at::kByte) || k < 0 || k > 64 || k > logits.size(1))
    return std::nullopt;
  const Tensor t = target.to(at::kLong).contiguous();
  if (!tracked({logits})) {
    const LpOut o = lp_forward(logits.stride(1) == 1 ? logits : logits.contiguous(), t, k);
    return std::make_tuple(o.lp, o.ent, o.top, o.idx);
  }
  const auto node = make_node<TokenLogprobsBackward>(logits);
  LpOut o;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor z = logits.stride(1) == 1 ? logits : logits.contiguous();
    o = lp_forward(z, t, k);
    node->logits_ = saved(z);
    node->target_ = saved(t);
    node->norm_ = saved(o.norm);
    node->index_ = saved(o.idx);
    node->k = k;
    node->rows = z.size(0);
    node->classes = z.size(1);
    node->type = z.scalar_type();
    node->device = z.device();
  }
  for (const Tensor& out : {o.lp, o.ent, o.top}) has_history(out, node);
  node->entropy_ = saved(o.ent, true);
  return std::make_tuple(o.lp, o.ent, o.top, o.idx);
}

// ------------------------------------------------------------------------------------------ Newton-Schulz and Muon
// out may be g itself (contiguous then)
Tensor newton_schulz(const Tensor& g0, const OptTensor& into, int64_t steps, double a, double b, double c, double eps, bool fast) {
  check_call("newton_schulz", g0);
  const Tensor g = g0.contiguous();
  const c10::DeviceGuard guard(g.device());
  const Tensor out = into.has_value() ? *into : at::empty_like(g);
  NewtonSchulz p;
  p.rows = g.size(-2); p.cols = g.size(-1); p.batch = g.numel() / (p.rows * p.cols);
  const Tensor work = at::empty({(int64_t)newton_schulz_workspace(p.batch, p.rows, p.cols)}, g.options().dtype(at::kByte));
  p.g = g.data_ptr(); p.out = out.data_ptr(); p.work = work.data_ptr();
  p.steps = (int)steps; p.a = (float)a; p.b = (float)b; p.c = (float)c; p.eps = eps; p.fast = fast;
  newton_schulz_launch(p, code(g), stream_of(g));
  return out;
}

void muon_begin(const Tensor& table, int n, long chunks, int g_dtype, const Tensor& hyper, const OptTensor& inv_scale,
                const OptTensor& found_inf, const Tensor& update) {
  const c10::DeviceGuard guard(update.device());
  muon_begin_launch(reinterpret_cast<const MuonTensor*>(table.data_ptr()), n, chunks, g_dtype, hyper.data_ptr<float>(),
                    data<float>(given(inv_scale)), data<float>(given(found_inf)), update.data_ptr<float>(), stream_of(update));
}
void muon_end(const Tensor& table, int n, long chunks, int lp_dtype, const Tensor& hyper, const OptTensor& found_inf,
              const Tensor& update) {
  const c10::DeviceGuard guard(update.device());
  muon_end_launch(reinterpret_cast<const MuonTensor*>(table.data_ptr()), n, chunks, lp_dtype, hyper.data_ptr<float>(),
                  data<float>(given(found_inf)), update.data_ptr<float>(), stream_of(update));
}

}  // namespace
}  // namespace dpa

PYBIND11_MODULE(_T, m) {
  m.doc() = "distributed_pytorch_amd transformer-block operators (gfx950 / MI355X)";
  m.def("residual_norm", &dpa::residual_norm);
  m.def("rotary", &dpa::rotary);
  m.def("token_logprobs", &dpa::token_logprobs);
  m.def("newton_schulz", &dpa::newton_schulz);
  m.def("muon_chunk_elems", &dpa::muon_chunk_elems);
  m.def("muon_table_entry_bytes", []() { return sizeof(dpa::MuonTensor); });
  m.def("muon_begin", &dpa::muon_begin);
  m.def("muon_end", &dpa::muon_end);
}
