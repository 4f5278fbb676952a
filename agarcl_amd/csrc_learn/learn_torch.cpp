// learn_torch.cpp -- the module agarcl_amd._learn: torch tensors in and out of the C ABI of include/agarcl_learn.h (host code only; agarcl_amd/learn.py documents
// the functions and gives them their keywords).  It checks the arguments, makes the outputs and the scratch memory, and holds the two autograd functions.
// In C++ because these calls sit between two steps of the env: checks, structures, and above all a backward pass that would have to take Python's lock in autograd's own thread took
// 23-155 us of host time per call from Python, a multiple of the kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <string>
#include <unordered_set>

#include "../../include/agarcl_learn.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Failure : std::runtime_error { int code; std::string text; Failure(int c, const std::string &t) : std::runtime_error("agarcl error " + std::to_string(c) + ": " + t), code(c), text(t) {} };      // -> AgarclError
[[noreturn]] void refuse(const std::string &m) { throw py::value_error(m); }
void done(int rc) {
  if (rc != 0) throw Failure(rc, agarcl_learn_error());      // (out of a backward pass it comes as the RuntimeError that it is)
}

// ---- arguments ------------------------------------------------------------------------------------------------------------------------------
std::string shape_text(at::IntArrayRef s) { std::string t = "("; for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]); return t + (s.size() == 1 ? ",)" : ")"); }
// t with its numbers in memory as they are: a view that negates when it is read lies there with the other sign, and torch's zeros without storage have a null address, which
// says "none" to the C ABI
Tensor stored(const Tensor &t) { return !t.defined() ? t : t._is_zerotensor() ? t.clone() : t.resolve_neg(); }
Tensor taken(py::handle h, const char *name) {
  const Tensor &t = THPVariable_Unpack(h.ptr());
  if (t._fw_grad(0).defined()) refuse(std::string(name) + " carries a forward-mode gradient: there are none through these operators");      // (better said than lost)
  return stored(t);
}
Tensor optional(py::handle h, const char *name) {      // undefined for None
  if (h.is_none()) return {};
  if (!THPVariable_Check(h.ptr())) refuse(std::string(name) + " must be a tensor");
  return taken(h, name);
}
Tensor needed(py::handle h, const char *name) { Tensor t = optional(h, name); if (!t.defined()) refuse(std::string(name) + " must be a tensor"); return t; }

int type_code(at::ScalarType t) { return t == at::kFloat ? AGARCL_F32 : t == at::kBFloat16 ? AGARCL_BF16 : t == at::kHalf ? AGARCL_F16 : -1; }
Tensor first(py::handle h, const char *name) {      // the tensor that says type and device for the others
  if (!THPVariable_Check(h.ptr()) || type_code(THPVariable_Unpack(h.ptr()).scalar_type()) < 0) refuse(std::string(name) + " must be a float32, bfloat16 or float16 tensor");
  return taken(h, name);
}
void like(const Tensor &t, const char *name, const Tensor &ref, at::ArrayRef<at::ScalarType> types, at::IntArrayRef shape) {
  if (t.device() != ref.device()) refuse(std::string(name) + " must live on " + ref.device().str());
  bool ok = false;
  for (auto k : types) ok = ok || t.scalar_type() == k;
  if (!ok) { std::string m; for (auto k : types) m += (m.empty() ? "" : " or ") + std::string(c10::toString(k)); refuse(std::string(name) + " must be " + m + ", got " + c10::toString(t.scalar_type())); }
  if (t.sizes() != shape) refuse(std::string(name) + " must have shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
}
const std::vector<at::ScalarType> F32 = {at::kFloat}, FLAGS = {at::kBool, at::kByte}, INTS = {at::kInt, at::kLong}, WEIGHTS = {at::kFloat, at::kBool};
void constant(std::initializer_list<std::pair<const char *, const Tensor *>> all) {      // gradients do not flow through these: better said than lost
  if (!at::GradMode::is_enabled()) return;
  for (auto &p : all) if (p.second->defined() && p.second->requires_grad()) refuse(std::string(p.first) + " is taken as a constant here: detach() it, or call under torch.no_grad()");
}
void on_gpu(const Tensor &t) { if (!t.is_cuda()) refuse("tensors must live on a GPU (there is no CPU path)"); }      // (the last of the checks)
void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
bool capturing(const Tensor &t) {
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing((hipStream_t)stream_of(t), &s) != hipSuccess) { (void)hipGetLastError(); return true; }      // (it cannot be asked now: the careful answer)
  return s != hipStreamCaptureStatusNone;
}
// A captured backward pass may not reach a node that another stream made: autograd would have that stream wait for the captured one, which ends the capture and
// with it the process.  That is so for a leaf whose eager graph still lives, since a leaf has one node for all its graphs.
void capture_reaches(const Tensor &ref, std::initializer_list<const Tensor *> inputs) {
  if (!capturing(ref)) return;
  const auto here = c10::hip::getCurrentHIPStream(ref.get_device()).unwrap().id();
  std::vector<std::shared_ptr<torch::autograd::Node>> nodes;
  std::unordered_set<torch::autograd::Node *> seen;
  const auto look = [&](const std::shared_ptr<torch::autograd::Node> &n) { if (n && seen.insert(n.get()).second) nodes.push_back(n); };
  for (const Tensor *t : inputs) if (t->defined() && t->requires_grad()) look(t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t));
  for (size_t i = 0; i < nodes.size(); ++i) {
    const auto s = nodes[i]->stream();
    if (s && s->id() != here) refuse("a graph that was made on another stream still holds a node of an input: drop it (its loss, its outputs) before the capture, and capture forward and backward together");
    for (const auto &e : nodes[i]->next_edges()) { const auto next = e.function; look(next); }
  }
}
int64_t product(at::IntArrayRef s) { int64_t n = 1; for (auto k : s) n *= k; return n; }
const void *ptr(const Tensor &t) {
  if (!t.defined()) return nullptr;
  const void *p = t.const_data_ptr();
  if (!p && t.numel()) refuse("a tensor without memory of its own (a wrapper's, a fake one)");      // (null says "none" to the C ABI)
  return p;
}
void *out(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor make(at::IntArrayRef shape, at::ScalarType type, const Tensor &ref) { return at::detail::empty_cuda(shape, type, ref.device(), std::nullopt); }      // (at::empty takes a microsecond)
// a tensor of its own on a part of another's memory, `at` elements behind its beginning and of its type: an allocation and its share of the host's time less
Tensor part(const Tensor &of, int64_t at, at::IntArrayRef shape) {
  auto t = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(of.storage()), of.key_set(), of.dtype());
  t->set_storage_offset(at);
  t->set_sizes_contiguous(shape);
  return Tensor(std::move(t));
}
Tensor floats(at::IntArrayRef shape, const Tensor &ref) { return make(shape, at::kFloat, ref); }
Tensor scratch(int64_t n, const Tensor &ref) { if (n < 0) refuse("sizes out of range"); return n ? floats({n}, ref) : Tensor(); }

// a tensor with every t[i] contiguous, and the elements from one index of the first axis to the next; a copy only where it has to be one
struct Strided { Tensor t; int64_t stride = 0; };
Strided steps(const Tensor &t) {
  if (!t.defined()) return {};
  const int64_t n = t.size(0), each = n ? t.numel() / n : 0;
  if (t.is_contiguous()) return {t, each};
  if (n && t.stride(0) >= each) {
    bool ok = true;
    int64_t want = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) { if (t.size(d) != 1 && t.stride(d) != want) ok = false; want *= t.size(d); }
    if (ok) return {t, t.stride(0)};
  }
  return {t.contiguous(), each};
}
// the same for [*rows, width] seen as rows
Strided rows_of(const Tensor &t) {
  if (!t.defined()) return {};
  const int64_t width = t.size(-1);
  if (!t.is_contiguous() && t.dim() == 2 && (width == 1 || t.stride(1) == 1) && t.stride(0) >= width) return {t, t.stride(0)};
  return {t.contiguous(), width};
}
Tensor whole(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// ---- the memory -------------------------------------------------------------------------------------------------------------------------------
agarcl_recurrence_args recurrence_args(const Tensor &ref, at::IntArrayRef shape, const Strided &x, const Strided &gate, const Strided &reset) {
  agarcl_recurrence_args a = {};
  a.steps = shape[0]; a.rows = product(shape.slice(1, shape.size() - 2)); a.width = shape.back();
  a.dtype = type_code(ref.scalar_type()); a.device = ref.get_device();
  a.x = ptr(x.t); a.gate = ptr(gate.t); a.x_stride = x.stride; a.gate_stride = gate.stride;
  a.reset = (const uint8_t *)ptr(reset.t); a.reset_stride = reset.stride; a.stream = stream_of(ref);
  return a;
}
struct Remembered { Tensor h, last, marks; };
Remembered recurrence_forward(const Tensor &x, const Tensor &gate, const Tensor &state, const Tensor &reset, bool marked) {
  const Strided xs = steps(x), gs = steps(gate), rs = steps(reset);
  const Tensor s = whole(state);
  agarcl_recurrence_args a = recurrence_args(x, x.sizes(), xs, gs, rs);
  const auto rest = x.sizes().slice(1);
  Remembered r{make(x.sizes(), x.scalar_type(), x), floats(rest, x), {}};
  if (marked) { std::vector<int64_t> m(x.sizes().begin(), x.sizes().end()); m[0] = (m[0] + AGARCL_MARK_STEPS - 1) / AGARCL_MARK_STEPS; r.marks = floats(m, x); }
  const Tensor work = scratch(agarcl_recurrence_work(a.steps, a.rows, a.width), x);
  a.state = (const float *)ptr(s); a.h = out(r.h); a.last = (float *)out(r.last); a.marks = (float *)out(r.marks); a.work = (float *)out(work);
  done(agarcl_recurrence(&a));
  return r;
}

void no_second_gradient() { if (at::GradMode::is_enabled()) throw std::runtime_error("agarcl_amd.learn has no gradients of gradients: call backward() / grad() without create_graph"); }

// A node of autograd's graph: what a backward pass reads is kept as SavedVariables, which notice a tensor that has been written since.
struct RecurrenceNode : torch::autograd::Node {
  SavedVariable x_, gate_, reset_, marks_;
  void keep(const Tensor &x, const Tensor &gate, const Tensor &reset, const Tensor &marks) {
    x_ = SavedVariable(x, false); gate_ = SavedVariable(gate, false); reset_ = SavedVariable(reset, false); marks_ = SavedVariable(marks, false);
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data(); gate_.reset_data(); reset_.reset_data(); marks_.reset_data();
  }
  variable_list apply(variable_list &&up) override {
    std::lock_guard<std::mutex> lock(mutex_);
    no_second_gradient();
    if (!up[0].defined() && !up[1].defined()) return variable_list(3);
    const Tensor x = x_.unpack(), gate = gate_.unpack(), reset = reset_.unpack(), marks = marks_.unpack();
    const Strided xs = steps(x), gs = steps(gate), rs = steps(reset), ds = steps(stored(up[0]));
    const Tensor dlast = whole(stored(up[1]));
    agarcl_recurrence_args a = recurrence_args(x, x.sizes(), xs, gs, rs);
    Tensor dx = make(x.sizes(), x.scalar_type(), x), dgate = make(x.sizes(), x.scalar_type(), x), dstate = floats(x.sizes().slice(1), x);
    const Tensor work = scratch(agarcl_recurrence_work(a.steps, a.rows, a.width), x);
    a.marks = (float *)out(marks); a.dh = ptr(ds.t); a.dh_stride = ds.stride; a.dlast = (const float *)ptr(dlast);
    a.dx = out(dx); a.dgate = out(dgate); a.dstate = (float *)out(dstate); a.work = (float *)out(work);
    done(agarcl_recurrence_grad(&a));
    const auto wanted = [&](size_t i, Tensor &t) { return task_should_compute_output(i) ? t : Tensor(); };
    return {wanted(0, dx), wanted(1, dgate), wanted(2, dstate)};
  }
};

py::tuple gated_recurrence(py::handle hx, py::handle hgate, py::handle hstate, py::handle hreset) {
  const Tensor x = first(hx, "x");
  if (x.dim() < 2) refuse("x must have shape [T, *rows, C], got " + shape_text(x.sizes()));
  const Tensor gate = needed(hgate, "gate"), state = optional(hstate, "state"), reset = optional(hreset, "reset");
  like(gate, "gate", x, {x.scalar_type()}, x.sizes());
  if (state.defined()) like(state, "state", x, F32, x.sizes().slice(1));
  if (reset.defined()) like(reset, "reset", x, FLAGS, x.sizes().slice(0, x.dim() - 1));
  on_gpu(x);
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (state.defined() && state.requires_grad()))) {
    capture_reaches(x, {&x, &gate, &state});
    auto node = std::shared_ptr<RecurrenceNode>(new RecurrenceNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, gate, state));
    Remembered r;
    {
      at::NoGradGuard off;
      r = recurrence_forward(x, gate, state, reset, true);
    }
    node->keep(x, gate, reset, r.marks);
    torch::autograd::set_history(r.h, node);
    torch::autograd::set_history(r.last, node);
    return py::make_tuple(r.h, r.last);
  }
  Remembered r = recurrence_forward(x, gate, state, reset, false);
  return py::make_tuple(r.h, r.last);
}

py::tuple recurrence_step(py::handle hx, py::handle hgate, py::handle hstate, py::handle hreset) {
  const Tensor x = first(hx, "x");
  if (x.dim() < 1) refuse("x must have shape [*rows, C]");
  const Tensor gate = needed(hgate, "gate"), state = needed(hstate, "state"), reset = optional(hreset, "reset");
  constant({{"x", &x}, {"gate", &gate}, {"state", &state}});
  like(gate, "gate", x, {x.scalar_type()}, x.sizes());
  like(state, "state", x, F32, x.sizes());
  if (reset.defined()) like(reset, "reset", x, FLAGS, x.sizes().slice(0, x.dim() - 1));
  on_gpu(x);
  const Tensor xc = x.contiguous(), gc = gate.contiguous(), sc = state.contiguous(), rc = whole(reset);
  agarcl_recurrence_args a = {};
  a.steps = 1; a.width = x.size(-1); a.rows = product(x.sizes().slice(0, x.dim() - 1)); a.dtype = type_code(x.scalar_type()); a.device = x.get_device();
  a.x = ptr(xc); a.gate = ptr(gc); a.x_stride = a.gate_stride = x.numel(); a.state = (const float *)ptr(sc); a.reset = (const uint8_t *)ptr(rc); a.reset_stride = a.rows;
  const Tensor h = make(x.sizes(), x.scalar_type(), x), last = floats(x.sizes(), x), work = scratch(agarcl_recurrence_work(1, a.rows, a.width), x);
  a.h = out(h); a.last = (float *)out(last); a.work = (float *)out(work); a.stream = stream_of(x);
  done(agarcl_recurrence(&a));
  return py::make_tuple(h, last);
}

// ---- the rollout ------------------------------------------------------------------------------------------------------------------------------
py::tuple advantages(py::handle hreward, py::handle hvalue, py::handle hnext, py::handle hterm, py::handle htrunc, py::handle hfinal, double gamma, double lam) {
  const Tensor value = first(hvalue, "value");
  if (value.dim() < 1) refuse("value must have shape [T, *rows]");
  const Tensor reward = needed(hreward, "reward"), next = needed(hnext, "next_value"), term = needed(hterm, "terminated"), trunc = optional(htrunc, "truncated"),
               final_value = optional(hfinal, "final_value");
  constant({{"reward", &reward}, {"value", &value}, {"next_value", &next}, {"final_value", &final_value}});
  like(reward, "reward", value, F32, value.sizes());
  like(next, "next_value", value, {value.scalar_type()}, value.sizes().slice(1));
  like(term, "terminated", value, FLAGS, value.sizes());
  if (trunc.defined()) like(trunc, "truncated", value, FLAGS, value.sizes());
  if (final_value.defined()) {
    if (!trunc.defined()) refuse("final_value without truncated");
    like(final_value, "final_value", value, {value.scalar_type()}, value.sizes());
  }
  if (!(gamma >= 0 && gamma <= 1 && lam >= 0 && lam <= 1)) refuse("gamma and lam must be in [0, 1]");
  on_gpu(value);
  const Strided r = steps(reward), v = steps(value), e = steps(term), u = steps(trunc), f = steps(final_value);
  const Tensor n = whole(next);
  agarcl_advantages_args a = {};
  a.steps = value.size(0); a.rows = product(value.sizes().slice(1)); a.dtype = type_code(value.scalar_type()); a.device = value.get_device();
  a.reward = (const float *)ptr(r.t); a.value = ptr(v.t); a.next_value = ptr(n); a.terminated = (const uint8_t *)ptr(e.t); a.truncated = (const uint8_t *)ptr(u.t); a.final_value = ptr(f.t);
  a.reward_stride = r.stride; a.value_stride = v.stride; a.terminated_stride = e.stride; a.truncated_stride = u.stride; a.final_stride = f.stride;
  a.gamma = (float)gamma; a.lambda = (float)lam;
  const Tensor adv = floats(value.sizes(), value), ret = floats(value.sizes(), value), work = scratch(agarcl_advantages_work(a.steps, a.rows), value);
  a.advantage = (float *)out(adv); a.returns = (float *)out(ret); a.work = (float *)out(work); a.stream = stream_of(value);
  done(agarcl_advantages(&a));
  return py::make_tuple(adv, ret);
}

// ---- the policy -------------------------------------------------------------------------------------------------------------------------------
// the checks that acting and training share; whether log_std has a row's stride
int policy_checks(const Tensor &logits, const Tensor &mean, py::handle hstd, const Tensor &allowed, Tensor &log_std) {
  if (logits.dim() < 1 || logits.size(-1) < 1) refuse("logits must have shape [*rows, kinds] with at least one kind, got " + shape_text(logits.sizes()));
  if (allowed.defined()) like(allowed, "allowed", logits, FLAGS, logits.sizes());
  if (mean.defined() == hstd.is_none()) refuse("mean and log_std belong together");
  if (!mean.defined()) return 0;
  std::vector<int64_t> two(logits.sizes().begin(), logits.sizes().end());
  two.back() = 2;
  like(mean, "mean", logits, {logits.scalar_type()}, two);
  log_std = needed(hstd, "log_std");
  if (log_std.dim() == 1 && log_std.size(0) == 2 && log_std.scalar_type() == at::kFloat && (two.size() > 1 || logits.scalar_type() != at::kFloat)) {
    like(log_std, "log_std", logits, F32, {2});
    return 0;
  }
  like(log_std, "log_std (float32 [2], or per row)", logits, {logits.scalar_type()}, two);
  return 1;
}

py::tuple sample_actions(py::handle hlogits, py::handle hmean, py::handle hstd, py::handle hgumbel, py::handle hnormal, py::handle hallowed) {
  const Tensor logits = first(hlogits, "logits"), mean = optional(hmean, "mean"), gumbel = optional(hgumbel, "gumbel"), normal = optional(hnormal, "normal"), allowed = optional(hallowed, "allowed");
  constant({{"logits", &logits}, {"mean", &mean}, {"gumbel", &gumbel}, {"normal", &normal}});
  Tensor log_std;
  const int per_row = policy_checks(logits, mean, hstd, allowed, log_std);
  constant({{"log_std", &log_std}});
  if (gumbel.defined()) like(gumbel, "gumbel", logits, F32, logits.sizes());
  if (normal.defined()) {
    if (!mean.defined()) refuse("normal without mean");
    like(normal, "normal", logits, F32, mean.sizes());
  }
  on_gpu(logits);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const Strided z = rows_of(logits), k = rows_of(allowed), g = rows_of(gumbel);
  const Tensor m = whole(mean), s = whole(log_std), n = whole(normal);
  agarcl_sample_args a = {};
  a.rows = product(lead); a.kinds = logits.size(-1); a.dtype = type_code(logits.scalar_type()); a.device = logits.get_device();
  a.logits = ptr(z.t); a.logits_stride = z.stride; a.allowed = (const uint8_t *)ptr(k.t); a.allowed_stride = k.stride; a.gumbel = (const float *)ptr(g.t); a.gumbel_stride = g.stride;
  a.mean = ptr(m); a.log_std = ptr(s); a.log_std_per_row = per_row; a.normal = (const float *)ptr(n);
  const int64_t moves = mean.defined() ? 2 * a.rows : 0;
  // (kind has an allocation of its own: torch does not save or copy tensors together that share their memory and differ in type)
  const Tensor all = floats({2 * moves + a.rows}, logits), kind = make(lead, at::kInt, logits), log_prob = part(all, 2 * moves, lead);
  Tensor raw, move;
  if (mean.defined()) { raw = part(all, 0, mean.sizes()); move = part(all, moves, mean.sizes()); }
  a.kind = (int32_t *)out(kind); a.log_prob = (float *)out(log_prob); a.raw = (float *)out(raw); a.move = (float *)out(move); a.stream = stream_of(logits);
  done(agarcl_sample_actions(&a));
  return mean.defined() ? py::make_tuple(move, kind, log_prob, raw) : py::make_tuple(py::none(), kind, log_prob, py::none());
}

// what of a loss call is not differentiated; the tensors in the order they are kept for the backward pass
struct LossCall {
  Tensor kind, old, adv, move, ref, allowed, weight;
  double low, high, kl, entropy;
  int over, per_row;
  bool need[3];                   // logits, mean, log_std
  Tensor results;                 // out, 16 numbers: the loss's stats from kStats on, its gradients of a shared log_std for an upstream gradient of 1 from kStdOne, the loss at kLoss
};
const int kStats = 0, kStdOne = 8, kLoss = 10;
agarcl_policy_loss_args loss_args(const Tensor &logits, const Tensor &mean, const Tensor &log_std, const LossCall &c, std::vector<Tensor> &kept) {
  const Strided z = rows_of(logits), k = rows_of(c.allowed);
  kept.reserve(16);
  const auto keep = [&](const Tensor &t) { kept.push_back(whole(t)); return ptr(kept.back()); };
  kept.push_back(z.t); kept.push_back(k.t);
  agarcl_policy_loss_args a = {};
  a.rows = product(logits.sizes().slice(0, logits.dim() - 1)); a.kinds = logits.size(-1); a.dtype = type_code(logits.scalar_type()); a.device = logits.get_device();
  a.logits = ptr(z.t); a.logits_stride = z.stride; a.allowed = (const uint8_t *)ptr(k.t); a.allowed_stride = k.stride;
  a.kind = (const int32_t *)keep(c.kind); a.mean = keep(mean); a.log_std = keep(log_std); a.log_std_per_row = c.per_row; a.mean_over_weight = c.over; a.move = (const float *)keep(c.move);
  a.old_log_prob = (const float *)keep(c.old); a.advantage = (const float *)keep(c.adv); a.ref_log_prob = (const float *)keep(c.ref); a.weight = (const float *)keep(c.weight);
  a.clip_low = (float)c.low; a.clip_high = (float)c.high; a.kl_coef = (float)c.kl; a.entropy_coef = (float)c.entropy; a.stream = stream_of(logits);
  return a;
}
// the tensors for the gradients of logits, mean, and a log_std per row
void loss_grads(const LossCall &c, const Tensor &logits, const Tensor &mean, const Tensor &log_std, Tensor (&g)[3]) {
  if (c.need[0]) g[0] = make(logits.sizes(), logits.scalar_type(), logits);
  if (c.need[1]) g[1] = make(mean.sizes(), mean.scalar_type(), mean);
  if (c.need[2] && c.per_row) g[2] = make(log_std.sizes(), log_std.scalar_type(), log_std);
}
// c.results; the gradients for an upstream gradient of 1 into what of g is defined, that of a shared log_std into c.results
void loss_forward(const Tensor &logits, const Tensor &mean, const Tensor &log_std, LossCall &c, const Tensor (&g)[3], bool shared_std) {
  std::vector<Tensor> kept;
  agarcl_policy_loss_args a = loss_args(logits, mean, log_std, c, kept);
  const Tensor work = make({agarcl_policy_loss_work()}, at::kDouble, logits);
  c.results = floats({16}, logits);
  float *r = (float *)out(c.results);
  a.want_stats = 1; a.loss = r + kLoss; a.stats = r + kStats; a.work = (double *)out(work);
  a.dlogits = out(g[0]); a.dmean = out(g[1]); a.dlog_std = shared_std ? r + kStdOne : out(g[2]);
  done(agarcl_policy_loss(&a));
}

// The gradients for an upstream gradient of 1 -- what loss.backward() brings -- are written by the forward pass, from the registers that hold the logits for the
// loss.  The first backward pass hands them out after its kernel has looked at the upstream gradient: it does nothing where that is 1 and works the
// gradients out from the logits otherwise.  Every other backward pass (a second one through a kept graph; one that is captured: its replays may bring other
// upstream gradients) works them out, into tensors of its own.  In float16 a loss is scaled as a rule, so there the forward pass leaves them.
struct PolicyLossNode : torch::autograd::Node {
  SavedVariable in_[3], fixed_[7], results_;
  LossCall c;                     // without its tensors
  Tensor ahead_[3];               // the gradients for an upstream gradient of 1
  bool ahead = false;
  void keep(const Tensor &logits, const Tensor &mean, const Tensor &log_std, LossCall &call) {
    const Tensor *in[3] = {&logits, &mean, &log_std}, *fixed[7] = {&call.kind, &call.old, &call.adv, &call.move, &call.ref, &call.allowed, &call.weight};
    for (int i = 0; i < 3; ++i) in_[i] = SavedVariable(*in[i], false);
    for (int i = 0; i < 7; ++i) fixed_[i] = SavedVariable(*fixed[i], false);
    results_ = SavedVariable(call.results, false);
    c = LossCall{{}, {}, {}, {}, {}, {}, {}, call.low, call.high, call.kl, call.entropy, call.over, call.per_row, {call.need[0], call.need[1], call.need[2]}, {}};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto &s : in_) s.reset_data();
    for (auto &s : fixed_) s.reset_data();
    results_.reset_data();
    for (auto &t : ahead_) t.reset();
    ahead = false;
  }
  variable_list apply(variable_list &&up) override {
    std::lock_guard<std::mutex> lock(mutex_);
    no_second_gradient();
    if (!up[0].defined()) return variable_list(3);
    const Tensor logits = in_[0].unpack(), mean = in_[1].unpack(), log_std = in_[2].unpack(), results = results_.unpack();
    LossCall now{fixed_[0].unpack(), fixed_[1].unpack(), fixed_[2].unpack(), fixed_[3].unpack(), fixed_[4].unpack(), fixed_[5].unpack(), fixed_[6].unpack(), c.low, c.high, c.kl, c.entropy,
                 c.over, c.per_row, {c.need[0], c.need[1], c.need[2]}, results};
    std::vector<Tensor> kept;
    agarcl_policy_loss_args a = loss_args(logits, mean, log_std, now, kept);
    const Tensor upstream = stored(up[0]).to(at::kFloat).contiguous();
    Tensor g[3];
    if (ahead && !capturing(logits)) {
      a.skip_if_one = 1; ahead = false;
      for (int i = 0; i < 3; ++i) g[i] = std::move(ahead_[i]);
    } else loss_grads(now, logits, mean, log_std, g);
    if (c.need[2] && !c.per_row) g[2] = floats({2}, logits);
    a.upstream = (const float *)ptr(upstream); a.weight_sum = (const float *)ptr(results) + kStats + 4;
    a.dlogits = out(g[0]); a.dmean = out(g[1]); a.dlog_std = out(g[2]); a.dlog_std_one = (const float *)ptr(results) + kStdOne;
    done(agarcl_policy_loss(&a));
    return {g[0], g[1], g[2]};
  }
};

py::tuple policy_loss(py::handle hlogits, py::handle hkind, py::handle hold, py::handle hadv, py::handle hmean, py::handle hstd, py::handle hmove, py::handle href, py::handle hallowed,
                      py::handle hweight, double low, double high, double kl, double entropy, int over) {
  const Tensor logits = first(hlogits, "logits"), mean = optional(hmean, "mean");
  LossCall c{needed(hkind, "kind"), needed(hold, "old_log_prob"), needed(hadv, "advantage"), optional(hmove, "move"), optional(href, "ref_log_prob"), optional(hallowed, "allowed"),
             optional(hweight, "weight"), low, high, kl, entropy, over, 0, {false, false, false}, {}};
  constant({{"old_log_prob", &c.old}, {"advantage", &c.adv}, {"move", &c.move}, {"ref_log_prob", &c.ref}, {"weight", &c.weight}});
  Tensor log_std;
  c.per_row = policy_checks(logits, mean, hstd, c.allowed, log_std);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  like(c.kind, "kind", logits, INTS, lead);
  like(c.old, "old_log_prob", logits, F32, lead);
  like(c.adv, "advantage", logits, F32, lead);
  if (mean.defined() != c.move.defined()) refuse("mean and move belong together");
  if (c.move.defined()) like(c.move, "move", logits, F32, mean.sizes());
  if (c.ref.defined()) like(c.ref, "ref_log_prob", logits, F32, lead);
  if (c.weight.defined()) like(c.weight, "weight", logits, WEIGHTS, lead);
  if (!(low >= 0 && high >= 0)) refuse("clip must not be negative");
  if (!(std::isfinite((float)kl) && std::isfinite((float)entropy))) refuse("kl_coef and entropy_coef must be finite");
  on_gpu(logits);
  if (c.weight.defined() && c.weight.scalar_type() != at::kFloat) c.weight = c.weight.to(at::kFloat);
  if (c.kind.scalar_type() != at::kInt) c.kind = c.kind.clamp(-1, logits.size(-1)).to(at::kInt);      // (what 32 bits cannot hold is outside all the same)
  c.need[0] = logits.requires_grad(); c.need[1] = mean.defined() && mean.requires_grad(); c.need[2] = log_std.defined() && log_std.requires_grad();
  std::shared_ptr<PolicyLossNode> node;
  if (at::GradMode::is_enabled() && (c.need[0] || c.need[1] || c.need[2])) {
    capture_reaches(logits, {&logits, &mean, &log_std});
    node = std::shared_ptr<PolicyLossNode>(new PolicyLossNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits, mean, log_std));
    {
      at::NoGradGuard off;
      node->ahead = logits.scalar_type() != at::kHalf && !capturing(logits);
      if (node->ahead) loss_grads(c, logits, mean, log_std, node->ahead_);
      loss_forward(logits, mean, log_std, c, node->ahead_, c.need[2] && !c.per_row);
    }
    node->keep(logits, mean, log_std, c);
  } else loss_forward(logits, mean, log_std, c, {}, false);
  const auto number = [&](int i) { return part(c.results, i, {}); };
  const Tensor loss = number(kLoss);
  if (node) torch::autograd::set_history(loss, node);
  return py::make_tuple(loss, number(kStats), number(kStats + 1), number(kStats + 2), number(kStats + 3));
}

}  // namespace

PYBIND11_MODULE(_learn, m) {
  m.doc() = "torch tensors in and out of include/agarcl_learn.h; documented in agarcl_amd/learn.py";
  static const py::object &error = *new py::object(py::module_::import("agarcl_amd._capi").attr("AgarclError"));      // (never destroyed: nothing runs after the interpreter)
  py::register_exception_translator([](std::exception_ptr p) {
    try { if (p) std::rethrow_exception(p); }
    catch (const Failure &f) { py::object e = error(f.code, f.text); PyErr_SetObject(error.ptr(), e.ptr()); }
  });
  m.def("gated_recurrence", &gated_recurrence);
  m.def("recurrence_step", &recurrence_step);
  m.def("advantages", &advantages);
  m.def("sample_actions", &sample_actions);
  m.def("policy_loss", &policy_loss);
}
