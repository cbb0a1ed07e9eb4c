// Host side of the token operators: checks, layouts, workspaces, streams and gradients of `ops.rotary_axes`, `ops.cross_attention` and
// `ops.adamw_step` over the C ABI of include/sleap_amd.h. In C++ because these calls are small beside what Python charges for them: a
// rotary call of a frame's queries runs 3.5 us on the GPU and cost its host 13 us through ctypes (now 5), an attention with its gradients 155 us
// (now 70, of which torch's engine alone takes 27), the step of 448 tensors 600 us (now 50, its four launches among them).
//
// Plain torch C++ on raw tensors: device memory, streams and the autograd graph. The entry points are handed over as addresses by
// sleap_amd/ops.py, from the library build that the rest of the package uses.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <map>
#include <sstream>
#include <unordered_set>

#include "../../include/sleap_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct {
  decltype(&sa_last_error) last_error;
  decltype(&sa_rotary_axes) rotary_axes;
  decltype(&sa_cross_attention_workspace) attention_workspace;
  decltype(&sa_cross_attention) attention;
  decltype(&sa_cross_attention_backward_workspace) backward_workspace;
  decltype(&sa_cross_attention_backward) attention_backward;
  decltype(&sa_adamw_step) adamw_step;
  PyObject* error;  // SleapAmdError
} entry;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
template <typename... A>
[[noreturn]] void bad_value(const A&... a) {
  throw py::value_error(text(a...));
}
template <typename... A>
[[noreturn]] void bad_type(const A&... a) {
  throw py::type_error(text(a...));
}

void check(int rc, const char* what) {
  if (rc == SA_OK) return;
  const std::string message = text(what, " failed (", rc, "): ", entry.last_error());
  if (!PyGILState_Check()) throw std::runtime_error(message);  // a gradient, in the engine's thread
  PyErr_SetString(entry.error, message.c_str());
  throw py::error_already_set();
}

void* stream_of(const at::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SA_F32;
    case at::kHalf: return SA_F16;
    case at::kBFloat16: return SA_BF16;
    default: return -1;
  }
}

// Forward-mode derivatives (torch.autograd.forward_ad) would be lost without a word: a kernel reads a tensor's values alone. Tensors carry them
// within a level only; outside of one they are not asked, since each answer takes a lock (448 tensors of an optimizer step: 50 us).
bool may_carry_tangents() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const char* who, const char* name, const Tensor& t) {
  if (t._fw_grad(/*level=*/0).defined()) throw std::runtime_error(text(who, ": ", name, " carries a forward-mode derivative: there are none"));
}

// The step has no gradient: a graph that it would cut, with what it leaves behind of it, is refused. (A parameter that is a leaf has none.)
void no_graph(const char* what, const Tensor& t, bool leaf) {
  if (t.requires_grad() && !(leaf && t.is_leaf()))
    throw std::runtime_error(text("adamw_step: there is no gradient through a step (", what, " requires one): call it under torch.no_grad()"));
}

void on_one_gpu(const char* who, std::initializer_list<std::pair<const char*, const Tensor*>> tensors) {
  if (may_carry_tangents())
    for (const auto& [name, t] : tensors)
      if (t->defined()) no_tangent(who, name, *t);
  const Tensor* first = nullptr;
  for (const auto& [name, t] : tensors) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) bad_value(who, ": ", name, " must be a CUDA tensor (there is no CPU fallback)");
    if (!first) first = t;
    else if (t->device() != first->device()) bad_value(who, ": ", name, " is on ", t->device(), ", not on ", first->device());
  }
}

bool capturing(const at::Device& d) {
  const c10::OptionalDeviceGuard guard(d);
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

// whether a stream is the current one or another that the capture has taken in, or, of a leaf's node, can take in and gives back by itself (the
// engine joins the streams of leaves when a backward pass ends). The default stream can not be captured, and is not asked.
bool captured(const c10::Stream& s, bool leaf) {
  const auto now = c10::hip::getCurrentHIPStream(s.device_index());
  if (s.id() == now.id()) return true;
  const hipStream_t other = c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, now.unwrap().device(), s.id())).stream();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return other && (leaf || (hipStreamIsCapturing(other, &status) == hipSuccess && status == hipStreamCaptureStatusActive));
}

// A graph that was built outside of a capture and still lives holds the gradient nodes of its leaves, and with them the stream that it was
// built on: a captured backward pass that reaches one of its nodes would pull that stream into the capture, where torch's engine ends the
// process. Refused before it starts; everything that the inputs hang on is looked at, while capturing only. (Leaves whose graph was
// built on a stream of its own, as a warm-up ahead of a capture is, are fine.)
void not_held_elsewhere(const char* who, std::initializer_list<const Tensor*> tensors) {
  if (!capturing((*tensors.begin())->device())) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  std::unordered_set<const torch::autograd::Node*> met;
  auto meet = [&](const std::shared_ptr<torch::autograd::Node>& node) {
    if (node && met.insert(node.get()).second) todo.push_back(node);
  };
  for (const Tensor* t : tensors)
    if (t->requires_grad()) meet(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
  while (!todo.empty()) {
    const auto node = std::move(todo.back());
    todo.pop_back();
    const auto held = node->stream();
    if (held && !captured(*held, node->next_edges().empty()))
      throw std::runtime_error(text(who, ": captured while a graph from outside of the capture holds the same leaf: delete that graph first (or capture a detached leaf)"));
    for (const auto& edge : node->next_edges()) meet(edge.function);
  }
}

// A (B, T, heads, D) tensor as the kernels take it: `t` itself if its last dimension is contiguous, every other stride and the address are
// whole multiples of `elements` values and 64 tokens and `group` heads span less than `limit` (if any); else a contiguous copy.
// Strides are 0 where there is nothing to step over.
struct Laid {
  Tensor t;
  std::array<int64_t, 3> s;
};
Laid laid_out(Tensor t, int64_t elements, int64_t limit = 0, int64_t group = 0) {
  t = t.resolve_neg();
  if (t.numel() == 0) return {std::move(t), {}};  // nothing to step over, whatever its strides say
  for (int turn = 0;; ++turn) {
    std::array<int64_t, 3> s;
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    const bool fits = (t.size(3) == 1 || t.stride(3) == 1) && s[0] % elements == 0 && s[1] % elements == 0 && s[2] % elements == 0 &&
                      reinterpret_cast<uintptr_t>(t.data_ptr()) % (elements * t.element_size()) == 0 && (!limit || 64 * s[1] + group * s[2] < limit);
    if (fits || turn) return {std::move(t), s};
    t = t.clone(at::MemoryFormat::Contiguous);
  }
}

// ---------------------------------------------------------------------------------------------- rotary positions
struct Turn {
  std::vector<int> sections;
  double theta;
  bool shared, interleaved, inverse;
};

Tensor turn(const Tensor& x_, const Tensor& positions_, const Turn& how) {
  const Laid x = laid_out(x_, how.interleaved ? 2 : 1);
  const Tensor positions = positions_.resolve_neg();
  const int64_t B = x.t.size(0), T = x.t.size(1), H = x.t.size(2), D = x.t.size(3);
  Tensor y = at::empty({B, T, H, D}, x.t.options());
  if (B == 0 || T == 0) return y;
  const int64_t n = positions.dim();
  const int64_t places[3] = {n == 3 && positions.size(0) > 1 ? positions.stride(0) : 0, positions.stride(n - 2), positions.stride(n - 1)};
  const int pos = positions.scalar_type() == at::kInt ? SA_POS_I32 : positions.scalar_type() == at::kLong ? SA_POS_I64 : SA_POS_F32;
  const c10::OptionalDeviceGuard guard(x.t.device());
  check(entry.rotary_axes(x.t.data_ptr(), type_of(x.t), (int)B, (int)T, (int)H, (int)D, x.s.data(), positions.data_ptr(), pos, places,
                        (int)how.sections.size(), how.sections.data(), how.theta, how.shared, how.interleaved, how.inverse, y.data_ptr(),
                        stream_of(x.t.device())),
        "sa_rotary_axes");
  return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Turn& how) {
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = std::vector<int64_t>(how.sections.begin(), how.sections.end());
    ctx->saved_data["theta"] = how.theta;
    ctx->saved_data["how"] = (int64_t)(how.shared | how.interleaved << 1 | how.inverse << 2);
    return turn(x, positions, how);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor dy = grads[0], positions = ctx->get_saved_variables()[0];
    if (!dy.defined()) return {Tensor(), Tensor(), Tensor()};
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const int64_t bits = ctx->saved_data["how"].toInt();
    // linear in x: its gradient is the turn the other way, which has a gradient again
    const Turn how = {{sections.begin(), sections.end()}, ctx->saved_data["theta"].toDouble(), (bits & 1) != 0, (bits & 2) != 0, (bits & 4) == 0};
    const bool again = at::GradMode::is_enabled() && dy.requires_grad();
    return {again ? Rotary::apply(dy, positions, how) : turn(dy, positions, how), Tensor(), Tensor()};
  }
};

Tensor rotary_axes(const Tensor& x, const Tensor& positions, const std::vector<int64_t>& sections, double theta, const std::string& ladder,
                   bool interleaved, bool inverse) {
  const char* who = "rotary_axes";
  on_one_gpu(who, {{"x", &x}, {"positions", &positions}});
  if (x.dim() != 4 || x.size(3) % 2 || x.size(3) < 2 || x.size(3) > 4096 || x.size(2) < 1 || x.size(2) > 4096)
    bad_value(who, ": x must be (B, T, heads, even size): got ", x.sizes());
  if (type_of(x) < 0) bad_type(who, ": x must be float32, float16 or bfloat16: got ", x.scalar_type());
  if (x.size(0) >= 1ll << 31 || x.size(1) >= 1ll << 31) bad_value(who, ": too many tokens: ", x.sizes());
  const auto kind = positions.scalar_type();
  if (kind != at::kInt && kind != at::kLong && kind != at::kFloat) bad_type(who, ": positions must be int32, int64 or float32: got ", kind);
  const int64_t B = x.size(0), T = x.size(1), D = x.size(3), A = (int64_t)sections.size();
  int64_t pairs = 0;
  bool fits = A >= 1 && A <= 8;
  for (const int64_t n : sections) {
    fits = fits && n >= 0 && n <= 128;
    pairs += fits ? n : 0;
  }
  if (!fits || pairs < 1 || pairs > std::min<int64_t>(D / 2, 128))
    bad_value(who, ": sections ", at::IntArrayRef(sections), " do not fit a head of ", D, " (at most 8 axes and 128 pairs of two values)");
  const int64_t n = positions.dim();
  if ((n != 2 && n != 3) || positions.size(n - 2) != T || positions.size(n - 1) != A || (n == 3 && positions.size(0) != B && positions.size(0) != 1))
    bad_value(who, ": positions ", positions.sizes(), " for ", B, " x ", T, " tokens and ", A, " axes");
  if (ladder != "axis" && ladder != "shared") bad_value(who, ": ladder '", ladder, "': 'axis' or 'shared'");
  if (!(theta > 0 && theta < 1e30)) bad_value(who, ": theta ", theta);
  if (positions.requires_grad() && at::GradMode::is_enabled()) bad_value(who, ": there is no gradient for positions");
  const Turn how = {{sections.begin(), sections.end()}, theta, ladder == "shared", interleaved, inverse};
  if (!x.requires_grad() || !at::GradMode::is_enabled()) return turn(x, positions, how);
  not_held_elsewhere(who, {&x});
  return Rotary::apply(x, positions, how);
}

// ---------------------------------------------------------------------------------------------- cross attention
// What the kernels address from one 64-bit base with 32 bits: 64 tokens of keys or values, and in the backward pass 64 tokens and the
// heads on one key head of q and dout, in elements. Wider layouts are copied.
constexpr int64_t KEY_SPAN = 64ll << 23, ROW_SPAN = 1ll << 30;

struct Keys {
  Tensor lengths, mask;
  float scale;
  const int32_t* n() const { return lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr; }
  const uint8_t* m() const { return mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr()) : nullptr; }
  std::array<int64_t, 2> strides() const {
    return mask.defined() ? std::array<int64_t, 2>{mask.size(0) > 1 ? mask.stride(0) : 0, mask.stride(1)} : std::array<int64_t, 2>{0, 0};
  }
};

Tensor workspace(size_t bytes, const Tensor& like) {  // of one call: the allocator orders its next use, a captured graph has its own
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Up to this many keys, or where lengths or a mask may leave no more, a forward pass that is to be differentiated keeps its output in two
// terms (attention.hip: LOW).
constexpr int64_t FEW_KEYS = 2048;

struct Attended {
  Tensor out, lse, low;
};
Attended attend(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Keys& keys, bool want_lse, bool want_low) {
  const Laid q = laid_out(q_, 8), k = laid_out(k_, 8, KEY_SPAN), v = laid_out(v_, 8, KEY_SPAN);
  const int B = (int)q.t.size(0), Tq = (int)q.t.size(1), H = (int)q.t.size(2), D = (int)q.t.size(3), Tk = (int)k.t.size(1), K = (int)k.t.size(2);
  Tensor out = at::empty({B, Tq, H, D}, q.t.options()), lse, low;
  if (want_low) low = at::empty_like(out);
  if (want_lse) lse = at::empty({B, H, Tq}, q.t.options().dtype(at::kFloat));
  if (B == 0 || Tq == 0) return {out, lse, low};
  const size_t bytes = entry.attention_workspace(B, Tq, Tk, H, K, D);
  const Tensor ws = workspace(bytes, q.t);
  const int64_t strides[9] = {q.s[0], q.s[1], q.s[2], k.s[0], k.s[1], k.s[2], v.s[0], v.s[1], v.s[2]};
  const auto ms = keys.strides();
  const c10::OptionalDeviceGuard guard(q.t.device());
  check(entry.attention(q.t.data_ptr(), k.t.data_ptr(), v.t.data_ptr(), type_of(q.t), B, Tq, Tk, H, K, D, strides, keys.n(), keys.m(), ms.data(),
                      keys.scale, out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr,
                      want_low ? low.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes,
                      stream_of(q.t.device())),
        "sa_cross_attention");
  return {out, lse, low};
}

std::array<Tensor, 3> attend_backward(const Tensor& dout_, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& out, const Tensor& lse,
                                      const Tensor& low, const Keys& keys, bool want_q, bool want_kv) {
  const int64_t group = q_.size(2) / k_.size(2);
  const Laid q = laid_out(q_, 8, ROW_SPAN, group), k = laid_out(k_, 8, KEY_SPAN), v = laid_out(v_, 8, KEY_SPAN), dout = laid_out(dout_, 8, ROW_SPAN, group);
  const int B = (int)q.t.size(0), Tq = (int)q.t.size(1), H = (int)q.t.size(2), D = (int)q.t.size(3), Tk = (int)k.t.size(1), K = (int)k.t.size(2);
  Tensor dq, dk, dv;
  if (want_q) dq = at::empty({B, Tq, H, D}, q.t.options());
  if (want_kv) {
    dk = at::empty({B, Tk, K, D}, q.t.options());
    dv = at::empty_like(dk);
  }
  if (B == 0 || (Tq == 0 && Tk == 0)) return {dq, dk, dv};
  const size_t bytes = entry.backward_workspace(B, Tq, Tk, H, K, D);
  const Tensor ws = workspace(bytes, q.t);
  const int64_t strides[9] = {q.s[0], q.s[1], q.s[2], k.s[0], k.s[1], k.s[2], v.s[0], v.s[1], v.s[2]};
  const auto ms = keys.strides();
  const c10::OptionalDeviceGuard guard(q.t.device());
  check(entry.attention_backward(q.t.data_ptr(), k.t.data_ptr(), v.t.data_ptr(), type_of(q.t), B, Tq, Tk, H, K, D, strides, keys.n(), keys.m(),
                               ms.data(), keys.scale, out.data_ptr(), low.defined() ? low.data_ptr() : nullptr, lse.data_ptr<float>(), dout.t.data_ptr(), dout.s.data(),
                               want_q ? dq.data_ptr() : nullptr, want_kv ? dk.data_ptr() : nullptr, want_kv ? dv.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q.t.device())),
        "sa_cross_attention_backward");
  return {dq, dk, dv};
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Keys& keys, bool want_lse) {
    const auto [out, lse, low] = attend(q, k, v, keys, true, k.size(1) <= FEW_KEYS || keys.lengths.defined() || keys.mask.defined());
    ctx->save_for_backward({q, k, v, out, lse, low, keys.lengths, keys.mask});
    ctx->saved_data["scale"] = (double)keys.scale;
    ctx->set_materialize_grads(false);
    if (!want_lse) return {out};
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const Keys keys = {saved[6], saved[7], (float)ctx->saved_data["scale"].toDouble()};
    const auto [dq, dk, dv] = attend_backward(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], keys,
                                            ctx->needs_input_grad(0), ctx->needs_input_grad(1) || ctx->needs_input_grad(2));
    variable_list got = {dq, dk, dv};
    if (at::GradMode::is_enabled()) {  // create_graph: a second gradient has to fail, not to miss what these depend on
      for (auto& t : got)
        if (t.defined()) t = t.detach().set_requires_grad(true);
      got = (*std::make_shared<torch::autograd::DelayedError>("cross_attention has first gradients only", 3))(std::move(got));
    }
    return {got[0], got[1], got[2], Tensor(), Tensor()};
  }
};

py::object cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& lengths_, const std::optional<Tensor>& mask_,
                           std::optional<double> scale_, bool return_lse) {
  const char* who = "cross_attention";
  Keys keys = {lengths_.value_or(Tensor()), mask_.value_or(Tensor()), 0.0f};
  on_one_gpu(who, {{"q", &q}, {"k", &k}, {"v", &v}, {"key_lengths", &keys.lengths}, {"key_mask", &keys.mask}});
  if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    bad_value(who, ": q (B, Tq, heads, D), k and v (B, Tk, key heads, D): got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  if ((q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    bad_type(who, ": q, k and v must all be float16 or all bfloat16: got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  const int64_t B = q.size(0), H = q.size(2), D = q.size(3), Tk = k.size(1), K = k.size(2);
  if (D % 8 || D < 8 || D > 128) bad_value(who, ": head size ", D, ": a multiple of 8, at most 128");
  if (H < 1 || K < 1 || H % K) bad_value(who, ": ", H, " query heads do not share ", K, " key heads evenly");
  if (std::max({B, q.size(1), H, Tk}) >= 1ll << 30) bad_value(who, ": too many tokens: ", q.sizes(), ", ", k.sizes());
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)D);
  if (!(scale >= 1e-30 && scale <= 1e30)) bad_value(who, ": scale ", scale, " must be positive and finite");
  keys.scale = (float)scale;
  if (keys.lengths.defined()) {
    const auto kind = keys.lengths.scalar_type();
    if ((kind != at::kInt && kind != at::kLong) || keys.lengths.dim() != 1 || keys.lengths.size(0) != B)
      bad_value(who, ": key_lengths must be (", B, ",) int32 or int64: got ", keys.lengths.sizes(), " ", kind);
    if (kind == at::kLong) keys.lengths = keys.lengths.clamp(0, Tk).to(at::kInt);
    keys.lengths = keys.lengths.resolve_neg().contiguous();
  }
  if (keys.mask.defined() && (keys.mask.scalar_type() != at::kBool || keys.mask.dim() != 2 || (keys.mask.size(0) != B && keys.mask.size(0) != 1) || keys.mask.size(1) != Tk))
    bad_value(who, ": key_mask must be (", B, ", ", Tk, ") bool, True where a key is visible: got ", keys.mask.sizes(), " ", keys.mask.scalar_type());
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    not_held_elsewhere(who, {&q, &k, &v});
    const auto got = CrossAttention::apply(q, k, v, keys, return_lse);
    return return_lse ? py::object(py::make_tuple(got[0], got[1])) : py::cast(got[0]);
  }
  const auto [out, lse, low] = attend(q, k, v, keys, return_lse, false);
  return return_lse ? py::object(py::make_tuple(out, lse)) : py::cast(out);
}

// ---------------------------------------------------------------------------------------------- AdamW
void adamw_step(const py::sequence& params, const py::sequence& grads, const py::sequence& exp_avgs, const py::sequence& exp_avg_sqs,
                const py::object& max_exp_avg_sqs, const py::object& step, const py::object& lr, std::pair<double, double> betas, double eps,
                double weight_decay) {
  const char* who = "adamw_step";
  const bool ams = !max_exp_avg_sqs.is_none(), tangents = may_carry_tangents(), recording = at::GradMode::is_enabled();
  const int lists = ams ? 5 : 4;
  const char* names[5] = {"params", "grads", "exp_avgs", "exp_avg_sqs", "max_exp_avg_sqs"};
  const py::object given[5] = {params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs};
  py::object fast[5];
  PyObject** items[5];
  Py_ssize_t n = 0;
  for (int j = 0; j < lists; ++j) {
    fast[j] = py::reinterpret_steal<py::object>(PySequence_Fast(given[j].ptr(), "adamw_step: lists of tensors"));
    if (!fast[j]) throw py::error_already_set();
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(fast[j].ptr());
    if (j && count != n) bad_value(who, ": lists of ", n, " and ", count, " tensors");
    n = count;
    items[j] = PySequence_Fast_ITEMS(fast[j].ptr());
  }
  const bool dev_step = THPVariable_Check(step.ptr()), dev_lr = THPVariable_Check(lr.ptr());
  const int64_t t = dev_step ? 1 : step.cast<int64_t>();
  const double rate = dev_lr ? 0.0 : lr.cast<double>();
  if (t < 1) bad_value(who, ": step ", t, ": the first is 1");
  const auto [b1, b2] = betas;
  if (!(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0 && weight_decay >= 0 && rate >= 0))
    bad_value(who, ": lr ", rate, ", betas (", b1, ", ", b2, "), eps ", eps, ", weight_decay ", weight_decay);
  for (const auto& [tensor, kind, what] : {std::tuple(&step, at::kLong, "a step tensor is one int64"), std::tuple(&lr, at::kFloat, "a learning rate tensor is one float32")})
    if (THPVariable_Check(tensor->ptr())) {
      const Tensor& x = THPVariable_Unpack(tensor->ptr());
      if (tangents) no_tangent(who, "a step or learning rate tensor", x);
      if (recording) no_graph("a step or learning rate tensor", x, false);
      if (x.scalar_type() != kind || x.numel() != 1 || !x.is_cuda()) bad_value(who, ": ", what, " on the GPU of the parameters");
      if (x.is_neg()) bad_value(who, ": ", what, ", not a negated view");
    }
  if (n == 0) return;

  std::map<std::pair<int, int>, std::vector<sa_adamw_tensor>> groups;  // by type and device
  std::pair<int, int> last_key = {-1, -1};
  std::vector<sa_adamw_tensor>* last = nullptr;
  using Range = std::pair<uintptr_t, uintptr_t>;  // where something that the step writes begins and ends
  std::vector<Range> written[5];
  std::vector<Range> read;  // the gradients; one may be its own parameter, whose values are read ahead of being written
  for (int j = 0; j < lists; ++j) (j == 1 ? read : written[j]).reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const Tensor* x[5] = {};
    for (int j = 0; j < lists; ++j) {
      if (!THPVariable_Check(items[j][i])) bad_value(who, ": lists of CUDA tensors: ", names[j], "[", i, "] is none");
      x[j] = &THPVariable_Unpack(items[j][i]);
      if (tangents) no_tangent(who, names[j], *x[j]);
      if (recording) no_graph(names[j], *x[j], j == 0);
      if (!x[j]->is_cuda() || x[j]->get_device() != x[0]->get_device())
        bad_value(who, ": CUDA tensors, a parameter, its gradient and its states on one GPU (there is no CPU fallback): ", names[j], "[", i, "] is on ", x[j]->device());
      if (x[j]->layout() != at::kStrided || !x[j]->is_contiguous()) bad_value(who, ": ", names[j], "[", i, "] must be contiguous");
      if (x[j]->is_neg()) bad_value(who, ": ", names[j], "[", i, "] is a negated view");  // its memory has the other sign
      if (x[j]->numel() != x[0]->numel()) bad_value(who, ": ", names[j], "[", i, "] differs in size from its parameter");
      if (j >= 2 && x[j]->scalar_type() != at::kFloat) bad_type(who, ": the states must be float32");
    }
    const int type = type_of(*x[0]);
    if (type < 0 || x[1]->scalar_type() != x[0]->scalar_type())
      bad_type(who, ": params and grads must be pairs of one type: float32, float16 or bfloat16");
    if (x[0]->numel() == 0) continue;
    const std::pair<int, int> key = {type, (int)x[0]->get_device()};
    if (key != last_key) {
      last_key = key;
      last = &groups[key];
      if (last->empty()) last->reserve(n);
    }
    const int64_t count = x[0]->numel();
    void* at[5] = {};
    for (int j = 0; j < lists; ++j) {
      at[j] = x[j]->data_ptr();
      const auto begin = reinterpret_cast<uintptr_t>(at[j]);
      const Range range = {begin, begin + count * (j >= 2 ? 4 : x[0]->element_size())};
      if (j != 1) written[j].push_back(range);
      else if (at[1] != at[0]) read.push_back(range);
    }
    last->push_back({at[0], at[1], static_cast<float*>(at[2]), static_cast<float*>(at[3]), static_cast<float*>(at[4]), count});
  }
  // Lists are mostly in the order of their addresses: sorted one by one where they are not, and merged, the whole check is linear.
  std::vector<Range> all;
  all.reserve(n * (lists - 1));
  for (auto& w : written) {
    if (!std::is_sorted(w.begin(), w.end())) std::sort(w.begin(), w.end());
    const auto middle = (ptrdiff_t)all.size();
    all.insert(all.end(), w.begin(), w.end());
    if (middle && !w.empty() && all[middle] < all[middle - 1]) std::inplace_merge(all.begin(), all.begin() + middle, all.end());
  }
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) bad_value(who, ": the same parameter or state twice, or two that overlap");
  if (!std::is_sorted(read.begin(), read.end())) std::sort(read.begin(), read.end());
  size_t next = 0;
  for (const Range& r : read) {
    while (next < all.size() && all[next].second <= r.first) ++next;
    if (next < all.size() && all[next].first < r.second) bad_value(who, ": a gradient overlaps with something that the step writes");
  }
  for (const auto& [key, tensors] : groups)
    for (const py::object* o : {&step, &lr})
      if (THPVariable_Check(o->ptr()) && THPVariable_Unpack(o->ptr()).get_device() != key.second)
        bad_value(who, ": step and learning rate tensors must be on the GPU of the parameters");
  auto device_of = [](const std::pair<int, int>& key) { return c10::Device(c10::kCUDA, (c10::DeviceIndex)key.second); };
  for (const auto& [key, tensors] : groups)
    if (!dev_step && capturing(device_of(key)))
      throw std::runtime_error("adamw_step: a captured step needs its count as a tensor (every replay would repeat this one)");
  for (const auto& [key, tensors] : groups) {
    const c10::Device device = device_of(key);
    const c10::OptionalDeviceGuard guard(device);
    check(entry.adamw_step(tensors.data(), (int)tensors.size(), key.first, ams, rate, dev_lr ? THPVariable_Unpack(lr.ptr()).data_ptr<float>() : nullptr, b1, b2,
                         eps, weight_decay, t, dev_step ? THPVariable_Unpack(step.ptr()).data_ptr<int64_t>() : nullptr, stream_of(device)),
          "sa_adamw_step");
  }
  for (int j = 0; j < lists; ++j)  // a graph that saved one of them has to notice
    for (Py_ssize_t i = 0; j != 1 && i < n; ++i) {
      const Tensor& x = THPVariable_Unpack(items[j][i]);
      if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
    }
}

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", [](const py::dict& addresses, const py::object& error) {
    take(entry.last_error, addresses, "sa_last_error");
    take(entry.rotary_axes, addresses, "sa_rotary_axes");
    take(entry.attention_workspace, addresses, "sa_cross_attention_workspace");
    take(entry.attention, addresses, "sa_cross_attention");
    take(entry.backward_workspace, addresses, "sa_cross_attention_backward_workspace");
    take(entry.attention_backward, addresses, "sa_cross_attention_backward");
    take(entry.adamw_step, addresses, "sa_adamw_step");
    entry.error = error.inc_ref().ptr();
  });
  m.def("rotary_axes", &rotary_axes);
  m.def("cross_attention", &cross_attention);
  m.def("adamw_step", &adamw_step);
}
