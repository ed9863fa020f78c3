// The sequence-block operators' calls from PyTorch without Python in between: argument checks, buffers, the current stream and the
// autograd nodes, over the C ABI of include/sound_bubble_seq.h.  A small call is its host time (a layer norm of 145 x 32: 3 us on the GPU), and a
// backward pass that is Python costs a change of thread and interpreter on top.
//
// These are the plain calls only.  Whatever is out of the ordinary -- a wrong type, nothing to compute, a copy that Python has to decide on --
// is "not taken" (an empty list, 0) before anything is launched: sound_bubble_amd/ops_seq.py then handles it, or says what is wrong.  What
// is raised is raised for good: nobody runs the call again.  The entry points' addresses come from there too (bind), so that one library serves both.
//
// Layer norm and scan are operators of the dispatcher (0.7 us a call).  AdamW's lists of tensors are not: a step over 160 parameters is 39 us of
// host time by the dispatcher, 18 by the module's function.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>

#include "../../../include/sound_bubble_seq.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&sb_layer_norm_fwd) layer_norm_fwd;
  decltype(&sb_layer_norm_bwd_scratch) layer_norm_bwd_scratch;
  decltype(&sb_layer_norm_bwd) layer_norm_bwd;
  decltype(&sb_gated_scan_plan) gated_scan_plan;
  decltype(&sb_gated_scan_fwd) gated_scan_fwd;
  decltype(&sb_gated_scan_bwd) gated_scan_bwd;
  decltype(&sb_gated_scan_step) gated_scan_step;
  decltype(&sb_adamw_chunk) adamw_chunk;
  decltype(&sb_adamw_norm) adamw_norm;
  decltype(&sb_adamw_step) adamw_step;
} entry = {};

void bind(at::IntArrayRef addresses) {
  TORCH_CHECK(addresses.size() * sizeof(void*) == sizeof(Entries), "sound_bubble_seq::bind: one address for each entry point");
  for (const int64_t a : addresses) TORCH_CHECK(a != 0, "sound_bubble_seq::bind: a null address");
  std::memcpy(&entry, addresses.data(), sizeof(Entries));
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SB_F32;
    case at::kBFloat16: return SB_BF16;
    case at::kHalf: return SB_F16;
    default: return -1;
  }
}
bool plain(const Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && type_of(t) >= 0; }
bool given(const Maybe& t) { return t.has_value() && t->defined(); }
Tensor or_none(const Maybe& t) { return given(t) ? *t : Tensor(); }
template <class T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor f32(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc, const char* what) { TORCH_CHECK(rc == 0, "sound_bubble: ", what, " failed with status ", rc); }

// passes `value` on and refuses its gradient: the second derivative that there is none of
struct NoSecond : torch::autograd::Function<NoSecond> {
  static Tensor forward(AutogradContext*, const Tensor& value, const Tensor&) { return value.alias(); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "sound_bubble: layer_norm and gated_scan have no second derivative");
  }
};
Tensor once(const Tensor& value, const Tensor& through) {
  return value.defined() && at::GradMode::is_enabled() && through.defined() && through.requires_grad() ? NoSecond::apply(value, through) : value;
}

// A leaf that an eager graph still holds has its gradient's node on that graph's stream; a backward pass under capture would wait for that stream,
// which ends the capture and the process.  Said here, in the forward call under capture.
void refuse_held_leaves(at::ArrayRef<const Tensor*> leaves, const Tensor& like) {
  const c10::OptionalDeviceGuard guard(like.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto id = c10::hip::getCurrentHIPStream(like.device().index()).id();
  for (const Tensor* t : leaves) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!stream || stream->id() == id, "sound_bubble: an eager graph of this leaf, made on another stream, is alive while a graph is captured: "
                "drop it (its outputs and losses) before the capture");
  }
}

void refuse_held(const std::vector<Tensor>& leaves) {
  std::vector<const Tensor*> at;
  for (const Tensor& t : leaves) at.push_back(&t);
  if (!leaves.empty()) refuse_held_leaves(at, leaves[0]);
}
// forward-mode tangents are refused where autograd is: by the Python functions
bool tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

// ---- layer norm ----
std::pair<Tensor, int64_t> rows_of(const Tensor& t, int64_t n) {
  if (t.is_contiguous()) return {t, n};
  Tensor r = t.reshape({-1, n});
  if (n > 1 && r.stride(1) != 1) r = r.contiguous();
  return {r, r.size(0) > 1 ? r.stride(0) : n};
}
bool norm_takes(const Tensor& x, const Maybe& weight, const Maybe& bias) {
  if (!plain(x) || x.dim() < 1 || x.numel() == 0 || tangent(x) || tangent(or_none(weight)) || tangent(or_none(bias))) return false;
  for (const Maybe* t : {&weight, &bias})
    if (given(*t) && (!plain(**t) || (*t)->device() != x.device() || (*t)->dim() != 1 || (*t)->size(0) != x.size(-1) ||
                      ((*t)->scalar_type() != x.scalar_type() && (*t)->scalar_type() != at::kFloat)))
      return false;
  return !given(weight) || !given(bias) || weight->scalar_type() == bias->scalar_type();
}
Tensor norm_fwd(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* mean, Tensor* rstd) {
  const c10::OptionalDeviceGuard guard(x.device());
  const int64_t n = x.size(-1);
  Tensor y = dense_like(x);
  if (mean) {
    *mean = f32(x, x.sizes().slice(0, x.dim() - 1));
    *rstd = f32(x, x.sizes().slice(0, x.dim() - 1));
  }
  const auto [xr, ldx] = rows_of(x, n);
  const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  sb_layer_norm_args a = {};
  a.rows = x.numel() / n; a.n = n; a.ldx = ldx;
  a.xtype = type_of(x);
  a.wtype = w.defined() ? type_of(w) : b.defined() ? type_of(b) : SB_F32;
  a.eps = (float)eps;
  a.x = ptr(xr); a.w = ptr(w); a.b = ptr(b); a.y = ptr(y);
  a.mean = mean ? ptr<float>(*mean) : nullptr;
  a.rstd = mean ? ptr<float>(*rstd) : nullptr;
  check(entry.layer_norm_fwd(&a, stream_of(x)), "sb_layer_norm_fwd");
  return y;
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    Tensor mean, rstd;
    const Tensor y = norm_fwd(x, or_none(weight), or_none(bias), eps, &mean, &rstd);
    ctx->save_for_backward({x, or_none(weight), mean, rstd});
    ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (given(weight) && weight->requires_grad()) << 1 | (given(bias) && bias->requires_grad()) << 2);
    ctx->saved_data["f32"] = given(bias) && bias->scalar_type() == at::kFloat;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &mean = saved[2], &rstd = saved[3], &dy = grads[0];
    const int64_t need = ctx->saved_data["need"].toInt();
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t n = x.size(-1), rows = x.numel() / n;
    const auto wt = weight.defined() ? weight.scalar_type() : ctx->saved_data["f32"].toBool() ? at::kFloat : x.scalar_type();
    TORCH_CHECK(dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes() && dy.device() == x.device(), "layer_norm: the gradient does not fit");
    Tensor dx = dense_like(x), dw, db, scratch;
    if (need & 2) dw = at::empty({n}, x.options().dtype(wt));
    if (need & 4) db = at::empty({n}, x.options().dtype(wt));
    if (need & 6) scratch = f32(x, {entry.layer_norm_bwd_scratch(rows, n, type_of(x))});
    const auto [xr, ldx] = rows_of(x, n);
    const auto [gr, ldg] = rows_of(dy.resolve_neg(), n);
    const Tensor w = weight.defined() ? weight.contiguous() : weight;
    sb_layer_norm_bwd_args a = {};
    a.rows = rows; a.n = n; a.ldx = ldx; a.lddy = ldg;
    a.xtype = type_of(x);
    a.wtype = wt == at::kFloat ? SB_F32 : type_of(x);
    a.x = ptr(xr); a.dy = ptr(gr); a.w = ptr(w); a.mean = ptr<float>(mean); a.rstd = ptr<float>(rstd);
    a.dx = ptr(dx); a.dw = ptr(dw); a.db = ptr(db); a.scratch = ptr<float>(scratch);
    check(entry.layer_norm_bwd(&a, stream_of(x)), "sb_layer_norm_bwd");
    const Tensor through = dy.requires_grad() ? dy : x.requires_grad() ? x : weight;
    return {need & 1 ? once(dx, through) : Tensor(), once(dw, through), once(db, through), Tensor()};
  }
};
std::vector<Tensor> layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  if (!norm_takes(x, weight, bias)) return {};
  if (at::GradMode::is_enabled() && (x.requires_grad() || (given(weight) && weight->requires_grad()) || (given(bias) && bias->requires_grad()))) {
    const Tensor w = or_none(weight), b = or_none(bias);
    refuse_held_leaves({&x, &w, &b}, x);
    return {LayerNorm::apply(x, weight, bias, eps)};
  }
  return {norm_fwd(x, or_none(weight), or_none(bias), eps, nullptr, nullptr)};
}

// ---- gated scan ----
struct Sizes { int64_t dim, outer = 1, steps = 0, inner = 1; std::vector<int64_t> rest; };
struct Steps { Tensor t; int64_t so, st; };
Steps steps_of(const Tensor& t, const Sizes& z) {
  if (t.is_contiguous()) return {t, z.steps * z.inner, z.inner};
  Tensor r = t.reshape({z.outer, z.steps, z.inner});
  if (z.inner > 1 && r.stride(2) != 1) r = r.contiguous();
  return {r, r.stride(0), r.stride(1)};
}
Sizes sizes_of(const Tensor& x, int64_t dim) {
  Sizes z;
  z.dim = dim < 0 ? dim + x.dim() : dim;
  for (int64_t i = 0; i < x.dim(); ++i) {
    if (i == z.dim) {
      z.steps = x.size(i);
      continue;
    }
    (i < z.dim ? z.outer : z.inner) *= x.size(i);
    z.rest.push_back(x.size(i));
  }
  return z;
}
struct Plan { int64_t chunks, fwd, bwd; };
Plan plan_of(const Sizes& z, const Tensor& x) {
  Plan p;
  check(entry.gated_scan_plan(z.outer, z.steps, z.inner, type_of(x), &p.chunks, &p.fwd, &p.bwd), "sb_gated_scan_plan");
  return p;
}
bool scan_takes(const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& lengths, int64_t dim, int64_t form) {
  if (!plain(x) || !plain(gate) || x.numel() == 0 || gate.device() != x.device() || gate.sizes() != x.sizes() || dim < -x.dim() || dim >= x.dim() ||
      (gate.scalar_type() != x.scalar_type() && gate.scalar_type() != at::kFloat) || form < 0 || form > 1 || tangent(x) || tangent(gate) ||
      tangent(or_none(h0)))
    return false;
  const Sizes z = sizes_of(x, dim);
  if (given(h0) && (!plain(*h0) || h0->scalar_type() != at::kFloat || h0->device() != x.device() || h0->sizes() != z.rest)) return false;
  return !given(lengths) || (lengths->is_cuda() && lengths->layout() == at::kStrided && lengths->device() == x.device() &&
                             lengths->sizes() == x.sizes().slice(0, z.dim) && (lengths->scalar_type() == at::kLong || lengths->scalar_type() == at::kInt));
}
std::pair<Tensor, Tensor> scan_fwd(const Tensor& x, const Tensor& gate, const Tensor& h0_, const Tensor& lengths, const Sizes& z, int64_t form,
                                   bool reverse, Tensor* states) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Plan p = plan_of(z, x);
  Tensor h = dense_like(x), last = f32(x, z.rest), scratch;
  if (states) *states = f32(x, {p.chunks * z.outer * z.inner});
  if (p.fwd) scratch = f32(x, {p.fwd});
  const Steps xs = steps_of(x, z), gs = steps_of(gate, z);
  const Tensor h0 = h0_.defined() ? h0_.contiguous() : h0_;
  sb_gated_scan_args a = {};
  a.outer = z.outer; a.steps = z.steps; a.inner = z.inner;
  a.xtype = type_of(x); a.gtype = type_of(gate); a.form = (int)form; a.reverse = reverse;
  a.x = ptr(xs.t); a.so_x = xs.so; a.st_x = xs.st;
  a.gate = ptr(gs.t); a.so_g = gs.so; a.st_g = gs.st;
  a.h0 = ptr<float>(h0); a.len = ptr<int64_t>(lengths); a.h = ptr(h); a.h_last = ptr<float>(last);
  a.states = states ? ptr<float>(*states) : nullptr; a.scratch = ptr<float>(scratch);
  check(entry.gated_scan_fwd(&a, stream_of(x)), "sb_gated_scan_fwd");
  return {h, last};
}
struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& lengths, int64_t dim, int64_t form,
                               bool reverse) {
    Tensor states;
    const auto [h, last] = scan_fwd(x, gate, or_none(h0), or_none(lengths), sizes_of(x, dim), form, reverse, &states);
    ctx->save_for_backward({x, gate, states, or_none(lengths)});
    ctx->saved_data["how"] = dim * 4 + form * 2 + (int64_t)reverse;
    ctx->saved_data["need"] = (int64_t)(x.requires_grad() | gate.requires_grad() << 1 | (given(h0) && h0->requires_grad()) << 2);
    ctx->set_materialize_grads(false);
    return {h, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate = saved[1], &states = saved[2], &lengths = saved[3];
    const int64_t need = ctx->saved_data["need"].toInt(), how = ctx->saved_data["how"].toInt();
    const c10::OptionalDeviceGuard guard(x.device());
    const Sizes z = sizes_of(x, how >> 2);
    const Plan p = plan_of(z, x);
    Tensor dx = dense_like(x), dgate = dense_like(gate), dh0, scratch;
    if (need & 4) dh0 = f32(x, z.rest);
    if (p.bwd) scratch = f32(x, {p.bwd});
    const Steps xs = steps_of(x, z), gs = steps_of(gate, z);
    Steps ds = {};
    if (grads[0].defined()) {
      TORCH_CHECK(grads[0].scalar_type() == x.scalar_type() && grads[0].sizes() == x.sizes() && grads[0].device() == x.device(),
                  "gated_scan: the gradient does not fit");
      ds = steps_of(grads[0].resolve_neg(), z);
    }
    Tensor dlast;
    if (grads[1].defined()) {
      TORCH_CHECK(grads[1].scalar_type() == at::kFloat && grads[1].sizes() == z.rest && grads[1].device() == x.device(), "gated_scan: the gradient does not fit");
      dlast = grads[1].resolve_neg().contiguous();
    }
    sb_gated_scan_bwd_args a = {};
    a.outer = z.outer; a.steps = z.steps; a.inner = z.inner;
    a.xtype = type_of(x); a.gtype = type_of(gate); a.form = how >> 1 & 1; a.reverse = how & 1;
    a.x = ptr(xs.t); a.so_x = xs.so; a.st_x = xs.st;
    a.gate = ptr(gs.t); a.so_g = gs.so; a.st_g = gs.st;
    a.dh = ptr(ds.t); a.so_d = ds.so; a.st_d = ds.st; a.dlast = ptr<float>(dlast);
    a.len = ptr<int64_t>(lengths); a.states = ptr<float>(states);
    a.dx = ptr(dx); a.dgate = ptr(dgate); a.dh0 = ptr<float>(dh0); a.scratch = ptr<float>(scratch);
    check(entry.gated_scan_bwd(&a, stream_of(x)), "sb_gated_scan_bwd");
    Tensor through = x.requires_grad() ? x : gate;
    for (const Tensor& g : grads)
      if (g.defined() && g.requires_grad()) through = g;
    if (need & 1) out[0] = once(dx, through);
    if (need & 2) out[1] = once(dgate, through);
    out[2] = once(dh0, through);
    return out;
  }
};
std::vector<Tensor> gated_scan(const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& lengths_, int64_t dim, int64_t form, bool reverse) {
  if (!scan_takes(x, gate, h0, lengths_, dim, form)) return {};
  Maybe lengths;
  if (given(lengths_)) {
    const c10::OptionalDeviceGuard guard(x.device());
    lengths = lengths_->to(at::kLong).contiguous();
  }
  const Sizes z = sizes_of(x, dim);
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (given(h0) && h0->requires_grad()))) {
    const Tensor first = or_none(h0);
    refuse_held_leaves({&x, &gate, &first}, x);
    return GatedScan::apply(x, gate, h0, lengths, z.dim, form, reverse);
  }
  const auto [h, last] = scan_fwd(x, gate, or_none(h0), or_none(lengths), z, form, reverse, nullptr);
  return {h, last};
}
// rows of a step's input; a copy where they lie on the state's memory in another order, in which other threads write it
std::pair<Tensor, int64_t> rows_beside(const Tensor& t, const Tensor& state, int64_t n) {
  auto got = rows_of(t, n);
  const auto& [r, ld] = got;
  const char *at = (const char*)r.data_ptr(), *to = (const char*)state.data_ptr();
  const int64_t size = ((t.numel() / n - 1) * ld + n) * r.element_size();
  if (at < to + state.nbytes() && to < at + size && !(at == to && ld == n && r.scalar_type() == at::kFloat)) got = {t.clone(at::MemoryFormat::Contiguous), n};
  return got;
}
std::vector<Tensor> gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state, int64_t form) {
  if (!plain(x) || !plain(gate) || !plain(state) || x.numel() == 0 || x.dim() < 1 || gate.sizes() != x.sizes() || state.sizes() != x.sizes() ||
      gate.device() != x.device() || state.device() != x.device() || (gate.scalar_type() != x.scalar_type() && gate.scalar_type() != at::kFloat) ||
      state.scalar_type() != at::kFloat || !state.is_contiguous() || form < 0 || form > 1 || tangent(x) || tangent(gate) || tangent(state) ||
      (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || state.requires_grad())))
    return {};
  const c10::OptionalDeviceGuard guard(x.device());
  const int64_t n = x.size(-1);
  Tensor y = dense_like(x);
  const auto [xr, ldx] = rows_beside(x, state, n);
  const auto [gr, ldg] = rows_beside(gate, state, n);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  check(entry.gated_scan_step(ptr(xr), ptr(gr), ptr<float>(state), ptr(y), x.numel() / n, n, ldx, ldg, type_of(x), type_of(gate), (int)form, stream_of(x)),
        "sb_gated_scan_step");
  return {y};
}

// ---- AdamW ----
using Tensors = std::vector<const Tensor*>;      // (the caller's)
struct AdamwCall {
  Tensors params, grads, state;      // state: exp_avg, exp_avg_sq, their scales (8 bits), master (16-bit parameters)
  int64_t bits, step;
  Maybe step_dev, lr_dev;
  double lr, beta1, beta2, eps, weight_decay, gscale, clip;
  uint32_t seed;
  const void* guard_word; void* skipped;
};
// 1: done, 0: not taken (nothing has been touched)
int adamw_step(const AdamwCall& call) {
  const auto& [params, grads, state, bits, step, step_dev, lr_dev, lr, beta1, beta2, eps, weight_decay, gscale, clip, seed, guard_word, skipped] = call;
  const size_t count = params.size();
  if (count == 0 || count != grads.size() || !plain(*params[0])) return 0;
  const auto device = params[0]->device();
  const auto ptype = params[0]->scalar_type(), gtype = grads[0]->scalar_type();
  if (gtype != ptype && gtype != at::kFloat) return 0;
  int64_t blocks = 0;
  for (size_t i = 0; i < count; ++i) {      // (one pair of types, a gradient for each: the usual call)
    const Tensor &p = *params[i], &g = *grads[i];
    if (!plain(p) || !plain(g) || p.device() != device || g.device() != device || p.scalar_type() != ptype || g.scalar_type() != gtype ||
        p.sizes() != g.sizes() || p.numel() == 0 || !p.is_contiguous() || !g.is_contiguous())
      return 0;
    blocks += (p.numel() + SB_ADAMW_BLOCK - 1) / SB_ADAMW_BLOCK;
  }
  std::vector<std::pair<const char*, const char*>> places(count);      // (no two may share memory: their workgroups would race)
  for (size_t i = 0; i < count; ++i) {
    const char* at = (const char*)params[i]->data_ptr();
    places[i] = {at, at + params[i]->nbytes()};
  }
  std::sort(places.begin(), places.end());
  for (size_t i = 1; i < count; ++i)
    if (places[i].first < places[i - 1].second) return 0;
  const auto rate = [](double v) { return v >= 0 && v < 1; };
  if (!rate(beta1) || !rate(beta2) || !(eps >= 0)) return 0;
  const size_t buffers = (bits == 8 ? 4 : 2) + (ptype != at::kFloat);
  const size_t slots_per = SB_ADAMW_NORM_SLOTS / ((count + SB_ADAMW_MAX - 1) / SB_ADAMW_MAX);
  if ((bits != 8 && bits != 32) || state.size() != buffers || blocks >= (1LL << 31) || slots_per == 0 || !(clip >= 0)) return 0;
  for (size_t i = 0; i < buffers; ++i) {
    const Tensor& t = *state[i];
    const bool scale = bits == 8 && (i == 2 || i == 3);
    const auto want = i + 1 == buffers && ptype != at::kFloat ? at::kFloat : bits == 32 ? at::kFloat : scale ? at::kFloat8_e8m0fnu : i == 0 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2;
    if (!t.defined() || t.device() != device || t.layout() != at::kStrided || t.scalar_type() != want || !t.is_contiguous() ||
        t.numel() != (scale ? blocks : blocks * SB_ADAMW_BLOCK) || (uintptr_t)t.data_ptr() % 16)
      return 0;
  }
  if (given(step_dev) ? !(step_dev->is_cuda() && step_dev->device() == device && step_dev->scalar_type() == at::kInt && step_dev->numel() == 1) : step < 1 || step >= (1LL << 31))
    return 0;
  if (given(lr_dev) && !(lr_dev->is_cuda() && lr_dev->device() == device && lr_dev->scalar_type() == at::kFloat && lr_dev->numel() == 1)) return 0;
  const c10::OptionalDeviceGuard guard(device);
  for (const Tensor* p : params) p->unsafeGetTensorImpl()->bump_version();
  sb_adamw_args a = {};
  a.ptype = type_of(*params[0]); a.gtype = type_of(*grads[0]); a.bits = (int)bits;
  a.m = ptr(*state[0]); a.v = ptr(*state[1]);
  if (bits == 8) {
    a.m_scale = ptr(*state[2]);
    a.v_scale = ptr(*state[3]);
  }
  if (ptype != at::kFloat) a.master = ptr<float>(*state[buffers - 1]);
  a.lr = lr; a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.weight_decay = weight_decay;
  a.lr_dev = given(lr_dev) ? ptr<float>(*lr_dev) : nullptr;
  a.step_dev = given(step_dev) ? ptr<int32_t>(*step_dev) : nullptr;
  a.step = (int32_t)step; a.seed = seed;
  a.gscale = (float)gscale; a.clip = (float)clip;
  a.guard = (const int*)guard_word; a.skipped = (int*)skipped;
  void* stream = stream_of(*params[0]);
  const int64_t chunk = entry.adamw_chunk();
  Tensor part;
  if (clip > 0) {
    part = at::empty({SB_ADAMW_NORM_SLOTS}, params[0]->options().dtype(at::kDouble));
    a.norm_part = (const double*)part.data_ptr();
    a.norm_slots = (int)(slots_per * ((count + SB_ADAMW_MAX - 1) / SB_ADAMW_MAX));
  }
  for (int pass = clip > 0 ? 0 : 1; pass < 2; ++pass) {      // the norm over all tensors comes first
    int64_t block = 0;
    for (size_t i0 = 0; i0 < count; i0 += SB_ADAMW_MAX) {
      const size_t n = std::min<size_t>(SB_ADAMW_MAX, count - i0);
      int64_t first = 0;
      for (size_t j = 0; j < n; ++j) {
        const Tensor& p = *params[i0 + j];
        a.t[j] = {p.data_ptr(), grads[i0 + j]->data_ptr(), p.numel(), (int32_t)block, (int32_t)first};
        block += (p.numel() + SB_ADAMW_BLOCK - 1) / SB_ADAMW_BLOCK;
        first += (p.numel() + chunk - 1) / chunk;
      }
      a.count = (int32_t)n;
      a.last = i0 + n == count;
      if (pass == 0)
        check(entry.adamw_norm(&a, (double*)part.data_ptr(), (int)(i0 / SB_ADAMW_MAX * slots_per), (int)slots_per, stream), "sb_adamw_norm");
      else
        check(entry.adamw_step(&a, stream), "sb_adamw_step");
    }
  }
  return 1;
}

struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};
bool tensors_of(PyObject* list, Tensors& out) {
  if (!PyList_Check(list)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(t)) return false;
    out.push_back(&THPVariable_Unpack(t));
  }
  return true;
}
// adamw_step(params, grads, state, bits, step, step_dev, lr, lr_dev, beta1, beta2, eps, weight_decay, gscale, clip, seed, guard, skipped) -> bool
PyObject* py_adamw_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 17, "adamw_step takes 17 arguments, got ", n);
  AdamwCall c;
  if (!tensors_of(args[0], c.params) || !tensors_of(args[1], c.grads) || !tensors_of(args[2], c.state)) Py_RETURN_FALSE;
  const auto maybe = [](PyObject* o) { return THPVariable_Check(o) ? Maybe(THPVariable_Unpack(o)) : Maybe(); };
  c.bits = PyLong_AsLongLong(args[3]);
  c.step = PyLong_AsLongLong(args[4]);
  c.step_dev = maybe(args[5]);
  c.lr_dev = maybe(args[7]);
  double* const to[] = {&c.lr, &c.beta1, &c.beta2, &c.eps, &c.weight_decay, &c.gscale, &c.clip};
  const int from[] = {6, 8, 9, 10, 11, 12, 13};
  for (int i = 0; i < 7; ++i) *to[i] = PyFloat_AsDouble(args[from[i]]);
  c.seed = (uint32_t)PyLong_AsUnsignedLongLong(args[14]);
  c.guard_word = PyLong_AsVoidPtr(args[15]);
  c.skipped = PyLong_AsVoidPtr(args[16]);
  if (PyErr_Occurred()) return nullptr;
  int done;
  {
    const WithoutGil without;
    done = adamw_step(c);
  }
  return PyBool_FromLong(done);
  END_HANDLE_TH_ERRORS
}

PyMethodDef functions[] = {{"adamw_step", (PyCFunction)(void*)py_adamw_step, METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "libsoundbubble_torch", nullptr, -1, functions, nullptr, nullptr, nullptr, nullptr};

}  // namespace

TORCH_LIBRARY(sound_bubble_seq, m) {
  m.def("bind(int[] addresses) -> ()", bind);
  m.def("refuse_held_leaves(Tensor[] leaves) -> ()", refuse_held);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor[]", layer_norm);
  m.def("gated_scan(Tensor x, Tensor gate, Tensor? h0, Tensor? lengths, int dim, int form, bool reverse) -> Tensor[]", gated_scan);
  m.def("gated_scan_step(Tensor x, Tensor gate, Tensor(a!) state, int form) -> Tensor[]", gated_scan_step);
}

PyMODINIT_FUNC PyInit_libsoundbubble_torch() { return PyModule_Create(&module); }
