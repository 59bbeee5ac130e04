// The dense layers' operators as torch sees them: checks of arguments, allocations, autograd nodes and the order of
// rows by expert, over the C ABI of libictc_mi355x.so.  The nodes are C++ ones because the engine runs a backward pass
// in a thread of its own: a node in Python costs two hand-overs of the interpreter's lock there, more than the kernels
// of a small layer take.  Work goes on the operand's current stream.
#include "torch_ops.h"

namespace {

// ---------------------------------------------------------------------------
// Layer norm
// ---------------------------------------------------------------------------

struct NormGrads {
  Tensor x, w, b;
};

NormGrads norm_backward(const Tensor& x_, const Tensor& w_, const Tensor& g_, const Tensor& stats, bool need_x,
                        bool need_w, bool need_b) {
  eager("layer_norm");
  const Tensor x = rows_of(x_), w = packed(w_), g = rows_of(g_);
  const int64_t N = x.size(0), C = x.size(1);
  const int dt = dtype_of(x);
  NormGrads out;
  Tensor ws;
  int64_t bytes = 0;
  if (need_x) out.x = at::empty({N, C}, x.options());
  if (need_w) out.w = at::empty({C}, x.options());
  if (need_b) out.b = at::empty({C}, x.options());
  if (need_w || need_b) {
    bytes = ictc_layer_norm_workspace_bytes(dt, N, (int)C);
    ws = floats(bytes / 4, x);
  }
  const float* st = stats.const_data_ptr<float>();
  done(ictc_layer_norm_bwd(dt, ptr(x), pitch(x), ptr(g), pitch(g), N, (int)C, ptr(w), st, st + N, ptr(out.x),
                           ptr(out.w), ptr(out.b), ptr(ws), bytes, stream_of(x)),
       "layer_norm");
  return out;
}

struct NormSeconds {
  Tensor x, w, g;
};

NormSeconds norm_backward2(const Tensor& x_, const Tensor& w_, const Tensor& g_, const Tensor& v_, const Tensor& vw_,
                           const Tensor& vb_, const Tensor& stats, bool need_x, bool need_w, bool need_g) {
  eager("layer_norm");
  const Tensor x = rows_of(x_), w = packed(w_), g = rows_of(g_), vw = packed(vw_), vb = packed(vb_);
  const Tensor v = v_.defined() ? rows_of(v_) : at::zeros_like(x, at::MemoryFormat::Contiguous);
  const int64_t N = x.size(0), C = x.size(1);
  const int dt = dtype_of(x);
  NormSeconds out;
  Tensor ws;
  int64_t bytes = 0;
  if (need_x) out.x = at::empty({N, C}, x.options());
  if (need_g) out.g = at::empty({N, C}, x.options());
  if (need_w) {
    out.w = at::empty({C}, x.options());
    bytes = ictc_layer_norm_workspace_bytes(dt, N, (int)C);
    ws = floats(bytes / 4, x);
  }
  const float* st = stats.const_data_ptr<float>();
  done(ictc_layer_norm_bwd2(dt, ptr(x), pitch(x), ptr(g), pitch(g), ptr(v), pitch(v), ptr(vw), ptr(vb), N, (int)C,
                            ptr(w), st, st + N, ptr(out.x), ptr(out.g), ptr(out.w), ptr(ws), bytes, stream_of(x)),
       "layer_norm");
  return out;
}

// The second derivative as a node of the graph, so that a third one raises wherever it would pass here.
struct LayerNormSecond : Function<LayerNormSecond> {
  static variable_list forward(AutogradContext*, const Tensor& x, const Tensor& g, const OptTensor& w,
                               const OptTensor& v, const OptTensor& vw, const OptTensor& vb, const Tensor& stats,
                               bool need_x, bool need_w, bool need_g) {
    const NormSeconds s =
        norm_backward2(x, value(w), g, value(v), value(vw), value(vb), stats, need_x, need_w, need_g);
    variable_list out;
    for (const Tensor& t : {s.x, s.w, s.g})
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "layer_norm: third derivatives are not supported");
  }
};

// (dx, dweight, dbias), those asked for, as functions of x, the output gradient g and the weight.
struct LayerNormGrad : Function<LayerNormGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const OptTensor& w,
                               const Tensor& stats, bool need_x, bool need_w, bool need_b) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, g, value(w), stats});
    ctx->saved_data["needs"] = (int64_t)(need_x | need_w << 1 | need_b << 2);
    const NormGrads s = norm_backward(x, value(w), g, stats, need_x, need_w, need_b);
    variable_list out;
    for (const Tensor& t : {s.x, s.w, s.b})
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &g = saved[1], &w = saved[2], &stats = saved[3];
    const int64_t needs = ctx->saved_data["needs"].toInt();
    Tensor v[3];
    size_t at = 0;
    for (int i = 0; i < 3; ++i)
      if (needs >> i & 1) v[i] = grads[at++];
    variable_list out(7);
    if (!v[0].defined() && !v[1].defined() && !v[2].defined()) return out;
    const std::vector<bool> want = wanted(ctx, {true, true, w.defined()});
    if (at::GradMode::is_enabled()) {
      const variable_list s =
          LayerNormSecond::apply(x, g, some(w), some(v[0]), some(v[1]), some(v[2]), stats, want[0], want[2], want[1]);
      size_t k = 0;
      if (want[0]) out[0] = s[k++];
      if (want[2]) out[2] = s[k++];
      if (want[1]) out[1] = s[k++];
    } else {
      const NormSeconds s = norm_backward2(x, w, g, v[0], v[1], v[2], stats, want[0], want[2], want[1]);
      out[0] = s.x;
      out[1] = s.g;
      out[2] = s.w;
    }
    return out;
  }
};

// stats: the rows' mean and 1 / deviation, or undefined
Tensor norm_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps, const Tensor& stats) {
  const Tensor x = rows_of(x_), w = packed(w_), b = packed(b_);
  const int64_t N = x.size(0), C = x.size(1);
  Tensor y = at::empty({N, C}, x.options());
  float* st = stats.defined() ? stats.mutable_data_ptr<float>() : nullptr;
  done(ictc_layer_norm_fwd(dtype_of(x), ptr(x), pitch(x), N, (int)C, ptr(w), ptr(b), (float)eps, ptr(y), st,
                           st ? st + N : nullptr, stream_of(x)),
       "layer_norm");
  return y;
}

struct LayerNorm : Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    const Tensor stats = floats(2 * x.size(0), x);
    ctx->save_for_backward({x, value(w), stats});
    ctx->saved_data["bias"] = b.has_value();
    return norm_forward(x, value(w), value(b), eps, stats);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const std::vector<bool> want = wanted(ctx, {true, w.defined(), ctx->saved_data["bias"].toBool()});
    variable_list out(4);
    if (!want[0] && !want[1] && !want[2]) return out;
    if (at::GradMode::is_enabled()) {   // the gradient will be differentiated
      const variable_list s = LayerNormGrad::apply(x, grads[0], some(w), stats,
                                                   want[0], want[1], want[2]);
      size_t k = 0;
      for (int i = 0; i < 3; ++i)
        if (want[i]) out[i] = s[k++];
    } else {
      const NormGrads s = norm_backward(x, w, grads[0], stats, want[0], want[1], want[2]);
      out[0] = s.x;
      out[1] = s.w;
      out[2] = s.b;
    }
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  eager("layer_norm");
  check_dense(x, "layer_norm", "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384,
                    "layer_norm: x must have a last axis of 1 to 16384 elements");
  const int64_t C = x.size(-1);
  for (const auto& [name, p] : {std::pair<const char*, const OptTensor*>("weight", &w), {"bias", &b}}) {
    if (!p->has_value()) continue;
    check_dense(**p, "layer_norm", name, &x);
    TORCH_CHECK_VALUE((*p)->dim() == 1 && (*p)->size(0) == C, "layer_norm: ", name, " must have shape [", C, "]");
  }
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "layer_norm: eps must be a finite number, zero or more");
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = x.dim() == 2 ? x : x.reshape({x.numel() / C, C}), wv = value(w), bv = value(b);
  const Tensor y = tracked({&rows, &wv, &bv}) ? LayerNorm::apply(rows, w, b, eps)
                                              : norm_forward(rows, wv, bv, eps, Tensor());
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---------------------------------------------------------------------------
// Expert linears
// ---------------------------------------------------------------------------

// (rows sorted by expert, first sorted row of each expert): what the kernels below take.
std::pair<Tensor, Tensor> expert_order(const Tensor& ids_, int64_t experts) {
  eager("expert_order");
  TORCH_CHECK_VALUE(ids_.is_cuda() && ids_.scalar_type() == at::kLong && ids_.dim() == 1,
                    "expert_order: ids must be an int64 vector on a ROCm (cuda) device");
  TORCH_CHECK_VALUE(experts >= 1 && experts <= 65535, "expert_order: experts must be an integer from 1 to 65535");
  TORCH_CHECK_VALUE(ids_.size(0) < (int64_t(1) << 31) - 2, "expert_order: up to 2^31 - 3 rows");
  const c10::DeviceGuard guard(ids_.device());
  return rows_by_id(packed(ids_), experts, "expert_order");
}

Tensor linear_rows(const Tensor& x_, const Tensor& W_, const Tensor& b_, const Tensor& perm, const Tensor& off,
                   bool trans) {
  eager("expert_linear");
  const Tensor x = rows_of(x_), W = packed(W_), b = packed(b_);
  const int64_t N = x.size(0), outputs = W.size(trans ? 2 : 1);
  Tensor out = at::empty({N, outputs}, x.options());
  done(ictc_expert_linear(dtype_of(x), ptr(x), pitch(x), N, (int)x.size(1), ptr(W), ptr(b), (int)outputs,
                          (int)W.size(0), perm.const_data_ptr<int>(), off.const_data_ptr<int>(), trans, ptr(out),
                          stream_of(x)),
       "expert_linear");
  return out;
}

// x: rows; or codes of them with their scales.
std::pair<Tensor, Tensor> linear_outer(const Tensor& g_, const Tensor& x_, const Tensor& perm, const Tensor& off,
                                       bool need_b, const Tensor& scales = Tensor()) {
  eager("expert_linear");
  const Tensor g = rows_of(g_);
  const int64_t N = g.size(0), M = g.size(1), K = x_.size(1), E = off.size(0) - 2;
  const int dt = dtype_of(g);
  const bool codes = scales.defined() && ictc_expert_outer_takes_codes(dt, ptr(g), pitch(g), N, (int)K, (int)M);
  const Tensor x = codes ? x_ : scales.defined() ? decode_rows(x_, scales, g.scalar_type()) : rows_of(x_);
  Tensor gW = at::empty({E, M, K}, g.options()), gb, ws;
  if (need_b) gb = at::empty({E, M}, g.options());
  const int64_t bytes = ictc_expert_outer_workspace_bytes(dt, N, (int)K, (int)M, (int)E);
  if (bytes > 0) ws = floats(bytes / 4, g);
  const int *p = perm.const_data_ptr<int>(), *o = off.const_data_ptr<int>();
  done(codes ? ictc_expert_outer_codes(dt, ptr(g), pitch(g), x.const_data_ptr<int8_t>(), scales.const_data_ptr<float>(), N,
                                       (int)K, (int)M, (int)E, p, o, ptr(gW), ptr(gb), ptr(ws), bytes, stream_of(g))
             : ictc_expert_outer(dt, ptr(g), pitch(g), ptr(x), pitch(x), N, (int)K, (int)M, (int)E, p, o, ptr(gW), ptr(gb),
                                 ptr(ws), bytes, stream_of(g)),
       "expert_linear");
  return {gW, gb};
}

struct ExpertOuter;

// y[n] = W[e] x[n] + b[e], or with trans W[e]^T x[n].  Its adjoints are the same map with the other orientation and
// ExpertOuter, whose adjoints are this map again: differentiable to any order.
struct ExpertLinear : Function<ExpertLinear> {
  // place, codes and scales: the rows are kept in 8 bits (torch_ops.h)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& W, const OptTensor& b,
                        const Tensor& perm, const Tensor& off, bool trans, const c10::IValue& place = c10::IValue(),
                        const Codes& kept = Codes()) {
    if (kept.codes.defined()) {
      ctx->save_for_backward({kept.codes, W, perm, off, kept.scales});
      ctx->saved_data["place"] = place;
    } else {
      ctx->save_for_backward({x, W, perm, off});
    }
    ctx->saved_data["trans"] = trans;
    ctx->saved_data["bias"] = b.has_value();
    return linear_rows(x, W, value(b), perm, off, trans);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

// Per expert the sum over its rows of g[n] x[n]^T and, need_b, the sum of g[n].
struct ExpertOuter : Function<ExpertOuter> {
  static variable_list forward(AutogradContext* ctx, const Tensor& g, const Tensor& x, const Tensor& perm,
                               const Tensor& off, bool need_b) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({g, x, perm, off});
    const auto [gW, gb] = linear_outer(g, x, perm, off, need_b);
    return need_b ? variable_list{gW, gb} : variable_list{gW};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &g = saved[0], &x = saved[1], &perm = saved[2], &off = saved[3];
    Tensor H = grads[0];
    const Tensor h = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(5);
    if (!H.defined() && !h.defined()) return out;
    if (!H.defined()) H = at::zeros({off.size(0) - 2, g.size(1), x.size(1)}, x.options());
    if (ctx->needs_input_grad(0))
      out[0] = ExpertLinear::apply(x, H, some(h), perm, off, false);
    if (ctx->needs_input_grad(1)) out[1] = ExpertLinear::apply(g, H, OptTensor(), perm, off, true);
    return out;
  }
};

variable_list ExpertLinear::backward(AutogradContext* ctx, variable_list grads) {
  const variable_list saved = ctx->get_saved_variables();
  const Tensor &W = saved[1], &perm = saved[2], &off = saved[3], &g = grads[0];
  const bool trans = ctx->saved_data["trans"].toBool();
  const std::vector<bool> want = wanted(ctx, {true, true, ctx->saved_data["bias"].toBool()});
  const bool again = at::GradMode::is_enabled();   // the gradient will be differentiated
  Tensor x = saved[0];
  const Tensor scales = saved.size() > 4 ? saved[4] : Tensor();   // (of codes, which are not transposed)
  if (scales.defined() && again && (want[1] || want[2]))
    x = Decoded::apply(ctx->saved_data["place"].toTensor(), saved[0], scales);
  variable_list out(8);
  if (want[0])
    out[0] = again ? ExpertLinear::apply(g, W, OptTensor(), perm, off, !trans)
                   : linear_rows(g, W, Tensor(), perm, off, !trans);
  if (want[1] || want[2]) {
    const Tensor &a = trans ? x : g, &b = trans ? g : x;
    if (again) {
      const variable_list s = ExpertOuter::apply(a, b, perm, off, want[2]);
      if (want[1]) out[1] = s[0];
      if (want[2]) out[2] = s[1];
    } else {
      auto [gW, gb] = linear_outer(a, b, perm, off, want[2], scales);
      if (want[1]) out[1] = gW;
      out[2] = gb;
    }
  }
  return out;
}

Tensor expert_linear(const Tensor& x, const Tensor& W, const OptTensor& b, const Tensor& perm, const Tensor& off,
                     int64_t rows, const std::optional<int64_t>& save_bits) {
  eager("expert_linear");
  check_dense(x, "expert_linear", "x");
  check_dense(W, "expert_linear", "weight", &x);
  TORCH_CHECK_VALUE(x.dim() == 2 && W.dim() == 3 && x.size(1) == W.size(2) && W.numel() > 0,
                    "expert_linear: expected x [N, inputs] and weight [experts, outputs, inputs]");
  TORCH_CHECK_VALUE(W.size(1) <= 65536 && W.size(2) <= 65536, "expert_linear: up to 65536 inputs and outputs");
  TORCH_CHECK_VALUE(rows == x.size(0) && off.size(0) - 2 == W.size(0) && perm.get_device() == x.get_device(),
                    "expert_linear: the order is of other rows, experts or another device");
  if (b.has_value()) {
    check_dense(*b, "expert_linear", "bias", &x);
    TORCH_CHECK_VALUE(b->dim() == 2 && b->size(0) == W.size(0) && b->size(1) == W.size(1),
                      "expert_linear: bias must have shape [experts, outputs]");
  }
  const bool eight = in_8_bits(save_bits, "expert_linear");
  const c10::DeviceGuard guard(x.device());
  const Tensor bv = value(b);
  if (!tracked({&x, &W, &bv})) return linear_rows(x, W, bv, perm, off, false);
  // (only the weights' gradient takes the rows)
  if (!eight || !W.requires_grad()) return ExpertLinear::apply(x, W, b, perm, off, false);
  return ExpertLinear::apply(x, W, b, perm, off, false, c10::IValue(Place8::apply(x)), encode_rows(x.detach()));
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------

constexpr int64_t kBlock = 256;

void check_moment(const Tensor& t, const char* name, at::ScalarType type, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == like.device() && t.is_contiguous(), "adamw: ", name,
                    " must be a contiguous ", type, " tensor on ", like.device());
}

void check_moments(const Tensor& m, const Tensor& v, const OptTensor& ms, const OptTensor& vs) {
  const bool eight = ms.has_value() || vs.has_value();
  TORCH_CHECK_VALUE(m.is_cuda(), "adamw: tensors must be on a ROCm (cuda) device");
  check_moment(m, "exp_avg", eight ? at::kFloat8_e4m3fn : at::kFloat, m);
  check_moment(v, "exp_avg_sq", eight ? at::kByte : at::kFloat, m);
  TORCH_CHECK_VALUE(m.numel() == v.numel(), "adamw: exp_avg and exp_avg_sq must have as many elements");
  if (!eight) return;
  TORCH_CHECK_VALUE(ms.has_value() && vs.has_value(), "adamw: moments in 8 bits have two scales");
  check_moment(*ms, "exp_avg_scale", at::kFloat, m);
  check_moment(*vs, "exp_avg_sq_scale", at::kFloat, m);
  TORCH_CHECK_VALUE(m.numel() % kBlock == 0 && ms->numel() * kBlock >= m.numel() && vs->numel() * kBlock >= m.numel(),
                    "adamw: 8-bit moments come in blocks of 256 elements with one scale each");
}

// Addresses and element counts of a list of tensors of one type on one device.
struct List {
  std::vector<int64_t> at, count;
  int dtype = -1;
};

List list_of(const std::vector<Tensor>& ts, const Tensor& like, const char* name) {
  List l;
  l.at.reserve(ts.size());
  l.count.reserve(ts.size());
  for (const Tensor& t : ts) {
    const int dt = dtype_of(t);
    TORCH_CHECK_VALUE(dt >= 0, "adamw: ", name, " must be float32, bfloat16 or float16");
    if (l.dtype < 0) l.dtype = dt;
    TORCH_CHECK_VALUE(dt == l.dtype && t.device() == like.device() && t.is_contiguous(), "adamw: ", name,
                      " must be contiguous, of one type and on one device");
    l.at.push_back((int64_t)t.data_ptr());
    l.count.push_back(t.numel());
  }
  return l;
}

// [0] the norm over the gradients, [1] the factor that holds it to max_norm (ictc_gradient_norm's workspace).
Tensor gradient_norm(const List& grads, double max_norm, const Tensor& like) {
  const int64_t bytes = ictc_gradient_norm_workspace_bytes((int)grads.at.size());
  const Tensor ws = floats(bytes / 4, like);
  done(ictc_gradient_norm(grads.dtype, (int)grads.at.size(), grads.at.data(), grads.count.data(), max_norm, ptr(ws),
                          bytes, stream_of(ws)),
       "adamw");
  return ws;
}

// One step of a list of parameters, whose moments begin at `starts` (empty: one behind another); the caller's lists.
struct Step {
  const std::vector<Tensor>&params, &grads;
  const Tensor &m, &v;
  const OptTensor &ms, &vs;
  const std::vector<int64_t>& starts;
  int64_t step;
  double lr, beta1, beta2, eps, decay;
};

struct Lists {
  List p, g;
};

// Everything that can be wrong with a step, found before anything of it is done.
Lists check_step(const Step& s) {
  check_moments(s.m, s.v, s.ms, s.vs);
  TORCH_CHECK_VALUE(s.params.size() == s.grads.size(), "adamw: as many gradients as parameters are needed");
  TORCH_CHECK_VALUE(s.starts.empty() || s.starts.size() == s.params.size(), "adamw: a segment per parameter is needed");
  const Lists l = {list_of(s.params, s.m, "parameters"), list_of(s.grads, s.m, "gradients")};
  TORCH_CHECK_VALUE(l.p.dtype == l.g.dtype, "adamw: gradients must have the type of their parameters");
  TORCH_CHECK_VALUE(l.p.count == l.g.count, "adamw: a gradient must have its parameter's shape");
  done(ictc_adamw_step(ICTC_F32, 32, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, s.lr,
                       s.beta1, s.beta2, s.eps, s.decay, s.step, nullptr, nullptr),   // (of no tensors: the numbers)
       "adamw");
  return l;
}

void launch_step(const Step& s, const Lists& l, const OptTensor& norm) {
  if (s.params.empty()) return;
  const c10::DeviceGuard guard(s.m.device());
  done(ictc_adamw_step(l.p.dtype, s.ms.has_value() ? 8 : 32, (int)s.params.size(), l.p.at.data(), l.g.at.data(),
                       l.p.count.data(), s.starts.empty() ? nullptr : s.starts.data(), ptr(s.m), ptr(s.v),
                       (float*)ptr(value(s.ms)), (float*)ptr(value(s.vs)), s.m.numel(), s.lr, s.beta1, s.beta2, s.eps,
                       s.decay, s.step, (const float*)ptr(value(norm)), stream_of(s.m)),
       "adamw");
  // what was read of these tensors before (a graph's saved inputs, copies of a weight) is out of date
  const auto changed = [](const Tensor& t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (const Tensor& t : s.params) changed(t);
  for (const Tensor& t : {s.m, s.v, value(s.ms), value(s.vs)}) changed(t);
}

// Gradients of one type share a norm's launch; the norms of several types are joined in FP64, and the factor made of them
// as ictc_gradient_norm makes it.
Tensor common_norm(const std::vector<List>& grads, double max_norm, const Tensor& like) {
  std::vector<Tensor> norms;
  for (const List& g : grads) norms.push_back(gradient_norm(g, max_norm, like));
  if (norms.empty()) return at::zeros({1}, like.options().dtype(at::kFloat));
  if (norms.size() == 1) return norms[0];
  for (Tensor& n : norms) n = n.narrow(0, 0, 4).view(at::kDouble).select(0, 1);   // (the FP64 norms)
  const Tensor norm = at::stack(norms).square().sum().sqrt();
  return at::stack({norm, at::clamp_max(max_norm / (norm + 1e-6), 1.0)}).to(at::kFloat);
}

// All steps with their gradients' common norm held to max_norm, which is returned; all are checked before the first is
// taken.
OptTensor take_steps(const std::vector<Step>& steps, const std::optional<double>& max_norm) {
  eager("adamw");
  TORCH_CHECK_VALUE(!max_norm.has_value() || *max_norm >= 0.0, "adamw: max_norm must be zero or more");
  std::vector<Lists> lists;
  std::vector<List> grads;   // of each type
  for (const Step& s : steps) {
    lists.push_back(check_step(s));
    const List& g = lists.back().g;
    if (!max_norm.has_value() || g.at.empty()) continue;
    TORCH_CHECK_VALUE(s.m.device() == steps[0].m.device(), "adamw: gradients of one norm must be on one device");
    size_t k = 0;
    while (k < grads.size() && grads[k].dtype != g.dtype) ++k;
    if (k == grads.size()) {
      grads.push_back(g);
      continue;
    }
    grads[k].at.insert(grads[k].at.end(), g.at.begin(), g.at.end());
    grads[k].count.insert(grads[k].count.end(), g.count.begin(), g.count.end());
  }
  OptTensor norm;
  if (max_norm.has_value() && !steps.empty()) {
    const c10::DeviceGuard guard(steps[0].m.device());
    norm = common_norm(grads, *max_norm, steps[0].m);
  }
  for (size_t i = 0; i < steps.size(); ++i) launch_step(steps[i], lists[i], norm);
  return norm.has_value() ? OptTensor(norm->select(0, 0)) : OptTensor();
}

OptTensor adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const Tensor& m,
                     const Tensor& v, const OptTensor& ms, const OptTensor& vs, int64_t step, double lr, double beta1,
                     double beta2, double eps, double decay, const std::optional<double>& max_norm) {
  const std::vector<int64_t> packed_starts;
  return take_steps({{params, grads, m, v, ms, vs, packed_starts, step, lr, beta1, beta2, eps, decay}}, max_norm);
}

using GroupStep = std::tuple<std::vector<Tensor>, std::vector<Tensor>, Tensor, Tensor, OptTensor, OptTensor,
                             std::vector<int64_t>, int64_t, double, double, double, double, double>;

OptTensor adamw_groups(const std::vector<GroupStep>& groups, const std::optional<double>& max_norm) {
  std::vector<Step> steps;
  for (const GroupStep& g : groups) steps.push_back(std::apply([](const auto&... part) -> Step { return {part...}; }, g));
  return take_steps(steps, max_norm);
}

std::pair<Tensor, Tensor> adamw_moments(const Tensor& m, const Tensor& v, const Tensor& ms, const Tensor& vs,
                                        at::ScalarType type) {
  eager("adamw");
  check_moments(m, v, ms, vs);
  const c10::DeviceGuard guard(m.device());
  const auto opts = m.options().dtype(type);
  Tensor mo = at::empty({m.numel()}, opts), vo = at::empty({m.numel()}, opts);
  const int dt = dtype_of(mo);
  TORCH_CHECK_VALUE(dt >= 0, "adamw: dtype must be float32, bfloat16 or float16");
  done(ictc_adamw_moments(dt, ptr(m), ptr(v), (const float*)ptr(ms), (const float*)ptr(vs), m.numel(), ptr(mo),
                          ptr(vo), stream_of(m)),
       "adamw");
  return {mo, vo};
}

}  // namespace

void bind_layers(pybind11::module_& mod);   // torch_layers.cpp

PYBIND11_MODULE(ictc_torch, mod) {
  // Launches may wait for room in a queue: other Python threads run meanwhile.
  using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
  mod.def("layer_norm", &layer_norm, Free());
  mod.def("expert_order", &expert_order, Free());
  mod.def("expert_linear", &expert_linear, pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("bias"),
          pybind11::arg("perm"), pybind11::arg("offsets"), pybind11::arg("rows"),
          pybind11::arg("save_bits") = pybind11::none(), Free());
  mod.def("adamw_step", &adamw_step, Free());
  mod.def("adamw_groups", &adamw_groups, Free());
  mod.def("adamw_moments", &adamw_moments, Free());
  bind_layers(mod);
}
