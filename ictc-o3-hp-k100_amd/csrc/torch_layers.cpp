// Embedding, group norm and 8-bit activations as torch sees them: checks, allocations and autograd nodes over the C ABI (see torch_ops.cpp).
#include "torch_ops.h"

namespace {

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------

Tensor embedding_rows(const Tensor& table_, const Tensor& ids, double scale) {
  eager("embedding");
  const c10::DeviceGuard guard(table_.device());
  const Tensor table = packed(table_);
  Tensor out = at::empty({ids.size(0), table.size(1)}, table.options());
  done(ictc_embedding_fwd(dtype_of(table), ptr(table), table.size(0), (int)table.size(1),
                          ids.const_data_ptr<int64_t>(), ids.size(0), (float)scale, ptr(out), stream_of(table)),
       "embedding");
  return out;
}

Tensor embedding_sums(const Tensor& g_, const Tensor& ids, const Tensor& perm_, const Tensor& off_, int64_t entries,
                      double scale) {
  eager("embedding");
  const c10::DeviceGuard guard(g_.device());
  const Tensor g = rows_of(g_);
  const int64_t N = g.size(0), C = g.size(1);
  const int dt = dtype_of(g);
  Tensor perm = perm_, off = off_, ws;
  if (!perm.defined() && ictc_embedding_needs_order(N)) std::tie(perm, off) = rows_by_id(ids, entries, "embedding");
  Tensor out = at::empty({entries, C}, g.options());
  const int64_t bytes = ictc_embedding_bwd_workspace_bytes(dt, N, entries, (int)C);
  if (bytes > 0) ws = floats(bytes / 4, g);
  done(ictc_embedding_bwd(dt, ptr(g), pitch(g), N, (int)C, ids.const_data_ptr<int64_t>(), entries, (const int*)ptr(perm),
                          (const int*)ptr(off), (float)scale, ptr(out), ptr(ws), bytes, stream_of(g)),
       "embedding");
  return out;
}

struct EmbeddingGrad;

// rows = scale table[ids].  Its adjoint is EmbeddingGrad, whose adjoint is this map again: differentiable to any order.
struct Embedding : Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, const OptTensor& perm,
                        const OptTensor& off, double scale) {
    ctx->save_for_backward({ids, value(perm), value(off)});
    ctx->saved_data["entries"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    return embedding_rows(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbeddingGrad : Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& g, const Tensor& ids, const OptTensor& perm,
                        const OptTensor& off, int64_t entries, double scale) {
    ctx->save_for_backward({ids, value(perm), value(off)});
    ctx->saved_data["scale"] = scale;
    return embedding_sums(g, ids, value(perm), value(off), entries, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    const double scale = ctx->saved_data["scale"].toDouble();
    out[0] = at::GradMode::is_enabled() ? Embedding::apply(grads[0], saved[0], some(saved[1]), some(saved[2]), scale)
                                        : embedding_rows(grads[0], saved[0], scale);
    return out;
  }
};

variable_list Embedding::backward(AutogradContext* ctx, variable_list grads) {
  const variable_list saved = ctx->get_saved_variables();
  const int64_t entries = ctx->saved_data["entries"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  variable_list out(5);
  out[0] = at::GradMode::is_enabled()
               ? EmbeddingGrad::apply(grads[0], saved[0], some(saved[1]), some(saved[2]), entries, scale)
               : embedding_sums(grads[0], saved[0], saved[1], saved[2], entries, scale);
  return out;
}

Tensor embedding(const Tensor& table, const Tensor& ids, double scale, const OptTensor& perm, const OptTensor& off) {
  eager("embedding");
  check_dense(table, "embedding", "table");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1 && table.size(1) <= 65536,
                    "embedding: table must have shape [entries, width], a width of 1 to 65536");
  TORCH_CHECK_VALUE(ids.is_cuda() && ids.scalar_type() == at::kLong && ids.get_device() == table.get_device(),
                    "embedding: ids must be int64 and on ", table.device());
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "embedding: scale must be a finite number");
  const int64_t N = ids.numel();
  TORCH_CHECK_VALUE(N < (int64_t(1) << 31) - 2 && table.size(0) < (int64_t(1) << 31) - 2,
                    "embedding: up to 2^31 - 3 ids and entries");
  if (perm.has_value())
    TORCH_CHECK_VALUE(off->size(0) - 2 == table.size(0) && perm->size(0) == std::max<int64_t>(N, 1) &&
                          perm->get_device() == table.get_device(),
                      "embedding: the order is of other ids, entries or another device");
  const c10::DeviceGuard guard(table.device());
  const Tensor flat = ids.dim() == 1 && ids.is_contiguous() ? ids : ids.reshape({N}).contiguous();
  const Tensor y = tracked({&table}) ? Embedding::apply(table, flat, perm, off, scale) : embedding_rows(table, flat, scale);
  if (ids.dim() == 1) return y;
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  return y.view(shape);
}

// ---------------------------------------------------------------------------
// Group norm
// ---------------------------------------------------------------------------

struct NormShape {
  int64_t samples, positions, groups;
  int channels;
  bool silu;
  int64_t units() const { return samples * groups; }
};

// Of a sample's groups: means and 1 / deviations [2 units], and where it counts what their rounding left of the means [units].
struct Stats {
  Tensor both, rest;
  float* mean() const { return both.defined() ? both.mutable_data_ptr<float>() : nullptr; }
  float* rstd(const NormShape& n) const { return both.defined() ? mean() + n.units() : nullptr; }
  float* left() const { return rest.defined() ? rest.mutable_data_ptr<float>() : nullptr; }
};

// What a backward pass has of x [samples, positions, channels]: itself, or codes and scales of its rows of channels.
struct Kept {
  Tensor x, codes, scales;
  const int8_t* code() const { return codes.defined() ? codes.const_data_ptr<int8_t>() : nullptr; }
  const float* scale() const { return scales.defined() ? scales.const_data_ptr<float>() : nullptr; }
};

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

struct GroupGrads {
  Tensor x, w, b;
};

GroupGrads group_backward(const Kept& kept, const Tensor& g_, const Tensor& w_, const Tensor& b_, const Stats& stats,
                          const NormShape& n, bool need_x, bool need_w, bool need_b) {
  eager("group_norm");
  const c10::DeviceGuard guard(g_.device());
  const Tensor x = packed(kept.x), g = packed(g_), w = packed(w_), b = packed(b_);
  const int dt = dtype_of(g);
  GroupGrads out;
  if (need_x) out.x = at::empty(g.sizes(), g.options());
  if (need_w) out.w = at::empty({n.channels}, g.options());
  if (need_b) out.b = at::empty({n.channels}, g.options());
  const int64_t bytes = ictc_group_norm_workspace_bytes(dt, 1, n.samples, n.positions, n.channels, (int)n.groups);
  const Tensor ws = workspace(bytes, g);
  done(ictc_group_norm_bwd_rest(dt, ptr(x), kept.code(), kept.scale(), ptr(g), n.samples, n.positions, n.channels,
                                (int)n.groups, ptr(w), ptr(b), n.silu, stats.mean(), stats.left(), stats.rstd(n),
                                ptr(out.x), ptr(out.w), ptr(out.b), ptr(ws), bytes, stream_of(g)),
       "group_norm");
  return out;
}

struct GroupSeconds {
  Tensor x, g, w, b;
};

GroupSeconds group_backward2(const Kept& kept, const Tensor& g_, const Tensor& w_, const Tensor& b_, const Tensor& v_,
                             const Tensor& vw_, const Tensor& vb_, const Stats& stats, const NormShape& n, bool need_x,
                             bool need_g, bool need_w, bool need_b) {
  eager("group_norm");
  const c10::DeviceGuard guard(g_.device());
  const Tensor x = packed(kept.x), g = packed(g_), w = packed(w_), b = packed(b_), vw = packed(vw_), vb = packed(vb_);
  const Tensor v = v_.defined() ? packed(v_) : at::zeros(g.sizes(), g.options());
  const int dt = dtype_of(g);
  GroupSeconds out;
  if (need_x) out.x = at::empty(g.sizes(), g.options());
  if (need_g) out.g = at::empty(g.sizes(), g.options());
  if (need_w) out.w = at::empty({n.channels}, g.options());
  if (need_b) out.b = at::empty({n.channels}, g.options());
  const int64_t bytes = ictc_group_norm_workspace_bytes(dt, 2, n.samples, n.positions, n.channels, (int)n.groups);
  const Tensor ws = workspace(bytes, g);
  done(ictc_group_norm_bwd2_rest(dt, ptr(x), kept.code(), kept.scale(), ptr(g), ptr(v), ptr(vw), ptr(vb), n.samples,
                                 n.positions, n.channels, (int)n.groups, ptr(w), ptr(b), n.silu, stats.mean(),
                                 stats.left(), stats.rstd(n), ptr(out.x), ptr(out.g), ptr(out.w), ptr(out.b), ptr(ws),
                                 bytes, stream_of(g)),
       "group_norm");
  return out;
}

// The second derivative as a node of the graph, so that a third one raises wherever it would pass here.
struct GroupNormSecond : Function<GroupNormSecond> {
  static variable_list forward(AutogradContext*, const OptTensor& place, const Tensor& g, const OptTensor& w,
                               const OptTensor& b, const OptTensor& v, const OptTensor& vw, const OptTensor& vb,
                               const Kept& kept, const Stats& stats, const NormShape& n, bool need_x, bool need_g,
                               bool need_w, bool need_b) {
    const GroupSeconds s = group_backward2(kept, g, value(w), value(b), value(v), value(vw), value(vb), stats, n, need_x,
                                           need_g, need_w, need_b);
    variable_list out;
    for (const Tensor& t : {s.x, s.g, s.w, s.b})
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "group_norm: third derivatives are not supported");
  }
};

void keep(AutogradContext* ctx, const NormShape& n) {
  ctx->saved_data["samples"] = n.samples;
  ctx->saved_data["positions"] = n.positions;
  ctx->saved_data["groups"] = n.groups;
  ctx->saved_data["channels"] = (int64_t)n.channels;
  ctx->saved_data["silu"] = n.silu;
}

NormShape kept_shape(AutogradContext* ctx) {
  auto& d = ctx->saved_data;
  return {d["samples"].toInt(), d["positions"].toInt(), d["groups"].toInt(), (int)d["channels"].toInt(),
          d["silu"].toBool()};
}

// (dx, dweight, dbias), those asked for, as functions of x (in 8 bits: of its place), the output gradient g, the weight and
// the bias.
struct GroupNormGrad : Function<GroupNormGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const OptTensor& w,
                               const OptTensor& b, const Kept& kept, const Stats& stats, const NormShape& n, bool need_x,
                               bool need_w, bool need_b) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, g, value(w), value(b), stats.both, stats.rest, kept.codes, kept.scales});
    ctx->saved_data["needs"] = (int64_t)(need_x | need_w << 1 | need_b << 2);
    keep(ctx, n);
    const GroupGrads s = group_backward(kept, g, value(w), value(b), stats, n, need_x, need_w, need_b);
    variable_list out;
    for (const Tensor& t : {s.x, s.w, s.b})
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &g = saved[1], &w = saved[2], &b = saved[3];
    const Stats stats = {saved[4], saved[5]};
    const bool eight = saved[6].defined();
    const Kept kept = {eight ? Tensor() : x, saved[6], saved[7]};
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const NormShape n = kept_shape(ctx);
    Tensor v[3];
    size_t at = 0;
    for (int i = 0; i < 3; ++i)
      if (needs >> i & 1) v[i] = grads[at++];
    variable_list out(10);
    if (!v[0].defined() && !v[1].defined() && !v[2].defined()) return out;
    const std::vector<bool> want = wanted(ctx, {true, true, w.defined(), b.defined()});
    if (at::GradMode::is_enabled()) {
      const variable_list s = GroupNormSecond::apply(some(x), g, some(w), some(b), some(v[0]), some(v[1]), some(v[2]), kept,
                                                     stats, n, want[0], want[1], want[2], want[3]);
      size_t k = 0;
      for (int i = 0; i < 4; ++i)
        if (want[i]) out[i] = s[k++];
    } else {
      const GroupSeconds s = group_backward2(kept, g, w, b, v[0], v[1], v[2], stats, n, want[0], want[1], want[2], want[3]);
      out[0] = s.x;
      out[1] = s.g;
      out[2] = s.w;
      out[3] = s.b;
    }
    return out;
  }
};

// stats: may be undefined
Tensor group_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps, const Stats& stats,
                     const NormShape& n, const Codes& codes = Codes()) {
  const Tensor x = packed(x_), w = packed(w_), b = packed(b_);
  Tensor y = at::empty(x.sizes(), x.options());
  const int64_t bytes =
      ictc_group_norm_workspace_bytes(dtype_of(x), 0, n.samples, n.positions, n.channels, (int)n.groups);
  const Tensor ws = workspace(bytes, x);
  done(ictc_group_norm_fwd_rest(dtype_of(x), ptr(x), n.samples, n.positions, n.channels, (int)n.groups, ptr(w), ptr(b),
                                (float)eps, n.silu, ptr(y), stats.mean(), stats.left(), stats.rstd(n),
                                (int8_t*)ptr(codes.codes), (float*)ptr(codes.scales), ptr(ws), bytes, stream_of(x)),
       "group_norm");
  return y;
}

struct GroupNorm : Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                        const NormShape& n, const c10::IValue& place) {
    Stats stats = {floats(2 * n.units(), x), Tensor()};
    Codes codes;
    if (!place.isNone()) {
      ctx->saved_data["place"] = place;
      codes = empty_codes(n.samples * n.positions, n.channels, x);
    } else if (ictc_group_norm_keeps_rest(dtype_of(x), n.samples, n.positions, n.channels, (int)n.groups)) {
      stats.rest = floats(n.units(), x);
    }
    ctx->save_for_backward({codes.codes.defined() ? Tensor() : x, value(w), value(b), stats.both, stats.rest, codes.codes,
                            codes.scales});
    keep(ctx, n);
    return group_forward(x, value(w), value(b), eps, stats, n, codes);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &w = saved[1], &b = saved[2];
    const Stats stats = {saved[3], saved[4]};
    const Kept kept = {saved[0], saved[5], saved[6]};
    const NormShape n = kept_shape(ctx);
    const std::vector<bool> want = wanted(ctx, {true, w.defined(), b.defined()});
    variable_list out(6);
    if (!want[0] && !want[1] && !want[2]) return out;
    if (at::GradMode::is_enabled()) {   // the gradient will be differentiated
      const Tensor x = kept.codes.defined() ? ctx->saved_data["place"].toTensor() : kept.x;
      const variable_list s = GroupNormGrad::apply(x, grads[0], some(w), some(b), kept, stats, n, want[0], want[1], want[2]);
      size_t k = 0;
      for (int i = 0; i < 3; ++i)
        if (want[i]) out[i] = s[k++];
    } else {
      const GroupGrads s = group_backward(kept, grads[0], w, b, stats, n, want[0], want[1], want[2]);
      out[0] = s.x;
      out[1] = s.w;
      out[2] = s.b;
    }
    return out;
  }
};

Tensor group_norm(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps,
                  const std::optional<std::string>& activation, const std::optional<int64_t>& save_bits) {
  eager("group_norm");
  check_dense(x, "group_norm", "x");
  TORCH_CHECK_VALUE(x.dim() >= 2 && x.size(-1) >= 1 && x.size(-1) <= 65536,
                    "group_norm: x must have shape [samples, ..., channels], 1 to 65536 channels");
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(groups >= 1 && C % groups == 0, "group_norm: groups must divide the ", C, " channels");
  for (const auto& [name, p] : {std::pair<const char*, const OptTensor*>("weight", &w), {"bias", &b}}) {
    if (!p->has_value()) continue;
    check_dense(**p, "group_norm", name, &x);
    TORCH_CHECK_VALUE((*p)->dim() == 1 && (*p)->size(0) == C, "group_norm: ", name, " must have shape [", C, "]");
  }
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "group_norm: eps must be a finite number, zero or more");
  TORCH_CHECK_VALUE(!activation.has_value() || *activation == "silu", "group_norm: activation must be 'silu' or None");
  const bool eight = in_8_bits(save_bits, "group_norm");
  const c10::DeviceGuard guard(x.device());
  int64_t positions = 1;
  for (int64_t i = 1; i + 1 < x.dim(); ++i) positions *= x.size(i);
  const NormShape n = {x.size(0), positions, groups, (int)C, activation.has_value()};
  const Tensor wv = value(w), bv = value(b);
  if (!tracked({&x, &wv, &bv})) return group_forward(x, wv, bv, eps, Stats(), n);
  return GroupNorm::apply(x, w, b, eps, n, eight ? c10::IValue(Place8::apply(x)) : c10::IValue());
}

// ---------------------------------------------------------------------------
// Activations in 8 bits
// ---------------------------------------------------------------------------

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> out = sizes.vec();
  out.back() = last;
  return out;
}

std::pair<Tensor, Tensor> encode_activations(const Tensor& x) {
  eager("encode_activations");
  check_dense(x, "encode_activations", "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= std::numeric_limits<int>::max(),
                    "encode_activations: x must have a last axis of 1 to 2^31 - 1 elements");
  const int64_t C = x.size(-1);
  const Codes k = encode_rows(x.detach().reshape({x.numel() / C, C}));
  return {k.codes.view(x.sizes()), k.scales.view(with_last(x.sizes(), k.scales.size(1)))};
}

Tensor decode_activations(const Tensor& codes, const Tensor& scales, at::ScalarType type) {
  eager("decode_activations");
  TORCH_CHECK_VALUE(codes.is_cuda() && codes.scalar_type() == at::kChar && codes.dim() >= 1 && codes.size(-1) >= 1 &&
                        codes.size(-1) <= std::numeric_limits<int>::max(),
                    "decode_activations: codes must be int8 on a ROCm (cuda) device");
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat && scales.device() == codes.device() &&
                        scales.sizes() == with_last(codes.sizes(), (codes.size(-1) + 127) / 128),
                    "decode_activations: scales must be float32, one for each 128 codes of a row, and on ",
                    codes.device());
  TORCH_CHECK_VALUE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
                    "decode_activations: dtype must be float32, bfloat16 or float16");
  const int64_t C = codes.size(-1), N = codes.numel() / C;
  const c10::DeviceGuard guard(codes.device());
  return decode_rows(codes.reshape({N, C}).contiguous(), scales.reshape({N, (C + 127) / 128}).contiguous(), type)
      .view(codes.sizes());
}

}  // namespace

void bind_layers(pybind11::module_& mod) {
  using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
  mod.def("embedding", &embedding, Free());
  mod.def("group_norm", &group_norm, Free());
  mod.def("encode_activations", &encode_activations, Free());
  mod.def("decode_activations", &decode_activations, Free());
}
