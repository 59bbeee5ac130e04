// Embedding lookup as torch sees it: checks, allocations and autograd nodes over the C ABI (see torch_ops.cpp).
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
  if (!perm.defined() && ictc_embedding_needs_order(N)) std::tie(perm, off) = rows_by_id(ids, entries);
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
  mod.def("encode_activations", &encode_activations, Free());
  mod.def("decode_activations", &decode_activations, Free());
}
