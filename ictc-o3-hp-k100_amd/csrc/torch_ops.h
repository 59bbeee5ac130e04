// What the torch layers of the dense operators share: checks of arguments, rows and pitches, which gradients are asked
// for, and refusals.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/ictc_mi355x.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Raises what the C ABI reported: an argument's fault as ValueError.
void done(int rc, const char* what) {
  if (rc == ICTC_OK) return;
  const std::string said = std::string(what) + ": " + ictc_last_error();
  TORCH_CHECK_VALUE(rc != ICTC_ERR_ARGUMENT && rc != ICTC_ERR_UNSUPPORTED, said);
  TORCH_CHECK(false, said);
}

// The results are written through raw pointers, which a trace does not see: it would keep their allocation and replay
// that.  So these operators run eagerly, as the equivariant ones do; forward and backward passes ask.
void eager(const char* op) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  bool traced = torch::jit::tracer::isTracing();
  if (Modes::any_modes_set())
    for (Key key : {Key::PROXY, Key::FAKE, Key::FUNCTIONAL}) traced |= Modes::get_mode(key).has_value();
  TORCH_CHECK_VALUE(!traced, op, ": cannot be traced; it requires eager execution");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ICTC_F32;
    case at::kBFloat16: return ICTC_BF16;
    case at::kHalf: return ICTC_F16;
    default: return -1;
  }
}

void check_dense(const Tensor& t, const char* op, const char* name, const Tensor* like = nullptr) {
  TORCH_CHECK_VALUE(t.is_cuda(), op, ": ", name, " must be on a ROCm (cuda) device");
  TORCH_CHECK_VALUE(dtype_of(t) >= 0, op, ": ", name, " must be float32, bfloat16 or float16");
  if (like) {
    TORCH_CHECK_VALUE(t.get_device() == like->get_device(), op, ": ", name, " must be on ", like->device());
    TORCH_CHECK_VALUE(t.scalar_type() == like->scalar_type(), op, ": ", name, " must have the type ",
                      like->scalar_type());
  }
}

// t [N, C] itself, or a copy, with unit column stride and a row pitch of at least C.
Tensor rows_of(const Tensor& t) {
  if (t.is_contiguous()) return t;
  if ((t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) <= 1)) return t;
  return t.contiguous();
}

int64_t pitch(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }   // (a single row's stride may be anything)

Tensor packed(const Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.contiguous(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor floats(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Whether an operator's call has to leave a node behind.  Without (inference) it goes past autograd, and layer norm writes
// no statistics: order and expert linear of 5 rows 10.7 -> 8.9 us, layer norm of one 5.5 -> 3.8.
bool tracked(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

// Which of a node's inputs the running backward pass asks for; inputs without a variable have no edge.
std::vector<bool> wanted(AutogradContext* ctx, std::initializer_list<bool> present) {
  std::vector<bool> out;
  size_t edge = 0;
  for (bool p : present) out.push_back(p && ctx->needs_input_grad(edge++));
  return out;
}

// (rows in the order of their id, first sorted row of each id) of ids [N] in [0, keys); those outside come last.  op: the
// operator that asks.
std::pair<Tensor, Tensor> rows_by_id(const Tensor& ids, int64_t keys, const char* op) {
  const int64_t N = ids.size(0), bytes = ictc_rows_by_id_workspace_bytes(N, keys);
  const auto ints = ids.options().dtype(at::kInt);
  const Tensor perm = at::empty({std::max<int64_t>(N, 1)}, ints), offsets = at::empty({keys + 2}, ints);
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, ids.options().dtype(at::kByte));
  done(ictc_rows_by_id(ids.const_data_ptr<int64_t>(), N, keys, perm.mutable_data_ptr<int>(),
                       offsets.mutable_data_ptr<int>(), ptr(ws), bytes, stream_of(ids)),
       op);
  return {perm, offsets};
}

// ---------------------------------------------------------------------------
// Activations in 8 bits
// ---------------------------------------------------------------------------

struct Codes {
  Tensor codes, scales;   // int8 [rows, width], float32 [rows, blocks of 128]
};

Codes empty_codes(int64_t N, int64_t C, const Tensor& like) {
  return {at::empty({N, C}, like.options().dtype(at::kChar)), at::empty({N, (C + 127) / 128}, like.options().dtype(at::kFloat))};
}

Codes encode_rows(const Tensor& x_) {
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows_of(x_);
  const int64_t N = x.size(0), C = x.size(1);
  Codes out = empty_codes(N, C, x);
  done(ictc_codes_encode(dtype_of(x), ptr(x), pitch(x), N, (int)C, out.codes.mutable_data_ptr<int8_t>(),
                         out.scales.mutable_data_ptr<float>(), stream_of(x)),
       "activations");
  return out;
}

Tensor decode_rows(const Tensor& codes, const Tensor& scales, at::ScalarType type) {
  const c10::DeviceGuard guard(codes.device());
  const int64_t N = codes.size(0), C = codes.size(1);
  Tensor out = at::empty({N, C}, codes.options().dtype(type));
  done(ictc_codes_decode(dtype_of(out), codes.const_data_ptr<int8_t>(), scales.const_data_ptr<float>(), N, (int)C,
                         ptr(out), stream_of(codes)),
       "activations");
  return out;
}

// Where a graph goes on from rows that are kept in 8 bits: a tensor of their shape without their memory, whose gradient
// is theirs.  A node keeps it beside the codes, and a backward pass that will be differentiated takes the values as a
// function of it (Decoded).
struct Place8 : Function<Place8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x) {
    ctx->set_materialize_grads(false);
    return at::empty({1}, x.options()).expand(x.sizes());
  }
  static variable_list backward(AutogradContext*, variable_list grads) { return {grads[0]}; }
};

struct Decoded : Function<Decoded> {
  static Tensor forward(AutogradContext* ctx, const Tensor& place, const Tensor& codes, const Tensor& scales) {
    ctx->set_materialize_grads(false);
    return decode_rows(codes, scales, place.scalar_type());
  }
  static variable_list backward(AutogradContext*, variable_list grads) { return {grads[0], Tensor(), Tensor()}; }
};

// save_bits of an operator: whether its rows are kept in 8 bits.
bool in_8_bits(const std::optional<int64_t>& save_bits, const char* op) {
  TORCH_CHECK_VALUE(!save_bits.has_value() || *save_bits == 8, op, ": save_bits must be 8 or None");
  return save_bits.has_value();
}

}  // namespace
