// The group norm's entry points: checks, workspaces and the choice of the element type (group_norm.h has the kernels).
#include "group_norm_launch.h"

namespace {

int64_t workspace_bytes(int dtype, int pass, int64_t samples, int64_t positions, int channels, int groups) {
  if (samples == 0 || positions == 0) samples = 0, positions = 1;   // (as the calls take them)
  const Plan p = plan_of(dtype == ICTC_F32 ? 4 : 2, samples, positions, channels, groups, pass == 2);
  const bool parts = p.form == Form::kParts;
  const int64_t units = samples * groups, each = units * p.tile.splits * p.tile.tiles_per;
  if (pass == 0) return parts ? each * 16 + units * 12 : 0;
  const int K = pass == 1 ? 2 : kSums;
  return 4 * (2 * p.parts * channels + (parts ? (each + units) * K : 0));
}

const char* bad_sizes(int dtype, int64_t samples, int64_t positions, int channels, int groups) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "group_norm: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (samples < 0 || positions < 0) return "group_norm: samples and positions must not be negative";
  if (channels < 1 || channels > 65536) return "group_norm: 1 to 65536 channels";
  if (groups < 1 || channels % groups) return "group_norm: groups must divide the channels";
  constexpr int64_t most = int64_t(1) << 40;   // (elements; 64-bit offsets hold far more)
  if (samples > 0 && (positions > most / samples || samples * std::max<int64_t>(positions, 1) > most / channels))
    return "group_norm: up to 2^40 elements";
  return nullptr;
}

bool workspace_fits(const ictc::GroupNormCall& a, int dtype, int pass) {
  const int64_t need = workspace_bytes(dtype, pass, a.samples, a.positions, a.channels, a.groups);
  return need == 0 || (a.ws && !(reinterpret_cast<uintptr_t>(a.ws) & 7) && a.ws_bytes >= need);
}

}  // namespace

#define GN_TYPED(f)                                \
  if (dtype == ICTC_F32)                           \
    ictc::f<float>(a);                             \
  else if (dtype == ICTC_BF16)                     \
    ictc::f<bf16>(a);                              \
  else                                             \
    ictc::f<f16>(a);

namespace ictc {
#define GN_EXTERN(T)                                      \
  extern template void group_norm_fwd<T>(const GroupNormCall&);  \
  extern template void group_norm_bwd<T>(const GroupNormCall&);  \
  extern template void group_norm_bwd2<T>(const GroupNormCall&);
GN_EXTERN(float)
GN_EXTERN(bf16)
GN_EXTERN(f16)
}  // namespace ictc

extern "C" {

int64_t ictc_group_norm_workspace_bytes(int dtype, int pass, int64_t samples, int64_t positions, int channels,
                                        int groups) {
  if (bad_sizes(dtype, samples, positions, channels, groups) || pass < 0 || pass > 2) return -1;
  return workspace_bytes(dtype, pass, samples, positions, channels, groups);
}

int ictc_group_norm_keeps_rest(int dtype, int64_t samples, int64_t positions, int channels, int groups) {
  return !bad_sizes(dtype, samples, positions, channels, groups) && samples > 0 && positions > 0 && dtype == ICTC_F32 &&
         plan_of(4, samples, positions, channels, groups, false).form != Form::kRows;
}

int ictc_group_norm_fwd_rest(int dtype, const void* x, int64_t samples, int64_t positions, int channels, int groups,
                             const void* weight, const void* bias, float eps, int activation, void* y, float* mean,
                             float* rest, float* rstd, int8_t* codes, float* scales, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, samples, positions, channels, groups)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (!(eps >= 0.f)) return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: eps must not be negative");
  if (activation != 0 && activation != 1) return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: activation must be 0 or 1");
  if (samples == 0 || positions == 0) return ICTC_OK;
  if (!x || !y || !mean != !rstd || (rest && !mean) || !codes != !scales)
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: null operand");
  ictc::GroupNormCall a = {};
  a.samples = samples, a.positions = positions, a.channels = channels, a.groups = groups;
  a.x = x, a.w = weight, a.b = bias, a.eps = eps, a.silu = activation, a.out = y, a.mean = mean, a.rest = rest,
  a.rstd = rstd;
  a.codes_out = codes, a.scales_out = scales;
  a.ws = workspace, a.ws_bytes = workspace_bytes, a.stream = (hipStream_t)stream;
  if (!workspace_fits(a, dtype, 0))
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: workspace smaller than ictc_group_norm_workspace_bytes");
  if (codes && !plan_of(dtype == ICTC_F32 ? 4 : 2, samples, positions, channels, groups, false).coded)
    if (const int rc = ictc_codes_encode(dtype, x, channels, samples * positions, channels, codes, scales, stream)) return rc;
  GN_TYPED(group_norm_fwd)
  return dense_status("group_norm_fwd launch");
}

int ictc_group_norm_bwd_rest(int dtype, const void* x, const int8_t* codes, const float* scales, const void* grad,
                             int64_t samples, int64_t positions, int channels, int groups, const void* weight,
                             const void* bias, int activation, const float* mean, const float* rest, const float* rstd,
                             void* dx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  if (const char* e = bad_sizes(dtype, samples, positions, channels, groups)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (activation != 0 && activation != 1) return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: activation must be 0 or 1");
  const bool none = samples == 0 || positions == 0;
  if (!none && ((!x && !codes) || !codes != !scales || !grad || !mean || !rstd))
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: null operand");
  if ((none || !dx) && !dweight && !dbias) return ICTC_OK;
  ictc::GroupNormCall a = {};
  a.samples = none ? 0 : samples, a.positions = none ? 1 : positions, a.channels = channels, a.groups = groups;
  a.x = x, a.codes = codes, a.scales = scales, a.g = grad, a.w = weight, a.b = bias, a.silu = activation;
  a.mean = (float*)mean, a.rest = (float*)rest, a.rstd = (float*)rstd, a.out = dx, a.out_w = dweight, a.out_b = dbias;
  a.ws = workspace, a.ws_bytes = workspace_bytes, a.stream = (hipStream_t)stream;
  if (!workspace_fits(a, dtype, 1))
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: workspace smaller than ictc_group_norm_workspace_bytes");
  GN_TYPED(group_norm_bwd)
  return dense_status("group_norm_bwd launch");
}

int ictc_group_norm_bwd2_rest(int dtype, const void* x, const int8_t* codes, const float* scales, const void* grad,
                              const void* v, const void* vweight, const void* vbias, int64_t samples, int64_t positions,
                              int channels, int groups, const void* weight, const void* bias, int activation,
                              const float* mean, const float* rest, const float* rstd, void* dx, void* dgrad,
                              void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, samples, positions, channels, groups)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (activation != 0 && activation != 1) return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: activation must be 0 or 1");
  const bool none = samples == 0 || positions == 0;
  if (!none && ((!x && !codes) || !codes != !scales || !grad || !v || !mean || !rstd))
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: null operand");
  if ((none || (!dx && !dgrad)) && !dweight && !dbias) return ICTC_OK;
  ictc::GroupNormCall a = {};
  a.samples = none ? 0 : samples, a.positions = none ? 1 : positions, a.channels = channels, a.groups = groups;
  a.x = x, a.codes = codes, a.scales = scales, a.g = grad, a.v = v, a.vw = vweight, a.vb = vbias;
  a.w = weight, a.b = bias, a.silu = activation, a.mean = (float*)mean, a.rest = (float*)rest, a.rstd = (float*)rstd;
  a.out = dx, a.out_g = dgrad, a.out_w = dweight, a.out_b = dbias;
  a.ws = workspace, a.ws_bytes = workspace_bytes, a.stream = (hipStream_t)stream;
  if (!workspace_fits(a, dtype, 2))
    return dense_fail(ICTC_ERR_ARGUMENT, "group_norm: workspace smaller than ictc_group_norm_workspace_bytes");
  GN_TYPED(group_norm_bwd2)
  return dense_status("group_norm_bwd2 launch");
}

int ictc_group_norm_fwd(int dtype, const void* x, int64_t samples, int64_t positions, int channels, int groups,
                        const void* weight, const void* bias, float eps, int activation, void* y, float* mean,
                        float* rstd, int8_t* codes, float* scales, void* workspace, int64_t workspace_bytes, void* stream) {
  return ictc_group_norm_fwd_rest(dtype, x, samples, positions, channels, groups, weight, bias, eps, activation, y, mean,
                                  nullptr, rstd, codes, scales, workspace, workspace_bytes, stream);
}

int ictc_group_norm_bwd(int dtype, const void* x, const int8_t* codes, const float* scales, const void* grad,
                        int64_t samples, int64_t positions, int channels, int groups, const void* weight,
                        const void* bias, int activation, const float* mean, const float* rstd, void* dx, void* dweight,
                        void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  return ictc_group_norm_bwd_rest(dtype, x, codes, scales, grad, samples, positions, channels, groups, weight, bias,
                                  activation, mean, nullptr, rstd, dx, dweight, dbias, workspace, workspace_bytes, stream);
}

int ictc_group_norm_bwd2(int dtype, const void* x, const int8_t* codes, const float* scales, const void* grad,
                         const void* v, const void* vweight, const void* vbias, int64_t samples, int64_t positions,
                         int channels, int groups, const void* weight, const void* bias, int activation,
                         const float* mean, const float* rstd, void* dx, void* dgrad, void* dweight, void* dbias,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  return ictc_group_norm_bwd2_rest(dtype, x, codes, scales, grad, v, vweight, vbias, samples, positions, channels, groups,
                                   weight, bias, activation, mean, nullptr, rstd, dx, dgrad, dweight, dbias, workspace,
                                   workspace_bytes, stream);
}

}  // extern "C"
