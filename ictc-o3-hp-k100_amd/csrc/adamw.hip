// AdamW over a list of tensors in one launch per kTensors of them:
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = (1 - rate decay) p - rate / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
// with g scaled by min(1, bound / (|g| + 1e-6)), |g| the norm over all tensors, where a bound is given.
// Everything is computed in FP32; a bfloat16 or FP16 parameter is rounded once, to nearest even.
//
// The moments are flat: the segment of each tensor begins at a multiple of 256 elements (a block).  With 8-bit
// moments a block has one power-of-two scale per moment (exact to multiply by):
//   first moment   E4M3 codes of m / scale, scale = 2^(floor(log2 max|m|) - 7), so the largest code is below 256
//   second moment  five exponent and three mantissa bits, no sign, no subnormals: code c > 0 is
//                  (1 + (c mod 8) / 8) 2^(c div 8 - 31) scale, 0 is zero; scale = 2^floor(log2 of the rounded max)
// The second moment divides, so it has range (2^31 within a block) and relative precision (2^-4) rather than a
// linear grid, and a nonzero value never becomes zero: a step would blow up on the next small gradient.  A block
// with NaN or infinity gets a NaN scale: the parameters it feeds become NaN, as they do with FP32 moments.
//
// Bound by memory: p and g in, p out, both moments in and out, 28 bytes an element in FP32, 16 with 8-bit moments; the
// norm reads g once more before.  Measured: 80 M bfloat16 parameters with FP32 moments 313 us (5.6 TB/s) and 67 us for
// the norm; 100 M FP32 with 8-bit moments 314 us (5.1 TB/s) and 127 us (3.2 TB/s: the moments that the update wrote are
// still on their way to memory; 83 us where nothing was written before); 1.2 M FP32 in 42 tensors 7.2 and 5.4 us.
// A block of 256 threads takes a run of 2,048 elements of one tensor; the tensors' pointers travel in the kernel's
// arguments, so no table is copied to the device.  A wave holds one 256-element block of the state, four elements
// a lane, so its largest value is a wave reduction.
#include "dense.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int kTensors = 120;   // tensors of one launch: their table is 3,840 bytes of kernel arguments
constexpr int kRun = 2048;      // elements of a block of threads
constexpr int kNormBlocks = 1024;
constexpr int kOneBlockRuns = 8;

struct Table {
  void* p[kTensors];
  const void* g[kTensors];
  int64_t n[kTensors];
  uint32_t segment[kTensors];   // first block of 256 elements of the tensor's moments
  uint32_t first[kTensors];     // first run of the tensor within this launch
  int tensors;
  int runs;
};

struct Hyper {
  float b1, c1, b2, c2, keep, rate, inv_bc2, eps;
};

// Tensor of run `b`: the last one whose first run is not past b (tensors without elements own no run).
__device__ __forceinline__ int find_tensor(const Table& t, int b) {
  const int lane = threadIdx.x & 63;
  int last = 0;
#pragma unroll
  for (int i = 0; i < (kTensors + 63) / 64; ++i) {
    const int k = i * 64 + lane;
    const bool in = k < t.tensors && t.first[k < kTensors ? k : 0] <= (uint32_t)b;
    last += __popcll(__ballot(in));
  }
  return __builtin_amdgcn_readfirstlane(last - 1);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, float* v) {
  if (n >= 4) {
    if (sizeof(T) == 4) {
      const u32x4 c = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(float, (uint32_t)c[i]);
    } else {
      union { u32x2 raw; T e[4]; } c;
      c.raw = *reinterpret_cast<const u32x2_any*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (float)c.e[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int n, const float* v) {
  if (n >= 4) {
    if (sizeof(T) == 4) {
      u32x4 c;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = __builtin_bit_cast(uint32_t, v[i]);
      *reinterpret_cast<u32x4_any*>(p) = c;
    } else {
      union { u32x2 raw; T e[4]; } c;
#pragma unroll
      for (int i = 0; i < 4; ++i) c.e[i] = (T)v[i];
      *reinterpret_cast<u32x2_any*>(p) = c.raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// Largest value over the wave of non-negative floats given as bits (their order; NaN above infinity above all).
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, s));
  return x;
}

constexpr uint32_t kInf = 0x7f800000u;

__device__ __forceinline__ float bits_float(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ uint32_t float_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

// 2^e as a float and its reciprocal, e in [-126, 126].
__device__ __forceinline__ float pow2(int e) { return bits_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ void decode_m(uint32_t codes, float scale, float* m) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  m[0] = lo[0] * scale;
  m[1] = lo[1] * scale;
  m[2] = hi[0] * scale;
  m[3] = hi[1] * scale;
}

__device__ __forceinline__ void decode_v(uint32_t codes, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = (codes >> (8 * i)) & 255u;
    v[i] = c ? bits_float((c + 96u * 8u) << 20) * scale : 0.f * scale;
  }
}

__device__ __forceinline__ uint32_t encode_m(const float* m, float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, float_bits(m[i]) & 0x7fffffffu);
  top = wave_max(top);
  if (top >= kInf) {
    scale = bits_float(0x7fc00000u);
    return 0;
  }
  const int e = min(126, max(-126, (int)(top >> 23) - 127 - 7));
  scale = pow2(e);
  const float inv = pow2(-e);
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * inv, m[1] * inv, 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(m[2] * inv, m[3] * inv, c, true);
  return (uint32_t)c;
}

// bits rounded to nearest even at the third mantissa bit, and shifted there
__device__ __forceinline__ uint32_t round20(uint32_t b) { return (b + 0x7ffffu + ((b >> 20) & 1u)) >> 20; }

__device__ __forceinline__ uint32_t encode_v(const float* v, float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, float_bits(v[i]) & 0x7fffffffu);
  top = wave_max(top);
  if (top >= kInf) {
    scale = bits_float(0x7fc00000u);
    return 0;
  }
  const int e = min(126, max(-126, (int)(round20(top) >> 3) - 127));
  scale = pow2(e);
  const float inv = pow2(-e);
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (int)round20(float_bits(v[i] * inv)) - 96 * 8;
    out |= (v[i] > 0.f ? (uint32_t)min(255, max(1, c)) : 0u) << (8 * i);
  }
  return out;
}

// Every operation rounded on its own: the moments are then the same bits as elementary operations give, so an
// 8-bit code does not depend on how a compiler fuses them.
__device__ __forceinline__ void update(const Hyper& h, float coef, float* p, const float* g, float* m, float* v) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float gi = g[i] * coef;
    m[i] = m[i] * h.b1 + gi * h.c1;
    v[i] = v[i] * h.b2 + gi * gi * h.c2;
    p[i] = p[i] * h.keep - h.rate * m[i] / (sqrtf(v[i] * h.inv_bc2) + h.eps);
  }
}

template <typename T, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(Table t, Hyper h, void* __restrict__ m_, void* __restrict__ v_,
                                                    float* __restrict__ m_scale, float* __restrict__ v_scale,
                                                    const float* __restrict__ norm) {
  const int b = blockIdx.x, k = find_tensor(t, b);
  const int64_t n = t.n[k], start = (int64_t)(b - (int)t.first[k]) * kRun;
  T* p = reinterpret_cast<T*>(t.p[k]) + start;
  const T* g = reinterpret_cast<const T*>(t.g[k]) + start;
  const int64_t seg = (int64_t)t.segment[k] * 256 + start;
  const float coef = norm ? norm[1] : 1.f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < kRun / 1024; ++j) {
    const int at = j * 1024 + wave * 256 + lane * 4;
    const int64_t left64 = n - start - at;
    const int left = (int)min<int64_t>(4, left64);
    // a wave past the tensor's last block of 256 has no state
    if (left64 + lane * 4 <= 0) continue;
    float pv[4], gv[4], mv[4], vv[4];
    load4(p + at, left, pv);
    load4(g + at, left, gv);
    const int64_t s = seg + at;
    if (EIGHT) {
      uint32_t* mc = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(m_) + s);
      uint32_t* vc = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(v_) + s);
      float ms = m_scale[s >> 8], vs = v_scale[s >> 8];
      decode_m(*mc, ms, mv);
      decode_v(*vc, vs, vv);
      update(h, coef, pv, gv, mv, vv);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= left) mv[i] = vv[i] = 0.f;
      *mc = encode_m(mv, ms);
      *vc = encode_v(vv, vs);
      if (lane == 0) {
        m_scale[s >> 8] = ms;
        v_scale[s >> 8] = vs;
      }
    } else {
      v4f* mp = reinterpret_cast<v4f*>(static_cast<float*>(m_) + s);
      v4f* vp = reinterpret_cast<v4f*>(static_cast<float*>(v_) + s);
      v4f mq = *mp, vq = *vp;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mv[i] = mq[i];
        vv[i] = vq[i];
      }
      update(h, coef, pv, gv, mv, vv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mq[i] = i < left ? mv[i] : 0.f;
        vq[i] = i < left ? vv[i] : 0.f;
      }
      *mp = mq;
      *vp = vq;
    }
    store4(p + at, left, pv);
  }
}

// out[0] = the norm, out[1] = the factor that holds it to `bound`, from the norm in FP64: one past FP32 still has one;
// out[2], out[3] = the FP64 norm.  NaN stays NaN.
__device__ __forceinline__ void write_norm(double squares, float bound, float* __restrict__ out) {
  const double norm = sqrt(squares), f = (double)bound / (norm + 1e-6);
  out[0] = (float)norm;
  out[1] = f >= 1.0 ? 1.f : (float)f;
  reinterpret_cast<double*>(out)[1] = norm;
}

// part[block] = sum of squares of the gradients of this launch's runs blockIdx, blockIdx + gridDim, ...: FP32 over the
// eight elements of a thread's run, FP64 above; and FP64 at once where the eight's sum is not well inside FP32's range
// (past it, or under 2^-100, to which squares below FP32's smallest still belong: any finite gradients have a norm).  Four
// runs are asked for before the first is added.  `out`: there is one block, which writes the norm and the factor too.
// (The test costs 2 to 4 %: alone, 80 M bfloat16 46.0 -> 47.7 us, 100 M FP32 81.4 -> 83.2.)
template <typename T>
__global__ __launch_bounds__(256) void grad_norm_kernel(Table t, double* __restrict__ part, float bound,
                                                        float* __restrict__ out) {
  constexpr int V = kChunk<T>, L = kRun / 256 / V, AHEAD = 4;
  __shared__ double lds[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = 0.0;
  int k = find_tensor(t, blockIdx.x);   // (1.3 M elements in 40 tensors: 5.5 us, walking there from tensor 0 7.9)
  for (int64_t b0 = blockIdx.x; b0 < t.runs; b0 += (int64_t)AHEAD * gridDim.x) {
    u32x4 raw[AHEAD][L];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t b = b0 + (int64_t)a * gridDim.x;
      const bool in = b < t.runs;
      while (in && k + 1 < t.tensors && t.first[k + 1] <= (uint32_t)b) ++k;
      const int64_t start = (b - t.first[k]) * kRun, left = in ? t.n[k] - start : 0;
      const T* g = reinterpret_cast<const T*>(t.g[k]) + start;
      if (left >= kRun) {   // (the same in every lane: a whole run needs no checks)
#pragma unroll
        for (int j = 0; j < L; ++j)
          raw[a][j] = *reinterpret_cast<const u32x4_any*>(g + (j * 256 + (int)threadIdx.x) * V);
      } else {
#pragma unroll
        for (int j = 0; j < L; ++j) {
          const int at = (j * 256 + (int)threadIdx.x) * V;
          raw[a][j] = load_raw(g + at, (int)max<int64_t>(0, min<int64_t>(V, left - at)));
        }
      }
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        float v[V];
        widen<T>(raw[a][j], v);
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i] * v[i];
      }
      double d = (double)s;
      if (sizeof(T) == 4 || __is_same(T, bf16)) {   // (FP16's squares are all in the range)
        if (!(s >= 0x1p-100f && s < bits_float(kInf))) {
          d = 0.0;
#pragma unroll
          for (int j = 0; j < L; ++j) {
            float v[V];
            widen<T>(raw[a][j], v);
#pragma unroll
            for (int i = 0; i < V; ++i) d += (double)v[i] * (double)v[i];
          }
        }
      }
      sum += d;
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);
  if (lane == 0) lds[wave] = sum;
  __syncthreads();
  if (threadIdx.x > 0) return;
  sum = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  if (out)
    write_norm(sum, bound, out);
  else
    part[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void norm_factor_kernel(const double* __restrict__ part, int n, float bound,
                                                          float* __restrict__ out) {
  __shared__ double lds[4];
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) sum += part[i];
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) write_norm((lds[0] + lds[1]) + (lds[2] + lds[3]), bound, out);
}

template <typename T>
__global__ __launch_bounds__(256) void moments_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                      const float* __restrict__ m_scale,
                                                      const float* __restrict__ v_scale, int64_t n,
                                                      T* __restrict__ m_out, T* __restrict__ v_out) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  float mv[4], vv[4];
  decode_m(*reinterpret_cast<const uint32_t*>(m + at), m_scale[at >> 8], mv);
  decode_v(*reinterpret_cast<const uint32_t*>(v + at), v_scale[at >> 8], vv);
  store4(m_out + at, 4, mv);
  store4(v_out + at, 4, vv);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T>
void launch_step(const Table& t, const Hyper& h, int bits, void* m, void* v, float* ms, float* vs, const float* norm,
                 hipStream_t st) {
  if (bits == 8)
    hipLaunchKernelGGL((adamw_kernel<T, true>), dim3((unsigned)t.runs), dim3(256), 0, st, t, h, m, v, ms, vs, norm);
  else
    hipLaunchKernelGGL((adamw_kernel<T, false>), dim3((unsigned)t.runs), dim3(256), 0, st, t, h, m, v, ms, vs, norm);
}

const char* bad_list(int dtype, int tensors, const int64_t* grads, const int64_t* counts) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "adamw: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (tensors < 0) return "adamw: negative count of tensors";
  if (tensors > 0 && (!grads || !counts)) return "adamw: null operand";
  for (int i = 0; i < tensors; ++i) {
    if (counts[i] < 0 || counts[i] / kRun >= (int64_t(1) << 30)) return "adamw: element count out of range";
    if (counts[i] > 0 && !grads[i]) return "adamw: null tensor";
  }
  return nullptr;
}

// Calls launch(table) for the tensors in order, up to kTensors and 2^30 runs at a time.
template <typename F>
void for_tables(int tensors, const int64_t* params, const int64_t* grads, const int64_t* counts,
                const int64_t* starts, F launch) {
  Table t;
  t.tensors = t.runs = 0;
  int64_t start = 0;
  for (int i = 0; i < tensors; ++i) {
    if (starts) start = starts[i];
    const int64_t runs = (counts[i] + kRun - 1) / kRun;
    if (t.runs > 0 && (t.tensors == kTensors || t.runs + runs > (int64_t(1) << 30))) {
      launch(t);
      t.tensors = t.runs = 0;
    }
    if (runs > 0) {
      t.p[t.tensors] = params ? reinterpret_cast<void*>(params[i]) : nullptr;
      t.g[t.tensors] = reinterpret_cast<const void*>(grads[i]);
      t.n[t.tensors] = counts[i];
      t.segment[t.tensors] = (uint32_t)(start / 256);
      t.first[t.tensors] = (uint32_t)t.runs;
      ++t.tensors;
      t.runs += (int)runs;
    }
    start += (counts[i] + 255) / 256 * 256;
  }
  if (t.runs > 0) launch(t);
}

}  // namespace

extern "C" {

int64_t ictc_gradient_norm_workspace_bytes(int tensors) {
  if (tensors < 0) return -1;
  return 16 + (int64_t)((tensors + kTensors - 1) / kTensors) * kNormBlocks * (int64_t)sizeof(double);
}

int ictc_gradient_norm(int dtype, int tensors, const int64_t* grads, const int64_t* counts, double max_norm,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_list(dtype, tensors, grads, counts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (!(max_norm >= 0.0)) return dense_fail(ICTC_ERR_ARGUMENT, "gradient_norm: max_norm must be zero or more");
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < ictc_gradient_norm_workspace_bytes(tensors))
    return dense_fail(ICTC_ERR_ARGUMENT, "gradient_norm: workspace smaller than ictc_gradient_norm_workspace_bytes");
  hipStream_t st = (hipStream_t)stream;
  double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  int parts = 0;
  // Few elements: one block and one launch (8 x 2,048: 4.9 us, two launches 7.7; 16 x 2,048 7.8 both).
  int64_t runs = 0;
  int used = 0;
  for (int i = 0; i < tensors; ++i) {
    runs += (counts[i] + kRun - 1) / kRun;
    used += counts[i] > 0;
  }
  const bool one = runs > 0 && runs <= kOneBlockRuns && used <= kTensors;
  float* out = one ? (float*)workspace : nullptr;
  const float bound = (float)max_norm;
  for_tables(tensors, nullptr, grads, counts, nullptr, [&](const Table& t) {
    const int blocks = one ? 1 : std::min(t.runs, kNormBlocks);
    if (dtype == ICTC_F32)
      hipLaunchKernelGGL(grad_norm_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, t, part + parts, bound,
                         out);
    else if (dtype == ICTC_BF16)
      hipLaunchKernelGGL(grad_norm_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, st, t, part + parts, bound,
                         out);
    else
      hipLaunchKernelGGL(grad_norm_kernel<f16>, dim3((unsigned)blocks), dim3(256), 0, st, t, part + parts, bound,
                         out);
    parts += blocks;
  });
  if (!one) hipLaunchKernelGGL(norm_factor_kernel, dim3(1), dim3(256), 0, st, part, parts, bound, (float*)workspace);
  return dense_status("gradient_norm launch");
}

int ictc_adamw_step(int dtype, int bits, int tensors, const int64_t* params, const int64_t* grads,
                    const int64_t* counts, const int64_t* starts, void* m, void* v, float* m_scale, float* v_scale,
                    int64_t state_elements, double lr, double beta1, double beta2, double eps, double weight_decay,
                    int64_t step, const float* norm, void* stream) {
  if (const char* e = bad_list(dtype, tensors, grads, counts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (bits != 32 && bits != 8) return dense_fail(ICTC_ERR_UNSUPPORTED, "adamw: moments of 32 or 8 bits");
  if (step < 1) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: steps count from 1");
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !std::isfinite(lr) ||
      !std::isfinite(weight_decay))
    return dense_fail(ICTC_ERR_ARGUMENT, "adamw: betas in [0, 1), eps zero or more, rate and decay finite");
  if (tensors > 0 && !params) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: null operand");
  int64_t end = 0;
  for (int i = 0; i < tensors; ++i) {
    if (counts[i] > 0 && !params[i]) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: null tensor");
    if (starts && (starts[i] < end || starts[i] % 256))
      return dense_fail(ICTC_ERR_ARGUMENT, "adamw: segments begin at multiples of 256, in order, without overlap");
    end = (starts ? starts[i] : end) + (counts[i] + 255) / 256 * 256;
  }
  if (end == 0) return ICTC_OK;
  if (end / 256 >= (int64_t(1) << 32)) return dense_fail(ICTC_ERR_UNSUPPORTED, "adamw: more than 2^40 elements");
  if (state_elements < end)
    return dense_fail(ICTC_ERR_ARGUMENT, "adamw: moments hold fewer elements than the tensors' blocks of 256");
  if (!m || !v || (bits == 8 && (!m_scale || !v_scale)))
    return dense_fail(ICTC_ERR_ARGUMENT, "adamw: null moments");
  if (!aligned(m, 16) || !aligned(v, 16)) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: moments must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  Hyper h;
  h.b1 = (float)beta1;
  h.c1 = (float)(1.0 - beta1);
  h.b2 = (float)beta2;
  h.c2 = (float)(1.0 - beta2);
  h.keep = (float)(1.0 - lr * weight_decay);
  h.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  h.inv_bc2 = (float)(1.0 / (1.0 - std::pow(beta2, (double)step)));
  h.eps = (float)eps;
  for_tables(tensors, params, grads, counts, starts, [&](const Table& t) {
    if (dtype == ICTC_F32)
      launch_step<float>(t, h, bits, m, v, m_scale, v_scale, norm, st);
    else if (dtype == ICTC_BF16)
      launch_step<bf16>(t, h, bits, m, v, m_scale, v_scale, norm, st);
    else
      launch_step<f16>(t, h, bits, m, v, m_scale, v_scale, norm, st);
  });
  return dense_status("adamw launch");
}

int ictc_adamw_moments(int dtype, const void* m, const void* v, const float* m_scale, const float* v_scale,
                       int64_t elements, void* m_out, void* v_out, void* stream) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16)
    return dense_fail(ICTC_ERR_ARGUMENT, "adamw: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16");
  if (elements < 0 || elements % 256) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: moments come in blocks of 256");
  if (elements / 1024 >= (int64_t(1) << 31) - 1) return dense_fail(ICTC_ERR_UNSUPPORTED, "adamw: too many elements");
  if (elements == 0) return ICTC_OK;
  if (!m || !v || !m_scale || !v_scale || !m_out || !v_out)
    return dense_fail(ICTC_ERR_ARGUMENT, "adamw: null operand");
  if (!aligned(m, 4) || !aligned(v, 4)) return dense_fail(ICTC_ERR_ARGUMENT, "adamw: moments must be 4-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((elements + 1023) / 1024));
  const uint8_t *mc = static_cast<const uint8_t*>(m), *vc = static_cast<const uint8_t*>(v);
  if (dtype == ICTC_F32)
    hipLaunchKernelGGL(moments_kernel<float>, grid, dim3(256), 0, st, mc, vc, m_scale, v_scale, elements, (float*)m_out,
                       (float*)v_out);
  else if (dtype == ICTC_BF16)
    hipLaunchKernelGGL(moments_kernel<bf16>, grid, dim3(256), 0, st, mc, vc, m_scale, v_scale, elements, (bf16*)m_out,
                       (bf16*)v_out);
  else
    hipLaunchKernelGGL(moments_kernel<f16>, grid, dim3(256), 0, st, mc, vc, m_scale, v_scale, elements, (f16*)m_out,
                       (f16*)v_out);
  return dense_status("adamw moments launch");
}

}  // extern "C"
