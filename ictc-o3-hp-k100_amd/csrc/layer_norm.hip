// Layer norm over rows of `width` elements (FP32, bfloat16 or FP16; every sum and statistic in FP32):
//   y = h w + b,  h = (x - mean) r,  r = 1 / sqrt(var + eps)
// with u = g w its gradients
//   dx = r (u - <u> - h <u h>),  dw = sum over rows g h,  db = sum over rows g        (<.> the mean over a row)
// and, for a loss that depends on dx itself, the gradients of <v, dx> + <vw, dw> + <vb, db>:
//   pv = r (v - <v> - h <v h>)                    dw' = sum over rows g pv
//   dg' = w pv + h vw + vb
//   t  = g vw - r (<v h> u + <u h> v)             q = <u v> - <u> <v> - <u h> <v h>
//   dx' = r (t - <t> - h <t h>) - r^2 q h
// (t is the gradient by h with r held fixed; dr/dx = -r^2 h / width gives the last term).
//
// All three are bound by memory: each element of each operand is read once and each output written once.  A row is
// held in the registers of a team of 8 to 512 lanes as 16-byte chunks, so the mean is subtracted before the
// squares are added (no cancellation) and nothing is read twice; teams of up to 64 lanes need no barrier.  Teams of
// 64 and more ask for their next row before they work on the present one (a team of 16 has three neighbours in its
// wave to wait with).  The gradients by w and b are added per lane over the rows that a team takes, then over the
// teams of a block in LDS, and the blocks' partial sums by a second kernel, always in the same order.
//
// Measured: 425,991 rows of 64 FP32 forward 38 us (5.7 TB/s), gradients 54 us (6.1 TB/s) and 4.7 us for the blocks'
// sums; 131,072 of 128 FP32 second derivative 55 us (6.1 TB/s); 8,191 of 2,176 bfloat16 forward 20 us and gradients
// 29 us (3.6 TB/s: a few rows a block, whose first loads and last stores wait for nothing else); 257 of 64 about 3 us
// each, the latency of a launch.  A large copy reaches 5.1 TB/s; operands that the caches still hold come faster.
#include "dense.h"

#include <algorithm>

namespace {

constexpr int kMaxWidth = 16384;

// Sums of K values over a team, in every lane of it.
template <int TEAM, int K>
__device__ __forceinline__ void team_sum(float (&s)[K], float* lds) {
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = lane_sum<(TEAM < 64 ? TEAM : 64)>(s[k]);
  if (TEAM > 64) {
    constexpr int W = TEAM / 64;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[w * K + k] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) a += lds[i * K + k];
      s[k] = a;
    }
    __syncthreads();
  }
}

template <int TEAM>
constexpr int kThreads = TEAM > 256 ? TEAM : 256;

// Whether a kernel reads one row ahead: where the registers for it are there.  (8,191 x 2,176 bfloat16: gradients 50
// us without, 36 us with; 2,048 x 8,192: 61 and 37 us.)
template <int TEAM, int EPL>
constexpr bool kAhead = TEAM >= 64 && EPL <= 16;

// A row's chunks as a lane of its team holds them.
template <typename T, int TEAM, int EPL>
struct Row {
  static constexpr int V = kChunk<T>, N = EPL / V;
  u32x4 raw[N];
  __device__ __forceinline__ void load(const T* __restrict__ row, int width, int lane) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * TEAM + lane) * V;
      raw[n] = load_raw(row + c, width - c);
    }
  }
  __device__ __forceinline__ void get(float (&v)[EPL]) const {
#pragma unroll
    for (int n = 0; n < N; ++n) widen<T>(raw[n], v + n * V);
  }
};

template <typename T, int TEAM, int EPL>
__global__ __launch_bounds__(kThreads<TEAM>) void ln_fwd_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                                int width, const T* __restrict__ weight,
                                                                const T* __restrict__ bias, float eps,
                                                                T* __restrict__ y, float* __restrict__ mean,
                                                                float* __restrict__ rstd) {
  constexpr int V = kChunk<T>, N = EPL / V, TEAMS = kThreads<TEAM> / TEAM;
  __shared__ float lds[TEAM > 64 ? TEAM / 64 : 1];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)width;
  float w[EPL], b[EPL];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * TEAM + lane) * V;
    if (weight) load_chunk(weight + c, width - c, w + n * V);
    if (bias) load_chunk(bias + c, width - c, b + n * V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (!weight) w[n * V + e] = 1.f;
      if (!bias) b[n * V + e] = 0.f;
    }
  }
  const int64_t gap = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  Row<T, TEAM, EPL> next;
  if (kAhead<TEAM, EPL> && row < rows) next.load(x + row * ldx, width, lane);
  for (; row < rows; row += gap) {
    float v[EPL], s[1] = {0.f};
    if (!kAhead<TEAM, EPL>) next.load(x + row * ldx, width, lane);
    next.get(v);
    if (kAhead<TEAM, EPL> && row + gap < rows) next.load(x + (row + gap) * ldx, width, lane);
#pragma unroll
    for (int i = 0; i < EPL; ++i) s[0] += v[i];
    team_sum<TEAM>(s, lds);
    const float mu = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * TEAM + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[n * V + e] -= mu;
        s[0] += c + e < width ? v[n * V + e] * v[n * V + e] : 0.f;
      }
    }
    team_sum<TEAM>(s, lds);
    float r = 1.f / sqrtf(s[0] * inv + eps);
    // (in the whole team) Finite deviations whose squares are past FP32 are added again, scaled.  Ordinary rows pay
    // nothing measurable: 425,991 x 64 FP32 34.8 us without the branch and 35.0 with, 8,191 x 2,176 24.7 both.
    if (s[0] == __builtin_inff()) {
      constexpr float SCALE = 0x1p-80f;
      s[0] = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * TEAM + lane) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = v[n * V + e] * SCALE;
          s[0] += c + e < width ? d * d : 0.f;
        }
      }
      team_sum<TEAM>(s, lds);
      r = SCALE / sqrtf(s[0] * inv + eps * SCALE * SCALE);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * TEAM + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) v[n * V + e] = v[n * V + e] * r * w[n * V + e] + b[n * V + e];
      store_chunk(y + row * (int64_t)width + c, width - c, v + n * V);
    }
    if (lane == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
  }
}

// Sums of acc over the teams of a block into part[columns of this block].
template <int TEAM, int EPL, int V>
__device__ __forceinline__ void block_columns(const float (&acc)[EPL], int width, float* __restrict__ part,
                                              float* lds) {
  constexpr int N = EPL / V, TEAMS = kThreads<TEAM> / TEAM;
  const int lane = threadIdx.x % TEAM;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (TEAMS == 1) {
      const int c = (n * TEAM + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < width) part[c + e] = acc[n * V + e];
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) lds[threadIdx.x * V + e] = acc[n * V + e];
      __syncthreads();
      for (int i = threadIdx.x; i < TEAM * V; i += kThreads<TEAM>) {
        float a = 0.f;
#pragma unroll
        for (int t = 0; t < TEAMS; ++t) a += lds[t * TEAM * V + i];
        if (n * TEAM * V + i < width) part[n * TEAM * V + i] = a;
      }
    }
  }
}

template <typename T, int TEAM, int EPL>
__global__ __launch_bounds__(kThreads<TEAM>) void ln_bwd_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ g, int64_t ldg, int64_t rows, int width,
    const T* __restrict__ weight, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
    float* __restrict__ part_w, float* __restrict__ part_b) {
  constexpr int V = kChunk<T>, N = EPL / V, TEAMS = kThreads<TEAM> / TEAM;
  __shared__ float lds[TEAM > 64 ? TEAM / 64 * 2 : 256 * V];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)width;
  float w[EPL], dw[EPL], db[EPL];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * TEAM + lane) * V;
    if (weight) load_chunk(weight + c, width - c, w + n * V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (!weight) w[n * V + e] = 1.f;
      dw[n * V + e] = db[n * V + e] = 0.f;
    }
  }
  const int64_t gap = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  Row<T, TEAM, EPL> nx, ng;
  float mu_next = 0.f, r_next = 0.f;
  auto load = [&](int64_t at) {
    nx.load(x + at * ldx, width, lane);
    ng.load(g + at * ldg, width, lane);
    mu_next = mean[at];
    r_next = rstd[at];
  };
  if (kAhead<TEAM, EPL> && row < rows) load(row);
  for (; row < rows; row += gap) {
    float h[EPL], u[EPL], s[2] = {0.f, 0.f};
    if (!kAhead<TEAM, EPL>) load(row);
    nx.get(h);
    ng.get(u);
    const float mu = mu_next, r = r_next;
    if (kAhead<TEAM, EPL> && row + gap < rows) load(row + gap);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      h[i] = (h[i] - mu) * r;
      dw[i] += u[i] * h[i];
      db[i] += u[i];
      u[i] *= w[i];
      s[0] += u[i];
      s[1] += u[i] * h[i];
    }
    if (dx) {
      team_sum<TEAM>(s, lds);
      const float a = s[0] * inv, b = s[1] * inv;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * TEAM + lane) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) u[n * V + e] = r * (u[n * V + e] - a - h[n * V + e] * b);
        store_chunk(dx + row * (int64_t)width + c, width - c, u + n * V);
      }
    }
  }
  if (part_w) block_columns<TEAM, EPL, V>(dw, width, part_w + (int64_t)blockIdx.x * width, lds);
  if (part_b) block_columns<TEAM, EPL, V>(db, width, part_b + (int64_t)blockIdx.x * width, lds);
}

template <typename T, int TEAM, int EPL>
__global__ __launch_bounds__(kThreads<TEAM>) void ln_bwd2_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ g, int64_t ldg, const T* __restrict__ v, int64_t ldv,
    const T* __restrict__ vw, const T* __restrict__ vb, int64_t rows, int width, const T* __restrict__ weight,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, T* __restrict__ dg,
    float* __restrict__ part_w) {
  constexpr int V = kChunk<T>, N = EPL / V, TEAMS = kThreads<TEAM> / TEAM;
  __shared__ float lds[TEAM > 64 ? TEAM / 64 * 7 : 256 * V];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)width;
  float dw[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) dw[i] = 0.f;
  // The row's parameters as they lie in memory, read once where the registers for it are there.  (Read twice a row from
  // the caches: 8,191 x 2,176 bfloat16 78 us, so 67; 65,536 x 250 FP32 82 and 70; 131,072 x 128 bfloat16 44 and 46.)
  constexpr bool KEEP = EPL <= 16;
  Row<T, TEAM, EPL> kw, kvw, kvb;
  if (KEEP && weight) kw.load(weight, width, lane);
  if (KEEP && vw) kvw.load(vw, width, lane);
  if (KEEP && vb) kvb.load(vb, width, lane);
  auto parameter = [&](const Row<T, TEAM, EPL>& kept, const T* p, int n, float* out) {
    const int c = (n * TEAM + lane) * V;
    if (KEEP)
      widen<T>(kept.raw[n], out);
    else
      load_chunk(p + c, width - c, out);
  };
  const int64_t gap = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  Row<T, TEAM, EPL> nx, ng, nv;
  float mu_next = 0.f, r_next = 0.f;
  auto load = [&](int64_t at) {
    nx.load(x + at * ldx, width, lane);
    ng.load(g + at * ldg, width, lane);
    nv.load(v + at * ldv, width, lane);
    mu_next = mean[at];
    r_next = rstd[at];
  };
  if (kAhead<TEAM, EPL> && row < rows) load(row);
  for (; row < rows; row += gap) {
    float h[EPL], gr[EPL], vr[EPL], s[7] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!kAhead<TEAM, EPL>) load(row);
    nx.get(h);
    ng.get(gr);
    nv.get(vr);
    const float mu = mu_next, r = r_next;
    if (kAhead<TEAM, EPL> && row + gap < rows) load(row + gap);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float w[V], q[V];
      if (weight) parameter(kw, weight, n, w);
      if (vw) parameter(kvw, vw, n, q);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = n * V + e;
        h[i] = (h[i] - mu) * r;
        const float u = weight ? gr[i] * w[e] : gr[i], t = vw ? gr[i] * q[e] : 0.f;
        s[0] += u;
        s[1] += u * h[i];
        s[2] += vr[i];
        s[3] += vr[i] * h[i];
        s[4] += u * vr[i];
        s[5] += t;
        s[6] += t * h[i];
      }
    }
    team_sum<TEAM>(s, lds);
#pragma unroll
    for (int k = 0; k < 7; ++k) s[k] *= inv;
    const float q = s[4] - s[0] * s[2] - s[1] * s[3];
    const float tm = s[5] - r * (s[3] * s[0] + s[1] * s[2]), th = s[6] - 2.f * r * s[1] * s[3];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * TEAM + lane) * V;
      float w[V], pw[V], pb[V];
      if (weight) parameter(kw, weight, n, w);
      if (vw) parameter(kvw, vw, n, pw);
      if (vb) parameter(kvb, vb, n, pb);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = n * V + e;
        const float u = weight ? gr[i] * w[e] : gr[i];
        const float pv = r * (vr[i] - s[2] - h[i] * s[3]);
        const float t = (vw ? gr[i] * pw[e] : 0.f) - r * (s[3] * u + s[1] * vr[i]);
        dw[i] += gr[i] * pv;
        vr[i] = (weight ? w[e] * pv : pv) + (vw ? h[i] * pw[e] : 0.f) + (vb ? pb[e] : 0.f);
        h[i] = r * (t - tm - h[i] * th) - r * r * q * h[i];
      }
      if (dx) store_chunk(dx + row * (int64_t)width + c, width - c, h + n * V);
      if (dg) store_chunk(dg + row * (int64_t)width + c, width - c, vr + n * V);
    }
  }
  if (part_w) block_columns<TEAM, EPL, V>(dw, width, part_w + (int64_t)blockIdx.x * width, lds);
}

// out[c] = sum over the blocks' partial rows, 16 slices of them added per column and then in order.
template <typename T>
__global__ __launch_bounds__(256) void ln_param_kernel(const float* __restrict__ part_a, T* __restrict__ out_a,
                                                       const float* __restrict__ part_b, T* __restrict__ out_b,
                                                       int blocks, int width) {
  __shared__ float lds[16][17];
  const float* part = blockIdx.y ? part_b : part_a;
  T* out = blockIdx.y ? out_b : out_a;
  if (!part) return;
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float a = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int b = slice; b < blocks; b += 16) a += part[(int64_t)b * width + c];
  }
  lds[slice][col] = a;
  __syncthreads();
  if (slice == 0 && c < width) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][col];
    out[c] = (T)s;
  }
}

// Lanes and elements per lane that hold a row.
struct Shape {
  int team, epl;
};

Shape shape_of(int width, int chunk) {
  if (width <= 64) return {64 / chunk, chunk};
  if (width <= 128) return {16, 8};
  if (width <= 256) return {16, 16};
  if (width <= 512) return {64, 8};
  if (width <= 1024) return {64, 16};
  if (width <= 2048) return {64, 32};
  if (width <= 4096) return {256, 16};
  if (width <= 8192) return {512, 16};
  return {512, 32};
}

int64_t blocks_of(int64_t rows, int team, int64_t most) {
  const int teams = team > 256 ? 1 : 256 / team;
  return std::max<int64_t>(1, std::min<int64_t>(most, (rows + teams - 1) / teams));
}

// Blocks of the forward kernel: four a unit, two for the widest rows.  Measured at 512 / 1,024 / 2,048 blocks: 425,991 x 64
// FP32 56 / 41 / 44 us, 8,191 x 2,176 FP32 32 / 30 / 35, bfloat16 26 / 20 / 21, 2,048 x 8,192 bfloat16 14 / 16 / 18, FP32
// 28 / 29 / 36; 32,768 x 500 bfloat16, the other way, 30 / 20 / 17.
int64_t fwd_blocks(int64_t rows, int team, int width) { return blocks_of(rows, team, width <= 4096 ? 1024 : 512); }

// The blocks of the gradient kernels each leave a partial row per parameter: fewer of them for wide rows.  Measured at
// 256 / 512 / 1,024 blocks: 425,991 x 64 FP32 103 / 65 / 67 us, 8,191 x 2,176 bfloat16 44 / 36 / 45 us, 2,048 x 8,192
// bfloat16 37 / 53 / 83 us.
int64_t grad_blocks(int64_t rows, int width, int chunk) {
  return blocks_of(rows, shape_of(width, chunk).team, width <= 256 ? 1024 : width <= 4096 ? 512 : 256);
}

// The second derivative's: 425,991 x 64 FP32 102 / 112 us at 512 / 1,024 blocks, 65,536 x 250 70 / 72.
int64_t second_blocks(int64_t rows, int width, int chunk) {
  return blocks_of(rows, shape_of(width, chunk).team, width <= 4096 ? 512 : 256);
}

#define LN_CASE(TEAM_, EPL_, ...)                      \
  if (s.team == TEAM_ && s.epl == EPL_) {              \
    constexpr int TEAM = TEAM_, EPL = EPL_;            \
    __VA_ARGS__;                                       \
  }
#define LN_DISPATCH(T, ...)                                                    \
  {                                                                            \
    LN_CASE(64 / kChunk<T>, kChunk<T>, __VA_ARGS__)                            \
    else LN_CASE(16, 8, __VA_ARGS__) else LN_CASE(16, 16, __VA_ARGS__)         \
    else LN_CASE(64, 8, __VA_ARGS__) else LN_CASE(64, 16, __VA_ARGS__)         \
    else LN_CASE(64, 32, __VA_ARGS__) else LN_CASE(256, 16, __VA_ARGS__)       \
    else LN_CASE(512, 16, __VA_ARGS__) else LN_CASE(512, 32, __VA_ARGS__)     \
  }

template <typename T>
int run_fwd(const void* x, int64_t ldx, int64_t rows, int width, const void* weight, const void* bias, float eps,
            void* y, float* mean, float* rstd, hipStream_t st) {
  const Shape s = shape_of(width, kChunk<T>);
  const dim3 grid((unsigned)fwd_blocks(rows, s.team, width));
  LN_DISPATCH(T, hipLaunchKernelGGL((ln_fwd_kernel<T, TEAM, EPL>), grid, dim3(kThreads<TEAM>), 0, st, (const T*)x,
                                    ldx, rows, width, (const T*)weight, (const T*)bias, eps, (T*)y, mean, rstd))
  return dense_status("layer_norm_fwd launch");
}

template <typename T>
int run_bwd(const void* x, int64_t ldx, const void* g, int64_t ldg, int64_t rows, int width, const void* weight,
            const float* mean, const float* rstd, void* dx, void* dw, void* db, float* ws, hipStream_t st) {
  const Shape s = shape_of(width, kChunk<T>);
  const int64_t blocks = grad_blocks(rows, width, kChunk<T>);
  float* pw = dw ? ws : nullptr;
  float* pb = db ? ws + blocks * width : nullptr;
  LN_DISPATCH(T, hipLaunchKernelGGL((ln_bwd_kernel<T, TEAM, EPL>), dim3((unsigned)blocks), dim3(kThreads<TEAM>), 0,
                                    st, (const T*)x, ldx, (const T*)g, ldg, rows, width, (const T*)weight, mean, rstd,
                                    (T*)dx, pw, pb))
  if (dw || db)
    hipLaunchKernelGGL(ln_param_kernel<T>, dim3((unsigned)((width + 15) / 16), 2), dim3(256), 0, st, pw, (T*)dw, pb,
                       (T*)db, (int)blocks, width);
  return dense_status("layer_norm_bwd launch");
}

template <typename T>
int run_bwd2(const void* x, int64_t ldx, const void* g, int64_t ldg, const void* v, int64_t ldv, const void* vw,
             const void* vb, int64_t rows, int width, const void* weight, const float* mean, const float* rstd,
             void* dx, void* dg, void* dw, float* ws, hipStream_t st) {
  const Shape s = shape_of(width, kChunk<T>);
  const int64_t blocks = second_blocks(rows, width, kChunk<T>);   // (at most grad_blocks)
  float* pw = dw ? ws : nullptr;
  LN_DISPATCH(T, hipLaunchKernelGGL((ln_bwd2_kernel<T, TEAM, EPL>), dim3((unsigned)blocks), dim3(kThreads<TEAM>), 0,
                                    st, (const T*)x, ldx, (const T*)g, ldg, (const T*)v, ldv, (const T*)vw,
                                    (const T*)vb, rows, width, (const T*)weight, mean, rstd, (T*)dx, (T*)dg, pw))
  if (dw)
    hipLaunchKernelGGL(ln_param_kernel<T>, dim3((unsigned)((width + 15) / 16), 1), dim3(256), 0, st, pw, (T*)dw,
                       (const float*)nullptr, (T*)nullptr, (int)blocks, width);
  return dense_status("layer_norm_bwd2 launch");
}

const char* bad_sizes(int dtype, int64_t rows, int width) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "layer_norm: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (rows < 0 || width < 1) return "layer_norm: rows must not be negative and width at least 1";
  return nullptr;
}

}  // namespace

extern "C" {

int64_t ictc_layer_norm_workspace_bytes(int dtype, int64_t rows, int width) {
  if (bad_sizes(dtype, rows, width) || width > kMaxWidth) return -1;
  return 2 * grad_blocks(rows, width, dtype == ICTC_F32 ? 4 : 8) * width * (int64_t)sizeof(float);
}

int ictc_layer_norm_fwd(int dtype, const void* x, int64_t ldx, int64_t rows, int width, const void* weight,
                        const void* bias, float eps, void* y, float* mean, float* rstd, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (width > kMaxWidth) return dense_fail(ICTC_ERR_UNSUPPORTED, "layer_norm: rows of up to 16384 elements");
  if (ldx < width && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: row pitch below the width");
  if (!(eps >= 0.f)) return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: eps must not be negative");
  if (rows == 0) return ICTC_OK;
  if (!x || !y || !mean != !rstd) return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: null operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ICTC_F32) return run_fwd<float>(x, ldx, rows, width, weight, bias, eps, y, mean, rstd, st);
  if (dtype == ICTC_BF16) return run_fwd<bf16>(x, ldx, rows, width, weight, bias, eps, y, mean, rstd, st);
  return run_fwd<f16>(x, ldx, rows, width, weight, bias, eps, y, mean, rstd, st);
}

int ictc_layer_norm_bwd(int dtype, const void* x, int64_t ldx, const void* grad, int64_t ldg, int64_t rows, int width,
                        const void* weight, const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (width > kMaxWidth) return dense_fail(ICTC_ERR_UNSUPPORTED, "layer_norm: rows of up to 16384 elements");
  if ((ldx < width || ldg < width) && rows > 1)
    return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: row pitch below the width");
  if (rows > 0 && (!x || !grad || !mean || !rstd)) return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: null operand");
  if ((dweight || dbias) && (!workspace || workspace_bytes < ictc_layer_norm_workspace_bytes(dtype, rows, width)))
    return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: workspace smaller than ictc_layer_norm_workspace_bytes");
  if ((rows == 0 || !dx) && !dweight && !dbias) return ICTC_OK;
  hipStream_t st = (hipStream_t)stream;
  float* ws = (float*)workspace;
  if (dtype == ICTC_F32)
    return run_bwd<float>(x, ldx, grad, ldg, rows, width, weight, mean, rstd, dx, dweight, dbias, ws, st);
  if (dtype == ICTC_BF16)
    return run_bwd<bf16>(x, ldx, grad, ldg, rows, width, weight, mean, rstd, dx, dweight, dbias, ws, st);
  return run_bwd<f16>(x, ldx, grad, ldg, rows, width, weight, mean, rstd, dx, dweight, dbias, ws, st);
}

int ictc_layer_norm_bwd2(int dtype, const void* x, int64_t ldx, const void* grad, int64_t ldg, const void* v,
                         int64_t ldv, const void* vweight, const void* vbias, int64_t rows, int width,
                         const void* weight, const float* mean, const float* rstd, void* dx, void* dgrad,
                         void* dweight, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (width > kMaxWidth) return dense_fail(ICTC_ERR_UNSUPPORTED, "layer_norm: rows of up to 16384 elements");
  if ((ldx < width || ldg < width || ldv < width) && rows > 1)
    return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: row pitch below the width");
  if (rows > 0 && (!x || !grad || !v || !mean || !rstd))
    return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: null operand");
  if (dweight && (!workspace || workspace_bytes < ictc_layer_norm_workspace_bytes(dtype, rows, width)))
    return dense_fail(ICTC_ERR_ARGUMENT, "layer_norm: workspace smaller than ictc_layer_norm_workspace_bytes");
  if ((rows == 0 || (!dx && !dgrad)) && !dweight) return ICTC_OK;
  hipStream_t st = (hipStream_t)stream;
  float* ws = (float*)workspace;
  if (dtype == ICTC_F32)
    return run_bwd2<float>(x, ldx, grad, ldg, v, ldv, vweight, vbias, rows, width, weight, mean, rstd, dx, dgrad,
                           dweight, ws, st);
  if (dtype == ICTC_BF16)
    return run_bwd2<bf16>(x, ldx, grad, ldg, v, ldv, vweight, vbias, rows, width, weight, mean, rstd, dx, dgrad,
                          dweight, ws, st);
  return run_bwd2<f16>(x, ldx, grad, ldg, v, ldv, vweight, vbias, rows, width, weight, mean, rstd, dx, dgrad, dweight,
                       ws, st);
}

}  // extern "C"
