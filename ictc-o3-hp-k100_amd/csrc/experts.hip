// Linears chosen per row: row n goes through the matrix of its expert (an atom's element),
//   y[n] = W[e(n)] x[n] + b[e(n)],   gx[n] = W[e(n)]^T gy[n],
//   gW[e] = sum over its rows gy[n] x[n]^T,   gb[e] = sum over its rows gy[n],
// W [experts, outputs, inputs] of any width, FP32, bfloat16 or FP16, FP32 sums, each result rounded once.
//
// Rows come in expert order (perm, offsets: ictc_csr_build), so a tile of 128 rows has one expert and its product is
// an ordinary matrix product; the gather and the scatter of the rows happen in the tile's own loads and stores.  The
// tile list is implicit: a block finds its (expert, first row) by a scan of the group sizes, one expert a lane, so
// nothing is counted on the host and the grid is the upper bound rows / 128 + experts.
//
// Products run on v_mfma_f32_16x16x32; FP32 operands are split exactly into three bfloat16 parts of which the six
// leading products are kept (FP32-level accuracy, see split_bf16.h; an infinite FP32 input may give NaN).  Both
// operands of a step are staged in LDS as [row][reduction index], 16-byte chunks XORed with the row so that neither
// the stores nor the fragment reads share banks.  An operand whose memory runs along the other axis (the weights of
// gx, both operands of gW) is transposed in registers on its way to LDS: eight rows of a few columns per thread.
#include "dense.h"
#include "split_bf16.h"

#include <algorithm>

namespace {

typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 128;   // rows and columns of an output tile: four waves of 64 x 64

template <typename T>
struct Config {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;    // parts of an operand in LDS
  static constexpr int BK = sizeof(T) == 4 ? 32 : 64;  // reduction indices of a step
  static constexpr int CH = BK / 8;                    // chunks of a row in LDS
  static constexpr int PER = kTile * CH / 256;         // chunks staged by a thread
  static constexpr int NC = BK / 16;                   // columns per thread of a transposed operand
  static constexpr int PART = kTile * BK;              // 16-bit values of a part of an operand
};

template <typename T>
struct alignas(16) Eight {
  T e[8];
};

// p[0 .. n), zero past n
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* __restrict__ p, int n) {
  Eight<T> r;
  if (n >= 8) {
    if (sizeof(T) == 4) {
      *reinterpret_cast<u32x4*>(&r.e[0]) = *reinterpret_cast<const u32x4_any*>(p);
      *reinterpret_cast<u32x4*>(&r.e[4]) = *reinterpret_cast<const u32x4_any*>(p + 4);
    } else {
      *reinterpret_cast<u32x4*>(&r.e[0]) = *reinterpret_cast<const u32x4_any*>(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

// NC (2 or 4) values, 8 bytes
template <typename T>
struct alignas(8) Few {
  T e[Config<T>::NC];
};

template <typename T>
__device__ __forceinline__ Few<T> load_few(const T* __restrict__ p, int n) {
  Few<T> r;
  if (n >= Config<T>::NC) {
    *reinterpret_cast<u32x2*>(&r) = *reinterpret_cast<const u32x2_any*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < Config<T>::NC; ++i) r.e[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

// 16-bit offset of chunk `ch` of row `row` in a part of an operand
template <typename T>
__device__ __forceinline__ int lds_at(int row, int ch) {
  constexpr int CH = Config<T>::CH;
  const int swz = CH == 8 ? (row ^ (row >> 3)) & 7 : (row >> 2) & 3;
  return (row * CH + (ch ^ swz)) * 8;
}

template <typename T>
__device__ __forceinline__ void put(uint16_t* __restrict__ lds, int row, int ch, const Eight<T>& v) {
  uint16_t* at = lds + lds_at<T>(row, ch);
  if constexpr (sizeof(T) == 4) {
    const Split s = split8(v.e);
    *reinterpret_cast<bf16x8*>(at) = s.hi;
    *reinterpret_cast<bf16x8*>(at + Config<T>::PART) = s.mid;
    *reinterpret_cast<bf16x8*>(at + 2 * Config<T>::PART) = s.lo;
  } else {
    *reinterpret_cast<u32x4*>(at) = *reinterpret_cast<const u32x4*>(&v.e[0]);
  }
}

template <typename T>
__device__ __forceinline__ v4f mma(u32x4 a, u32x4 b, v4f c) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// The product of one 16 x 16 block over 32 reduction indices from the operands' parts.
template <typename T>
__device__ __forceinline__ v4f product(const u32x4 (&a)[Config<T>::NP], const u32x4 (&b)[Config<T>::NP], v4f c) {
  if constexpr (sizeof(T) == 4) {
    c = mma<T>(a[2], b[0], c);
    c = mma<T>(a[0], b[2], c);
    c = mma<T>(a[1], b[1], c);
    c = mma<T>(a[1], b[0], c);
    c = mma<T>(a[0], b[1], c);
  }
  return mma<T>(a[0], b[0], c);
}

template <typename T>
__device__ __forceinline__ void fragment(const uint16_t* __restrict__ lds, int row, int ch, u32x4 (&f)[Config<T>::NP]) {
  const uint16_t* at = lds + lds_at<T>(row, ch);
#pragma unroll
  for (int p = 0; p < Config<T>::NP; ++p) f[p] = *reinterpret_cast<const u32x4*>(at + p * Config<T>::PART);
}

// acc[i][j] += the block's step: rows 64 wa + 16 i of operand A by rows 64 wb + 16 j of operand B.
template <typename T>
__device__ __forceinline__ void step(const uint16_t* __restrict__ A, const uint16_t* __restrict__ B, int wa, int wb,
                                     v4f (&acc)[4][4]) {
  const int li = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int kk = 0; kk < Config<T>::BK / 32; ++kk) {
    u32x4 a[4][Config<T>::NP];
#pragma unroll
    for (int i = 0; i < 4; ++i) fragment<T>(A, 64 * wa + 16 * i + li, 4 * kk + g, a[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4 b[Config<T>::NP];
      fragment<T>(B, 64 * wb + 16 * j + li, 4 * kk + g, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] = product<T>(a[i], b, acc[i][j]);
    }
  }
}

// Run `t` of groups 0 .. G - 1 cut into runs of `rows` sorted rows: its group, first row, row count, index within
// the group and the group's runs.  ONE: a group without rows has one empty run.  False past the last run.  The same
// values in every lane of the wave, which has to be whole.
struct Run {
  int group, start, count, index, runs;
};

template <bool ONE>
__device__ __forceinline__ bool find_run(const int* __restrict__ off, int G, int rows, int t, Run& r) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < G; s0 += 64) {
    const int s = s0 + lane;
    int lo = 0, n = 0, runs = 0;
    if (s < G) {
      lo = off[s];
      n = off[s + 1] - lo;
      runs = (n + rows - 1) / rows;
      if (ONE && runs == 0) runs = 1;
    }
    int sum = runs;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (t < base + total) {
      const int f = __builtin_ctzll(__ballot(base + sum > t));
      r.group = s0 + f;
      r.runs = __builtin_amdgcn_readlane(runs, f);
      r.index = t - (base + __builtin_amdgcn_readlane(sum, f) - r.runs);
      r.start = __builtin_amdgcn_readlane(lo, f) + r.index * rows;
      r.count = min(rows, __builtin_amdgcn_readlane(n, f) - r.index * rows);
      return true;
    }
    base += total;
  }
  return false;
}

// Block `b` of `blocks` in an order that gives each of the eight dies (blocks go to them in turn) a contiguous part.
__device__ __forceinline__ int die_order(int b, int blocks) {
  const int per = blocks / 8, rest = blocks % 8, die = b & 7;
  return die * per + min(die, rest) + (b >> 3);
}

// A 128-row operand whose rows run along the reduction index.
template <typename T>
struct Straight {
  const T* row[Config<T>::PER];
  bool ok[Config<T>::PER];
  Eight<T> v[Config<T>::PER];

  static __device__ __forceinline__ int row_of(int i) { return (i * 256 + (int)threadIdx.x) / Config<T>::CH; }
  static __device__ __forceinline__ int chunk_of(int i) { return (i * 256 + (int)threadIdx.x) % Config<T>::CH; }

  __device__ __forceinline__ void load(int k0, int K) {
#pragma unroll
    for (int i = 0; i < Config<T>::PER; ++i) {
      const int k = k0 + 8 * chunk_of(i);
      v[i] = load8(row[i] + k, ok[i] ? K - k : 0);
    }
  }
  __device__ __forceinline__ void store(uint16_t* lds) const {
#pragma unroll
    for (int i = 0; i < Config<T>::PER; ++i) put(lds, row_of(i), chunk_of(i), v[i]);
  }
};

// An operand whose memory runs along its 128 rows: thread (kb, cg) takes reduction indices 8 kb .. and rows NC cg ...
template <typename T>
struct Across {
  static constexpr int NC = Config<T>::NC;
  Few<T> v[8];

  static __device__ __forceinline__ int column() { return (int)threadIdx.x % (kTile / NC) * NC; }
  static __device__ __forceinline__ int block() { return (int)threadIdx.x / (kTile / NC); }

  __device__ __forceinline__ void store(uint16_t* lds) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      Eight<T> e;
#pragma unroll
      for (int j = 0; j < 8; ++j) e.e[j] = v[j].e[c];
      put(lds, column() + c, block(), e);
    }
  }
};

// out[perm[r]] = M x[perm[r]] + b over the 128 columns of a block, M = W[e] [N, K] or, TRANS, the transpose of
// W[e] [K, N].  Operand A is the weights, so a lane ends with four consecutive columns of one row.
template <typename T, bool TRANS>
__global__ __launch_bounds__(256) void experts_rows_kernel(const T* __restrict__ x, int64_t ldx, int K,
                                                           const T* __restrict__ W, const T* __restrict__ bias, int N,
                                                           int experts, const int* __restrict__ perm,
                                                           const int* __restrict__ off, T* __restrict__ out) {
  using C = Config<T>;
  __shared__ __attribute__((aligned(16))) uint16_t As[C::NP * C::PART];
  __shared__ __attribute__((aligned(16))) uint16_t Bs[C::NP * C::PART];
  const int columns = (N + kTile - 1) / kTile;
  const int b = die_order(blockIdx.x, gridDim.x);
  Run run;
  if (!find_run<false>(off, experts + 1, kTile, b / columns, run)) return;
  const int n0 = b % columns * kTile;
  if (run.group == experts) {   // ids outside [0, experts): zero rows
    const int width = min(kTile, N - n0);
    for (int i = threadIdx.x; i < run.count * kTile; i += 256)
      if (i % kTile < width) out[(int64_t)perm[run.start + i / kTile] * N + n0 + i % kTile] = (T)0.f;
    return;
  }
  const T* w = W + (int64_t)run.group * N * K;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  Straight<T> xs, ws;
  Across<T> wt;
#pragma unroll
  for (int i = 0; i < C::PER; ++i) {
    const int r = xs.row_of(i);
    xs.ok[i] = r < run.count;
    xs.row[i] = x + (xs.ok[i] ? (int64_t)perm[run.start + r] * ldx : 0);
    ws.ok[i] = n0 + r < N;
    ws.row[i] = w + (ws.ok[i] ? (int64_t)(n0 + r) * K : 0);
  }
  auto load = [&](int k0) {
    xs.load(k0, K);
    if (!TRANS) {
      ws.load(k0, K);
    } else {
      const int c = n0 + wt.column();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = k0 + 8 * wt.block() + j;
        wt.v[j] = load_few(w + (int64_t)k * N + c, k < K ? N - c : 0);
      }
    }
  };
  v4f acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  load(0);
  for (int k0 = 0; k0 < K; k0 += C::BK) {
    xs.store(Bs);
    if (TRANS)
      wt.store(As);
    else
      ws.store(As);
    __syncthreads();
    if (k0 + C::BK < K) load(k0 + C::BK);
    step<T>(As, Bs, wave >> 1, wave & 1, acc);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = n0 + 64 * (wave >> 1) + 16 * i + 4 * g;
    float bv[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) bv[r] = bias && c + r < N ? (float)bias[(int64_t)run.group * N + c + r] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 64 * (wave & 1) + 16 * j + li;
      if (r >= run.count || c >= N) continue;
      T* o = out + (int64_t)perm[run.start + r] * N + c;
      T v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = (T)(acc[i][j][q] + bv[q]);
      if (c + 4 <= N) {
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<u32x4_any*>(o) = *reinterpret_cast<const u32x4*>(v);
        else
          *reinterpret_cast<u32x2_any*>(o) = *reinterpret_cast<const u32x2*>(v);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (c + q < N) o[q] = v[q];
      }
    }
  }
}

// Partial gradients of one run of an expert's rows: [M, K] of W (g^T x) and [M] of b (the blocks of column tile 0:
// the product of g with ones).  A group of one run is done; the others leave FP32 sums, run by run, in `part`.
template <typename T>
__global__ __launch_bounds__(256) void experts_outer_kernel(const T* __restrict__ gy, int64_t ldg, int M,
                                                            const T* __restrict__ x, int64_t ldx, int K, int experts,
                                                            int rows, const int* __restrict__ perm,
                                                            const int* __restrict__ off, T* __restrict__ gW,
                                                            T* __restrict__ gb, float* __restrict__ part) {
  using C = Config<T>;
  __shared__ __attribute__((aligned(16))) uint16_t As[C::NP * C::PART];
  __shared__ __attribute__((aligned(16))) uint16_t Bs[C::NP * C::PART];
  const int ct = (K + kTile - 1) / kTile, tiles = ct * ((M + kTile - 1) / kTile);
  const int b = die_order(blockIdx.x, gridDim.x), t = b / tiles;
  Run run;
  if (!find_run<true>(off, experts, rows, t, run)) return;
  const int k0 = b % tiles % ct * kTile, m0 = b % tiles / ct * kTile;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  Across<T> xs, gs;
  const int cx = k0 + xs.column(), cg = m0 + gs.column(), r0 = 8 * xs.block();
  auto load = [&](int s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = s + r0 + j;
      const bool ok = r < run.count;
      const int64_t node = ok ? perm[run.start + r] : 0;
      xs.v[j] = load_few(x + node * ldx + cx, ok ? K - cx : 0);
      gs.v[j] = load_few(gy + node * ldg + cg, ok ? M - cg : 0);
    }
  };
  const bool bias = gb != nullptr && k0 == 0 && wave < 2;
  const uint32_t one = sizeof(T) == 4 || __is_same(T, bf16) ? 0x3f803f80u : 0x3c003c00u;
  v4f acc[4][4], accb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    accb[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  load(0);
  for (int s = 0; s < run.count; s += C::BK) {
    xs.store(As);
    gs.store(Bs);
    __syncthreads();
    if (s + C::BK < run.count) load(s + C::BK);
    step<T>(As, Bs, wave >> 1, wave & 1, acc);
    if (bias) {
#pragma unroll
      for (int kk = 0; kk < C::BK / 32; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u32x4 f[C::NP];
          fragment<T>(Bs, 64 * (wave & 1) + 16 * j + li, 4 * kk + g, f);
#pragma unroll
          for (int p = C::NP - 1; p >= 0; --p) accb[j] = mma<T>(u32x4{one, one, one, one}, f[p], accb[j]);
        }
    }
    __syncthreads();
  }
  const bool whole = run.runs == 1;
  const int64_t MK = (int64_t)M * K;
  float* pw = part + (int64_t)t * (MK + M);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 64 * (wave & 1) + 16 * j + li;
    if (m >= M) continue;
    if (bias && g == 0) {
      if (whole)
        gb[(int64_t)run.group * M + m] = (T)accb[j][0];
      else
        pw[MK + m] = accb[j][0];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + 64 * (wave >> 1) + 16 * i + 4 * g;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (k + q >= K) continue;
        if (whole)
          gW[(int64_t)run.group * MK + (int64_t)m * K + k + q] = (T)acc[i][j][q];
        else
          pw[(int64_t)m * K + k + q] = acc[i][j][q];
      }
    }
  }
}

// Sums of the runs' partial gradients in run order, for experts of more than one run.
template <typename T>
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ part, int64_t MK, int M,
                                                          const int* __restrict__ off, int rows, T* __restrict__ gW,
                                                          T* __restrict__ gb) {
  const int s = blockIdx.y, lane = threadIdx.x & 63;
  const int runs = (off[s + 1] - off[s] + rows - 1) / rows;
  if (runs < 2) return;
  int first = 0;   // runs of the experts before this one
  for (int e = lane; e < s; e += 64) first += max(1, (off[e + 1] - off[e] + rows - 1) / rows);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) first += __shfl_xor(first, d);
  const int64_t size = MK + M, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size || (i >= MK && !gb)) return;
  const float* p = part + (int64_t)first * size + i;
  float a = 0.f;
#pragma unroll 4
  for (int r = 0; r < runs; ++r) a += p[(int64_t)r * size];
  if (i < MK)
    gW[(int64_t)s * MK + i] = (T)a;
  else
    gb[(int64_t)s * M + i - MK] = (T)a;
}

// Rows of a run of the weight gradient: enough runs to fill the card where there are few tiles, but no run so short
// that its partial sums (4 bytes a weight) cost more than its rows.
int outer_rows(int64_t n, int experts, int M, int K) {
  const int64_t tiles = (int64_t)((M + kTile - 1) / kTile) * ((K + kTile - 1) / kTile);
  const int64_t wanted = std::max<int64_t>(1, 1024 / tiles);
  const int64_t rows = std::max<int64_t>(512, (n + wanted - 1) / wanted);
  return (int)std::min<int64_t>((rows + 63) / 64 * 64, int64_t(1) << 30);
}

int64_t outer_runs(int64_t n, int experts, int rows) { return n / rows + experts; }

const char* bad_sizes(int dtype, int64_t rows, int64_t inputs, int64_t outputs, int experts) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "expert_linear: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (rows < 0 || rows >= (int64_t(1) << 31) - 2) return "expert_linear: up to 2^31 - 3 rows";
  if (inputs < 1 || outputs < 1 || inputs > 65536 || outputs > 65536) return "expert_linear: 1 to 65536 inputs and outputs";
  if (experts < 1 || experts > 65535) return "expert_linear: 1 to 65535 experts";
  return nullptr;
}

template <typename T>
void launch_rows(const void* x, int64_t ldx, int K, const void* W, const void* bias, int N, int experts,
                 const int* perm, const int* off, int transpose, void* out, unsigned blocks, hipStream_t st) {
  if (transpose)
    hipLaunchKernelGGL((experts_rows_kernel<T, true>), dim3(blocks), dim3(256), 0, st, (const T*)x, ldx, K,
                       (const T*)W, (const T*)bias, N, experts, perm, off, (T*)out);
  else
    hipLaunchKernelGGL((experts_rows_kernel<T, false>), dim3(blocks), dim3(256), 0, st, (const T*)x, ldx, K,
                       (const T*)W, (const T*)bias, N, experts, perm, off, (T*)out);
}

template <typename T>
void launch_outer(const void* gy, int64_t ldg, int M, const void* x, int64_t ldx, int K, int64_t n, int experts,
                  int rows, const int* perm, const int* off, void* gW, void* gb, float* part, unsigned blocks,
                  hipStream_t st) {
  hipLaunchKernelGGL(experts_outer_kernel<T>, dim3(blocks), dim3(256), 0, st, (const T*)gy, ldg, M, (const T*)x, ldx,
                     K, experts, rows, perm, off, (T*)gW, (T*)gb, part);
  if (n > rows) {   // an expert may have several runs
    const int64_t MK = (int64_t)M * K;
    hipLaunchKernelGGL(experts_sum_kernel<T>, dim3((unsigned)((MK + M + 255) / 256), (unsigned)experts), dim3(256), 0,
                       st, part, MK, M, off, rows, (T*)gW, (T*)gb);
  }
}

}  // namespace

extern "C" {

int ictc_expert_linear(int dtype, const void* x, int64_t ldx, int64_t rows, int inputs, const void* weight,
                       const void* bias, int outputs, int experts, const int32_t* perm, const int32_t* offsets,
                       int transpose, void* out, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, inputs, outputs, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (rows == 0) return ICTC_OK;
  if (ldx < inputs && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "expert_linear: row pitch below the inputs");
  if (!x || !weight || !perm || !offsets || !out) return dense_fail(ICTC_ERR_ARGUMENT, "expert_linear: null operand");
  const int64_t blocks = (rows / kTile + experts + 1) * ((outputs + kTile - 1) / kTile);
  if (blocks >= (int64_t(1) << 31)) return dense_fail(ICTC_ERR_UNSUPPORTED, "expert_linear: too many tiles");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ICTC_F32)
    launch_rows<float>(x, ldx, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, (unsigned)blocks, st);
  else if (dtype == ICTC_BF16)
    launch_rows<bf16>(x, ldx, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, (unsigned)blocks, st);
  else
    launch_rows<f16>(x, ldx, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, (unsigned)blocks, st);
  return dense_status("expert_linear launch");
}

int64_t ictc_expert_outer_workspace_bytes(int dtype, int64_t rows, int inputs, int outputs, int experts) {
  if (bad_sizes(dtype, rows, inputs, outputs, experts)) return -1;
  const int run = outer_rows(rows, experts, outputs, inputs);
  return rows > run ? outer_runs(rows, experts, run) * ((int64_t)outputs * inputs + outputs) * (int64_t)sizeof(float) : 0;
}

int ictc_expert_outer(int dtype, const void* grad, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int inputs,
                      int outputs, int experts, const int32_t* perm, const int32_t* offsets, void* dweight,
                      void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, inputs, outputs, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if ((ldx < inputs || ldg < outputs) && rows > 1)
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: row pitch below the row");
  if (!offsets || !dweight || (rows > 0 && (!grad || !x || !perm)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: null operand");
  const int64_t need = ictc_expert_outer_workspace_bytes(dtype, rows, inputs, outputs, experts);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: workspace smaller than ictc_expert_outer_workspace_bytes");
  const int run = outer_rows(rows, experts, outputs, inputs);
  const int64_t tiles = (int64_t)((outputs + kTile - 1) / kTile) * ((inputs + kTile - 1) / kTile);
  const int64_t blocks = outer_runs(rows, experts, run) * tiles;
  if (blocks >= (int64_t(1) << 31)) return dense_fail(ICTC_ERR_UNSUPPORTED, "expert_outer: too many tiles");
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  if (dtype == ICTC_F32)
    launch_outer<float>(grad, ldg, outputs, x, ldx, inputs, rows, experts, run, perm, offsets, dweight, dbias, part, (unsigned)blocks, st);
  else if (dtype == ICTC_BF16)
    launch_outer<bf16>(grad, ldg, outputs, x, ldx, inputs, rows, experts, run, perm, offsets, dweight, dbias, part, (unsigned)blocks, st);
  else
    launch_outer<f16>(grad, ldg, outputs, x, ldx, inputs, rows, experts, run, perm, offsets, dweight, dbias, part, (unsigned)blocks, st);
  return dense_status("expert_outer launch");
}

}  // extern "C"
