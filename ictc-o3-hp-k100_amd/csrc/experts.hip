// Linears chosen per row: row n goes through the matrix of its expert (an atom's element),
//   y[n] = W[e(n)] x[n] + b[e(n)],   gx[n] = W[e(n)]^T gy[n],
//   gW[e] = sum over its rows gy[n] x[n]^T,   gb[e] = sum over its rows gy[n],
// W [experts, outputs, inputs] of any width, FP32, bfloat16 or FP16, FP32 sums, each result rounded once.
//
// Rows come in expert order (perm, offsets: ictc_expert_order), so a tile of rows has one expert and its product is an
// ordinary matrix product; the gather and the scatter of the rows happen in the tile's own loads and stores.  The tile
// list is implicit: a block finds its (expert, first row) by a scan of the group sizes, one expert a lane, so nothing is
// counted on the host and the grid is an upper bound (most_runs).
//
// Products run on v_mfma_f32_16x16x32; FP32 operands are split exactly into three bfloat16 parts of which the six
// leading products are kept (FP32-level accuracy, see split_bf16.h; an infinite FP32 input may give NaN).  Here are the
// order, the products of few rows, the sums of partial gradients, the choice among the kernels, and kernels for rows of
// under 16 bytes; those of experts_direct.hip take the rest.  Both operands of a step here are staged in LDS as
// [row][reduction index], 16-byte chunks XORed with the row so that neither the stores nor the fragment reads share
// banks.  An operand whose memory runs along the other axis (the weights of gx, both operands of gW) is transposed in
// registers on its way to LDS: eight rows of a few columns per thread.
#include <algorithm>

#include "experts.h"

namespace {

// Rows of under 16 bytes: tiles of 64 x 64 outputs by four waves of 32 x 32.
constexpr int TILE = 64;

template <typename T>
struct Config {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;                     // parts of an operand in LDS
  static constexpr int BK = 64;                                         // reduction indices of a step
  static constexpr int CH = BK / 8;                                     // chunks of a row in LDS
  static constexpr int PER = TILE * CH / 256;                           // chunks staged by a thread
  static constexpr int NC = TILE * BK / 2048;                           // columns per thread of a transposed operand
  static constexpr int PART = TILE * BK;                                // 16-bit values of a part of an operand
  static constexpr int NI = TILE / 32;                                  // blocks of 16 a side of a wave's tile
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

// NC (2 or 4) values, 4 or 8 bytes
template <typename T, int NC>
struct alignas(NC * sizeof(T)) Few {
  T e[NC];
};

template <typename T, int NC>
__device__ __forceinline__ Few<T, NC> load_few(const T* __restrict__ p, int n) {
  typedef uint32_t u32_any __attribute__((aligned(2)));
  Few<T, NC> r;
  if (n >= NC) {
    if constexpr (NC * sizeof(T) == 8)
      *reinterpret_cast<u32x2*>(&r) = *reinterpret_cast<const u32x2_any*>(p);
    else
      *reinterpret_cast<uint32_t*>(&r) = *reinterpret_cast<const u32_any*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i) r.e[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

// 16-bit offset of chunk `ch` of row `row` in a part of an operand
__device__ __forceinline__ int lds_at(int row, int ch) { return (row * 8 + (ch ^ ((row ^ (row >> 3)) & 7))) * 8; }

template <typename T>
__device__ __forceinline__ void put(uint16_t* __restrict__ lds, int row, int ch, const Eight<T>& v) {
  using C = Config<T>;
  uint16_t* at = lds + lds_at(row, ch);
  if constexpr (sizeof(T) == 4) {
    const Split s = split8_pairs(v.e);
    *reinterpret_cast<bf16x8*>(at) = s.hi;
    *reinterpret_cast<bf16x8*>(at + C::PART) = s.mid;
    *reinterpret_cast<bf16x8*>(at + 2 * C::PART) = s.lo;
  } else {
    *reinterpret_cast<u32x4*>(at) = *reinterpret_cast<const u32x4*>(&v.e[0]);
  }
}

template <typename T>
__device__ __forceinline__ void fragment(const uint16_t* __restrict__ lds, int row, int ch,
                                         u32x4 (&f)[Config<T>::NP]) {
  using C = Config<T>;
  const uint16_t* at = lds + lds_at(row, ch);
#pragma unroll
  for (int p = 0; p < C::NP; ++p) f[p] = *reinterpret_cast<const u32x4*>(at + p * C::PART);
}

// acc[i][j] += the block's step: rows 16 (wa NI + i) of operand A by rows 16 (wb NI + j) of operand B.
template <typename T>
__device__ __forceinline__ void step(const uint16_t* __restrict__ A, const uint16_t* __restrict__ B, int wa, int wb,
                                     v4f (&acc)[Config<T>::NI][Config<T>::NI]) {
  using C = Config<T>;
  const int li = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int kk = 0; kk < C::BK / 32; ++kk) {
    u32x4 a[C::NI][C::NP];
#pragma unroll
    for (int i = 0; i < C::NI; ++i) fragment<T>(A, 16 * (wa * C::NI + i) + li, 4 * kk + g, a[i]);
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      u32x4 b[C::NP];
      fragment<T>(B, 16 * (wb * C::NI + j) + li, 4 * kk + g, b);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) acc[i][j] = product<T>(a[i], b, acc[i][j]);
    }
  }
}

// An operand whose rows run along the reduction index.
template <typename T>
struct Straight {
  using C = Config<T>;
  const T* row[C::PER];
  bool ok[C::PER];
  Eight<T> v[C::PER];

  static __device__ __forceinline__ int row_of(int i) { return (i * 256 + (int)threadIdx.x) / C::CH; }
  static __device__ __forceinline__ int chunk_of(int i) { return (i * 256 + (int)threadIdx.x) % C::CH; }

  __device__ __forceinline__ void load(int k0, int K) {
#pragma unroll
    for (int i = 0; i < C::PER; ++i) {
      const int k = k0 + 8 * chunk_of(i);
      v[i] = load8(row[i] + k, ok[i] ? K - k : 0);
    }
  }
  __device__ __forceinline__ void store(uint16_t* lds) const {
#pragma unroll
    for (int i = 0; i < C::PER; ++i) put<T>(lds, row_of(i), chunk_of(i), v[i]);
  }
};

// An operand whose memory runs along its rows: thread (kb, cg) takes reduction indices 8 kb .. and rows NC cg ...
template <typename T>
struct Across {
  static constexpr int NC = Config<T>::NC;
  Few<T, NC> v[8];

  static __device__ __forceinline__ int column() { return (int)threadIdx.x % (TILE / NC) * NC; }
  static __device__ __forceinline__ int block() { return (int)threadIdx.x / (TILE / NC); }

  __device__ __forceinline__ void store(uint16_t* lds) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      Eight<T> e;
#pragma unroll
      for (int j = 0; j < 8; ++j) e.e[j] = v[j].e[c];
      put<T>(lds, column() + c, block(), e);
    }
  }
};

// out[perm[r]] = M x[perm[r]] + b over the columns of a tile, M = W[e] [N, K] or, TRANS, the transpose of
// W[e] [K, N].  Operand A is the weights, so a lane ends with four consecutive columns of one row.
template <typename T, bool TRANS>
__global__ __launch_bounds__(256) void experts_rows_kernel(const T* __restrict__ x, int64_t ldx, int K,
                                                           const T* __restrict__ W, const T* __restrict__ bias, int N,
                                                           int experts, const int* __restrict__ perm,
                                                           const int* __restrict__ off, T* __restrict__ out) {
  using C = Config<T>;
  __shared__ __attribute__((aligned(16))) uint16_t As[C::NP * C::PART];
  __shared__ __attribute__((aligned(16))) uint16_t Bs[C::NP * C::PART];
  const int columns = (N + TILE - 1) / TILE;
  const int b = die_order(blockIdx.x, gridDim.x);
  Run run;
  if (!find_run(off, experts + 1, TILE, b / columns, run)) return;
  const int n0 = b % columns * TILE;
  if (run.group == experts) {   // ids outside [0, experts): zero rows
    const int width = min(TILE, N - n0);
    for (int i = threadIdx.x; i < run.count * TILE; i += 256)
      if (i % TILE < width) out[(int64_t)perm[run.start + i / TILE] * N + n0 + i % TILE] = (T)0.f;
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
        wt.v[j] = load_few<T, C::NC>(w + (int64_t)k * N + c, k < K ? N - c : 0);
      }
    }
  };
  v4f acc[C::NI][C::NI];
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NI; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
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
  // all of the bias and row numbers are asked for before the first is needed
  T bv[C::NI][4];
  T* row[C::NI];
#pragma unroll
  for (int i = 0; i < C::NI; ++i) {
    const int c = n0 + TILE / 2 * (wave >> 1) + 16 * i + 4 * g;
    const T* bp = bias + (int64_t)run.group * N + c;
#pragma unroll
    for (int q = 0; q < 4; ++q) bv[i][q] = bias && c + q < N ? bp[q] : (T)0.f;
    const int r = TILE / 2 * (wave & 1) + 16 * i + li;
    row[i] = out + (int64_t)perm[run.start + (r < run.count ? r : 0)] * N;
  }
#pragma unroll
  for (int j = 0; j < C::NI; ++j) {
    if (TILE / 2 * (wave & 1) + 16 * j + li >= run.count) continue;
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      const int c = n0 + TILE / 2 * (wave >> 1) + 16 * i + 4 * g;
      if (c >= N) continue;
      T* o = row[j] + c;
      T v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = (T)(acc[i][j][q] + (float)bv[i][q]);
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

// The same for few rows: a block takes 16 rows of an expert and 32 columns, its eight waves share the reduction, and
// every lane reads its fragments' values from memory itself, so a call is one round of loads, not a chain of steps (16
// rows of 1,024 -> 1,024 FP32 over eight experts: 8.9 us, 25 in tiles of 64).  The waves' sums are added in order.  Two
// blocks share a unit.
constexpr int kFewRows = 16, kFewColumns = 32, kFewWaves = 8;

template <typename T>
__device__ __forceinline__ void parts(const Eight<T>& v, u32x4 (&f)[sizeof(T) == 4 ? 3 : 1]) {
  if constexpr (sizeof(T) == 4) {
    const Split s = split8_pairs(v.e);
    f[0] = __builtin_bit_cast(u32x4, s.hi);
    f[1] = __builtin_bit_cast(u32x4, s.mid);
    f[2] = __builtin_bit_cast(u32x4, s.lo);
  } else {
    f[0] = *reinterpret_cast<const u32x4*>(&v.e[0]);
  }
}

template <typename T, bool TRANS>
__global__ __launch_bounds__(kFewWaves * 64, 4) void experts_few_kernel(const T* __restrict__ x, int64_t ldx, int K,
                                                                    const T* __restrict__ W,
                                                                    const T* __restrict__ bias, int N, int experts,
                                                                    const int* __restrict__ perm,
                                                                    const int* __restrict__ off,
                                                                    T* __restrict__ out) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1, AHEAD = 4;
  __shared__ v4f sums[kFewWaves][2][64];
  const int columns = (N + kFewColumns - 1) / kFewColumns;
  Run run;
  if (!find_run(off, experts + 1, kFewRows, blockIdx.x / columns, run)) return;
  const int n0 = blockIdx.x % columns * kFewColumns;
  const bool valid = run.group < experts;   // rows of no expert: zeros
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* w = W + (int64_t)(valid ? run.group : 0) * N * K;
  const bool row = valid && li < run.count;
  const T* xr = x + (row ? (int64_t)perm[run.start + li] * ldx : 0);
  const int per = (K + kFewWaves * 32 - 1) / (kFewWaves * 32) * 32, end = min(K, (wave + 1) * per);
  v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
  for (int k0 = wave * per; valid && k0 < end; k0 += 32 * AHEAD) {
    Eight<T> xv[AHEAD], wv[AHEAD][2];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int k = k0 + 32 * s + 8 * g, left = end - k;
      xv[s] = load8(xr + k, row ? left : 0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = n0 + 16 * i + li;
        if (!TRANS) {
          wv[s][i] = load8(w + (int64_t)c * K + k, c < N ? left : 0);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) wv[s][i].e[e] = c < N && e < left ? w[(int64_t)(k + e) * N + c] : (T)0.f;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      u32x4 b[NP];
      parts(xv[s], b);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4 a[NP];
        parts(wv[s][i], a);
        acc[i] = product<T>(a, b, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= 2 || li >= run.count) return;   // wave i adds the column block i: four columns of one row a lane
  v4f t = sums[0][wave][lane];
#pragma unroll
  for (int v = 1; v < kFewWaves; ++v) t += sums[v][wave][lane];
  const int c = n0 + 16 * wave + 4 * g;
  T* o = out + (int64_t)perm[run.start + li] * N + c;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (c + q < N) o[q] = valid ? (T)(t[q] + (bias ? (float)bias[(int64_t)run.group * N + c + q] : 0.f)) : (T)0.f;
}

// The stable order of the rows by expert (ids outside [0, experts) last).  A block takes up to kOrderRows of them: each
// wave counts the experts of a run of rows, the counts are scanned expert by expert and wave by wave, and the waves place
// their rows.  Lanes of one expert find each other by one ballot for each bit of the id.  What a row needs for its place,
// the expert, the lanes of it below and how many there are, is kept in one register, so the ids are read once, all of a
// lane's at once.  One block does it alone; of several, each has `span` rows and adds up, from all blocks' counts
// ([blocks, experts + 1], the kernel below), what lies before its own.  Bound by latency: a chain of loads, ballots and
// barriers (8,192 rows of ten ids in one block 7.9 us; 131,072 in 128 blocks 3 + 5 us).
//
// More than 1,023 experts (entries of a table) are ordered by the low bits of the id and then, stably, by the ones above, up
// to ten at a time: each pass leaves ids and row numbers, the last the row numbers and sorted ids, of which
// order_offsets_kernel makes the offsets (425,991 rows of 7,921 ids: 31 us, 125 by the general sort).
constexpr int kOrderExperts = 1023, kOrderWaves = 16, kOrderAtOnce = 16, kOrderBlocks = 1024;
constexpr int kOrderRows = kOrderWaves * kOrderAtOnce * 64;

// What a pass takes and leaves: row i's id, or of a later pass the key and number that the one before left at i.
enum class Pass { kOnly, kFirst, kLater };
struct OrderIn {
  const int64_t* ids;
  const int *keys, *rows;
  int experts, shift, groups;   // digit: key >> shift & (groups - 1); of the only pass the key, groups = experts + 1
};
struct OrderOut {
  int *perm, *keys, *off;
};

// A row's id or key as it lies in memory (-1: there is no row), and the key.  (Apart, so that loads are not waited for one
// by one.)
template <Pass P>
__device__ __forceinline__ int64_t order_raw(const OrderIn& in, int row, bool there) {
  if (P == Pass::kLater) return there ? in.keys[row] : -1;
  return there ? in.ids[row] : -1;
}

template <Pass P>
__device__ __forceinline__ uint32_t order_key(const OrderIn& in, int64_t raw) {
  if (P == Pass::kLater) return (uint32_t)raw;
  return (uint64_t)raw < (uint64_t)in.experts ? (uint32_t)raw : (uint32_t)in.experts;
}

template <Pass P>
__device__ __forceinline__ uint32_t order_digit(const OrderIn& in, uint32_t key) {
  return P == Pass::kOnly ? key : key >> in.shift & (uint32_t)(in.groups - 1);
}

template <Pass P>
__global__ __launch_bounds__(1024) void experts_count_kernel(OrderIn in, int n, int span, int* __restrict__ counts) {
  __shared__ int count[kOrderExperts + 1];
  if ((int)threadIdx.x < in.groups) count[threadIdx.x] = 0;
  __syncthreads();
  const int begin = blockIdx.x * span, end = min(n, begin + span);
  for (int r0 = begin + (int)threadIdx.x; r0 < end; r0 += 4096) {
    int64_t raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = order_raw<P>(in, r0 + i * 1024, r0 + i * 1024 < end);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r0 + i * 1024 < end) atomicAdd(&count[order_digit<P>(in, order_key<P>(in, raw[i]))], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x < in.groups) counts[blockIdx.x * in.groups + threadIdx.x] = count[threadIdx.x];
}

template <Pass P>
__global__ __launch_bounds__(1024) void experts_order_kernel(OrderIn in, int n, int bits, int span,
                                                             const int* __restrict__ counts, OrderOut out) {
  __shared__ int count[kOrderWaves][kOrderExperts + 1];
  __shared__ int wave_total[kOrderWaves];
  const int lane = threadIdx.x & 63, groups = in.groups, group = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ int totals[kOrderExperts + 1], befores[kOrderExperts + 1];   // of each group: all rows, those of the blocks before
  for (int i = threadIdx.x; i < kOrderWaves * groups; i += 1024) count[i / groups][i % groups] = 0;
  totals[threadIdx.x] = befores[threadIdx.x] = 0;
  __syncthreads();
  if (counts) {   // the threads left over share a group's blocks
    const int width = 1 << bits, at = threadIdx.x & (width - 1);
    int all = 0, earlier = 0;
    if (at < groups) {
      constexpr int AT_ONCE = 16;
      const int step = 1024 / width;
      for (int b0 = threadIdx.x / width; b0 < (int)gridDim.x; b0 += AT_ONCE * step) {
        int c[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) c[i] = b0 + i * step < (int)gridDim.x ? counts[(b0 + i * step) * groups + at] : 0;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          all += c[i];
          earlier += b0 + i * step < (int)blockIdx.x ? c[i] : 0;
        }
      }
      atomicAdd(&totals[at], all);
      atomicAdd(&befores[at], earlier);
    }
  }
  const int first = blockIdx.x * span, rows = min(span, n - first);
  const int per = ((rows + kOrderWaves - 1) / kOrderWaves + 63) / 64 * 64;
  const int begin = first + wave * per, end = min(first + rows, begin + per);
  int* mine = count[wave];
  uint32_t place[kOrderAtOnce];   // digit | lanes below << 10 | lanes << 16
  int64_t raw[kOrderAtOnce];
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) raw[i] = order_raw<P>(in, begin + i * 64 + lane, begin + i * 64 + lane < end);
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) {
    const int r0 = begin + i * 64;
    if (r0 >= end) break;
    const uint32_t digit = order_digit<P>(in, order_key<P>(in, raw[i]));
    const uint64_t here = __ballot(r0 + lane < end);
    uint32_t lo = (uint32_t)here, hi = (uint32_t)(here >> 32);   // the lanes whose row has this lane's digit
    int x = (int)(digit << (32 - bits));
    for (int b = 0; b < bits; ++b, x <<= 1) {
      const uint64_t set = __ballot(x < 0);
      lo &= ~((uint32_t)set ^ (uint32_t)(x >> 31));
      hi &= ~((uint32_t)(set >> 32) ^ (uint32_t)(x >> 31));
    }
    const uint64_t m = (uint64_t)hi << 32 | lo;
    const int below = __popcll(m & ((uint64_t(1) << lane) - 1)), lanes = __popcll(m);
    place[i] = digit | below << 10 | lanes << 16;
    if (r0 + lane < end && below == 0) atomicAdd(&mine[digit], lanes);
  }
  __syncthreads();
  int here = 0, total = totals[group], before = befores[group];
  if (group < groups) {
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) {
      const int c = count[w][group];
      count[w][group] = here;
      here += c;
    }
  }
  if (!counts) total = here;
  int sum = scan_lanes(total);
  if (lane == 63) wave_total[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += wave_total[w];
  if (group < groups) {
    const int start = sum - total;
    if (P == Pass::kOnly && blockIdx.x == 0) out.off[group] = start;
    if (P == Pass::kOnly && blockIdx.x == 0 && group == in.experts) out.off[groups] = n;
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) count[w][group] += start + before;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) {
    const int r0 = begin + i * 64;
    if (r0 >= end) break;
    const bool ok = r0 + lane < end;
    const int digit = place[i] & 1023u, below = place[i] >> 10 & 63u, lanes = place[i] >> 16;
    if (ok) {
      const int to = mine[digit] + below;
      out.perm[to] = P == Pass::kLater ? in.rows[r0 + lane] : r0 + lane;
      if (P != Pass::kOnly) out.keys[to] = (int)order_key<P>(in, raw[i]);
    }
    wave_meet();
    if (ok && below == 0) atomicAdd(&mine[digit], lanes);   // (before the next rows' reads: LDS keeps a wave's order)
    wave_meet();
  }
}

// First place of sorted keys [n] that holds `key` or more, by a wave: 64 places looked at together, then 64 of the part
// between two of them.
__device__ __forceinline__ int first_place(const int* __restrict__ keys, int n, uint32_t key) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t m = __ballot(at < hi && (uint32_t)keys[at < hi ? at : lo] >= key);
    const int f = m ? __builtin_ctzll(m) : (hi - lo - 1) / step + 1;   // looked at: f are below the key
    if (m) hi = lo + f * step;
    if (f > 0) lo += (f - 1) * step + 1;
  }
  return lo;
}

// off[k] = the first place of sorted keys [n] that holds k or more, for k of 0 .. experts + 1.  A place fills the offsets
// from the key before it to its own, long gaps with its wave; but of a gap the whole spans of kSpan offsets (from
// multiples of it) are filled by a wave each, of the blocks behind the places', so that few rows, or ids side by side, of
// many entries do not keep one wave; and a wave has only eight places where most gaps are long (the whole order of 5 rows
// of a million entries 484 -> 16 us, of 33.5 million 15.8 ms -> 34 us).  Offsets are unsigned: experts + 2 may be
// 2^31 - 1, and a step past it.
constexpr uint32_t kSpan = 1024;
__global__ __launch_bounds__(256) void order_offsets_kernel(const int* __restrict__ keys, int n, uint32_t experts,
                                                            int each, int place_blocks, int* __restrict__ off) {
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x >= place_blocks) {
    const uint32_t first = ((blockIdx.x - place_blocks) * 4 + (threadIdx.x >> 6)) * kSpan;
    if (first + kSpan > experts + 2) return;
    const int p = first_place(keys, n, first);
    if (p < n && (uint32_t)keys[p] + 1 < first + kSpan) return;   // a key within it
    for (uint32_t k = lane; k < kSpan; k += 64) off[first + k] = p;
    return;
  }
  const int p = (blockIdx.x * 4 + (threadIdx.x >> 6)) * each + lane;
  uint32_t from = 0, to = 0;   // offsets from .. to - 1 are p
  if (lane < each && p <= n) {
    from = p > 0 ? (uint32_t)keys[p - 1] + 1 : 0;
    to = p < n ? (uint32_t)keys[p] + 1 : experts + 2;
  }
  const bool wide = to - from > 8;
  if (!wide)
    for (uint32_t k = from; k < to; ++k) off[k] = p;
  for (uint64_t m = __ballot(wide); m; m &= m - 1) {
    const int l = __builtin_ctzll(m);
    const uint32_t a = __builtin_amdgcn_readlane(from, l), b = __builtin_amdgcn_readlane(to, l),
                   q = __builtin_amdgcn_readlane(p, l);
    uint32_t spans = (a + kSpan - 1) / kSpan * kSpan, behind = b / kSpan * kSpan;   // whole ones: from, to
    if (behind <= spans) spans = behind = b;
    for (uint32_t k = a + lane; k < spans; k += 64) off[k] = q;
    for (uint32_t k = behind + lane; k < b; k += 64) off[k] = q;
  }
}

int64_t tiles_of(int64_t n, int tile) { return (n + tile - 1) / tile; }

int id_bits(int64_t experts) {
  int bits = 1;
  while (experts >> bits) ++bits;
  return bits;
}

// Rows of a block: all of few rows; 1,024, and more once those would be more than 256 blocks (over 255 ids 2,048 and 128);
// and zero: the general sort.  Measured in us, one block / several: ten experts 500 rows 4.6 / 8.0, 8,192 8.0 / 8.5.
// Both kernels at 64 / 128 / 256 blocks and 4,096 / 2,048 / 1,024 rows at least: 131,072 rows of ten experts 10.5 / 8.9 /
// 8.3, 30,011 of 89 11.1 / 9.5 / 9.0, 425,991 of 1,000 25 / 24 / 29; both passes of 60,013 rows of 50,021 ids 34 / 28 / 22,
// of 425,991 of 7,921 42 / 35 / 32.  Several / the general sort, ten experts: 4.2 million rows 32 / 83.
//
// Every block reads all blocks' counts, so very many rows go to the general sort: over ten bits from 12.6 million on (1,000
// experts: 12 million rows 256 / 264, 16.8 million 425 / 350; 500: 259 / 348), in several passes from 2.1 million (2 and 4.2
// million rows of 7,921 ids 67 / 93 and 144 / 115, of 65,535 86 / 92 and 184 / 116, of a million 134 / 137 and 259 / 165).
int order_span(int64_t rows, int bits, int passes) {
  if (rows > (int64_t)kOrderBlocks * kOrderRows || (passes > 1 && rows > 1 << 21) || (bits > 9 && rows > 12 << 20)) return 0;
  if (rows <= kOrderRows && rows * (3 + bits) <= 60000) return (int)std::max<int64_t>(rows, 1);
  const int blocks = bits <= 8 ? 256 : 128;
  return (int)std::min<int64_t>(kOrderRows, std::max<int64_t>(262144 / blocks, (rows / blocks + 1023) / 1024 * 1024));
}

// The passes over the bits of an id, none: the general sort.
struct OrderPlan {
  int passes, bits, digit, span;   // bits of an id and of a pass; rows of a block
  int64_t blocks, counts;          // of each pass; ints of its counts
};

OrderPlan order_plan(int64_t rows, int64_t experts) {
  OrderPlan p = {};
  p.bits = id_bits(experts);
  p.passes = experts <= kOrderExperts ? 1 : (p.bits + 9) / 10;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.span = order_span(rows, p.digit, p.passes);
  if (p.span == 0) return OrderPlan{};
  p.blocks = std::max<int64_t>(1, tiles_of(rows, p.span));
  const int64_t groups = p.passes == 1 ? experts + 1 : int64_t(1) << p.digit;
  p.counts = rows <= p.span ? 0 : p.blocks * groups;
  return p;
}

// Ids and row numbers between two passes, both twice where there are more than two; the sorted ids.
int64_t order_bytes(int64_t rows, int64_t experts) {
  const OrderPlan p = order_plan(rows, experts);
  if (p.passes == 0) return ictc_csr_workspace_bytes(rows, experts);
  return 4 * (p.counts + (p.passes == 1 ? 0 : p.passes == 2 ? 3 : 4) * rows);
}

template <Pass P>
void order_pass(const OrderIn& in, int n, int bits, const OrderPlan& p, int* counts, const OrderOut& out, hipStream_t st) {
  if (counts)
    hipLaunchKernelGGL(experts_count_kernel<P>, dim3((unsigned)p.blocks), dim3(1024), 0, st, in, n, p.span, counts);
  hipLaunchKernelGGL(experts_order_kernel<P>, dim3((unsigned)p.blocks), dim3(1024), 0, st, in, n, bits, p.span, counts, out);
}

// The order of rows by id in [0, experts), those of no id last.  small, launch: what the caller says of too small a workspace
// and of a launch that fails.
int order_rows(const int64_t* ids, int64_t rows, int64_t experts, int* perm, int* off, void* workspace, int64_t bytes,
               hipStream_t st, const char* small, const char* launch) {
  const OrderPlan p = order_plan(rows, experts);
  if (p.passes == 0) {   // (what is left for it to refuse is the workspace)
    const int rc = ictc_csr_build(ids, rows, experts, off, perm, workspace, bytes, st);
    return rc == ICTC_ERR_ARGUMENT ? dense_fail(rc, small) : rc;
  }
  const int64_t need = order_bytes(rows, experts);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || bytes < need))
    return dense_fail(ICTC_ERR_ARGUMENT, small);
  const int n = (int)rows;
  int* counts = p.counts ? (int*)workspace : nullptr;
  OrderIn in = {ids, nullptr, nullptr, (int)experts, 0, (int)experts + 1};
  if (p.passes == 1) {
    order_pass<Pass::kOnly>(in, n, p.bits, p, counts, {perm, nullptr, off}, st);
    return dense_status(launch);
  }
  int* half[2][2];   // ids and row numbers that pass 0, 2, .. and 1, 3, .. leave; the last pass: sorted ids
  for (int k = 0; k < 4; ++k) half[k / 2][k % 2] = (int*)workspace + p.counts + k * rows;
  in.groups = 1 << p.digit;
  order_pass<Pass::kFirst>(in, n, p.digit, p, counts, {half[0][1], half[0][0], nullptr}, st);
  for (int k = 1; k < p.passes; ++k) {
    int *const *from = half[(k - 1) % 2], *const *to = half[k % 2];
    const int shift = k * p.digit, bits = std::min(p.digit, p.bits - shift);
    const OrderIn next = {nullptr, from[0], from[1], (int)experts, shift, 1 << bits};
    order_pass<Pass::kLater>(next, n, bits, p, counts, {k + 1 < p.passes ? to[1] : perm, to[0], nullptr}, st);
  }
  const int each = experts >= 8 * rows ? 8 : 64, places = (int)tiles_of(rows + 1, 4 * each);
  const int64_t spans = (experts + 2) / kSpan;
  hipLaunchKernelGGL(order_offsets_kernel, dim3((unsigned)(places + tiles_of(spans, 4))), dim3(256), 0, st,
                     half[(p.passes - 1) % 2][0], n, (uint32_t)experts, each, places, off);
  return dense_status(launch);
}

// Gradients of W ([M, K], g^T x) and of b ([M], the product of g with ones, by the blocks of column tile 0): one tile
// over one range of rows.
template <typename T>
__global__ __launch_bounds__(256, 2) void experts_outer_kernel(const T* __restrict__ gy, int64_t ldg, int M,
                                                            const T* __restrict__ x, int64_t ldx, int K, int experts,
                                                            int ranges, const int* __restrict__ perm,
                                                            const int* __restrict__ off, T* __restrict__ gW,
                                                            T* __restrict__ gb, float* __restrict__ part) {
  using C = Config<T>;
  __shared__ __attribute__((aligned(16))) uint16_t As[C::NP * C::PART];
  __shared__ __attribute__((aligned(16))) uint16_t Bs[C::NP * C::PART];
  const int ct = (K + TILE - 1) / TILE, tiles = ct * ((M + TILE - 1) / TILE);
  const int b = die_order(blockIdx.x, gridDim.x), q = b / tiles;
  const int k0 = b % tiles % ct * TILE, m0 = b % tiles / ct * TILE;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  const int64_t MK = (int64_t)M * K;
  const bool bias = gb != nullptr && k0 == 0 && wave < 2;
  const uint32_t one = sizeof(T) == 4 || __is_same(T, bf16) ? 0x3f803f80u : 0x3c003c00u;
  const int parts = gridDim.x / tiles;
  for (int e = q; e < experts; e += parts)   // experts without rows: zeros, shared out over the blocks of a tile
    if (off[e + 1] == off[e]) zero_tile<T, TILE, 256>(gW + e * MK, gb ? gb + (int64_t)e * M : nullptr, M, K, m0, k0);
  if (q >= ranges) return;
  const Ranges r = find_ranges(off, experts, C::BK, ranges);
  Across<T> xs, gs;
  const int cx = k0 + xs.column(), cg = m0 + gs.column(), r0 = 8 * xs.block();
  Segment s;
  for (int u = q * r.per; find_segment(off, experts, C::BK, r, q, u, s); u += s.steps) {
    alignas(16) int node[8];   // the row numbers of a step are read one step before its rows
    auto name = [&](int row) {
      typedef u32x4 u32x4_int __attribute__((aligned(4)));
      const int* p = perm + s.start + row + r0;
      if (row + r0 + 8 <= s.count) {
        *reinterpret_cast<u32x4*>(node) = *reinterpret_cast<const u32x4_int*>(p);
        *reinterpret_cast<u32x4*>(node + 4) = *reinterpret_cast<const u32x4_int*>(p + 4);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) node[j] = row + r0 + j < s.count ? p[j] : -1;
      }
    };
    auto load = [&]() {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t n = max(node[j], 0);
        xs.v[j] = load_few<T, C::NC>(x + n * ldx + cx, node[j] >= 0 ? K - cx : 0);
        gs.v[j] = load_few<T, C::NC>(gy + n * ldg + cg, node[j] >= 0 ? M - cg : 0);
      }
    };
    v4f acc[C::NI][C::NI], accb[C::NI];
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      accb[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < C::NI; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    name(0);
    load();
    name(C::BK);
    for (int row = 0; row < s.count; row += C::BK) {
      xs.store(As);
      gs.store(Bs);
      __syncthreads();
      if (row + C::BK < s.count) {
        load();
        name(row + 2 * C::BK);
      }
      step<T>(As, Bs, wave >> 1, wave & 1, acc);
      if (bias) {
#pragma unroll
        for (int kk = 0; kk < C::BK / 32; ++kk)
#pragma unroll
          for (int j = 0; j < C::NI; ++j) {
            u32x4 f[C::NP];
            fragment<T>(Bs, TILE / 2 * (wave & 1) + 16 * j + li, 4 * kk + g, f);
#pragma unroll
            for (int p = C::NP - 1; p >= 0; --p) accb[j] = mma<T>(u32x4{one, one, one, one}, f[p], accb[j]);
          }
      }
      __syncthreads();
    }
    float* pw = part + (int64_t)(2 * q + s.slot) * (MK + M);
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int m = m0 + TILE / 2 * (wave & 1) + 16 * j + li;
      if (m >= M) continue;
      if (bias && g == 0) {
        if (s.whole)
          gb[(int64_t)s.expert * M + m] = (T)accb[j][0];
        else
          pw[MK + m] = accb[j][0];
      }
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const int k = k0 + TILE / 2 * (wave >> 1) + 16 * i + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (k + e >= K) continue;
          if (s.whole)
            gW[(int64_t)s.expert * MK + (int64_t)m * K + k + e] = (T)acc[i][j][e];
          else
            pw[(int64_t)m * K + k + e] = acc[i][j][e];
        }
      }
    }
  }
}

// Sums of the ranges' partial gradients in order, for the experts that cross ranges.
template <typename T>
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ part, int64_t MK, int M,
                                                          const int* __restrict__ off, int experts, int rows,
                                                          int ranges, T* __restrict__ gW, T* __restrict__ gb) {
  const int s = blockIdx.y, lane = threadIdx.x & 63;
  const int units = (off[s + 1] - off[s] + rows - 1) / rows;
  if (units < 2) return;
  const Ranges r = find_ranges(off, experts, rows, ranges);
  int first = 0;   // steps of the experts before this one
  for (int e = lane; e < s; e += 64) first += (off[e + 1] - off[e] + rows - 1) / rows;
  first = __builtin_amdgcn_readlane(scan_lanes(first), 63);
  const int q0 = first / r.per, q1 = (first + units - 1) / r.per;
  if (q0 == q1) return;
  const int64_t size = MK + M, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const int n = (int)min<int64_t>(4, size - i);   // this thread's sums
  if (n <= 0) return;
  const bool four = n == 4 && size % 4 == 0;
  auto read = [&](int slot) {
    const float* p = part + (int64_t)slot * size + i;
    if (four) return *reinterpret_cast<const v4f*>(p);
    v4f v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? p[e] : 0.f;
    return v;
  };
  v4f a = read(2 * q0 + (first > q0 * r.per));
#pragma unroll 4
  for (int q = q0 + 1; q <= q1; ++q) a += read(2 * q);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e >= n) continue;
    if (i + e < MK)
      gW[(int64_t)s * MK + i + e] = (T)a[e];
    else if (gb)
      gb[(int64_t)s * M + i + e - MK] = (T)a[e];
  }
}

// Whether `blocks` of experts_few_kernel beat tiles of 64 x 64, from both measured in us (straight and transposed within
// 0.5): tiles of FP32 5.8 / 13.8 / 24 / 45 at 128 / 512 / 1,024 / 2,048 inputs, of 16 bits 3.8 / 5.5 / 7.9 / 12.7, up to
// some thousand rows; the others at those inputs, of one round (256 blocks) FP32 6.2 / 7.5 / 9.6 / 16 and 16 bits 5.2 / 5.5
// / 5.7 / 8.4, of two rounds FP32 7.2 / 10.4 / 15.4 / 26 and 16 bits 5.5 / 6.8 / 8.3 / 13.9.
bool few_is_faster(int dtype, int64_t blocks, int inputs) {
  const double rounds = (double)((blocks + 255) / 256), k = inputs;
  return dtype == ICTC_F32 ? 5.0 + rounds * (1.0 + k / 230.0) < 3.2 + k / 49.0
                           : 4.2 + rounds * k / 450.0 < 3.3 + k / 230.0;
}

// Ranges of the weights' gradient: two blocks for each of the card's 256 units; one in 16 bits where a block would have
// under a thousand rows, unless experts have so few; and no range shorter than a step.  Measured, in us, at 256 / 512
// blocks: bfloat16 131,072 rows of 128 -> 128 20.3 / 22.4, of 512 -> 512 146 / 99, 30,000 of 512 -> 512 over 40 experts 80
// / 62; FP32 30,000 of 512 -> 512 over 40 experts 223 / 136, 16,384 of 512 -> 512 over ten 90 / 82.  FP32 in tiles of 64
// where a block of 128 x 128 would have under 256 rows (2,000 of 336 -> 520 34 against 45 us; 16,384 of 512 -> 512 100
// against 82).
OuterPlan outer_plan(bool direct, int dtype, int64_t n, int M, int K, int experts) {
  OuterPlan p;
  p.direct = direct;
  p.tile = 128;
  int64_t tiles = tiles_of(M, 128) * tiles_of(K, 128);
  const int64_t blocks = dtype == ICTC_F32 || n * tiles >= 512 * 1024 || n < 1024 * (int64_t)experts ? 512 : 256;
  if (!direct || (dtype == ICTC_F32 && n * tiles < 512 * 256)) {
    p.tile = 64;
    tiles = tiles_of(M, 64) * tiles_of(K, 64);
  }
  p.rows = p.tile == 128 && dtype == ICTC_F32 ? 32 : 64;
  const int64_t steps = n / p.rows + std::min<int64_t>(n, experts);   // about as many as there are
  p.ranges = (int)std::max<int64_t>(1, std::min<int64_t>(blocks / tiles, steps));
  // Experts of few rows: a range for each of them, not several one after another (64 rows of ten experts, 128 -> 128
  // FP32: 58 us in one range).
  if (n < 256 * (int64_t)experts)
    p.ranges = (int)std::max<int64_t>(p.ranges, std::min(std::min<int64_t>(n, experts), 2048 / tiles));
  p.sums = p.ranges > 1 && n > p.rows;   // (an expert of one step lies within a range)
  p.fill = (int)std::max<int64_t>(1, std::min<int64_t>(512 / tiles, experts));
  return p;
}

int64_t outer_bytes(const OuterPlan& p, int M, int K) {
  return p.sums ? 2 * (int64_t)p.ranges * ((int64_t)M * K + M) * (int64_t)sizeof(float) : 0;
}

const char* bad_sizes(int dtype, int64_t rows, int64_t inputs, int64_t outputs, int experts) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "expert_linear: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (rows < 0 || rows >= (int64_t(1) << 31) - 2) return "expert_linear: up to 2^31 - 3 rows";
  if (inputs < 1 || outputs < 1 || inputs > 65536 || outputs > 65536) return "expert_linear: 1 to 65536 inputs and outputs";
  if (experts < 1 || experts > 65535) return "expert_linear: 1 to 65535 experts";
  return nullptr;
}

template <typename T>
void launch_rows(const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias, int N, int experts,
                 const int* perm, const int* off, int transpose, void* out, hipStream_t st) {
  const dim3 grid((unsigned)(most_runs(rows, experts, 64) * tiles_of(N, 64)));
  if (transpose)
    hipLaunchKernelGGL((experts_rows_kernel<T, true>), grid, dim3(256), 0, st, (const T*)x, ldx, K, (const T*)W,
                       (const T*)bias, N, experts, perm, off, (T*)out);
  else
    hipLaunchKernelGGL((experts_rows_kernel<T, false>), grid, dim3(256), 0, st, (const T*)x, ldx, K, (const T*)W,
                       (const T*)bias, N, experts, perm, off, (T*)out);
}

template <typename T>
void launch_few(const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias, int N, int experts,
                const int* perm, const int* off, int transpose, void* out, hipStream_t st) {
  const dim3 grid((unsigned)(most_runs(rows, experts, kFewRows) * tiles_of(N, kFewColumns))), block(kFewWaves * 64);
  if (transpose)
    hipLaunchKernelGGL((experts_few_kernel<T, true>), grid, block, 0, st, (const T*)x, ldx, K, (const T*)W,
                       (const T*)bias, N, experts, perm, off, (T*)out);
  else
    hipLaunchKernelGGL((experts_few_kernel<T, false>), grid, block, 0, st, (const T*)x, ldx, K, (const T*)W,
                       (const T*)bias, N, experts, perm, off, (T*)out);
}

template <typename T>
void launch_outer(const OuterPlan& plan, const void* gy, int64_t ldg, int M, const void* x, int64_t ldx, int K,
                  int experts, const int* perm, const int* off, void* gW, void* gb, float* part, hipStream_t st) {
  const dim3 grid((unsigned)(std::max(plan.ranges, plan.fill) * tiles_of(M, plan.tile) * tiles_of(K, plan.tile)));
  hipLaunchKernelGGL(experts_outer_kernel<T>, grid, dim3(256), 0, st, (const T*)gy, ldg, M,
                     (const T*)x, ldx, K, experts, plan.ranges, perm, off, (T*)gW, (T*)gb, part);
}

template <typename T>
void launch_sum(const OuterPlan& plan, int M, int K, int experts, const int* off, void* gW, void* gb, const float* part,
                hipStream_t st) {
  const int64_t MK = (int64_t)M * K;
  hipLaunchKernelGGL(experts_sum_kernel<T>, dim3((unsigned)((MK + M + 1023) / 1024), (unsigned)experts), dim3(256), 0, st,
                     part, MK, M, off, experts, plan.rows, plan.ranges, (T*)gW, (T*)gb);
}

// The weights' gradient of rows x, or of codes; the caller has looked at these.
int run_outer(int dtype, const void* grad, int64_t ldg, const void* x, int64_t ldx, const int8_t* codes, const float* scales,
              int64_t rows, int inputs, int outputs, int experts, const int* perm, const int* offsets, void* dweight,
              void* dbias, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  if (ldg < outputs && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: row pitch below the row");
  if (!offsets || !dweight || (rows > 0 && (!grad || !perm)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: null operand");
  const OuterPlan plan = outer_plan(rows > 0 && experts_direct_outer_fits(dtype, outputs, inputs),
                                    dtype, rows, outputs, inputs, experts);
  if (outer_bytes(plan, outputs, inputs) > 0 &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
       workspace_bytes < ictc_expert_outer_workspace_bytes(dtype, rows, inputs, outputs, experts)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: workspace smaller than ictc_expert_outer_workspace_bytes");
  float* part = (float*)workspace;
  if (codes)
    experts_codes_outer(dtype, plan, grad, ldg, outputs, codes, scales, inputs, experts, perm, offsets, dweight, dbias, part,
                        st);
  else if (plan.direct)
    experts_direct_outer(dtype, plan, grad, ldg, outputs, x, ldx, inputs, experts, perm, offsets, dweight, dbias, part,
                         st);
  else if (dtype == ICTC_F32)
    launch_outer<float>(plan, grad, ldg, outputs, x, ldx, inputs, experts, perm, offsets, dweight, dbias, part, st);
  else if (dtype == ICTC_BF16)
    launch_outer<bf16>(plan, grad, ldg, outputs, x, ldx, inputs, experts, perm, offsets, dweight, dbias, part, st);
  else
    launch_outer<f16>(plan, grad, ldg, outputs, x, ldx, inputs, experts, perm, offsets, dweight, dbias, part, st);
  if (plan.sums) {
    if (dtype == ICTC_F32)
      launch_sum<float>(plan, outputs, inputs, experts, offsets, dweight, dbias, part, st);
    else if (dtype == ICTC_BF16)
      launch_sum<bf16>(plan, outputs, inputs, experts, offsets, dweight, dbias, part, st);
    else
      launch_sum<f16>(plan, outputs, inputs, experts, offsets, dweight, dbias, part, st);
  }
  return dense_status("expert_outer launch");
}

}  // namespace

extern "C" {

int64_t ictc_expert_order_workspace_bytes(int64_t rows, int experts) {
  if (bad_sizes(ICTC_F32, rows, 1, 1, experts)) return -1;
  return order_bytes(rows, experts);
}

int ictc_expert_order(const int64_t* ids, int64_t rows, int experts, int32_t* perm, int32_t* offsets, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(ICTC_F32, rows, 1, 1, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (!offsets || (rows > 0 && (!ids || !perm))) return dense_fail(ICTC_ERR_ARGUMENT, "expert_order: null operand");
  return order_rows(ids, rows, experts, perm, offsets, workspace, workspace_bytes, (hipStream_t)stream,
                    "expert_order: workspace smaller than ictc_expert_order_workspace_bytes", "expert_order launch");
}

int64_t ictc_rows_by_id_workspace_bytes(int64_t rows, int64_t entries) {
  if (rows < 0 || entries < 1 || std::max(rows, entries) >= (int64_t(1) << 31) - 2) return -1;
  return order_bytes(rows, entries);
}

int ictc_rows_by_id(const int64_t* ids, int64_t rows, int64_t entries, int32_t* perm, int32_t* offsets, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  if (ictc_rows_by_id_workspace_bytes(rows, entries) < 0)
    return dense_fail(ICTC_ERR_ARGUMENT, "rows_by_id: up to 2^31 - 3 rows and entries");
  if (!offsets || (rows > 0 && (!ids || !perm))) return dense_fail(ICTC_ERR_ARGUMENT, "rows_by_id: null operand");
  return order_rows(ids, rows, entries, perm, offsets, workspace, workspace_bytes, (hipStream_t)stream,
                    "rows_by_id: workspace smaller than ictc_rows_by_id_workspace_bytes", "rows_by_id launch");
}

int ictc_expert_linear(int dtype, const void* x, int64_t ldx, int64_t rows, int inputs, const void* weight,
                       const void* bias, int outputs, int experts, const int32_t* perm, const int32_t* offsets,
                       int transpose, void* out, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, inputs, outputs, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (rows == 0) return ICTC_OK;
  if (ldx < inputs && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "expert_linear: row pitch below the inputs");
  if (!x || !weight || !perm || !offsets || !out) return dense_fail(ICTC_ERR_ARGUMENT, "expert_linear: null operand");
  const bool direct = experts_direct_rows_fit(dtype, inputs, outputs, transpose != 0);
  const bool wide = outputs > 64 && experts_tiles(rows, outputs, experts) >= 1024 && direct;
  const int tile = wide ? 128 : 64;   // the least that is taken
  if (most_runs(rows, experts, tile) * tiles_of(outputs, tile) >= (int64_t(1) << 24))
    return dense_fail(ICTC_ERR_UNSUPPORTED, "expert_linear: more than 2^24 tiles");
  hipStream_t st = (hipStream_t)stream;
  if (few_is_faster(dtype, most_runs(rows, experts, kFewRows) * tiles_of(outputs, kFewColumns), inputs)) {
    if (dtype == ICTC_F32)
      launch_few<float>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
    else if (dtype == ICTC_BF16)
      launch_few<bf16>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
    else
      launch_few<f16>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
    return dense_status("expert_linear launch");
  }
  if (direct)
    experts_direct_rows(dtype, x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose != 0, out,
                        st);
  else if (dtype == ICTC_F32)
    launch_rows<float>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
  else if (dtype == ICTC_BF16)
    launch_rows<bf16>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
  else
    launch_rows<f16>(x, ldx, rows, inputs, weight, bias, outputs, experts, perm, offsets, transpose, out, st);
  return dense_status("expert_linear launch");
}

int64_t ictc_expert_outer_workspace_bytes(int dtype, int64_t rows, int inputs, int outputs, int experts) {
  if (bad_sizes(dtype, rows, inputs, outputs, experts)) return -1;
  return std::max(outer_bytes(outer_plan(false, dtype, rows, outputs, inputs, experts), outputs, inputs),
                  outer_bytes(outer_plan(true, dtype, rows, outputs, inputs, experts), outputs, inputs));
}

int ictc_expert_outer(int dtype, const void* grad, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int inputs,
                      int outputs, int experts, const int32_t* perm, const int32_t* offsets, void* dweight,
                      void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, inputs, outputs, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (ldx < inputs && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: row pitch below the row");
  if (rows > 0 && !x) return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: null operand");
  return run_outer(dtype, grad, ldg, x, ldx, nullptr, nullptr, rows, inputs, outputs, experts, perm, offsets, dweight, dbias,
                   workspace, workspace_bytes, (hipStream_t)stream);
}

int ictc_expert_outer_takes_codes(int dtype, const void* grad, int64_t ldg, int64_t rows, int inputs, int outputs) {
  return !bad_sizes(dtype, rows, inputs, outputs, 1) && rows > 0 && experts_direct_outer_fits(dtype, outputs, inputs) &&
         experts_codes_outer_fits(dtype, grad, ldg, outputs, inputs);
}

int ictc_expert_outer_codes(int dtype, const void* grad, int64_t ldg, const int8_t* codes, const float* scales, int64_t rows,
                            int inputs, int outputs, int experts, const int32_t* perm, const int32_t* offsets,
                            void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, inputs, outputs, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (!codes || !scales) return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: null operand");
  if (!ictc_expert_outer_takes_codes(dtype, grad, ldg, rows, inputs, outputs))
    return dense_fail(ICTC_ERR_UNSUPPORTED, "expert_outer: codes need rows, and whole aligned 16-byte chunks of them");
  return run_outer(dtype, grad, ldg, nullptr, inputs, codes, scales, rows, inputs, outputs, experts, perm, offsets, dweight,
                   dbias, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
