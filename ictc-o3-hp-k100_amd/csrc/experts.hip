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
// ([blocks, experts + 1], the kernel below), what lies before its own.
constexpr int kOrderExperts = 1023, kOrderWaves = 16, kOrderAtOnce = 16, kOrderBlocks = 256;
constexpr int kOrderRows = kOrderWaves * kOrderAtOnce * 64;

__global__ __launch_bounds__(1024) void experts_count_kernel(const int64_t* __restrict__ ids, int n, int experts,
                                                             int span, int* __restrict__ counts) {
  __shared__ int count[kOrderExperts + 1];
  if ((int)threadIdx.x <= experts) count[threadIdx.x] = 0;
  __syncthreads();
  const int begin = blockIdx.x * span, end = min(n, begin + span);
  for (int r0 = begin + (int)threadIdx.x; r0 < end; r0 += 4096) {
    int64_t id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = r0 + i * 1024 < end ? ids[r0 + i * 1024] : -1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r0 + i * 1024 < end) atomicAdd(&count[(uint64_t)id[i] < (uint64_t)experts ? (int)id[i] : experts], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x <= experts) counts[blockIdx.x * (experts + 1) + threadIdx.x] = count[threadIdx.x];
}

__global__ __launch_bounds__(1024) void experts_order_kernel(const int64_t* __restrict__ ids, int n, int experts,
                                                             int bits, int span, const int* __restrict__ counts,
                                                             int* __restrict__ off, int* __restrict__ perm) {
  __shared__ int count[kOrderWaves][kOrderExperts + 1];
  __shared__ int wave_total[kOrderWaves];
  const int lane = threadIdx.x & 63, groups = experts + 1, group = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int i = threadIdx.x; i < kOrderWaves * groups; i += 1024) count[i / groups][i % groups] = 0;
  int total = 0, before = 0;   // of this group: all rows, and those of the blocks before
  if (counts && group < groups) {
#pragma unroll 8
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int c = counts[b * groups + group];
      total += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
  }
  __syncthreads();
  const int first = blockIdx.x * span, rows = min(span, n - first);
  const int per = ((rows + kOrderWaves - 1) / kOrderWaves + 63) / 64 * 64;
  const int begin = first + wave * per, end = min(first + rows, begin + per);
  int* mine = count[wave];
  uint32_t place[kOrderAtOnce];   // expert | lanes below << 10 | lanes << 16
  int64_t id[kOrderAtOnce];
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) {
    const int row = begin + i * 64 + lane;
    id[i] = row < end ? ids[row] : -1;
  }
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) {
    const int r0 = begin + i * 64;
    if (r0 >= end) break;
    const uint32_t key = (uint64_t)id[i] < (uint64_t)experts ? (uint32_t)id[i] : (uint32_t)experts;
    const uint64_t in = __ballot(r0 + lane < end);
    uint32_t lo = (uint32_t)in, hi = (uint32_t)(in >> 32);   // the lanes whose row has this lane's expert
    int x = (int)(key << (32 - bits));
    for (int b = 0; b < bits; ++b, x <<= 1) {
      const uint64_t set = __ballot(x < 0);
      lo &= ~((uint32_t)set ^ (uint32_t)(x >> 31));
      hi &= ~((uint32_t)(set >> 32) ^ (uint32_t)(x >> 31));
    }
    const uint64_t m = (uint64_t)hi << 32 | lo;
    const int below = __popcll(m & ((uint64_t(1) << lane) - 1)), lanes = __popcll(m);
    place[i] = key | below << 10 | lanes << 16;
    if (r0 + lane < end && below == 0) atomicAdd(&mine[key], lanes);
  }
  __syncthreads();
  int here = 0;
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
    if (blockIdx.x == 0) off[group] = start;
    if (blockIdx.x == 0 && group == experts) off[groups] = n;
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) count[w][group] += start + before;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOrderAtOnce; ++i) {
    const int r0 = begin + i * 64;
    if (r0 >= end) break;
    const bool in = r0 + lane < end;
    const int key = place[i] & 1023u, below = place[i] >> 10 & 63u, lanes = place[i] >> 16;
    if (in) perm[mine[key] + below] = r0 + lane;
    wave_meet();
    if (in && below == 0) atomicAdd(&mine[key], lanes);   // (before the next rows' reads: LDS keeps a wave's order)
    wave_meet();
  }
}

int64_t tiles_of(int64_t n, int tile) { return (n + tile - 1) / tile; }

int id_bits(int experts) {
  int bits = 1;
  while (experts >> bits) ++bits;
  return bits;
}

// Rows of a block: all of few rows; 4,096; more once those would be more than 64 blocks; and zero: the general sort.
// Measured in us, one block / several: ten experts 500 rows 4.6 / 8.0, 8,192 8.0 / 8.5, 16,384 12.9 / 9.0; 89 experts 6,000
// rows 8.2 / 8.7, 16,384 16.4 / 10.1.  Several / the general sort, ten experts: 30,011 rows 8.8 / 10.8, 262,145 11.8 / 106,
// 4.2 million 32 / 83.
int order_span(int64_t rows, int experts) {
  if (experts > kOrderExperts || rows > (int64_t)kOrderBlocks * kOrderRows) return 0;
  if (rows <= kOrderRows && rows * (3 + id_bits(experts)) <= 60000) return (int)std::max<int64_t>(rows, 1);
  return (int)std::min<int64_t>(kOrderRows, std::max<int64_t>(4096, (rows / 64 + 1023) / 1024 * 1024));
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

}  // namespace

extern "C" {

int64_t ictc_expert_order_workspace_bytes(int64_t rows, int experts) {
  if (bad_sizes(ICTC_F32, rows, 1, 1, experts)) return -1;
  const int span = order_span(rows, experts);
  if (span == 0) return ictc_csr_workspace_bytes(rows, experts);
  return rows <= span ? 0 : tiles_of(rows, span) * (experts + 1) * (int64_t)sizeof(int);
}

int ictc_expert_order(const int64_t* ids, int64_t rows, int experts, int32_t* perm, int32_t* offsets, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(ICTC_F32, rows, 1, 1, experts)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (!offsets || (rows > 0 && (!ids || !perm))) return dense_fail(ICTC_ERR_ARGUMENT, "expert_order: null operand");
  const int span = order_span(rows, experts);
  if (span == 0) return ictc_csr_build(ids, rows, experts, offsets, perm, workspace, workspace_bytes, stream);
  const bool several = rows > span;
  if (several && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
                  workspace_bytes < ictc_expert_order_workspace_bytes(rows, experts)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_order: workspace smaller than ictc_expert_order_workspace_bytes");
  const dim3 blocks((unsigned)std::max<int64_t>(1, tiles_of(rows, span)));
  int* counts = several ? (int*)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (several)
    hipLaunchKernelGGL(experts_count_kernel, blocks, dim3(1024), 0, st, ids, (int)rows, experts, span, counts);
  hipLaunchKernelGGL(experts_order_kernel, blocks, dim3(1024), 0, st, ids, (int)rows, experts, id_bits(experts), span,
                     counts, offsets, perm);
  return dense_status("expert_order launch");
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
  if ((ldx < inputs || ldg < outputs) && rows > 1)
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: row pitch below the row");
  if (!offsets || !dweight || (rows > 0 && (!grad || !x || !perm)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: null operand");
  const OuterPlan plan = outer_plan(rows > 0 && experts_direct_outer_fits(dtype, outputs, inputs),
                                    dtype, rows, outputs, inputs, experts);
  if (outer_bytes(plan, outputs, inputs) > 0 &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
       workspace_bytes < ictc_expert_outer_workspace_bytes(dtype, rows, inputs, outputs, experts)))
    return dense_fail(ICTC_ERR_ARGUMENT, "expert_outer: workspace smaller than ictc_expert_outer_workspace_bytes");
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  if (plan.direct)
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

}  // extern "C"
