// The expert linears' products over rows of 16 bytes or more: where all rows begin at multiples of 16 bytes the tiles go
// from memory to LDS without passing through registers (global_load_lds, 16 bytes a lane), one step ahead of the matrix
// instructions; else through registers (load_chunk_of), 16 bits then at 0.6 to 0.75 of the speed.
//
// A tile of an operand whose rows run along the reduction index is kept [row][step]; one whose memory runs along the
// rows is kept as it lies, [step][row], and its fragments are transposed as they are read: 16 bits by
// ds_read_b64_tr_b16 (sixteen lanes read four rows of sixteen values and receive four of a column each), FP32 by eight
// reads of one value.  A load writes lane l's 16 bytes at base + 16 l, so the exchange of chunks that spreads the
// fragment reads over the banks is made by the lanes' source addresses.  Chunks past the end of the reduction come from
// a block of zeros; rows and columns past the tile's end repeat valid ones and are not stored.  FP32 values are split
// after they are read from LDS, by each of the two waves that use them: 3.5 vector instructions a value, which cost less
// than the 6 bytes that split values would take in LDS (30,000 rows of 256 -> 256, split on their way there: rows 43
// against 38 us, weights' gradient 77 against 59).
//
// Tiles of 128 x 128 by four waves of 64 x 64, or of 256 columns by eight.  For the rows' products in 16 bits a step has 32
// reduction indices, so that sixteen waves share a compute unit and one block's first loads and last stores run under
// another's products: at 131,072 rows of 512 -> 1,024 bfloat16 in tiles of 128 x 128 this measured 211 us and its adjoint
// 182 us (1,024 -> 512).  256 x 256 tiles, one block of eight waves and steps of 64, took 204 / 188 us there and lost a
// factor of two at 128 -> 128 (41 against 17 us).  For the weights' gradient a step has 64 rows and two blocks share a
// unit.
//
// At 131,072 rows of 512 -> 512 over ten experts, rows / adjoint / weights' gradient in us: bfloat16 102 / 97 / 116 (674,
// 708 and 592 TFLOP/s; a library product of these sizes with one matrix 83 / 91 / 363), FP32 394 / 401 / 441 (174, 171 and
// 156 TFLOP/s, six times that on the matrix cores; 497 / 505 / 640), bound by the matrix cores' rate at the clock that they
// leave; 511 -> 511 FP16, through registers, 149 / 177 / 185.
#include <algorithm>
#include <type_traits>

#include "experts.h"

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// How an element is kept in LDS, and the parts of it that the matrix instructions take.
template <typename T>
using Word = std::conditional_t<sizeof(T) == 4, float, uint16_t>;
template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;

__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

__device__ __forceinline__ void to_lds(const void* p, void* lds) {
  __builtin_amdgcn_global_load_lds((global_void*)p, (lds_void*)lds, 16, 0, 0);
}

// Rows that do not begin at multiples of 16 bytes go through registers, to the same places.  The chunk at p has `n`
// elements of its row left: of a chunk that passes the row's end the last 16 bytes of the row are read (a row has a chunk
// or more) and moved down, and what has none left reads zeros; so no load passes a row's end.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk_of(const T* p, int n) {
  const T* at = n <= 0 ? reinterpret_cast<const T*>(kZeros) : p - max(0, kChunk<T> - n);
  return *reinterpret_cast<const u32x4_any*>(at);
}
template <typename T>
__device__ __forceinline__ u32x4 move_chunk(u32x4 raw, int n) {
  if (n > 0 && n < kChunk<T>) {
    const int s = 8 * (int)sizeof(T) * (kChunk<T> - n);
    uint64_t lo = (uint64_t)raw[1] << 32 | raw[0], hi = (uint64_t)raw[3] << 32 | raw[2];
    lo = s >= 64 ? hi >> (s - 64) : lo >> s | hi << (64 - s);
    hi = s >= 64 ? 0 : hi >> s;
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  return raw;
}

// Chunk exchange of row `r` of an operand kept [S][R].  16 bits: pairs of chunks (16 columns, R / 16 of them); FP32: fours
// of chunks (16 columns too).
template <typename T, int R>
__device__ __forceinline__ int across_swap(int r) {
  if (sizeof(T) == 4) return (r >> 3 & 3) << 2;
  return (((r & 3) | ((r >> 3) & 1) << 2) & (R / 16 - 1)) << 1;
}

// Loads of an operand of R rows by a wave: blocks of 1 KB of a step of S reduction indices over WAVES waves.
template <typename T, int R, int S, int WAVES>
constexpr int kLoads = R * S / (64 * kChunk<T>) / WAVES;

// Chunk exchange of row `r` of an operand kept [R][S], eight chunks a row or four.
template <typename T, int S>
__device__ __forceinline__ int row_swap(int r) { return S == 8 * kChunk<T> ? r & 7 : (r >> 2) & 3; }

// 16 bits, kept [R][S]: where a lane's part of a fragment lies, 16 x 32 values at rows r0 .. r0 + 15 of an operand,
// reduction indices 32 kk ..., r0 a multiple of 16: + r0 * S.
template <typename T, int S>
__device__ __forceinline__ int straight_at(int kk) {
  const int lane = threadIdx.x & 63, li = lane & 15;
  return li * S + (((4 * kk + (lane >> 4)) ^ row_swap<T, S>(li)) * 8);
}

// 16 bits, kept [S][R]: the lane's row of the tile and its exchange; ^ the first column, a multiple of 16 below R.
template <typename T, int R>
__device__ __forceinline__ int across_at() {
  const int lane = threadIdx.x & 63, i = lane & 15, k = 8 * (lane >> 4) + (i >> 2);
  return k * R + across_swap<T, R>(k) * 8 + (i & 3) * 4;
}

template <int R>
__device__ __forceinline__ u32x4 across_fragment(const uint16_t* p) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * R));
  const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
  return u32x4{l[0], l[1], h[0], h[1]};
}

// N fragments of an operand of R rows from row 16 N w + 16 first on.
template <typename T, bool ACROSS, int R, int S, int N, int OF>
__device__ __forceinline__ void fragments(const Word<T>* lds, int kk, int w, int first, u32x4 (&f)[N][kParts<T>]) {
  if constexpr (sizeof(T) == 4) {
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      alignas(16) float v[8];
      const int r0 = (w * OF + first + i) * 16;
      if (ACROSS) {
        const float* p = lds + (32 * kk + 8 * g) * R + (r0 ^ (g * 16)) + li;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[e * R];
      } else {
        const float* p = lds + (r0 + li) * S;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<u32x4*>(v + 4 * h) =
              *reinterpret_cast<const u32x4*>(p + (((8 * kk + 2 * g + h) ^ row_swap<T, S>(li)) * 4));
      }
      const Split s = split8_pairs(v);
      f[i][0] = __builtin_bit_cast(u32x4, s.hi);
      f[i][1] = __builtin_bit_cast(u32x4, s.mid);
      f[i][2] = __builtin_bit_cast(u32x4, s.lo);
    }
  } else if constexpr (ACROSS) {
    int at = across_at<T, R>() ^ (w * OF * 16);
    asm volatile("" : "+v"(at));   // (keeps one address in a register, not one for each fragment over the whole loop)
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][0] = across_fragment<R>(lds + (at ^ ((first + i) * 16)) + kk * 32 * R);
  } else {
    const uint16_t* p = lds + straight_at<T, S>(kk) + (w * OF + first) * 16 * S;
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][0] = *reinterpret_cast<const u32x4*>(p + i * 16 * S);
  }
}

// ones: the sums of operand B's rows over the step are added to accb too.  16 bits: all fragments of 32 reduction indices,
// then their products; FP32: operand B's one after another, which are split while the products before them run.
template <typename T, bool ACROSS_A, bool ACROSS_B, int TA, int TB, int S, int GA, int GB, bool SUMS>
__device__ __forceinline__ void direct_step(const Word<T>* A, const Word<T>* B, int wa, int wb,
                                            v4f (&acc)[TA / GA / 16][TB / GB / 16], bool ones,
                                            v4f (&accb)[SUMS ? TB / GB / 16 : 1]) {
  constexpr int NA = TA / GA / 16, NB = TB / GB / 16, NP = kParts<T>, AT_ONCE = sizeof(T) == 4 ? 1 : NB;
#pragma unroll
  for (int kk = 0; kk < S / 32; ++kk) {
    u32x4 a[NA][NP], b[AT_ONCE][NP];
    if (sizeof(T) == 2) fragments<T, ACROSS_B, TB, S, AT_ONCE, NB>(B, kk, wb, 0, b);
    fragments<T, ACROSS_A, TA, S, NA, NA>(A, kk, wa, 0, a);
#pragma unroll
    for (int j0 = 0; j0 < NB; j0 += AT_ONCE) {
      if (sizeof(T) == 4) fragments<T, ACROSS_B, TB, S, AT_ONCE, NB>(B, kk, wb, j0, b);
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) acc[i][j0 + j] = product<T>(a[i], b[j], acc[i][j0 + j]);
      if (SUMS && ones) {
        constexpr uint32_t one = __is_same(T, f16) ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) accb[j0 + j] = mma<T>(u32x4{one, one, one, one}, b[j][p], accb[j0 + j]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // (the next half's fragments would not fit the registers beside these)
  }
}

// All waves are here, with their reads of LDS behind them and, LOADS, this wave's loads in LDS.  (The wait is the
// builtin's: the compiler then knows of it and adds none of its own before the fragment reads.)
template <bool LOADS>
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(LOADS ? 0x0070 : 0xc07f);   // vmcnt(0) lgkmcnt(0); lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// out[perm[r]] = M x[perm[r]] + b, M = W[e] [N, K] or, TRANS, the transpose of W[e] [K, N].  Operand A is the
// weights (TA output columns), operand B the rows (TB of them).
template <typename T, bool ALIGNED, bool TRANS, int TA, int TB, int S, int GA, int GB>
__global__ __launch_bounds__(GA * GB * 64, sizeof(T) == 2 && S == 32 ? 4 : 2) void experts_direct_kernel(
    const T* __restrict__ x, int64_t ldx, int K, const T* __restrict__ W, const T* __restrict__ bias, int N,
    int experts, const int* __restrict__ perm, const int* __restrict__ off, T* __restrict__ out) {
  constexpr int WAVES = GA * GB, LA = kLoads<T, TA, S, WAVES>, LB = kLoads<T, TB, S, WAVES>;
  constexpr int NA = TA / GA / 16, NB = TB / GB / 16, V = kChunk<T>, KB = 64 * V;   // (KB: elements of a load)
  __shared__ __attribute__((aligned(16))) Word<T> A0[TA * S], A1[TA * S], B0[TB * S], B1[TB * S];
  __shared__ __attribute__((aligned(16))) uint16_t stage[sizeof(T) == 2 ? WAVES * NA * 256 : 8];
  const int columns = (N + TA - 1) / TA;
  const int blk = die_order(blockIdx.x, gridDim.x);
  Run run;
  if (!find_run(off, experts + 1, TB, blk / columns, run)) return;
  const int n0 = blk % columns * TA;
  if (run.group == experts) {   // ids outside [0, experts): zero rows
    const int width = min(TA, N - n0);
    for (int i = threadIdx.x; i < run.count * TA; i += WAVES * 64)
      if (i % TA < width) out[(int64_t)perm[run.start + i / TA] * N + n0 + i % TA] = (T)0.f;
    return;
  }
  const T* w = W + (int64_t)run.group * N * K;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wa = wave / GB, wb = wave % GB;
  // the lanes' source addresses at step 0, and the reduction index that each stands at
  const T *pa[LA], *pb[LB];
  int ka[LA], na[LA];   // (na: TRANS, the weights' columns from there on)
  constexpr int RC = S / V, RR = 64 / RC;   // chunks of a row kept [R][S], rows of a load
  const int kb = ((lane % RC) ^ row_swap<T, S>(lane / RC)) * V;
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int block = wave * LA + i;
    if (TRANS) {
      constexpr int CH = TA / V;   // chunks of a row kept [S][R]
      const int r = block * (64 / CH) + lane / CH, c = (lane % CH) ^ across_swap<T, TA>(r);
      ka[i] = r;
      na[i] = N - n0 - V * c;
      pa[i] = w + (int64_t)r * N + (na[i] > 0 ? n0 + V * c : n0);
    } else {
      const int r = block * RR + lane / RC;
      ka[i] = kb;
      pa[i] = w + (int64_t)(n0 + r < N ? n0 + r : n0) * K + kb;
    }
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int r = (wave * LB + i) * RR + lane / RC;
    pb[i] = x + (int64_t)perm[run.start + (r < run.count ? r : 0)] * ldx + kb;
  }
  u32x4 ra[LA], rb[LB];   // (not ALIGNED)
  auto load = [&](Word<T>* A, Word<T>* B, int k0) {
    const int left = K - k0;   // reduction indices from here on
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const T* p = pa[i] + (TRANS ? (int64_t)k0 * N : (int64_t)k0);
      if (ALIGNED)
        to_lds(ka[i] < left ? (const void*)p : (const void*)kZeros, A + (wave * LA + i) * KB);
      else
        ra[i] = load_chunk_of(p, TRANS ? (ka[i] < left ? na[i] : 0) : left - kb);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      if (ALIGNED)
        to_lds(kb < left ? (const void*)(pb[i] + k0) : (const void*)kZeros, B + (wave * LB + i) * KB);
      else
        rb[i] = load_chunk_of(pb[i] + k0, left - kb);
    }
  };
  auto put = [&](Word<T>* A, Word<T>* B, int k0) {   // not ALIGNED: what load read
    const int left = K - k0;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      *reinterpret_cast<u32x4*>(A + (wave * LA + i) * KB + lane * V) = move_chunk<T>(ra[i], TRANS ? na[i] : left - kb);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      *reinterpret_cast<u32x4*>(B + (wave * LB + i) * KB + lane * V) = move_chunk<T>(rb[i], left - kb);
  };
  v4f acc[NA][NB], none[1];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  load(A0, B0, 0);
  if (!ALIGNED) put(A0, B0, 0);
  for (int k0 = 0; k0 < K; k0 += 2 * S) {   // the two buffers are separate objects: a step's reads wait for no load
    meet<ALIGNED>();
    if (k0 + S < K) load(A1, B1, k0 + S);
    direct_step<T, TRANS, false, TA, TB, S, GA, GB, false>(A0, B0, wa, wb, acc, false, none);
    if (k0 + S < K) {
      if (!ALIGNED) put(A1, B1, k0 + S);
      meet<ALIGNED>();
      if (k0 + 2 * S < K) load(A0, B0, k0 + 2 * S);
      direct_step<T, TRANS, false, TA, TB, S, GA, GB, false>(A1, B1, wa, wb, acc, false, none);
      if (!ALIGNED && k0 + 2 * S < K) put(A0, B0, k0 + 2 * S);
    }
  }
  const int c0 = n0 + wa * NA * 16;
  T bv[NA][4];   // all of the bias and row numbers are asked for before the first is needed
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const int c = c0 + 16 * i + 4 * g;
    const T* bp = bias + (int64_t)run.group * N + c;
    if (bias && c + 4 <= N) {
      __builtin_memcpy(bv[i], bp, sizeof(bv[i]));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) bv[i][q] = bias && c + q < N ? bp[q] : (T)0.f;
    }
  }
  if constexpr (sizeof(T) == 4) {   // a lane's four columns of a row are a store
    int at[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int r = (wb * NB + j) * 16 + li;
      at[j] = r < run.count ? perm[run.start + r] : -1;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (at[j] < 0) continue;
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int c = c0 + 16 * i + 4 * g;
        T* o = out + (int64_t)at[j] * N + c;
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = acc[i][j][q] + bv[i][q];
        store_chunk(o, N - c, v);
      }
    }
  } else {
    // 16 bits: the results go through LDS, 16 rows of this wave's columns at a time, so that a store writes runs of them.
    constexpr int CH = NA * 2, PER = 64 / CH;   // chunks of a row here; rows of a store
    // An output larger than the caches is not kept in them (131,072 x 1,024: 233 us without, 216 us with).
    const bool stream = (int64_t)off[experts + 1] * N * (int64_t)sizeof(T) > (int64_t(1) << 27);
    const int cc = c0 + lane % CH * 8;
    int at[NB][16 / PER];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int h = 0; h < 16 / PER; ++h) {
        const int r = (wb * NB + j) * 16 + h * PER + lane / CH;
        at[j][h] = r < run.count ? perm[run.start + r] : -1;
      }
    uint16_t* st = stage + wave * NA * 256;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        T v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = (T)(acc[i][j][q] + (float)bv[i][q]);
        *reinterpret_cast<u32x2*>(st + (li * CH + ((2 * i + (g >> 1)) ^ (li % CH))) * 8 + (g & 1) * 4) =
            *reinterpret_cast<const u32x2*>(v);
      }
      wave_meet();
#pragma unroll
      for (int h = 0; h < 16 / PER; ++h) {
        const int r = h * PER + lane / CH;
        Chunk<T> v;
        v.raw = *reinterpret_cast<const u32x4*>(st + (r * CH + ((lane % CH) ^ (r % CH))) * 8);
        if (at[j][h] < 0) continue;
        T* o = out + (int64_t)at[j][h] * N + cc;
        if (cc + 8 <= N) {
          if (stream)
            __builtin_nontemporal_store(v.raw, reinterpret_cast<u32x4_any*>(o));
          else
            *reinterpret_cast<u32x4_any*>(o) = v.raw;
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (cc + q < N) o[q] = v.e[q];
        }
      }
      wave_meet();
    }
  }
}

template <typename T, bool ALIGNED, bool TRANS, int TA, int TB, int S>
void launch_direct(const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias, int N, int experts,
                   const int* perm, const int* off, void* out, hipStream_t st) {
  constexpr int GA = TA == 256 ? 4 : 2;
  const int64_t blocks = most_runs(rows, experts, TB) * ((N + TA - 1) / TA);
  hipLaunchKernelGGL((experts_direct_kernel<T, ALIGNED, TRANS, TA, TB, S, GA, 2>), dim3((unsigned)blocks),
                     dim3(GA * 128), 0, st, (const T*)x, ldx, K, (const T*)W, (const T*)bias, N, experts, perm, off,
                     (T*)out);
}

template <typename T, bool ALIGNED, bool TRANS>
void direct_rows(const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias, int N, int experts,
                 const int* perm, const int* off, void* out, hipStream_t st) {
  // Tiles of 64 x 64 where those of 128 x 128 are fewer than the card's units or half empty: 8,192 rows of 128 -> 128 4.4
  // against 6.2 us, 131,072 of 64 -> 64 11 against 15; 16,384 of 256 -> 256 10.1 against 9.6.  (FP32: 30,000 of 256 -> 256
  // 38 against 45, 16,384 of 512 -> 512 72 against 75, 8,192 of 1,024 -> 1,024 141 both.)
  constexpr int SMALL = sizeof(T) == 4 ? 32 : 64;
  // (transposed through registers: four blocks a unit leave too few for the loads)
  constexpr int LARGE = sizeof(T) == 4 || ALIGNED || !TRANS ? 32 : 64;
  const int64_t tiles = experts_tiles(rows, N, experts);
  if (N <= 64 || tiles < (sizeof(T) == 4 ? 1024 : 256)) {
    launch_direct<T, ALIGNED, TRANS, 64, 64, SMALL>(x, ldx, rows, K, W, bias, N, experts, perm, off, out, st);
    return;
  }
  // 16 bits, aligned: 256 columns by eight waves where those tiles are as full and there are many.  Both in us: 131,072 rows
  // of 512 -> 1,024 211 / 204, of 512 -> 512 103 / 99, 60,000 of 512 -> 512 over 40 experts 50 / 45; the other way 131,072 of
  // 256 -> 256 37 / 39, of 128 -> 512 39 / 41, 20,000 of 512 -> 1,024 35 / 37.
  if constexpr (sizeof(T) == 2 && ALIGNED) {
    if (N > 256 && K >= 256 && (N + 127) / 128 % 2 == 0 && tiles >= 1536) {
      launch_direct<T, ALIGNED, TRANS, 256, 128, 32>(x, ldx, rows, K, W, bias, N, experts, perm, off, out, st);
      return;
    }
  }
  launch_direct<T, ALIGNED, TRANS, 128, 128, LARGE>(x, ldx, rows, K, W, bias, N, experts, perm, off, out, st);
}

// Gradients of W (g^T x; operand A is x, so a lane ends with four consecutive columns of one row) and of b over one
// range of rows: see experts_outer_kernel.
template <typename T, bool ALIGNED, int TA, int TB, int S, int GA, int GB>
__global__ __launch_bounds__(GA * GB * 64, 2) void experts_direct_outer_kernel(
    const T* __restrict__ gy, int64_t ldg, int M, const T* __restrict__ x, int64_t ldx, int K, int experts, int ranges,
    const int* __restrict__ perm, const int* __restrict__ off, T* __restrict__ gW, T* __restrict__ gb,
    float* __restrict__ part) {
  static_assert(TA == TB, "one row number serves both operands");
  constexpr int WAVES = GA * GB, L = kLoads<T, TA, S, WAVES>, V = kChunk<T>, CH = TA / V, PER = 64 / CH;
  constexpr int KB = 64 * V;   // elements of a load
  constexpr int NA = TA / GA / 16, NB = TB / GB / 16;
  __shared__ __attribute__((aligned(16))) Word<T> A0[TA * S], A1[TA * S], B0[TB * S], B1[TB * S];
  const int ct = (K + TA - 1) / TA, tiles = ct * ((M + TB - 1) / TB);
  const int blk = die_order(blockIdx.x, gridDim.x), q = blk / tiles;
  const int k0 = blk % tiles % ct * TA, m0 = blk % tiles / ct * TB;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wa = wave / GB, wb = wave % GB;
  const int64_t MK = (int64_t)M * K;
  const bool bias = gb != nullptr && k0 == 0 && wa == 0;
  const int parts = gridDim.x / tiles;
  for (int e = q; e < experts; e += parts)   // experts without rows: zeros, shared out over the blocks of a tile
    if (off[e + 1] == off[e])
      zero_tile<T, TA, WAVES * 64>(gW + e * MK, gb ? gb + (int64_t)e * M : nullptr, M, K, m0, k0);
  if (q >= ranges) return;
  const Ranges range = find_ranges(off, experts, S, ranges);
  // this lane's row within a load, and its columns of both operands
  const int sub = lane / CH;
  Segment seg;
  for (int u = q * range.per; find_segment(off, experts, S, range, q, u, seg); u += seg.steps) {
    int node[L];   // row numbers, read a step before their rows
    auto name = [&](int row) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int r = row + (wave * L + i) * PER + sub;
        node[i] = r < seg.count ? perm[seg.start + r] : -1;
      }
    };
    u32x4 ra[L], rb[L];   // (not ALIGNED)
    auto column = [&](int i) { return ((lane % CH) ^ across_swap<T, TA>((wave * L + i) * PER + sub)) * V; };
    auto load = [&](Word<T>* A, Word<T>* B) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int c = column(i), ca = k0 + c < K ? k0 + c : k0, cb = m0 + c < M ? m0 + c : m0;
        const bool ok = node[i] >= 0;
        const T *px = x + (int64_t)node[i] * ldx + ca, *pg = gy + (int64_t)node[i] * ldg + cb;
        if (ALIGNED) {
          to_lds(ok ? (const void*)px : (const void*)kZeros, A + (wave * L + i) * KB);
          to_lds(ok ? (const void*)pg : (const void*)kZeros, B + (wave * L + i) * KB);
        } else {
          ra[i] = load_chunk_of(px, ok ? K - k0 - c : 0);
          rb[i] = load_chunk_of(pg, ok ? M - m0 - c : 0);
        }
      }
    };
    auto put = [&](Word<T>* A, Word<T>* B) {   // not ALIGNED: what load read
#pragma unroll
      for (int i = 0; i < L; ++i) {
        *reinterpret_cast<u32x4*>(A + (wave * L + i) * KB + lane * V) = move_chunk<T>(ra[i], K - k0 - column(i));
        *reinterpret_cast<u32x4*>(B + (wave * L + i) * KB + lane * V) = move_chunk<T>(rb[i], M - m0 - column(i));
      }
    };
    v4f acc[NA][NB], accb[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      accb[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NA; ++i) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    name(0);
    load(A0, B0);
    if (!ALIGNED) put(A0, B0);
    name(S);
    for (int row = 0; row < seg.count; row += 2 * S) {
      meet<ALIGNED>();
      if (row + S < seg.count) {
        load(A1, B1);
        name(row + 2 * S);
      }
      direct_step<T, true, true, TA, TB, S, GA, GB, true>(A0, B0, wa, wb, acc, bias, accb);
      if (row + S < seg.count) {
        if (!ALIGNED) put(A1, B1);
        meet<ALIGNED>();
        if (row + 2 * S < seg.count) {
          load(A0, B0);
          name(row + 3 * S);
        }
        direct_step<T, true, true, TA, TB, S, GA, GB, true>(A1, B1, wa, wb, acc, bias, accb);
        if (!ALIGNED && row + 2 * S < seg.count) put(A0, B0);
      }
    }
    meet<false>();   // the next segment's first load overwrites what a wave may still read
    float* pw = part + (int64_t)(2 * q + seg.slot) * (MK + M);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int m = m0 + (wb * NB + j) * 16 + li;
      if (m >= M) continue;
      if (bias && g == 0) {
        if (seg.whole)
          gb[(int64_t)seg.expert * M + m] = (T)accb[j][0];
        else
          pw[MK + m] = accb[j][0];
      }
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int k = k0 + (wa * NA + i) * 16 + 4 * g;
        if (k >= K) continue;
        T* w = gW + (int64_t)seg.expert * MK + (int64_t)m * K + k;
        float* p = pw + (int64_t)m * K + k;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)acc[i][j][e];
        if (ALIGNED || k + 4 <= K) {   // (ALIGNED: K is a multiple of 4)
          if (seg.whole)
            __builtin_memcpy(w, v, sizeof(v));
          else
            *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, acc[i][j]);
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e) {
            if (k + e >= K) continue;
            if (seg.whole)
              w[e] = v[e];
            else
              p[e] = acc[i][j][e];
          }
        }
      }
    }
  }
}

template <typename T, bool ALIGNED, int TILE, int S>
void launch_outer(const OuterPlan& plan, const void* gy, int64_t ldg, int M, const void* x, int64_t ldx, int K,
                  int experts, const int* perm, const int* off, void* gW, void* gb, float* part, hipStream_t st) {
  const int64_t tiles = (int64_t)((M + TILE - 1) / TILE) * ((K + TILE - 1) / TILE);
  const dim3 grid((unsigned)(std::max(plan.ranges, plan.fill) * tiles));
  hipLaunchKernelGGL((experts_direct_outer_kernel<T, ALIGNED, TILE, TILE, S, 2, 2>), grid, dim3(256), 0, st, (const T*)gy,
                     ldg, M, (const T*)x, ldx, K, experts, plan.ranges, perm, off, (T*)gW, (T*)gb, part);
}

template <typename T, bool ALIGNED>
void direct_outer(const OuterPlan& plan, const void* gy, int64_t ldg, int M, const void* x, int64_t ldx, int K,
                  int experts, const int* perm, const int* off, void* gW, void* gb, float* part, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    launch_outer<T, ALIGNED, 128, 64>(plan, gy, ldg, M, x, ldx, K, experts, perm, off, gW, gb, part, st);
  else if (plan.tile == 64)
    launch_outer<T, ALIGNED, 64, 64>(plan, gy, ldg, M, x, ldx, K, experts, perm, off, gW, gb, part, st);
  else
    launch_outer<T, ALIGNED, 128, 32>(plan, gy, ldg, M, x, ldx, K, experts, perm, off, gW, gb, part, st);
}

bool whole16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool ALIGNED, bool TRANS, typename... A>
void typed_rows(int dtype, A... a) {
  if (dtype == ICTC_F32)
    direct_rows<float, ALIGNED, TRANS>(a...);
  else if (dtype == ICTC_BF16)
    direct_rows<bf16, ALIGNED, TRANS>(a...);
  else
    direct_rows<f16, ALIGNED, TRANS>(a...);
}

template <bool ALIGNED, typename... A>
void either_rows(int dtype, bool transpose, A... a) {
  if (transpose)
    typed_rows<ALIGNED, true>(dtype, a...);
  else
    typed_rows<ALIGNED, false>(dtype, a...);
}

template <bool ALIGNED, typename... A>
void typed_outer(int dtype, A... a) {
  if (dtype == ICTC_F32)
    direct_outer<float, ALIGNED>(a...);
  else if (dtype == ICTC_BF16)
    direct_outer<bf16, ALIGNED>(a...);
  else
    direct_outer<f16, ALIGNED>(a...);
}

}  // namespace

static int chunk_of(int dtype) { return dtype == ICTC_F32 ? 4 : 8; }

bool experts_direct_rows_fit(int dtype, int K, int N, bool transpose) {
  return K >= chunk_of(dtype) && (!transpose || N >= chunk_of(dtype));
}

void experts_direct_rows(int dtype, const void* x, int64_t ldx, int64_t rows, int K, const void* W, const void* bias,
                         int N, int experts, const int* perm, const int* off, bool transpose, void* out,
                         hipStream_t st) {
  // 16-byte chunks of x, and of the weights along their memory, whole and aligned
  const int v = chunk_of(dtype);
  if (whole16(x) && ldx % v == 0 && K % v == 0 && whole16(W) && (!transpose || N % v == 0))
    either_rows<true>(dtype, transpose, x, ldx, rows, K, W, bias, N, experts, perm, off, out, st);
  else
    either_rows<false>(dtype, transpose, x, ldx, rows, K, W, bias, N, experts, perm, off, out, st);
}

bool experts_direct_outer_fits(int dtype, int M, int K) { return M >= chunk_of(dtype) && K >= chunk_of(dtype); }

void experts_direct_outer(int dtype, const OuterPlan& plan, const void* gy, int64_t ldg, int M, const void* x,
                          int64_t ldx, int K, int experts, const int* perm, const int* off, void* gW, void* gb,
                          float* part, hipStream_t st) {
  const int v = chunk_of(dtype);
  if (whole16(gy) && whole16(x) && ldg % v == 0 && ldx % v == 0 && M % v == 0 && K % v == 0)
    typed_outer<true>(dtype, plan, gy, ldg, M, x, ldx, K, experts, perm, off, gW, gb, part, st);
  else
    typed_outer<false>(dtype, plan, gy, ldg, M, x, ldx, K, experts, perm, off, gW, gb, part, st);
}
