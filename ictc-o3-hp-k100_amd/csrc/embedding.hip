// Rows of a table chosen by an id and scaled, and the table's gradient (FP32, bfloat16 or FP16):
//   out[n] = scale table[ids[n]]            (a zero row where the id is outside [0, entries))
//   dtable[v] = scale sum over the rows n of id v of g[n]    (zeros for an id without rows)
// Both are bound by memory: the lookup writes its output, the gradient reads its rows once and writes the table once.
// 131,072 rows of 128 FP32, ten entries: lookup 13 us (5.1 TB/s), order 8, gradient 15.5 (4.3 TB/s) and join 6; 60,013 rows of
// 1,021 FP16, 50,021 entries: lookup 49 us, order 28, gradient 63 (3.6 TB/s), join 9; 425,991 rows of 64 bfloat16, 7,921
// entries: lookup 13 us, order 31, gradient 21, join 4.
//
// The gradient takes the rows in the order of their id (perm, offsets: what ictc_expert_order and ictc_csr_build give),
// cut into equal ranges whatever the ids' shares, so an id that a tenth of all rows has costs no more than many rare
// ones.  A team of lanes holds a chunk of columns in registers and adds consecutive sorted rows; a run of one id that
// lies within the team's rows is written at once, the first and the last run of a team meet the neighbours' in LDS, and
// those of a block that continue in other blocks leave FP32 partial sums (slot 0: continued from before; slot 1: begun
// here) that a second kernel adds in order, in FP64.  Every sum has a fixed order.  Up to 128 rows are added by one kernel
// that looks the ids over itself.
#include <algorithm>

#include "dense.h"

namespace {

constexpr int kMaxWidth = 65536, kUnroll = 4, kFewRows = 128, kMaxBlocks = 1 << 20;

// Lanes of a row's chunks (16 bytes; of narrower rows single elements): the power of two that covers the width, at most a
// wave.
int chunk_of(int64_t width, int chunk) { return width < chunk ? 1 : chunk; }

int team_of(int64_t width, int chunk) {
  int lanes = 1;
  while (lanes < 64 && (int64_t)lanes * chunk < width) lanes *= 2;
  return lanes;
}

// First column of a lane's chunk: a row's last chunk is read back from its end, so that none is in part.  Two lanes then
// have some columns alike, and write the same there.  (60,013 rows of 1,021 FP16: lookup 61 -> 50 us, gradient 85 -> 65.)
template <int V>
__device__ __forceinline__ int column_of(int c, int width) {
  return min(c, width - V);
}

template <typename T, int V, int L>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, int64_t entries, int width,
                                                        const int64_t* __restrict__ ids, int64_t rows, float scale,
                                                        T* __restrict__ out) {
  constexpr int TEAMS = 256 / L;
  const int c0 = (blockIdx.y * L + threadIdx.x % L) * V, c = column_of<V>(c0, width);
  if (c0 >= width) return;
  for (int64_t first = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / L) * kUnroll; first < rows;
       first += (int64_t)gridDim.x * TEAMS * kUnroll) {
    int64_t id[kUnroll];
    Pack<T, V> raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) id[i] = first + i < rows ? ids[first + i] : -1;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const bool in = (uint64_t)id[i] < (uint64_t)entries;
      raw[i] = load_pack<T, V>(table + (in ? id[i] * width + c : 0), in);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (first + i >= rows) break;
      const bool in = (uint64_t)id[i] < (uint64_t)entries;
      float v[V];
      get<T, V>(raw[i], v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = in ? held(v[e] * scale) : 0.f;
      store_pack<T, V>(out + (first + i) * width + c, v);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void write_scaled(T* __restrict__ p, const float (&acc)[V], float scale) {
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = held(acc[e] * scale);
  store_pack<T, V>(p, v);
}

// Few rows: a team per entry adds the rows whose id is its own, in their order.  Its lanes hold the ids, kFewRows / L
// each, and compare them with the entry all at once, so an entry without rows costs a ballot and its store.  Measured in
// us, 128 rows this way / 129 in order with the order's launches, FP32: ten entries of 64 5 / 12; 10,000 5 / 19; 150,000
// 14 / 28; a million 67 / 66, of 128 78 / 121.  (Each team looking all ids over in LDS: 28, 29, 133, 774 and 1,533.)
template <typename T, int V, int L>
__global__ __launch_bounds__(256) void embed_few_kernel(const T* __restrict__ g, int64_t ldg, int rows, int width,
                                                        const int64_t* __restrict__ ids, int entries, float scale,
                                                        T* __restrict__ out) {
  constexpr int TEAMS = 256 / L, IDS = kFewRows / L;
  const int lane = threadIdx.x % L, shift = (threadIdx.x & 63) / L * L;
  const int c0 = (blockIdx.y * L + lane) * V, c = column_of<V>(c0, width);
  const bool live = c0 < width;
  int id[IDS];   // of rows i L + lane; -1: none, or outside the table
#pragma unroll
  for (int i = 0; i < IDS; ++i) {
    const int64_t k = i * L + lane < rows ? ids[i * L + lane] : -1;
    id[i] = (uint64_t)k < (uint64_t)entries ? (int)k : -1;
  }
  const auto mine = [&](bool hit) {   // the team's lanes that say so
    const uint64_t m = __ballot(hit) >> shift;
    return L == 64 ? m : m & ((uint64_t(1) << (L & 63)) - 1);
  };
  for (int64_t v = (int64_t)blockIdx.x * TEAMS + threadIdx.x / L; v < entries; v += (int64_t)gridDim.x * TEAMS) {
    float acc[V] = {};
    bool any = false;
#pragma unroll
    for (int i = 0; i < IDS; ++i) any |= id[i] == (int)v;
    if (mine(any)) {
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        uint64_t m = mine(id[i] == (int)v);
        while (m) {   // the next rows of this entry
          Pack<T, V> raw[kUnroll];
#pragma unroll
          for (int k = 0; k < kUnroll; ++k) {
            const bool in = live && m != 0;
            raw[k] = load_pack<T, V>(g + (in ? (i * L + __builtin_ctzll(m)) * ldg + c : 0), in);
            m &= m - 1;
          }
#pragma unroll
          for (int k = 0; k < kUnroll; ++k) {
            float x[V];
            get<T, V>(raw[k], x);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += x[e];
          }
        }
      }
    }
    if (live) write_scaled<T, V>(out + v * width + c, acc, scale);
  }
}

// part [ranges][2][width]; a block takes `per` sorted rows a team.  open [ranges]: the id of the run that begins in the
// range and goes on behind it, or -1.
template <typename T, int V, int L>
__global__ __launch_bounds__(256) void embed_grad_kernel(const T* __restrict__ g, int64_t ldg, int width,
                                                         const int64_t* __restrict__ ids, int64_t entries,
                                                         const int* __restrict__ perm, const int* __restrict__ off,
                                                         float scale, int per, int ranges, float* __restrict__ part,
                                                         int* __restrict__ open, T* __restrict__ out) {
  constexpr int TEAMS = 256 / L, W = L * V, AHEAD = 8;
  extern __shared__ int staged[];         // the range's row numbers, and their ids
  __shared__ float sums[2][TEAMS][V + W];   // of each team's first run, and of its last where that is another (V: see column_of)
  __shared__ int keys[2][TEAMS];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const int c0 = blockIdx.y * W, c = column_of<V>(c0 + lane * V, width);
  const bool live = c0 + lane * V < width;
  const int at_lds = V + c - c0;
  const int64_t n = off[entries], start = (int64_t)blockIdx.x * TEAMS * per;   // (ids outside the table come last)
  const int count = (int)max<int64_t>(0, min(n - start, (int64_t)TEAMS * per));
  int *row = staged, *id = staged + TEAMS * per;
  for (int k = threadIdx.x; k < count; k += 256) {
    row[k] = perm[start + k];
    id[k] = (int)ids[row[k]];
  }
  const float zero[V] = {};
  for (int64_t e = (int64_t)blockIdx.x * TEAMS + team; e < entries; e += (int64_t)gridDim.x * TEAMS)
    if (live && off[e] == off[e + 1]) store_pack<T, V>(out + e * width + c, zero);
  if (open && blockIdx.y == 0 && threadIdx.x == 0 && (int)blockIdx.x < ranges) open[blockIdx.x] = -1;
  if (count == 0) return;
  __syncthreads();
  auto write = [&](int key, const float (&acc)[V]) {
    if (live && key >= 0 && key < entries) write_scaled<T, V>(out + (int64_t)key * width + c, acc, scale);
  };
  float acc[V] = {};
  int key = -1;
  bool first = true;
  const int end = min(count, (team + 1) * per);
  for (int p = team * per; p < end; p += AHEAD) {
    Pack<T, V> raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const bool in = live && p + i < end;
      raw[i] = load_pack<T, V>(g + (in ? row[p + i] * ldg + c : 0), in);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p + i >= end) break;
      const int k = id[p + i];
      if (key != k) {
        if (key >= 0) {
          if (first) {
            if (live) {
#pragma unroll
              for (int e = 0; e < V; ++e) sums[0][team][at_lds + e] = acc[e];
            }
            if (lane == 0) keys[0][team] = key;
            first = false;
          } else {
            write(key, acc);
          }
        }
        key = k;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
      }
      float x[V];
      get<T, V>(raw[i], x);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += x[e];
    }
  }
  if (live) {
#pragma unroll
    for (int e = 0; e < V; ++e) sums[first ? 0 : 1][team][at_lds + e] = acc[e];
  }
  if (lane == 0) {
    keys[first ? 0 : 1][team] = key;
    if (first) keys[1][team] = -1;
  }
  __syncthreads();
  // The runs that meet other teams', each by the team that it begins in (or the first): its last run takes the first runs of
  // the teams behind it, in order, as long as they are of its id.
  if (!live || keys[0][team] < 0) return;
  const int64_t last = start + count;
  const int before = start > 0 ? (int)ids[perm[start - 1]] : -1, after = last < n ? (int)ids[perm[last]] : -1;
  const int k0 = keys[0][team], k1 = keys[1][team];
  const int previous = team == 0 ? before : keys[1][team - 1] >= 0 ? keys[1][team - 1] : keys[0][team - 1];
  auto own = [&](int which) {
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = sums[which][team][at_lds + e];
  };
  auto keep = [&](int slot) {
    if (!part) return;
    float* p = part + ((int64_t)blockIdx.x * 2 + slot) * width + c;
#pragma unroll
    for (int e = 0; e < V; ++e) p[e] = acc[e];
  };
  if (k1 >= 0) {
    own(0);
    if (k0 != previous)
      write(k0, acc);
    else if (team == 0)
      keep(0);
  }
  const int key_last = k1 >= 0 ? k1 : k0;
  const bool begins = k1 >= 0 || k0 != previous;
  if (!begins && team > 0) return;
  own(k1 >= 0 ? 1 : 0);
  bool goes_on = true;   // to the end of the block
  for (int t = team + 1; t < TEAMS && keys[0][t] >= 0; ++t) {
    if (keys[0][t] != key_last) {
      goes_on = false;
      break;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] += sums[0][t][at_lds + e];
    if (keys[1][t] >= 0) {
      goes_on = false;
      break;
    }
  }
  if (!begins) {
    keep(0);
  } else if (goes_on && key_last == after) {
    keep(1);
    if (open && c == 0) open[blockIdx.x] = key_last < entries ? key_last : -1;
  } else {
    write(key_last, acc);
  }
}

// The runs that cross ranges, each by the blocks of the range that it begins in, 64 columns a block: its partial sums added
// by 16 slices and those in order, in FP64, for a run may have a tenth of all rows and more (4.2 million rows of 256 in a run
// are 2,048 sums a slice: values alike lose 480 units of 2^-24 in FP32).
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(const float* __restrict__ part, const int* __restrict__ open,
                                                         int width, const int* __restrict__ off, float scale,
                                                         int64_t range, T* __restrict__ out) {
  __shared__ double lds[16][64];
  const int64_t q = blockIdx.x;
  const int key = open[q];
  if (key < 0) return;
  const int64_t count = (off[key + 1] - 1) / range - q + 1;
  const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int c = blockIdx.y * 64 + lane * 4, left = width - c;
  double a[4] = {};
#pragma unroll 8
  for (int64_t j = slice; j < count; j += 16) {
    float x[4];
    load_chunk<float>(part + ((q + j) * 2 + (j == 0 ? 1 : 0)) * width + c, left, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += x[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) lds[slice][lane * 4 + e] = a[e];
  __syncthreads();
  const int col = threadIdx.x;
  if (col < 64 && blockIdx.y * 64 + col < width) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][col];
    out[(int64_t)key * width + blockIdx.y * 64 + col] = (T)held(held((float)s) * scale);
  }
}

// How the sorted rows are cut: `per` rows a team, `ranges` blocks, `blocks` with those that only write zeros.
struct GradPlan {
  int lanes, per;
  int64_t range, ranges, blocks;
  int columns;
};

GradPlan grad_plan(int dtype, int64_t rows, int64_t entries, int64_t width) {
  const int chunk = chunk_of(width, dtype == ICTC_F32 ? 4 : 8);
  GradPlan p;
  // eight lanes at least, some idle, so that a block has few teams whose runs meet (60,013 rows of one element 45 -> 11 us)
  p.lanes = std::max(8, team_of(width, chunk));
  p.columns = (int)((width + p.lanes * chunk - 1) / (p.lanes * chunk));
  const int64_t teams = 256 / p.lanes;
  const int64_t want = (rows * p.columns + teams * 2048 - 1) / (teams * 2048);
  p.per = (int)((std::min<int64_t>(32, std::max<int64_t>(4, want)) + 3) / 4 * 4);
  p.range = teams * p.per;
  p.ranges = (rows + p.range - 1) / p.range;
  p.blocks = std::max<int64_t>(std::max<int64_t>(1, p.ranges), std::min<int64_t>(2048, (entries + teams - 1) / teams));
  return p;
}

const char* bad_sizes(int dtype, int64_t rows, int64_t entries, int64_t width) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "embedding: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (rows < 0 || rows >= (int64_t(1) << 31) - 2) return "embedding: up to 2^31 - 3 rows";
  if (entries < 1 || entries >= (int64_t(1) << 31) - 2) return "embedding: 1 to 2^31 - 3 entries";
  if (width < 1 || width > kMaxWidth) return "embedding: rows of 1 to 65536 elements";
  return nullptr;
}

#define EMBED_CASE(V_, L_, ...)           \
  case L_: {                              \
    constexpr int V = V_, L = L_;         \
    __VA_ARGS__;                          \
    break;                                \
  }
#define EMBED_LANES(width, n, ...)            \
  if ((width) < kChunk<T>) {                  \
    switch (n) {                              \
      EMBED_CASE(1, 1, __VA_ARGS__)           \
      EMBED_CASE(1, 2, __VA_ARGS__)           \
      EMBED_CASE(1, 4, __VA_ARGS__)           \
      EMBED_CASE(1, 8, __VA_ARGS__)           \
    }                                         \
  } else {                                    \
    switch (n) {                              \
      EMBED_CASE(kChunk<T>, 1, __VA_ARGS__)   \
      EMBED_CASE(kChunk<T>, 2, __VA_ARGS__)   \
      EMBED_CASE(kChunk<T>, 4, __VA_ARGS__)   \
      EMBED_CASE(kChunk<T>, 8, __VA_ARGS__)   \
      EMBED_CASE(kChunk<T>, 16, __VA_ARGS__)  \
      EMBED_CASE(kChunk<T>, 32, __VA_ARGS__)  \
      EMBED_CASE(kChunk<T>, 64, __VA_ARGS__)  \
    }                                         \
  }
#define EMBED_TEAMS(width, n, ...)            \
  if ((width) < kChunk<T>) {                  \
    constexpr int V = 1, L = 8;               \
    __VA_ARGS__;                              \
  } else {                                    \
    switch (n) {                              \
      EMBED_CASE(kChunk<T>, 8, __VA_ARGS__)   \
      EMBED_CASE(kChunk<T>, 16, __VA_ARGS__)  \
      EMBED_CASE(kChunk<T>, 32, __VA_ARGS__)  \
      EMBED_CASE(kChunk<T>, 64, __VA_ARGS__)  \
    }                                         \
  }

template <typename T>
void run_fwd(const void* table, int64_t entries, int width, const int64_t* ids, int64_t rows, float scale, void* out,
             hipStream_t st) {
  const int chunk = chunk_of(width, kChunk<T>), lanes = team_of(width, chunk);
  const int columns = (width + lanes * chunk - 1) / (lanes * chunk);
  const int64_t block = 256 / lanes * kUnroll;
  const dim3 grid((unsigned)std::min<int64_t>(kMaxBlocks, (rows + block - 1) / block), columns);
  EMBED_LANES(width, lanes, hipLaunchKernelGGL((embed_fwd_kernel<T, V, L>), grid, dim3(256), 0, st, (const T*)table, entries,
                                        width, ids, rows, scale, (T*)out))
}

template <typename T>
void run_bwd(const void* g, int64_t ldg, int64_t rows, int width, int64_t entries, const int64_t* ids, const int* perm,
             const int* off, float scale, void* out, float* part, hipStream_t st) {
  constexpr int dtype = sizeof(T) == 4 ? ICTC_F32 : ICTC_BF16;   // (only the size counts)
  const GradPlan p = grad_plan(dtype, rows, entries, width);
  if (rows <= kFewRows) {
    const int64_t teams = 256 / p.lanes;
    const dim3 grid((unsigned)std::min<int64_t>(kMaxBlocks, (entries + teams - 1) / teams), p.columns);
    EMBED_TEAMS(width, p.lanes, hipLaunchKernelGGL((embed_few_kernel<T, V, L>), grid, dim3(256), 0, st, (const T*)g, ldg,
                                            (int)rows, width, ids, (int)entries, scale, (T*)out))
    return;
  }
  const dim3 grid((unsigned)p.blocks, p.columns);
  int* open = p.ranges > 1 ? (int*)(part + p.ranges * 2 * width) : nullptr;
  EMBED_TEAMS(width, p.lanes, hipLaunchKernelGGL((embed_grad_kernel<T, V, L>), grid, dim3(256), (unsigned)(p.range * 8), st,
                                          (const T*)g, ldg, width, ids, entries, perm, off, scale, p.per, (int)p.ranges,
                                          open ? part : nullptr, open, (T*)out))
  if (open)
    hipLaunchKernelGGL(embed_join_kernel<T>, dim3((unsigned)(p.ranges - 1), (unsigned)((width + 63) / 64)), dim3(256), 0,
                       st, part, open, width, off, scale, p.range, (T*)out);
}

}  // namespace

extern "C" {

int ictc_embedding_fwd(int dtype, const void* table, int64_t entries, int width, const int64_t* ids, int64_t rows,
                       float scale, void* out, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, entries, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (rows == 0) return ICTC_OK;
  if (!table || !ids || !out) return dense_fail(ICTC_ERR_ARGUMENT, "embedding: null operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ICTC_F32)
    run_fwd<float>(table, entries, width, ids, rows, scale, out, st);
  else if (dtype == ICTC_BF16)
    run_fwd<bf16>(table, entries, width, ids, rows, scale, out, st);
  else
    run_fwd<f16>(table, entries, width, ids, rows, scale, out, st);
  return dense_status("embedding_fwd launch");
}

int ictc_embedding_needs_order(int64_t rows) { return rows > kFewRows; }

int64_t ictc_embedding_bwd_workspace_bytes(int dtype, int64_t rows, int64_t entries, int width) {
  if (bad_sizes(dtype, rows, entries, width)) return -1;
  const GradPlan p = grad_plan(dtype, rows, entries, width);
  return rows <= kFewRows || p.ranges < 2 ? 0 : p.ranges * (2 * width + 1) * (int64_t)sizeof(float);
}

int ictc_embedding_bwd(int dtype, const void* grad, int64_t ldg, int64_t rows, int width, const int64_t* ids,
                       int64_t entries, const int32_t* perm, const int32_t* offsets, float scale, void* dtable,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* e = bad_sizes(dtype, rows, entries, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (ldg < width && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "embedding: row pitch below the width");
  if (!dtable || (rows > 0 && (!grad || !ids))) return dense_fail(ICTC_ERR_ARGUMENT, "embedding: null operand");
  if (rows > kFewRows && (!perm || !offsets))
    return dense_fail(ICTC_ERR_ARGUMENT, "embedding: more than 128 rows need their order");
  const int64_t need = ictc_embedding_bwd_workspace_bytes(dtype, rows, entries, width);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || workspace_bytes < need))
    return dense_fail(ICTC_ERR_ARGUMENT, "embedding: workspace smaller than ictc_embedding_bwd_workspace_bytes");
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  if (dtype == ICTC_F32)
    run_bwd<float>(grad, ldg, rows, width, entries, ids, perm, offsets, scale, dtable, part, st);
  else if (dtype == ICTC_BF16)
    run_bwd<bf16>(grad, ldg, rows, width, entries, ids, perm, offsets, scale, dtable, part, st);
  else
    run_bwd<f16>(grad, ldg, rows, width, entries, ids, perm, offsets, scale, dtable, part, st);
  return dense_status("embedding_bwd launch");
}

}  // extern "C"
