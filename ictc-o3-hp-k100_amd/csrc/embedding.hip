// Rows of a table chosen by an id and scaled, and the table's gradient (FP32, bfloat16 or FP16):
//   out[n] = scale table[ids[n]]            (a zero row where the id is outside [0, entries))
//   dtable[v] = scale sum over the rows n of id v of g[n]    (zeros for an id without rows)
// Both are bound by memory: the lookup writes its output, the gradient reads its rows once and writes the table once.
//
// The gradient takes the rows in the order of their id (perm, offsets: what ictc_expert_order and ictc_csr_build give),
// cut into equal ranges whatever the ids' shares, so an id that a tenth of all rows has costs no more than many rare
// ones.  A team of lanes holds a chunk of columns in registers and adds consecutive sorted rows; a run of one id that
// lies within the team's rows is written at once, the first and the last run of a team meet the neighbours' in LDS, and
// those of a block that continue in other blocks leave FP32 partial sums (slot 0: continued from before; slot 1: begun
// here) that a second kernel adds in order.  Every sum has a fixed order.  Up to 128 rows are added by one kernel that
// looks the ids over itself.
#include <algorithm>

#include "dense.h"

namespace {

constexpr int kMaxWidth = 65536, kUnroll = 4, kFewRows = 128, kMaxBlocks = 1 << 20;

// Lanes of a row's chunks: the power of two that covers the width, at most a wave.
int team_of(int64_t width, int chunk) {
  int lanes = 1;
  while (lanes < 64 && (int64_t)lanes * chunk < width) lanes *= 2;
  return lanes;
}

template <typename T, int L>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, int64_t entries, int width,
                                                        const int64_t* __restrict__ ids, int64_t rows, float scale,
                                                        T* __restrict__ out) {
  constexpr int V = kChunk<T>, TEAMS = 256 / L;
  const int c = (blockIdx.y * L + threadIdx.x % L) * V;
  if (c >= width) return;
  for (int64_t first = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / L) * kUnroll; first < rows;
       first += (int64_t)gridDim.x * TEAMS * kUnroll) {
    int64_t id[kUnroll];
    u32x4 raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) id[i] = first + i < rows ? ids[first + i] : -1;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const bool in = (uint64_t)id[i] < (uint64_t)entries;
      raw[i] = load_raw(table + (in ? id[i] * width + c : 0), in ? width - c : 0);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (first + i >= rows) break;
      const bool in = (uint64_t)id[i] < (uint64_t)entries;
      float v[V];
      widen<T>(raw[i], v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = in ? held(v[e] * scale) : 0.f;
      store_chunk(out + (first + i) * width + c, width - c, v);
    }
  }
}

template <typename T>
__device__ __forceinline__ void write_scaled(T* __restrict__ p, int n, const float* acc, float scale) {
  float v[kChunk<T>];
#pragma unroll
  for (int e = 0; e < kChunk<T>; ++e) v[e] = held(acc[e] * scale);
  store_chunk(p, n, v);
}

// Few rows: a team per entry adds the rows whose id is its own, in their order.
template <typename T, int L>
__global__ __launch_bounds__(256) void embed_few_kernel(const T* __restrict__ g, int64_t ldg, int rows, int width,
                                                        const int64_t* __restrict__ ids, int64_t entries, float scale,
                                                        T* __restrict__ out) {
  constexpr int V = kChunk<T>, TEAMS = 256 / L;
  __shared__ int64_t id[kFewRows];
  if ((int)threadIdx.x < rows) id[threadIdx.x] = ids[threadIdx.x];
  __syncthreads();
  const int c = (blockIdx.y * L + threadIdx.x % L) * V;
  if (c >= width) return;
  for (int64_t v = (int64_t)blockIdx.x * TEAMS + threadIdx.x / L; v < entries; v += (int64_t)gridDim.x * TEAMS) {
    float acc[V] = {};
    for (int r = 0; r < rows;) {
      int64_t row[kUnroll] = {};
      int n = 0;
      while (n < kUnroll) {   // the next rows of this id
        while (r < rows && id[r] != v) ++r;
        if (r >= rows) break;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) row[i] = i == n ? r : row[i];
        ++r;
        ++n;
      }
      u32x4 raw[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) raw[i] = load_raw(g + (i < n ? row[i] * ldg + c : 0), i < n ? width - c : 0);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        float x[V];
        widen<T>(raw[i], x);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += x[e];
      }
    }
    write_scaled(out + v * width + c, width - c, acc, scale);
  }
}

// part [ranges][2][width]; a block takes `per` sorted rows a team.
template <typename T, int L>
__global__ __launch_bounds__(256) void embed_grad_kernel(const T* __restrict__ g, int64_t ldg, int width,
                                                         const int64_t* __restrict__ ids, int64_t entries,
                                                         const int* __restrict__ perm, const int* __restrict__ off,
                                                         float scale, int per, float* __restrict__ part,
                                                         T* __restrict__ out) {
  constexpr int V = kChunk<T>, TEAMS = 256 / L, W = L * V;
  __shared__ float sums[2][TEAMS][W];     // of each team's first run, and of its last where that is another
  __shared__ int64_t keys[2][TEAMS];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const int c0 = blockIdx.y * W, c = c0 + lane * V, left = width - c;
  const float zero[V] = {};
  for (int64_t e = (int64_t)blockIdx.x * TEAMS + team; e < entries; e += (int64_t)gridDim.x * TEAMS)
    if (off[e] == off[e + 1]) store_chunk(out + e * width + c, left, zero);
  const int64_t n = off[entries], start = (int64_t)blockIdx.x * TEAMS * per;   // (ids outside the table come last)
  if (start >= n) return;
  const int64_t end = min(n, start + (int64_t)TEAMS * per);
  const int64_t p1 = min(end, start + (int64_t)(team + 1) * per);
  auto write = [&](int64_t key, const float* acc) {
    if ((uint64_t)key < (uint64_t)entries) write_scaled(out + key * width + c, left, acc, scale);
  };
  float acc[V] = {};
  int64_t key = -1;
  bool first = true;
  for (int64_t p = start + (int64_t)team * per; p < p1; p += kUnroll) {
    int64_t row[kUnroll], id[kUnroll];
    u32x4 raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) row[i] = p + i < p1 ? perm[p + i] : -1;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      id[i] = row[i] >= 0 ? ids[row[i]] : -1;
      raw[i] = load_raw(g + (row[i] >= 0 ? row[i] * ldg + c : 0), row[i] >= 0 ? left : 0);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (p + i >= p1) break;
      if (key != id[i]) {
        if (key >= 0) {
          if (first) {
#pragma unroll
            for (int e = 0; e < V; ++e) sums[0][team][lane * V + e] = acc[e];
            if (lane == 0) keys[0][team] = key;
            first = false;
          } else {
            write(key, acc);
          }
        }
        key = id[i];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
      }
      float x[V];
      widen<T>(raw[i], x);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sums[first ? 0 : 1][team][lane * V + e] = acc[e];
  if (lane == 0) {
    keys[first ? 0 : 1][team] = key;
    if (first) keys[1][team] = -1;
  }
  __syncthreads();
  // the block's open runs: a column a thread, the teams in order
  const int64_t before = start > 0 ? ids[perm[start - 1]] : -1, after = end < n ? ids[perm[end]] : -1;
  for (int col = threadIdx.x; col < W && c0 + col < width; col += 256) {
    float a = 0.f;
    int64_t at = keys[0][0];
    bool begins = at != before;    // the present run begins in this block
    auto flush = [&](bool ends) {
      if (at < 0 || at >= entries) return;
      if (begins && ends)
        out[at * width + c0 + col] = (T)held(a * scale);
      else
        part[((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * width + c0 + col] = a;
    };
#pragma unroll 4
    for (int t = 0; t < TEAMS; ++t) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t k = keys[s][t];
        if (k < 0) continue;
        const float x = sums[s][t][col];
        if (k != at) {
          flush(true);
          at = k;
          begins = true;
          a = x;
        } else {
          a += x;
        }
      }
    }
    flush(at != after);
  }
}

// The runs that cross ranges, each by the block of the first boundary that it crosses: its partial sums added by 32
// slices and those in order.
template <typename T>
__global__ __launch_bounds__(512) void embed_join_kernel(const float* __restrict__ part, int width,
                                                         const int64_t* __restrict__ ids, int64_t entries,
                                                         const int* __restrict__ perm, const int* __restrict__ off,
                                                         float scale, int64_t range, T* __restrict__ out) {
  __shared__ float lds[32][17];
  const int64_t q = blockIdx.x, p = (q + 1) * range;
  if (p >= off[entries]) return;
  const int64_t key = ids[perm[p]];
  if (ids[perm[p - 1]] != key || (uint64_t)key >= (uint64_t)entries || off[key] / range != q) return;
  const int64_t count = (off[key + 1] - 1) / range - q + 1;
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int c = blockIdx.y * 16 + col;
  float a = 0.f;
  if (c < width) {
#pragma unroll 4
    for (int64_t j = slice; j < count; j += 32) a += part[((q + j) * 2 + (j == 0 ? 1 : 0)) * width + c];
  }
  lds[slice][col] = a;
  __syncthreads();
  if (slice == 0 && c < width) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += lds[i][col];
    out[key * width + c] = (T)held(s * scale);
  }
}

// How the sorted rows are cut: `per` rows a team, `ranges` blocks, `blocks` with those that only write zeros.
struct GradPlan {
  int lanes, per;
  int64_t range, ranges, blocks;
  int columns;
};

GradPlan grad_plan(int dtype, int64_t rows, int64_t entries, int64_t width) {
  const int chunk = dtype == ICTC_F32 ? 4 : 8;
  GradPlan p;
  p.lanes = team_of(width, chunk);
  p.columns = (int)((width + p.lanes * chunk - 1) / (p.lanes * chunk));
  const int64_t teams = 256 / p.lanes;
  const int64_t want = (rows * p.columns + teams * 2048 - 1) / (teams * 2048);
  const int64_t most = std::max<int64_t>(32, rows / (teams << 20) + 1);   // (no more than about a million ranges)
  p.per = (int)((std::min(most, std::max<int64_t>(4, want)) + kUnroll - 1) / kUnroll * kUnroll);
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

#define EMBED_CASE(L_, ...)      \
  case L_: {                     \
    constexpr int L = L_;        \
    __VA_ARGS__;                 \
    break;                       \
  }
#define EMBED_LANES(n, ...)                                                                                  \
  switch (n) {                                                                                               \
    EMBED_CASE(1, __VA_ARGS__)                                                                               \
    EMBED_CASE(2, __VA_ARGS__)                                                                               \
    EMBED_CASE(4, __VA_ARGS__)                                                                               \
    EMBED_CASE(8, __VA_ARGS__)                                                                               \
    EMBED_CASE(16, __VA_ARGS__)                                                                              \
    EMBED_CASE(32, __VA_ARGS__)                                                                              \
    EMBED_CASE(64, __VA_ARGS__)                                                                              \
  }

template <typename T>
void run_fwd(const void* table, int64_t entries, int width, const int64_t* ids, int64_t rows, float scale, void* out,
             hipStream_t st) {
  const int lanes = team_of(width, kChunk<T>), columns = (width + lanes * kChunk<T> - 1) / (lanes * kChunk<T>);
  const int64_t block = 256 / lanes * kUnroll;
  const dim3 grid((unsigned)std::min<int64_t>(kMaxBlocks, (rows + block - 1) / block), columns);
  EMBED_LANES(lanes, hipLaunchKernelGGL((embed_fwd_kernel<T, L>), grid, dim3(256), 0, st, (const T*)table, entries,
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
    EMBED_LANES(p.lanes, hipLaunchKernelGGL((embed_few_kernel<T, L>), grid, dim3(256), 0, st, (const T*)g, ldg,
                                            (int)rows, width, ids, entries, scale, (T*)out))
    return;
  }
  const dim3 grid((unsigned)p.blocks, p.columns);
  EMBED_LANES(p.lanes, hipLaunchKernelGGL((embed_grad_kernel<T, L>), grid, dim3(256), 0, st, (const T*)g, ldg, width,
                                          ids, entries, perm, off, scale, p.per, part, (T*)out))
  if (p.ranges > 1)
    hipLaunchKernelGGL(embed_join_kernel<T>, dim3((unsigned)(p.ranges - 1), (unsigned)((width + 15) / 16)), dim3(512), 0,
                       st, part, width, ids, entries, perm, off, scale, p.range, (T*)out);
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
  return rows <= kFewRows || p.ranges < 2 ? 0 : p.ranges * 2 * width * (int64_t)sizeof(float);
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
