// Activations to 8 bits and back (codes.h has the format): what a backward pass needs of a row in a byte an element and
// four a block of 128, for 2 to 4 times less memory between the passes.
//
// Both are bound by memory.  A team of lanes has one block, a 16-byte chunk a lane, so that its largest magnitude is
// found in registers, and asks for four blocks before it works on the first.  131,072 x 512 bfloat16: to codes 40 us, back
// 31 us, 5.1 and 6.6 TB/s (the codes are still in the caches).
#include <algorithm>

#include "codes.h"

namespace {

constexpr int kAtOnce = 4;

// Where block b begins: its row, and its first column.
struct Where {
  int64_t row;
  int column;
};

__device__ __forceinline__ Where where(int64_t b, int per) {
  if (per == 1) return {b, 0};
  const int64_t row = b < (int64_t(1) << 32) ? (int64_t)((uint32_t)b / (uint32_t)per) : b / per;
  return {row, (int)(b - row * per) * kCodeBlock};
}

template <typename T, int TEAM>
__global__ __launch_bounds__(256) void encode_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int width,
                                                     int per, int8_t* __restrict__ codes, float* __restrict__ scales) {
  constexpr int V = kChunk<T>, TEAMS = 256 / TEAM;
  const int lane = threadIdx.x % TEAM;
  const int64_t blocks = rows * per;
  for (int64_t b0 = (int64_t)blockIdx.x * TEAMS * kAtOnce + threadIdx.x / TEAM; b0 < blocks;
       b0 += (int64_t)gridDim.x * TEAMS * kAtOnce) {
    u32x4 raw[kAtOnce];
    Where at[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t b = b0 + i * TEAMS;
      at[i] = where(b < blocks ? b : 0, per);
      const int c = at[i].column + lane * V;
      raw[i] = load_raw(x + at[i].row * ldx + c, b < blocks ? width - c : 0);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t b = b0 + i * TEAMS;
      if (b >= blocks) break;
      float v[V];
      widen<T>(raw[i], v);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) top = max(top, magnitude(v[e]));
      const float scale = code_scale(lane_top<TEAM>(top)), inverse = 1.f / scale;
      Codes<V> q;
#pragma unroll
      for (int e = 0; e < V; ++e) q.e[e] = (int8_t)code_of(v[e], inverse);
      const int c = at[i].column + lane * V;
      store_codes<V>(codes + at[i].row * width + c, width - c, q);
      if (lane == 0) scales[b] = scale;
    }
  }
}

template <typename T, int TEAM>
__global__ __launch_bounds__(256) void decode_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                     int64_t rows, int width, int per, T* __restrict__ out) {
  constexpr int V = kChunk<T>, TEAMS = 256 / TEAM;
  const int lane = threadIdx.x % TEAM;
  const int64_t blocks = rows * per;
  for (int64_t b0 = (int64_t)blockIdx.x * TEAMS * kAtOnce + threadIdx.x / TEAM; b0 < blocks;
       b0 += (int64_t)gridDim.x * TEAMS * kAtOnce) {
    Codes<V> q[kAtOnce];
    float scale[kAtOnce];
    Where at[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t b = b0 + i * TEAMS;
      at[i] = where(b < blocks ? b : 0, per);
      const int c = at[i].column + lane * V;
      q[i] = load_codes<V>(codes + at[i].row * width + c, b < blocks ? width - c : 0);
      scale[i] = scales[b < blocks ? b : 0];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (b0 + i * TEAMS >= blocks) break;
      float v[V];
      code_products<V>(q[i].raw, scale[i], v);
      const int c = at[i].column + lane * V;
      store_chunk(out + at[i].row * width + c, width - c, v);
    }
  }
}

// Blocks of a row.  (Of any width that an int holds: a row of 2^31 - 1 elements has 2^24, the last chunk's column is
// below 2^31.)
int blocks_of(int width) { return (width - 1) / kCodeBlock + 1; }

// Lanes of a block's chunks: all of 128 elements, fewer where rows are shorter.
int team_of(int width, int chunk) {
  int lanes = 1;
  while (lanes * chunk < std::min(width, kCodeBlock)) lanes *= 2;
  return lanes;
}

#define CODES_CASE(TEAM_, ...)     \
  case TEAM_: {                    \
    constexpr int TEAM = TEAM_;    \
    __VA_ARGS__;                   \
    break;                         \
  }
#define CODES_TEAMS(n, ...)                                                                                      \
  switch (n) {                                                                                                   \
    CODES_CASE(1, __VA_ARGS__)                                                                                   \
    CODES_CASE(2, __VA_ARGS__)                                                                                   \
    CODES_CASE(4, __VA_ARGS__)                                                                                   \
    CODES_CASE(8, __VA_ARGS__)                                                                                   \
    CODES_CASE(16, __VA_ARGS__)                                                                                  \
    default:                                                                                                     \
      if constexpr (kChunk<T> == 4) {                                                                            \
        constexpr int TEAM = 32;                                                                                 \
        __VA_ARGS__;                                                                                             \
      }                                                                                                          \
  }

dim3 grid_of(int64_t blocks, int team) {
  const int64_t per = 256 / team * kAtOnce;
  return dim3((unsigned)std::min<int64_t>(1 << 20, (blocks + per - 1) / per));
}

template <typename T>
void run_encode(const void* x, int64_t ldx, int64_t rows, int width, int8_t* codes, float* scales, hipStream_t st) {
  const int per = blocks_of(width), team = team_of(width, kChunk<T>);
  CODES_TEAMS(team, hipLaunchKernelGGL((encode_kernel<T, TEAM>), grid_of(rows * per, team), dim3(256), 0, st,
                                       (const T*)x, ldx, rows, width, per, codes, scales))
}

template <typename T>
void run_decode(const int8_t* codes, const float* scales, int64_t rows, int width, void* out, hipStream_t st) {
  const int per = blocks_of(width), team = team_of(width, kChunk<T>);
  CODES_TEAMS(team, hipLaunchKernelGGL((decode_kernel<T, TEAM>), grid_of(rows * per, team), dim3(256), 0, st, codes,
                                       scales, rows, width, per, (T*)out))
}

const char* bad_sizes(int dtype, int64_t rows, int width) {
  if (dtype < ICTC_F32 || dtype > ICTC_F16) return "activations: dtype must be ICTC_F32, ICTC_BF16 or ICTC_F16";
  if (rows < 0 || width < 1) return "activations: rows must not be negative and width at least 1";
  return nullptr;
}

}  // namespace

extern "C" {

int ictc_codes_encode(int dtype, const void* x, int64_t ldx, int64_t rows, int width, int8_t* codes, float* scales,
                      void* stream) {
  if (const char* e = bad_sizes(dtype, rows, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (ldx < width && rows > 1) return dense_fail(ICTC_ERR_ARGUMENT, "activations: row pitch below the width");
  if (rows == 0) return ICTC_OK;
  if (!x || !codes || !scales) return dense_fail(ICTC_ERR_ARGUMENT, "activations: null operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ICTC_F32)
    run_encode<float>(x, ldx, rows, width, codes, scales, st);
  else if (dtype == ICTC_BF16)
    run_encode<bf16>(x, ldx, rows, width, codes, scales, st);
  else
    run_encode<f16>(x, ldx, rows, width, codes, scales, st);
  return dense_status("codes_encode launch");
}

int ictc_codes_decode(int dtype, const int8_t* codes, const float* scales, int64_t rows, int width, void* out,
                      void* stream) {
  if (const char* e = bad_sizes(dtype, rows, width)) return dense_fail(ICTC_ERR_ARGUMENT, e);
  if (rows == 0) return ICTC_OK;
  if (!codes || !scales || !out) return dense_fail(ICTC_ERR_ARGUMENT, "activations: null operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ICTC_F32)
    run_decode<float>(codes, scales, rows, width, out, st);
  else if (dtype == ICTC_BF16)
    run_decode<bf16>(codes, scales, rows, width, out, st);
  else
    run_decode<f16>(codes, scales, rows, width, out, st);
  return dense_status("codes_decode launch");
}

}  // extern "C"
