// Layer norm of rows, forward and backward.
//
//   y = (x - m) r w + b,  m the row's mean, r = 1 / sqrt(mean((x - m)^2) + eps)
//   u = (x - m) r, g = dy w:  dx = r (g - mean(g) - u mean(g u)),  dw = sum over rows of dy u,  db = sum over rows of dy
//
// A row is read once, into registers: 16 bytes a lane and unit, by 16, 32 or 64 lanes (short rows share a wavefront, and need no
// barrier) or by up to 16 wavefronts.  All sums are fp32.  The squares are summed about the mean of what a wavefront holds, and
// wavefronts' means and squares joined as those of parts of a sample, so that a large common offset costs no digits and one barrier
// serves both sums.
#pragma once

#include "row_access.hpp"

namespace flexsae {

constexpr int kNormThreads = 256;  // of a block whose rows share wavefronts
constexpr int kNormMostWaves = 16;

struct NormArgs {
  const void *x, *weight, *bias;  // weight, bias: NULL for none
  const void *dy;
  void *y;  // backward: dx (NULL: not wanted)
  float *mean, *rstd;  // forward: written where not NULL
  float *partial;      // backward: [blocks][2][cols] sums of dy u and dy, or NULL
  int64_t rows, cols, x_stride, dy_stride;
  int64_t per_block;  // forward: rows of a group of lanes, one after another
  float eps;
  int weight_dtype, bias_dtype;
};

// How a block's lanes share rows.  LANES == 0: the block has one row at a time.
template <int LANES>
struct NormShare {
  static constexpr bool kMulti = LANES == 0;
  int lanes, groups, group, me;
  __device__ __forceinline__ NormShare() {
    lanes = kMulti ? static_cast<int>(blockDim.x) : LANES;
    groups = kMulti ? 1 : kNormThreads / (kMulti ? 1 : LANES);
    group = kMulti ? 0 : static_cast<int>(threadIdx.x) / (kMulti ? 1 : LANES);
    me = kMulti ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % (kMulti ? 1 : LANES);
  }
};

// Sum over the lanes of a row of two numbers at once; `turn` alternates between calls of a block (its part of `sh` is read until
// the next barrier).
template <int LANES>
__device__ __forceinline__ float2 row_sums(float a, float b, float2 (*sh)[kNormMostWaves], int turn) {
  if constexpr (LANES != 0) {
    return make_float2(group_sum<LANES>(a), group_sum<LANES>(b));
  } else {
    const float2 mine = make_float2(group_sum<kWave>(a), group_sum<kWave>(b));
    const int waves = static_cast<int>(blockDim.x) / kWave;
    if (waves == 1) return mine;
    if (lane_id() == 0) sh[turn][wave_index()] = mine;
    __syncthreads();
    float2 all = make_float2(0.f, 0.f);
    for (int w = 0; w < waves; ++w) {
      all.x += sh[turn][w].x;
      all.y += sh[turn][w].y;
    }
    return all;
  }
}

// Mean of a row and its mean square about it, from what the wavefronts hold: UNITS units of N elements a lane, of which the first
// `left[u]` are in the row.
template <int LANES, int UNITS, int N>
__device__ __forceinline__ float2 row_moments(const float (&x)[UNITS][N], int64_t cols, const NormShare<LANES> &sh_of,
                                              float2 (*sh)[kNormMostWaves], int turn) {
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) sum += x[u][i];  // (zeros behind the row's end)
  constexpr int kGroup = LANES == 0 ? kWave : LANES;
  sum = group_sum<kGroup>(sum);
  int64_t held = cols;
  if constexpr (LANES == 0) {
    held = 0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t rest = cols - (static_cast<int64_t>(u) * sh_of.lanes + wave_index() * kWave) * N;
      held += rest < 0 ? 0 : rest > kWave * N ? kWave * N : rest;
    }
  }
  const float mean = held > 0 ? sum / static_cast<float>(held) : 0.f;
  float squares = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t left = cols - (static_cast<int64_t>(u) * sh_of.lanes + sh_of.me) * N;
    if (left >= N) {
#pragma unroll
      for (int i = 0; i < N; ++i) squares = fmaf(x[u][i] - mean, x[u][i] - mean, squares);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) squares = fmaf(x[u][i] - mean, x[u][i] - mean, squares);
    }
  }
  squares = group_sum<kGroup>(squares);
  if constexpr (LANES != 0) {
    return make_float2(mean, squares / static_cast<float>(cols));
  } else {
    const int waves = sh_of.lanes / kWave;
    if (waves == 1) return make_float2(mean, squares / static_cast<float>(cols));
    if (lane_id() == 0) sh[turn][wave_index()] = make_float2(mean, squares);
    __syncthreads();
    auto held_by = [&](int w) {
      int64_t n = 0;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int64_t rest = cols - (static_cast<int64_t>(u) * sh_of.lanes + w * kWave) * N;
        n += rest < 0 ? 0 : rest > kWave * N ? kWave * N : rest;
      }
      return static_cast<float>(n);
    };
    float all = 0.f, m2 = 0.f;
    for (int w = 0; w < waves; ++w) all += held_by(w) * sh[turn][w].x;
    all /= static_cast<float>(cols);
    for (int w = 0; w < waves; ++w) {
      const float d = sh[turn][w].x - all;
      m2 += sh[turn][w].y + held_by(w) * d * d;
    }
    return make_float2(all, m2 / static_cast<float>(cols));
  }
}

template <typename T, int LANES, int UNITS>
__global__ __launch_bounds__(LANES == 0 ? 1024 : kNormThreads) void layer_norm_fwd_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const NormShare<LANES> share;
  float w[UNITS][N], b[UNITS][N];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
    if (a.weight) load_typed<N>(a.weight, a.weight_dtype, c, a.cols - c, w[u]);
    if (a.bias) load_typed<N>(a.bias, a.bias_dtype, c, a.cols - c, b[u]);
  }
  for (int64_t i = 0; i < a.per_block; ++i) {
    const int64_t row = (block_index() * a.per_block + i) * share.groups + share.group;
    if (row >= a.rows) return;  // (of all lanes of a row at once)
    const S *const in = static_cast<const S *>(a.x) + row * a.x_stride;
    float x[UNITS][N];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
      unpack<T>(load_upto<T>(in + c, a.cols - c), x[u]);
    }
    const float2 moments = row_moments<LANES, UNITS, N>(x, a.cols, share, sh, static_cast<int>(i & 1));
    const float mean = moments.x, rstd = 1.f / sqrtf(moments.y + a.eps);
    S *const out = static_cast<S *>(a.y) + row * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float v = (x[u][k] - mean) * rstd;
        if (a.weight) v *= w[u][k];
        if (a.bias) v += b[u][k];
        x[u][k] = v;
      }
      store_upto<T>(out + c, pack<T>(x[u]), a.cols - c);
    }
    if (share.me == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

// Rows that no block holds: walked three times, a block a row.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_fwd_long_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const int64_t row = block_index();
  if (row >= a.rows) return;
  const S *const in = static_cast<const S *>(a.x) + row * a.x_stride;
  const int64_t step = static_cast<int64_t>(blockDim.x) * N;
  float x[N], w[N], b[N];
  float sum = 0.f, squares = 0.f;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * N; c < a.cols; c += step) {
    unpack<T>(load_upto<T>(in + c, a.cols - c), x);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += x[i];
  }
  const float mean = row_sums<0>(sum, 0.f, sh, 0).x / static_cast<float>(a.cols);
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * N; c < a.cols; c += step) {
    unpack<T>(load_upto<T>(in + c, a.cols - c), x);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < a.cols) squares = fmaf(x[i] - mean, x[i] - mean, squares);
  }
  const float rstd = 1.f / sqrtf(row_sums<0>(squares, 0.f, sh, 1).x / static_cast<float>(a.cols) + a.eps);
  S *const out = static_cast<S *>(a.y) + row * a.cols;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * N; c < a.cols; c += step) {
    unpack<T>(load_upto<T>(in + c, a.cols - c), x);
    if (a.weight) load_typed<N>(a.weight, a.weight_dtype, c, a.cols - c, w);
    if (a.bias) load_typed<N>(a.bias, a.bias_dtype, c, a.cols - c, b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v = (x[i] - mean) * rstd;
      if (a.weight) v *= w[i];
      if (a.bias) v += b[i];
      x[i] = v;
    }
    store_upto<T>(out + c, pack<T>(x), a.cols - c);
  }
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
}

// Blocks go over the rows, each keeping the column sums of its own in registers, and leave one row of partial sums each.  (Atomics
// into one row of sums would make their order, and so the last bits, a matter of chance.)  Dynamic LDS: 2 groups cols floats where
// groups of lanes share a block.
template <typename T, int LANES, int UNITS>
__global__ __launch_bounds__(LANES == 0 ? 1024 : kNormThreads) void layer_norm_bwd_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const NormShare<LANES> share;
  float w[UNITS][N], dw[UNITS][N], db[UNITS][N];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[u][i] = 1.f;
      dw[u][i] = 0.f;
      db[u][i] = 0.f;
    }
    if (a.weight) load_typed<N>(a.weight, a.weight_dtype, c, a.cols - c, w[u]);
  }
  int turn = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * share.groups;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * share.groups + share.group; row < a.rows; row += step, turn ^= 1) {
    const S *const in = static_cast<const S *>(a.x) + row * a.x_stride;
    const S *const grad = static_cast<const S *>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    words_t xr[UNITS], gr[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
      xr[u] = load_upto<T>(in + c, a.cols - c);
      gr[u] = load_upto<T>(grad + c, a.cols - c);
    }
    float c1 = 0.f, c2 = 0.f;
    float x[UNITS][N], g[UNITS][N];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      unpack<T>(xr[u], x[u]);
      unpack<T>(gr[u], g[u]);
#pragma unroll
      for (int i = 0; i < N; ++i) {  // (behind the row's end all gradients are zeros)
        const float unit = (x[u][i] - mean) * rstd;
        dw[u][i] = fmaf(g[u][i], unit, dw[u][i]);
        db[u][i] += g[u][i];
        g[u][i] *= w[u][i];
        c1 += g[u][i];
        c2 = fmaf(g[u][i], unit, c2);
        x[u][i] = unit;
      }
    }
    if (a.y == nullptr) continue;
    const float2 sums = row_sums<LANES>(c1, c2, sh, turn);
    c1 = sums.x / static_cast<float>(a.cols);
    c2 = sums.y / static_cast<float>(a.cols);
    S *const out = static_cast<S *>(a.y) + row * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] = rstd * (g[u][i] - c1 - x[u][i] * c2);
      store_upto<T>(out + c, pack<T>(x[u]), a.cols - c);
    }
  }
  if (a.partial == nullptr) return;
  float *const out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
  if constexpr (LANES == 0) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < a.cols) {
          out[c + i] = dw[u][i];
          out[a.cols + c + i] = db[u][i];
        }
    }
  } else {
    extern __shared__ float sums[];  // [groups][2][cols]
    float *const mine = sums + static_cast<int64_t>(share.group) * 2 * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t c = (static_cast<int64_t>(u) * share.lanes + share.me) * N;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < a.cols) {
          mine[c + i] = dw[u][i];
          mine[a.cols + c + i] = db[u][i];
        }
    }
    __syncthreads();
    for (int64_t c = threadIdx.x; c < 2 * a.cols; c += kNormThreads) {
      float s = 0.f;
      for (int k = 0; k < share.groups; ++k) s += sums[static_cast<int64_t>(k) * 2 * a.cols + c];
      out[c] = s;
    }
  }
}

// Rows that no block holds: dx by walking the row twice, and the column sums by a kernel of their own.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_bwd_long_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const int64_t row = block_index();
  if (row >= a.rows) return;
  const S *const in = static_cast<const S *>(a.x) + row * a.x_stride;
  const S *const grad = static_cast<const S *>(a.dy) + row * a.dy_stride;
  const float mean = a.mean[row], rstd = a.rstd[row];
  const int64_t step = static_cast<int64_t>(blockDim.x) * N;
  float x[N], g[N], w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = 1.f;
  auto load = [&](int64_t c) {
    unpack<T>(load_upto<T>(in + c, a.cols - c), x);
    unpack<T>(load_upto<T>(grad + c, a.cols - c), g);
    if (a.weight) load_typed<N>(a.weight, a.weight_dtype, c, a.cols - c, w);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = (x[i] - mean) * rstd;
      g[i] *= w[i];
    }
  };
  float c1 = 0.f, c2 = 0.f;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * N; c < a.cols; c += step) {
    load(c);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c1 += g[i];
      c2 = fmaf(g[i], x[i], c2);
    }
  }
  const float2 sums = row_sums<0>(c1, c2, sh, 0);
  c1 = sums.x / static_cast<float>(a.cols);
  c2 = sums.y / static_cast<float>(a.cols);
  S *const out = static_cast<S *>(a.y) + row * a.cols;
  for (int64_t c = static_cast<int64_t>(threadIdx.x) * N; c < a.cols; c += step) {
    load(c);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = rstd * (g[i] - c1 - x[i] * c2);
    store_upto<T>(out + c, pack<T>(x), a.cols - c);
  }
}

// Column sums of the rows b, b + gridDim.y, ... of block (., b); a thread has N columns.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void layer_norm_columns_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x) * N;
  if (c >= a.cols) return;
  float dw[N], db[N];
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float x[N], g[N];
    unpack<T>(load_upto<T>(static_cast<const S *>(a.x) + row * a.x_stride + c, a.cols - c), x);
    unpack<T>(load_upto<T>(static_cast<const S *>(a.dy) + row * a.dy_stride + c, a.cols - c), g);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      dw[i] = fmaf(g[i], (x[i] - mean) * rstd, dw[i]);
      db[i] += g[i];
    }
  }
  float *const out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (c + i < a.cols) {
      out[c + i] = dw[i];
      out[a.cols + c + i] = db[i];
    }
}

// Partial sums [parts][2][cols] to dw and db in their types (NULL: not wanted): a block has 64 columns of one of them, its
// wavefronts every 16th part.
__global__ __launch_bounds__(1024) void layer_norm_finish_kernel(const float *__restrict__ partial, int64_t parts, int64_t cols,
                                                                 void *dw, int dw_dtype, void *db, int db_dtype) {
  __shared__ float sh[kNormMostWaves][kWave];
  void *const out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kWave + lane_id();
  const int wv = wave_index();
  float s = 0.f;
  if (c < cols)
    for (int64_t p = wv; p < parts; p += kNormMostWaves) s += partial[(p * 2 + blockIdx.y) * cols + c];
  sh[wv][lane_id()] = s;
  __syncthreads();
  if (wv != 0 || c >= cols) return;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < kNormMostWaves; ++k) s += sh[k][lane_id()];
  store_typed(out, blockIdx.y == 0 ? dw_dtype : db_dtype, c, s);
}

}  // namespace flexsae
