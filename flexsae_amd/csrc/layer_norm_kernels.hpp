// Layer norm of rows, forward and backward.
//
//   y = (x - m) r w + b,  m the row's mean, r = 1 / sqrt(mean((x - m)^2) + eps)
//   u = (x - m) r, g = dy w:  dx = r (g - mean(g) - u mean(g u)),  dw = sum over rows of dy u,  db = sum over rows of dy
//
// A row is read once, into registers: 16 bytes a lane and unit, by 16, 32 or 64 lanes (short rows share a wavefront, and need no
// barrier) or by up to 16 wavefronts.  All sums are fp32.  The squares are summed about the mean of what a wavefront holds, and
// wavefronts' means and squares joined as those of parts of a sample, so that a large common offset costs no digits and one barrier
// serves both sums.
//
// Memory bounds it: 16384 x 8192 bf16 forward 86 us (6.2 TB/s), 65536 x 2304 forward 115 us (5.2) and backward 172 us (5.3), each one call
// after another, where a lane has less of a row to keep on its way.  (A trace of single kernels says 132 and 185 + 5: there each waits for
// its last stores.)  What that took (us of the last forward, traced): weight and bias once for several rows, whose next one is on its way
// while a row is worked on, 304 to 194; the wavefronts' sums by one read of the LDS, not one after another, to 158; sixteen elements a
// lane instead of eight, to 142.
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

// A lane's units of a row.  WHOLE: rows have N elements and more; where one ends inside a unit, the lane has its last N elements
// instead, the first `again` of which the lane before has too: both compute and store the same, and sums leave them out.  Else a row
// is a part of one unit.
template <typename T, int UNITS, bool WHOLE>
struct RowUnits {
  static constexpr int N = kUnitOf<T>;
  int cols, column[UNITS], again[UNITS];
  __device__ __forceinline__ RowUnits(int me, int lanes, int64_t row_cols) : cols(static_cast<int>(row_cols)) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = (u * lanes + me) * N;
      column[u] = !WHOLE ? at : at >= cols ? 0 : at + N > cols ? cols - N : at;
      again[u] = at >= cols ? N : at - column[u];
    }
  }
  __device__ __forceinline__ words_t load(const elem_t<T> *row, int u) const {
    if constexpr (WHOLE) return load_words<T, true>(row + column[u]);
    else return load_upto<T>(row + column[u], cols - column[u]);
  }
  __device__ __forceinline__ void store(elem_t<T> *row, int u, words_t v) const {
    if constexpr (WHOLE) store_whole<T, true>(row + column[u], v, again[u] < N);
    else store_upto<T>(row + column[u], v, cols - column[u]);
  }
  // f(i) for each element of unit u that is in the row and that no other lane has
  template <typename F>
  __device__ __forceinline__ void once(int u, F f) const {
    if (WHOLE && again[u] == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) f(i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (WHOLE ? i >= again[u] : column[u] + i < cols) f(i);
    }
  }
  // the same of all elements that are in the row
  template <typename F>
  __device__ __forceinline__ void each(int u, F f) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (WHOLE ? again[u] < N : column[u] + i < cols) f(i);
  }
  __device__ __forceinline__ void typed(const void *base, int dtype, int u, float (&o)[N]) const {
    load_typed<N>(base, dtype, column[u], WHOLE ? N : cols - column[u], o);
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
    // (a wavefront's sums in a lane of each 16, and one read of the LDS instead of one after another)
    const int w = lane_id() % kNormMostWaves;
    const float2 theirs = w < waves ? sh[turn][w] : make_float2(0.f, 0.f);
    return make_float2(group_sum<kNormMostWaves>(theirs.x), group_sum<kNormMostWaves>(theirs.y));
  }
}

// Mean of a row and its mean square about it, from what the wavefronts hold.
template <typename T, int LANES, int UNITS, bool WHOLE>
__device__ __forceinline__ float2 row_moments(const float (&x)[UNITS][kUnitOf<T>], const RowUnits<T, UNITS, WHOLE> &units,
                                              const NormShare<LANES> &share, float2 (*sh)[kNormMostWaves], int turn) {
  constexpr int kGroup = LANES == 0 ? kWave : LANES, kSpan = kWave * kUnitOf<T>;
  const int cols = units.cols;
  float sum = 0.f, squares = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) units.once(u, [&](int i) { sum += x[u][i]; });
  sum = group_sum<kGroup>(sum);
  auto held_by = [&](int wave) {  // elements
    int n = 0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int rest = cols - (u * share.lanes + wave * kWave) * kUnitOf<T>;
      n += rest < 0 ? 0 : rest > kSpan ? kSpan : rest;
    }
    return static_cast<float>(n);
  };
  const float held = LANES == 0 ? held_by(wave_index()) : static_cast<float>(cols);
  const float mean = held > 0.f ? sum / held : 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) units.once(u, [&](int i) { squares = fmaf(x[u][i] - mean, x[u][i] - mean, squares); });
  squares = group_sum<kGroup>(squares);
  const int waves = LANES == 0 ? share.lanes / kWave : 1;
  if (waves == 1) return make_float2(mean, squares / static_cast<float>(cols));
  if (lane_id() == 0) sh[turn][wave_index()] = make_float2(mean, squares);
  __syncthreads();
  // (as in row_sums)
  const int w = lane_id() % kNormMostWaves;
  const float2 theirs = w < waves ? sh[turn][w] : make_float2(0.f, 0.f);
  const float n = w < waves ? held_by(w) : 0.f;
  const float all = group_sum<kNormMostWaves>(n * theirs.x) / static_cast<float>(cols), d = theirs.x - all;
  return make_float2(all, group_sum<kNormMostWaves>(theirs.y + n * d * d) / static_cast<float>(cols));
}

// Consecutive rows by a group of lanes, the next one's elements on their way while a row is worked on; weight and bias stay in
// registers.
template <typename T, int LANES, int UNITS, bool WHOLE>
__global__ __launch_bounds__(LANES == 0 ? 1024 : kNormThreads) void layer_norm_fwd_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const NormShare<LANES> share;
  const RowUnits<T, UNITS, WHOLE> units(share.me, share.lanes, a.cols);
  const int64_t first = block_index() * a.per_block * share.groups + share.group;
  if (first >= a.rows) return;  // (of all lanes of a row at once)
  auto source = [&](int64_t row) { return static_cast<const S *>(a.x) + (row < a.rows ? row : first) * a.x_stride; };
  words_t raw[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) raw[u] = units.load(source(first), u);
  float w[UNITS][N], b[UNITS][N];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (a.weight) units.typed(a.weight, a.weight_dtype, u, w[u]);
    if (a.bias) units.typed(a.bias, a.bias_dtype, u, b[u]);
  }
  for (int64_t i = 0; i < a.per_block; ++i) {
    const int64_t row = first + i * share.groups;
    if (row >= a.rows) return;
    float x[UNITS][N];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) unpack<T>(raw[u], x[u]);
    if (i + 1 < a.per_block) {
      const S *const in = source(row + share.groups);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) raw[u] = units.load(in, u);
    }
    const float2 moments = row_moments<T, LANES>(x, units, share, sh, static_cast<int>(i & 1));
    const float mean = moments.x, rstd = 1.f / sqrtf(moments.y + a.eps);
    S *const out = static_cast<S *>(a.y) + row * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float v = (x[u][k] - mean) * rstd;
        if (a.weight) v *= w[u][k];
        if (a.bias) v += b[u][k];
        x[u][k] = v;
      }
      units.store(out, u, pack<T>(x[u]));
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
template <typename T, int LANES, int UNITS, bool WHOLE>
__global__ __launch_bounds__(LANES == 0 ? 1024 : kNormThreads) void layer_norm_bwd_kernel(const NormArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[2][kNormMostWaves];
  const NormShare<LANES> share;
  const RowUnits<T, UNITS, WHOLE> units(share.me, share.lanes, a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * share.groups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * share.groups + share.group;
  words_t xr[UNITS], gr[UNITS];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t r) {
    r = r < a.rows ? r : 0;
    const S *const in = static_cast<const S *>(a.x) + r * a.x_stride;
    const S *const grad = static_cast<const S *>(a.dy) + r * a.dy_stride;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      xr[u] = units.load(in, u);
      gr[u] = units.load(grad, u);
    }
    mean = a.mean[r];
    rstd = a.rstd[r];
  };
  load(row);
  float w[UNITS][N], dw[UNITS][N], db[UNITS][N];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[u][i] = 1.f;
      dw[u][i] = 0.f;
      db[u][i] = 0.f;
    }
    if (a.weight) units.typed(a.weight, a.weight_dtype, u, w[u]);
  }
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    float c1 = 0.f, c2 = 0.f;
    float x[UNITS][N], g[UNITS][N];
    const float r = rstd;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      unpack<T>(xr[u], x[u]);
      unpack<T>(gr[u], g[u]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float unit = (x[u][i] - mean) * r;
        dw[u][i] = fmaf(g[u][i], unit, dw[u][i]);
        db[u][i] += g[u][i];
        g[u][i] *= w[u][i];
        x[u][i] = unit;
      }
      units.once(u, [&](int i) {
        c1 += g[u][i];
        c2 = fmaf(g[u][i], x[u][i], c2);
      });
    }
    load(row + step);
    if (a.y == nullptr) continue;
    const float2 sums = row_sums<LANES>(c1, c2, sh, turn);
    c1 = sums.x / static_cast<float>(a.cols);
    c2 = sums.y / static_cast<float>(a.cols);
    S *const out = static_cast<S *>(a.y) + row * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] = r * (g[u][i] - c1 - x[u][i] * c2);
      units.store(out, u, pack<T>(x[u]));
    }
  }
  if (a.partial == nullptr) return;
  float *const out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
  auto put = [&](float *to) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      units.each(u, [&](int i) {
        to[units.column[u] + i] = dw[u][i];
        to[a.cols + units.column[u] + i] = db[u][i];
      });
  };
  if constexpr (LANES == 0) {
    put(out);
  } else {
    extern __shared__ float sums[];  // [groups][2][cols]
    put(sums + static_cast<int64_t>(share.group) * 2 * a.cols);
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
#pragma unroll 8
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
