// Distillation from a teacher's top logits: the divergence between what the teacher's stored logits t[k] (of vocabulary entries
// i[k]) say among themselves and what a student's row of logits z says of them, and its gradient.
//
//   p = softmax over the stored k of t / T,  q = softmax over the vocabulary of z / T
//   L = T^2 a sum over k of p[k] (log p[k] - log q[i[k]]),   dL / dz[v] = T a (q[v] - sum over k with i[k] = v of p[k])
//
// with a the row's weight, divided by the sum of all where the mean is taken.  A place with an index that is negative or beyond the
// vocabulary holds no logit.  A row of weight zero, or without a stored logit above minus infinity, is not read: it counts as zero
// and has a gradient of zeros.
//
// The row's statistics are its maximum m and s = sum of exp((z - m) / T), in one pass: a running maximum per lane, sums rescaled
// when it moves.  Exponents are of differences from the maximum, so that large logits cost no digits.
#pragma once

#include <float.h>

#include "row_access.hpp"

namespace flexsae {

constexpr int kDistillThreads = 256;
constexpr int kDistillSplits = 64;  // most parts of a row
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  const void *logits, *top;
  const int64_t *index;
  const float *row_weights;  // or NULL
  float2 *parts;             // [rows][splits]: maximum and sum of a part of a row
  float4 *stats;             // [rows]: m, ln s, the teacher's maximum, 1 / sum of its exponentials (0: the row is not used);
                             // [rows].x: one over the sum of the weights
  float *row_loss;           // [rows]
  float *loss;
  const float *grad;  // upstream gradient: one number, or one of every row; NULL: one
  void *dlogits;
  int *flag;
  int64_t rows, vocab, k, stride, part;  // part: columns of a part of a row, whole units
  int splits;
  float inv_t, t;
  int top_dtype;
  bool by_row;       // losses of rows, not their mean
  bool skip_if_one;  // dlogits holds the gradient for an upstream gradient of one already
};

// exp(x / T) by the base-2 exponential; c = log2(e) / T.
__device__ __forceinline__ float exp_of(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }

// The maximum and sum of two parts.  (A maximum is never minus infinity: it begins as the least finite number.)
__device__ __forceinline__ float2 join(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  return make_float2(m, a.y * exp_of(a.x - m, c) + b.y * exp_of(b.x - m, c));
}

template <int N>
__device__ __forceinline__ void take(float2 &ms, const float (&x)[N], float c) {
  float m = ms.x;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  float s = ms.y * exp_of(ms.x - m, c);
#pragma unroll
  for (int i = 0; i < N; ++i) s += exp_of(x[i] - m, c);
  ms = make_float2(m, s);
}

__device__ __forceinline__ float2 wave_join(float2 v, float c) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v = join(v, make_float2(__shfl_xor(v.x, d), __shfl_xor(v.y, d)), c);
  return v;
}

// One over the sum of the rows' weights, for the mean; one block.
__global__ __launch_bounds__(1024) void distill_weights_kernel(const DistillArgs a) {
  __shared__ double sh[1024 / kWave];
  double s = 0.;
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) s += static_cast<double>(a.row_weights[r]);
  s = wave_sum_lane63(s);
  if (lane_id() == kWave - 1) sh[wave_index()] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.;
  for (int w = 0; w < 1024 / kWave; ++w) s += sh[w];
  a.stats[a.rows].x = s == 0. ? 0.f : static_cast<float>(1. / s);  // (the mean of no rows is zero)
}

// Weight of a row with regard to the mean.
__device__ __forceinline__ float row_weight(const DistillArgs &a, int64_t row) { return a.row_weights ? a.row_weights[row] : 1.f; }
__device__ __forceinline__ float mean_factor(const DistillArgs &a) {
  if (a.by_row) return 1.f;
  return a.row_weights ? a.stats[a.rows].x : 1.f / static_cast<float>(a.rows);
}

// Statistics of a part of a row: block = row * splits + part.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_parts_kernel(const DistillArgs a) {
  using S = typename Traits<T>::store_t;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[kDistillThreads / kWave];
  const int64_t block = block_index(), row = block / a.splits, split = block - row * a.splits;
  if (row >= a.rows || row_weight(a, row) == 0.f) return;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  const int64_t end = (split + 1) * a.part < a.vocab ? (split + 1) * a.part : a.vocab;
  const float c = kLog2e * a.inv_t;
  float2 ms = make_float2(-FLT_MAX, 0.f);
  for (int64_t at = split * a.part + static_cast<int64_t>(threadIdx.x) * N; at < end; at += kDistillThreads * N) {
    float x[N];
    const int64_t left = end - at;
    unpack_raw<T, N>(load_upto<T, N>(in + at, left), x);
    if (left < N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i >= left) x[i] = -INFINITY;
    }
    take<N>(ms, x, c);
  }
  ms = wave_join(ms, c);
  if (lane_id() == 0) sh[wave_index()] = ms;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < kDistillThreads / kWave; ++w) ms = join(ms, sh[w], c);
  a.parts[block] = ms;
}

// The teacher's side of a row and its loss, by one wavefront that has the row's statistics; fills stats[row] and the row's loss.
template <typename T>
__device__ __forceinline__ void finish_row(const DistillArgs &a, int64_t row, float2 ms) {
  using S = typename Traits<T>::store_t;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  const int lane = lane_id();
  const float weight = row_weight(a, row);
  float2 t = make_float2(-INFINITY, 0.f);
  const float c = kLog2e * a.inv_t;
  bool beyond = false;
  for (int64_t k = lane; k < a.k; k += kWave) {
    const int64_t i = a.index[row * a.k + k];
    beyond = beyond || i < -1 || i >= a.vocab;
    if (i < 0 || i >= a.vocab) continue;
    const float v = load_scalar(a.top, a.top_dtype, row * a.k + k);
    t.x = v == v ? fmaxf(t.x, v) : INFINITY;  // (a NaN makes the row's loss one)
  }
  if (a.flag && beyond) atomicOr(a.flag, FLEXSAE_FLAG_TOKEN_RANGE);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) t.x = fmaxf(t.x, __shfl_xor(t.x, d));
  const bool used = weight != 0.f && t.x != -INFINITY;
  float loss = 0.f, log_s = 0.f, log_t = 0.f;
  if (used) {
    for (int64_t k = lane; k < a.k; k += kWave) {
      const int64_t i = a.index[row * a.k + k];
      if (i >= 0 && i < a.vocab) t.y += exp_of(load_scalar(a.top, a.top_dtype, row * a.k + k) - t.x, c);
    }
    t.y = group_sum<kWave>(t.y);
    log_t = logf(t.y);
    log_s = logf(ms.y);
    for (int64_t k = lane; k < a.k; k += kWave) {
      const int64_t i = a.index[row * a.k + k];
      if (i < 0 || i >= a.vocab) continue;
      const float d = load_scalar(a.top, a.top_dtype, row * a.k + k) - t.x;
      const float p = exp_of(d, c) / t.y;
      if (p == 0.f) continue;
      const float e = Traits<T>::up(in[i]) - ms.x;
      loss = fmaf(p, (d - e) * a.inv_t - (log_t - log_s), loss);
    }
    loss = group_sum<kWave>(loss);
  }
  if (lane != 0) return;
  a.stats[row] = make_float4(ms.x, log_s, t.x, used ? 1.f / t.y : 0.f);
  a.row_loss[row] = used ? a.t * a.t * weight * loss : 0.f;
}

// Rows whose parts are there: a wavefront a row.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_rows_kernel(const DistillArgs a) {
  const int64_t row = block_index() * (kDistillThreads / kWave) + wave_index();
  if (row >= a.rows) return;
  const float c = kLog2e * a.inv_t;
  float2 ms = make_float2(-FLT_MAX, 0.f);
  if (row_weight(a, row) != 0.f && lane_id() < a.splits) ms = a.parts[row * a.splits + lane_id()];
  finish_row<T>(a, row, wave_join(ms, c));
}

// The rows' losses to their mean; one block.
__global__ __launch_bounds__(1024) void distill_mean_kernel(const DistillArgs a) {
  __shared__ double sh[1024 / kWave];
  double s = 0.;
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) s += static_cast<double>(a.row_loss[r]);
  s = wave_sum_lane63(s);
  if (lane_id() == kWave - 1) sh[wave_index()] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.;
  for (int w = 0; w < 1024 / kWave; ++w) s += sh[w];
  a.loss[0] = static_cast<float>(s * static_cast<double>(mean_factor(a)));
}

// The entries of a part of a row that the teacher has stored: gradients in the place of those that `dlogits` holds without the
// teacher.  Run by the whole block, behind a barrier.  An entry that is stored twice is written by the first of its places.
template <typename T, int THREADS>
__device__ __forceinline__ void stored_entries(const DistillArgs &a, int64_t row, int64_t from, int64_t end, float4 st, float coef) {
  using S = typename Traits<T>::store_t;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  S *const out = static_cast<S *>(a.dlogits) + row * a.vocab;
  const int64_t *const index = a.index + row * a.k;
  const float c = kLog2e * a.inv_t;
  for (int64_t k = threadIdx.x; k < a.k; k += THREADS) {
    const int64_t i = index[k];
    if (i < from || i >= end) continue;
    float p = 0.f;
    bool first = true;
    for (int64_t j = 0; j < a.k && first; ++j) {
      if (index[j] != i) continue;
      first = j >= k;
      p += exp_of(load_scalar(a.top, a.top_dtype, row * a.k + j) - st.z, c) * st.w;
    }
    if (!first) continue;
    const float q = __builtin_amdgcn_exp2f((Traits<T>::up(in[i]) - st.x) * c - st.y * kLog2e);
    out[i] = Traits<T>::down(coef * (q - p));
  }
}

// Gradient of a part of a row: block = row * splits + part.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_grad_kernel(const DistillArgs a) {
  using S = typename Traits<T>::store_t;
  constexpr int N = kUnitOf<T>;
  if (a.skip_if_one && a.grad[0] == 1.f) return;
  const int64_t block = block_index(), row = block / a.splits, split = block - row * a.splits;
  if (row >= a.rows) return;
  const float4 st = a.stats[row];
  const int64_t from = split * a.part, end = from + a.part < a.vocab ? from + a.part : a.vocab;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  S *const out = static_cast<S *>(a.dlogits) + row * a.vocab;
  const float upstream = a.grad == nullptr ? 1.f : a.grad[a.by_row ? row : 0];
  const float coef = a.t * row_weight(a, row) * mean_factor(a) * upstream;
  const bool used = st.w != 0.f;
  const float c = kLog2e * a.inv_t, shift = st.y * kLog2e;
  for (int64_t at = from + static_cast<int64_t>(threadIdx.x) * N; at < end; at += kDistillThreads * N) {
    float x[N];
    const int64_t left = end - at;
    if (used) {
      unpack_raw<T, N>(load_upto<T, N>(in + at, left), x);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = coef * __builtin_amdgcn_exp2f((x[i] - st.x) * c - shift);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = 0.f;
    }
    store_upto<T, N>(out + at, pack<T, N>(x), left);
  }
  if (!used) return;
  __syncthreads();
  stored_entries<T, kDistillThreads>(a, row, from, end, st, coef);
}

}  // namespace flexsae
