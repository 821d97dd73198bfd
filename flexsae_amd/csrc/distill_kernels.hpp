// Distillation from a teacher's top logits: the divergence between what the teacher's stored logits t[k] (of vocabulary entries
// i[k]) say among themselves and what a student's row of logits z says of them, and its gradient.
//
//   p = softmax over the stored k of t / T,  q = softmax over the vocabulary of z / T
//   L = T^2 a sum over k of p[k] (log p[k] - log q[i[k]]),   dL / dz[v] = T a (q[v] - sum over k with i[k] = v of p[k])
//
// with a the row's weight, divided by the sum of all where the mean is taken.  A place with an index that is negative or beyond the
// vocabulary holds no logit.  A row of weight zero, or without a stored logit above minus infinity, counts as zero and has a gradient of
// zeros, whatever its logits are.
//
// Three ways.  With the gradient of a mean a row is read once, into the registers of one block (distill_held_kernel): maximum, sum
// and gradient from there.  8192 rows of 131072 bf16: 855 us, 5.0 TB/s of reads and writes where a copy by the library reaches 4.8;
// statistics and gradient by passes of their own take 1440, and one block a row that reads it twice 1270: a second read comes no
// faster from the Infinity Cache.  At this size a block fills its compute unit, whose memory rests while it takes the sum.
// Few long rows, rows that no block holds and losses without a gradient go by parts of rows (121 us for 537 MB), joined by a wavefront a
// row; and gradients for an upstream gradient that the forward did not know by parts of rows again (38 us for 102 MB read and as much
// written), which the gradient that was made with the loss comes on top of: 8192 x 131072 bf16 1805 us for 948.
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
  float4 *stats;             // [rows]: m, s, the teacher's maximum, 1 / sum of its exponentials (0: the row is not used);
                             // [rows]: one over the sum of the weights, in 64 bits
  float *row_loss;           // [rows], times their weights' shares
  float *loss;
  const float *grad;  // upstream gradient: one number, or one of every row; NULL: one
  void *dlogits;
  int *flag;
  int64_t rows, vocab, k, stride, part;  // part: columns of a part of a row, whole units
  int splits, slots;  // slots: of the table of stored entries
  float inv_t, t;
  int top_dtype;
  bool by_row;       // losses of rows, not their mean
  bool skip_if_one;  // dlogits holds the gradient for an upstream gradient of one already
};

// exp(x / T) by the base-2 exponential; c = log2(e) / T.
__device__ __forceinline__ float exp_of(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }

// exp((x - m) / T) of a row.  (Of the difference, which is exact where it matters: one operation less, 2^(c x - c m), would have
// the rounding of c m in every exponent.)
struct RowExp {
  float m, c;
  __device__ __forceinline__ RowExp(float m, float inv_t) : m(m), c(kLog2e * inv_t) {}
  __device__ __forceinline__ float of(float x) const { return exp_of(x - m, c); }
};

// The maximum and sum of two parts.  (A maximum is never minus infinity: it begins as the least finite number.)
__device__ __forceinline__ float2 join(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  return make_float2(m, a.y * exp_of(a.x - m, c) + b.y * exp_of(b.x - m, c));
}

// Takes the elements [from, end) of a row, THREADS units at a time, to `with` (first column, elements, how many of them are in the
// row), with kAhead units of a thread on their way at once.
template <typename T, int THREADS, bool NT, typename F>
__device__ __forceinline__ void walk(const elem_t<T> *in, int64_t from, int64_t end, F with) {
  constexpr int N = kUnitOf<T>, kAhead = 4;
  constexpr int64_t kStep = THREADS * N;
  int64_t at = from + static_cast<int64_t>(threadIdx.x) * N;
  float x[N];
  for (; at + (kAhead - 1) * kStep + N <= end; at += kAhead * kStep) {
    words_t v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = load_words<T, NT>(in + at + u * kStep);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      unpack<T>(v[u], x);
      with(at + u * kStep, x, int64_t{N});
    }
  }
  for (; at < end; at += kStep) {
    unpack<T>(load_upto<T>(in + at, end - at), x);
    with(at, x, end - at);
  }
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
  *reinterpret_cast<double *>(a.stats + a.rows) = s == 0. ? 0. : 1. / s;  // (the mean of no rows is zero)
}

// Weight of a row, and its share of a mean.  (Of weights by 64 bits: their sum, and one over it, may be beyond the normal numbers of
// fp32 where they are not.)
__device__ __forceinline__ float row_weight(const DistillArgs &a, int64_t row) { return a.row_weights ? a.row_weights[row] : 1.f; }
__device__ __forceinline__ float weight_share(const DistillArgs &a, float weight) {
  return a.by_row || !a.row_weights ? weight : static_cast<float>(weight * *reinterpret_cast<const double *>(a.stats + a.rows));
}
// ... times this: where there are no weights the rows share it evenly
__device__ __forceinline__ float mean_factor(const DistillArgs &a) {
  return a.by_row || a.row_weights ? 1.f : 1.f / static_cast<float>(a.rows);
}

// Statistics of a part of a row: block = row * splits + part.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_parts_kernel(const DistillArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  __shared__ float2 sh[kDistillThreads / kWave];
  const int64_t block = block_index(), row = block / a.splits, split = block - row * a.splits;
  if (row >= a.rows || row_weight(a, row) == 0.f) return;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  const int64_t end = (split + 1) * a.part < a.vocab ? (split + 1) * a.part : a.vocab;
  const float c = kLog2e * a.inv_t;
  float2 ms = make_float2(-FLT_MAX, 0.f);
  walk<T, kDistillThreads, true>(in, split * a.part, end, [&](int64_t, float (&x)[N], int64_t left) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= left) x[i] = -INFINITY;
    take<N>(ms, x, c);
  });
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
  using S = elem_t<T>;
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
  a.stats[row] = make_float4(ms.x, ms.y, t.x, used ? 1.f / t.y : 0.f);
  a.row_loss[row] = used ? a.t * a.t * weight_share(a, weight) * loss : 0.f;
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

// For sums of probabilities that no order changes: p 2^up as a whole number.
__device__ __forceinline__ int exponent_of(float p) { return __builtin_amdgcn_frexp_expf(p); }
__device__ __forceinline__ int64_t scaled(float p, int up) { return static_cast<int64_t>(ldexpf(p, up)); }

// The entries of a part of a row that the teacher has stored, each once, with the sum of their places' probabilities, in a table in the
// LDS.  A place finds its entry's slot by a hash where the table has twice as many as there are places; else a slot is an entry, of as many
// entries at a time, and the places are read again for the next ones.  A search of each place among all the others would grow with the
// square of their number (us of a backward, 1000 x 32000 fp16, with it and now: 64 places 61 and 48, 256 179 and 50, 1000 2009 and 68;
// 32000 are 2300).  The sums are those of whole numbers, as many bits of the entry's largest as leave room for all places.
constexpr int64_t kStoredMost = 2048;  // places that a hash finds the slots of
constexpr int kStoredBytes = 16;       // of a slot

// U: of the teacher's logits.  (A type that is known at run time alone is a branch in loops that lanes leave one after another; the
// compiler kept its condition as a mask of the lanes that were left in one of them, and used it for all lanes in the next.)
template <typename U, int THREADS>
struct StoredEntries {
  int *key;         // the entry, or -1
  uint32_t *most;   // bits of the largest
  uint64_t *sum;
  int slots;        // a power of two
  int bits;
  __device__ __forceinline__ StoredEntries(void *lds, int slots, int64_t k)
      : key(reinterpret_cast<int *>(static_cast<uint64_t *>(lds) + slots)), most(reinterpret_cast<uint32_t *>(key + slots)),
        sum(static_cast<uint64_t *>(lds)), slots(slots) {
    const int rest = 31 + __builtin_clz(static_cast<unsigned>(k));  // (fewer than 2^(63 - rest) places)
    bits = rest < 52 ? rest : 52;
  }
  __device__ __forceinline__ int slot_of(int entry, bool hashed, int64_t from) const {
    if (!hashed) {
      const int slot = static_cast<int>(entry - from);
      key[slot] = entry;  // (every place writes the same)
      return slot;
    }
    uint32_t slot = static_cast<uint32_t>(entry) * 2654435761u >> 16;
    for (;; ++slot) {  // (ends: half of the slots stay free)
      slot &= static_cast<uint32_t>(slots) - 1u;
      const int there = atomicCAS(&key[slot], -1, entry);
      if (there == -1 || there == entry) return static_cast<int>(slot);
    }
  }
  // f(entry, probability) for the places of a row whose entries are in [from, end), but for those without a share (of a teacher that
  // has any to give)
  template <typename F>
  __device__ __forceinline__ void places(const DistillArgs &a, int64_t row, int64_t from, int64_t end, float top, F f) const {
    constexpr int kAhead = 4;
    const int64_t *const index = a.index + row * a.k;
    const auto *const logit = static_cast<const elem_t<U> *>(a.top) + row * a.k;
    const float c = kLog2e * a.inv_t;
    for (int64_t k = threadIdx.x; k < a.k; k += kAhead * THREADS) {
      int64_t i[kAhead];
#pragma unroll
      for (int r = 0; r < kAhead; ++r) i[r] = k + r * THREADS < a.k ? index[k + r * THREADS] : -1;
#pragma unroll
      for (int r = 0; r < kAhead; ++r) {
        if (i[r] < from || i[r] >= end) continue;
        const float p = exp_of(Traits<U>::up(logit[k + r * THREADS]) - top, c);
        if (p != 0.f || top == INFINITY) f(static_cast<int>(i[r]), p);
      }
    }
  }
  // By the whole block, behind a barrier where the table was in use.
  __device__ __forceinline__ void gather(const DistillArgs &a, int64_t row, int64_t from, int64_t end, float top, bool hashed) const {
    for (int s = threadIdx.x; s < slots; s += THREADS) {
      key[s] = -1;
      most[s] = 0u;
      sum[s] = 0u;
    }
    __syncthreads();
    places(a, row, from, end, top, [&](int entry, float p) { atomicMax(&most[slot_of(entry, hashed, from)], __float_as_uint(p)); });
    __syncthreads();
    places(a, row, from, end, top, [&](int entry, float p) {
      const int slot = slot_of(entry, hashed, from);
      atomicAdd(reinterpret_cast<unsigned long long *>(&sum[slot]), static_cast<unsigned long long>(scaled(p, up(slot))));
    });
  }
  // f(entry, probability) for the slots in use, behind a barrier.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int s = threadIdx.x; s < slots; s += THREADS)
      if (key[s] >= 0) f(key[s], ldexpf(static_cast<float>(sum[s]), -up(s)));
  }
  __device__ __forceinline__ int up(int slot) const { return bits - exponent_of(__uint_as_float(most[slot])); }
};

// Gradient of a part of a row: block = row * splits + part.
template <typename T, typename U>
__global__ __launch_bounds__(kDistillThreads) void distill_grad_kernel(const DistillArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  if (a.skip_if_one && a.grad[0] == 1.f) return;
  const int64_t block = block_index(), row = block / a.splits, split = block - row * a.splits;
  if (row >= a.rows) return;
  const float4 st = a.stats[row];
  const int64_t from = split * a.part, end = from + a.part < a.vocab ? from + a.part : a.vocab;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  S *const out = static_cast<S *>(a.dlogits) + row * a.vocab;
  const float upstream = a.grad == nullptr ? 1.f : a.grad[a.by_row ? row : 0];
  const float coef = a.t * weight_share(a, row_weight(a, row)) * mean_factor(a) * upstream;
  const bool used = st.w != 0.f;
  if (!used) {
    for (int64_t at = from + static_cast<int64_t>(threadIdx.x) * N; at < end; at += kDistillThreads * N)
      store_upto<T>(out + at, words_t(0u), end - at);
    return;
  }
  extern __shared__ __align__(16) uint64_t table[];
  const StoredEntries<U, kDistillThreads> stored(table, a.slots, a.k);
  const bool hashed = a.k <= kStoredMost;
  if (hashed) stored.gather(a, row, from, end, st.z, true);
  const RowExp e(st.x, a.inv_t);
  const float each = coef / st.y;
  walk<T, kDistillThreads, false>(in, from, end, [&](int64_t at, float (&x)[N], int64_t left) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = each * e.of(x[i]);
    store_upto<T>(out + at, pack<T>(x), left);
  });
  // in the places of gradients without the teacher, which are there behind a barrier
  const auto put = [&](int i, float p) { out[i] = Traits<T>::down(each * e.of(Traits<T>::up(in[i])) - coef * (p * st.w)); };
  if (hashed) {
    __syncthreads();
    stored.each(put);
    return;
  }
  for (int64_t first = from; first < end; first += a.slots) {
    __syncthreads();
    stored.gather(a, row, first, first + a.slots < end ? first + a.slots : end, st.z, false);
    __syncthreads();
    stored.each(put);
  }
}

// ---- a row in the registers of one block ------------------------------------------------------

// Words of minus infinities.
template <typename T>
constexpr uint32_t kMinusInfinities = Traits<T>::dtype == FLEXSAE_F32 ? 0xff800000u : Traits<T>::dtype == FLEXSAE_BF16 ? 0xff80ff80u : 0xfc00fc00u;

// The largest of what a lane has seen, without converting it: 16-bit floats that are not negative are ordered as their bits, and
// negative ones the other way round.  (A NaN that is passed over shows in the sum.)
template <typename T>
struct LargestBits {
  typedef int16_t pair_t __attribute__((ext_vector_type(2)));
  pair_t most = -32768, least = 32767;
  __device__ __forceinline__ void take(words_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pair_t p;
      const uint32_t w = v[i];
      __builtin_memcpy(&p, &w, 4);
      most = __builtin_elementwise_max(most, p);
      least = __builtin_elementwise_min(least, p);
    }
  }
  __device__ __forceinline__ float value() const {
    const int16_t hi = most.x > most.y ? most.x : most.y, lo = least.x < least.y ? least.x : least.y;
    return Traits<T>::up(static_cast<uint16_t>(hi >= 0 ? hi : lo));
  }
};
template <>
struct LargestBits<float> {
  float most = -INFINITY;
  __device__ __forceinline__ void take(words_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) most = fmaxf(most, __uint_as_float(v[i]));
  }
  __device__ __forceinline__ float value() const { return most; }
};

// A row that is not used: a gradient of zeros, and no loss.
template <typename T, int THREADS>
__device__ __forceinline__ void unused_row(const DistillArgs &a, int64_t row) {
  constexpr int N = kUnitOf<T>;
  if (threadIdx.x == 0) {
    a.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    a.row_loss[row] = 0.f;
  }
  elem_t<T> *const out = static_cast<elem_t<T> *>(a.dlogits) + row * a.vocab;
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * N; at < a.vocab; at += THREADS * N) store_upto<T>(out + at, words_t(0u), a.vocab - at);
}

// Loads are unconditional (lanes behind the row's end read its first elements, and put them aside): one that waits for its own
// condition waits for those before it, which made the whole of this kernel 1.2 times as long.  The stored entries are put in their
// places by the threads whose columns they are, so that no barrier waits for the stores; a search for entries that are stored twice, by
// each against all, was 5 us a row.
template <typename T, int THREADS, int UNITS>
__global__ __launch_bounds__(THREADS) void distill_held_kernel(const DistillArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>, kWaves = THREADS / kWave;
  __shared__ float2 maxima[kWaves];  // of logits and teacher
  __shared__ float2 sums[kWaves];    // of both exponentials
  // the teacher's places: entry, exponential, the student's logit; the two logits
  // apart; those of a thread's columns in a chain
  __shared__ int stored[THREADS], chain[THREADS], head[THREADS];
  __shared__ float stored_p[THREADS], stored_z[THREADS], apart[THREADS];
  const int64_t row = block_index();
  if (row >= a.rows) return;
  const float weight = row_weight(a, row);
  if (weight == 0.f) {
    if (static_cast<int64_t>(threadIdx.x) < a.k && a.flag) {
      const int64_t i = a.index[row * a.k + threadIdx.x];
      if (i < -1 || i >= a.vocab) atomicOr(a.flag, FLEXSAE_FLAG_TOKEN_RANGE);
    }
    return unused_row<T, THREADS>(a, row);
  }
  // whole units, and behind them up to N - 1 elements, one of a thread
  const uint32_t cols = static_cast<uint32_t>(a.vocab), whole = cols - cols % N, first = threadIdx.x * N, last = whole + threadIdx.x;
  const S *const in = static_cast<const S *>(a.logits) + row * a.stride;
  S *const out = static_cast<S *>(a.dlogits) + row * a.vocab;
  const int places = static_cast<int>(a.k), k = static_cast<int>(threadIdx.x);
  words_t held[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const uint32_t at = first + u * THREADS * N;
    held[u] = load_words<T>(in + (at < whole ? at : 0u));
  }
  // (behind the row's loads: what waits for these does not hold those up)
  const int64_t place = row * a.k + (k < places ? k : places - 1);
  S last_one = in[last < cols ? last : 0u];
  int64_t index = a.index[place];
  const uint32_t t_bits = load_scalar_bits(a.top, a.top_dtype, place);
  const float tail = last < cols ? Traits<T>::up(last_one) : -INFINITY, t = scalar_from_bits(t_bits, a.top_dtype);
  if (k >= places) index = -1;
  if (index < -1 || index >= a.vocab) {
    if (a.flag) atomicOr(a.flag, FLEXSAE_FLAG_TOKEN_RANGE);
    index = -1;
  }
  const S z_one = in[index < 0 ? 0 : index];
  head[k] = -1;
  stored[k] = static_cast<int>(index);
  float top = wave_max(index < 0 ? -INFINITY : t == t ? t : INFINITY);  // (a NaN makes the row's loss one)
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
    if ((u + 1) * THREADS * N > whole) held[u] = first + u * THREADS * N < whole ? held[u] : words_t(kMinusInfinities<T>);
  LargestBits<T> largest;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) largest.take(held[u]);
  float m = wave_max(fmaxf(largest.value(), tail));
  if (lane_id() == 0) maxima[wave_index()] = make_float2(m, top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    m = fmaxf(m, maxima[w].x);
    top = fmaxf(top, maxima[w].y);
  }
  if (top == -INFINITY) return unused_row<T, THREADS>(a, row);
  const RowExp e(m, a.inv_t);
  const float p = index < 0 ? 0.f : exp_of(t - top, kLog2e * a.inv_t);
  stored_p[k] = p;
  // (a place without a share is left out, but not of a teacher that has none to give, whose shares are all NaN)
  if (index >= 0 && (p != 0.f || top == INFINITY)) {
    chain[k] = atomicExch(&head[static_cast<uint32_t>(index) < whole ? static_cast<uint32_t>(index) / N % THREADS : static_cast<uint32_t>(index) - whole], k);
  }
  float sum = e.of(tail);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float x[N];
    unpack<T>(held[u], x);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += e.of(x[i]);
  }
  // (the compiler would keep the exponentials, which take twice the registers of the row, instead of taking them again)
#pragma unroll
  for (int u = 0; u < UNITS; ++u) asm volatile("" : "+v"(held[u]));
  const float z = Traits<T>::up(z_one);
  stored_z[k] = z;
  apart[k] = ((t - top) - (z - m)) * a.inv_t;
  sum = group_sum<kWave>(sum);
  float sum_top = group_sum<kWave>(p);
  if (lane_id() == 0) sums[wave_index()] = make_float2(sum, sum_top);
  __syncthreads();
  sum = sum_top = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sum += sums[w].x;
    sum_top += sums[w].y;
  }
  const float inv_top = 1.f / sum_top, log_s = logf(sum), share = weight_share(a, weight);
  if (wave_index() == 0) {
    const float logs = logf(sum_top) - log_s;
    float loss = 0.f;
    for (int j = k; j < places; j += kWave)
      if (stored_p[j] != 0.f) loss = fmaf(stored_p[j] * inv_top, apart[j] - logs, loss);
    loss = group_sum<kWave>(loss);
    if (k == 0) {
      a.stats[row] = make_float4(m, sum, top, inv_top);
      a.row_loss[row] = a.t * a.t * share * loss;
    }
  }
  const float coef = a.t * share * mean_factor(a), each = coef / sum;
  auto gradient = [&](float x) { return each * e.of(x); };
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const uint32_t at = first + u * THREADS * N;
    float x[N];
    unpack<T>(held[u], x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = gradient(x[i]);
    store_whole<T>(out + at, pack<T>(x), at < whole);
  }
  if (last < cols) out[last] = Traits<T>::down(gradient(tail));
  // The stored entries among the thread's columns, in whose places the gradients above have been stored by this very thread.  What an
  // entry's places have is summed in 52 bits of the largest of them, exact numbers of which no order changes the sum (the chain's order is
  // that of the exchanges above), and its places leave the chain.
  for (int j = head[k]; j >= 0; j = chain[j]) {
    const int entry = stored[j];
    float all = stored_p[j], most = all;
    bool more = false;
    for (int i = chain[j]; i >= 0; i = chain[i])
      if (stored[i] == entry) {
        most = fmaxf(most, stored_p[i]);
        more = true;
      }
    if (more) {
      const int up = 52 - exponent_of(most);
      int64_t sum_up = scaled(all, up);
      for (int before = j, i = chain[j]; i >= 0; i = chain[i]) {
        if (stored[i] != entry) {
          before = i;
          continue;
        }
        sum_up += scaled(stored_p[i], up);
        chain[before] = chain[i];
      }
      all = ldexpf(static_cast<float>(sum_up), -up);
    }
    out[entry] = Traits<T>::down(gradient(stored_z[j]) - coef * (all * inv_top));
  }
}

}  // namespace flexsae
