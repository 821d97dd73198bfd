// Rows of a table by token, scaled, and their gradients.
//
//   out[n] = f s[n] W[token[n]];   dW[v] = f sum over n with token[n] = v of s[n] dout[n];   ds[n] = f <dout[n], W[token[n]]>
//
// A token that is negative or no row of the table gives zeros and takes no part in the gradients (its row of dout is not read).
//
// The gradient of the table goes by the sorted places of the tokens (the losses' pair list, one pair a row): every row of dW is
// written once, by the lanes that add up its places in their order, so that the bits are the same on every run; rows without a
// token get zeros in the same pass.  A frequent token would be one long walk: tokens with more than kLookupChunk places are added
// up in pieces first, those that fall into the aligned stretches of kLookupChunk sorted places, by blocks that know nothing but
// their stretch.  A stretch that holds pieces of two such tokens holds the end of one and the beginning of the other.
#pragma once

#include "row_access.hpp"

namespace flexsae {

constexpr int kLookupThreads = 256;
constexpr int kLookupChunk = 64;

struct LookupArgs {
  const int64_t *tokens;
  const void *weight, *scale;  // scale: NULL for none
  const void *dout;
  void *out;  // backward: dW
  const uint32_t *begin, *map;  // of the sorted places
  float *pieces;      // [chunks][2][columns of whole tiles]: the end of a token that began before the stretch, and the beginning of one that ends behind it
  float *dots;        // [n][tiles] shares of ds, or NULL
  void *dscale;
  int *flag;
  int64_t n, vocab, cols, weight_stride, dout_stride;
  int64_t tiles;  // of a row: LANES * UNITS units of 16 bytes each
  float factor;
  int scale_dtype;
};

// Row of the table, or -1.
__device__ __forceinline__ int64_t row_of(int64_t token, int64_t vocab) { return token >= 0 && token < vocab ? token : -1; }

// What a group of lanes works on: item (a row of out, a row of dW, a stretch) and tile of the row.
template <typename T, int LANES, int UNITS>
struct LookupPlace {
  static constexpr int N = kUnitOf<T>;
  int64_t item, tile, first;  // first: the lane's first column; unit u begins LANES * N columns further on
  __device__ __forceinline__ explicit LookupPlace(int64_t tiles) {
    const int64_t task = block_index() * (kLookupThreads / LANES) +
                         (LANES == kWave ? wave_index() : static_cast<int>(threadIdx.x) / LANES);
    item = task / tiles;
    tile = task - item * tiles;
    first = tile * (LANES * UNITS * N) + (static_cast<int>(threadIdx.x) % LANES) * N;
  }
  // columns of whole tiles, which rows of fp32 sums have
  __device__ __forceinline__ int64_t width(int64_t tiles) const { return tiles * (LANES * UNITS * N); }
  __device__ __forceinline__ int64_t column(int u) const { return first + static_cast<int64_t>(u) * LANES * N; }
};

template <typename T, int LANES, int UNITS>
__global__ __launch_bounds__(kLookupThreads) void lookup_fwd_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS> at(a.tiles);
  if (at.item >= a.n) return;
  const int64_t token = a.tokens[at.item], row = row_of(token, a.vocab);
  if (a.flag && at.first == 0 && (token < -1 || token >= a.vocab)) atomicOr(a.flag, FLEXSAE_FLAG_TOKEN_RANGE);
  S *const out = static_cast<S *>(a.out) + at.item * a.cols;
  words_t v[UNITS];
  if (row < 0) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      v[u] = 0;
      store_upto<T>(out + at.column(u), v[u], a.cols - at.column(u));
    }
    return;
  }
  const S *const in = static_cast<const S *>(a.weight) + row * a.weight_stride;
  const float scale = a.scale ? a.factor * load_scalar(a.scale, a.scale_dtype, at.item) : a.factor;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) v[u] = load_upto<T>(in + at.column(u), a.cols - at.column(u));
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (scale != 1.f) {
      float x[N];
      unpack<T>(v[u], x);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] *= scale;
      v[u] = pack<T>(x);
    }
    store_upto<T>(out + at.column(u), v[u], a.cols - at.column(u));
  }
}

// Adds the rows of dout at sorted places [from, to), all of one token, to `sum`; W: the token's row (used with dots).
// `here`: whether place 0 of the list may hold tokens that are no row (they are filed under row 0).
template <typename T, int LANES, int UNITS, bool DOTS>
__device__ __forceinline__ void add_places(const LookupArgs &a, const LookupPlace<T, LANES, UNITS> &at, uint32_t from, uint32_t to,
                                           bool check, const float (&w)[UNITS][kUnitOf<T>], float (&sum)[UNITS][kUnitOf<T>]) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  for (uint32_t p = from; p < to; ++p) {
    const int64_t n = a.map[p];
    if (check && row_of(a.tokens[n], a.vocab) < 0) continue;
    const S *const in = static_cast<const S *>(a.dout) + n * a.dout_stride;
    const float scale = a.scale ? a.factor * load_scalar(a.scale, a.scale_dtype, n) : a.factor;
    float dot = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      float x[N];
      unpack<T>(load_upto<T>(in + at.column(u), a.cols - at.column(u)), x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sum[u][i] = fmaf(scale, x[i], sum[u][i]);
        if constexpr (DOTS) dot = fmaf(x[i], w[u][i], dot);
      }
    }
    if constexpr (DOTS) {
      dot = group_sum<LANES>(dot);
      if (static_cast<int>(threadIdx.x) % LANES == 0) a.dots[n * a.tiles + at.tile] = dot;
    }
  }
}

template <typename T, int LANES, int UNITS>
__device__ __forceinline__ void load_row(const LookupArgs &a, const LookupPlace<T, LANES, UNITS> &at, int64_t row,
                                         float (&w)[UNITS][kUnitOf<T>]) {
  constexpr int N = kUnitOf<T>;
  const auto *const in = static_cast<const typename Traits<T>::store_t *>(a.weight) + row * a.weight_stride;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) unpack<T>(load_upto<T>(in + at.column(u), a.cols - at.column(u)), w[u]);
}

template <int UNITS, int N>
__device__ __forceinline__ void clear(float (&x)[UNITS][N]) {
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) x[u][i] = 0.f;
}

// The pieces of frequent tokens in a stretch of kLookupChunk sorted places.
template <typename T, int LANES, int UNITS, bool DOTS>
__global__ __launch_bounds__(kLookupThreads) void lookup_pieces_kernel(const LookupArgs a) {
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS> at(a.tiles);
  const int64_t from = at.item * kLookupChunk;
  if (from >= a.n) return;
  const uint32_t lo = static_cast<uint32_t>(from);
  const uint32_t hi = static_cast<uint32_t>(from + kLookupChunk < a.n ? from + kLookupChunk : a.n);
  auto token_at = [&](uint32_t p) {
    const int64_t row = row_of(a.tokens[a.map[p]], a.vocab);
    return row < 0 ? 0 : row;
  };
  auto add = [&](int64_t token, uint32_t b, uint32_t e, int which) {
    float w[UNITS][N], sum[UNITS][N];
    clear(sum);
    if constexpr (DOTS) load_row(a, at, token, w);
    add_places<T, LANES, UNITS, DOTS>(a, at, b > lo ? b : lo, e < hi ? e : hi, token == 0, w, sum);
    float *const out = a.pieces + (at.item * 2 + which) * at.width(a.tiles);
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int h = 0; h < N; h += 4) *reinterpret_cast<float4 *>(out + at.column(u) + h) = make_float4(sum[u][h], sum[u][h + 1], sum[u][h + 2], sum[u][h + 3]);
  };
  const int64_t first = token_at(lo), last = token_at(hi - 1);
  const uint32_t first_begin = a.begin[first], first_end = a.begin[first + 1];
  if (first_end - first_begin > kLookupChunk) add(first, first_begin, first_end, first_begin > lo);
  if (last == first) return;
  const uint32_t last_begin = a.begin[last], last_end = a.begin[last + 1];
  if (last_end - last_begin > kLookupChunk) add(last, last_begin, last_end, last_begin > lo);
}

template <typename T, int LANES, int UNITS, bool DOTS>
__global__ __launch_bounds__(kLookupThreads) void lookup_bwd_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS> at(a.tiles);
  if (at.item >= a.vocab) return;
  const uint32_t from = a.begin ? a.begin[at.item] : 0u, to = a.begin ? a.begin[at.item + 1] : 0u;
  float sum[UNITS][N];
  clear(sum);
  if (to - from > kLookupChunk) {
    for (uint32_t chunk = from / kLookupChunk; chunk <= (to - 1) / kLookupChunk; ++chunk) {
      const int which = from > chunk * kLookupChunk;
      const float *const piece = a.pieces + (static_cast<int64_t>(chunk) * 2 + which) * at.width(a.tiles);
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int h = 0; h < N; h += 4) {
          const float4 x = *reinterpret_cast<const float4 *>(piece + at.column(u) + h);
          sum[u][h] += x.x;
          sum[u][h + 1] += x.y;
          sum[u][h + 2] += x.z;
          sum[u][h + 3] += x.w;
        }
    }
  } else if (to > from) {
    float w[UNITS][N];
    if constexpr (DOTS) load_row(a, at, at.item, w);
    add_places<T, LANES, UNITS, DOTS>(a, at, from, to, at.item == 0, w, sum);
  }
  S *const out = static_cast<S *>(a.out) + at.item * a.cols;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) store_upto<T>(out + at.column(u), pack<T>(sum[u]), a.cols - at.column(u));
}

// Shares of ds by rows of dout, where no gradient of the table is wanted.
template <typename T, int LANES, int UNITS>
__global__ __launch_bounds__(kLookupThreads) void lookup_dots_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS> at(a.tiles);
  if (at.item >= a.n) return;
  const int64_t row = row_of(a.tokens[at.item], a.vocab);
  if (row < 0) return;
  const S *const in = static_cast<const S *>(a.weight) + row * a.weight_stride;
  const S *const grad = static_cast<const S *>(a.dout) + at.item * a.dout_stride;
  float dot = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float x[N], g[N];
    unpack<T>(load_upto<T>(in + at.column(u), a.cols - at.column(u)), x);
    unpack<T>(load_upto<T>(grad + at.column(u), a.cols - at.column(u)), g);
#pragma unroll
    for (int i = 0; i < N; ++i) dot = fmaf(x[i], g[i], dot);
  }
  dot = group_sum<LANES>(dot);
  if (static_cast<int>(threadIdx.x) % LANES == 0) a.dots[at.item * a.tiles + at.tile] = dot;
}

__global__ __launch_bounds__(kLookupThreads) void lookup_dscale_kernel(const LookupArgs a) {
  const int64_t n = block_index() * kLookupThreads + threadIdx.x;
  if (n >= a.n) return;
  float s = 0.f;
  if (row_of(a.tokens[n], a.vocab) >= 0)
    for (int64_t t = 0; t < a.tiles; ++t) s += a.dots[n * a.tiles + t];
  store_typed(a.dscale, a.scale_dtype, n, a.factor * s);
}

}  // namespace flexsae
