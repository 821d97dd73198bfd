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
// their stretch (64 places: 131072 tokens whose frequencies fall as one over their rank have two fifths of them there).  A stretch that
// holds pieces of two such tokens holds the end of one and the beginning of the other.  Tokens that are no row are filed under row 0,
// whose walk passes over them (half of 131072 tokens: the backward of 65536 x 2048 bf16 194 us without them, 291 with).
#pragma once

#include <type_traits>

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

// What a group of lanes works on: item (a row of out, a row of dW, a stretch) and tile of the row.  WHOLE: rows have N elements and
// more; where one ends inside a lane's unit, the lane has its last N elements instead, some of which the lane before has too (both
// compute and store the same), so that every access is a whole one.  Else a row is a part of one unit.
template <typename T, int LANES, int UNITS, bool WHOLE>
struct LookupPlace {
  static constexpr int N = kUnitOf<T>;
  int64_t item, tile, cols;
  int64_t column[UNITS];  // first of the unit's
  bool there[UNITS];      // any of it in the row
  int again[UNITS];       // elements that the lane before has too
  __device__ __forceinline__ LookupPlace(int64_t tiles, int64_t cols) : cols(cols) {
    // (fewer than 2^32 of them: a division of 64-bit numbers is longer than the rest of a row without a token)
    const uint32_t task = static_cast<uint32_t>(block_index()) * (kLookupThreads / LANES) +
                          static_cast<uint32_t>(LANES == kWave ? wave_index() : static_cast<int>(threadIdx.x) / LANES);
    const uint32_t per = static_cast<uint32_t>(tiles), quotient = task / per;
    item = quotient;
    tile = task - quotient * per;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int64_t at = (tile * UNITS + u) * (LANES * N) + (static_cast<int>(threadIdx.x) % LANES) * N;
      there[u] = at < cols;
      column[u] = !WHOLE ? at : at >= cols ? 0 : at + N > cols ? cols - N : at;
      again[u] = there[u] ? static_cast<int>(at - column[u]) : N;
    }
  }
  __device__ __forceinline__ words_t load(const elem_t<T> *row, int u) const {
    if constexpr (WHOLE) return load_words<T>(row + column[u]);
    else return load_upto<T>(row + column[u], cols - column[u]);
  }
  __device__ __forceinline__ void store(elem_t<T> *row, int u, words_t v) const {
    if constexpr (WHOLE) store_whole<T, true>(row + column[u], v, there[u]);
    else store_upto<T>(row + column[u], v, cols - column[u]);
  }
  // Sum of products, each element once.
  __device__ __forceinline__ float dot(int u, const float (&x)[N], const float (&y)[N]) const {
    float s = 0.f;
    if (again[u] == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(x[i], y[i], s);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) s = i < again[u] ? s : fmaf(x[i], y[i], s);
    }
    return s;
  }
  // fp32 sums of whole tiles
  __device__ __forceinline__ int64_t width(int64_t tiles) const { return tiles * (LANES * UNITS * N); }
  __device__ __forceinline__ int64_t sums(int u) const {
    return (tile * UNITS + u) * (LANES * N) + (static_cast<int>(threadIdx.x) % LANES) * N;
  }
};

// The value of a lane of the group.
template <int LANES>
__device__ __forceinline__ int of_lane(int v, int lane) {
  if constexpr (LANES == kWave) return __builtin_amdgcn_readlane(v, lane);
  else return __shfl(v, lane, LANES);
}
template <int LANES>
__device__ __forceinline__ float of_lane(float v, int lane) { return __int_as_float(of_lane<LANES>(__float_as_int(v), lane)); }

// ROWS consecutive tokens of a group of lanes, on their way together: a wavefront that waits for one token and then for its row leaves
// memory idle twice (us of 131072 rows of 262144 x 4096 bf16: 350 with one row, 293 with four, 266 with streaming stores).
template <typename T, int LANES, int UNITS, bool WHOLE, int ROWS>
__global__ __launch_bounds__(kLookupThreads) void lookup_fwd_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS, WHOLE> at(a.tiles, a.cols);
  const int64_t first = at.item * ROWS;
  if (first >= a.n) return;
  int64_t row[ROWS];
  float scale[ROWS];
  words_t v[ROWS][UNITS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t i = first + r < a.n ? first + r : first, token = a.tokens[i];
    row[r] = row_of(token, a.vocab);
    scale[r] = a.scale ? a.factor * load_scalar(a.scale, a.scale_dtype, i) : a.factor;
    if (a.flag && at.tile == 0 && static_cast<int>(threadIdx.x) % LANES == 0 && (token < -1 || token >= a.vocab))
      atomicOr(a.flag, FLEXSAE_FLAG_TOKEN_RANGE);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const S *const in = static_cast<const S *>(a.weight) + (row[r] < 0 ? 0 : row[r]) * a.weight_stride;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) v[r][u] = at.load(in, u);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (first + r >= a.n) return;
    S *const out = static_cast<S *>(a.out) + (first + r) * a.cols;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (row[r] < 0) {
        v[r][u] = 0u;
      } else if (scale[r] != 1.f) {
        float x[N];
        unpack<T>(v[r][u], x);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= scale[r];
        v[r][u] = pack<T>(x);
      }
      at.store(out, u, v[r][u]);
    }
  }
}

// Brings the places of tokens that are rows, among the group's `count`, to its first lanes, in their order; -> how many there are.
template <int LANES>
__device__ __forceinline__ int rows_first(const LookupArgs &a, int count, uint32_t &place) {
  const int me = static_cast<int>(threadIdx.x) % LANES, first = lane_id() - me;
  const bool there = me < count && row_of(a.tokens[place], a.vocab) >= 0;
  const uint64_t group = (__ballot(there) >> first) & (LANES == kWave ? ~uint64_t{0} : (uint64_t{1} << LANES) - 1);
  const int kept = __popcll(group), before = __popcll(group & ((uint64_t{1} << me) - 1));
  const int to = there ? before : kept + me - before;
  place = static_cast<uint32_t>(__builtin_amdgcn_ds_permute((first + to) * 4, static_cast<int>(place)));
  return kept;
}

// Adds the rows of dout at sorted places [from, to), all of one token, to `sum`; w: the token's row (used with dots).  check: the
// places may be of tokens that are no row (they are filed under row 0), whose rows of dout are not read.  Places and scales of LANES
// tokens are read at once, a lane each, and AHEAD rows are on their way together: a walk that waits for each place and then for its row
// takes 3 latencies a row.
template <typename T, int LANES, int UNITS, bool WHOLE, bool DOTS, int AHEAD>
__device__ __forceinline__ void add_places(const LookupArgs &a, const LookupPlace<T, LANES, UNITS, WHOLE> &at, uint32_t from, uint32_t to,
                                           bool check, const float (&w)[UNITS][kUnitOf<T>], float (&sum)[UNITS][kUnitOf<T>]) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const int me = static_cast<int>(threadIdx.x) % LANES;
  for (uint32_t base = from; base < to; base += LANES) {
    int count = static_cast<int>(to - base < LANES ? to - base : LANES);
    uint32_t n_mine = a.map[base + (me < count ? me : 0)];
    if (check) count = rows_first<LANES>(a, count, n_mine);
    const float scale_mine = a.scale ? a.factor * load_scalar(a.scale, a.scale_dtype, n_mine) : a.factor;
    auto together = [&](auto ahead, int j) {
      constexpr int A = decltype(ahead)::value;
      words_t v[A][UNITS];
      uint32_t n[A];
      float scale[A];
#pragma unroll
      for (int r = 0; r < A; ++r) {
        const int lane = j + r < count ? j + r : j;  // (a row that is there stands in for one behind the last)
        n[r] = static_cast<uint32_t>(of_lane<LANES>(static_cast<int>(n_mine), lane));
        scale[r] = of_lane<LANES>(scale_mine, lane);
        const S *const in = static_cast<const S *>(a.dout) + n[r] * a.dout_stride;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) v[r][u] = at.load(in, u);
      }
#pragma unroll
      for (int r = 0; r < A; ++r) {
        if (A != AHEAD && j + r >= count) continue;
        float dot = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          float x[N];
          unpack<T>(v[r][u], x);
#pragma unroll
          for (int i = 0; i < N; ++i) sum[u][i] = fmaf(scale[r], x[i], sum[u][i]);
          if constexpr (DOTS) dot += at.dot(u, x, w[u]);
        }
        if constexpr (DOTS) {
          dot = group_sum<LANES>(dot);
          if (me == 0) a.dots[static_cast<int64_t>(n[r]) * a.tiles + at.tile] = dot;
        }
      }
    };
    int j = 0;
    for (; j + AHEAD <= count; j += AHEAD) together(std::integral_constant<int, AHEAD>(), j);
    for (; j < count; j += 2) together(std::integral_constant<int, 2>(), j);
  }
}

template <typename T, int LANES, int UNITS, bool WHOLE>
__device__ __forceinline__ void load_row(const LookupArgs &a, const LookupPlace<T, LANES, UNITS, WHOLE> &at, int64_t row,
                                         float (&w)[UNITS][kUnitOf<T>]) {
  const auto *const in = static_cast<const elem_t<T> *>(a.weight) + row * a.weight_stride;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) unpack<T>(at.load(in, u), w[u]);
}

template <int UNITS, int N>
__device__ __forceinline__ void clear(float (&x)[UNITS][N]) {
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) x[u][i] = 0.f;
}

// The pieces of frequent tokens in a stretch of kLookupChunk sorted places.
template <typename T, int LANES, int UNITS, bool WHOLE, bool DOTS>
__global__ __launch_bounds__(kLookupThreads) void lookup_pieces_kernel(const LookupArgs a) {
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS, WHOLE> at(a.tiles, a.cols);
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
    add_places<T, LANES, UNITS, WHOLE, DOTS, 8>(a, at, b > lo ? b : lo, e < hi ? e : hi, token == 0, w, sum);
    float *const out = a.pieces + (at.item * 2 + which) * at.width(a.tiles);
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int h = 0; h < N; h += 4) *reinterpret_cast<float4 *>(out + at.sums(u) + h) = make_float4(sum[u][h], sum[u][h + 1], sum[u][h + 2], sum[u][h + 3]);
  };
  const int64_t first = token_at(lo), last = token_at(hi - 1);
  const uint32_t first_begin = a.begin[first], first_end = a.begin[first + 1];
  if (first_end - first_begin > kLookupChunk) add(first, first_begin, first_end, first_begin > lo);
  if (last == first) return;
  const uint32_t last_begin = a.begin[last], last_end = a.begin[last + 1];
  if (last_end - last_begin > kLookupChunk) add(last, last_begin, last_end, last_begin > lo);
}

// ROWS consecutive rows of dW of a group of lanes: where most tokens do not occur, a row is two numbers to wait for and a store.
template <typename T, int LANES, int UNITS, bool WHOLE, bool DOTS, int ROWS>
__global__ __launch_bounds__(kLookupThreads) void lookup_bwd_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS, WHOLE> at(a.tiles, a.cols);
  const int64_t first = at.item * ROWS;
  if (first >= a.vocab) return;
  uint32_t begin[ROWS + 1];
#pragma unroll
  for (int r = 0; r <= ROWS; ++r) begin[r] = a.begin ? a.begin[first + r < a.vocab ? first + r : a.vocab] : 0u;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t row = first + r;
    if (row >= a.vocab) return;
    const uint32_t from = begin[r], to = begin[r + 1];
    S *const out = static_cast<S *>(a.out) + row * a.cols;
    if (to == from) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) at.store(out, u, words_t(0u));
      continue;
    }
    float sum[UNITS][N];
    clear(sum);
    if (to - from > kLookupChunk) {
#pragma unroll 4
      for (uint32_t chunk = from / kLookupChunk; chunk <= (to - 1) / kLookupChunk; ++chunk) {
        const int which = from > chunk * kLookupChunk;
        const float *const piece = a.pieces + (static_cast<int64_t>(chunk) * 2 + which) * at.width(a.tiles);
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
          for (int h = 0; h < N; h += 4) {
            const float4 x = *reinterpret_cast<const float4 *>(piece + at.sums(u) + h);
            sum[u][h] += x.x;
            sum[u][h + 1] += x.y;
            sum[u][h + 2] += x.z;
            sum[u][h + 3] += x.w;
          }
      }
    } else {
      float w[UNITS][N];
      if constexpr (DOTS) load_row(a, at, row, w);
      add_places<T, LANES, UNITS, WHOLE, DOTS, 4>(a, at, from, to, row == 0, w, sum);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) at.store(out, u, pack<T>(sum[u]));
  }
}

// Shares of ds by rows of dout, where no gradient of the table is wanted.
template <typename T, int LANES, int UNITS, bool WHOLE>
__global__ __launch_bounds__(kLookupThreads) void lookup_dots_kernel(const LookupArgs a) {
  using S = elem_t<T>;
  constexpr int N = kUnitOf<T>;
  const LookupPlace<T, LANES, UNITS, WHOLE> at(a.tiles, a.cols);
  if (at.item >= a.n) return;
  const int64_t row = row_of(a.tokens[at.item], a.vocab);
  if (row < 0) return;
  const S *const grad = static_cast<const S *>(a.dout) + at.item * a.dout_stride;
  float w[UNITS][N], dot = 0.f;
  words_t v[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) v[u] = at.load(grad, u);
  load_row(a, at, row, w);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float g[N];
    unpack<T>(v[u], g);
    dot += at.dot(u, g, w[u]);
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
