// AdamW over many tensors in one launch, with states in 32 bits or in 8, on tensors as they are stored or on rows that are
// held at length one; the gradients' global norm; the values of 8-bit states.
//
// With c the factor of the gradient (inverse loss scale, clipping) and t the number of this step:
//   g <- c g;  unit rows: g <- g - (<g,w> / <w,w>) w
//   m <- b1 m + (1-b1) g,  v <- b2 v + (1-b2) g^2
//   w <- (1 - lr wd) w - lr / (1-b1^t) * m / (sqrt(v) / sqrt(1-b2^t) + eps);  unit rows: w <- w / |w|
//
// 8-bit states: blocks of 256 consecutive elements (of a row, where rows have length one; the last block of a tensor or row may
// be shorter) with two 32-bit maxima, of |m| and of v.  Of the two bytes of an element the first, c, stands for
// sign(c-128) ((c-128)/127)^2 a_m and the second for (c/255)^4 a_v: square-root codes of m and of sqrt(v).  Elements of a block
// differ by orders of magnitude (a power of four spans 2e-10 to 1), and a uniform decay is carried by the maxima alone and
// leaves the codes as they are.  A v above zero gets at least code 1, so that no m is divided by a v that was lost.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace flexsae {

constexpr int kAdamwThreads = 256;
constexpr int kAdamwLane = 8;                              // consecutive elements of a lane
constexpr int kAdamwTile = kAdamwThreads * kAdamwLane;     // of a block at a time
constexpr int kAdamwQuant = 256;                           // elements that share the maxima of 8-bit states
constexpr int kAdamwTensors = 48;                          // of one launch: the table travels in the kernel's arguments (4 KiB)
constexpr int kNormTensors = 128;

struct AdamwTensor {
  void *param;
  const void *grad;
  void *s0, *s1;  // exp_avg, exp_avg_sq; or codes, maxima
  float *master;  // (NULL: none)
  int64_t rows, cols;
  float lr, weight_decay;
  int32_t dtype;
};

struct AdamwTable {
  AdamwTensor tensor[kAdamwTensors];
  uint32_t first[kAdamwTensors + 1];  // tile (unit rows: group of rows) at which each tensor begins; the number of them
  int32_t count;
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, inv_scale, max_norm;
  int32_t last;  // the call's last launch: counts the step
  double log_beta1, log_beta2;
  const float *grad_norm, *lr;  // device (NULL: none)
  int64_t *counter;             // device: steps taken; blocks of this launch that have ended
};
static_assert(sizeof(AdamwTable) <= 4096, "kernel arguments");

struct AdamwCoefs {
  float b1, omb1, b2, omb2, eps, grad, inv_bc1, inv_sqrt_bc2, lr;
  bool go;
};

__device__ __forceinline__ AdamwCoefs adamw_coefs(const AdamwTable &a) {
  AdamwCoefs c;
  const double t = static_cast<double>(a.counter[0] + 1);
  c.b1 = a.beta1;
  c.omb1 = a.one_minus_beta1;
  c.b2 = a.beta2;
  c.omb2 = a.one_minus_beta2;
  c.eps = a.eps;
  c.grad = a.inv_scale;
  c.go = true;
  if (a.grad_norm) {
    const float norm = *a.grad_norm;
    c.go = __builtin_isfinite(norm);
    if (a.max_norm > 0.f) c.grad *= fminf(1.f, a.max_norm / (norm * a.inv_scale + 1e-6f));
  }
  // 1 - b^t without cancellation
  c.inv_bc1 = -1.f / expm1f(static_cast<float>(t * a.log_beta1));
  c.inv_sqrt_bc2 = 1.f / sqrtf(-expm1f(static_cast<float>(t * a.log_beta2)));
  c.lr = a.lr ? *a.lr : 1.f;
  c.inv_bc1 *= c.lr;
  return c;
}

// The last block of the call's last launch counts the step: by then every block has read the number of steps.
__device__ __forceinline__ void adamw_count(const AdamwTable &a) {
  if (!a.last) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long *ended = reinterpret_cast<unsigned long long *>(a.counter + 1);
    if (atomicAdd(ended, 1ull) + 1 == gridDim.x) {
      atomicExch(ended, 0ull);
      a.counter[0] += 1;
    }
  }
}

// The tensor of a tile: the largest i with first[i] <= tile (tensors without tiles are not in the table).
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table &a, uint32_t tile) {
  int i = 0;
#pragma unroll
  for (int s = 64; s > 0; s >>= 1)
    if (i + s < a.count && tile >= a.first[i + s]) i += s;
  return i;
}

// Sixteen bytes through memory that is aligned to ALIGN (2 or 4: to the elements; rows and views start anywhere).
typedef uint32_t words_at4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t words_at2_t __attribute__((ext_vector_type(4), aligned(2)));
template <int ALIGN>
__device__ __forceinline__ void load16(const void *p, uint32_t *w) {
  vec_t<uint32_t, 4> x;
  if constexpr (ALIGN == 4) x = __builtin_nontemporal_load(static_cast<const words_at4_t *>(p));
  else x = __builtin_nontemporal_load(static_cast<const words_at2_t *>(p));
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = x[k];
}
template <int ALIGN>
__device__ __forceinline__ void store16(void *p, const uint32_t *w) {
  const vec_t<uint32_t, 4> x = {w[0], w[1], w[2], w[3]};
  if constexpr (ALIGN == 4) __builtin_nontemporal_store(x, static_cast<words_at4_t *>(p));
  else __builtin_nontemporal_store(x, static_cast<words_at2_t *>(p));
}

// Eight elements as stored.
template <typename T>
struct Raw8 {
  static constexpr int kWords = 2 * static_cast<int>(sizeof(typename Traits<T>::store_t));
  uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ void load8(const void *base, int64_t at, int left, Raw8<T> &r) {
  using S = typename Traits<T>::store_t;
  const S *p = static_cast<const S *>(base) + at;
  if (left >= kAdamwLane) {
#pragma unroll
    for (int j = 0; j < Raw8<T>::kWords; j += 4) load16<sizeof(S)>(reinterpret_cast<const char *>(p) + 4 * j, r.w + j);
  } else {
    S x[kAdamwLane];
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j) x[j] = j < left ? p[j] : S{};
    __builtin_memcpy(r.w, x, sizeof(x));
  }
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, float (&o)[kAdamwLane]) {
  if constexpr (Traits<T>::dtype == FLEXSAE_F32) {
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j) o[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j) o[j] = Traits<T>::up(static_cast<uint16_t>(r.w[j / 2] >> (16 * (j % 2))));
  }
}

template <typename T>
__device__ __forceinline__ void store8(void *base, int64_t at, int left, const float (&x)[kAdamwLane]) {
  using S = typename Traits<T>::store_t;
  S *p = static_cast<S *>(base) + at;
  if (left >= kAdamwLane) {
    uint32_t w[Raw8<T>::kWords];
#pragma unroll
    for (int j = 0; j < Raw8<T>::kWords; ++j) {
      if constexpr (Traits<T>::dtype == FLEXSAE_F32) w[j] = __float_as_uint(x[j]);
      else if constexpr (Traits<T>::dtype == FLEXSAE_BF16) w[j] = f32x2_to_bf16x2_bits(x[2 * j], x[2 * j + 1]);
      else w[j] = static_cast<uint32_t>(f32_to_f16_bits(x[2 * j])) | (static_cast<uint32_t>(f32_to_f16_bits(x[2 * j + 1])) << 16);
    }
#pragma unroll
    for (int j = 0; j < Raw8<T>::kWords; j += 4) store16<sizeof(S)>(reinterpret_cast<char *>(p) + 4 * j, w + j);
  } else {
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j)
      if (j < left) p[j] = Traits<T>::down(x[j]);
  }
}

// ---- 8-bit states --------------------------------------------------------------------------
// Sixteen bytes: (code of m, code of v) of eight elements.
struct Codes8 {
  uint32_t w[4];
};

__device__ __forceinline__ void load_codes(const void *base, int64_t at, int left, Codes8 &c) {
  const uint16_t *p = static_cast<const uint16_t *>(base) + at;
  if (left >= kAdamwLane) {
    load16<2>(p, c.w);
  } else {
    uint16_t x[kAdamwLane];
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j) x[j] = j < left ? p[j] : uint16_t{128};
    __builtin_memcpy(c.w, x, sizeof(x));
  }
}

__device__ __forceinline__ void store_codes(void *base, int64_t at, int left, const Codes8 &c) {
  uint16_t *p = static_cast<uint16_t *>(base) + at;
  if (left >= kAdamwLane) {
    store16<2>(p, c.w);
  } else {
#pragma unroll
    for (int j = 0; j < kAdamwLane; ++j)
      if (j < left) p[j] = static_cast<uint16_t>(c.w[j / 2] >> (16 * (j % 2)));
  }
}

__device__ __forceinline__ void decode8(const Codes8 &c, float a_m, float a_v, float (&m)[kAdamwLane], float (&v)[kAdamwLane]) {
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) {
    const uint32_t pair = c.w[j / 2] >> (16 * (j % 2));
    // (the squares of codes are exact; what follows is a rounding each, and none is raised to a power but that of 1 / 255^2)
    const float x = static_cast<float>(pair & 0xffu) - 128.f;
    m[j] = x * fabsf(x) * (1.f / (127.f * 127.f)) * a_m;
    float y = static_cast<float>((pair >> 8) & 0xffu);
    y = y * y * (1.f / (255.f * 255.f));
    v[j] = y * y * a_v;
  }
}

// The largest of the 32 lanes of each half of the wavefront.  As whole numbers: the bits of non-negative floats are in their
// order, infinity and NaN above all.
__device__ __forceinline__ uint32_t half_wave_max(uint32_t x) {
  auto move = [](uint32_t y, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(y), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = max(x, move(x, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
  x = max(x, move(x, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
  x = max(x, move(x, std::integral_constant<int, 0x141>{}));  // the other quad of each 8
  x = max(x, move(x, std::integral_constant<int, 0x140>{}));  // the other half of each 16-lane row
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false);  // the other row of each two
  return max(r[0], r[1]);
}

// What a maximum is kept as: zero below the smallest normal number (its inverse would overflow), NaN where the block has
// infinities or NaN.
__device__ __forceinline__ float kept_max(uint32_t bits) {
  return bits < 0x00800000u ? 0.f : bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(bits);
}

__device__ __forceinline__ void maxima8(const float (&m)[kAdamwLane], const float (&v)[kAdamwLane], float &a_m, float &a_v) {
  uint32_t bm = 0, bv = 0;
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) {
    bm = max(bm, __float_as_uint(m[j]) & 0x7fffffffu);
    bv = max(bv, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  a_m = kept_max(half_wave_max(bm));
  a_v = kept_max(half_wave_max(bv));
}

__device__ __forceinline__ void encode8(const float (&m)[kAdamwLane], const float (&v)[kAdamwLane], float a_m, float a_v, Codes8 &c) {
  const float per_m = a_m > 0.f ? 1.f / a_m : 0.f, per_v = a_v > 0.f ? 1.f / a_v : 0.f;
#pragma unroll
  for (int j = 0; j < kAdamwLane / 2; ++j) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // (the hardware's square root, one unit in the last place: which of two codes a value between them gets)
      const float x = __builtin_amdgcn_sqrtf(fabsf(m[2 * j + k]) * per_m);
      const uint32_t cm = static_cast<uint32_t>(fmaf(copysignf(x, m[2 * j + k]), 127.f, 128.5f));
      const float part = v[2 * j + k] * per_v;
      const float y = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(part));
      const uint32_t cv = max(static_cast<uint32_t>(fmaf(y, 255.f, 0.5f)), part > 0.f ? 1u : 0u);
      w |= (cm | (cv << 8)) << (16 * k);
    }
    c.w[j] = w;
  }
}

// ---- the step ------------------------------------------------------------------------------
__device__ __forceinline__ void adamw_moments(const AdamwCoefs &c, const float (&g)[kAdamwLane], float (&m)[kAdamwLane],
                                              float (&v)[kAdamwLane]) {
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) {
    m[j] = fmaf(c.b1, m[j], c.omb1 * g[j]);
    v[j] = fmaf(c.b2, v[j], c.omb2 * g[j] * g[j]);
  }
}

__device__ __forceinline__ void adamw_move(const AdamwCoefs &c, float step, float keep, const float (&m)[kAdamwLane],
                                           const float (&v)[kAdamwLane], float (&w)[kAdamwLane]) {
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) {
    const float by = m[j] / fmaf(sqrtf(v[j]), c.inv_sqrt_bc2, c.eps);
    w[j] = fmaf(-step, by, keep * w[j]);
  }
}

// A lane's eight elements of the tensors that a step works on: as loaded, and as numbers.
template <typename T, bool MASTER, bool EIGHT>
struct AdamwLane {
  using W = std::conditional_t<MASTER, float, T>;
  Raw8<T> rg;
  Raw8<W> rw;
  Raw8<float> rm, rv;  // states in 32 bits,
  Codes8 codes;        // in 8
  float2 top;
  int64_t at, block;
  int left;

  // elements [at, at + 8) of a tensor, of which `left` (at most 8) exist; block: that of their 8-bit states
  __device__ __forceinline__ void load(const AdamwTensor &t, int64_t at_, int64_t rest, int64_t block_) {
    at = at_;
    block = block_;
    left = rest > kAdamwLane ? kAdamwLane : rest < 0 ? 0 : static_cast<int>(rest);
    load8<T>(t.grad, at, left, rg);
    load8<W>(MASTER ? t.master : t.param, at, left, rw);
    if constexpr (EIGHT) {
      load_codes(t.s0, at, left, codes);
      top = left > 0 ? static_cast<const float2 *>(t.s1)[block] : float2{0.f, 0.f};
    } else {
      load8<float>(t.s0, at, left, rm);
      load8<float>(t.s1, at, left, rv);
    }
  }

  // m, v from g and what they were; stored; w moved
  __device__ __forceinline__ void step(const AdamwTensor &t, const AdamwCoefs &c, const float (&g)[kAdamwLane],
                                       float (&w)[kAdamwLane], bool store) {
    float m[kAdamwLane], v[kAdamwLane];
    if constexpr (EIGHT) {
      decode8(codes, top.x, top.y, m, v);
    } else {
      unpack8(rm, m);
      unpack8(rv, v);
    }
    adamw_moments(c, g, m, v);
    adamw_move(c, t.lr * c.inv_bc1, 1.f - t.lr * c.lr * t.weight_decay, m, v, w);
    if (!store) return;
    if constexpr (EIGHT) {
      float a_m, a_v;
      maxima8(m, v, a_m, a_v);
      Codes8 now;
      encode8(m, v, a_m, a_v, now);
      store_codes(t.s0, at, left, now);
      if (left > 0 && (threadIdx.x & 31) == 0) static_cast<float2 *>(t.s1)[block] = float2{a_m, a_v};
    } else {
      store8<float>(t.s0, at, left, m);
      store8<float>(t.s1, at, left, v);
    }
  }

  __device__ __forceinline__ void store(const AdamwTensor &t, const float (&w)[kAdamwLane]) const {
    store8<T>(t.param, at, left, w);
    if constexpr (MASTER) store8<float>(t.master, at, left, w);
  }
};

template <typename T, bool MASTER, bool EIGHT>
__device__ __forceinline__ void adamw_tile(const AdamwTensor &t, int64_t base, const AdamwCoefs &c) {
  const int64_t at = base + static_cast<int64_t>(threadIdx.x) * kAdamwLane;
  AdamwLane<T, MASTER, EIGHT> lane;
  lane.load(t, at, t.cols - at, at / kAdamwQuant);
  float g[kAdamwLane], w[kAdamwLane];
  unpack8(lane.rg, g);
  unpack8(lane.rw, w);
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) g[j] *= c.grad;
  lane.step(t, c, g, w, true);
  lane.store(t, w);
}

template <bool EIGHT>
__global__ __launch_bounds__(kAdamwThreads) void adamw_kernel(const AdamwTable a) {
  const AdamwCoefs c = adamw_coefs(a);
  if (!c.go) return;
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const AdamwTensor &t = a.tensor[i];
    const int64_t base = static_cast<int64_t>(tile - a.first[i]) * kAdamwTile;
    if (t.dtype == FLEXSAE_F32) adamw_tile<float, false, EIGHT>(t, base, c);
    else if (t.dtype == FLEXSAE_BF16) t.master ? adamw_tile<bf16_t, true, EIGHT>(t, base, c) : adamw_tile<bf16_t, false, EIGHT>(t, base, c);
    else t.master ? adamw_tile<f16_t, true, EIGHT>(t, base, c) : adamw_tile<f16_t, false, EIGHT>(t, base, c);
  }
  adamw_count(a);
}

// Sums over the WAVES wavefronts of a row; `turn` alternates between two places so that one barrier a sum is enough.
template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float (*place)[16], int turn) {
  x = wave_sum_bcast(x);
  if constexpr (WAVES > 1) {
    if (lane_id() == 0) place[turn][wave_in_block()] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += place[turn][i];
  }
  return x;
}

// Rows of length one.  WAVES wavefronts hold a row, SEGMENTS stretches of 512 elements each, in registers: every tensor is
// read and written once.  SEGMENTS = 0: a row of any length is walked three times (the two products; the length of the moved
// row; the step), nothing stored before the last walk.
template <typename T, bool MASTER, bool EIGHT, int WAVES, int SEGMENTS>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * kWave) void adamw_rows_kernel(const AdamwTable a) {
  constexpr int kRows = WAVES < 4 ? 4 / WAVES : 1;  // of a block at a time
  constexpr int kSegment = kWave * kAdamwLane;
  __shared__ float place[2][16];
  const AdamwCoefs c = adamw_coefs(a);
  if (!c.go) return;
  const int wave = wave_in_block() % WAVES;
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const AdamwTensor &t = a.tensor[i];
    const int64_t row = static_cast<int64_t>(tile - a.first[i]) * kRows + wave_in_block() / WAVES;
    if (row >= t.rows) continue;  // (of a whole wavefront: a block of several rows has no barriers)
    const int64_t start = row * t.cols, blocks = (t.cols + kAdamwQuant - 1) / kAdamwQuant;
    auto load = [&](AdamwLane<T, MASTER, EIGHT> &lane, int64_t s) {
      const int64_t col = (s * WAVES + wave) * kSegment + lane_id() * kAdamwLane;
      lane.load(t, start + col, t.cols - col, row * blocks + col / kAdamwQuant);
    };
    auto products = [&](const AdamwLane<T, MASTER, EIGHT> &lane, float (&g)[kAdamwLane], float (&w)[kAdamwLane], float &gw, float &ww) {
      unpack8(lane.rg, g);
      unpack8(lane.rw, w);
#pragma unroll
      for (int j = 0; j < kAdamwLane; ++j) {
        g[j] *= c.grad;
        gw = fmaf(g[j], w[j], gw);
        ww = fmaf(w[j], w[j], ww);
      }
    };
    auto across = [&](float along, float (&g)[kAdamwLane], const float (&w)[kAdamwLane]) {
#pragma unroll
      for (int j = 0; j < kAdamwLane; ++j) g[j] = fmaf(-along, w[j], g[j]);
    };
    auto squares = [&](const float (&w)[kAdamwLane], float &s) {
#pragma unroll
      for (int j = 0; j < kAdamwLane; ++j) s = fmaf(w[j], w[j], s);
    };
    auto scaled = [&](float by, float (&w)[kAdamwLane]) {
#pragma unroll
      for (int j = 0; j < kAdamwLane; ++j) w[j] *= by;
    };
    float gw = 0.f, ww = 0.f, nn = 0.f;
    if constexpr (SEGMENTS > 0) {
      AdamwLane<T, MASTER, EIGHT> lane[SEGMENTS];
      float g[SEGMENTS][kAdamwLane], w[SEGMENTS][kAdamwLane];
#pragma unroll
      for (int s = 0; s < SEGMENTS; ++s) load(lane[s], s);
#pragma unroll
      for (int s = 0; s < SEGMENTS; ++s) products(lane[s], g[s], w[s], gw, ww);
      gw = row_sum<WAVES>(gw, place, 0);
      ww = row_sum<WAVES>(ww, place, 1);
      const float along = ww > 0.f ? gw / ww : 0.f;
#pragma unroll
      for (int s = 0; s < SEGMENTS; ++s) {
        across(along, g[s], w[s]);
        lane[s].step(t, c, g[s], w[s], true);
        squares(w[s], nn);
      }
      nn = row_sum<WAVES>(nn, place, 0);
      const float by = nn > 0.f ? 1.f / sqrtf(nn) : 1.f;
#pragma unroll
      for (int s = 0; s < SEGMENTS; ++s) {
        scaled(by, w[s]);
        lane[s].store(t, w[s]);
      }
    } else {
      const int64_t segments = (t.cols + WAVES * kSegment - 1) / (WAVES * kSegment);
      AdamwLane<T, MASTER, EIGHT> lane;
      float g[kAdamwLane], w[kAdamwLane];
      for (int64_t s = 0; s < segments; ++s) {
        load(lane, s);
        products(lane, g, w, gw, ww);
      }
      gw = row_sum<WAVES>(gw, place, 0);
      ww = row_sum<WAVES>(ww, place, 1);
      const float along = ww > 0.f ? gw / ww : 0.f;
      float unused_gw = 0.f, unused_ww = 0.f;
      for (int64_t s = 0; s < segments; ++s) {
        load(lane, s);
        products(lane, g, w, unused_gw, unused_ww);
        across(along, g, w);
        lane.step(t, c, g, w, false);
        squares(w, nn);
      }
      nn = row_sum<WAVES>(nn, place, 0);
      const float by = nn > 0.f ? 1.f / sqrtf(nn) : 1.f;
      for (int64_t s = 0; s < segments; ++s) {
        load(lane, s);
        products(lane, g, w, unused_gw, unused_ww);
        across(along, g, w);
        lane.step(t, c, g, w, true);
        scaled(by, w);
        lane.store(t, w);
      }
    }
    // (the next row's first sum may write place[0] while a wavefront still reads it for this one's length)
    if constexpr (WAVES > 1) __syncthreads();
  }
  adamw_count(a);
}

// ---- the gradients' norm -------------------------------------------------------------------
struct NormTensor {
  const void *grad;
  int64_t n;
  int32_t dtype;
};
// (No table here has an array of bytes beside its wider ones: an index that addresses both lets the compiler take the address of
// a wider entry apart as base + i and 7 i, and scalar loads drop the two low bits of each part.)
struct NormTable {
  NormTensor tensor[kNormTensors];
  uint32_t first[kNormTensors + 1];
  int32_t count;
  double *partial;  // one of each block
};
static_assert(sizeof(NormTable) <= 4096, "kernel arguments");

// Squares are summed in 64 bits: those of finite 32-bit numbers neither overflow nor vanish there, and the order of the sum,
// which is the same on every run, hardly matters.
template <typename T>
__device__ __forceinline__ double squares_of_tile(const void *grad, int64_t n, int64_t base) {
  double sum = 0.0;
  const int64_t at = base + static_cast<int64_t>(threadIdx.x) * kAdamwLane;
  const int64_t rest = n - at;
  Raw8<T> r;
  load8<T>(grad, at, rest > kAdamwLane ? kAdamwLane : rest < 0 ? 0 : static_cast<int>(rest), r);
  float x[kAdamwLane];
  unpack8(r, x);
#pragma unroll
  for (int j = 0; j < kAdamwLane; ++j) sum = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
  return sum;
}

// The block's sum, in thread 0 (in a fixed order).
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double place[kAdamwThreads / kWave];
  x = wave_sum_lane63(x);
  if (lane_id() == kWave - 1) place[wave_in_block()] = x;
  __syncthreads();
  x = 0.0;
  for (int i = 0; i < kAdamwThreads / kWave; ++i) x += place[i];
  return x;
}

__global__ __launch_bounds__(kAdamwThreads) void norm_partial_kernel(const NormTable a) {
  double sum = 0.0;
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const NormTensor &t = a.tensor[i];
    const int64_t base = static_cast<int64_t>(tile - a.first[i]) * kAdamwTile;
    if (t.dtype == FLEXSAE_F32) sum += squares_of_tile<float>(t.grad, t.n, base);
    else if (t.dtype == FLEXSAE_BF16) sum += squares_of_tile<bf16_t>(t.grad, t.n, base);
    else sum += squares_of_tile<f16_t>(t.grad, t.n, base);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kAdamwThreads) void norm_finish_kernel(const double *partial, int64_t n, float *norm) {
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kAdamwThreads) sum += partial[i];
  sum = block_sum(sum);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(sum));
}

// ---- the values of 8-bit states ------------------------------------------------------------
struct MomentsTensor {
  const void *codes;
  const float *maxima;
  void *m, *v;
  int64_t rows, cols;
};
constexpr int kMomentsTensors = 64;
struct MomentsTable {
  MomentsTensor tensor[kMomentsTensors];
  uint32_t first[kMomentsTensors + 1];
  int32_t count;
};
static_assert(sizeof(MomentsTable) <= 4096, "kernel arguments");

// A tile is 2048 elements of one row.
template <typename T>
__global__ __launch_bounds__(kAdamwThreads) void adamw8_moments_kernel(const MomentsTable a) {
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const MomentsTensor &t = a.tensor[i];
    const int64_t per_row = (t.cols + kAdamwTile - 1) / kAdamwTile, blocks = (t.cols + kAdamwQuant - 1) / kAdamwQuant;
    const int64_t row = (tile - a.first[i]) / per_row, part = (tile - a.first[i]) % per_row;
    const int64_t col = part * kAdamwTile + static_cast<int64_t>(threadIdx.x) * kAdamwLane, rest = t.cols - col;
    if (rest <= 0) continue;
    const int left = rest > kAdamwLane ? kAdamwLane : static_cast<int>(rest);
    Codes8 codes;
    load_codes(t.codes, row * t.cols + col, left, codes);
    const float2 top = reinterpret_cast<const float2 *>(t.maxima)[row * blocks + col / kAdamwQuant];
    float m[kAdamwLane], v[kAdamwLane];
    decode8(codes, top.x, top.y, m, v);
    store8<T>(t.m, row * t.cols + col, left, m);
    store8<T>(t.v, row * t.cols + col, left, v);
  }
}

}  // namespace flexsae
