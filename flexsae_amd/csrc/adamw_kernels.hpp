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
constexpr int kAdamwTile = 2048;                           // elements of a block at a time
constexpr int kAdamwQuant = 256;                           // elements that share the maxima of 8-bit states
constexpr int kAdamwTensors = 66;                          // of one launch: the table travels in the kernel's arguments (4 KiB)
constexpr int kNormTensors = 200;
constexpr int kNormTile = 8192;
constexpr int kNormSums = 4;  // of a thread

struct AdamwTensor {
  void *param;
  const void *grad;
  void *s0, *s1;  // exp_avg, exp_avg_sq; or codes, maxima
  float *master;  // (NULL: none)
  uint64_t size;  // elements and type (sized); unit rows: columns in the high word, rows in the low one
  float lr, weight_decay;
};

// A number of elements (at most 2^40) and a flexsae_dtype in one word.
constexpr int kDtypeBit = 56;
constexpr uint64_t sized(int64_t n, int dtype) { return static_cast<uint64_t>(n) | (static_cast<uint64_t>(dtype) << kDtypeBit); }
__device__ __forceinline__ int64_t elements(uint64_t size) { return static_cast<int64_t>(size & ((uint64_t{1} << kDtypeBit) - 1)); }
__device__ __forceinline__ int dtype_of(uint64_t size) { return static_cast<int>(size >> kDtypeBit); }

struct AdamwTable {
  AdamwTensor tensor[kAdamwTensors];
  uint32_t first[kAdamwTensors + 1];  // tile (unit rows: group of rows) at which each tensor begins; the number of them
  int32_t count;
  uint32_t per_block;  // consecutive tiles of a block
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, inv_scale, max_norm;
  const float *grad_norm, *lr;  // device (NULL: none)
  const float2 *bias;           // device: 1 / (1 - b1^t), 1 / sqrt(1 - b2^t)
};
static_assert(sizeof(AdamwTable) <= 4096, "kernel arguments");

struct AdamwCoefs {
  float b1, omb1, b2, omb2, eps, grad, inv_bc1, inv_sqrt_bc2, lr;
  bool go;
};

// 1 - b^t = -(e^x - 1) for x = t log(b) <= 0, without cancellation: the series to x^9 where x is small (off by less than
// 2^-30 of it), one exponential elsewhere.
__device__ __forceinline__ float one_minus_power(double t, double log_b) {
  const float x = static_cast<float>(t * log_b);
  if (x < -0.5f) return 1.f - __expf(x);
  float s = 1.f;
#pragma unroll
  for (int k = 9; k > 1; --k) s = fmaf(s, x * (1.f / static_cast<float>(k)), 1.f);
  return -x * s;
}

__device__ __forceinline__ AdamwCoefs adamw_coefs(const AdamwTable &a) {
#pragma clang fp contract(off)
  AdamwCoefs c;
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
  const float2 bias = *a.bias;
  c.lr = a.lr ? *a.lr : 1.f;
  c.inv_bc1 = bias.x * c.lr;
  c.inv_sqrt_bc2 = bias.y;
  return c;
}

// Every block needs the number of the step, so none may count it before all have read it: a kernel of one thread does, before the
// first of a call, and leaves what depends on the number in the word beside it.  (Tickets of blocks that end, the last of which
// counts, come at 160 a microsecond: at 148 000 blocks 1.8 ms instead of 0.6.)
__global__ void adamw_count_kernel(int64_t *counter, const float *grad_norm, double log_beta1, double log_beta2) {
  if (grad_norm && !__builtin_isfinite(*grad_norm)) return;
  const int64_t steps = counter[0] + 1;
  counter[0] = steps;
  const double t = static_cast<double>(steps);
  *reinterpret_cast<float2 *>(counter + 1) = float2{1.f / one_minus_power(t, log_beta1), 1.f / sqrtf(one_minus_power(t, log_beta2))};
}

// The tensor of a tile: the largest i with first[i] <= tile (tensors without tiles are not in the table).
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table &a, uint32_t tile) {
  int i = 0;
#pragma unroll
  for (int s = 128; s > 0; s >>= 1)
    if (i + s < a.count && tile >= a.first[i + s]) i += s;
  return i;
}

// N consecutive elements of a lane as stored.  Vector accesses ask for the elements' own alignment only (rows and views start
// anywhere); they stream: every byte is used once in a call.
template <typename T, int N>
struct Raw {
  static constexpr int kWords = N * static_cast<int>(sizeof(typename Traits<T>::store_t)) / 4;
  uint32_t w[kWords];
};

typedef uint32_t words4_at4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t words4_at2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words2_at4_t __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t words2_at2_t __attribute__((ext_vector_type(2), aligned(2)));

// WORDS (2, 4 or 8) dwords through memory that is aligned to ALIGN (2 or 4) bytes
template <int WORDS, int ALIGN>
__device__ __forceinline__ void load_words(const void *p, uint32_t *w) {
  if constexpr (WORDS == 2) {
    vec_t<uint32_t, 2> x;
    if constexpr (ALIGN == 4) x = __builtin_nontemporal_load(static_cast<const words2_at4_t *>(p));
    else x = __builtin_nontemporal_load(static_cast<const words2_at2_t *>(p));
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int j = 0; j < WORDS; j += 4) {
      const void *at = static_cast<const char *>(p) + 4 * j;
      vec_t<uint32_t, 4> x;
      if constexpr (ALIGN == 4) x = __builtin_nontemporal_load(static_cast<const words4_at4_t *>(at));
      else x = __builtin_nontemporal_load(static_cast<const words4_at2_t *>(at));
#pragma unroll
      for (int k = 0; k < 4; ++k) w[j + k] = x[k];
    }
  }
}
template <int WORDS, int ALIGN>
__device__ __forceinline__ void store_words(void *p, const uint32_t *w) {
  if constexpr (WORDS == 2) {
    const vec_t<uint32_t, 2> x = {w[0], w[1]};
    if constexpr (ALIGN == 4) __builtin_nontemporal_store(x, static_cast<words2_at4_t *>(p));
    else __builtin_nontemporal_store(x, static_cast<words2_at2_t *>(p));
  } else {
#pragma unroll
    for (int j = 0; j < WORDS; j += 4) {
      void *at = static_cast<char *>(p) + 4 * j;
      const vec_t<uint32_t, 4> x = {w[j], w[j + 1], w[j + 2], w[j + 3]};
      if constexpr (ALIGN == 4) __builtin_nontemporal_store(x, static_cast<words4_at4_t *>(at));
      else __builtin_nontemporal_store(x, static_cast<words4_at2_t *>(at));
    }
  }
}

// Where a lane's elements are: `start` and `block`, the same for the wavefront where it works on one row, stay in scalar registers,
// and the lane's part fits 32 bits.
struct Place {
  int64_t start;  // element of the tensor at which the row, or the tile, begins
  int64_t block;  // block of 8-bit states that begins there
  uint32_t col;   // of the lane's first element
  int left;       // elements of the lane that exist
};
template <typename S>
__device__ __forceinline__ S *element(S *base, const Place &at) {
  using C = std::conditional_t<std::is_const_v<S>, const char, char>;
  return reinterpret_cast<S *>(reinterpret_cast<C *>(base + at.start) + at.col * static_cast<uint32_t>(sizeof(S)));
}

// at.left (at most N) of the elements exist; the others are zeros, or are not stored.
template <typename T, int N>
__device__ __forceinline__ void load_raw_upto(const void *base, const Place &at, Raw<T, N> &r) {
  using S = typename Traits<T>::store_t;
  const S *p = element(static_cast<const S *>(base), at);
  const int left = at.left;
  if (left >= N) {
    load_words<Raw<T, N>::kWords, sizeof(S)>(p, r.w);
  } else {
    S x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = j < left ? p[j] : S{};
    __builtin_memcpy(r.w, x, sizeof(x));
  }
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N> &r, float (&o)[N]) {
  if constexpr (Traits<T>::dtype == FLEXSAE_F32) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = Traits<T>::up(static_cast<uint16_t>(r.w[j / 2] >> (16 * (j % 2))));
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_upto(void *base, const Place &at, const float (&x)[N]) {
  using S = typename Traits<T>::store_t;
  S *p = element(static_cast<S *>(base), at);
  const int left = at.left;
  if (left >= N) {
    uint32_t w[Raw<T, N>::kWords];
#pragma unroll
    for (int j = 0; j < Raw<T, N>::kWords; ++j) {
      if constexpr (Traits<T>::dtype == FLEXSAE_F32) w[j] = __float_as_uint(x[j]);
      else if constexpr (Traits<T>::dtype == FLEXSAE_BF16) w[j] = f32x2_to_bf16x2_bits(x[2 * j], x[2 * j + 1]);
      else w[j] = static_cast<uint32_t>(f32_to_f16_bits(x[2 * j])) | (static_cast<uint32_t>(f32_to_f16_bits(x[2 * j + 1])) << 16);
    }
    store_words<Raw<T, N>::kWords, sizeof(S)>(p, w);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < left) p[j] = Traits<T>::down(x[j]);
  }
}

// ---- 8-bit states --------------------------------------------------------------------------
// (code of m, code of v) of N elements
template <int N>
struct Codes {
  uint32_t w[N / 2];
};

template <int N>
__device__ __forceinline__ void load_codes(const void *base, const Place &at, Codes<N> &c) {
  const uint16_t *p = element(static_cast<const uint16_t *>(base), at);
  const int left = at.left;
  if (left >= N) {
    load_words<N / 2, 2>(p, c.w);
  } else {
    uint16_t x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = j < left ? p[j] : uint16_t{128};
    __builtin_memcpy(c.w, x, sizeof(x));
  }
}

template <int N>
__device__ __forceinline__ void store_codes(void *base, const Place &at, const Codes<N> &c) {
  uint16_t *p = element(static_cast<uint16_t *>(base), at);
  const int left = at.left;
  if (left >= N) {
    store_words<N / 2, 2>(p, c.w);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < left) p[j] = static_cast<uint16_t>(c.w[j / 2] >> (16 * (j % 2)));
  }
}

template <int N>
__device__ __forceinline__ void decode(const Codes<N> &c, float a_m, float a_v, float (&m)[N], float (&v)[N]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t pair = c.w[j / 2] >> (16 * (j % 2));
    // (the squares of codes are exact; what follows is a rounding each, and none is raised to a power but that of 1 / 255^2)
    const float x = static_cast<float>(pair & 0xffu) - 128.f;
    m[j] = x * fabsf(x) * (1.f / (127.f * 127.f)) * a_m;
    float y = static_cast<float>((pair >> 8) & 0xffu);
    y = y * y * (1.f / (255.f * 255.f));
    v[j] = y * y * a_v;
  }
}

// Sum or maximum over each LANES (16, 32 or 64) consecutive lanes, in all of them.
template <int LANES, typename T, typename F>
__device__ __forceinline__ T across_lanes(T x, F join) {
  static_assert(sizeof(T) == 4 && (LANES == 16 || LANES == 32 || LANES == 64), "");
  auto bits = [](T y) {
    uint32_t u;
    __builtin_memcpy(&u, &y, 4);
    return u;
  };
  auto value = [](uint32_t u) {
    T y;
    __builtin_memcpy(&y, &u, 4);
    return y;
  };
  auto move = [&](T y, auto ctrl) {
    return value(static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(bits(y)), decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  x = join(x, move(x, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
  x = join(x, move(x, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
  x = join(x, move(x, std::integral_constant<int, 0x141>{}));  // the other quad of each 8
  x = join(x, move(x, std::integral_constant<int, 0x140>{}));  // the other half of each 16-lane row
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  if constexpr (LANES >= 32) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(bits(x), bits(x), false, false);  // the other row of each two
    x = join(value(r[0]), value(r[1]));
  }
  if constexpr (LANES == 64) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(bits(x), bits(x), false, false);  // the other half
    x = join(value(r[0]), value(r[1]));
  }
  return x;
}

// 1 / a of a positive normal number, rounded once: a reciprocal, its error put right, and the exponent by itself (the result may
// lie below the normal numbers).
__device__ __forceinline__ float inverse(float a) {
  const float x = __builtin_amdgcn_frexp_mantf(a), r = __builtin_amdgcn_rcpf(x);
  return __builtin_amdgcn_ldexpf(fmaf(r, fmaf(-x, r, 1.f), r), -__builtin_amdgcn_frexp_expf(a));
}

// The maxima of |m| and of v over a block that LANES lanes hold, and their inverses (zero for zero).  A maximum is kept as zero
// below the smallest normal number (its inverse would overflow), as NaN where the block has infinities or NaN: as whole numbers
// the bits of non-negative floats are in their order, infinity and NaN above all.
struct Maxima {
  float m, v, per_m, per_v, root_per_v;
};

__device__ __forceinline__ float kept(uint32_t bits) {
  return bits < 0x00800000u ? 0.f : bits < 0x7f800000u ? __uint_as_float(bits) : __uint_as_float(0x7fc00000u);
}

template <int LANES, int N>
__device__ __forceinline__ Maxima maxima(const float (&m)[N], const float (&v)[N], float m_before) {
  Maxima r;
  uint32_t bv = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) bv = max(bv, __float_as_uint(v[j]));
  if constexpr (N == 4) {
    // After the first exchange even lanes carry m's and odd lanes v's, so that the other exchanges and the inverses serve both:
    // what a block costs is shared by few elements (24571 x 1538 fp32 122 -> 118 us, 2.1M fp32 11.0 -> 10.7).  With eight the registers
    // it takes cost more (302M bf16 512 -> 536 us).
    uint32_t bm = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) bm = max(bm, __float_as_uint(m[j]) & 0x7fffffffu);
    auto move = [](uint32_t y, auto ctrl) {
      return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(y), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    const bool odd = (threadIdx.x & 1) != 0;
    uint32_t x = odd ? bv : bm;
    x = max(x, move(odd ? bm : bv, std::integral_constant<int, 0xB1>{}));  // lane ^ 1 gives what it does not carry
    x = max(x, move(x, std::integral_constant<int, 0x4E>{}));              // lane ^ 2
    x = max(x, move(x, std::integral_constant<int, 0x124>{}));             // 4 lanes on, in the row of 16
    x = max(x, move(x, std::integral_constant<int, 0x128>{}));             // 8 lanes on
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    if constexpr (LANES >= 32) {
      const u32x2 y = __builtin_amdgcn_permlane16_swap(x, x, false, false);  // the other row of each two
      x = max(y[0], y[1]);
    }
    if constexpr (LANES == 64) {
      const u32x2 y = __builtin_amdgcn_permlane32_swap(x, x, false, false);  // the other half
      x = max(y[0], y[1]);
    }
    const float a = kept(x), per = a > 0.f ? inverse(a) : 0.f;
    auto even_of = [&](float y) { return __uint_as_float(move(__float_as_uint(y), std::integral_constant<int, 0xA0>{})); };
    auto odd_of = [&](float y) { return __uint_as_float(move(__float_as_uint(y), std::integral_constant<int, 0xF5>{})); };
    r.m = even_of(a);
    r.v = odd_of(a);
    r.per_m = even_of(per);
    r.per_v = odd_of(per);
    r.root_per_v = odd_of(__builtin_amdgcn_sqrtf(per));
  } else {
    // The floating-point maximum passes over NaN, and m has infinities or NaN only where v has, or its maximum was NaN before (a
    // finite g whose square overflows leaves m as it is): such blocks are asked again.
    float bm = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) bm = fmaxf(bm, fabsf(m[j]));
    bm = across_lanes<LANES>(bm, [](float x, float y) { return fmaxf(x, y); });
    bv = across_lanes<LANES>(bv, [](uint32_t x, uint32_t y) { return max(x, y); });
    r.m = kept(__float_as_uint(bm));
    if (__any(bv >= 0x7f800000u || m_before != m_before)) {
      uint32_t all = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) all = max(all, __float_as_uint(m[j]) & 0x7fffffffu);
      r.m = kept(across_lanes<LANES>(all, [](uint32_t x, uint32_t y) { return max(x, y); }));
    }
    r.v = kept(bv);
    r.per_m = r.m > 0.f ? inverse(r.m) : 0.f;
    r.per_v = r.v > 0.f ? inverse(r.v) : 0.f;
    r.root_per_v = __builtin_amdgcn_sqrtf(r.per_v);
  }
  return r;
}

// Codes of two elements, (m, v) each, from |m| / a_m and v / a_v: whole numbers nearest to 127 sqrt and 255 sqrt sqrt of them, as
// correctly rounded operations give them, whatever unit computes them.  EXACT: such operations.  Otherwise the hardware's roots,
// `root_v` = sqrt(v) sqrt(1 / a_v) among them, off by a unit in the last place each: with the roundings on either side 2.5e-7 of
// the result for m and 5.5e-7 for v.  Both ends of that stretch are rounded; where they are not the same, true comes back.
// Adding kMagic rounds to a whole number, which then stands in the low bits.
// The hardware's root takes a number below the normal ones for zero.  Maxima above 2^126 have such an inverse, and beside
// one below 2^-96 such a v has a code above one ((2^-126 / 2^-96)^(1/4) is 1.41 / 255): blocks of these are EXACT (rooted).
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
constexpr float kOffM = 2.5e-7f, kOffV = 5.5e-7f;

// Whether the hardware's roots serve a block of this maximum of v (one that is kept as zero or NaN has no codes to speak of).
__device__ __forceinline__ bool rooted(float a_v) { return !(a_v > 0x1p126f || (a_v > 0.f && a_v < 0x1p-96f)); }

template <bool EXACT>
__device__ __forceinline__ bool codes_of_two(const float *m, const float *v, const Maxima &a, uint32_t least, const float *s,
                                             uint32_t &w) {
#pragma clang fp contract(off)
  uint32_t pair[2], differ = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float x, y;
    if constexpr (EXACT) {
      x = copysignf(sqrtf(fabsf(m[k]) * a.per_m) * 127.f, m[k]) + (kMagic + 128.f);
      y = sqrtf(sqrtf(v[k] * a.per_v)) * 255.f + kMagic;
    } else {
      const float rm = copysignf(__builtin_amdgcn_sqrtf(fabsf(m[k]) * a.per_m), m[k]);
      const float rv = __builtin_amdgcn_sqrtf(s[k] * a.root_per_v);
      x = fmaf(rm, 127.f * (1.f + kOffM), kMagic + 128.f);
      y = fmaf(rv, 255.f * (1.f + kOffV), kMagic);
      differ |= (__float_as_uint(x) ^ __float_as_uint(fmaf(rm, 127.f * (1.f - kOffM), kMagic + 128.f))) |
                (__float_as_uint(y) ^ __float_as_uint(fmaf(rv, 255.f * (1.f - kOffV), kMagic)));
    }
    // (a v above zero never becomes zero: `least` is one where the block has a maximum)
    pair[k] = __builtin_amdgcn_perm(max(__float_as_uint(y) & 0xffu, min(__float_as_uint(v[k]), least)), __float_as_uint(x), 0x0c0c0400u);
  }
  w = pair[0] | (pair[1] << 16);
  return differ != 0;
}

// s: the hardware's square roots of v
template <int N>
__device__ __forceinline__ void encode(const float (&m)[N], const float (&v)[N], const float (&s)[N], const Maxima &a, Codes<N> &c) {
  const uint32_t least = a.v > 0.f ? 1u : 0u;
  const bool all = !rooted(a.v);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    // (one such pair of a wavefront in 30 to 50: 128 elements, each with 1.1e-6 of its code of v, and half of that of m's, between)
    const bool near = codes_of_two<false>(m + j, v + j, a, least, s + j, c.w[j / 2]);
    if (__any(near || all)) (void)codes_of_two<true>(m + j, v + j, a, least, s + j, c.w[j / 2]);
  }
}

// ---- the step ------------------------------------------------------------------------------
constexpr float kRootFloor = 1.0842022e-19f;  // 2^-63

template <int N>
__device__ __forceinline__ void adamw_moments(const AdamwCoefs &c, const float (&g)[N], float (&m)[N], float (&v)[N]) {
// (each operation rounded by itself, like the roots of the codes: 8-bit states do not depend on what a compiler contracts)
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < N; ++j) {
    m[j] = m[j] * c.b1 + g[j] * c.omb1;
    v[j] = v[j] * c.b2 + g[j] * g[j] * c.omb2;
  }
}

// s: square roots of v.  The hardware's root and reciprocal, each off by a unit in the last place: of the update, which is a small
// part of the weight.  (It takes a v below the smallest normal number for zero: the root's floor keeps the quotient finite
// where eps is zero.  The larger of two whole numbers: a NaN, which the larger of two floats passes over, reaches the weight.)
template <int N>
__device__ __forceinline__ void adamw_move(const AdamwCoefs &c, float step, float keep, const float (&m)[N], const float (&s)[N],
                                           float (&w)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float root = __uint_as_float(max(__float_as_uint(s[j]), __float_as_uint(kRootFloor)));
    const float per = __builtin_amdgcn_rcpf(fmaf(root, c.inv_sqrt_bc2, c.eps));
    w[j] = fmaf(-step, m[j] * per, keep * w[j]);
  }
}

// Elements of a lane that follow each other: as many as make sixteen bytes of the widest tensor, so that every access of a
// wavefront is one stretch of memory (two accesses of half a stretch each cost a tenth of the bandwidth).
template <typename T, bool MASTER, bool EIGHT>
constexpr int kUnit = EIGHT && !MASTER && sizeof(typename Traits<T>::store_t) == 2 ? 8 : 4;

// A lane's elements of the tensors that a step works on: as loaded, and as numbers.
template <typename T, bool MASTER, bool EIGHT>
struct AdamwUnit {
  static constexpr int N = kUnit<T, MASTER, EIGHT>;
  static constexpr int kQuantLanes = kAdamwQuant / N;  // that hold a block of 8-bit states
  using W = std::conditional_t<MASTER, float, T>;
  Raw<T, N> rg;
  Raw<W, N> rw;
  Raw<float, EIGHT ? 0 : N> rm, rv;  // states in 32 bits,
  Codes<EIGHT ? N : 0> codes;        // in 8
  float2 top;

  __device__ __forceinline__ void load(const AdamwTensor &t, const Place &at) {
    load_raw_upto(t.grad, at, rg);
    load_raw_upto(MASTER ? t.master : t.param, at, rw);
    if constexpr (EIGHT) {
      load_codes(t.s0, at, codes);
      top = at.left > 0 ? static_cast<const float2 *>(t.s1)[at.block + at.col / kAdamwQuant] : float2{0.f, 0.f};
    } else {
      load_raw_upto(t.s0, at, rm);
      load_raw_upto(t.s1, at, rv);
    }
  }

  // m, v from g and what they were; w moved; STORE: m and v stored.  LANES share a row.
  template <bool STORE, int LANES>
  __device__ __forceinline__ void step(const AdamwTensor &t, const AdamwCoefs &c, const Place &at, const float (&g)[N], float (&w)[N]) {
    float m[N], v[N], s[N];
    if constexpr (EIGHT) {
      decode(codes, top.x, top.y, m, v);
    } else {
      unpack(rm, m);
      unpack(rv, v);
    }
    adamw_moments(c, g, m, v);
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = __builtin_amdgcn_sqrtf(v[j]);
    adamw_move(c, t.lr * c.inv_bc1, 1.f - t.lr * c.lr * t.weight_decay, m, s, w);
    if constexpr (STORE && EIGHT) {
      constexpr int kLanes = LANES < kQuantLanes ? LANES : kQuantLanes;
      const Maxima a = maxima<kLanes>(m, v, top.x);
      Codes<N> now;
      encode(m, v, s, a, now);
      store_codes(t.s0, at, now);
      if (at.left > 0 && (threadIdx.x & (kLanes - 1)) == 0)
        static_cast<float2 *>(t.s1)[at.block + at.col / kAdamwQuant] = float2{a.m, a.v};
    } else if constexpr (STORE) {
      store_upto<float>(t.s0, at, m);
      store_upto<float>(t.s1, at, v);
    }
  }

  __device__ __forceinline__ void store(const AdamwTensor &t, const Place &at, const float (&w)[N]) const {
    if constexpr (MASTER) {
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] = w[j];
        // the 32-bit number itself is what is rounded (an instruction that multiplies, adds and rounds to fp16 would leave it out)
        if constexpr (Traits<T>::dtype == FLEXSAE_F16) asm("" : "+v"(x[j]));
      }
      store_upto<T>(t.param, at, x);
      store_upto<float>(t.master, at, x);
    } else {
      store_upto<T>(t.param, at, w);
    }
  }
};

// What exists of N elements of which `rest` are left.
template <int N>
__device__ __forceinline__ int upto(int64_t rest) {
  return rest > N ? N : rest < 0 ? 0 : static_cast<int>(rest);
}

// FULL: the tile ends within the tensor.
template <typename T, bool MASTER, bool EIGHT, bool FULL>
__device__ __forceinline__ void adamw_tile(const AdamwTensor &t, int64_t base, const AdamwCoefs &c) {
  using Unit = AdamwUnit<T, MASTER, EIGHT>;
  constexpr int N = Unit::N, kUnits = kAdamwTile / (kAdamwThreads * N);
  Unit unit[kUnits];
  auto place = [&](int u) -> Place {
    const uint32_t col = (u * kAdamwThreads + threadIdx.x) * N;
    return {base, base / kAdamwQuant, col, FULL ? N : upto<N>(elements(t.size) - base - col)};
  };
#pragma unroll
  for (int u = 0; u < kUnits; ++u) unit[u].load(t, place(u));
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float g[N], w[N];
    unpack(unit[u].rg, g);
    unpack(unit[u].rw, w);
    if (c.grad != 1.f) {
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] *= c.grad;
    }
    unit[u].template step<true, kWave>(t, c, place(u), g, w);
    unit[u].store(t, place(u), w);
  }
}

// Tensors as they are stored.  States in 32 bits: bound by memory, every byte moved once (302M bf16 parameters with masters:
// 1394 us, 6.07 TB/s, where a copy reaches 6.5).  States in 8 bits: 62 vector instructions an element, of which four or five are roots
// and a reciprocal that take four times as long, fill nearly the time that memory takes (302M bf16 parameters: 510 us, 6.0 TB/s;
// a table of the codes' values in the LDS, maxima exchanged for both moments at once, five or seven wavefronts a SIMD instead of
// six: the same or slower).
template <bool EIGHT>
__global__ __launch_bounds__(kAdamwThreads) void adamw_kernel(const AdamwTable a) {
  const AdamwCoefs c = adamw_coefs(a);
  if (!c.go) return;
  const uint32_t end = min(a.first[a.count], (blockIdx.x + 1) * a.per_block);
  for (uint32_t tile = blockIdx.x * a.per_block; tile < end; ++tile) {
    const int i = tensor_of(a, tile);
    const AdamwTensor &t = a.tensor[i];
    const int64_t base = static_cast<int64_t>(tile - a.first[i]) * kAdamwTile;
    const int dtype = dtype_of(t.size);
    auto tile_of = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      if (dtype == FLEXSAE_F32) adamw_tile<float, false, EIGHT, kFull>(t, base, c);
      else if (dtype == FLEXSAE_BF16) t.master ? adamw_tile<bf16_t, true, EIGHT, kFull>(t, base, c) : adamw_tile<bf16_t, false, EIGHT, kFull>(t, base, c);
      else t.master ? adamw_tile<f16_t, true, EIGHT, kFull>(t, base, c) : adamw_tile<f16_t, false, EIGHT, kFull>(t, base, c);
    };
    if (base + kAdamwTile <= elements(t.size)) tile_of(std::true_type{});
    else tile_of(std::false_type{});
  }
}

// Sums over a row that LANES lanes of a wavefront, or WAVES wavefronts of a block, hold; `turn` alternates between two places so
// that one barrier a sum is enough.
template <int WAVES, int LANES>
__device__ __forceinline__ float row_sum(float x, float (*place)[16], int turn) {
  x = across_lanes<LANES>(x, [](float y, float z) { return y + z; });
  if constexpr (WAVES > 1) {
    if (lane_id() == 0) place[turn][wave_in_block()] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += place[turn][i];
  }
  return x;
}

// (blocks of eight wavefronts and more: registers for sixteen on a compute unit, two blocks of eight or one of sixteen)
constexpr int rows_threads(int waves) { return waves < 4 ? 256 : waves * kWave; }

// Rows of length one.  LANES (64 at least with more than one) of each of WAVES wavefronts hold a row, UNITS units of elements each,
// in registers: every tensor is read and written once.  UNITS = 0: a row of any length is walked three times (the two products;
// the length of the moved row; the step), nothing stored before the last walk.  Bound by memory with states in 32 bits (65536 x 2304
// bf16 with masters: 749 us, 5.64 TB/s), by arithmetic in 8 (24571 x 1538 fp32: 118 us, 5.1 TB/s: 109 vector instructions an element,
// among them the seventh stretch of a wavefront for the last two columns, and the block's maxima and inverses of every four elements).
template <typename T, bool MASTER, bool EIGHT, int WAVES, int LANES, int UNITS>
__global__ __launch_bounds__(rows_threads(WAVES), WAVES < 8 ? 1 : 4) void adamw_rows_kernel(const AdamwTable a) {
  static_assert(LANES == kWave || (WAVES == 1 && UNITS == 1), "less than a wavefront: one unit");
  using Unit = AdamwUnit<T, MASTER, EIGHT>;
  constexpr int N = Unit::N, kStretch = LANES * N;
  static_assert(WAVES == 1 || WAVES >= 4, "a block has a barrier only where it holds one row");
  constexpr int kRows = rows_threads(WAVES) / (WAVES * LANES);  // of a block at a time
  __shared__ float place[2][16];
  const AdamwCoefs c = adamw_coefs(a);
  if (!c.go) return;
  const int wave = wave_in_block() % WAVES;
  const uint32_t end = min(a.first[a.count], (blockIdx.x + 1) * a.per_block);
  for (uint32_t tile = blockIdx.x * a.per_block; tile < end; ++tile) {
    const int i = tensor_of(a, tile);
    const AdamwTensor &t = a.tensor[i];
    const int64_t rows = static_cast<uint32_t>(t.size);
    int64_t row = static_cast<int64_t>(tile - a.first[i]) * kRows + wave_in_block() / WAVES * (kWave / LANES);
    if (row >= rows) continue;  // (of a whole wavefront: a block of several rows has no barriers)
    if constexpr (LANES < kWave) row += lane_id() / LANES;
    const bool live = LANES == kWave || row < rows;
    const int cols = static_cast<int>(t.size >> 32);
    const int64_t start = row * cols, block = row * ((cols + kAdamwQuant - 1) / kAdamwQuant);
    auto stretch = [&](int u) { return (u * WAVES + wave) * kStretch; };
    auto at = [&](int u) -> Place {
      const int col = stretch(u) + lane_id() % LANES * N;
      return {start, block, static_cast<uint32_t>(col), live ? upto<N>(cols - col) : 0};
    };
    auto products = [&](const Unit &unit, float (&g)[N], float (&w)[N], float &gw, float &ww) {
      unpack(unit.rg, g);
      unpack(unit.rw, w);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        g[j] *= c.grad;
        gw = fmaf(g[j], w[j], gw);
        ww = fmaf(w[j], w[j], ww);
      }
    };
    auto across = [&](float along, float (&g)[N], const float (&w)[N]) {
#pragma clang fp contract(off)
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] = g[j] - along * w[j];
    };
    auto squares = [&](const float (&w)[N], float &s) {
#pragma unroll
      for (int j = 0; j < N; ++j) s = fmaf(w[j], w[j], s);
    };
    auto scaled = [&](float by, float (&w)[N]) {
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] *= by;
    };
    float gw = 0.f, ww = 0.f, nn = 0.f;
    if constexpr (UNITS > 0) {
      // (units beyond the row's end, the same ones for the whole wavefront, are left out)
      Unit unit[UNITS];
      float g[UNITS][N], w[UNITS][N];
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (u == 0 || stretch(u) < cols) unit[u].load(t, at(u));
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (u == 0 || stretch(u) < cols) products(unit[u], g[u], w[u], gw, ww);
      gw = row_sum<WAVES, LANES>(gw, place, 0);
      ww = row_sum<WAVES, LANES>(ww, place, 1);
      const float along = ww > 0.f ? gw / ww : 0.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (u == 0 || stretch(u) < cols) {
          across(along, g[u], w[u]);
          unit[u].template step<true, LANES>(t, c, at(u), g[u], w[u]);
          squares(w[u], nn);
        }
      nn = row_sum<WAVES, LANES>(nn, place, 0);
      const float by = nn > 0.f ? 1.f / sqrtf(nn) : 1.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (u == 0 || stretch(u) < cols) {
          scaled(by, w[u]);
          unit[u].store(t, at(u), w[u]);
        }
    } else {
      const int units = (cols - 1) / (WAVES * kStretch) + 1;
      Unit unit;
      float g[N], w[N];
      for (int u = 0; u < units; ++u) {
        unit.load(t, at(u));
        products(unit, g, w, gw, ww);
      }
      gw = row_sum<WAVES, LANES>(gw, place, 0);
      ww = row_sum<WAVES, LANES>(ww, place, 1);
      const float along = ww > 0.f ? gw / ww : 0.f;
      float unused_gw = 0.f, unused_ww = 0.f;
      for (int u = 0; u < units; ++u) {
        unit.load(t, at(u));
        products(unit, g, w, unused_gw, unused_ww);
        across(along, g, w);
        unit.template step<false, LANES>(t, c, at(u), g, w);
        squares(w, nn);
      }
      nn = row_sum<WAVES, LANES>(nn, place, 0);
      const float by = nn > 0.f ? 1.f / sqrtf(nn) : 1.f;
      for (int u = 0; u < units; ++u) {
        unit.load(t, at(u));
        products(unit, g, w, unused_gw, unused_ww);
        across(along, g, w);
        unit.template step<true, LANES>(t, c, at(u), g, w);
        scaled(by, w);
        unit.store(t, at(u), w);
      }
    }
    // (the next row's first sum may write place[0] while a wavefront still reads it for this one's length)
    if constexpr (WAVES > 1) __syncthreads();
  }
}

// ---- the gradients' norm -------------------------------------------------------------------
struct NormTensor {
  const void *grad;
  uint64_t size;
};
// (No table here has an array of bytes beside its wider ones: an index that addresses both lets the compiler take the address of
// a wider entry apart as base + i and 7 i, and scalar loads drop the two low bits of each part.)
// TENSORS: a launch with four kilobytes of arguments takes the host a microsecond longer than one with few.
template <int TENSORS>
struct NormTable {
  NormTensor tensor[TENSORS];
  uint32_t first[TENSORS + 1];
  int32_t count;
  double *partial;  // one of each block
};
constexpr int kNormFew = 8;
static_assert(sizeof(NormTable<kNormTensors>) <= 4096, "kernel arguments");

// Squares are summed in 64 bits: those of finite 32-bit numbers neither overflow nor vanish there, and the order of the sum,
// which is the same on every run, hardly matters.
template <typename T, bool FULL>
__device__ __forceinline__ void squares_of_tile(const void *grad, int64_t n, int64_t base, double (&sum)[kNormSums]) {
  constexpr int N = 16 / static_cast<int>(sizeof(typename Traits<T>::store_t)), kLoads = kNormTile / (kAdamwThreads * N);
  Raw<T, N> r[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint32_t col = (u * kAdamwThreads + threadIdx.x) * N;
    load_raw_upto(grad, Place{base, 0, col, FULL ? N : upto<N>(n - base - col)}, r[u]);
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    float x[N];
    unpack(r[u], x);
#pragma unroll
    for (int j = 0; j < N; ++j)
      sum[u % kNormSums] = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum[u % kNormSums]);
  }
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

template <int TENSORS>
__global__ __launch_bounds__(kAdamwThreads) void norm_partial_kernel(const NormTable<TENSORS> a) {
  double sum[kNormSums] = {};
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const NormTensor &t = a.tensor[i];
    const int64_t base = static_cast<int64_t>(tile - a.first[i]) * kNormTile, n = elements(t.size);
    const int dtype = dtype_of(t.size);
    auto tile_of = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      if (dtype == FLEXSAE_F32) squares_of_tile<float, kFull>(t.grad, n, base, sum);
      else if (dtype == FLEXSAE_BF16) squares_of_tile<bf16_t, kFull>(t.grad, n, base, sum);
      else squares_of_tile<f16_t, kFull>(t.grad, n, base, sum);
    };
    if (base + kNormTile <= n) tile_of(std::true_type{});
    else tile_of(std::false_type{});
  }
  double all = 0.0;
#pragma unroll
  for (int u = 0; u < kNormSums; ++u) all += sum[u];
  all = block_sum(all);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = all;
}

// Bound by memory: 2.1e9 bf16 elements in 615 us, 7.0 TB/s, what reading alone reaches; with one load of a thread in flight instead
// of four 948 us.
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

// A tile is 2048 elements of the flattened tensor, wherever rows end.  Bound by memory: 302M elements to bf16 in 280 us, 6.5 TB/s;
// rows that are no multiple of 256 by their places: 41 vector instructions an element instead of 17, and maxima fetched by the lane
// (24571 x 1538: 49 us, 4.7 TB/s).
template <typename T>
__global__ __launch_bounds__(kAdamwThreads) void adamw8_moments_kernel(const MomentsTable a) {
  constexpr int N = 16 / static_cast<int>(sizeof(typename Traits<T>::store_t));
  for (uint32_t tile = blockIdx.x; tile < a.first[a.count]; tile += gridDim.x) {
    const int i = tensor_of(a, tile);
    const MomentsTensor &t = a.tensor[i];
    const int64_t base = static_cast<int64_t>(tile - a.first[i]) * kAdamwTile, blocks = (t.cols + kAdamwQuant - 1) / kAdamwQuant;
    const int64_t row = t.rows == 1 ? 0 : base / t.cols, from = base - row * t.cols;
    const float2 *const top = reinterpret_cast<const float2 *>(t.maxima) + row * blocks;
#pragma unroll
    for (int u = 0; u < kAdamwTile / (kAdamwThreads * N); ++u) {
      const uint32_t offset = (u * kAdamwThreads + threadIdx.x) * N;
      const Place at = {base, 0, offset, upto<N>(t.rows * t.cols - base - offset)};
      if (at.left == 0) continue;
      // the lane's row, counted from the tile's first, and column
      int64_t col = from + offset;
      uint32_t r = 0;
      if (col >= t.cols) {
        r = t.cols >= 2 * kAdamwTile ? 1u : static_cast<uint32_t>(col) / static_cast<uint32_t>(t.cols);
        col -= r * t.cols;
      }
      Codes<N> codes;
      load_codes(t.codes, at, codes);
      float m[N], v[N];
      if (col % kAdamwQuant + at.left <= kAdamwQuant && col + at.left <= t.cols) {
        const float2 x = top[r * blocks + col / kAdamwQuant];
        decode(codes, x.x, x.y, m, v);
      } else {  // more than one block
        decode(codes, 1.f, 1.f, m, v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (j >= at.left) break;
          if (col == t.cols) {
            col = 0;
            ++r;
          }
          const float2 x = top[r * blocks + col / kAdamwQuant];
          m[j] *= x.x;
          v[j] *= x.y;
          ++col;
        }
      }
      store_upto<T>(t.m, at, m);
      store_upto<T>(t.v, at, v);
    }
  }
}

}  // namespace flexsae
