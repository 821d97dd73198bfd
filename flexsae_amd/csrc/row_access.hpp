// Rows that start anywhere: vectors of elements at any element's address, rows that end inside a vector, and sums over the lanes
// that share a row.
#pragma once

#include "common.hpp"

namespace flexsae {

template <typename T>
constexpr int kUnitOf = 16 / static_cast<int>(sizeof(typename Traits<T>::store_t));  // elements of 16 bytes, one access of a lane

// What a lane reads or writes at once, as four words.
typedef uint32_t words_t __attribute__((ext_vector_type(4)));

// The same in memory, aligned to its elements only: rows of an odd number of 16-bit elements begin at odd addresses.  (The HSA ABI
// runs kernels with unaligned access on, and the compiler forms the same 16-byte accesses.)
template <typename T>
struct LooseWords;
template <>
struct LooseWords<float> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct LooseWords<bf16_t> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct LooseWords<f16_t> : LooseWords<bf16_t> {};

template <typename T>
using elem_t = typename Traits<T>::store_t;

template <typename T>
__device__ __forceinline__ uint32_t bits_of(elem_t<T> v) {
  if constexpr (sizeof(v) == 4) return __float_as_uint(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ elem_t<T> from_bits(uint32_t v) {
  if constexpr (sizeof(elem_t<T>) == 4) return __uint_as_float(v);
  else return static_cast<uint16_t>(v);
}

// NT: streaming, for what is read or written once and not soon again.
template <typename T, bool NT = false>
__device__ __forceinline__ words_t load_words(const elem_t<T> *p) {
  const auto *q = reinterpret_cast<const typename LooseWords<T>::type *>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}

template <typename T, bool NT = false>
__device__ __forceinline__ void store_whole(elem_t<T> *p, words_t v, bool there) {
  using L = typename LooseWords<T>::type;
  if (!there) return;
  if constexpr (NT) __builtin_nontemporal_store(static_cast<L>(v), reinterpret_cast<L *>(p));
  else *reinterpret_cast<L *>(p) = v;
}

// The first `left` of the elements at p, zeros for the rest.
template <typename T>
__device__ __forceinline__ words_t load_upto(const elem_t<T> *p, int64_t left) {
  constexpr int N = kUnitOf<T>, kPer = N / 4;
  words_t v = 0u;
  if (left >= N) {
    v = *reinterpret_cast<const typename LooseWords<T>::type *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (i < left) v[i / kPer] |= bits_of<T>(p[i]) << (i % kPer * 16);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store_upto(elem_t<T> *p, words_t v, int64_t left) {
  constexpr int N = kUnitOf<T>, kPer = N / 4;
  if (left >= N) {
    *reinterpret_cast<typename LooseWords<T>::type *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (i < left) p[i] = from_bits<T>(v[i / kPer] >> (i % kPer * 16));
  }
}

template <typename T>
__device__ __forceinline__ void unpack(words_t v, float (&x)[kUnitOf<T>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Traits<T>::dtype == FLEXSAE_F32) {
      x[i] = __uint_as_float(v[i]);
    } else if constexpr (Traits<T>::dtype == FLEXSAE_BF16) {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    } else {
      x[2 * i] = f16_bits_to_f32(static_cast<uint16_t>(v[i]));
      x[2 * i + 1] = f16_bits_to_f32(static_cast<uint16_t>(v[i] >> 16));
    }
  }
}

template <typename T>
__device__ __forceinline__ words_t pack(const float (&x)[kUnitOf<T>]) {
  words_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Traits<T>::dtype == FLEXSAE_F32) v[i] = __float_as_uint(x[i]);
    else if constexpr (Traits<T>::dtype == FLEXSAE_BF16) v[i] = f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
    else v[i] = static_cast<uint32_t>(f32_to_f16_bits(x[2 * i])) | static_cast<uint32_t>(f32_to_f16_bits(x[2 * i + 1])) << 16;
  }
  return v;
}

// N elements of a type that is known at run time, as fp32; zeros behind `left`.
template <int N>
__device__ __forceinline__ void load_typed(const void *base, int dtype, int64_t off, int64_t left, float (&o)[N]) {
  static_assert(N == 4 || N == 8, "units of 16 bytes");
  if (dtype == FLEXSAE_F32) {
#pragma unroll
    for (int h = 0; h < N; h += 4) {
      float x[4];
      unpack<float>(load_upto<float>(static_cast<const float *>(base) + off + h, left - h), x);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[h + i] = x[i];
    }
  } else {
    // (of a unit of four elements the second half is not there)
    const words_t v = load_upto<bf16_t>(static_cast<const uint16_t *>(base) + off, N == 8 ? left : left < 4 ? left : 4);
    float x[8];
    if (dtype == FLEXSAE_BF16) unpack<bf16_t>(v, x);
    else unpack<f16_t>(v, x);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = x[i];
  }
}

__device__ __forceinline__ void store_typed(void *base, int dtype, int64_t off, float v) {
  if (dtype == FLEXSAE_F32) static_cast<float *>(base)[off] = v;
  else static_cast<uint16_t *>(base)[off] = dtype == FLEXSAE_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

// Sum over LANES (16, 32 or 64) consecutive lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(LANES == 16 || LANES == 32 || LANES == 64, "whole rows of 16 lanes");
  v += dpp_move<0xB1>(v);   // quad_perm [1,0,3,2]: lane ^ 1
  v += dpp_move<0x4E>(v);   // quad_perm [2,3,0,1]: lane ^ 2
  v += dpp_move<0x141>(v);  // row_half_mirror: the other quad of each 8
  v += dpp_move<0x140>(v);  // row_mirror: the other half of each 16-lane row
  if constexpr (LANES == 64) return add_across_rows(v);
  if constexpr (LANES == 32) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return v;
}

// The largest over a wavefront, in all lanes.
__device__ __forceinline__ float wave_max(float v) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Blocks beyond the first kGridRow go into further rows of the grid (threads of a grid are counted in 32 bits along an axis).
constexpr int64_t kGridRow = int64_t{1} << 21;
__device__ __forceinline__ int64_t block_index() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6); }

}  // namespace flexsae
