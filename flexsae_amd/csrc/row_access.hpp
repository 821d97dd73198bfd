// Rows that start anywhere: vectors of elements at any element's address, rows that end inside a vector, and sums over the lanes
// that share a row.
#pragma once

#include "common.hpp"

namespace flexsae {

template <typename T>
constexpr int kUnitOf = 16 / static_cast<int>(sizeof(typename Traits<T>::store_t));  // elements of 16 bytes, one access of a lane

// Vectors that are aligned to their elements only: rows of an odd number of 16-bit elements begin at odd addresses.  (The HSA ABI
// runs kernels with unaligned access on, and the compiler forms the same 16-byte accesses.)
template <typename S, int N>
using loose_vec_t = S __attribute__((ext_vector_type(N), aligned(sizeof(S))));

// The N elements at p of which the first `left` are there; zeros (or `fill`'s bits) for the rest.
template <typename T, int N, bool NT = false>
__device__ __forceinline__ raw_vec_t<T, N> load_upto(const typename Traits<T>::store_t *p, int64_t left,
                                                     typename Traits<T>::store_t fill = 0) {
  using S = typename Traits<T>::store_t;
  raw_vec_t<T, N> v;
  if (left >= N) {
    const auto *q = reinterpret_cast<const loose_vec_t<S, N> *>(p);
    if constexpr (NT) v = __builtin_nontemporal_load(q);
    else v = *q;
    return v;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < left ? p[i] : fill;
  return v;
}

template <typename T, int N>
__device__ __forceinline__ raw_vec_t<T, N> pack(const float (&x)[N]) {
  raw_vec_t<T, N> v;
  if constexpr (Traits<T>::dtype == FLEXSAE_BF16) {
    vec_t<uint32_t, N / 2> w;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
    __builtin_memcpy(&v, &w, sizeof v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Traits<T>::down(x[i]);
  }
  return v;
}

template <typename T, int N, bool NT = false>
__device__ __forceinline__ void store_upto(typename Traits<T>::store_t *p, const raw_vec_t<T, N> &v, int64_t left) {
  using S = typename Traits<T>::store_t;
  if (left >= N) {
    auto *q = reinterpret_cast<loose_vec_t<S, N> *>(p);
    const loose_vec_t<S, N> w = v;
    if constexpr (NT) __builtin_nontemporal_store(w, q);
    else *q = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < left) p[i] = v[i];
}

// N elements of a type that is known at run time, as fp32; zeros behind `left`.
template <int N>
__device__ __forceinline__ void load_typed(const void *base, int dtype, int64_t off, int64_t left, float (&o)[N]) {
  if (dtype == FLEXSAE_F32) {
    unpack_raw<float, N>(load_upto<float, N>(static_cast<const float *>(base) + off, left), o);
  } else {
    const auto v = load_upto<bf16_t, N>(static_cast<const uint16_t *>(base) + off, left);
    if (dtype == FLEXSAE_BF16) unpack_raw<bf16_t, N>(v, o);
    else unpack_raw<f16_t, N>(v, o);
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

// Blocks beyond the first kGridRow go into further rows of the grid (threads of a grid are counted in 32 bits along an axis).
constexpr int64_t kGridRow = int64_t{1} << 21;
__device__ __forceinline__ int64_t block_index() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6); }

}  // namespace flexsae
