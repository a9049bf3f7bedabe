// Rows of any width and alignment: vectors of 16 bytes, and sums over lanes.
//
// A row of `dim` elements is read in vectors of 16 bytes (8 bf16, 4 fp32) from its
// first element on.  Global loads and stores of 16 bytes need no more than their
// element's alignment on gfx950 (unaligned access mode), so rows of an odd width
// or at an odd offset take the same instructions as aligned ones; only the vector
// that the row ends in goes element by element.
#pragma once

#include "mf_common.h"

namespace mf {

template <typename T> struct RowVec;
template <> struct RowVec<bf16> {
  static constexpr int N = 8;
  typedef bf16 V __attribute__((ext_vector_type(8)));
  typedef bf16 U __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct RowVec<float> {
  static constexpr int N = 4;
  typedef float V __attribute__((ext_vector_type(4)));
  typedef float U __attribute__((ext_vector_type(4), aligned(4)));
};
template <typename T> using Vec = typename RowVec<T>::V;
template <typename T> constexpr int kVec = RowVec<T>::N;

// Elements col .. col + N - 1 of a row of `dim`, `fill` past its end (TAIL: a
// vector may be cut; otherwise it is whole or beyond the row).
template <typename T, bool TAIL, bool STREAM = false>
__device__ __forceinline__ Vec<T> load_row(const T* row, int col, int dim, float fill = 0.f) {
  typedef typename RowVec<T>::U U;
  constexpr int N = kVec<T>;
  Vec<T> v;
  if (col + N <= dim) {
    const U* p = reinterpret_cast<const U*>(row + col);
    const U u = STREAM ? __builtin_nontemporal_load(p) : *p;
    v = u;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)fill;
    if constexpr (TAIL) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (col + i < dim) v[i] = row[col + i];
    }
  }
  return v;
}

template <typename T, bool TAIL, bool STREAM = false>
__device__ __forceinline__ void store_row(T* row, int col, int dim, const float (&x)[kVec<T>]) {
  typedef typename RowVec<T>::U U;
  constexpr int N = kVec<T>;
  if (col + N <= dim) {
    U u;
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = (T)x[i];
    U* p = reinterpret_cast<U*>(row + col);
    if constexpr (STREAM)
      __builtin_nontemporal_store(u, p);
    else
      *p = u;
  } else if constexpr (TAIL) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col + i < dim) row[col + i] = (T)x[i];
  }
}

// Element `i` of an array that holds fp32 or bf16.
__device__ __forceinline__ float element(const void* p, bool f32, size_t i) {
  return f32 ? reinterpret_cast<const float*>(p)[i] : (float)reinterpret_cast<const bf16*>(p)[i];
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}

__device__ __forceinline__ float rows16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rows16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sum over each group of 16 lanes, in all of them: neighbours, pairs, quads
// (mirrored halves), eights (mirrored rows).
__device__ __forceinline__ float sum16(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  return x;
}
__device__ __forceinline__ float sum64(float x) { return halves_sum(rows16_sum(sum16(x))); }

__device__ __forceinline__ float max64(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  x = fmaxf(x, dpp<0x140>(x));
  return halves_max(rows16_max(x));
}

}  // namespace mf
