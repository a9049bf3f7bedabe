// Rows of any width and alignment: vectors of 16 bytes, and sums over lanes.
//
// A row of `dim` elements is taken in vectors of 16 bytes (8 bf16, 4 fp32).  Global loads
// and stores of 16 bytes need no more than their element's alignment on gfx950
// (unaligned access mode), so rows of an odd width or at an odd offset take the same
// instructions as aligned ones.  Loads have no condition: a wait counts the loads
// behind it, and behind a branch it can only wait for all.  A lane whose vector is
// beyond the row loads one inside, and one that the row ends in (EDGE_CUT) takes the
// row's last N elements, those in front of its own twice with another lane.  Rows
// shorter than a vector (EDGE_SHORT) go element by element.
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

enum Edge { EDGE_WHOLE, EDGE_CUT, EDGE_SHORT };

template <typename T>
inline Edge edge_of(int dim) {
  return dim < kVec<T> ? EDGE_SHORT : dim % kVec<T> ? EDGE_CUT : EDGE_WHOLE;
}

// Where the lane that owns vector `v` of a row loads and stores.
template <typename T, Edge E>
struct RowPlace {
  static constexpr int N = kVec<T>;
  int at;    // first element
  int own;   // elements in front of this index in the vector are another lane's; N: all are
  int dim;

  __device__ __forceinline__ RowPlace() {}
  __device__ __forceinline__ RowPlace(int v, int dim_) : dim(dim_) {
    const int col = v * N;
    if constexpr (E == EDGE_SHORT) {
      at = 0;
      own = v == 0 ? 0 : N;
    } else {
      at = min(col, dim - N);
      own = col < dim ? col - at : N;
    }
  }
  __device__ __forceinline__ bool any() const { return own < N; }
  // whether element i counts in sums
  __device__ __forceinline__ bool mine(int i) const {
    if constexpr (E == EDGE_WHOLE) return true;  // (with any())
    if constexpr (E == EDGE_CUT) return i >= own;
    return i < dim;
  }
  template <bool STREAM = false>
  __device__ __forceinline__ Vec<T> load(const T* row) const {
    typedef typename RowVec<T>::U U;
    Vec<T> x;
    if constexpr (E == EDGE_SHORT) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = i < dim ? row[i] : (T)0.f;
    } else {
      const U* p = reinterpret_cast<const U*>(row + at);
      x = STREAM ? __builtin_nontemporal_load(p) : *p;
    }
    return x;
  }
  template <bool STREAM = false>
  __device__ __forceinline__ void store(T* row, const float (&x)[N]) const {
    typedef typename RowVec<T>::U U;
    if (!any()) return;
    if constexpr (E == EDGE_SHORT) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < dim) row[i] = (T)x[i];
    } else {
      U u;
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = (T)x[i];
      U* p = reinterpret_cast<U*>(row + at);
      if constexpr (STREAM)
        __builtin_nontemporal_store(u, p);
      else
        *p = u;
    }
  }
};

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

template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over the wave in 64 bits, in all lanes.
__device__ __forceinline__ double sum64(double x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
#pragma unroll
  for (int rows = 1; rows <= 2; ++rows) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    const auto l = rows == 1 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false)
                             : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = rows == 1 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false)
                             : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    x = __builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]) +
        __builtin_bit_cast(double, (uint64_t)h[1] << 32 | l[1]);
  }
  return x;
}

__device__ __forceinline__ float max64(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  x = fmaxf(x, dpp<0x140>(x));
  return halves_max(rows16_max(x));
}

}  // namespace mf
