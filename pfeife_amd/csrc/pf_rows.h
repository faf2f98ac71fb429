// Copies between matrices whose rows differ in width, for operands that the vector kernels cannot take as they lie.
#pragma once
#include "pf_common.h"

// dst [rows][to_width] = src [rows][width] (contiguous), zeros behind it; elements of `size` 2 or 4 bytes, to_width * size a multiple of
// 16, dst on a boundary of 16 bytes
void pf_rows_widen(const void* src, int64_t rows, int64_t width, void* dst, int64_t to_width, int size, hipStream_t st);
// dst [rows][width] (contiguous) = the first columns of src [rows][ld], 16-bit elements; ld a multiple of 8, src on a boundary of 16 bytes
void pf_rows_narrow(const void* src, int64_t ld, void* dst, int64_t rows, int64_t width, hipStream_t st);

#ifdef __HIPCC__
// 16 bytes that begin at any element (one access: global memory asks for no alignment), of which `left` elements are there; zeros for
// the others
template <typename U> __device__ __forceinline__ uint4 pf_load_loose(const U* from, int64_t left) {
  constexpr int N = 16 / sizeof(U);
  uint4 o;
  if (left >= N) {
    __builtin_memcpy(&o, from, 16);
  } else {
    U v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < left ? from[k] : (U)0;
    __builtin_memcpy(&o, v, 16);
  }
  return o;
}
template <typename U> __device__ __forceinline__ void pf_store_loose(U* to, int64_t left, const uint4& o) {
  constexpr int N = 16 / sizeof(U);
  if (left >= N) {
    __builtin_memcpy(to, &o, 16);
  } else {
    U v[N];
    __builtin_memcpy(v, &o, 16);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < left) to[k] = v[k];
  }
}
#endif
