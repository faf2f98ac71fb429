// The gated projection's matrix products, one object file per 16-bit operand type.
#pragma once
#include "pf_common.h"

enum { PF_KEEP_NONE = 0, PF_KEEP_SAME = 1, PF_KEEP_8BIT = 2 };
#define PF_GATED_BLOCK 16      // neighbouring columns that share an exponent

// y = act(x Wg^T) * (x Wu^T) and what is kept of the two products
struct PfGatedProduct {
  int64_t rows, depth, ffn;    // depth a multiple of 8, at least 64
  const void* x;
  int64_t ldx;
  const void* w;               // [2 ffn][ldw], the gate's rows first
  int64_t ldw;
  int act, keep;
  void* y;
  int64_t ldy;
  void* kept;                  // the two halves of a row side by side, each `half` columns; with 8 bits codes
  int64_t half;                // a multiple of 8 (8 bits: of 16)
  uint8_t* exps;               // 8 bits: exponents + 127, those of four rows' same columns side by side: [rows / 4][2 half / 16][4]
};
int pf_gated_forward_1(const PfGatedProduct& p, hipStream_t st);
int pf_gated_forward_2(const PfGatedProduct& p, hipStream_t st);
// C[M][N] (16 bits) = A^T B over K rows, A [K][lda], B [K][ldb]; batch: so many of them, `step` columns of A apart, their results one behind
// the other
int pf_gated_weight_1(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int batch, int64_t step, hipStream_t st);
int pf_gated_weight_2(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int batch, int64_t step, hipStream_t st);

#ifdef __HIPCC__
// 1 / (1 + e^-x) by one exponential and one reciprocal of the hardware, each off by a unit in the last place: far below what
// 16-bit results can hold.  (The forward product's epilogue waits for these: 8192 x 2048 x 5632 332 us with the library's exponential and
// division, 313 with this.)  -inf and +inf give 0 and 1.
__device__ __forceinline__ float pf_sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }
__device__ __forceinline__ float pf_silu_fast(float x) { return x * pf_sigmoid_fast(x); }
// 2^e for e + 127 in 1 .. 254
__device__ __forceinline__ float pf_pow2(int biased) { return __uint_as_float((uint32_t)biased << 23); }
// The biased exponent of the smallest power of two that brings `top` to 448 (the largest e4m3) or below; 127 for zero
__device__ __forceinline__ int pf_e4m3_exponent(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);     // 448 = 1.75 * 2^8
  return top == 0.f ? 127 : (e < 1 ? 1 : e > 253 ? 253 : e);
}
#endif
