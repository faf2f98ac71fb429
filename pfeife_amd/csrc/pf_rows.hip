// Copies between matrices whose rows differ in width.  A product over rows that do not begin on 16 bytes would load and store
// element by element; a copy of such an operand or result moves its bytes twice more, 16 at a time on the aligned side.  The other
// side's elements are neighbours, in lines that the neighbouring threads take the rest of.
#include "pf_rows.h"

namespace {

// 16 bytes of dst to a thread
template <typename U>
__global__ __launch_bounds__(256) void rows_widen_kernel(const U* src, int64_t rows, int64_t width, uint4* dst, int64_t to_rows, int64_t to_width, int64_t total) {
  constexpr int N = 16 / sizeof(U);
  const int64_t per = to_width / N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t line = i / per, c = i % per * N, half = line / to_rows, r = line % to_rows;
    U v[N];
    const U* from = src + (half * rows + r) * width + c;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = r < rows && c + k < width ? from[k] : (U)0;
    uint4 o;
    __builtin_memcpy(&o, v, 16);
    dst[i] = o;
  }
}

// Eight neighbours of dst to a thread, which may belong to several rows; the first `head` elements, before a boundary of 16 bytes, and
// the last ones one by one
__global__ __launch_bounds__(256) void rows_narrow_kernel(const uint16_t* src, int64_t ld, uint16_t* dst, int64_t width, int64_t total, int head) {
  const int64_t units = (total - head + 7) / 8 + (head > 0 ? 1 : 0);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < units; i += (int64_t)gridDim.x * 256) {
    const int64_t at = head > 0 ? (i == 0 ? 0 : head + (i - 1) * 8) : i * 8;
    const int many = head > 0 && i == 0 ? head : (total - at < 8 ? (int)(total - at) : 8);
    int64_t r = at / width, c = at % width;
    uint16_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = k < many ? src[r * ld + c] : (uint16_t)0;
      if (++c == width) { c = 0; ++r; }
    }
    if (many == 8) {
      uint4 o;
      __builtin_memcpy(&o, v, 16);
      *(uint4*)(dst + at) = o;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < many) dst[at + k] = v[k];
    }
  }
}

unsigned blocks_of(int64_t units) {
  const int64_t b = (units + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b < 16384 ? b : 16384);
}

}  // namespace

void pf_rows_widen(const void* src, int64_t rows, int64_t width, void* dst, int64_t to_rows, int64_t to_width, int halves, int size, hipStream_t st) {
  const int64_t total = halves * to_rows * (to_width * size / 16);
  if (total == 0) return;
  if (size == 4)
    hipLaunchKernelGGL(rows_widen_kernel<uint32_t>, dim3(blocks_of(total)), dim3(256), 0, st, (const uint32_t*)src, rows, width, (uint4*)dst, to_rows, to_width, total);
  else
    hipLaunchKernelGGL(rows_widen_kernel<uint16_t>, dim3(blocks_of(total)), dim3(256), 0, st, (const uint16_t*)src, rows, width, (uint4*)dst, to_rows, to_width, total);
}

void pf_rows_narrow(const void* src, int64_t ld, void* dst, int64_t rows, int64_t width, hipStream_t st) {
  const int64_t total = rows * width;
  if (total == 0) return;
  int64_t head = (16 - (int64_t)((uintptr_t)dst & 15)) % 16 / 2;
  if (head > total) head = total;
  hipLaunchKernelGGL(rows_narrow_kernel, dim3(blocks_of(total / 8 + 2)), dim3(256), 0, st, (const uint16_t*)src, ld, (uint16_t*)dst, width, total, (int)head);
}
