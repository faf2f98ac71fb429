// Copies between matrices whose rows differ in width.  A product over rows that do not begin on 16 bytes would load and store
// element by element; a copy of such an operand or result moves its bytes twice more, 16 at a time on either side, on any element's
// boundary on one of them (49999 x 1000 to 1024, 16 bits: 31 us; element by element on that side 54).
#include "pf_rows.h"

namespace {

// 16 bytes of dst to a thread
template <typename U>
__global__ __launch_bounds__(256) void rows_widen_kernel(const U* src, int64_t width, uint4* dst, uint32_t per, uint32_t total) {
  constexpr int N = 16 / sizeof(U);
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const uint32_t r = i / per;
    const int64_t c = (int64_t)(i % per) * N;
    dst[i] = pf_load_loose(src + r * width + c, width - c);
  }
}

// 16 bytes of src to a thread
__global__ __launch_bounds__(256) void rows_narrow_kernel(const uint4* src, uint32_t per_src, uint16_t* dst, int64_t width, uint32_t per, uint32_t total) {
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const uint32_t r = i / per;
    const int64_t c = (int64_t)(i % per) * 8;
    pf_store_loose(dst + r * width + c, width - c, src[(int64_t)r * per_src + i % per]);
  }
}

unsigned blocks_of(int64_t units) {
  const int64_t b = (units + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b < 16384 ? b : 16384);
}

constexpr int64_t MOST = 1ll << 30;      // units of a launch

template <typename U>
void widen(const void* src, int64_t rows, int64_t width, void* dst, int64_t to_width, hipStream_t st) {
  const int64_t per = to_width * (int64_t)sizeof(U) / 16, step = MOST / per;
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t n = rows - r < step ? rows - r : step;
    hipLaunchKernelGGL(rows_widen_kernel<U>, dim3(blocks_of(n * per)), dim3(256), 0, st, (const U*)src + r * width, width, (uint4*)dst + r * per, (uint32_t)per,
                       (uint32_t)(n * per));
  }
}

}  // namespace

void pf_rows_widen(const void* src, int64_t rows, int64_t width, void* dst, int64_t to_width, int size, hipStream_t st) {
  if (size == 4) widen<uint32_t>(src, rows, width, dst, to_width, st);
  else widen<uint16_t>(src, rows, width, dst, to_width, st);
}

void pf_rows_narrow(const void* src, int64_t ld, void* dst, int64_t rows, int64_t width, hipStream_t st) {
  const int64_t per = (width + 7) / 8, step = MOST / per;
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t n = rows - r < step ? rows - r : step;
    hipLaunchKernelGGL(rows_narrow_kernel, dim3(blocks_of(n * per)), dim3(256), 0, st, (const uint4*)src + r * (ld / 8), (uint32_t)(ld / 8), (uint16_t*)dst + r * width, width,
                       (uint32_t)per, (uint32_t)(n * per));
  }
}
