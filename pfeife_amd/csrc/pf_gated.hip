// Gated projection y = act(x Wg^T) * (x Wu^T), weight [2 ffn, D] with the gate's rows first, and its backward pass.
//
//   g = x Wg^T, u = x Wu^T (fp32);  y = act(g) u
//   dg = dy u act'(g);  du = dy act(g);  dx = [dg du] W;  dW = [dg du]^T x
//
// The backward pass starts from g and u as they were kept: in the operands' type, or (16-bit operands) as e4m3 codes, 16 neighbouring columns
// of a row under one power of two, 17 instead of 32 bytes for 16 of them.  The power of two is the smallest that brings the
// largest of the 16 to 448 or below, so that nothing saturates, and decoding is exact.  The pass over the elements that
// makes dg and du reads the codes as they are: 4.1 bytes instead of 6 an element of y, and 4 written.
#include "pf_gated.h"
#include "pf_gemm_common.h"
#include "pf_rows.h"

namespace {

inline int64_t round_up(int64_t n, int64_t k) { return (n + k - 1) / k * k; }

template <int ACT> __device__ __forceinline__ void act_and_slope(float g, float& value, float& slope) {
  if constexpr (ACT == PF_ACT_SILU) {
    const float p = pf_sigmoid_fast(g);
    value = g * p;
    slope = p * (1.f + g * (1.f - p));
  } else {
    value = ACT == PF_ACT_RELU && g != g ? g : pf_act(ACT, g);
    slope = pf_act_grad(ACT, g);
  }
}

// W neighbouring values of what was kept
template <int DT, int KEEP, int W>
__device__ __forceinline__ void kept_load(const void* kept, const uint8_t* exps, int64_t half, int64_t row, int64_t at, float (&v)[W]) {
  if constexpr (KEEP == PF_KEEP_SAME) {
    Vec8<DT>::load(kept, row * 2 * half + at, v);
  } else {
    const uint2 c = *(const uint2*)((const uint8_t*)kept + row * 2 * half + at);
    const float by = pf_pow2(exps[(row / 4 * 2 * half + at) / PF_GATED_BLOCK * 4 + row % 4]);
    v[0] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 0) * by; v[1] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 1) * by;
    v[2] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 2) * by; v[3] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 3) * by;
    v[4] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 0) * by; v[5] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 1) * by;
    v[6] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 2) * by; v[7] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 3) * by;
  }
}

// dg and du side by side in rows of 2 wide columns (zeros past ffn), eight columns of a row to a thread; bound by memory: 8192 x 5632, bf16:
// 79 us, 461 MB at 5.8 TB/s; from 8-bit codes 16384 rows in 128 us, 750 MB
template <int DT, int KEEP, int ACT>
__global__ __launch_bounds__(256) void gated_backward_kernel(const void* dy, const void* kept, const uint8_t* exps, int64_t half, int64_t rows, int64_t ffn,
                                                             void* dgu, int64_t wide) {
  const int64_t per = wide / 8, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per, c = i % per * 8;
    float d[8], g[8], u[8], dg[8], du[8];
    const uint4 bits = pf_load_loose((const uint16_t*)dy + row * ffn + c, ffn - c);
    Vec8<DT>::load(&bits, 0, d);
    kept_load<DT, KEEP, 8>(kept, exps, half, row, c, g);
    kept_load<DT, KEEP, 8>(kept, exps, half, row, half + c, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float value, slope;
      act_and_slope<ACT>(g[k], value, slope);
      const bool in = c + k < ffn;      // (what is kept past the last column may be anything)
      dg[k] = in ? d[k] * u[k] * slope : 0.f;
      du[k] = in ? d[k] * value : 0.f;
    }
    Vec8<DT>::store(dgu, row * 2 * wide + c, dg);
    Vec8<DT>::store(dgu, row * 2 * wide + wide + c, du);
  }
}

template <int DT, int KEEP>
void backward_launch(const void* dy, const void* kept, const uint8_t* exps, int64_t half, int64_t rows, int64_t ffn, void* dgu, int64_t wide, int act, hipStream_t st) {
  const int64_t blocks = (rows * (wide / 8) + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
#define PF_GB(A) hipLaunchKernelGGL((gated_backward_kernel<DT, KEEP, A>), grid, dim3(256), 0, st, dy, kept, exps, half, rows, ffn, dgu, wide)
  switch (act) {
    case PF_ACT_SILU: PF_GB(PF_ACT_SILU); break;
    case PF_ACT_GELU: PF_GB(PF_ACT_GELU); break;
    case PF_ACT_GELU_TANH: PF_GB(PF_ACT_GELU_TANH); break;
    default: PF_GB(PF_ACT_RELU); break;
  }
#undef PF_GB
}

void split_launch(int dtype, int keep, const void* dy, const void* kept, int64_t half, int64_t rows, int64_t ffn, void* dgu, int64_t wide, int act, hipStream_t st) {
  const uint8_t* exps = keep == PF_KEEP_8BIT ? (const uint8_t*)kept + rows * 2 * half : nullptr;
  if (dtype == PF_F16) {
    if (keep == PF_KEEP_SAME) backward_launch<PF_F16, PF_KEEP_SAME>(dy, kept, exps, half, rows, ffn, dgu, wide, act, st);
    else backward_launch<PF_F16, PF_KEEP_8BIT>(dy, kept, exps, half, rows, ffn, dgu, wide, act, st);
  } else {
    if (keep == PF_KEEP_SAME) backward_launch<PF_BF16, PF_KEEP_SAME>(dy, kept, exps, half, rows, ffn, dgu, wide, act, st);
    else backward_launch<PF_BF16, PF_KEEP_8BIT>(dy, kept, exps, half, rows, ffn, dgu, wide, act, st);
  }
}

// Both halves of the weight transposed, 64 x 64 elements to a workgroup: wt[d][z * wide + f] = w[z * ffn + f][d], zeros for f from ffn to wide
// (2 x 2732 x 1000: 6.4 us, where a fill and a transpose for each half took 13.6)
__global__ __launch_bounds__(256) void gated_transpose_kernel(const uint16_t* w, int64_t ffn, int64_t D, uint16_t* wt, int64_t wide) {
  __shared__ __align__(16) uint16_t tile[64][66];
  const int t = threadIdx.x;
  const int64_t d0 = (int64_t)blockIdx.x * 64, f0 = (int64_t)blockIdx.y * 64, z = blockIdx.z;
#pragma unroll
  for (int i = t >> 3; i < 64; i += 32) {
    const int64_t f = f0 + i, d = d0 + (t & 7) * 8;
    const uint16_t* from = w + (z * ffn + f) * D + d;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (f < ffn && d < D) v = pf_load_loose(from, D - d);
    uint32_t* to = (uint32_t*)&tile[i][(t & 7) * 8];
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  }
  __syncthreads();
#pragma unroll
  for (int i = t >> 3; i < 64; i += 32) {
    const int64_t d = d0 + i, f = f0 + (t & 7) * 8;
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (uint32_t)tile[(t & 7) * 8 + 2 * j][i] | (uint32_t)tile[(t & 7) * 8 + 2 * j + 1][i] << 16;
    if (d < D && f < wide) *(uint4*)(wt + d * 2 * wide + z * wide + f) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// dx from the sums of its shares, [splits][rows][ld] in fp32
template <int W>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* acc, int64_t ld, int splits, int64_t rows, int64_t D, void* dx, int dt) {
  const int64_t per = (D + 64 * W - 1) / (64 * W), total = rows * per;      // (a wavefront to 64 W columns of a row)
  for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < total; q += (int64_t)gridDim.x * 4) {
    const int64_t r = q / per, i = q % per * 64 * W + (threadIdx.x & 63) * W;
    if (i >= D) continue;
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = 0.f;
#pragma unroll 4
    for (int p = 0; p < splits; ++p) {
      float w[W];
      ld_vec<W>(acc, (p * rows + r) * ld + i, PF_F32, w);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += w[k];
    }
    st_vec<W>(dx, r * D + i, dt, v);
  }
}

// What a few rows' kernel left in fp32 as it is kept: a thread to 16 columns of one half of a row
__global__ __launch_bounds__(256) void gated_encode_kernel(const float* gu, int64_t rows, int64_t ffn, int64_t half, uint8_t* codes, uint8_t* exps) {
  const int64_t per = half / PF_GATED_BLOCK, total = rows * 2 * per;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / (2 * per), block = i % (2 * per), c = block % per * PF_GATED_BLOCK;
  const float* from = gu + row * 2 * half + block * PF_GATED_BLOCK;
  float v[PF_GATED_BLOCK], top = 0.f;
#pragma unroll
  for (int k = 0; k < PF_GATED_BLOCK; ++k) {
    v[k] = c + k < ffn ? from[k] : 0.f;
    top = fmaxf(top, fabsf(v[k]));
  }
  const int e = pf_e4m3_exponent(top);
  const float by = pf_pow2(254 - e);
  int w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k] * by, v[4 * k + 1] * by, 0, false);
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2] * by, v[4 * k + 3] * by, w[k], true);
  }
  *(int4*)(codes + row * 2 * half + block * PF_GATED_BLOCK) = make_int4(w[0], w[1], w[2], w[3]);
  exps[(row / 4 * 2 * per + block) * 4 + row % 4] = (uint8_t)e;
}

// A few rows: a wavefront takes a column of y, i.e. one row of either half of the weight, and R rows of x from LDS.  Bound by the
// weight's way from memory: all of a wavefront's loads are independent, and ffn wavefronts are on their way at once (one row, 2048 to
// 5632, bf16: 46 MB in 9.7 us).
// kept_f32: both products as they are, for the 8-bit codes.
template <int DT, int R>
__global__ __launch_bounds__(256) void gated_few_kernel(const void* x, const void* w, int64_t depth, int64_t rows, int64_t ffn, int act, void* y, void* kept, int64_t half,
                                                        int kept_f32) {
  extern __shared__ __align__(16) char xs[];
  typedef typename Codec<DT>::storage S;
  for (int64_t i = (int64_t)threadIdx.x * 8; i < R * depth; i += 256 * 8) {
    float v[8] = {};
    if (i < rows * depth) Vec8<DT>::load(x, i, v);
    Vec8<DT>::store(xs, i, v);
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (f >= ffn) return;
  const S* wg = (const S*)w + f * depth;
  const S* wu = (const S*)w + (ffn + f) * depth;
  float g[R], u[R];
#pragma unroll
  for (int r = 0; r < R; ++r) g[r] = u[r] = 0.f;
#pragma unroll 4
  for (int64_t k = lane * 8; k < depth; k += 512) {
    float a[8], b[8];
    Vec8<DT>::load(wg, k, a);
    Vec8<DT>::load(wu, k, b);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[8];
      Vec8<DT>::load(xs, r * depth + k, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) { g[r] = fmaf(a[q], v[q], g[r]); u[r] = fmaf(b[q], v[q], u[r]); }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float gs = pf_wave_sum(g[r]), us = pf_wave_sum(u[r]);
    if (lane == 0 && r < rows) {
      const float v = act == PF_ACT_RELU && gs != gs ? gs : pf_act(act, gs);
      Codec<DT>::store(y, r * ffn + f, v * us);
      if (kept != nullptr && kept_f32) {
        ((float*)kept)[r * 2 * half + f] = gs;
        ((float*)kept)[r * 2 * half + half + f] = us;
      } else if (kept != nullptr) {
        Codec<DT>::store(kept, r * 2 * half + f, gs);
        Codec<DT>::store(kept, r * 2 * half + half + f, us);
      }
    }
  }
}
template <int DT, int R>
int few_launch(const void* x, const void* w, int64_t depth, int64_t rows, int64_t ffn, int act, void* y, void* kept, int64_t half, int kept_f32, hipStream_t st) {
  const size_t lds = (size_t)(R * depth * pf_dtype_size(DT));
  hipLaunchKernelGGL((gated_few_kernel<DT, R>), dim3((unsigned)((ffn + 3) / 4)), dim3(256), lds, st, x, w, depth, rows, ffn, act, y, kept, half, kept_f32);
  PF_CHECK_LAUNCH("pf_gated_linear_fwd");
  return PF_OK;
}
// How many rows such a launch would hold in LDS, 0: it cannot run, or the product's 64x64 tile is no slower.  us of either, bf16: one row, 2048 to 5632 9.7
// and 12.3, 4096 to 11008 27.9 and 31; two 10.8 and 12.3, 30.5 and 31; three 12.6 and 12.3, 39 and 31
int few_rows(int64_t rows, int64_t depth, int64_t es) {
  const int r = rows <= 2 ? (int)rows : 0;
  return depth % 8 == 0 && r * depth * es <= 64 * 1024 ? r : 0;
}
template <int DT>
int few(int r, const void* x, const void* w, int64_t depth, int64_t rows, int64_t ffn, int act, void* y, void* kept, int64_t half, int kept_f32, hipStream_t st) {
  return r == 1 ? few_launch<DT, 1>(x, w, depth, rows, ffn, act, y, kept, half, kept_f32, st) : few_launch<DT, 2>(x, w, depth, rows, ffn, act, y, kept, half, kept_f32, st);
}

// A few rows' backward pass in 16 bits, without a transposed weight and without copies of odd widths: bound by the weight's way from memory and its gradient's
// way there.  us, 2048 to 5632, bf16: dx with its join 21 for one row, 26 for four, 35 for eight, where transpose, product and join take 31; the weight's
// gradient 10, 11 and 15, 22 for sixteen, and as a matrix product 36.
constexpr int FEW_DX = 4, FEW_DW = 16, FEW_PARTS = 64;

// dx's shares: a wavefront takes 512 columns and every so many 32 rows of the weight, a workgroup's four wavefronts add up in LDS; part [share][row][ld]
template <int DT, int R>
__global__ __launch_bounds__(256) void gated_few_dx_kernel(const uint16_t* __restrict__ dgu, int64_t wide, const uint16_t* __restrict__ w, int64_t rows, int64_t ffn, int64_t D, float* __restrict__ part,
                                                           int64_t ld) {
  __shared__ float sums[3][R][512];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t c = (int64_t)blockIdx.x * 512 + lane * 8, left = D - c, blocks = (ffn + 31) / 32;
  float acc[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[r][k] = 0.f;
  for (int64_t q = (int64_t)blockIdx.y * 4 + wave; q < 2 * blocks; q += (int64_t)gridDim.y * 4) {
    const int64_t z = q / blocks, k0 = q % blocks * 32, k1 = k0 + 32 < ffn ? k0 + 32 : ffn;
    for (int64_t k = k0; k < k1; k += 8) {      // (columns of dg and du past ffn are zeros up to a multiple of 8)
      float v[8][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint4 bits = left > 0 ? pf_load_loose(w + (z * ffn + (k + j < ffn ? k + j : ffn - 1)) * D + c, left) : make_uint4(0, 0, 0, 0);
        Vec8<DT>::load(&bits, 0, v[j]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float d[8];
        Vec8<DT>::load(dgu, (r < rows ? r : rows - 1) * 2 * wide + z * wide + k, d);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(d[j], v[j][e], acc[r][e]);
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[wave - 1][r][e * 64 + lane] = acc[r][e];
  }
  __syncthreads();
  if (wave > 0 || left <= 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] += sums[s][r][e * 64 + lane];
    Vec8<PF_F32>::store(part, (blockIdx.y * rows + r) * ld + c, acc[r]);
  }
}

// The weight's gradient: a wavefront takes 16 of its rows and 512 columns
template <int DT>
__global__ __launch_bounds__(256) void gated_few_dw_kernel(const uint16_t* __restrict__ dgu, int64_t wide, const uint16_t* __restrict__ x, int64_t rows, int64_t ffn, int64_t D,
                                                           uint16_t* __restrict__ dw) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t f0 = ((int64_t)blockIdx.x * 4 + wave) * 16, c = (int64_t)blockIdx.y * 512 + (threadIdx.x & 63) * 8, z = blockIdx.z;
  if (f0 >= ffn || c >= D) return;
  float acc[16][8];
#pragma unroll
  for (int f = 0; f < 16; ++f)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[f][e] = 0.f;
#pragma unroll 2
  for (int64_t r = 0; r < rows; ++r) {
    float v[8], d[16];
    const uint4 bits = pf_load_loose(x + r * D + c, D - c);
    Vec8<DT>::load(&bits, 0, v);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float half[8];
      Vec8<DT>::load(dgu, r * 2 * wide + z * wide + (f0 + 8 * h < wide ? f0 + 8 * h : f0), half);
#pragma unroll
      for (int k = 0; k < 8; ++k) d[8 * h + k] = half[k];
    }
#pragma unroll
    for (int f = 0; f < 16; ++f)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[f][e] = fmaf(d[f], v[e], acc[f][e]);
  }
#pragma unroll
  for (int f = 0; f < 16; ++f)
    if (f0 + f < ffn) {
      uint4 o;
      Vec8<DT>::store(&o, 0, acc[f]);
      pf_store_loose(dw + (z * ffn + f0 + f) * D + c, D - c, o);
    }
}

template <int DT>
void few_dx(const void* dgu, int64_t wide, const void* w, int64_t rows, int64_t ffn, int64_t D, float* part, int64_t ld, int parts, hipStream_t st) {
  const dim3 grid((unsigned)((D + 511) / 512), (unsigned)parts);
  if (rows == 1)
    hipLaunchKernelGGL((gated_few_dx_kernel<DT, 1>), grid, dim3(256), 0, st, (const uint16_t*)dgu, wide, (const uint16_t*)w, rows, ffn, D, part, ld);
  else
    hipLaunchKernelGGL((gated_few_dx_kernel<DT, FEW_DX>), grid, dim3(256), 0, st, (const uint16_t*)dgu, wide, (const uint16_t*)w, rows, ffn, D, part, ld);
}
template <int DT>
void few_dw(const void* dgu, int64_t wide, const void* x, int64_t rows, int64_t ffn, int64_t D, void* dw, hipStream_t st) {
  hipLaunchKernelGGL(gated_few_dw_kernel<DT>, dim3((unsigned)((ffn + 63) / 64), (unsigned)((D + 511) / 512), 2), dim3(256), 0, st, (const uint16_t*)dgu, wide,
                     (const uint16_t*)x, rows, ffn, D, (uint16_t*)dw);
}

// What lies where.  depth: the width of the rows that the products read, of x and of the weight, which are copied where theirs is
// another (16 bytes have to lie at their front); wide: that of one half of dg and du, and with 16 bits of the transposed weight; half: that
// of one half of what is kept.
int64_t half_of(int dtype, int64_t ffn, int keep) { return round_up(ffn, keep == PF_KEEP_8BIT ? PF_GATED_BLOCK : dtype == PF_F32 ? 4 : 8); }
int64_t kept_bytes(int dtype, int64_t rows, int64_t ffn, int keep) {
  const int64_t half = half_of(dtype, ffn, keep);
  return keep == PF_KEEP_8BIT ? rows * 2 * half + (rows + 3) / 4 * 4 * (2 * half / PF_GATED_BLOCK) : rows * 2 * half * (dtype == PF_F32 ? 4 : 2);
}
struct Plan {
  int64_t es, depth, wide, half, chunk;
  bool copy_x, copy_w, narrow;
  bool few_dx, few_dw;         // kernels of a few rows
  int splits;                  // of dx's sums (with `parts`)
  char* x; char* w; char* wt; char* dgu; char* dw; float* parts; float* gu;
  int64_t bytes;
};

int check(const char* who, int dtype, int64_t rows, int64_t D, int64_t ffn, int act, int keep) {
  PF_REQUIRE(dtype == PF_F32 || dtype == PF_F16 || dtype == PF_BF16, "%s: bad dtype", who);
  PF_REQUIRE(rows >= 0 && D > 0 && ffn > 0, "%s: bad sizes", who);
  PF_REQUIRE(act >= PF_ACT_GELU && act <= PF_ACT_RELU, "%s: bad activation", who);
  PF_REQUIRE(keep >= PF_KEEP_NONE && keep <= PF_KEEP_8BIT && (keep != PF_KEEP_8BIT || dtype != PF_F32), "%s: fp32 is not kept in 8 bits", who);
  return PF_OK;
}
int too_large(const char* who) {
  pf_set_error("%s: too large for one call: the weight, and with a gradient the kept rows and x, have to stay below 2 GiB each", who);
  return PF_ERR_INVALID;
}

// batch: shares of the depth, with results of their own; what does not divide is added to the first
int product(int dtype, int c_dtype, int a_trans, int b_trans, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb, void* C,
            int64_t ldc, int beta, hipStream_t st, int splits = 1) {
  pf_gemm_desc d = {};
  d.in_dtype = dtype;
  d.c_dtype = c_dtype;
  d.a_trans = a_trans; d.b_trans = b_trans;
  d.M = M; d.N = N; d.K = K;
  d.A = A; d.lda = lda; d.B = B; d.ldb = ldb; d.C = C; d.ldc = ldc;
  d.batch1 = d.batch2 = 1;
  d.alpha = 1.f;
  d.beta = beta;
  const int64_t share = splits > 1 ? K / splits / 64 * 64 : 0;
  if (share == 0) return pf_gemm(&d, st);
  const int64_t es = dtype == PF_F32 ? 4 : 2;
  d.K = share;
  d.batch2 = splits;
  d.a_stride2 = share * (a_trans ? lda : 1);
  d.b_stride2 = share * (b_trans ? ldb : 1);
  d.c_stride2 = M * ldc;
  const int rc = pf_gemm(&d, st);
  if (rc != PF_OK || share * splits == K) return rc;
  d.K = K - share * splits;
  d.batch2 = 1;
  d.A = (const char*)A + splits * d.a_stride2 * es;
  d.B = (const char*)B + splits * d.b_stride2 * es;
  d.beta = 1;
  return pf_gemm(&d, st);
}

// In how many shares dx is best summed: few rows make few tiles, whose depth is both halves of the weight
int splits_of(int dtype, int64_t rows, int64_t D, int64_t K) {
  int best = 1;
  double best_t = 0;
  for (int s = 1; s <= 16 && (s == 1 || K / s >= 256); ++s) {
    double t = 0;
    pf_gemm_desc d = {};
    d.in_dtype = dtype;
    d.c_dtype = PF_F32;
    d.M = rows; d.N = D; d.K = K / s / 64 * 64 > 0 ? K / s / 64 * 64 : K;
    d.batch1 = 1;
    d.batch2 = s;
    if (dtype == PF_F32) {
      t = pf_gemm_f32_depth_us(d);
    } else {
      pf_gemm_best_tile(d, &t);
    }
    if (s > 1) t += 4.0 + (double)(rows * D) * s * 8.0 / 5.0e6;      // a launch, and the shares' way through memory at 5 TB/s
    if (s > 1 && K / s / 64 * 64 * s != K) t += 5.0;                 // another for what does not divide
    if (s == 1 || t < best_t) { best = s; best_t = t; }
  }
  return best;
}

bool plan_of(Plan& p, const void* x, const void* w, int dtype, int64_t rows, int64_t D, int64_t ffn, int keep, bool back, char* base) {
  const bool f32 = dtype == PF_F32;
  p.es = f32 ? 4 : 2;
  p.depth = f32 ? round_up(D, 4) : (D < 64 ? 64 : round_up(D, 8));
  p.wide = round_up(ffn, f32 ? 4 : 8);
  p.half = half_of(dtype, ffn, keep);
  p.copy_x = p.depth != D || !pf_aligned(x, 16);
  p.copy_w = p.depth != D || !pf_aligned(w, 16);
  // Whole stages of the fastest tile, where both operands are copied anyway and where many rows pay for the copies.  us of a forward and a backward pass, 1000 to
  // 2736, bf16, without and with: 2048 rows 151 and 148, 4096 208 and 211, 8192 366 and 352
  if (!f32 && rows > 128 && ((p.copy_x && p.copy_w) || rows >= 8192) && p.depth % 64 != 0) {
    p.depth = round_up(p.depth, 64);
    p.copy_x = p.copy_w = true;
  }
  p.few_dx = back && !f32 && rows <= FEW_DX;
  p.few_dw = back && !f32 && rows <= FEW_DW;
  p.narrow = !f32 && D % 8 != 0;
  const int64_t blocks = (ffn + 31) / 32 * 2;      // (of the weight's rows, to four wavefronts each)
  const int64_t deep = f32 && p.wide != ffn ? ffn : 2 * p.wide;      // (16 bits: one sum over both halves, whatever ffn is)
  p.splits = !back ? 1 : p.few_dx ? (int)(blocks < 4 * FEW_PARTS ? (blocks + 3) / 4 : FEW_PARTS) : splits_of(dtype, rows, D, deep);
  // rows of one launch: everything it addresses by 32-bit offsets stays below 2 GiB
  const int64_t widest = p.depth > 2 * p.half ? p.depth : 2 * p.half;
  p.chunk = ((1ll << 31) / (widest * p.es) - 512) / 256 * 256;
  p.x = p.w = p.wt = p.dgu = p.dw = nullptr;
  p.parts = p.gu = nullptr;
  int64_t used = 0;
  auto take = [&](int64_t bytes) {
    char* q = base == nullptr ? nullptr : base + used;
    used += round_up(bytes, 256);
    return q;
  };
  // (the 16-bit backward pass reads x as the right-hand operand of a reduction over its rows, and of the weight a transposed copy)
  const bool x_as_is = back && !f32 && D % 8 == 0 && pf_aligned(x, 16);
  if (p.copy_x && !x_as_is && !p.few_dw) p.x = take(rows * p.depth * p.es);
  if (p.copy_w && (!back || f32)) p.w = take(2 * ffn * p.depth * p.es);
  if (back) {
    p.dgu = take(rows * 2 * p.wide * p.es);
    if (!f32 && !p.few_dx) p.wt = take(p.depth * 2 * p.wide * 2);
    if (p.narrow && !p.few_dw) p.dw = take(2 * ffn * p.depth * 2);
    if (p.splits > 1 || p.narrow || p.few_dx) p.parts = (float*)take(p.splits * rows * p.depth * 4);
  } else if (keep == PF_KEEP_8BIT && few_rows(rows, p.depth, 2) > 0) {
    p.gu = (float*)take(rows * 2 * p.half * 4);
  } else if (f32 && keep == PF_KEEP_NONE) {
    p.dgu = take(rows * 2 * p.wide * 4);
  }
  p.bytes = used;
  return p.depth < (1ll << 19) && p.half < (1ll << 18) && p.chunk > 0 && (2 * ffn + 512) * p.depth * 2 < (1ll << 31) && (p.depth + 512) * 2 * p.wide * 2 < (1ll << 31) &&
         (keep == PF_KEEP_NONE ? rows < (1ll << 31) : f32 || rows <= p.chunk);
}

}  // namespace

extern "C" int64_t pf_gated_linear_kept(int dtype, int64_t rows, int64_t ffn, int keep) {
  const int rc = check("pf_gated_linear_kept", dtype, rows, 1, ffn, PF_ACT_SILU, keep);
  if (rc != PF_OK || keep == PF_KEEP_NONE) return rc;
  return kept_bytes(dtype, rows, ffn, keep);
}

extern "C" int64_t pf_gated_linear_workspace(const void* x, const void* weight, int dtype, int64_t rows, int64_t D, int64_t ffn, int keep, int backward) {
  const char* who = "pf_gated_linear_workspace";
  const int rc = check(who, dtype, rows, D, ffn, PF_ACT_SILU, keep);
  if (rc != PF_OK) return rc;
  Plan p;
  if (!plan_of(p, x, weight, dtype, rows, D, ffn, keep, backward != 0, nullptr)) return too_large(who);
  return p.bytes;
}

extern "C" int pf_gated_linear_fwd(const void* x, int dtype, int64_t rows, int64_t D, const void* weight, int64_t ffn, int act, int keep, void* y, void* kept,
                                   void* workspace, void* stream) {
  const char* who = "pf_gated_linear_fwd";
  int rc = check(who, dtype, rows, D, ffn, act, keep);
  if (rc != PF_OK || rows == 0) return rc;
  Plan p;
  if (!plan_of(p, x, weight, dtype, rows, D, ffn, keep, false, (char*)workspace)) return too_large(who);
  PF_REQUIRE(x && weight && y && (keep == PF_KEEP_NONE || kept) && (p.bytes == 0 || workspace), "%s: null pointer", who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(workspace, 16), "%s: kept and the workspace lie on boundaries of 16 and 256 bytes", who);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PF_F32) {
    const int r = D % 8 == 0 && !p.copy_x && !p.copy_w ? few_rows(rows, D, 4) : 0;
    if (r > 0) return few<PF_F32>(r, x, weight, D, rows, ffn, act, y, kept, p.half, 0, st);
    if (p.copy_x) pf_rows_widen(x, rows, D, p.x, p.depth, 4, st);
    if (p.copy_w) pf_rows_widen(weight, 2 * ffn, D, p.w, p.depth, 4, st);
    const float* xs = p.copy_x ? (const float*)p.x : (const float*)x;
    const float* ws = p.copy_w ? (const float*)p.w : (const float*)weight;
    float* gu = keep == PF_KEEP_NONE ? (float*)p.dgu : (float*)kept;
    if (p.wide == ffn) {
      rc = product(PF_F32, PF_F32, 0, 0, rows, 2 * ffn, D, xs, p.depth, ws, p.depth, gu, 2 * ffn, 0, st);
    } else {
      for (int h = 0; h < 2 && rc == PF_OK; ++h)
        rc = product(PF_F32, PF_F32, 0, 0, rows, ffn, D, xs, p.depth, ws + h * ffn * p.depth, p.depth, gu + h * p.wide, 2 * p.wide, 0, st);
    }
    if (rc != PF_OK) return rc;
    return pf_glu_fwd(gu, 2 * p.wide, gu + p.wide, 2 * p.wide, y, ffn, PF_F32, act, rows, ffn, stream);
  }
  if (p.copy_x) pf_rows_widen(x, rows, D, p.x, p.depth, 2, st);
  if (p.copy_w) pf_rows_widen(weight, 2 * ffn, D, p.w, p.depth, 2, st);
  PF_CHECK_LAUNCH(who);
  const int r = few_rows(rows, p.depth, 2);
  if (r > 0) {
    const void* xs = p.copy_x ? p.x : x;
    const void* ws = p.copy_w ? p.w : weight;
    const int codes = keep == PF_KEEP_8BIT;
    void* to = codes ? (void*)p.gu : kept;
    rc = dtype == PF_F16 ? few<PF_F16>(r, xs, ws, p.depth, rows, ffn, act, y, to, p.half, codes, st) : few<PF_BF16>(r, xs, ws, p.depth, rows, ffn, act, y, to, p.half, codes, st);
    if (rc != PF_OK || !codes) return rc;
    hipLaunchKernelGGL(gated_encode_kernel, dim3((unsigned)((rows * 2 * p.half / PF_GATED_BLOCK + 255) / 256)), dim3(256), 0, st, p.gu, rows, ffn, p.half, (uint8_t*)kept,
                       (uint8_t*)kept + rows * 2 * p.half);
    PF_CHECK_LAUNCH(who);
    return PF_OK;
  }
  const int64_t row_k = 2 * p.half * (keep == PF_KEEP_8BIT ? 1 : 2);
  for (int64_t r = 0; r < rows; r += p.chunk) {
    PfGatedProduct q = {};
    q.rows = rows - r < p.chunk ? rows - r : p.chunk;
    q.depth = p.depth; q.ffn = ffn;
    q.x = (p.copy_x ? p.x : (const char*)x) + r * p.depth * 2; q.ldx = p.depth;
    q.w = p.copy_w ? p.w : weight; q.ldw = p.depth;
    q.act = act; q.keep = keep;
    q.y = (char*)y + r * ffn * 2; q.ldy = ffn;
    q.kept = keep == PF_KEEP_NONE ? nullptr : (char*)kept + r * row_k;
    q.half = p.half;
    q.exps = keep == PF_KEEP_8BIT ? (uint8_t*)kept + rows * 2 * p.half + r * (2 * p.half / PF_GATED_BLOCK) : nullptr;
    rc = dtype == PF_F16 ? pf_gated_forward_1(q, st) : pf_gated_forward_2(q, st);
    if (rc != PF_OK) return rc;
  }
  return PF_OK;
}

extern "C" int pf_gated_linear_split(const void* dy, int dtype, int64_t rows, int64_t ffn, int act, int keep, const void* kept, void* dgu, void* stream) {
  const char* who = "pf_gated_linear_split";
  const int rc = check(who, dtype, rows, 1, ffn, act, keep);
  if (rc != PF_OK) return rc;
  PF_REQUIRE(keep != PF_KEEP_NONE, "%s: nothing was kept", who);
  PF_REQUIRE(ffn % 8 == 0, "%s: a multiple of 8 columns", who);
  if (rows == 0) return PF_OK;
  PF_REQUIRE(dy && kept && dgu, "%s: null pointer", who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(dgu, 16), "%s: kept and dgu lie on boundaries of 16 bytes", who);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PF_F32) {
    const float* gu = (const float*)kept;
    float* d = (float*)dgu;
    return pf_glu_bwd(dy, ffn, gu, 2 * ffn, gu + ffn, 2 * ffn, d, 2 * ffn, d + ffn, 2 * ffn, PF_F32, act, rows, ffn, stream);
  }
  split_launch(dtype, keep, dy, kept, half_of(dtype, ffn, keep), rows, ffn, dgu, ffn, act, st);
  PF_CHECK_LAUNCH(who);
  return PF_OK;
}

extern "C" int pf_gated_linear_bwd(const void* x, int dtype, int64_t rows, int64_t D, const void* weight, int64_t ffn, int act, int keep, const void* kept,
                                   const void* dy, void* dx, void* dweight, void* workspace, void* stream) {
  const char* who = "pf_gated_linear_bwd";
  int rc = check(who, dtype, rows, D, ffn, act, keep);
  if (rc != PF_OK) return rc;
  PF_REQUIRE(keep != PF_KEEP_NONE, "%s: nothing was kept", who);
  Plan p;
  if (!plan_of(p, x, weight, dtype, rows, D, ffn, keep, true, (char*)workspace)) return too_large(who);
  hipStream_t st = (hipStream_t)stream;
  if (rows == 0) return dweight == nullptr ? PF_OK : pf_fill(dweight, dtype, 0.f, 2 * ffn * D, stream);
  PF_REQUIRE(x && weight && kept && dy && workspace, "%s: null pointer", who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(workspace, 16), "%s: kept and the workspace lie on boundaries of 16 and 256 bytes", who);
  PF_REQUIRE(dtype == PF_F32 || (pf_aligned(dx, 16) && pf_aligned(dweight, 16)), "%s: the gradients lie on boundaries of 16 bytes", who);
  const bool f32 = dtype == PF_F32;
  const int es = f32 ? 4 : 2;
  const int halves = p.wide == ffn ? 1 : 2;      // products over both halves of the weight at once, or one by one
  if (f32) {
    const float* gu = (const float*)kept;
    float* d = (float*)p.dgu;
    rc = pf_glu_bwd(dy, ffn, gu, 2 * p.wide, gu + p.wide, 2 * p.wide, d, 2 * p.wide, d + p.wide, 2 * p.wide, PF_F32, act, rows, ffn, stream);
    if (rc != PF_OK) return rc;
  } else {
    split_launch(dtype, keep, dy, kept, p.half, rows, ffn, p.dgu, p.wide, act, st);
  }
  auto join = [&] {
    const int64_t lanes = D % 8 == 0 ? 512 : 64, units = (rows * ((D + lanes - 1) / lanes) + 3) / 4;
    const dim3 grid((unsigned)(units < 16384 ? units : 16384));
    if (D % 8 == 0) hipLaunchKernelGGL(gated_join_kernel<8>, grid, dim3(256), 0, st, p.parts, p.depth, p.splits, rows, D, dx, dtype);
    else hipLaunchKernelGGL(gated_join_kernel<1>, grid, dim3(256), 0, st, p.parts, p.depth, p.splits, rows, D, dx, dtype);
  };
  const bool wide_x = p.x != nullptr && dweight != nullptr;
  if (wide_x) pf_rows_widen(x, rows, D, p.x, p.depth, es, st);
  PF_CHECK_LAUNCH(who);
  const char* xs = wide_x ? p.x : (const char*)x;
  const int64_t ldx = wide_x ? p.depth : D;
  if (dx && p.few_dx) {
    if (dtype == PF_F16) few_dx<PF_F16>(p.dgu, p.wide, weight, rows, ffn, D, p.parts, p.depth, p.splits, st);
    else few_dx<PF_BF16>(p.dgu, p.wide, weight, rows, ffn, D, p.parts, p.depth, p.splits, st);
    join();
  } else if (dx) {
    const bool parts = p.parts != nullptr;
    void* c = parts ? (void*)p.parts : dx;
    const int64_t ldc = parts ? p.depth : D, n = parts && !f32 ? round_up(D, 8) : D;
    const int c_dtype = parts ? PF_F32 : dtype;
    if (f32) {
      if (p.copy_w) pf_rows_widen(weight, 2 * ffn, D, p.w, p.depth, 4, st);
      const float* ws = p.copy_w ? (const float*)p.w : (const float*)weight;
      const float* d = (const float*)p.dgu;
      for (int h = 0; h < halves && rc == PF_OK; ++h)
        rc = product(dtype, c_dtype, 0, 1, rows, n, halves == 1 ? 2 * ffn : ffn, d + h * p.wide, 2 * p.wide, ws + h * ffn * p.depth, p.depth, c, ldc, h, st, p.splits);
    } else {
      // The reduction runs along the weight's rows, its transposed copy makes it contiguous: 13 us and a product of 242, where the product
      // of the weight as it lies takes 441 (8192 x 11264 x 2048, bf16).  (Columns past ffn, of zeros in dg and du, are zeros here too.)
      if (halves == 1) {
        rc = pf_transpose_cast(weight, dtype, D, p.wt, dtype, 2 * ffn, 2 * ffn, D, stream);
      } else {
        hipLaunchKernelGGL(gated_transpose_kernel, dim3((unsigned)((D + 63) / 64), (unsigned)((p.wide + 63) / 64), 2), dim3(256), 0, st, (const uint16_t*)weight, ffn, D,
                           (uint16_t*)p.wt, p.wide);
      }
      if (rc == PF_OK) rc = product(dtype, c_dtype, 0, 0, rows, n, 2 * p.wide, p.dgu, 2 * p.wide, p.wt, 2 * p.wide, c, ldc, 0, st, p.splits);
    }
    if (rc != PF_OK) return rc;
    if (parts) join();
  }
  if (dweight && p.few_dw) {
    if (dtype == PF_F16) few_dw<PF_F16>(p.dgu, p.wide, x, rows, ffn, D, dweight, st);
    else few_dw<PF_BF16>(p.dgu, p.wide, x, rows, ffn, D, dweight, st);
  } else if (dweight) {
    char* out = p.narrow ? p.dw : (char*)dweight;
    const int64_t ldc = p.narrow ? p.depth : D, n = p.narrow ? round_up(D, 8) : D;
    const int64_t m = halves == 1 ? 2 * ffn : ffn;
    if (f32) {
      for (int h = 0; h < halves && rc == PF_OK; ++h)
        rc = product(dtype, dtype, 1, 1, m, n, rows, p.dgu + h * p.wide * es, 2 * p.wide, xs, ldx, out + h * ffn * ldc * es, ldc, 0, st);
    } else if (dtype == PF_F16) {
      rc = pf_gated_weight_1(m, n, rows, p.dgu, 2 * p.wide, xs, ldx, out, ldc, halves, p.wide, st);
    } else {
      rc = pf_gated_weight_2(m, n, rows, p.dgu, 2 * p.wide, xs, ldx, out, ldc, halves, p.wide, st);
    }
    if (rc != PF_OK) return rc;
    if (p.narrow) pf_rows_narrow(p.dw, p.depth, dweight, 2 * ffn, D, st);
  }
  PF_CHECK_LAUNCH(who);
  return PF_OK;
}
