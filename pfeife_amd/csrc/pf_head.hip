// Softmax cross entropy of a large vocabulary from the last hidden state: loss and gradients without the logits in memory.
//
//   z = h W^T (fp32, never rounded);  lse = ln sum exp z;  loss = lse - z[label] + z_loss lse^2
//   dz = c (p (1 + 2 z_loss lse) - onehot);  dh = dz W;  dW = dz^T h
//
// Forward: one product whose epilogue keeps, of every block of vocabulary rows, each token's maximum and sum (pf_head_x.hip), and
// a merge of those.  Backward: piece by piece of the vocabulary the same product again, now with dz in its epilogue, and the two
// products that read it.  A piece's dz is all that is ever in memory.  Of the three products that any backward pass
// needs one is thus done twice: the price of 2 N V bytes that are not kept, a quarter of the arithmetic.
//
// Tokens whose label is ignored take no part in any of this: the others are gathered to the front first, and how many they are is
// read by the kernels.  (The gathered copy is also where strides, odd widths and the gap of a shifted label end.)
// dz is rounded to the operands' type before the products, as the logits' gradient of any step in 16 bits is.  It is rounded as a
// multiple of the largest factor c, which the products multiply by in fp32: the label's entry, 1 - p of it, is what weighs most in
// both gradients, and is the more exact the less sure the model is (c (1 - p) would take over c's own rounding for all tokens
// alike: 131072 classes, bf16, relative error of the gradients 2.8e-3 so, 1.9e-3 as it is, 1.7e-3 being the results' own rounding).  Where the
// tokens' factors differ (a gradient for every token) the rounding of c is there.  fp16: 2^13 times that, which keeps probabilities down
// to 2^-38.
// fp32: the same through the fp32 products, with a piece's logits in memory.
#include "pf_gemm_common.h"
#include "pf_head.h"
#include "pf_rows.h"

#include <math.h>

#define PF_HEAD_DECL(DT)                                                   \
  int pf_head_stats_##DT(const PfHeadProduct&, hipStream_t);               \
  int pf_head_dz_##DT(const PfHeadProduct&, hipStream_t);                  \
  int pf_head_dh_##DT(const PfHeadProduct&, hipStream_t);                  \
  int pf_head_dw_##DT(const PfHeadProduct&, hipStream_t);
PF_HEAD_DECL(1)
PF_HEAD_DECL(2)
#undef PF_HEAD_DECL
static_assert(PF_F16 == 1 && PF_BF16 == 2, "the names above are written out for these ids");

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.69314718055994530942;
constexpr float LOWEST = -3.0e38f;

// What the forward pass leaves for the backward pass; n_max entries each
struct Kept {
  int* count;      // tokens that take part
  int* rows;       // their places among B * T, in order
  int* lab;        // their labels (-2: outside the vocabulary; -1 behind the last of them)
  int* inv;        // [B * T] a place's number among them, -1: none
  float* top;      // a logit near the largest
  float* bias;     // -log2 of the sum of exponentials beside it
};
inline int64_t round_up(int64_t n, int64_t k) { return (n + k - 1) / k * k; }
inline int64_t kept_bytes(int64_t n_max) { return 64 + 20 * n_max; }
inline Kept kept_of(void* p, int64_t n_max) {
  int* q = (int*)p;
  return {q, q + 16, q + 16 + n_max, q + 16 + 2 * n_max, (float*)(q + 16 + 3 * n_max), (float*)(q + 16 + 4 * n_max)};
}

struct Sizes {
  int64_t n, n_max, depth, piece, dim8;
  PfHeadShares shares;
  bool copy_w, narrow;
};

struct Labels {
  const int64_t* labels;
  int64_t n, T, V, ignore, n_max;
  int shift;
  __device__ __forceinline__ int64_t at(int64_t r) const { return r >= n || (shift && r % T == T - 1) ? ignore : labels[r + shift]; }
  __device__ __forceinline__ int64_t out(int64_t r) const { return r / T * (T - shift) + r % T; }
  __device__ __forceinline__ bool scored(int64_t r) const { return r < n && !(shift && r % T == T - 1); }
  __device__ __forceinline__ int label(int64_t l) const { return l >= 0 && l < V ? (int)l : -2; }
};

// Which tokens take part: groups of 1024, each of which counts for itself what lies before it: one launch, no order of arrival in the
// result
__global__ __launch_bounds__(1024) void head_index_kernel(const Labels y, Kept k, float* out) {
  __shared__ float sm[16];
  __shared__ int before[17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int ahead = 0;
#pragma unroll 4
  for (int64_t r = tid; r < (int64_t)blockIdx.x * 1024; r += 1024) ahead += y.at(r) != y.ignore;
  // (at most 2^24 tokens: exact in fp32)
  const int base = (int)pf_block_sum<16>((float)ahead, sm);
  const int64_t r = (int64_t)blockIdx.x * 1024 + tid;
  const int64_t l = y.at(r);
  const bool in = l != y.ignore;
  const unsigned long long mask = __ballot(in);
  if (lane == 0) before[wave + 1] = __popcll(mask);
  __syncthreads();
  if (tid == 0) {
    before[0] = base;
    for (int w = 1; w <= 16; ++w) before[w] += before[w - 1];
  }
  __syncthreads();
  const int c = before[wave] + __popcll(mask & ((1ull << lane) - 1));
  if (r < y.n) k.inv[r] = in ? c : -1;
  if (in) {
    k.rows[c] = (int)r;
    k.lab[c] = y.label(l);
  } else if (out != nullptr && y.scored(r)) {
    out[y.out(r)] = 0.f;
  }
  if (blockIdx.x == gridDim.x - 1) {
    const int total = before[16];
    if (tid == 0) *k.count = total;
    for (int64_t i = total + tid; i < y.n_max; i += 1024) k.lab[i] = -1;
  }
}

__device__ __forceinline__ int64_t rows_needed(int n) { return n > 64 ? (n + 63) / 64 * 64 : 64; }

struct Hidden {
  const char* h;
  int64_t T, sb, st, D, depth;
  char* hc;
};
// One token's row by one wavefront, or zeros; U: an element, as bits
template <typename U>
__device__ __forceinline__ void gather_row(const Hidden& x, int64_t c, int64_t r) {
  constexpr int N = 16 / sizeof(U);
  uint4* dst = (uint4*)((U*)x.hc + c * x.depth);
  const U* src = (const U*)x.h + (r / x.T) * x.sb + (r % x.T) * x.st;
  const int64_t width = r >= 0 ? x.D : 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x & 63; i < x.depth / N; i += 64) dst[i] = i * N < width ? pf_load_loose(src + i * N, width - i * N) : make_uint4(0, 0, 0, 0);
}

// The tokens that take part, one behind the other, zeros behind them and in columns D .. depth - 1
template <typename U>
__global__ __launch_bounds__(256) void head_gather_kernel(const Hidden x, const Kept k) {
  const int n = *k.count;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c < rows_needed(n)) gather_row<U>(x, c, c < n ? k.rows[c] : -1);
}

// Both in one launch for up to 4096 tokens, where every workgroup can count all of them: four tokens to a workgroup, and the rows of
// zeros behind the last one dealt out too.  (us of a forward pass with 512 classes of 512 columns, one launch and two: 1024 tokens 38 and 40, 4096 42.4 and 43.1, 8192
// 55 and 47)
template <typename U>
__global__ __launch_bounds__(256) void head_index_gather_kernel(const Labels y, const Hidden x, Kept k, float* out) {
  __shared__ int sm[4], sa[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * 4;
  int ahead = 0, total = 0;
#pragma unroll 4
  for (int64_t r = tid; r < y.n; r += 256) {
    const int in = y.at(r) != y.ignore;
    total += in;
    ahead += r < r0 ? in : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    ahead += __shfl_xor(ahead, o, 64);
    total += __shfl_xor(total, o, 64);
  }
  if (lane == 0) { sm[wave] = total; sa[wave] = ahead; }
  __syncthreads();
  total = sm[0] + sm[1] + sm[2] + sm[3];
  int c = sa[0] + sa[1] + sa[2] + sa[3];
  const int64_t r = r0 + wave;
  for (int64_t q = r0; q < r; ++q) c += y.at(q) != y.ignore;
  const int64_t l = y.at(r);
  const bool in = l != y.ignore;
  if (in) gather_row<U>(x, c, r);
  if (lane == 0 && r < y.n) {
    k.inv[r] = in ? c : -1;
    if (in) {
      k.rows[c] = (int)r;
      k.lab[c] = y.label(l);
    } else if (out != nullptr && y.scored(r)) {
      out[y.out(r)] = 0.f;
    }
  }
  const int64_t zeros = rows_needed(total);
  for (int64_t z = total + (int64_t)blockIdx.x * 4 + wave; z < zeros; z += (int64_t)gridDim.x * 4) gather_row<U>(x, z, -1);
  if (blockIdx.x == 0) {
    if (tid == 0) *k.count = total;
    for (int64_t i = total + tid; i < y.n_max; i += 256) k.lab[i] = -1;
  }
}

// Every token's statistics of all blocks merged, its loss; TOKENS to a workgroup, 1024 / TOKENS threads to a token.  The sum in 64 bits: a
// loss near zero is the logarithm of a sum near one.  A chain of latencies; us with 8 and 32 tokens to a workgroup: 16 of them with 1000 blocks each 4.4 / 7.5, 2048 with
// 1024 9.8 / 10.7, 4662 with 391 7.6 / 6.6, 8192 with 250 11.8 / 7.0.
template <int TOKENS>
__global__ __launch_bounds__(1024) void head_merge_kernel(const PfHeadPart* part, int64_t blocks, int64_t n_max, const float* zl, Kept k, double z_loss,
                                                          int64_t T, int shift, double* terms, float* out) {
  constexpr int SLICES = 1024 / TOKENS;
  __shared__ float tops[16][TOKENS];
  __shared__ double sums[16][TOKENS];
  const int t = threadIdx.x % TOKENS, slice = threadIdx.x / TOKENS;
  const int n = *k.count;
  const int64_t c = (int64_t)blockIdx.x * TOKENS + t;
  float m = LOWEST;
  double s = 0;
  if (c < n) {
    for (int64_t i0 = slice; i0 < blocks; i0 += SLICES * 8) {      // (eight loads on their way at once)
      PfHeadPart p[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) p[q] = i0 + SLICES * q < blocks ? part[(i0 + SLICES * q) * n_max + c] : PfHeadPart{LOWEST, 0.f};
      float x = m;
#pragma unroll
      for (int q = 0; q < 8; ++q) x = fmaxf(x, p[q].top);
      s *= (double)__builtin_amdgcn_exp2f((m - x) * LOG2E);
#pragma unroll
      for (int q = 0; q < 8; ++q) s += (double)(p[q].sum * __builtin_amdgcn_exp2f((p[q].top - x) * LOG2E));
      m = x;
    }
  }
#pragma unroll
  for (int o = TOKENS; o < 64; o <<= 1) {
    const float om = __shfl_xor(m, o, 64);
    const double os = __shfl_xor(s, o, 64);
    const float x = fmaxf(m, om);
    s = s * (double)__builtin_amdgcn_exp2f((m - x) * LOG2E) + os * (double)__builtin_amdgcn_exp2f((om - x) * LOG2E);
    m = x;
  }
  if ((int)(threadIdx.x & 63) < TOKENS) {
    tops[threadIdx.x >> 6][t] = m;
    sums[threadIdx.x >> 6][t] = s;
  }
  __syncthreads();
  if (threadIdx.x >= TOKENS) return;
  double term = 0;
  if (c < n) {
    float top = LOWEST;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, tops[i][t]);
    double total = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += sums[i][t] * (double)__builtin_amdgcn_exp2f((tops[i][t] - top) * LOG2E);
    const double ls = log(total), lse = (double)top + ls;
    const int l = k.lab[c];
    term = l < 0 ? (double)NAN : ((double)top - (double)zl[c]) + ls + z_loss * lse * lse;
    k.top[c] = top;
    k.bias[c] = (float)(-ls / LN2);
    if (out != nullptr) {
      const int64_t r = k.rows[c];
      out[r / T * (T - shift) + r % T] = (float)term;
    }
  }
  if (terms != nullptr && c < n_max) terms[c] = term;
}

__global__ __launch_bounds__(1024) void head_reduce_kernel(const double* terms, const int* count, int mean, float* loss) {
  __shared__ double sm[1024];
  const int n = *count;
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += terms[i];
  sm[threadIdx.x] = s;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) sm[threadIdx.x] += sm[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = (float)(mean && n > 0 ? sm[0] / n : sm[0]);
}

// What every token's gradient is multiplied by: the factor of its probabilities and that of its label
struct Upstream {
  const float* grad;       // of the loss, or of every token's
  int64_t g_sb, g_st;      // 0, 0: one number
  int64_t T;
  int mean;
  double z_loss;
  Kept k;
};
__device__ __forceinline__ void factors(const Upstream& u, int n, int64_t c, float& f, float& g) {
  const int64_t r = u.k.rows[c];
  const double up = (double)u.grad[(r / u.T) * u.g_sb + (r % u.T) * u.g_st] / (u.mean ? (double)n : 1.0);
  const double lse = (double)u.k.top[c] - (double)u.k.bias[c] * LN2;
  g = u.k.lab[c] < 0 ? NAN : (float)up;
  f = u.k.lab[c] < 0 ? NAN : (float)(up * (1.0 + 2.0 * u.z_loss * lse));
}
// The number that brings the largest factor to `most`; nothing to scale by where all factors are zero, one is infinite, or the
// quotient would be
__device__ __forceinline__ float scale_of(float top, float most) { return top > 1e-30f && top < INFINITY ? most / top : 1.f; }
__device__ __forceinline__ float largest_factor(const Upstream& u, int n, int first, int step) {
  float top = 0.f;
  for (int c = first; c < n; c += step) {
    float f, g;
    factors(u, n, c, f, g);
    top = fmaxf(top, fmaxf(fabsf(f), fabsf(g)));
  }
  return top;
}
__global__ __launch_bounds__(1024) void head_scale_kernel(const Upstream u, float most, float* scale) {
  __shared__ float sm[16];
  const float top = pf_block_max<16>(largest_factor(u, *u.k.count, threadIdx.x, 1024), sm);
  if (threadIdx.x == 0) *scale = scale_of(top, most);
}

// What the backward pass's products read, in one launch: each token's factors (the first `factor` workgroups), the gathered rows (the
// next `rows`) and their transpose (the others, 64 x 64 elements each).  Bound by memory: 8192 x 2048, bf16: 26 us, 134 MB (52 with
// the transpose by two bytes to a lane).
struct Ready {
  Upstream u;
  Hidden x;
  PfHeadColumn* col;
  float* scale;            // null: none
  float most;
  int known;               // 0: to be found; 1: there already; 2: all tokens' factors are alike
  int factor, rows, tiles_n;
  int64_t n_max, dim8;
  uint16_t* ht;
};
template <typename U>
__global__ __launch_bounds__(256) void head_ready_kernel(const Ready q) {
  __shared__ __align__(16) uint16_t tile[64][66];      // (rows of 33 words: neither way do lanes meet in a bank)
  __shared__ float sm[4];
  const Kept& k = q.u.k;
  const int n = *k.count, t = threadIdx.x;
  if ((int)blockIdx.x < q.factor) {
    float s = 1.f;
    if (q.scale != nullptr) {
      if (q.known == 1) s = *q.scale;
      else if (q.known == 2) s = scale_of((float)(fabs((double)*q.u.grad) / (q.u.mean && n > 0 ? (double)n : 1.0)), q.most);
      else s = scale_of(pf_block_max<4>(largest_factor(q.u, n, t, 256), sm), q.most);
      if (q.known != 1 && blockIdx.x == 0 && t == 0) *q.scale = s;
    }
    const int64_t c = (int64_t)blockIdx.x * 256 + t;
    if (c >= q.n_max) return;
    PfHeadColumn o = {0.f, 0.f, 0.f, 0.f};     // (behind the last token: zeros times exp(0))
    if (c < n) {
      o.top = k.top[c];
      o.bias = k.bias[c];
      factors(q.u, n, c, o.f, o.g);
      o.f *= s;
      o.g *= s;
    }
    q.col[c] = o;
    return;
  }
  const int64_t padded = rows_needed(n);
  const int block = (int)blockIdx.x - q.factor;
  if (block < q.rows) {
    const int64_t c = (int64_t)block * 4 + (t >> 6);
    if (c < padded) gather_row<U>(q.x, c, c < n ? k.rows[c] : -1);
    return;
  }
  const int64_t c0 = (int64_t)((block - q.rows) / q.tiles_n) * 64, d0 = (int64_t)((block - q.rows) % q.tiles_n) * 64;
  if (c0 >= padded) return;
#pragma unroll
  for (int i = t >> 3; i < 64; i += 32) {      // eight elements of a row to a thread, either way
    const int64_t c = c0 + i, d = d0 + (t & 7) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < n && d < q.x.D) {
      const int64_t r = k.rows[c];
      v = pf_load_loose((const uint16_t*)q.x.h + (r / q.x.T) * q.x.sb + (r % q.x.T) * q.x.st + d, q.x.D - d);
    }
    uint32_t* to = (uint32_t*)&tile[i][(t & 7) * 8];
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  }
  __syncthreads();
#pragma unroll
  for (int i = t >> 3; i < 64; i += 32) {
    const int64_t d = d0 + i;
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (uint32_t)tile[(t & 7) * 8 + 2 * j][i] | (uint32_t)tile[(t & 7) * 8 + 2 * j + 1][i] << 16;
    if (d < q.dim8) *(uint4*)(q.ht + d * q.n_max + c0 + (t & 7) * 8) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The gradient of every row of the hidden state: a token's sum rounded once (times a loss scale first), zeros where it took no part
template <int W>
__global__ __launch_bounds__(256) void head_spread_kernel(const float* acc, int64_t ld, const PfHeadShares shares, int64_t n_max, const int* count, const int* inv, int64_t n,
                                                          int64_t D, const float* times, void* dh, int dt) {
  const float by = times != nullptr ? *times : 1.f;
  const int splits = shares.of(*count, ld);
  const int64_t step = shares.by_count ? *count : n_max;
  const int64_t per = (D + 64 * W - 1) / (64 * W), total = n * per;      // (a wavefront to 64 W columns of a row)
  for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < total; q += (int64_t)gridDim.x * 4) {
    const int64_t r = q / per, i = q % per * 64 * W + (threadIdx.x & 63) * W;
    if (i >= D) continue;
    const int c = inv[r];
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = 0.f;
    if (c >= 0) {
#pragma unroll 4
      for (int p = 0; p < splits; ++p) {
        float w[W];
        ld_vec<W>(acc, (p * step + c) * ld + i, PF_F32, w);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] += w[k];
      }
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] *= by;
    }
    st_vec<W>(dh, r * D + i, dt, v);
  }
}

// fp32: statistics of ROWS32 vocabulary rows of a piece in memory, z[row][token]
constexpr int ROWS32 = 32;
__global__ __launch_bounds__(256) void head_stats32_kernel(const float* z, int64_t rows, int64_t n_max, int64_t v0, const int* lab, const int* count, PfHeadPart* part,
                                                           float* zl) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, r0 = (int64_t)blockIdx.y * ROWS32;
  if (c >= *count) return;
  const int64_t r1 = r0 + ROWS32 < rows ? r0 + ROWS32 : rows;
  const int64_t at = (int64_t)lab[c] - v0;
  float m = LOWEST, s = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float x = z[r * n_max + c];
    if (r == at) zl[c] = x;
    const float t = fmaxf(m, x);
    s = s * __builtin_amdgcn_exp2f((m - t) * LOG2E) + __builtin_amdgcn_exp2f((x - t) * LOG2E);
    m = t;
  }
  part[(int64_t)blockIdx.y * n_max + c] = {m, s};
}
__global__ __launch_bounds__(256) void head_dz32_kernel(float* z, int64_t rows, int64_t n_max, int64_t v0, const int* lab, const int* count, const PfHeadColumn* col) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, r0 = (int64_t)blockIdx.y * ROWS32;
  if (c >= *count) return;
  const int64_t r1 = r0 + ROWS32 < rows ? r0 + ROWS32 : rows;
  const int64_t at = lab[c] >= 0 ? (int64_t)lab[c] - v0 : -1;
  const PfHeadColumn k = col[c];
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float v = k.f * __builtin_amdgcn_exp2f(fmaf(z[r * n_max + c] - k.top, LOG2E, k.bias));
    z[r * n_max + c] = r == at ? v - k.g : v;
  }
}

// fp32, few tokens: the weight's gradient as the outer products that it is, 16 rows of it to a wavefront, 4 columns to a lane.  Bound by its way to
// memory, where a matrix tile mostly waits for its one stage of operands: 2 tokens, 4080 columns, 26156 classes 103 us, 427 MB, against 246.  us of a step of the
// weight alone, 2048 columns, 32000 classes, so and by matrix tiles: 8 tokens 245 and 316, 32 277 and 312, 64 350 and 336.
constexpr int FEW_ROWS32 = 16, FEW_TOKENS32 = 48;
__global__ __launch_bounds__(256) void head_weight_grad32_kernel(const float* dz, int64_t n_max, const int* count, const float* hc, int64_t ld, float* dw, int64_t rows,
                                                                 int64_t D) {
  const int n = *count, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r0 = ((int64_t)blockIdx.x * 4 + wave) * FEW_ROWS32, c = ((int64_t)blockIdx.y * 64 + (threadIdx.x & 63)) * 4;
  if (r0 >= rows || c >= D) return;
  float acc[FEW_ROWS32][4];
#pragma unroll
  for (int r = 0; r < FEW_ROWS32; ++r)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[r][k] = 0.f;
#pragma unroll 4
  for (int t = 0; t < n; ++t) {
    const float4 h = *(const float4*)(hc + t * ld + c);
#pragma unroll
    for (int r = 0; r < FEW_ROWS32; ++r) {
      const float x = dz[(r0 + r < rows ? r0 + r : rows - 1) * n_max + t];
      acc[r][0] = fmaf(x, h.x, acc[r][0]);
      acc[r][1] = fmaf(x, h.y, acc[r][1]);
      acc[r][2] = fmaf(x, h.z, acc[r][2]);
      acc[r][3] = fmaf(x, h.w, acc[r][3]);
    }
  }
#pragma unroll
  for (int r = 0; r < FEW_ROWS32; ++r)
    if (r0 + r < rows)
      pf_store_loose((uint32_t*)dw + (r0 + r) * D + c, D - c,
                     make_uint4(__float_as_uint(acc[r][0]), __float_as_uint(acc[r][1]), __float_as_uint(acc[r][2]), __float_as_uint(acc[r][3])));
}

int bad(const char* who, const char* what) {
  pf_set_error("%s: %s", who, what);
  return PF_ERR_INVALID;
}

// Vocabulary rows of a piece: its dz (fp32: its logits) in 256 MB, in whole tiles.  (16384 tokens, 2048 columns, 32000 classes, bf16: 6.62 ms; with 512 MB 6.60, with
// 128 7.35)
int64_t piece_rows(int64_t n_max, int64_t V, int64_t size) {
  int64_t rows = (256ll << 20) / (n_max * size) / 256 * 256;
  if (rows < 256) rows = 256;
  return rows < V ? rows : V;
}
// Rows that a buffer's 32-bit offsets reach
int64_t reach_rows(int64_t ldw) { return ((1ll << 31) / (ldw * 2) - 512) / 256 * 256; }

struct Call {
  const char* who;
  const void* h;
  int dtype;
  int64_t B, T, D, sb, st;
  const void* w;
  int64_t V;
};

bool sizes_of(const Call& c, Sizes& s, bool back) {
  const int64_t es = c.dtype == PF_F32 ? 4 : 2;
  s.n = c.B * c.T;
  s.n_max = round_up(s.n > 0 ? s.n : 1, 64);
  s.depth = c.dtype == PF_F32 ? round_up(c.D, 4) : (c.D < 64 ? 64 : round_up(c.D, 8));
  s.copy_w = s.depth != c.D || !pf_aligned(c.w, 16);
  // Whole stages of the fastest tile: where the weight is copied anyway, and where many tokens pay for a copy.  us of a step, 1000 columns, 50000 classes, bf16,
  // on the tile for any multiple of 8 and on the other behind copies: 1024 tokens 567 and 589, 2048 937 and 875, 4096 1780 and 1546.
  if (es == 2 && s.n_max > 256 && (s.copy_w || s.n_max >= 2048)) {
    s.depth = round_up(s.depth, 64);
    s.copy_w = s.copy_w || s.depth != c.D;
  }
  s.dim8 = round_up(c.D, 8);
  s.narrow = es == 2 && s.dim8 != c.D;
  s.piece = piece_rows(s.n_max, c.V, es);
  if (es == 2 && s.piece > reach_rows(s.depth)) s.piece = reach_rows(s.depth);
  if (back) s.shares = pf_head_shares(c.dtype, es == 4 && s.n > 0 ? s.n : s.n_max, s.depth, s.piece);
  if (s.n >= (1ll << 24) || c.V >= (1ll << 31) || s.depth >= (1ll << 19)) return false;
  // what is addressed by 32-bit offsets: forward the gathered rows (fp32: and a piece's logits), backward the fp32 sums of their gradient and a piece's dz
  if (es == 2 && !back) return s.n_max <= reach_rows(s.depth);
  return s.n_max * s.depth * 4 < (1ll << 31) - 64 && s.piece * s.n_max * es < (1ll << 31) - 64;
}

// A block of device memory handed out front to back, each part on a boundary of 256 bytes
struct Carve {
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base == nullptr ? nullptr : base + used;
    used += round_up(bytes, 256);
    return p;
  }
};
struct Work {
  char* hc; char* wide; PfHeadPart* part; float* zl; double* terms;             // forward (hc and wide: backward too)
  char* dz; char* ht; char* dw; float* acc; PfHeadColumn* col; float* scale;     // backward (dz: fp32's logits in both)
};
Work carve(Carve& a, const Call& c, const Sizes& s, bool back) {
  const int64_t es = c.dtype == PF_F32 ? 4 : 2;
  Work w = {};
  w.hc = (char*)a.take(s.n_max * s.depth * es);
  if (s.copy_w) w.wide = (char*)a.take(c.V * s.depth * es);
  if (back || es == 4) w.dz = (char*)a.take(s.piece * s.n_max * es);
  if (!back) {
    w.part = (PfHeadPart*)a.take((es == 4 ? (c.V + ROWS32 - 1) / ROWS32 : pf_head_blocks(c.V, s.n_max, s.depth)) * s.n_max * 8);
    w.zl = (float*)a.take(s.n_max * 4);
    w.terms = (double*)a.take(s.n_max * 8);
  } else {
    if (es == 2) w.ht = (char*)a.take(s.dim8 * s.n_max * 2);
    if (s.narrow) w.dw = (char*)a.take(s.piece * s.depth * 2);
    w.col = (PfHeadColumn*)a.take(s.n_max * 16);
    w.scale = (float*)a.take(4);
    w.acc = (float*)a.take(s.shares.bytes(s.n_max, s.depth));
  }
  return w;
}

int check_call(const Call& c, const Sizes& s, bool back, bool ok) {
  if (c.dtype != PF_F32 && c.dtype != PF_F16 && c.dtype != PF_BF16) return bad(c.who, "bad dtype");
  if (c.B < 0 || c.T < 0 || c.D <= 0 || c.V <= 0) return bad(c.who, "bad sizes");
  if (!ok) {
    pf_set_error("%s: %lld tokens of width %lld and %lld classes: too many for one call (the tokens%s to stay below 2 GiB)", c.who, (long long)s.n, (long long)c.D,
                 (long long)c.V, back ? "' fp32 gradient has" : " have");
    return PF_ERR_INVALID;
  }
  return PF_OK;
}

Hidden hidden_of(const Call& c, const Sizes& s, const Work& w) {
  return {(const char*)c.h, c.T > 0 ? c.T : 1, c.sb, c.st, c.D, s.depth, w.hc};
}
#define PF_BY_SIZE(KERNEL, ...)                                                          \
  do {                                                                                   \
    if (c.dtype == PF_F32) hipLaunchKernelGGL(KERNEL<uint32_t>, __VA_ARGS__);            \
    else hipLaunchKernelGGL(KERNEL<uint16_t>, __VA_ARGS__);                              \
  } while (0)

void widen(const Call& c, const Sizes& s, const Work& w, hipStream_t st) {
  if (s.copy_w) pf_rows_widen(c.w, c.V, c.D, w.wide, s.depth, c.dtype == PF_F32 ? 4 : 2, st);
}

// A product over fp32 operands of the tokens that take part, all of them at most (N, M or K of it, see pf_gemm_f32_counted); splits: shares of the
// depth, with results of their own
int product32(int a_trans, int b_trans, int64_t M, int64_t N, int64_t K, const float* A, int64_t lda, const float* B, int64_t ldb, float* C, int64_t ldc, int beta,
              const int* count, hipStream_t st, int splits = 1, int64_t c_stride = 0) {
  pf_gemm_desc d = {};
  d.in_dtype = d.c_dtype = PF_F32;
  d.a_trans = a_trans; d.b_trans = b_trans;
  d.M = M; d.N = N; d.K = pf_head_share(K, splits);
  d.A = A; d.lda = lda; d.B = B; d.ldb = ldb; d.C = C; d.ldc = ldc;
  d.batch1 = 1; d.batch2 = (K + d.K - 1) / d.K;
  d.a_stride2 = d.K * lda;
  d.b_stride2 = d.K * ldb;
  d.c_stride2 = c_stride;
  d.alpha = 1.f;
  d.beta = beta;
  return pf_gemm_f32_counted(d, count, K, st);
}

}  // namespace

int pf_head_stats(int dtype, const PfHeadProduct& p, hipStream_t st) { return dtype == PF_F16 ? pf_head_stats_1(p, st) : pf_head_stats_2(p, st); }
int pf_head_dz(int dtype, const PfHeadProduct& p, hipStream_t st) { return dtype == PF_F16 ? pf_head_dz_1(p, st) : pf_head_dz_2(p, st); }
int pf_head_dh(int dtype, const PfHeadProduct& p, hipStream_t st) { return dtype == PF_F16 ? pf_head_dh_1(p, st) : pf_head_dh_2(p, st); }
int pf_head_dw(int dtype, const PfHeadProduct& p, hipStream_t st) { return dtype == PF_F16 ? pf_head_dw_1(p, st) : pf_head_dw_2(p, st); }

extern "C" int64_t pf_linear_ce_kept(int64_t tokens) { return kept_bytes(round_up(tokens > 0 ? tokens : 1, 64)); }

extern "C" int64_t pf_linear_ce_workspace(const void* weight, int dtype, int64_t tokens, int64_t D, int64_t V, int backward) {
  const Call c = {"pf_linear_ce_workspace", nullptr, dtype, 1, tokens, D, 0, D, weight, V};
  Sizes s = {};
  const int rc = check_call(c, s, backward != 0, tokens < 0 || D <= 0 || V <= 0 || sizes_of(c, s, backward != 0));
  if (rc != PF_OK) return rc;
  Carve a = {nullptr};
  carve(a, c, s, backward != 0);
  return a.used;
}

extern "C" int pf_linear_ce_fwd(const void* hidden, int dtype, int64_t B, int64_t T, int64_t D, int64_t sb, int64_t st_, const void* weight, int64_t V,
                                const int64_t* labels, int shift, int64_t ignore_index, double z_loss, int reduction, float* loss, void* kept,
                                void* workspace, void* stream) {
  const Call c = {"pf_linear_ce_fwd", hidden, dtype, B, T, D, sb, st_, weight, V};
  Sizes s = {};
  int rc = check_call(c, s, false, B < 0 || T < 0 || D <= 0 || V <= 0 || sizes_of(c, s, false));
  if (rc != PF_OK) return rc;
  PF_REQUIRE((shift == 0 || shift == 1) && reduction >= 0 && reduction <= 2, "%s: shift is 0 or 1, reduction 0, 1 or 2", c.who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(workspace, 16), "%s: kept and the workspace lie on boundaries of 256 bytes", c.who);
  PF_REQUIRE((loss || (reduction == 0 && B * (T - shift) <= 0)) && kept && workspace && weight && (s.n == 0 || (hidden && labels)), "%s: null pointer", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of(kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, false);
  float* out = reduction == 0 ? loss : nullptr;
  const Labels y = {labels, s.n, T > 0 ? T : 1, V, ignore_index, s.n_max, shift};
  const Hidden x = hidden_of(c, s, w);
  if (s.n <= 4096) {
    PF_BY_SIZE(head_index_gather_kernel, dim3((unsigned)(s.n_max / 4)), dim3(256), 0, st, y, x, k, out);
  } else {
    hipLaunchKernelGGL(head_index_kernel, dim3((unsigned)((s.n + 1023) / 1024)), dim3(1024), 0, st, y, k, out);
    PF_BY_SIZE(head_gather_kernel, dim3((unsigned)(s.n_max / 4)), dim3(256), 0, st, x, k);
  }
  widen(c, s, w, st);
  PF_CHECK_LAUNCH(c.who);
  const char* wide = s.copy_w ? w.wide : (const char*)weight;
  int64_t blocks = 0;
  if (dtype == PF_F32) {
    const int64_t n = s.n > 0 ? s.n : 1;
    for (int64_t v0 = 0; v0 < V; v0 += s.piece) {
      const int64_t rows = V - v0 < s.piece ? V - v0 : s.piece;
      rc = product32(0, 0, rows, n, D, (const float*)wide + v0 * s.depth, s.depth, (const float*)w.hc, s.depth, (float*)w.dz, s.n_max, 0, k.count, st);
      if (rc != PF_OK) return rc;
      hipLaunchKernelGGL(head_stats32_kernel, dim3((unsigned)((s.n_max + 255) / 256), (unsigned)((rows + ROWS32 - 1) / ROWS32)), dim3(256), 0, st, (const float*)w.dz, rows,
                         s.n_max, v0, k.lab, k.count, w.part + blocks * s.n_max, w.zl);
      blocks += (rows + ROWS32 - 1) / ROWS32;
    }
  } else {
    PfHeadProduct p = {};
    p.ldw = s.depth; p.depth = s.depth;
    p.hc = w.hc; p.ldh = s.depth; p.n_max = s.n_max;
    p.count = k.count; p.lab = k.lab; p.zl = w.zl;
    // (at most 2^23 workgroups of 512 threads to a launch)
    const int64_t most = (1ll << 23) / ((s.n_max + 127) / 128) * 256, reach = reach_rows(s.depth) < most ? reach_rows(s.depth) : most;
    for (int64_t v0 = 0; v0 < V; v0 += reach) {
      p.v0 = v0;
      p.rows = V - v0 < reach ? V - v0 : reach;
      p.w = wide + v0 * s.depth * 2;
      p.part = w.part + blocks * s.n_max;
      rc = pf_head_stats(dtype, p, st);
      if (rc != PF_OK) return rc;
      blocks += pf_head_blocks(p.rows, s.n_max, s.depth);
    }
  }
#define PF_HM(TOKENS) \
  hipLaunchKernelGGL(head_merge_kernel<TOKENS>, dim3((unsigned)(s.n_max / TOKENS)), dim3(1024), 0, st, w.part, blocks, s.n_max, w.zl, k, z_loss, T > 0 ? T : 1, shift, \
                     reduction == 0 ? nullptr : w.terms, out)
  if (s.n_max <= 2048) PF_HM(8);
  else PF_HM(32);
#undef PF_HM
  if (reduction != 0) hipLaunchKernelGGL(head_reduce_kernel, dim3(1), dim3(1024), 0, st, w.terms, k.count, reduction == 1, loss);
  PF_CHECK_LAUNCH(c.who);
  return PF_OK;
}

extern "C" int pf_linear_ce_bwd(const void* hidden, int dtype, int64_t B, int64_t T, int64_t D, int64_t sb, int64_t st_, const void* weight, int64_t V,
                                double z_loss, int mean, const void* kept, const float* grad, int64_t g_sb, int64_t g_st, void* dhidden, void* dweight,
                                void* workspace, void* stream) {
  const Call c = {"pf_linear_ce_bwd", hidden, dtype, B, T, D, sb, st_, weight, V};
  Sizes s = {};
  int rc = check_call(c, s, true, B < 0 || T < 0 || D <= 0 || V <= 0 || sizes_of(c, s, true));
  if (rc != PF_OK) return rc;
  PF_REQUIRE(kept && workspace && weight && grad && (s.n == 0 || hidden), "%s: null pointer", c.who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(workspace, 16), "%s: kept and the workspace lie on boundaries of 256 bytes", c.who);
  PF_REQUIRE(dtype == PF_F32 || pf_aligned(dweight, 16), "%s: dweight lies on a boundary of 16 bytes", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of((void*)kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, true);
  const Upstream u = {grad, g_sb, g_st, T > 0 ? T : 1, mean, z_loss, k};
  const bool half = dtype != PF_F32;
  Ready q = {};
  q.u = u;
  q.x = hidden_of(c, s, w);
  q.col = w.col;
  q.scale = half ? w.scale : nullptr;
  q.most = dtype == PF_F16 ? 8192.f : 1.f;
  if (g_sb == 0 && g_st == 0 && z_loss == 0) {
    q.known = 2;
  } else if (half && s.n > 1024) {      // (fewer: every workgroup finds the largest factor for itself; at 1024 the same, at 8192 10 us longer)
    hipLaunchKernelGGL(head_scale_kernel, dim3(1), dim3(1024), 0, st, u, q.most, w.scale);
    q.known = 1;
  }
  q.factor = (int)((s.n_max + 255) / 256);
  q.rows = (int)(s.n_max / 4);
  q.n_max = s.n_max; q.dim8 = s.dim8;
  q.ht = (uint16_t*)w.ht;
  q.tiles_n = (int)((s.dim8 + 63) / 64);
  const int tiles = half && dweight ? (int)(s.n_max / 64) * q.tiles_n : 0;
  PF_BY_SIZE(head_ready_kernel, dim3((unsigned)(q.factor + q.rows + tiles)), dim3(256), 0, st, q);
  widen(c, s, w, st);
  PF_CHECK_LAUNCH(c.who);
  const char* wide = s.copy_w ? w.wide : (const char*)weight;
  const int64_t n = s.n > 0 ? s.n : 1;
  for (int64_t v0 = 0; v0 < V; v0 += s.piece) {
    const int64_t rows = V - v0 < s.piece ? V - v0 : s.piece;
    if (!half) {
      const float* wp = (const float*)wide + v0 * s.depth;
      float* dz = (float*)w.dz;
      rc = product32(0, 0, rows, n, D, wp, s.depth, (const float*)w.hc, s.depth, dz, s.n_max, 0, k.count, st);
      if (rc != PF_OK) return rc;
      hipLaunchKernelGGL(head_dz32_kernel, dim3((unsigned)((s.n_max + 255) / 256), (unsigned)((rows + ROWS32 - 1) / ROWS32)), dim3(256), 0, st, dz, rows, s.n_max, v0, k.lab,
                         k.count, w.col);
      if (dhidden) rc = product32(1, 1, n, D, rows, dz, s.n_max, wp, s.depth, w.acc, s.depth, v0 > 0, k.count, st, s.shares.most, s.n_max * s.depth);
      if (rc != PF_OK) return rc;
      float* dw = (float*)dweight + v0 * D;
      if (dweight && s.n <= FEW_TOKENS32) {
        hipLaunchKernelGGL(head_weight_grad32_kernel, dim3((unsigned)((rows + 4 * FEW_ROWS32 - 1) / (4 * FEW_ROWS32)), (unsigned)((D + 255) / 256)), dim3(256), 0, st, dz, s.n_max,
                           k.count, (const float*)w.hc, s.depth, dw, rows, D);
      } else if (dweight) {
        rc = product32(0, 1, rows, D, n, dz, s.n_max, (const float*)w.hc, s.depth, dw, D, 0, k.count, st);
        if (rc != PF_OK) return rc;
      }
      continue;
    }
    PfHeadProduct p = {};
    p.w = wide + v0 * s.depth * 2;
    p.ldw = s.depth; p.v0 = v0; p.rows = rows; p.depth = s.depth;
    p.hc = w.hc; p.ldh = s.depth; p.n_max = s.n_max;
    p.count = k.count; p.lab = k.lab; p.col = w.col; p.dz = w.dz; p.ht = w.ht; p.dim = s.dim8;
    char* dw = (char*)dweight + v0 * D * 2;
    p.dw = s.narrow ? w.dw : dw;
    p.ldw_out = s.narrow ? s.depth : D;
    p.dh = w.acc; p.add = v0 > 0; p.shares = s.shares;
    p.unscale = w.scale;
    rc = pf_head_dz(dtype, p, st);
    if (rc == PF_OK && dhidden) rc = pf_head_dh(dtype, p, st);
    if (rc == PF_OK && dweight) rc = pf_head_dw(dtype, p, st);
    if (rc != PF_OK) return rc;
    if (dweight && s.narrow) pf_rows_narrow(w.dw, s.depth, dw, rows, D, st);
  }
  PF_CHECK_LAUNCH(c.who);
  if (!dhidden) return PF_OK;
  return pf_linear_ce_hidden_grad(weight, dtype, s.n, D, V, kept, nullptr, dhidden, workspace, stream);
}

extern "C" int pf_linear_ce_hidden_grad(const void* weight, int dtype, int64_t tokens, int64_t D, int64_t V, const void* kept, const float* times, void* dhidden,
                                        const void* workspace, void* stream) {
  const Call c = {"pf_linear_ce_hidden_grad", nullptr, dtype, 1, tokens, D, 0, D, weight, V};
  Sizes s = {};
  const int rc = check_call(c, s, true, tokens < 0 || D <= 0 || V <= 0 || sizes_of(c, s, true));
  if (rc != PF_OK) return rc;
  if (s.n == 0) return PF_OK;
  PF_REQUIRE(kept && dhidden && workspace, "%s: null pointer", c.who);
  PF_REQUIRE(pf_aligned(kept, 16) && pf_aligned(workspace, 16), "%s: kept and the workspace lie on boundaries of 256 bytes", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of((void*)kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, true);
  const int64_t lanes = D % 8 == 0 && pf_aligned(dhidden, 16) ? 512 : 64, units = (s.n * ((D + lanes - 1) / lanes) + 3) / 4;
  const dim3 grid((unsigned)(units < 16384 ? units : 16384));
  if (D % 8 == 0 && pf_aligned(dhidden, 16))
    hipLaunchKernelGGL(head_spread_kernel<8>, grid, dim3(256), 0, st, w.acc, s.depth, s.shares, s.n_max, k.count, k.inv, s.n, D, times, dhidden, dtype);
  else
    hipLaunchKernelGGL(head_spread_kernel<1>, grid, dim3(256), 0, st, w.acc, s.depth, s.shares, s.n_max, k.count, k.inv, s.n, D, times, dhidden, dtype);
  PF_CHECK_LAUNCH(c.who);
  return PF_OK;
}
