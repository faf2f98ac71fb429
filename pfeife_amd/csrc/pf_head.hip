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
// alike: 131072 classes, bf16, relative error of the gradients 2.8e-3 so, 1.7e-3 being the results' own rounding).  fp16: 2^13 times
// that, which keeps probabilities down to 2^-38.
// fp32: the same through pf_gemm, with a piece's logits in memory.
#include "pf_head.h"

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
  int64_t n, n_max, depth, piece;
  bool copy_w;
};

// tokens in groups of 1024, each of which counts for itself what lies before it: one launch, no order of arrival in the result
__global__ __launch_bounds__(1024) void head_index_kernel(const int64_t* labels, int64_t n, int64_t T, int shift, int64_t ignore, int64_t V,
                                                          int64_t n_max, Kept k, float* out) {
  __shared__ float sm[16];
  __shared__ int before[17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto label = [&](int64_t r) -> int64_t {
    if (r >= n || (shift && r % T == T - 1)) return ignore;
    return labels[r + shift];
  };
  int ahead = 0;
  for (int64_t r = tid; r < (int64_t)blockIdx.x * 1024; r += 1024) ahead += label(r) != ignore;
  // (at most 2^24 tokens: exact in fp32)
  const int base = (int)pf_block_sum<16>((float)ahead, sm);
  const int64_t r = (int64_t)blockIdx.x * 1024 + tid;
  const int64_t l = label(r);
  const bool in = l != ignore;
  const unsigned long long mask = __ballot(in);
  if (lane == 0) before[wave + 1] = __popcll(mask);
  __syncthreads();
  if (tid == 0) {
    before[0] = base;
    for (int w = 1; w <= 16; ++w) before[w] += before[w - 1];
  }
  __syncthreads();
  const int c = before[wave] + __popcll(mask & ((1ull << lane) - 1));
  if (r < n) k.inv[r] = in ? c : -1;
  if (in) {
    k.rows[c] = (int)r;
    k.lab[c] = l >= 0 && l < V ? (int)l : -2;
  } else if (out != nullptr && r < n && !(shift && r % T == T - 1)) {
    out[r / T * (T - shift) + r % T] = 0.f;
  }
  if (blockIdx.x == gridDim.x - 1) {
    const int total = before[16];
    if (tid == 0) *k.count = total;
    for (int64_t i = total + tid; i < n_max; i += 1024) k.lab[i] = -1;
  }
}

// The tokens that take part, one behind the other, zeros behind them up to a multiple of 64 (all: up to n_max) and in columns D .. depth - 1.
// One wavefront to a row.  U: 16 bytes, or one element where something is not aligned.
template <typename U>
__global__ __launch_bounds__(256) void head_gather_kernel(const char* h, int64_t T, int64_t sb, int64_t st, int64_t D, int64_t depth, const int* count,
                                                          const int* rows, char* hc, int64_t n_max, int all) {
  const int n = *count;
  const int64_t padded = all ? n_max : (n > 64 ? (n + 63) / 64 * 64 : 64);
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= padded) return;
  U* dst = (U*)hc + c * depth;
  const U* src = nullptr;
  if (c < n) {
    const int64_t r = rows[c];
    src = (const U*)h + (r / T) * sb + (r % T) * st;
  }
  const U zero = {};
  for (int64_t i = threadIdx.x & 63; i < depth; i += 64) dst[i] = src != nullptr && i < D ? src[i] : zero;
}

// a matrix with its rows' width raised, zeros in the new columns
template <typename U>
__global__ __launch_bounds__(256) void head_widen_kernel(const U* src, int64_t ld, int64_t D, U* dst, int64_t depth, int64_t rows) {
  const int64_t total = rows * depth;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / depth, c = i % depth;
    dst[i] = c < D ? src[r * ld + c] : (U)0;
  }
}

// Every token's statistics of all blocks merged, its loss; 32 tokens to a workgroup, 32 threads to a token.  The sum in 64 bits: a
// loss near zero is the logarithm of a sum near one.
__global__ __launch_bounds__(1024) void head_merge_kernel(const PfHeadPart* part, int64_t blocks, int64_t n_max, const float* zl, Kept k, double z_loss,
                                                          int64_t T, int shift, double* terms, float* out) {
  __shared__ float tops[32][33];
  __shared__ double sums[32][33];
  const int t = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int n = *k.count;
  const int64_t c = (int64_t)blockIdx.x * 32 + t;
  float m = LOWEST;
  double s = 0;
  if (c < n) {
#pragma unroll 4
    for (int64_t i = slice; i < blocks; i += 32) {
      const PfHeadPart p = part[i * n_max + c];
      const float x = fmaxf(m, p.top);
      s = s * (double)__builtin_amdgcn_exp2f((m - x) * LOG2E) + (double)(p.sum * __builtin_amdgcn_exp2f((p.top - x) * LOG2E));
      m = x;
    }
  }
  tops[slice][t] = m;
  sums[slice][t] = s;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  double term = 0;
  if (c < n) {
    float top = LOWEST;
    for (int i = 0; i < 32; ++i) top = fmaxf(top, tops[i][t]);
    double total = 0;
    for (int i = 0; i < 32; ++i) total += sums[i][t] * (double)__builtin_amdgcn_exp2f((tops[i][t] - top) * LOG2E);
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
// The number that brings the largest factor to `most`
__global__ __launch_bounds__(1024) void head_scale_kernel(const Upstream u, float most, float* scale) {
  __shared__ float sm[16];
  const int n = *u.k.count;
  float top = 0.f;
  for (int c = threadIdx.x; c < n; c += 1024) {
    float f, g;
    factors(u, n, c, f, g);
    top = fmaxf(top, fmaxf(fabsf(f), fabsf(g)));
  }
  top = pf_block_max<16>(top, sm);
  // (nothing to scale by where all factors are zero, one is infinite, or the quotient would be)
  if (threadIdx.x == 0) *scale = top > 1e-30f && top < INFINITY ? most / top : 1.f;
}
__global__ __launch_bounds__(256) void head_factor_kernel(const Upstream u, const float* scale, PfHeadColumn* col, int64_t n_max) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= n_max) return;
  const int n = *u.k.count;
  PfHeadColumn o = {0.f, 0.f, 0.f, 0.f};     // (behind the last token: zeros times exp(0))
  if (c < n) {
    const float s = scale != nullptr ? *scale : 1.f;
    o.top = u.k.top[c];
    o.bias = u.k.bias[c];
    factors(u, n, c, o.f, o.g);
    o.f *= s;
    o.g *= s;
  }
  col[c] = o;
}

// The gradient of every row of the hidden state: a token's sum rounded once (times a loss scale first), zeros where it took no part
template <int W>
__global__ __launch_bounds__(256) void head_spread_kernel(const float* acc, int64_t ld, const int* inv, int64_t n, int64_t D, const float* times, void* dh, int dt) {
  const float by = times != nullptr ? *times : 1.f;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4) {
    const int c = inv[r];
    for (int64_t i = (int64_t)(threadIdx.x & 63) * W; i < D; i += 64 * W) {
      float v[W];
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = 0.f;
      if (c >= 0) {
        ld_vec<W>(acc, c * ld + i, PF_F32, v);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] *= by;
      }
      st_vec<W>(dh, r * D + i, dt, v);
    }
  }
}

// fp32: statistics of 128 vocabulary rows of a piece in memory, z[row][token]
__global__ __launch_bounds__(256) void head_stats32_kernel(const float* z, int64_t rows, int64_t n_max, int64_t v0, const int* lab, const int* count, PfHeadPart* part,
                                                           float* zl) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, r0 = (int64_t)blockIdx.y * 128;
  if (c >= *count) return;
  const int64_t r1 = r0 + 128 < rows ? r0 + 128 : rows;
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
__global__ __launch_bounds__(256) void head_dz32_kernel(float* z, int64_t rows, int64_t n_max, int64_t v0, const int* lab, const PfHeadColumn* col) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, r0 = (int64_t)blockIdx.y * 128;
  if (c >= n_max) return;
  const int64_t r1 = r0 + 128 < rows ? r0 + 128 : rows;
  const int64_t at = lab[c] >= 0 ? (int64_t)lab[c] - v0 : -1;
  const PfHeadColumn k = col[c];
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float v = k.f * __builtin_amdgcn_exp2f(fmaf(z[r * n_max + c] - k.top, LOG2E, k.bias));
    z[r * n_max + c] = r == at ? v - k.g : v;
  }
}

int bad(const char* who, const char* what) {
  pf_set_error("%s: %s", who, what);
  return PF_ERR_INVALID;
}

// Vocabulary rows of a piece: its dz (fp32: its logits) in 256 MB, in whole tiles
int64_t piece_rows(int64_t n_max, int64_t V, int64_t size) {
  int64_t rows = (256ll << 20) / (n_max * size) / 256 * 256;
  if (rows < 256) rows = 256;
  return rows < V ? rows : V;
}
// ... and of one whose weights a buffer's 32-bit offsets reach
int64_t reach_rows(int64_t ldw) { return ((1ll << 31) / (ldw * 2) - 512) / 256 * 256; }

struct Call {
  const char* who;
  const void* h;
  int dtype;
  int64_t B, T, D, sb, st;
  const void* w;
  int64_t V;
};

bool sizes_of(const Call& c, Sizes& s) {
  const int64_t es = c.dtype == PF_F32 ? 4 : 2;
  s.n = c.B * c.T;
  s.n_max = round_up(s.n > 0 ? s.n : 1, 64);
  s.depth = c.dtype == PF_F32 ? round_up(c.D, 4) : (c.D < 64 ? 64 : round_up(c.D, 8));
  s.copy_w = c.dtype != PF_F32 && (s.depth != c.D || !pf_aligned(c.w, 16));
  s.piece = piece_rows(s.n_max, c.V, es);
  if (es == 2 && s.piece > reach_rows(s.depth)) s.piece = reach_rows(s.depth);
  return s.n < (1ll << 24) && c.V < (1ll << 31) && s.n_max * s.depth * 4 < (1ll << 31) - 64 && s.piece * s.n_max * es < (1ll << 31) - 64 &&
         s.depth < (1ll << 19);
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
  char* dz; char* ht; float* acc; PfHeadColumn* col; float* scale;               // backward (dz: fp32's logits in both)
};
Work carve(Carve& a, const Call& c, const Sizes& s, bool back) {
  const int64_t es = c.dtype == PF_F32 ? 4 : 2;
  Work w = {};
  w.hc = (char*)a.take(s.n_max * s.depth * es);
  if (s.copy_w) w.wide = (char*)a.take(c.V * s.depth * 2);
  if (back || es == 4) w.dz = (char*)a.take(s.piece * s.n_max * es);
  if (!back) {
    w.part = (PfHeadPart*)a.take((es == 4 ? (c.V + 127) / 128 : pf_head_blocks(c.V, s.n_max, s.depth)) * s.n_max * 8);
    w.zl = (float*)a.take(s.n_max * 4);
    w.terms = (double*)a.take(s.n_max * 8);
  } else {
    if (es == 2) w.ht = (char*)a.take(c.D * s.n_max * 2);
    w.col = (PfHeadColumn*)a.take(s.n_max * 16);
    w.scale = (float*)a.take(4);
    w.acc = (float*)a.take(s.n_max * s.depth * 4);
  }
  return w;
}

int check_call(const Call& c, const Sizes& s, bool ok) {
  if (c.dtype != PF_F32 && c.dtype != PF_F16 && c.dtype != PF_BF16) return bad(c.who, "bad dtype");
  if (c.B < 0 || c.T < 0 || c.D <= 0 || c.V <= 0) return bad(c.who, "bad sizes");
  if (!ok) {
    pf_set_error("%s: %lld tokens of width %lld and %lld classes: too many for one call (the tokens' fp32 gradient has to stay below 2 GiB)", c.who, (long long)s.n,
                 (long long)c.D, (long long)c.V);
    return PF_ERR_INVALID;
  }
  return PF_OK;
}

void gather(const Call& c, const Sizes& s, const Work& w, const Kept& k, hipStream_t st) {
  const int64_t es = c.dtype == PF_F32 ? 4 : 2, per = 16 / es;
  const int all = es == 4;
  const dim3 grid((unsigned)((s.n_max + 3) / 4));
  if (pf_aligned(c.h, 16) && c.D % per == 0 && s.depth % per == 0 && c.sb % per == 0 && c.st % per == 0)
    hipLaunchKernelGGL(head_gather_kernel<uint4>, grid, dim3(256), 0, st, (const char*)c.h, c.T, c.sb / per, c.st / per, c.D / per, s.depth / per, k.count, k.rows, w.hc,
                       s.n_max, all);
  else if (es == 4)
    hipLaunchKernelGGL(head_gather_kernel<uint32_t>, grid, dim3(256), 0, st, (const char*)c.h, c.T, c.sb, c.st, c.D, s.depth, k.count, k.rows, w.hc, s.n_max, all);
  else
    hipLaunchKernelGGL(head_gather_kernel<uint16_t>, grid, dim3(256), 0, st, (const char*)c.h, c.T, c.sb, c.st, c.D, s.depth, k.count, k.rows, w.hc, s.n_max, all);
}
void widen(const Call& c, const Sizes& s, const Work& w, hipStream_t st) {
  if (s.copy_w)
    hipLaunchKernelGGL(head_widen_kernel<uint16_t>, dim3(4096), dim3(256), 0, st, (const uint16_t*)c.w, c.D, c.D, (uint16_t*)w.wide, s.depth, c.V);
}

// a product over fp32 operands
int product32(int a_trans, int b_trans, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int beta,
              hipStream_t st) {
  pf_gemm_desc d = {};
  d.in_dtype = d.c_dtype = PF_F32;
  d.a_trans = a_trans; d.b_trans = b_trans;
  d.M = M; d.N = N; d.K = K;
  d.A = A; d.lda = lda; d.B = B; d.ldb = ldb; d.C = C; d.ldc = ldc;
  d.batch1 = d.batch2 = 1;
  d.alpha = 1.f;
  d.beta = beta;
  return pf_gemm(&d, st);
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
  const int rc = check_call(c, s, tokens < 0 || D <= 0 || V <= 0 || sizes_of(c, s));
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
  int rc = check_call(c, s, B < 0 || T < 0 || D <= 0 || V <= 0 || sizes_of(c, s));
  if (rc != PF_OK) return rc;
  PF_REQUIRE((shift == 0 || shift == 1) && reduction >= 0 && reduction <= 2, "%s: shift is 0 or 1, reduction 0, 1 or 2", c.who);
  PF_REQUIRE(loss && kept && workspace && weight && (s.n == 0 || (hidden && labels)), "%s: null pointer", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of(kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, false);
  float* out = reduction == 0 ? loss : nullptr;
  hipLaunchKernelGGL(head_index_kernel, dim3((unsigned)((s.n + 1023) / 1024 > 0 ? (s.n + 1023) / 1024 : 1)), dim3(1024), 0, st, labels, s.n, T > 0 ? T : 1, shift,
                     ignore_index, V, s.n_max, k, out);
  gather(c, s, w, k, st);
  widen(c, s, w, st);
  PF_CHECK_LAUNCH(c.who);
  int64_t blocks = 0;
  if (dtype == PF_F32) {
    for (int64_t v0 = 0; v0 < V; v0 += s.piece) {
      const int64_t rows = V - v0 < s.piece ? V - v0 : s.piece;
      rc = product32(0, 0, rows, s.n_max, D, (const float*)weight + v0 * D, D, w.hc, s.depth, w.dz, s.n_max, 0, st);
      if (rc != PF_OK) return rc;
      hipLaunchKernelGGL(head_stats32_kernel, dim3((unsigned)((s.n_max + 255) / 256), (unsigned)((rows + 127) / 128)), dim3(256), 0, st, (const float*)w.dz, rows,
                         s.n_max, v0, k.lab, k.count, w.part + blocks * s.n_max, w.zl);
      blocks += (rows + 127) / 128;
    }
  } else {
    PfHeadProduct p = {};
    p.ldw = s.depth; p.depth = s.depth;
    p.hc = w.hc; p.ldh = s.depth; p.n_max = s.n_max;
    p.count = k.count; p.lab = k.lab; p.zl = w.zl;
    const int64_t reach = reach_rows(s.depth);
    for (int64_t v0 = 0; v0 < V; v0 += reach) {
      p.v0 = v0;
      p.rows = V - v0 < reach ? V - v0 : reach;
      p.w = (s.copy_w ? w.wide : (const char*)weight) + v0 * s.depth * 2;
      p.part = w.part + blocks * s.n_max;
      rc = pf_head_stats(dtype, p, st);
      if (rc != PF_OK) return rc;
      blocks += pf_head_blocks(p.rows, s.n_max, s.depth);
    }
  }
  hipLaunchKernelGGL(head_merge_kernel, dim3((unsigned)((s.n_max + 31) / 32)), dim3(1024), 0, st, w.part, blocks, s.n_max, w.zl, k, z_loss, T > 0 ? T : 1, shift,
                     reduction == 0 ? nullptr : w.terms, out);
  if (reduction != 0) hipLaunchKernelGGL(head_reduce_kernel, dim3(1), dim3(1024), 0, st, w.terms, k.count, reduction == 1, loss);
  PF_CHECK_LAUNCH(c.who);
  return PF_OK;
}

extern "C" int pf_linear_ce_bwd(const void* hidden, int dtype, int64_t B, int64_t T, int64_t D, int64_t sb, int64_t st_, const void* weight, int64_t V,
                                double z_loss, int mean, const void* kept, const float* grad, int64_t g_sb, int64_t g_st, void* dhidden, void* dweight,
                                void* workspace, void* stream) {
  const Call c = {"pf_linear_ce_bwd", hidden, dtype, B, T, D, sb, st_, weight, V};
  Sizes s = {};
  int rc = check_call(c, s, B < 0 || T < 0 || D <= 0 || V <= 0 || sizes_of(c, s));
  if (rc != PF_OK) return rc;
  PF_REQUIRE(kept && workspace && weight && grad && (s.n == 0 || hidden), "%s: null pointer", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of((void*)kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, true);
  const Upstream u = {grad, g_sb, g_st, T > 0 ? T : 1, mean, z_loss, k};
  const bool narrow = dtype != PF_F32;
  if (narrow) hipLaunchKernelGGL(head_scale_kernel, dim3(1), dim3(1024), 0, st, u, dtype == PF_F16 ? 8192.f : 1.f, w.scale);
  hipLaunchKernelGGL(head_factor_kernel, dim3((unsigned)((s.n_max + 255) / 256)), dim3(256), 0, st, u, (const float*)(narrow ? w.scale : nullptr), w.col, s.n_max);
  gather(c, s, w, k, st);
  widen(c, s, w, st);
  PF_CHECK_LAUNCH(c.who);
  if (dtype != PF_F32 && dweight) {
    rc = pf_transpose_cast(w.hc, dtype, s.depth, w.ht, dtype, s.n_max, s.n_max, D, stream);
    if (rc != PF_OK) return rc;
  }
  for (int64_t v0 = 0; v0 < V; v0 += s.piece) {
    const int64_t rows = V - v0 < s.piece ? V - v0 : s.piece;
    if (dtype == PF_F32) {
      const float* wp = (const float*)weight + v0 * D;
      rc = product32(0, 0, rows, s.n_max, D, wp, D, w.hc, s.depth, w.dz, s.n_max, 0, st);
      if (rc != PF_OK) return rc;
      hipLaunchKernelGGL(head_dz32_kernel, dim3((unsigned)((s.n_max + 255) / 256), (unsigned)((rows + 127) / 128)), dim3(256), 0, st, (float*)w.dz, rows, s.n_max, v0,
                         k.lab, w.col);
      if (dhidden) rc = product32(1, 1, s.n_max, D, rows, w.dz, s.n_max, wp, D, w.acc, s.depth, v0 > 0, st);
      if (rc == PF_OK && dweight) rc = product32(0, 1, rows, D, s.n_max, w.dz, s.n_max, w.hc, s.depth, (float*)dweight + v0 * D, D, 0, st);
      if (rc != PF_OK) return rc;
      continue;
    }
    PfHeadProduct p = {};
    p.w = (s.copy_w ? w.wide : (const char*)weight) + v0 * s.depth * 2;
    p.ldw = s.depth; p.v0 = v0; p.rows = rows; p.depth = s.depth;
    p.hc = w.hc; p.ldh = s.depth; p.n_max = s.n_max;
    p.count = k.count; p.lab = k.lab; p.col = w.col; p.dz = w.dz; p.ht = w.ht; p.dim = D;
    p.dw = dweight ? (char*)dweight + v0 * D * 2 : nullptr;
    p.dh = w.acc; p.add = v0 > 0;
    p.unscale = w.scale;
    rc = pf_head_dz(dtype, p, st);
    if (rc == PF_OK && dhidden) rc = pf_head_dh(dtype, p, st);
    if (rc == PF_OK && dweight) rc = pf_head_dw(dtype, p, st);
    if (rc != PF_OK) return rc;
  }
  if (!dhidden) return PF_OK;
  return pf_linear_ce_hidden_grad(weight, dtype, s.n, D, V, kept, nullptr, dhidden, workspace, stream);
}

extern "C" int pf_linear_ce_hidden_grad(const void* weight, int dtype, int64_t tokens, int64_t D, int64_t V, const void* kept, const float* times, void* dhidden,
                                        const void* workspace, void* stream) {
  const Call c = {"pf_linear_ce_hidden_grad", nullptr, dtype, 1, tokens, D, 0, D, weight, V};
  Sizes s = {};
  const int rc = check_call(c, s, tokens < 0 || D <= 0 || V <= 0 || sizes_of(c, s));
  if (rc != PF_OK) return rc;
  if (s.n == 0) return PF_OK;
  PF_REQUIRE(kept && dhidden && workspace, "%s: null pointer", c.who);
  hipStream_t st = (hipStream_t)stream;
  const Kept k = kept_of((void*)kept, s.n_max);
  Carve a = {(char*)workspace};
  const Work w = carve(a, c, s, true);
  const dim3 grid((unsigned)((s.n + 3) / 4 < 8192 ? (s.n + 3) / 4 : 8192));
  if (D % 8 == 0 && pf_aligned(dhidden, 16))
    hipLaunchKernelGGL(head_spread_kernel<8>, grid, dim3(256), 0, st, w.acc, s.depth, k.inv, s.n, D, times, dhidden, dtype);
  else
    hipLaunchKernelGGL(head_spread_kernel<1>, grid, dim3(256), 0, st, w.acc, s.depth, k.inv, s.n, D, times, dhidden, dtype);
  PF_CHECK_LAUNCH(c.who);
  return PF_OK;
}
