// Log-probabilities of given tokens, and the preference and policy losses over them, straight from the logits.
//
// A row of logits x (classes V) scores the label y: with m = max x, c = log2(e) / temperature and Z = sum_j 2^((x_j - m) c),
//   logprob = (x_y - m) / temperature - ln Z,      p_j = 2^((x_j - m) c) / Z,
// and whatever is formed from the logprobs has the gradient  dx_j = g (onehot_j - p_j) / temperature  with g = d loss / d logprob.
// Rows whose label is ignore_index take no part: they are not read, their logprob is 0 and their gradient zeros.  A label outside
// the vocabulary reads nothing either and gives NaN.  Exponentials and their partial sums are fp32 (relative error some 1e-7 each, of
// random sign); what a row ends in, (x_y - m) / temperature - ln Z, and every sum over tokens is formed in double, because a sequence's
// log-probability is compared with another that differs from it in the fourth digit, and a ratio with a clip border.
// Sums run in a fixed order: results are the same from run to run.
#include "pf_common.h"

namespace {

// [B, T] rows of V logits, and the labels [B, T] contiguous; row t of a sequence is scored against label t + shift, so a sequence has
// T - shift scored rows; the rows behind them have zeros for a gradient.
struct TokenRows {
  const void* logits;
  int64_t sb, st;         // elements between sequences and between rows
  const int64_t* labels;
  int64_t B, T, V;
  int64_t ignore_index;
  int shift;
  float c, c_lo;          // log2(e) / temperature, and what its rounding lost
  double inv_temp;
};
struct GradRows {
  void* dx;               // null: none wanted
  int64_t sb, st;
};

enum LabelKind { LABEL_SKIP, LABEL_OK, LABEL_BAD };
__device__ __forceinline__ LabelKind label_kind(const TokenRows& r, int64_t y) {
  if (y == r.ignore_index) return LABEL_SKIP;
  return y >= 0 && y < r.V ? LABEL_OK : LABEL_BAD;
}

struct RowStats { float m, z; };

// Maximum and sum of exponentials of one row by the whole workgroup (256 threads).
template <int DT>
__device__ RowStats row_stats(const TokenRows& r, const void* x, int64_t at, float* sm) {
  float m = -INFINITY;
  for (int64_t j = threadIdx.x; j < r.V; j += 256) m = fmaxf(m, Codec<DT>::load(x, at + j));
  m = pf_block_max<4>(m, sm);
  float z = 0.f;
  for (int64_t j = threadIdx.x; j < r.V; j += 256) {
    const float t = Codec<DT>::load(x, at + j) - m;
    z += exp2f(fmaf(t, r.c, t == -INFINITY ? 0.f : t * r.c_lo));      // (a sum of many tokens' logprobs would show c's rounding)
  }
  return {m, pf_block_sum<4>(z, sm)};
}

template <int DT>
__device__ __forceinline__ double row_logprob(const TokenRows& r, int64_t at, int64_t y, const RowStats& s) {
  return ((double)Codec<DT>::load(r.logits, at + y) - (double)s.m) * r.inv_temp - log((double)s.z);
}

// dx = g (onehot - p) / temperature over one row
template <int DT>
__device__ __forceinline__ void row_gradient(const TokenRows& r, int64_t at, int64_t y, float m, float inv_z, float g, void* dx, int64_t to) {
  g *= (float)r.inv_temp;
  for (int64_t j = threadIdx.x; j < r.V; j += 256) {
    const float p = exp2f((Codec<DT>::load(r.logits, at + j) - m) * r.c) * inv_z;
    Codec<DT>::store(dx, to + j, g * ((j == y ? 1.f : 0.f) - p));
  }
}
template <int DT>
__device__ __forceinline__ void row_zeros(const TokenRows& r, void* dx, int64_t to) {
  for (int64_t j = threadIdx.x; j < r.V; j += 256) Codec<DT>::store(dx, to + j, 0.f);
}

// stats[row] = {maximum, 1 / sum}; for rows that take no part {0, 0}
template <int DT, typename Out>
__global__ __launch_bounds__(256) void token_logprob_kernel(const TokenRows r, Out* logprobs, float2* stats) {
  __shared__ float sm[4];
  const int64_t R = r.T - r.shift, rows = r.B * R;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t b = row / R, t = row % R, at = b * r.sb + t * r.st;
    const int64_t y = r.labels[b * r.T + t + r.shift];
    const LabelKind kind = label_kind(r, y);
    RowStats s = {0.f, 0.f};
    if (kind == LABEL_OK) s = row_stats<DT>(r, r.logits, at, sm);
    if (threadIdx.x == 0) {
      logprobs[row] = kind == LABEL_OK ? (Out)row_logprob<DT>(r, at, y, s) : kind == LABEL_BAD ? (Out)NAN : (Out)0;
      if (stats) stats[row] = kind == LABEL_OK ? make_float2(s.m, 1.f / s.z) : make_float2(0.f, kind == LABEL_BAD ? NAN : 0.f);
    }
  }
}

// dlogits from the rows' statistics and g = coef[b * g_sb + t * g_st] (* scale[0]).  unless_one: nothing is done where scale[0] is one.
template <int DT>
__global__ __launch_bounds__(256) void token_gradient_kernel(const TokenRows r, const GradRows d, const float2* stats, const float* coef,
                                                             int64_t g_sb, int64_t g_st, const float* scale, int unless_one) {
  const float by = scale ? scale[0] : 1.f;
  if (unless_one && by == 1.f) return;
  const int64_t R = r.T - r.shift, rows = r.B * r.T;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t b = row / r.T, t = row % r.T, at = b * r.sb + t * r.st, to = b * d.sb + t * d.st;
    const int64_t y = t < R ? r.labels[row + r.shift] : 0;
    const LabelKind kind = t < R ? label_kind(r, y) : LABEL_SKIP;
    if (kind == LABEL_SKIP) {
      row_zeros<DT>(r, d.dx, to);
    } else {
      const float2 s = stats[b * R + t];
      row_gradient<DT>(r, at, y, s.x, s.y, coef[b * g_sb + t * g_st] * by, d.dx, to);
    }
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int NW>
__device__ __forceinline__ double block_sum(double v, double* sm) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += sm[i];
  return s;
}

// ---- preference ------------------------------------------------------------------------------------------------------------
// A workgroup to a pair (sequences 2i, 2i + 1):  reward = beta (sum or mean of logprobs - ref),  D = reward_2i - reward_2i+1,
//   loss_i = -(1 - e) ln sigma(D) - e ln sigma(-D),   d loss_i / dD = sigma(D) - (1 - e).
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }   // -ln sigma(-x)

__global__ __launch_bounds__(256) void preference_pair_kernel(const double* logprobs, const int64_t* labels, int64_t T, int shift, int64_t ignore_index,
                                                              const float* ref, double beta, double smoothing, int average, int64_t pairs,
                                                              float* rewards, float* coef, double* pair_loss) {
  __shared__ double sm[4];
  const int64_t R = T - shift;
  for (int64_t i = blockIdx.x; i < pairs; i += gridDim.x) {
    double reward[2], per_token[2];
    for (int k = 0; k < 2; ++k) {
      const int64_t b = 2 * i + k;
      double s = 0.0, n = 0.0;
      for (int64_t t = threadIdx.x; t < R; t += 256) {
        s += logprobs[b * R + t];
        if (average) n += labels[b * T + t + shift] != ignore_index ? 1.0 : 0.0;
      }
      s = block_sum<4>(s, sm);
      per_token[k] = 1.0;
      if (average) {
        n = block_sum<4>(n, sm);
        per_token[k] = n > 0.0 ? 1.0 / n : 0.0;
      }
      reward[k] = beta * (s * per_token[k] - (double)ref[b]);
    }
    if (threadIdx.x == 0) {
      const double D = reward[0] - reward[1];
      const double up = 1.0 / (1.0 + exp(-D)) - (1.0 - smoothing);
      pair_loss[i] = (1.0 - smoothing) * softplus(-D) + smoothing * softplus(D);
      for (int k = 0; k < 2; ++k) {
        rewards[2 * i + k] = (float)reward[k];
        coef[2 * i + k] = (float)((k ? -up : up) * beta * per_token[k] / (double)pairs);
      }
    }
  }
}

// out[k] = sum over n of in[k * n + i] (* scale), in double
__global__ __launch_bounds__(256) void sums_kernel(const double* in, int64_t n, double scale, float* out0, float* out1) {
  __shared__ double sm[4];
  for (int k = 0; k < (out1 ? 2 : 1); ++k) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) s += in[k * n + i];
    s = block_sum<4>(s, sm);
    if (threadIdx.x == 0) (k ? out1 : out0)[0] = (float)(s * scale);
  }
}

// ---- policy ----------------------------------------------------------------------------------------------------------------
// weight of every token of sequence b: 1 / (tokens that count), or by_sequence 1 / (its own such tokens * sequences that have any)
__global__ __launch_bounds__(256) void token_weights_kernel(const TokenRows r, int by_sequence, double* weights) {
  __shared__ double sm[4];
  const int64_t R = r.T - r.shift;
  double total = 0.0;
  for (int64_t b = 0; b < r.B; ++b) {
    double n = 0.0;
    for (int64_t t = threadIdx.x; t < R; t += 256) n += r.labels[b * r.T + t + r.shift] != r.ignore_index ? 1.0 : 0.0;
    n = block_sum<4>(n, sm);
    if (threadIdx.x == 0) weights[b] = n;
    total += by_sequence ? (n > 0.0 ? 1.0 : 0.0) : n;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < r.B; b += 256) {
    const double n = weights[b];
    weights[b] = n > 0.0 ? 1.0 / (by_sequence ? n * total : total) : 0.0;
  }
}

struct PolicyArgs {
  const float* old;      // [B, R]
  const float* ref;      // [B, R] or null
  const float* adv;
  int64_t a_sb, a_st;
  double low, high, kl_coef;
};

// One token:  -min(r A, clip(r) A) + kl_coef (e^q - q - 1)  with r = e^(logprob - old), q = ref - logprob; g is its derivative by
// the logprob (at the clip's borders that of r A).
struct TokenTerms { double loss, kl, g; };
__device__ __forceinline__ TokenTerms policy_token(const PolicyArgs& a, int64_t row, int64_t b, int64_t t, double logprob) {
  const double ratio = exp(logprob - (double)a.old[row]);
  const double A = (double)a.adv[b * a.a_sb + t * a.a_st];
  const double clipped = ratio < a.low ? a.low : ratio > a.high ? a.high : ratio;
  const bool outside = A >= 0.0 ? ratio > a.high : ratio < a.low;
  TokenTerms o;
  o.loss = -(outside ? clipped : ratio) * A;
  o.g = outside ? 0.0 : -ratio * A;
  o.kl = 0.0;
  if (a.ref) {
    const double q = (double)a.ref[row] - logprob, e = expm1(q);
    o.kl = e - q;
    o.loss += a.kl_coef * o.kl;
    o.g -= a.kl_coef * e;
  }
  return o;
}

// A row's log-probability, its part of the loss and, where wanted, its gradient.  terms: [2][B * R], weighted
template <int DT>
__global__ __launch_bounds__(256) void policy_kernel(const TokenRows r, const GradRows d, const PolicyArgs a, const double* weights, float* logprobs,
                                                     float2* stats, float* coef, double* terms) {
  __shared__ float sm[4];
  __shared__ float shared_g;
  const int64_t R = r.T - r.shift, all = r.B * R, rows = r.B * r.T;
  for (int64_t place = blockIdx.x; place < rows; place += gridDim.x) {
    const int64_t b = place / r.T, t = place % r.T, at = b * r.sb + t * r.st, to = b * d.sb + t * d.st, row = b * R + t;
    const int64_t y = t < R ? r.labels[place + r.shift] : 0;
    const LabelKind kind = t < R ? label_kind(r, y) : LABEL_SKIP;
    RowStats s = {0.f, 0.f};
    if (kind == LABEL_OK) s = row_stats<DT>(r, r.logits, at, sm);
    if (threadIdx.x == 0 && t < R) {
      TokenTerms o = {0.0, 0.0, 0.0};
      double lp = 0.0;
      if (kind != LABEL_SKIP) {
        lp = kind == LABEL_OK ? row_logprob<DT>(r, at, y, s) : (double)NAN;
        o = policy_token(a, row, b, t, lp);
      }
      const double w = weights[b];
      logprobs[row] = (float)lp;
      terms[row] = kind == LABEL_SKIP ? 0.0 : w * o.loss;
      terms[all + row] = kind == LABEL_SKIP ? 0.0 : w * o.kl;
      const float g = kind == LABEL_SKIP ? 0.f : (float)(w * o.g);
      shared_g = g;
      if (coef) {
        coef[row] = g;
        stats[row] = kind == LABEL_OK ? make_float2(s.m, 1.f / s.z) : make_float2(0.f, kind == LABEL_BAD ? NAN : 0.f);
      }
    }
    if (!d.dx) continue;
    __syncthreads();
    if (kind == LABEL_SKIP) row_zeros<DT>(r, d.dx, to);
    else row_gradient<DT>(r, at, y, s.m, kind == LABEL_OK ? 1.f / s.z : NAN, shared_g, d.dx, to);
    __syncthreads();
  }
}

constexpr int64_t MAX_BLOCKS = 1 << 20;
inline dim3 rows_grid(int64_t rows) { return dim3((unsigned)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS)); }

int check_rows(const char* who, const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
               double temperature) {
  PF_REQUIRE(pf_is_float_dtype(dtype), "%s: logits are fp32, fp16 or bf16", who);
  PF_REQUIRE(B >= 0 && T >= 0 && V >= 1 && sb >= 0 && st >= 0, "%s: bad sizes", who);
  PF_REQUIRE(shift == 0 || shift == 1, "%s: shift is 0 or 1", who);
  PF_REQUIRE(temperature > 0.0 && temperature >= 1e-6 && temperature <= 1e6, "%s: temperature must lie in [1e-6, 1e6]", who);
  PF_REQUIRE(B * T == 0 || (logits && labels), "%s: null pointer", who);
  PF_REQUIRE(T < (1ll << 31) && B < (1ll << 31) && B * T < (1ll << 40), "%s: too many rows", who);
  return PF_OK;
}

TokenRows token_rows(const void* logits, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
                     int64_t ignore_index, double temperature) {
  const double c = 1.4426950408889634 / temperature;
  return {logits, sb, st, labels, B, T, V, ignore_index, shift, (float)c, (float)(c - (double)(float)c), 1.0 / temperature};
}

}  // namespace

#define PF_BY_DTYPE(dt, CALL)                \
  do {                                       \
    if (dt == PF_F32) { CALL(PF_F32); }      \
    else if (dt == PF_F16) { CALL(PF_F16); } \
    else { CALL(PF_BF16); }                  \
  } while (0)

extern "C" int pf_token_logprob_fwd(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels,
                                    int shift, int64_t ignore_index, double temperature, float* logprobs, float* stats, void* stream) {
  if (int rc = check_rows("pf_token_logprob_fwd", logits, dtype, B, T, V, sb, st, labels, shift, temperature)) return rc;
  if (B == 0 || T <= shift) return PF_OK;
  PF_REQUIRE(logprobs, "pf_token_logprob_fwd: null pointer");
  const TokenRows r = token_rows(logits, B, T, V, sb, st, labels, shift, ignore_index, temperature);
#define CALL(DT) hipLaunchKernelGGL((token_logprob_kernel<DT, float>), rows_grid(B * (T - shift)), dim3(256), 0, (hipStream_t)stream, r, logprobs, (float2*)stats)
  PF_BY_DTYPE(dtype, CALL);
#undef CALL
  PF_CHECK_LAUNCH("pf_token_logprob_fwd");
  return PF_OK;
}

extern "C" int pf_token_logprob_bwd(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels,
                                    int shift, int64_t ignore_index, double temperature, const float* stats, const float* coef, int64_t g_sb,
                                    int64_t g_st, const float* scale, int unless_one, void* dlogits, int64_t d_sb, int64_t d_st, void* stream) {
  if (int rc = check_rows("pf_token_logprob_bwd", logits, dtype, B, T, V, sb, st, labels, shift, temperature)) return rc;
  PF_REQUIRE(g_sb >= 0 && g_st >= 0 && d_sb >= 0 && d_st >= 0, "pf_token_logprob_bwd: bad strides");
  PF_REQUIRE(!unless_one || scale, "pf_token_logprob_bwd: unless_one needs a scale");
  if (B * T == 0) return PF_OK;
  PF_REQUIRE(dlogits && (T <= shift || (stats && coef)), "pf_token_logprob_bwd: null pointer");
  const TokenRows r = token_rows(logits, B, T, V, sb, st, labels, shift, ignore_index, temperature);
  const GradRows d = {dlogits, d_sb, d_st};
#define CALL(DT)                                                                                                                        \
  hipLaunchKernelGGL(token_gradient_kernel<DT>, rows_grid(B * T), dim3(256), 0, (hipStream_t)stream, r, d, (const float2*)stats, coef, g_sb, g_st, \
                     scale, unless_one)
  PF_BY_DTYPE(dtype, CALL);
#undef CALL
  PF_CHECK_LAUNCH("pf_token_logprob_bwd");
  return PF_OK;
}

extern "C" int64_t pf_preference_workspace(int64_t B, int64_t T, int shift) { return B / 2 + B * (T > shift ? T - shift : 0); }

extern "C" int pf_preference_loss(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels,
                                  int shift, int64_t ignore_index, const float* ref, double beta, double label_smoothing, int length_average,
                                  float* loss, float* rewards, float* stats, float* coef, double* workspace, void* stream) {
  if (int rc = check_rows("pf_preference_loss", logits, dtype, B, T, V, sb, st, labels, shift, 1.0)) return rc;
  PF_REQUIRE(B >= 2 && B % 2 == 0, "pf_preference_loss: sequences come in pairs");
  PF_REQUIRE(label_smoothing >= 0.0 && label_smoothing <= 1.0, "pf_preference_loss: label_smoothing must lie in [0, 1]");
  PF_REQUIRE(ref && loss && rewards && coef && workspace, "pf_preference_loss: null pointer");
  const int64_t pairs = B / 2, R = T > shift ? T - shift : 0;
  double* logprobs = workspace + pairs;
  if (R > 0) {
    const TokenRows r = token_rows(logits, B, T, V, sb, st, labels, shift, ignore_index, 1.0);
#define CALL(DT) hipLaunchKernelGGL((token_logprob_kernel<DT, double>), rows_grid(B * R), dim3(256), 0, (hipStream_t)stream, r, logprobs, (float2*)stats)
    PF_BY_DTYPE(dtype, CALL);
#undef CALL
  }
  hipLaunchKernelGGL(preference_pair_kernel, rows_grid(pairs), dim3(256), 0, (hipStream_t)stream, logprobs, labels, R + shift, shift, ignore_index, ref,
                     beta, label_smoothing, length_average, pairs, rewards, coef, workspace);
  hipLaunchKernelGGL(sums_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, workspace, pairs, 1.0 / (double)pairs, loss, (float*)nullptr);
  PF_CHECK_LAUNCH("pf_preference_loss");
  return PF_OK;
}

extern "C" int64_t pf_policy_workspace(int64_t B, int64_t T, int shift) { return B + 2 * B * (T > shift ? T - shift : 0); }

extern "C" int pf_policy_loss(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
                              int64_t ignore_index, double temperature, const float* old_logprobs, const float* advantages, int64_t a_sb, int64_t a_st,
                              const float* ref_logprobs, double clip_low, double clip_high, double kl_coef, int by_sequence, float* loss, float* kl,
                              float* logprobs, float* stats, float* coef, void* dlogits, int64_t d_sb, int64_t d_st, double* workspace, void* stream) {
  if (int rc = check_rows("pf_policy_loss", logits, dtype, B, T, V, sb, st, labels, shift, temperature)) return rc;
  PF_REQUIRE(a_sb >= 0 && a_st >= 0 && d_sb >= 0 && d_st >= 0, "pf_policy_loss: bad strides");
  PF_REQUIRE(clip_low >= 0.0 && clip_high >= 0.0, "pf_policy_loss: clip bounds must not be negative");
  PF_REQUIRE(loss && kl, "pf_policy_loss: null pointer");
  PF_REQUIRE(B * T == 0 || (T <= shift && !dlogits) || workspace, "pf_policy_loss: null workspace");
  PF_REQUIRE(B == 0 || T <= shift || (old_logprobs && advantages && logprobs), "pf_policy_loss: null pointer");
  PF_REQUIRE((stats != nullptr) == (coef != nullptr), "pf_policy_loss: stats and coef go together");
  hipStream_t s = (hipStream_t)stream;
  const TokenRows r = token_rows(logits, B, T, V, sb, st, labels, shift, ignore_index, temperature);
  const GradRows d = {dlogits, d_sb, d_st};
  const PolicyArgs a = {old_logprobs, ref_logprobs, advantages, a_sb, a_st, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
  const int64_t R = T > shift ? T - shift : 0;
  double* terms = workspace ? workspace + B : nullptr;
  if (B * T > 0 && (R > 0 || dlogits)) {
    if (R > 0) hipLaunchKernelGGL(token_weights_kernel, dim3(1), dim3(256), 0, s, r, by_sequence, workspace);
#define CALL(DT) \
  hipLaunchKernelGGL(policy_kernel<DT>, rows_grid(B * T), dim3(256), 0, s, r, d, a, workspace, logprobs, (float2*)stats, coef, terms)
    PF_BY_DTYPE(dtype, CALL);
#undef CALL
  }
  hipLaunchKernelGGL(sums_kernel, dim3(1), dim3(256), 0, s, terms, B * R, 1.0, loss, kl);
  PF_CHECK_LAUNCH("pf_policy_loss");
  return PF_OK;
}
