// The 16-bit matrix products of the cross entropy from the last hidden state, on the direct-to-LDS kernel: compiled once per
// operand type with -DPF_X_DT=<PF_F16|PF_BF16 value>.
//
// All of them look at the logits as z^T = W H^T, vocabulary rows by tokens, so that a lane of the matrix instruction keeps whole
// tokens: the softmax's maximum and sum run over a lane's own registers (two exchanges between lanes per token at the end
// instead of four per row and element), and the gradient dz^T leaves in runs of tokens, which is the layout that both products
// of the backward pass read: dW = dz^T H as row-major x row-major of H^T, dH = (dz^T)^T W with both operands stored along the
// reduction.  Nothing is transposed but H, the smallest of the three.
//
// All are bound by the matrix units.  8192 tokens, 2048 columns, 32000 classes, bf16 (1.07 TFLOP each over all of the vocabulary): the
// statistics 0.85 ms, 1.26 PFLOP/s; dz 0.84, 1.28; dh 0.76 and dW 0.71, 1.41 and 1.51 (a plain product of 8192 cubed: 1.35).  What the first two
// lack is their epilogue, which one wavefront to a SIMD does not hide.
//
// How many tokens take part is known to the device alone.  The grid covers all of them; the kernels read the number and leave
// the rest of the grid, so prompts and padding cost no arithmetic and the host does not wait.
#include "pf_gemm_x.h"
#include "pf_head.h"

#if !defined(PF_X_DT)
#error "compile with -DPF_X_DT=<dtype id>"
#endif

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.0e38f;     // (stands for "no logit yet": what is below it, -inf, adds nothing)

// one 16-row block's accumulators by a rolled loop's index (unrolled, the arithmetic's code would stream through a cold
// instruction cache)
template <bool AGPR, int TM, int TN>
__device__ __forceinline__ void block_of(float4_t (&x)[TN], const float4_t (&acc)[TM][TN], int h) {
  static_for<TM>([&](auto cc) {
    constexpr int c = decltype(cc)::value;
    if (h == c) acc_read<AGPR>(x, acc[c]);
  });
}

// Maximum and sum of exponentials of each token over this wavefront's vocabulary rows, in one pass over the accumulators
struct StatsTail {
  static constexpr bool PAIR = false;
  PfHeadPart* part;
  int64_t ldp;
  const int* lab;
  float* zl;
  int v0;
  template <int TM, int TN, bool AGPR>
  __device__ __forceinline__ void run(const float4_t (&acc)[TM][TN], int64_t row0, int64_t c0, int64_t M, int64_t N, int lane, int blk) const {
    float m[TN], s[TN];
    int rel[TN];       // the label's place counted from this lane's first row
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      m[j] = LOWEST;
      s[j] = 0.f;
      const int l = c0 < N ? lab[c0 + j] : -1;
      rel[j] = l >= 0 ? l - v0 - (int)row0 : -1;
    }
    const int left = (int)(M - row0);
#pragma nounroll
    for (int h = 0; h < TM; ++h) {
      float4_t x[TN];
      block_of<AGPR>(x, acc, h);
      if (16 * h + 3 >= left) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[j][r] = 16 * h + r < left ? x[j][r] : -INFINITY;
      }
      bool hit = false;
#pragma unroll
      for (int j = 0; j < TN; ++j) hit |= (unsigned)(rel[j] - 16 * h) < 4u;
      if (hit) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (rel[j] == 16 * h + r) zl[c0 + j] = x[j][r];
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float t = fmaxf(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])), m[j]);
        float a = s[j] * __builtin_amdgcn_exp2f((m[j] - t) * LOG2E);
#pragma unroll
        for (int r = 0; r < 4; ++r) a += __builtin_amdgcn_exp2f((x[j][r] - t) * LOG2E);
        s[j] = a;
        m[j] = t;
      }
    }
#pragma unroll
    for (int off = 16; off < 64; off <<= 1)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float om = __shfl_xor(m[j], off, 64), os = __shfl_xor(s[j], off, 64);
        const float t = fmaxf(m[j], om);
        s[j] = s[j] * __builtin_amdgcn_exp2f((m[j] - t) * LOG2E) + os * __builtin_amdgcn_exp2f((om - t) * LOG2E);
        m[j] = t;
      }
    if (lane < 16 && c0 < N) {
      PfHeadPart* out = part + (int64_t)blk * ldp + c0;
#pragma unroll
      for (int j = 0; j < TN; ++j) out[j] = {m[j], s[j]};
    }
  }
};

// dz = f p - g [row is the label], rounded to the operands' type: what both gradient products read
template <int DT> struct GradTail {
  static constexpr bool PAIR = false;
  const PfHeadColumn* col;
  const int* lab;
  uint16_t* dz;
  int64_t ldz;
  int v0;
  template <int TM, int TN, bool AGPR>
  __device__ __forceinline__ void run(const float4_t (&acc)[TM][TN], int64_t row0, int64_t c0, int64_t M, int64_t N, int lane, int) const {
    PfHeadColumn c[TN];
    int rel[TN];
    const bool in = c0 < N;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int l = in ? lab[c0 + j] : -1;
      rel[j] = l >= 0 ? l - v0 - (int)row0 : -1;
      c[j] = col[in ? c0 + j : 0];
    }
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(dz, (uint32_t)(((M - 1) * ldz + N) * 2));
    uint32_t at = in ? (uint32_t)((row0 * ldz + c0) * 2) : 0x80000000u;
    const uint32_t step = (uint32_t)(ldz * 2);
#pragma nounroll
    for (int h = 0; h < TM; ++h) {
      float4_t x[TN];
      block_of<AGPR>(x, acc, h);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j][r] = c[j].f * __builtin_amdgcn_exp2f(fmaf(x[j][r] - c[j].top, LOG2E, c[j].bias));
      bool hit = false;
#pragma unroll
      for (int j = 0; j < TN; ++j) hit |= (unsigned)(rel[j] - 16 * h) < 4u;
      if (hit) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (rel[j] == 16 * h + r) x[j][r] -= c[j].g;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        Words<TN / 2> o;
#pragma unroll
        for (int k = 0; k < TN / 2; ++k) o.w[k] = (int)pack2<DT>(x[2 * k][r], x[2 * k + 1][r]);
        o.store(rs, at + (uint32_t)r * step);
      }
      at += 16 * step;
    }
  }
};

__device__ __forceinline__ int padded_count(const int* count) { return *count > 64 ? (*count + 63) / 64 * 64 : 64; }

// the grid's share of a product with fewer tiles than it was launched for; false: none
template <int BM, int BN>
__device__ __forceinline__ bool shrink(const pf_gemm_desc& p, GemmGrid& g) {
  g.tiles_m = (int)((p.M + BM - 1) / BM);
  g.tiles_n = (int)((p.N + BN - 1) / BN);
  g.per_xcd = (g.tiles_m * g.tiles_n + 7) / 8;
  return (int)(blockIdx.x >> 3) < g.per_xcd;
}

#define PF_H_TILE T::BM, T::BN, T::BK, T::WGM, T::WGN, T::KS, T::ST
#define PF_H_BOUNDS __launch_bounds__(64 * XTile<XT>::WGM * XTile<XT>::WGN, (XTile<XT>::BM == 64 ? 2 : 1))

// z^T of one piece, its tokens counted on the device
template <int XT, bool RAG, class Tail>
__global__ PF_H_BOUNDS void head_logits_kernel(const pf_gemm_desc d, const int* count, const Tail tail) {
  using T = XTile<XT>;
  pf_gemm_desc p = d;
  GemmGrid g;
  p.N = padded_count(count);
  g.vec_epi = 1;
  if (!shrink<T::BM, T::BN>(p, g)) return;
  gemm16x_body<PF_X_DT, PF_H_TILE, false, false, EC_OWN, RAG, Tail>(p, g, (int)blockIdx.x, tail);
}
// The piece's `rows` in shares, the last one shorter
template <int XT, int EC>
__global__ PF_H_BOUNDS void head_hidden_grad_kernel(const pf_gemm_desc d, const int* count, int64_t rows, const PfHeadShares shares) {
  using T = XTile<XT>;
  pf_gemm_desc p = d;
  GemmGrid g;
  p.M = *count;
  const int64_t share = pf_head_share(rows, shares.of(p.M, p.N)), left = rows - (int64_t)blockIdx.y * share;
  if (left <= 0) return;
  p.K = left < share ? left : share;
  p.a_stride2 = share * p.lda;
  p.b_stride2 = share * p.ldb;
  p.c_stride2 = (shares.by_count ? p.M : d.M) * p.N;
  g.vec_epi = 1;
  if (p.M == 0 || !shrink<T::BM, T::BN>(p, g)) return;
  gemm16x_body<PF_X_DT, PF_H_TILE, true, true, EC>(p, g, (int)blockIdx.x);
}
template <int XT, int EC>
__global__ PF_H_BOUNDS void head_weight_grad_kernel(const pf_gemm_desc d, const GemmGrid g, const int* count) {
  using T = XTile<XT>;
  pf_gemm_desc p = d;
  p.K = padded_count(count);
  gemm16x_body<PF_X_DT, PF_H_TILE, false, false, EC>(p, g, (int)blockIdx.x);
}

template <int XT> constexpr size_t tile_lds() {
  using T = XTile<XT>;
  return (size_t)T::ST * (T::BM + T::BN) * T::BK * 2 + (T::ST == 2 ? (size_t)T::BN * T::BK * 2 : 0);
}
template <int XT, class K, class... A>
int launch(K kern, int64_t M, int64_t N, int batch, hipStream_t st, const A&... args) {
  using T = XTile<XT>;
  const int rc = pf_allow_lds((const void*)kern, tile_lds<XT>(), "pf_linear_ce");
  if (rc != PF_OK) return rc;
  const int64_t tiles = ((M + T::BM - 1) / T::BM) * ((N + T::BN - 1) / T::BN);
  hipLaunchKernelGGL(kern, dim3((unsigned)((tiles + 7) / 8 * 8), (unsigned)batch), dim3(64 * T::WGM * T::WGN), tile_lds<XT>(), st, args...);
  PF_CHECK_LAUNCH("pf_linear_ce");
  return PF_OK;
}

pf_gemm_desc plain_desc() {
  pf_gemm_desc d = {};
  d.in_dtype = PF_X_DT;
  d.batch1 = d.batch2 = 1;
  d.alpha = 1.f;
  return d;
}
pf_gemm_desc logits_desc(const PfHeadProduct& p) {
  pf_gemm_desc d = plain_desc();
  d.M = p.rows; d.N = p.n_max; d.K = p.depth;
  d.A = p.w; d.lda = p.ldw; d.B = p.hc; d.ldb = p.ldh;
  return d;
}
template <class Tail> int logits_launch(const PfHeadProduct& p, const Tail& tail, hipStream_t st) {
  const pf_gemm_desc d = logits_desc(p);
  static_assert(XTile<PF_XT_64x64>::BM / XTile<PF_XT_64x64>::WGM == 32 && XTile<PF_XT_256x128w8>::BM / XTile<PF_XT_256x128w8>::WGM == 64 &&
                XTile<PF_XT_256x256w4>::BM / XTile<PF_XT_256x256w4>::WGM == 128, "pf_head_blocks");
  switch (pf_head_tile(p.n_max, p.depth)) {
    case PF_HEAD_64x64: return launch<PF_XT_64x64>(head_logits_kernel<PF_XT_64x64, true, Tail>, p.rows, p.n_max, 1, st, d, p.count, tail);
    case PF_HEAD_256x128: return launch<PF_XT_256x128w8>(head_logits_kernel<PF_XT_256x128w8, true, Tail>, p.rows, p.n_max, 1, st, d, p.count, tail);
    default: return launch<PF_XT_256x256w4>(head_logits_kernel<PF_XT_256x256w4, false, Tail>, p.rows, p.n_max, 1, st, d, p.count, tail);
  }
}

template <int XT> int hidden_launch(const pf_gemm_desc& d, const PfHeadProduct& p, hipStream_t st) {
  return d.beta ? launch<XT>(head_hidden_grad_kernel<XT, EC_ACC32>, d.M, d.N, (int)d.batch2, st, d, p.count, p.rows, p.shares)
                : launch<XT>(head_hidden_grad_kernel<XT, EC_STORE32>, d.M, d.N, (int)d.batch2, st, d, p.count, p.rows, p.shares);
}
int hidden_grad(const pf_gemm_desc& d, const PfHeadProduct& p, hipStream_t st) {
  switch (p.shares.by_count ? PF_XT_256x256w4 : pf_gemm_best_tile(d)) {
    case PF_XT_64x64: return hidden_launch<PF_XT_64x64>(d, p, st);
    case PF_XT_128x128w8: return hidden_launch<PF_XT_128x128w8>(d, p, st);
    case PF_XT_256x128w8: return hidden_launch<PF_XT_256x128w8>(d, p, st);
    default: return hidden_launch<PF_XT_256x256w4>(d, p, st);
  }
}

}  // namespace

#define PF_H_CAT_(a, b) a##b
#define PF_H_CAT(a, b) PF_H_CAT_(a, b)

int PF_H_CAT(pf_head_stats_, PF_X_DT)(const PfHeadProduct& p, hipStream_t st) {
  return logits_launch(p, StatsTail{p.part, p.n_max, p.lab, p.zl, (int)p.v0}, st);
}

int PF_H_CAT(pf_head_dz_, PF_X_DT)(const PfHeadProduct& p, hipStream_t st) {
  return logits_launch(p, GradTail<PF_X_DT>{p.col, p.lab, (uint16_t*)p.dz, p.n_max, (int)p.v0}, st);
}

int PF_H_CAT(pf_head_dh_, PF_X_DT)(const PfHeadProduct& p, hipStream_t st) {
  pf_gemm_desc d = plain_desc();
  d.c_dtype = PF_F32;
  d.a_trans = d.b_trans = 1;
  d.M = p.n_max; d.N = p.depth; d.K = pf_head_share(p.rows, p.shares.most);
  d.A = p.dz; d.lda = p.n_max; d.B = p.w; d.ldb = p.ldw; d.C = p.dh; d.ldc = p.depth;
  d.beta = p.add;
  d.unscale_by = p.unscale;
  d.batch2 = p.shares.most;
  return hidden_grad(d, p, st);
}

int PF_H_CAT(pf_head_dw_, PF_X_DT)(const PfHeadProduct& p, hipStream_t st) {
  pf_gemm_desc d = plain_desc();
  d.c_dtype = PF_X_DT;
  d.M = p.rows; d.N = p.dim; d.K = p.n_max;
  d.A = p.dz; d.lda = p.n_max; d.B = p.ht; d.ldb = p.n_max; d.C = p.dw; d.ldc = p.ldw_out;
  d.unscale_by = p.unscale;
  // (one tile for all sizes, the widest runs of a row's stores: a step of the weight alone with 64 tokens, 2048 columns, 32000 classes, bf16 100 us, on 256x128
  // 104, 128x128 113, 64x64 137; with 2048 tokens 653, 682, 726, 838)
  using T = XTile<PF_XT_256x256w4>;
  GemmGrid g;
  g.tiles_m = (int)((d.M + T::BM - 1) / T::BM);
  g.tiles_n = (int)((d.N + T::BN - 1) / T::BN);
  g.per_xcd = (int)(((int64_t)g.tiles_m * g.tiles_n + 7) / 8);
  g.vec_epi = epi_vec_ok(d);
  return launch<PF_XT_256x256w4>(head_weight_grad_kernel<PF_XT_256x256w4, EC_STORE16>, d.M, d.N, 1, st, d, g, p.count);
}

#if PF_X_DT == 1
PfHeadShares pf_head_shares(int dtype, int64_t n_max, int64_t depth, int64_t rows) {
  PfHeadShares best = {1, 0, rows};
  int tile = 0;
  double best_t = 0;
  for (int s = 1; s <= 16 && (s == 1 || (rows / s >= 256 && n_max * depth * 4 * s < (1ll << 31) - 64)); ++s) {
    double t = 0;
    pf_gemm_desc d = plain_desc();
    d.c_dtype = PF_F32;
    d.a_trans = d.b_trans = 1;
    d.M = n_max; d.N = depth; d.K = pf_head_share(rows, s);
    d.batch2 = (rows + d.K - 1) / d.K;
    const int on = dtype == PF_F32 ? 0 : pf_gemm_best_tile(d, &t);
    if (dtype == PF_F32) t = pf_gemm_f32_depth_us(d);
    t += (double)(n_max * depth) * s * 8.0 / 5.0e6;      // the shares' way through memory, written and read at 5 TB/s
    if (s == 1 || t < best_t) { best.most = (int)d.batch2; best_t = t; tile = on; }
  }
  if (tile == PF_XT_256x256w4) {      // (half again as many as fill a round with all tokens: the workgroups that find nothing to do wait for a CU all the same)
    int64_t most = 384 / ((n_max + 255) / 256 * ((depth + 255) / 256));
    if (most > rows / 256) most = rows / 256;
    if (most > 16) most = 16;
    if (most > 1) best = {(int)most, 1, rows};
  }
  return best;
}
#endif
