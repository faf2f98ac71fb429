// The gated projection's 16-bit products on the direct-to-LDS kernel: compiled once per operand type with
// -DPF_X_DT=<PF_F16|PF_BF16 value>.
//
// Forward: ONE product over both halves of the weight.  The right-hand tile holds as many rows of the gate's half as of the other
// (DTile's PAIR), dealt to the matrix instructions so that a lane's accumulators are the same columns of both: the activation and the
// product of the two happen in registers, and what is kept for the backward pass leaves from there, in the operands' type or
// as 8-bit codes.  Without that the two results make a trip through memory, 6 bytes an element of y.
//
// Bound by the matrix units, and by the epilogue, which the four-wavefront tile (one wavefront to a SIMD) cannot hide: 8192 x 2048 x 5632,
// silu, bf16: 309 us with both products kept, 0.378 TFLOP at 1.22 PFLOP/s, against 0.280 ms that the same tile's plain product would take at its
// 1.35; the activation by the library's exponential and division made that 332.  With 8-bit codes 16384 rows take 630 us (681 with the
// largest of a block by way of LDS and an exponent to a store).
#include "pf_gemm_x.h"
#include "pf_gated.h"

#if !defined(PF_X_DT)
#error "compile with -DPF_X_DT=<dtype id>"
#endif

namespace {

// N (1, 2 or 4) neighbouring 16-bit values
template <int N>
__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t rs, uint32_t at, const float (&v)[N]) {
  if constexpr (N == 1) {
    __builtin_amdgcn_raw_buffer_store_b16((short)(PF_X_DT == PF_BF16 ? pf_f32_to_bf16_bits(v[0]) : pf_f32_to_f16_bits(v[0])), rs, (int)at, 0, 0);
  } else {
    Words<N / 2> w;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) w.w[k] = (int)pack2<PF_X_DT>(v[2 * k], v[2 * k + 1]);
    w.store(rs, at);
  }
}
// N neighbouring values over `scale` as e4m3 codes
template <int N>
__device__ __forceinline__ void store8(__amdgpu_buffer_rsrc_t rs, uint32_t at, const float (&v)[N], float by) {
  if constexpr (N == 4) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * by, v[1] * by, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * by, v[3] * by, w, true);
    __builtin_amdgcn_raw_buffer_store_b32(w, rs, (int)at, 0, 0);
  } else {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * by, v[N - 1] * by, 0, false);
    if constexpr (N == 2) __builtin_amdgcn_raw_buffer_store_b16((short)w, rs, (int)at, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b8((char)w, rs, (int)at, 0, 0);
  }
}

// The largest of N neighbouring lanes' values (N = 4, 8 or 16), which share a data-parallel row: no trip through LDS
template <int N> __device__ __forceinline__ float largest(float v) {
  auto with = [&](auto c) {
    const int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(c)::value, 0xf, 0xf, true);
    v = fmaxf(v, __int_as_float(o));
  };
  with(std::integral_constant<int, 0xB1>{});                            // lanes 1 0 3 2
  with(std::integral_constant<int, 0x4E>{});                            // lanes 2 3 0 1
  if constexpr (N >= 8) with(std::integral_constant<int, 0x141>{});     // mirrored in 8
  if constexpr (N >= 16) with(std::integral_constant<int, 0x140>{});    // mirrored in 16
  return v;
}

template <int KEEP> struct GatedTail {
  static constexpr bool PAIR = true;
  uint16_t* y;
  int64_t ldy;
  void* kept;
  int64_t half;
  uint8_t* exps;
  int act, vec;
  template <int TM, int TN, bool AGPR>
  __device__ __forceinline__ void run(const float4_t (&acc)[TM][TN], int64_t row0, int64_t c0, int64_t M, int64_t N, int lane, int) const {
    constexpr int P = TN / 2;                       // columns of a lane
    constexpr int GROUP = PF_GATED_BLOCK / P;       // lanes that share an exponent
    constexpr int KS = KEEP == PF_KEEP_8BIT ? 1 : 2;
    constexpr uint32_t OOB = 0x80000000u;
    const __amdgpu_buffer_rsrc_t rs_y = make_rsrc(y, (uint32_t)(((M - 1) * ldy + N) * 2));
    const __amdgpu_buffer_rsrc_t rs_k = make_rsrc(KEEP ? kept : (void*)y, KEEP ? (uint32_t)(M * half * 2 * KS) : 0u);
    const __amdgpu_buffer_rsrc_t rs_e =
        make_rsrc(KEEP == PF_KEEP_8BIT ? (void*)exps : (void*)y, KEEP == PF_KEEP_8BIT ? (uint32_t)((M + 3) / 4 * (half / PF_GATED_BLOCK) * 8) : 0u);
    const bool in = c0 < half;                      // (of what is kept; with 8 bits whole groups of lanes)
    uint32_t at_y = c0 < N ? (uint32_t)((row0 * ldy + c0) * 2) : OOB;
    uint32_t at_k = in ? (uint32_t)((row0 * half * 2 + c0) * KS) : OOB;
    uint32_t at_e = in && lane % GROUP == 0 ? (uint32_t)(row0 * (half / PF_GATED_BLOCK) * 2 + c0 / PF_GATED_BLOCK * 4) : OOB;
    const uint32_t step_y = (uint32_t)(ldy * 2), step_k = (uint32_t)(half * 2 * KS), step_e = (uint32_t)(half / PF_GATED_BLOCK * 2);
#pragma nounroll
    for (int h = 0; h < TM; ++h) {
      float4_t x[TN];
      static_for<TM>([&](auto cc) {
        constexpr int c = decltype(cc)::value;
        if (h == c) acc_read<AGPR>(x, acc[c]);
      });
      if (c0 + P > N) {      // columns past the last: rows of the other half, or of nothing
#pragma unroll
        for (int k = 0; k < P; ++k)
          if (c0 + k >= N) x[k] = x[k + P] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
      float4_t v[P];
      auto gate = [&](auto fn) {
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[k][r] = fn(x[k][r]) * x[k + P][r];
      };
      switch (act) {
        case PF_ACT_SILU: gate([](float t) { return pf_silu_fast(t); }); break;
        case PF_ACT_GELU: gate([](float t) { return pf_gelu_erf(t); }); break;
        case PF_ACT_GELU_TANH: gate([](float t) { return pf_gelu_tanh(t); }); break;
        default: gate([](float t) { return t > 0.f ? t : (t != t ? t : 0.f); }); break;
      }
      uint32_t eg4 = 0, eu4 = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float o[P], g[P], u[P];
#pragma unroll
        for (int k = 0; k < P; ++k) { o[k] = v[k][r]; g[k] = x[k][r]; u[k] = x[k + P][r]; }
        if (vec) {
          store16<P>(rs_y, at_y + (uint32_t)r * step_y, o);
        } else {
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const float one[1] = {o[k]};
            store16<1>(rs_y, c0 + k < N ? at_y + (uint32_t)r * step_y + 2 * k : OOB, one);
          }
        }
        if constexpr (KEEP == PF_KEEP_SAME) {
          store16<P>(rs_k, at_k + (uint32_t)r * step_k, g);
          store16<P>(rs_k, at_k + (uint32_t)r * step_k + (uint32_t)half * 2, u);
        }
        if constexpr (KEEP == PF_KEEP_8BIT) {
          float tg = 0.f, tu = 0.f;
#pragma unroll
          for (int k = 0; k < P; ++k) { tg = fmaxf(tg, fabsf(g[k])); tu = fmaxf(tu, fabsf(u[k])); }
          const int eg = pf_e4m3_exponent(largest<GROUP>(tg)), eu = pf_e4m3_exponent(largest<GROUP>(tu));
          store8<P>(rs_k, at_k + (uint32_t)r * step_k, g, pf_pow2(254 - eg));
          store8<P>(rs_k, at_k + (uint32_t)r * step_k + (uint32_t)half, u, pf_pow2(254 - eu));
          eg4 |= (uint32_t)eg << (8 * r);
          eu4 |= (uint32_t)eu << (8 * r);
        }
      }
      if constexpr (KEEP == PF_KEEP_8BIT) {
        __builtin_amdgcn_raw_buffer_store_b32((int)eg4, rs_e, (int)at_e, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32((int)eu4, rs_e, (int)(at_e + (uint32_t)(half / PF_GATED_BLOCK * 4)), 0, 0);
      }
      at_y += 16 * step_y;
      at_k += 16 * step_k;
      at_e += 16 * step_e;
    }
  }
};

#define PF_T_TILE T::BM, T::BN, T::BK, T::WGM, T::WGN, T::KS, T::ST
#define PF_T_BOUNDS __launch_bounds__(64 * XTile<XT>::WGM * XTile<XT>::WGN, (XTile<XT>::BM == 64 ? 2 : 1))

template <int XT, bool RAG, int KEEP>
__global__ PF_T_BOUNDS void gated_forward_kernel(const pf_gemm_desc d, const GemmGrid g, const GatedTail<KEEP> tail) {
  using T = XTile<XT>;
  gemm16x_body<PF_X_DT, PF_T_TILE, false, false, EC_OWN, RAG, GatedTail<KEEP>>(d, g, (int)blockIdx.x, tail);
}
template <int XT, int EC>
__global__ PF_T_BOUNDS void gated_weight_kernel(const pf_gemm_desc d, const GemmGrid g) {
  using T = XTile<XT>;
  gemm16x_body<PF_X_DT, PF_T_TILE, true, true, EC>(d, g, (int)blockIdx.x);
}

template <int XT, class K, class... A>
int launch(K kern, int64_t M, int64_t N, int bn, hipStream_t st, const pf_gemm_desc& d, const A&... args) {
  using T = XTile<XT>;
  constexpr size_t lds = (size_t)T::ST * (T::BM + T::BN) * T::BK * 2 + (T::ST == 2 ? (size_t)T::BN * T::BK * 2 : 0);
  const int rc = pf_allow_lds((const void*)kern, lds, "pf_gated_linear");
  if (rc != PF_OK) return rc;
  GemmGrid g;
  g.tiles_m = (int)((M + T::BM - 1) / T::BM);
  g.tiles_n = (int)((N + bn - 1) / bn);
  g.per_xcd = (int)(((int64_t)g.tiles_m * g.tiles_n + 7) / 8);
  g.vec_epi = 1;
  hipLaunchKernelGGL(kern, dim3((unsigned)(g.per_xcd * 8), (unsigned)d.batch2), dim3(64 * T::WGM * T::WGN), lds, st, d, g, args...);
  PF_CHECK_LAUNCH("pf_gated_linear");
  return PF_OK;
}

template <int KEEP> int forward(const PfGatedProduct& p, hipStream_t st) {
  pf_gemm_desc d = {};
  d.in_dtype = d.c_dtype = PF_X_DT;
  d.M = p.rows; d.N = 2 * p.ffn; d.K = p.depth;
  d.A = p.x; d.lda = p.ldx; d.B = p.w; d.ldb = p.ldw; d.C = p.y; d.ldc = 2 * p.ffn;
  d.batch1 = d.batch2 = 1;
  d.alpha = 1.f;
  const int best = pf_gemm_best_tile(d);
  d.N = p.ffn;
  const GatedTail<KEEP> tail = {(uint16_t*)p.y, p.ldy, p.kept, p.half, p.exps, p.act, p.ldy % 8 == 0 && pf_aligned(p.y, 16)};
  // The plain product's choice, at most 4 % off the fastest of the four for 16 to 4096 rows of 1024, 2048 and 4096 columns.  (Where pf_gemm would take a
  // tile of 192 rows the next larger of its kind runs, or the four-wavefront one: three kernels an instantiation.)
  switch (best) {
    case PF_XT_64x64: return launch<PF_XT_64x64>(gated_forward_kernel<PF_XT_64x64, true, KEEP>, d.M, d.N, 32, st, d, tail);
    case PF_XT_128x128w8: return launch<PF_XT_128x128w8>(gated_forward_kernel<PF_XT_128x128w8, true, KEEP>, d.M, d.N, 64, st, d, tail);
    case PF_XT_192x128w8:
    case PF_XT_256x128w8: return launch<PF_XT_256x128w8>(gated_forward_kernel<PF_XT_256x128w8, true, KEEP>, d.M, d.N, 64, st, d, tail);
    default:
      if (p.depth % 64 != 0) return launch<PF_XT_256x128w8>(gated_forward_kernel<PF_XT_256x128w8, true, KEEP>, d.M, d.N, 64, st, d, tail);
      return launch<PF_XT_256x256w4>(gated_forward_kernel<PF_XT_256x256w4, false, KEEP>, d.M, d.N, 128, st, d, tail);
  }
}

}  // namespace

#define PF_T_CAT_(a, b) a##b
#define PF_T_CAT(a, b) PF_T_CAT_(a, b)

int PF_T_CAT(pf_gated_forward_, PF_X_DT)(const PfGatedProduct& p, hipStream_t st) {
  return p.keep == PF_KEEP_NONE ? forward<PF_KEEP_NONE>(p, st) : p.keep == PF_KEEP_SAME ? forward<PF_KEEP_SAME>(p, st) : forward<PF_KEEP_8BIT>(p, st);
}

// A weight gradient in the operands' type.  pf_gemm has straight-line code for fp32 results of such products only (it accumulates
// them); here the result is a tensor of its own, and 6 bytes an element less to move.  Where columns lie between the halves (ffn no multiple of
// 8) their products are one launch's two batches: 777 x 1000 x 2732, fp16: 33 us, one by one 2 x 19.5.
int PF_T_CAT(pf_gated_weight_, PF_X_DT)(int64_t M, int64_t N, int64_t K, const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int batch, int64_t step,
                                     hipStream_t st) {
  pf_gemm_desc d = {};
  d.in_dtype = PF_X_DT; d.c_dtype = PF_X_DT;
  d.a_trans = d.b_trans = 1;
  d.M = M; d.N = N; d.K = K;
  d.A = A; d.lda = lda; d.B = B; d.ldb = ldb; d.C = C; d.ldc = ldc;
  d.batch1 = 1; d.batch2 = batch;
  d.a_stride2 = step; d.c_stride2 = M * ldc;
  d.alpha = 1.f;
  const bool runs = epi_class(d, epi_vec_ok(d)) == EC_STORE16 && (M + 255) / 256 * 256 * ldc * 2 < (1ll << 31);
  const int64_t rows = runs && batch == 1 ? pf_gemm_strided_rows(d) : M;
  const int best = pf_gemm_best_tile(d);
  if (!runs || (rows == M && best != PF_XT_256x256w4)) return pf_gemm(&d, st);
  d.M = rows;
  const int rc = launch<PF_XT_256x256w4>(gated_weight_kernel<PF_XT_256x256w4, EC_STORE16>, rows, N, 256, st, d);
  if (rc != PF_OK || rows == M) return rc;
  d.M = M - rows;
  d.A = (const char*)A + rows * 2;
  d.C = (char*)C + rows * ldc * 2;
  return pf_gemm(&d, st);
}
