// AdamW over many tensors at once with moments of 8 bits (or of 32 where a tensor is small).
//
//   m = m + (1 - beta1)(g - m),  v = beta2 v + (1 - beta2) g^2,
//   p = p (1 - lr wd) - step_size m / (sqrt(v) / sqrt(1 - beta2^t) + eps),       step_size = lr / (1 - beta1^t)
//
// in fp32, one rounding to an operation (no contraction: the results do not depend on what the compiler joins).  In 8 bits a moment is
// e4m3 codes with an fp32 scale to every 256 consecutive elements, the block's largest magnitude / 448: the codes then span 2^18.  The
// second moment is held as its root r = sqrt(v): half the range to cover, and the root is what the update divides by.
//
// Rounding.  beta2 = 0.999 changes v by 0.1 % a step, a sixtieth of half a code: rounded to nearest it would never decay.  A code is
// therefore rounded up with the probability of its distance from the lower neighbour, which keeps the mean; the random bits are a hash
// of element, tensor and step, so a step is the same from run to run, in any order of blocks.  A root that is not zero is never rounded to zero: a
// first moment that is rounded up meets a denominator of at least 2^-9 scale, not one of eps.  A block whose largest magnitude is below 2^-100 is
// held as zeros; one with an infinity or a NaN gets the scale NaN, so that it shows.
#include "pf_common.h"

#pragma clang fp contract(off)

namespace {

constexpr int BLOCK = 256;           // elements to a scale: a wavefront, four to a lane

// one row of the device table, eight 64-bit words
struct Adam8Item {
  float* param;
  const float* grad;
  void* m;               // e4m3 codes, or with m_scale == null fp32
  float* m_scale;
  void* r;               // e4m3 codes of sqrt(v), or fp32 v
  float* r_scale;
  int64_t n;
  int64_t tensor;        // which of the optimizer's tensors: a part of the rounding's random bits
};
static_assert(sizeof(Adam8Item) == 64, "eight words");

struct Adam8Coef {
  float keep, omb1, beta2, omb2, eps, step_size, bias_c2_sqrt, inv_bias;     // keep = 1 - lr wd
  uint32_t step;
};

// a / b, correctly rounded, from the rounded reciprocal y of b: a y is within an ulp, and its remainder, exact in an FMA, rounds it right (P. Markstein,
// 1990), while nothing underflows: a third of a division's instructions, for a b that many share.
__device__ __forceinline__ float divide_by(float a, float b, float y) {
  const float q = a * y;
  const float r = fmaf(fmaf(-q, b, a), y, q);
  return a < INFINITY ? r : a;
}

// 32 bits to 32 bits, one to one: shifts and products with odd constants, 0x9E3779B1 the prime next to 2^32 over the golden ratio (the
// multiplicative hash of D. Knuth), 0x93D765DD a multiplier of 32 bits from the tables of G. Steele and S. Vigna (2021)
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x93D765DDu;
  x = (x ^ (x >> 15)) * 0x9E3779B1u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ void update(const Adam8Coef& c, float& p, float g, float& m, float& v, float& root) {
  m = m + c.omb1 * (g - m);
  v = c.beta2 * v + c.omb2 * (g * g);
  root = sqrtf(v);
  p = p * c.keep - c.step_size * (m / (divide_by(root, c.bias_c2_sqrt, c.inv_bias) + c.eps));
}

// |x| inv = a in [0, 448] to an e4m3 value: a's lowest 20 bits of mantissa are rounded by `bits` (16 of them).  Below 2^-6, where codes are 2^-9
// apart, a + 2^-6 has just those 20 bits.
__device__ __forceinline__ float round_code(float x, float inv, uint32_t bits) {
  const float a = fabsf(x) * inv;
  const bool fine = a < 0.015625f;
  const float t = fine ? a + 0.015625f : a;
  const float q = __uint_as_float((__float_as_uint(t) + (bits << 4)) & 0xFFF00000u);
  return copysignf(fminf(fine ? q - 0.015625f : q, 448.f), x);
}

// Of both moments' largest magnitudes; `bad`: not all finite.  The four divisions are one, by lanes that differ in their operands.
struct BlockScale { float inv, scale; };
__device__ __forceinline__ void block_scales(float m_top, bool m_bad, float r_top, bool r_bad, BlockScale& m, BlockScale& r) {
  const float top = threadIdx.x & 2 ? r_top : m_top;
  const float q = __fdiv_rn(threadIdx.x & 1 ? top : 448.f, threadIdx.x & 1 ? 448.f : top);
  const auto lane = [&](int k) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q), k)); };
  m = m_bad ? BlockScale{0.f, NAN} : m_top >= 0x1p-100f ? BlockScale{lane(0), lane(1)} : BlockScale{0.f, 0.f};
  r = r_bad ? BlockScale{0.f, NAN} : r_top >= 0x1p-100f ? BlockScale{lane(2), lane(3)} : BlockScale{0.f, 0.f};
}

__device__ __forceinline__ uint32_t pack4(const float (&q)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}
__device__ __forceinline__ void unpack4(uint32_t w, float scale, float (&x)[4]) {
  x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
  x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
  x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
  x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
}

// Four values from element i on.  FULL: all of them are the tensor's; else those where i + k < n.  Everything is next used a step later and
// bypasses the caches.
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t word_any __attribute__((aligned(1)));
template <bool FULL> __device__ __forceinline__ void load4(const float* p, int64_t i, int64_t n, float (&x)[4]) {
  if constexpr (FULL) {
    const float4_any v = __builtin_nontemporal_load((const float4_any*)(p + i));
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k < n ? p[i + k] : 0.f;
  }
}
template <bool FULL> __device__ __forceinline__ void store4(float* p, int64_t i, int64_t n, const float (&x)[4]) {
  if constexpr (FULL) {
    const float4_any v = {x[0], x[1], x[2], x[3]};
    __builtin_nontemporal_store(v, (float4_any*)(p + i));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = x[k];
  }
}
template <bool FULL> __device__ __forceinline__ uint32_t load_codes(const void* p, int64_t i, int64_t n) {
  if constexpr (FULL) return __builtin_nontemporal_load((const word_any*)((const uint8_t*)p + i));
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) w |= (uint32_t)((const uint8_t*)p)[i + k] << (8 * k);
  return w;
}
template <bool FULL> __device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t n, uint32_t w) {
  if constexpr (FULL) {
    __builtin_nontemporal_store(w, (word_any*)((uint8_t*)p + i));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) ((uint8_t*)p)[i + k] = (uint8_t)(w >> (8 * k));
  }
}

// one block, by a wavefront
template <bool FULL> __device__ __forceinline__ void step_block(const Adam8Item& it, int64_t block, const Adam8Coef& c) {
  const int lane = threadIdx.x & 63;
  const int64_t i = block * BLOCK + lane * 4;
  float p[4], g[4], m[4], v[4], root[4];
  load4<FULL>(it.param, i, it.n, p);
  load4<FULL>(it.grad, i, it.n, g);
  if (it.m_scale == nullptr) {
    load4<FULL>((const float*)it.m, i, it.n, m);
    load4<FULL>((const float*)it.r, i, it.n, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) update(c, p[j], g[j], m[j], v[j], root[j]);
    store4<FULL>(it.param, i, it.n, p);
    store4<FULL>((float*)it.m, i, it.n, m);
    store4<FULL>((float*)it.r, i, it.n, v);
    return;
  }
  const uint32_t mw = load_codes<FULL>(it.m, i, it.n), rw = load_codes<FULL>(it.r, i, it.n);
  unpack4(mw, it.m_scale[block], m);
  unpack4(rw, it.r_scale[block], root);
  float m_top = 0.f, r_top = 0.f;
  bool m_bad = false, r_bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = root[j] * root[j];
    update(c, p[j], g[j], m[j], v[j], root[j]);
    if (!FULL && i + j >= it.n) m[j] = root[j] = 0.f;      // (not of the tensor: a NaN scale would show there too)
    m_top = fmaxf(m_top, fabsf(m[j]));
    r_top = fmaxf(r_top, root[j]);
    m_bad |= !(fabsf(m[j]) < INFINITY);
    r_bad |= !(root[j] < INFINITY);
  }
  store4<FULL>(it.param, i, it.n, p);
  BlockScale ms, rs;
  block_scales(pf_wave_max(m_top), __any(m_bad), pf_wave_max(r_top), __any(r_bad), ms, rs);
  const uint32_t key = mix(mix((uint32_t)block + (uint32_t)it.tensor * 0x9E3779B1u) + c.step * 0x93D765DDu);
  float mq[4], rq[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t bits = mix(key + (uint32_t)(lane * 4 + j) * 0x9E3779B1u);
    mq[j] = round_code(m[j], ms.inv, bits >> 16);
    rq[j] = round_code(root[j], rs.inv, bits & 0xFFFFu);
    if (root[j] > 0.f && rs.inv > 0.f) rq[j] = fmaxf(rq[j], 0x1p-9f);
  }
  store_codes<FULL>(it.m, i, it.n, pack4(mq));
  store_codes<FULL>(it.r, i, it.n, pack4(rq));
  if (lane == 0) {
    it.m_scale[block] = ms.scale;
    it.r_scale[block] = rs.scale;
  }
}

// A workgroup of four wavefronts to every 1024 elements, a wavefront to a block: 16 bytes a lane of parameters and gradients, one word of each
// code, the block's maximum by lane exchanges.  Bound by memory, 16.06 bytes a parameter: 117 M parameters in eight tensors 368 us, 5.1 TB/s (the
// 32-bit step moves 28); 1.8 M in four 10.  Some 80 instructions an element (square root and quotient correctly rounded, the hash) keep the
// arithmetic units busy two thirds of that time.
__global__ __launch_bounds__(256) void adam8_kernel(const Adam8Item* items, const int64_t* ends, int64_t first, int n_items, Adam8Coef c,
                                                    const float* scaler_state) {
  if (scaler_state) {
    if (scaler_state[2] != 0.f) return;
    c.step_size = scaler_state[4];
    c.bias_c2_sqrt = scaler_state[5];
    c.inv_bias = __fdiv_rn(1.f, scaler_state[5]);
    c.step = (uint32_t)scaler_state[3] + 1u;
  }
  const int64_t chunk = first + blockIdx.x;
  const int k = pf_find_item(ends, n_items, chunk);
  const Adam8Item it = items[k];
  const int64_t block = (chunk - (k > 0 ? ends[k - 1] : 0)) * (PF_ADAM_CHUNK / BLOCK) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((block + 1) * BLOCK <= it.n) step_block<true>(it, block, c);
  else if (block * BLOCK < it.n) step_block<false>(it, block, c);
}

}  // namespace

extern "C" int pf_adam8_step(const int64_t* items_dev, const int64_t* chunk_ends_dev, int n_items, int64_t n_chunks, double lr, double beta1,
                             double beta2, double eps, double weight_decay, int64_t step, float* scaler_state, void* stream) {
  PF_REQUIRE(n_items >= 0 && n_chunks >= 0 && (scaler_state != nullptr || step >= 1), "pf_adam8_step: bad arguments");
  if (n_items == 0 || n_chunks == 0) return PF_OK;
  PF_REQUIRE(items_dev != nullptr && chunk_ends_dev != nullptr, "pf_adam8_step: bad item list");
  if (scaler_state != nullptr) pf_adam_coefficients(scaler_state, lr, beta1, beta2, stream);
  const double t = scaler_state != nullptr ? 1.0 : (double)step;
  const float bias = (float)sqrt(1.0 - pow(beta2, t));
  const Adam8Coef c = {(float)(1.0 - lr * weight_decay), (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps,
                       (float)(lr / (1.0 - pow(beta1, t))), bias, 1.f / bias, (uint32_t)step};
  constexpr int64_t most = 1 << 23;      // (a launch has less than 2^32 threads)
  for (int64_t first = 0; first < n_chunks; first += most)
    hipLaunchKernelGGL(adam8_kernel, dim3((unsigned)(n_chunks - first < most ? n_chunks - first : most)), dim3(256), 0, (hipStream_t)stream,
                       (const Adam8Item*)items_dev, chunk_ends_dev, first, n_items, c, scaler_state);
  PF_CHECK_LAUNCH("pf_adam8_step");
  return PF_OK;
}
