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
  float c;                // log2(e) / temperature
  double c_off;           // what its rounding added to it, relative
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

// ---- a row's sum of exponentials --------------------------------------------------------------------------------------------
// A row is read once, 16 bytes to a lane and access, NV accesses of a lane in flight; the row stays in the registers that it was loaded to, so that a gradient of the same pass is formed from there.  Each lane sums 2^(x c - ref) against a
// reference of its own, the whole number from its largest x c on: no exchange between lanes before the end, and one FMA and one exponential
// to an element.  Sums of eight go into a double.  What such arithmetic cannot do (a row of nothing but the lowest values, where
// x c overflows, infinities, NaN, x c past 2^29, where a whole number near it is no longer within 32 of it) shows as a sum outside
// (2^-32, 2^60), and is done again as (x - m) c.  (Below 2^24 the largest element's term lies between 1/4 and 2; there are 2^28 classes at most.)
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
typedef uint32_t raw4_any __attribute__((ext_vector_type(4), aligned(2)));      // (the memory unit takes any alignment)

template <int DT> constexpr int VE = DT == PF_F32 ? 4 : 8;       // elements of 16 bytes

template <int DT>
__device__ __forceinline__ void unpack(const raw4& w, float (&x)[VE<DT>]) {
  if constexpr (DT == PF_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == PF_BF16) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        x[2 * k] = pf_f16_bits_to_f32((uint16_t)(w[k] & 0xffffu));
        x[2 * k + 1] = pf_f16_bits_to_f32((uint16_t)(w[k] >> 16));
      }
    }
  }
}
template <int DT>
__device__ __forceinline__ raw4 pack(const float (&x)[VE<DT>]) {
  raw4 w;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == PF_F32) w[k] = __float_as_uint(x[k]);
    else if constexpr (DT == PF_BF16) w[k] = pf_pack2_bf16(x[2 * k], x[2 * k + 1]);
    else w[k] = pf_pack2_f16(x[2 * k], x[2 * k + 1]);
  }
  return w;
}
constexpr float NOTHING = -1e30f;      // the reference of a lane that has seen nothing

// the largest of three, NaN aside (one instruction: fmaxf would first quieten each operand)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
// the largest of a vector's elements and `top`
template <int DT>
__device__ __forceinline__ float max_of(const raw4& w, float top) {
  if constexpr (DT == PF_F32) {
    return max3(max3(top, __uint_as_float(w[0]), __uint_as_float(w[1])), __uint_as_float(w[2]), __uint_as_float(w[3]));
  } else if constexpr (DT == PF_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max3(top, __uint_as_float(w[k] & 0xffff0000u), __uint_as_float(w[k] << 16));
    return top;
  } else {
    uint32_t m, n;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(w[0]), "v"(w[1]));
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(n) : "v"(w[2]), "v"(w[3]));
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(m), "v"(n));
    return max3(top, pf_f16_bits_to_f32((uint16_t)(m & 0xffffu)), pf_f16_bits_to_f32((uint16_t)(m >> 16)));
  }
}

// Sum of 2^(x c - ref), ref a whole number, so that sums of different references meet without a rounding.  With FIRST also that of
// x 2^(x c - ref): what c's rounding does to the sum is some 1e-8 times the mean of x, of one sign in every row, and a sum over the tokens
// of a sequence shows it.
template <bool FIRST> struct Sums {
  float ref = NOTHING;
  double s = 0.0, s1 = 0.0;
  __device__ __forceinline__ void raise(float top) {      // the reference to the whole number from top on, if that is more
    top = ceilf(top);
    const float to = max3(ref, top, top);
    const int by = (int)(ref - to);
    s = ldexp(s, by);
    if (FIRST) s1 = ldexp(s1, by);
    ref = to;
  }
  template <int N> __device__ __forceinline__ void add(const float (&x)[N], float c, bool valid) {
    float e[N], f = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      e[k] = __builtin_amdgcn_exp2f(fmaf(x[k], c, -ref));
      if (FIRST) f = fmaf(e[k], x[k], f);
    }
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
      for (int k = 0; k < d; ++k) e[k] += e[k + d];
    s += (double)(valid ? e[0] : 0.f);
    if (FIRST) s1 += (double)(valid && f == f ? f : 0.f);      // (0 times -inf: a masked class among the eight leaves them out of the mean)
  }
  __device__ __forceinline__ void join(float other, double os, double os1) {
    const float to = max3(ref, other, other);
    const int a = (int)(ref - to), b = (int)(other - to);
    s = ldexp(s, a) + ldexp(os, b);
    if (FIRST) s1 = ldexp(s1, a) + ldexp(os1, b);
    ref = to;
  }
  __device__ __forceinline__ void join_lanes(int width) {
    for (int o = width / 2; o > 0; o >>= 1) {
      const float other = __shfl_xor(ref, o, 64);
      const double os = __shfl_xor(s, o, 64), os1 = FIRST ? __shfl_xor(s1, o, 64) : 0.0;
      join(other, os, os1);
    }
  }
};

// The whole row's: by one wavefront, or by the workgroup (`sm`: a slot to each wavefront).
template <bool FIRST> struct SumSlots { float ref[16]; double s[16], s1[16]; };
template <bool ONE, bool FIRST>
__device__ __forceinline__ void join_row(Sums<FIRST>& a, SumSlots<FIRST>* sm) {
  a.join_lanes(64);
  if constexpr (!ONE) {
    const int waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    if (waves == 1) return;
    __syncthreads();
    if (lane == 0) {
      sm->ref[threadIdx.x >> 6] = a.ref;
      sm->s[threadIdx.x >> 6] = a.s;
      if (FIRST) sm->s1[threadIdx.x >> 6] = a.s1;
    }
    __syncthreads();
    const int at = lane & 15;            // (lanes 16 apart hold the same)
    const bool in = at < waves;
    a.ref = in ? sm->ref[at] : NOTHING;
    a.s = in ? sm->s[at] : 0.0;
    if (FIRST) a.s1 = in ? sm->s1[at] : 0.0;
    a.join_lanes(16);
  }
}

// What follows from a row's sums.  slow: p = 2^((x - ref) c) inv, else 2^(x c - ref) inv
struct RowStats { float ref, inv; bool slow; double logprob; };
__device__ __forceinline__ float2 pack_stats(const RowStats& s) { return make_float2(s.ref, s.slow ? -s.inv : s.inv); }

// The row by (x - m) c, an element at a time; -> its sum
template <int DT, bool ONE>
__device__ double slow_sums(const char* x, int V, float c, float* m_out, double* shared) {
  const int tid = ONE ? (threadIdx.x & 63) : threadIdx.x, n = ONE ? 64 : blockDim.x, waves = ONE ? 1 : blockDim.x >> 6;
  float m = -INFINITY;
  for (int j = tid; j < V; j += n) m = fmaxf(m, Codec<DT>::load(x, j));
  m = pf_wave_max(m);
  if (waves > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = (double)m;
    __syncthreads();
    for (int w = 0; w < waves; ++w) m = fmaxf(m, (float)shared[w]);
  }
  double z = 0.0;
  for (int j = tid; j < V; j += n) z += (double)exp2f((Codec<DT>::load(x, j) - m) * c);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
  if (waves > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = z;
    __syncthreads();
    z = 0.0;
    for (int w = 0; w < waves; ++w) z += shared[w];
  }
  *m_out = m;
  return z;
}

template <int DT> constexpr int pf_es = DT == PF_F32 ? 4 : 2;

// A row in vectors of 16 bytes from the first address of `where` (the row itself, or its gradient) that is a multiple of 16 on: `head` elements
// stand before them and less than a vector's behind them, those of both ends a lane each.
template <int DT> struct Split {
  int head, full, loose;      // elements before the vectors, vectors, elements at both ends
  __device__ __forceinline__ Split(const char* where, int V) {
    head = (int)((16u - ((uint32_t)(uintptr_t)where & 15u)) & 15u) / pf_es<DT>;
    if (head > V) head = V;
    full = (V - head) / VE<DT>;
    loose = V - full * VE<DT>;
  }
  __device__ __forceinline__ int element(int lane) const { return lane < head ? lane : full * VE<DT> + lane; }      // (lane < loose)
  __device__ __forceinline__ size_t start() const { return (size_t)head * pf_es<DT>; }
};

// LOOP: the row takes several tiles of NV vectors to a lane; else one (rows of no vector at all have none).
template <int DT, int NV, bool ONE, bool LOOP> struct RowReader {
  const char* x;       // the row
  Split<DT> cut;
  int full;            // its vectors
  int tid, n;          // this lane among those of the row
  raw4 v[NV];
  float last;          // the loose element that this lane has (tid < cut.loose)

  __device__ __forceinline__ RowReader(const char* row, const char* where, int V)
      : x(row), cut(where, V), full(cut.full), tid(ONE ? (threadIdx.x & 63) : threadIdx.x), n(ONE ? 64 : blockDim.x) {}

  __device__ __forceinline__ int tiles() const { return full == 0 ? 0 : LOOP ? (full + n * NV - 1) / (n * NV) : 1; }
  __device__ __forceinline__ void load_loose() {
    last = -INFINITY;
    if (tid < cut.loose) last = Codec<DT>::load(x, cut.element(tid));
  }
  // lanes that have an i-th vector of a tile: those below this (uniform)
  __device__ __forceinline__ int left(int tile, int i) const { return full - (tile * NV + i) * n; }
  __device__ __forceinline__ void load(int tile) {
    const char* from = x + cut.start();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      int k = (tile * NV + i) * n + tid;
      if (k > full - 1) k = full - 1;
      v[i] = *(const raw4_any*)(from + (uint32_t)k * 16u);
    }
  }
  template <bool FIRST> __device__ __forceinline__ void sum(int tile, float c, Sums<FIRST>& a) {
    float top = NOTHING;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max_of<DT>(v[i], top);
    a.raise(top * c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      asm("" : "+v"(v[i]));      // (what the maximum unpacked is not worth keeping)
      float e[VE<DT>];
      unpack<DT>(v[i], e);
      a.add(e, c, tid < left(tile, i));      // (lanes past the end hold the last vector again)
    }
  }
  template <bool FIRST> __device__ __forceinline__ void sum_loose(float c, Sums<FIRST>& a) {
    if (cut.loose == 0) return;
    float e[1] = {last};
    a.raise(last * c);
    a.add(e, c, tid < cut.loose);
  }
};

template <int DT> __device__ __forceinline__ float element(const char* x, int j) { return Codec<DT>::load(x, j); }

// Statistics of a row whose label counts; the logprob where `lane_wants` (all lanes for the policy, one otherwise).
template <bool FIRST, int DT, int NV, bool ONE, bool LOOP>
__device__ __forceinline__ RowStats row_stats(const TokenRows& r, RowReader<DT, NV, ONE, LOOP>& row, float xy, SumSlots<FIRST>* sm, bool lane_wants) {
  Sums<FIRST> a;
  row.load_loose();
  const int tiles = row.tiles();
  for (int tile = 0; tile < tiles; ++tile) {
    row.load(tile);
    row.sum(tile, r.c, a);
  }
  row.sum_loose(r.c, a);
  join_row<ONE, FIRST>(a, sm);
  RowStats o = {a.ref, 0.f, !(a.s > 0x1p-32 && a.s < 0x1p60), 0.0};      // (1 / s times a small gradient is then no subnormal number)
  if (o.slow) {
    a.s = slow_sums<DT, ONE>(row.x, (int)r.V, r.c, &o.ref, sm ? sm->s : nullptr);
    o.logprob = ((double)xy - (double)o.ref) * r.inv_temp - log(a.s);
  } else if (lane_wants) {
    if (FIRST)   // ln sum exp(x / temperature) = ln sum 2^(x c) - c's relative error times the mean of x / temperature
      o.logprob = (double)xy * r.inv_temp - ((double)a.ref * 0.693147180559945309 + log(a.s) - r.c_off * r.inv_temp * (a.s1 / a.s));
    else
      o.logprob = ((double)xy * (double)r.c - (double)a.ref) * 0.693147180559945309 - log(a.s);
  }
  o.inv = (float)(1.0 / a.s);
  return o;
}

// PAST: past the caches
template <bool PAST> __device__ __forceinline__ void store_vector(char* dx, const raw4& w) {
  if (PAST) __builtin_nontemporal_store(w, (raw4_any*)dx);
  else *(raw4_any*)dx = w;
}

// What a lane needs for dx = g (onehot - p) / temperature = scaled 2^(..), scaled = -g inv / temperature; and the whole of it at the label
struct RowGrad { float scaled, at_label; };
template <bool SLOW> __device__ __forceinline__ float power(float x, const RowStats& s, float c) {
  return __builtin_amdgcn_exp2f(SLOW ? (x - s.ref) * c : fmaf(x, c, -s.ref));
}
__device__ __forceinline__ RowGrad row_grad(const TokenRows& r, const RowStats& s, float g, float xy) {
  g *= (float)r.inv_temp;
  const float scaled = -g * s.inv;
  return {scaled, fmaf(scaled, s.slow ? power<true>(xy, s, r.c) : power<false>(xy, s, r.c), g)};
}
// of the vector at dx; label: whose element in it, else negative or VE and more
template <int DT, bool SLOW, bool PAST>
__device__ __forceinline__ void gradient_vector(raw4 w, int label, const RowStats& s, const RowGrad& g, float c, char* dx) {
  asm volatile("" : "+v"(w));      // (unpacked here and not before: a tile's elements would not fit the registers)
  float x[VE<DT>];
  unpack<DT>(w, x);
#pragma unroll
  for (int e = 0; e < VE<DT>; ++e) x[e] = g.scaled * power<SLOW>(x[e], s, c);
  if ((unsigned)label < (unsigned)VE<DT>) {
    asm volatile("" : "+v"(label));      // (compared here and not ahead for every vector of a tile)
#pragma unroll
    for (int e = 0; e < VE<DT>; ++e) x[e] = e == label ? g.at_label : x[e];
  }
  store_vector<PAST>(dx, pack<DT>(x));
}
template <int DT>
__device__ __forceinline__ void gradient_element(float x, int j, int y, const RowStats& s, const RowGrad& g, float c, char* dx) {
  Codec<DT>::store(dx, j, j == y ? g.at_label : g.scaled * (s.slow ? power<true>(x, s, c) : power<false>(x, s, c)));
}

template <int DT, bool PAST>
__device__ __forceinline__ void fill_row(char* dx, int V, float value, int tid, int n) {
  float x[VE<DT>];
#pragma unroll
  for (int e = 0; e < VE<DT>; ++e) x[e] = value;
  const raw4 w = pack<DT>(x);
  const Split<DT> cut(dx, V);
  for (int k = tid; k < cut.full; k += n) store_vector<PAST>(dx + cut.start() + (uint32_t)k * 16u, w);
  if (tid < cut.loose) Codec<DT>::store(dx, cut.element(tid), value);
}

// The place of a workgroup's row in its sequence or, with ONE, of a wavefront's (four to a workgroup), uniform; the sequence is b0 + blockIdx.y
template <bool ONE> __device__ __forceinline__ int row_of_group(int t0) {
  return t0 + (ONE ? (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)blockIdx.x);
}

// stats[row] = {reference, 1 / sum}; for rows that take no part {0, 0}.  Bound by memory: 5371 of 8 x 1021 rows of 32000 classes in bf16 58 us,
// 5.9 TB/s; 8192 x 32000 in fp32 165, 6.4, in fp16 93, 5.6.  One row takes 5 us, a chain of a label's, a row's and a sum's latencies, which few
// rows do not hide: fp32 of 10007 classes 10.2 us for 855 rows (3.3 TB/s, three rows to a CU), 16 for 1710 (4.2), 57 for 8192 (5.7).
template <int DT, int NV, bool ONE, bool LOOP, typename Out>
__global__ __launch_bounds__(ONE ? 256 : 1024) void token_logprob_kernel(const TokenRows r, int b0, int t0, Out* logprobs, float2* stats) {
  constexpr bool FIRST = sizeof(Out) == 8;
  __shared__ SumSlots<FIRST> slots[1];
  const int R = (int)r.T - r.shift, t = row_of_group<ONE>(t0);
  const int64_t b = b0 + (int)blockIdx.y;
  if (t >= R) return;
  const int64_t y = r.labels[b * r.T + t + r.shift], at = b * R + t;
  const LabelKind kind = label_kind(r, y);
  RowStats s = {0.f, kind == LABEL_BAD ? NAN : 0.f, false, kind == LABEL_BAD ? (double)NAN : 0.0};
  const int tid = ONE ? threadIdx.x & 63 : threadIdx.x;
  if (kind == LABEL_OK) {
    const char* x = (const char*)r.logits + (b * r.sb + t * r.st) * pf_es<DT>;
    RowReader<DT, NV, ONE, LOOP> row(x, x, (int)r.V);
    s = row_stats<FIRST>(r, row, element<DT>(row.x, (int)y), slots, tid == 0);
  }
  if (tid == 0) {
    logprobs[at] = (Out)s.logprob;
    if (stats) stats[at] = pack_stats(s);
  }
}

// dlogits from the rows' statistics and g = coef[b * g_sb + t * g_st] (* scale[0]).  unless_one: nothing is done where scale[0] is one.
// A wavefront to 64 * GNV vectors of a row, without a word to others.  Rows are taken from the last one back: what the forward pass read
// last is what the caches may still hold.  Bound by memory: [4, 2048] x 32000 in bf16, 4745 rows of it scored, 828 MB (by the counters 306 read and
// 524 written past L2, so nothing twice) in 123 us, 6.7 TB/s; writing alone reaches 6.9, a copy 5.2.
constexpr int GNV = 4;
template <int DT, bool PAST>
__global__ __launch_bounds__(256) void token_gradient_kernel(const TokenRows r, const GradRows d, const float2* stats, const float* coef,
                                                             int64_t g_sb, int64_t g_st, const float* scale, int unless_one, unsigned pieces) {
  const float by = scale ? scale[0] : 1.f;
  if (unless_one && by == 1.f) return;
  const int64_t R = r.T - r.shift, units = r.T * pieces;
  const int lane = threadIdx.x & 63;
  for (int64_t b = r.B - 1 - (int64_t)blockIdx.y; b >= 0; b -= gridDim.y) {
    for (int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units; u += (int64_t)gridDim.x * 4) {
      const int64_t t = r.T - 1 - u / pieces;
      const int piece = (int)(u % pieces);
      char* dx = (char*)d.dx + (b * d.sb + t * d.st) * pf_es<DT>;
      const Split<DT> cut(dx, (int)r.V);
      const int first = piece * 64 * GNV + lane;      // this lane's vectors: this one and every 64th from it on
      const bool loose = piece == 0 && lane < cut.loose;
      const int64_t y = t < R ? r.labels[b * r.T + t + r.shift] : 0;
      const LabelKind kind = t < R ? label_kind(r, y) : LABEL_SKIP;
      char* to = dx + cut.start() + (uint32_t)first * 16u;
      if (kind == LABEL_SKIP) {
#pragma unroll
        for (int i = 0; i < GNV; ++i)
          if (first + i * 64 < cut.full) store_vector<PAST>(to + i * 1024, raw4{0, 0, 0, 0});
        if (loose) Codec<DT>::store(dx, cut.element(lane), 0.f);
        continue;
      }
      const char* x = (const char*)r.logits + (b * r.sb + t * r.st) * pf_es<DT>;
      const int yi = kind == LABEL_OK ? (int)y : -1;      // (no vector's and no element's)
      raw4 v[GNV];
      if (cut.full > 0) {
#pragma unroll
        for (int i = 0; i < GNV; ++i) {
          const int k = first + i * 64;
          v[i] = *(const raw4_any*)(x + cut.start() + (uint32_t)(k < cut.full ? k : cut.full - 1) * 16u);
        }
      }
      const float2 packed = stats[b * R + t];
      const RowStats s = {packed.x, fabsf(packed.y), packed.y < 0.f, 0.0};
      const RowGrad g = row_grad(r, s, coef[b * g_sb + t * g_st] * by, kind == LABEL_OK ? element<DT>(x, yi) : NAN);
      const int label = yi < cut.head ? -1 : yi - cut.head - first * VE<DT>;
      if (s.slow) {
#pragma unroll
        for (int i = 0; i < GNV; ++i)
          if (first + i * 64 < cut.full) gradient_vector<DT, true, PAST>(v[i], label - i * 64 * VE<DT>, s, g, r.c, to + i * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < GNV; ++i)
          if (first + i * 64 < cut.full) gradient_vector<DT, false, PAST>(v[i], label - i * 64 * VE<DT>, s, g, r.c, to + i * 1024);
      }
      if (loose) gradient_element<DT>(element<DT>(x, cut.element(lane)), cut.element(lane), yi, s, g, r.c, dx);
    }
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// sum of f(i) for i = first, first + n, ... below `end`, eight of them requested at a time
template <typename F> __device__ __forceinline__ double sum_in_eights(int64_t first, int64_t end, int64_t n, F f) {
  double s = 0.0;
  for (int64_t i = first; i < end; i += 8 * n) {
    double x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = f(i + j * n < end ? i + j * n : end - 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += i + j * n < end ? x[j] : 0.0;
  }
  return s;
}

// ---- preference ------------------------------------------------------------------------------------------------------------
// A workgroup to a pair, half of it to a sequence (2i, 2i + 1):  reward = beta (sum or mean of logprobs - ref),  D = reward_2i - reward_2i+1,
//   loss_i = -(1 - e) ln sigma(D) - e ln sigma(-D),   d loss_i / dD = e sigma(D) - (1 - e) sigma(-D)
// (= sigma(D) - (1 - e), which would cancel for a pair far apart).
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }   // -ln sigma(-x)

struct PairArgs {
  const double* logprobs;
  const int64_t* labels;
  int64_t T;
  int shift;
  int64_t ignore_index;
  const float* ref;
  double beta, smoothing;
  int average;
  int64_t pairs;
  float* rewards;
  float* coef;
};
// sum of the logprobs of sequence b's tokens and, for an average, how many count: this lane's part, lane of n
__device__ __forceinline__ void sequence_part(const PairArgs& a, int64_t b, int lane, int n, double& s, double& count) {
  const int64_t R = a.T - a.shift;
  s = sum_in_eights(lane, R, n, [&](int64_t t) { return a.logprobs[b * R + t]; });
  count = a.average ? sum_in_eights(lane, R, n, [&](int64_t t) { return a.labels[b * a.T + t + a.shift] != a.ignore_index ? 1.0 : 0.0; }) : 0.0;
}
// -> the pair's loss
__device__ double pair_terms(const PairArgs& a, int64_t i, const double (&total)[2], const double (&count)[2]) {
  double reward[2], per_token[2];
  for (int k = 0; k < 2; ++k) {
    per_token[k] = !a.average ? 1.0 : count[k] > 0.0 ? 1.0 / count[k] : 0.0;
    reward[k] = a.beta * (total[k] * per_token[k] - (double)a.ref[2 * i + k]);
  }
  const double D = reward[0] - reward[1], t = exp(-fabs(D)), most = 1.0 / (1.0 + t), least = t / (1.0 + t);      // sigma(|D|), sigma(-|D|)
  const double up = a.smoothing * (D >= 0.0 ? most : least) - (1.0 - a.smoothing) * (D >= 0.0 ? least : most);
  for (int k = 0; k < 2; ++k) {
    a.rewards[2 * i + k] = (float)reward[k];
    a.coef[2 * i + k] = (float)((k ? -up : up) * a.beta * per_token[k] / (double)a.pairs);
  }
  double loss = 0.0;      // (a term of factor zero is none, where the other answer has a token of no probability too)
  if (a.smoothing < 1.0) loss += (1.0 - a.smoothing) * softplus(-D);
  if (a.smoothing > 0.0) loss += a.smoothing * softplus(D);
  return loss;
}

__global__ __launch_bounds__(512) void preference_pair_kernel(const PairArgs a, double* pair_loss) {
  __shared__ double sums[8], counts[8];
  const int wave = threadIdx.x >> 6;
  for (int64_t i = blockIdx.x; i < a.pairs; i += gridDim.x) {
    double s, n;
    sequence_part(a, 2 * i + (threadIdx.x >> 8), threadIdx.x & 255, 256, s, n);
    s = wave_sum(s);
    n = wave_sum(n);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      sums[wave] = s;
      counts[wave] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      double total[2], count[2];
      for (int k = 0; k < 2; ++k) {
        total[k] = sums[4 * k] + sums[4 * k + 1] + sums[4 * k + 2] + sums[4 * k + 3];
        count[k] = counts[4 * k] + counts[4 * k + 1] + counts[4 * k + 2] + counts[4 * k + 3];
      }
      pair_loss[i] = pair_terms(a, i, total, count);
    }
  }
}

// All pairs by one workgroup, and their mean: the wavefronts share the sequences, a lane each takes a pair.
constexpr int FEW_SEQUENCES = 32;
__global__ __launch_bounds__(1024) void preference_few_kernel(const PairArgs a, float* loss) {
  __shared__ double sums[FEW_SEQUENCES][16], counts[FEW_SEQUENCES][16];
  const int B = 2 * (int)a.pairs, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int share = B <= 2 ? 8 : B <= 4 ? 4 : B <= 8 ? 2 : 1;      // wavefronts to a sequence
  for (int b = wave / share; b < B; b += 16 / share) {
    double s, n;
    sequence_part(a, b, (wave % share) * 64 + lane, share * 64, s, n);
    s = wave_sum(s);
    n = wave_sum(n);
    if (lane == 0) {
      sums[b][wave % share] = s;
      counts[b][wave % share] = n;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  double mine = 0.0;
  if (lane < (int)a.pairs) {
    double total[2] = {0.0, 0.0}, count[2] = {0.0, 0.0};
    for (int k = 0; k < 2; ++k)
      for (int j = 0; j < share; ++j) {
        total[k] += sums[2 * lane + k][j];
        count[k] += counts[2 * lane + k][j];
      }
    mine = pair_terms(a, lane, total, count);
  }
  mine = wave_sum(mine);
  if (lane == 0) loss[0] = (float)(mine / (double)a.pairs);
}

// out_k = scale * sum over n of in[k * n + i], in double.  One workgroup: 4 us for two sums over 8 x 1021 tokens, 19 over 64 x 1024, 278 over
// 1024 x 1024 (a third of what a policy loss of 64 classes takes for so many, 3 % with 32000).
__global__ __launch_bounds__(1024) void sums_kernel(const double* in, int64_t n, double scale, float* out0, float* out1) {
  __shared__ double sm[2][16];
  double total[2] = {0.0, 0.0};
  total[0] = sum_in_eights(threadIdx.x, n, 1024, [&](int64_t i) { return in[i]; });
  if (out1) total[1] = sum_in_eights(threadIdx.x, n, 1024, [&](int64_t i) { return in[n + i]; });
  for (int k = 0; k < 2; ++k) {
    total[k] = wave_sum(total[k]);
    if ((threadIdx.x & 63) == 0) sm[k][threadIdx.x >> 6] = total[k];
  }
  __syncthreads();
  if (threadIdx.x < 2 && (threadIdx.x == 0 || out1)) {
    double s = 0.0;
    for (int i = 0; i < 16; ++i) s += sm[threadIdx.x][i];
    (threadIdx.x ? out1 : out0)[0] = (float)(s * scale);
  }
}

// ---- policy ----------------------------------------------------------------------------------------------------------------
// Weight of every token of sequence b: 1 / (tokens that count), or by_sequence 1 / (its own such tokens * sequences that have any).  One
// workgroup: 3 us for 8 x 1021 labels, 10 for 64 x 1024, 135 for 1024 x 1024.
__global__ __launch_bounds__(1024) void token_weights_kernel(const TokenRows r, int by_sequence, double* weights) {
  __shared__ double sm[16];
  const int64_t R = r.T - r.shift, all = r.B * r.T;
  double total = 0.0;
  if (by_sequence) {      // a wavefront to a sequence
    for (int64_t b = threadIdx.x >> 6; b < r.B; b += 16) {
      const double n = wave_sum(sum_in_eights(threadIdx.x & 63, R, 64, [&](int64_t t) { return r.labels[b * r.T + t + r.shift] != r.ignore_index ? 1.0 : 0.0; }));
      if ((threadIdx.x & 63) == 0) weights[b] = n;
      total += n > 0.0 ? 1.0 : 0.0;
    }
  } else {
    double n = sum_in_eights(threadIdx.x, all, 1024, [&](int64_t i) { return r.labels[i] != r.ignore_index ? 1.0 : 0.0; });
    if (r.shift)      // no row is scored against a sequence's first label
      for (int64_t b = threadIdx.x; b < r.B; b += 1024) n -= r.labels[b * r.T] != r.ignore_index ? 1.0 : 0.0;
    total = wave_sum(n);
  }
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = total;
  __syncthreads();
  total = 0.0;
  for (int i = 0; i < 16; ++i) total += sm[i];
  for (int64_t b = threadIdx.x; b < r.B; b += 1024) {
    const double n = by_sequence ? weights[b] * total : total;
    weights[b] = n > 0.0 ? 1.0 / n : 0.0;
  }
}

struct PolicyArgs {
  const float* old;      // [B, R]
  const float* ref;      // [B, R] or null
  const float* adv;
  int64_t a_sb, a_st;
  double low, high;      // ln(1 - clip_low), ln(1 + clip_high)
  float low_ratio, high_ratio, kl_coef;
  double scale;          // of the loss
};

// One token:  -min(r A, clip(r) A) + kl_coef (e^q - q - 1)  with r = e^d, d = logprob - old, q = ref - logprob; g is its derivative by the
// logprob (at the clip's borders that of r A).  The differences and the comparison are in double; e^q - 1 - q is summed up as
// the series it is where the subtraction would lose its digits.
struct TokenTerms { float loss, kl, g; };
__device__ __forceinline__ TokenTerms policy_token(const PolicyArgs& a, float old, float A, float ref, double logprob) {
  const double d = logprob - (double)old;
  const float ratio = expf((float)d);
  const bool outside = A >= 0.f ? d > a.high : d < a.low;
  TokenTerms o;
  o.loss = -(outside ? (A >= 0.f ? a.high_ratio : a.low_ratio) : ratio) * A;
  o.g = outside ? 0.f : -ratio * A;
  o.kl = 0.f;
  if (a.ref) {
    const double dq = (double)ref - logprob;
    const float q = (float)dq;
    float e, k;
    if (fabsf(q) < 0.5f) {      // q^2 / 2! + q^3 / 3! + ...: eight terms leave 2^-26 of it
      float h = fmaf(q, 1.f / 9.f, 1.f);
      h = fmaf(h * q, 1.f / 8.f, 1.f);
      h = fmaf(h * q, 1.f / 7.f, 1.f);
      h = fmaf(h * q, 1.f / 6.f, 1.f);
      h = fmaf(h * q, 1.f / 5.f, 1.f);
      h = fmaf(h * q, 1.f / 4.f, 1.f);
      h = fmaf(h * q, 1.f / 3.f, 1.f);
      k = 0.5f * q * q * h;
      e = q + k;
    } else {
      e = expf(q) - 1.f;
      k = e - q;
    }
    o.kl = k;
    if (a.kl_coef != 0.f) {      // (else it is for the log alone, where it may be infinite)
      o.loss = fmaf(a.kl_coef, k, o.loss);
      o.g = fmaf(-a.kl_coef, e, o.g);
    }
  }
  return o;
}

// A row's log-probability, its part of the loss and, where wanted, its gradient.  terms: [2][B * R], weighted.  Every lane forms the token's
// terms itself, which spares a second exchange.  Bound by memory: 5371 of 8 x 1021 rows of 32000 classes in bf16 scored, 867 MB in 161 us, 5.4 TB/s;
// 131072 classes, whose row takes half a CU's registers, 969 MB in 187, 5.2.
template <int DT, int NV, bool ONE, bool LOOP, bool PAST>
__global__ __launch_bounds__(ONE ? 256 : 1024) void policy_kernel(const TokenRows r, int b0, int t0, const GradRows d, const PolicyArgs a, const double* weights,
                                                                  float* logprobs, float2* stats, float* coef, double* terms) {
  __shared__ SumSlots<false> slots[1];
  const int T = (int)r.T, R = T - r.shift, t = row_of_group<ONE>(t0);
  const int64_t b = b0 + (int)blockIdx.y, at = b * R + t;
  if (t >= T) return;
  const int tid = ONE ? threadIdx.x & 63 : threadIdx.x, n = ONE ? 64 : blockDim.x;
  const int64_t y = t < R ? r.labels[b * T + t + r.shift] : 0;
  const LabelKind kind = t < R ? label_kind(r, y) : LABEL_SKIP;
  char* dx = (char*)d.dx + (b * d.sb + t * d.st) * pf_es<DT>;
  if (kind != LABEL_OK) {
    const float none = kind == LABEL_BAD ? NAN : 0.f;
    if (tid == 0 && t < R) {
      logprobs[at] = none;
      terms[at] = terms[r.B * R + at] = none;
      if (coef) {
        coef[at] = none;
        stats[at] = make_float2(0.f, none);
      }
    }
    if (d.dx) fill_row<DT, PAST>(dx, (int)r.V, none, tid, n);
    return;
  }
  const float old = a.old[at], A = a.adv[b * a.a_sb + t * a.a_st], ref = a.ref ? a.ref[at] : 0.f;
  const double w = weights[b];
  const char* x = (const char*)r.logits + (b * r.sb + t * r.st) * pf_es<DT>;
  RowReader<DT, NV, ONE, LOOP> row(x, d.dx ? dx : x, (int)r.V);
  const float xy = element<DT>(row.x, (int)y);
  const RowStats s = row_stats<false>(r, row, xy, slots, true);
  const TokenTerms o = policy_token(a, old, A, ref, s.logprob);
  const float g = (float)(w * a.scale * (double)o.g);
  if (tid == 0) {
    logprobs[at] = (float)s.logprob;
    terms[at] = w * a.scale * (double)o.loss;
    terms[r.B * R + at] = w * (double)o.kl;
    if (coef) {
      coef[at] = g;
      stats[at] = pack_stats(s);
    }
  }
  if (!d.dx) return;
  const RowGrad rg = row_grad(r, s, g, xy);
  const int tiles = row.tiles(), label = (int)y < row.cut.head ? -1 : (int)y - row.cut.head - tid * VE<DT>;
  for (int tile = tiles - 1; tile >= 0; --tile) {
    if (LOOP && tile != tiles - 1) row.load(tile);      // (the last one is still there)
    char* to = dx + row.cut.start() + (size_t)((unsigned)(tile * NV * n) * 16u);
    if (s.slow) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid < row.left(tile, i))
          gradient_vector<DT, true, PAST>(row.v[i], label - (tile * NV + i) * n * VE<DT>, s, rg, r.c, to + (unsigned)(i * n) * 16u + (unsigned)tid * 16u);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid < row.left(tile, i))
          gradient_vector<DT, false, PAST>(row.v[i], label - (tile * NV + i) * n * VE<DT>, s, rg, r.c, to + (unsigned)(i * n) * 16u + (unsigned)tid * 16u);
    }
  }
  if (tid < row.cut.loose) gradient_element<DT>(row.last, row.cut.element(tid), (int)y, s, rg, r.c, dx);
}

// ---- launches --------------------------------------------------------------------------------------------------------------
// How a row is dealt out.  NV accesses of a lane in flight, WAVES wavefronts to a row; ONE: a wavefront alone, four rows to a workgroup; LOOP: in
// several tiles.  A row that is only read goes through eight wavefronts at most, so that several workgroups share a CU and one loads while
// another sums: us for 400 MB, 2 wavefronts of 8 / 4 of 4 at 8192 classes 69 / 72 (in bf16), 8 of 8 / 4 of 16 at 32000 67 / 69, 13 wavefronts of 8 /
// loops of 8 at 49999 88 / 59, 13 of 16 / loops at 100000 91 / 75.  One whose gradient follows is kept whole as far as registers go: 4 wavefronts of 4 /
// 2 of 8 at 8192 191 / 197, 8 of 8 / 4 of 16 at 32000 187 / 190, 13 of 8 / 7 of 16 at 49999 208 / 176, 13 of 16 / loops of 8 at 100000 195 / 219.
struct RowPlan { int nv, waves; bool one, loop; };
RowPlan row_plan(int dtype, int64_t V, bool gradient) {
  const int64_t full = V / (dtype == PF_F32 ? 4 : 8);
  const auto waves = [&](int nv) { return (int)((full + 64 * nv - 1) / (64 * nv)); };
  if (full <= 64 * 4) return {4, 1, true, false};
  if (gradient && full <= 64 * 4 * 4) return {4, waves(4), false, false};
  if (full <= 64 * 8 * 8) return {8, waves(8), false, false};
  if (gradient && full <= 64 * 16 * 16) return {16, waves(16), false, false};
  return {8, gradient ? 16 : 8, false, true};
}
// A gradient of this many bytes goes past the caches, which it would only empty of logits that are still to be read: preference loss at [4, 2048] x
// 32000 in bf16 272 -> 232 us, policy loss 198 -> 190.  In the policy loss's one pass that holds for rows of whole cache lines; a line that two workgroups
// write goes out twice (49999 classes in fp16 172 -> 179, 10007 in fp32 230 -> 243).
constexpr int64_t PAST_BYTES = 256ll << 20;

// rows along x, sequences along y; a launch has less than 2^32 threads, and kernels loop over what is beyond
dim3 rows_grid(int64_t units, int64_t B, int per_group, int threads, int64_t most = 1ll << 40) {
  const int64_t y = B < 65535 ? B : 65535;
  int64_t x = (units + per_group - 1) / per_group, limit = ((1ll << 32) - 1) / threads / y;
  if (limit > most / y) limit = most / y;
  if (limit < 1) limit = 1;
  if (x > limit) x = limit;
  return dim3((unsigned)(x < 1 ? 1 : x), (unsigned)y);
}

int check_rows(const char* who, const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
               double temperature) {
  PF_REQUIRE(pf_is_float_dtype(dtype), "%s: logits are fp32, fp16 or bf16", who);
  PF_REQUIRE(B >= 0 && T >= 0 && V >= 1 && sb >= 0 && st >= 0, "%s: bad sizes", who);
  PF_REQUIRE(shift == 0 || shift == 1, "%s: shift is 0 or 1", who);
  PF_REQUIRE(temperature > 0.0 && temperature >= 1e-6 && temperature <= 1e6, "%s: temperature must lie in [1e-6, 1e6]", who);
  PF_REQUIRE(B * T == 0 || (logits && labels), "%s: null pointer", who);
  PF_REQUIRE(T <= (1ll << 30) && B < (1ll << 31), "%s: too many rows", who);
  PF_REQUIRE(V <= (1ll << 28), "%s: too many classes", who);
  return PF_OK;
}

TokenRows token_rows(const void* logits, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
                     int64_t ignore_index, double temperature) {
  const double c = 1.4426950408889634 / temperature;
  return {logits, sb, st, labels, B, T, V, ignore_index, shift, (float)c, (double)(float)c / c - 1.0, 1.0 / temperature};
}

}  // namespace

#define PF_BY_DTYPE(dt, CALL)                \
  do {                                       \
    if (dt == PF_F32) { CALL(PF_F32); }      \
    else if (dt == PF_F16) { CALL(PF_F16); } \
    else { CALL(PF_BF16); }                  \
  } while (0)
// CALL(dtype, NV, ONE, LOOP), or OTHER where a plan for a gradient has another kernel, with grid, block, b0 and t0 for rows of V classes: a
// launch has less than 2^32 threads, so many rows or sequences go in several
#define PF_ONE(DT) CALL(DT, 4, true, false)
#define PF_SOME(DT) CALL(DT, 8, false, false)
#define PF_LOOP(DT) CALL(DT, 8, false, true)
#define PF_FEW(DT) CALL(DT, 4, false, false)
#define PF_MANY(DT) CALL(DT, 16, false, false)
constexpr int64_t ROWS_MOST = 1 << 20;
#define PF_BY_ROW(dt, V, rows, B, gradient, OTHER)                                                  \
  do {                                                                                              \
    const RowPlan plan = row_plan(dt, V, gradient);                                                 \
    const dim3 block(plan.one ? 256 : 64 * plan.waves);                                             \
    for (int64_t t0 = 0; t0 < (rows); t0 += ROWS_MOST) {                                            \
      const int64_t here = (rows) - t0 < ROWS_MOST ? (rows) - t0 : ROWS_MOST;                       \
      const unsigned groups = (unsigned)(plan.one ? (here + 3) / 4 : here);                         \
      int64_t most = ((1ll << 32) - 1) / ((int64_t)groups * block.x);                               \
      if (most > 65535) most = 65535;                                                               \
      for (int64_t b0 = 0; b0 < (B); b0 += most) {                                                  \
        const dim3 grid(groups, (unsigned)((B) - b0 < most ? (B) - b0 : most));                     \
        if (plan.one) { PF_BY_DTYPE(dt, PF_ONE); }                                                  \
        else if (plan.loop) { PF_BY_DTYPE(dt, PF_LOOP); }                                           \
        else if (plan.nv == 8) { PF_BY_DTYPE(dt, PF_SOME); }                                        \
        OTHER(dt)                                                                                   \
      }                                                                                             \
    }                                                                                               \
  } while (0)
#define PF_NO_OTHER(dt)
#define PF_FEW_OR_MANY(dt)                                                                          \
  else if (plan.nv == 4) { PF_BY_DTYPE(dt, PF_FEW); }                                               \
  else { PF_BY_DTYPE(dt, PF_MANY); }

extern "C" int pf_token_logprob_fwd(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels,
                                    int shift, int64_t ignore_index, double temperature, float* logprobs, float* stats, void* stream) {
  if (int rc = check_rows("pf_token_logprob_fwd", logits, dtype, B, T, V, sb, st, labels, shift, temperature)) return rc;
  if (B == 0 || T <= shift) return PF_OK;
  PF_REQUIRE(logprobs, "pf_token_logprob_fwd: null pointer");
  const TokenRows r = token_rows(logits, B, T, V, sb, st, labels, shift, ignore_index, temperature);
#define CALL(DT, NV, ONE, LOOP) hipLaunchKernelGGL((token_logprob_kernel<DT, NV, ONE, LOOP, float>), grid, block, 0, (hipStream_t)stream, r, (int)b0, (int)t0, logprobs, (float2*)stats)
  PF_BY_ROW(dtype, V, T - shift, B, false, PF_NO_OTHER);
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
  const int64_t full = V / (dtype == PF_F32 ? 4 : 8), pieces = full > 64 * GNV ? (full + 64 * GNV - 1) / (64 * GNV) : 1;
  // (with unless_one most calls have nothing to do: few workgroups, that loop where there is something)
  const dim3 grid = rows_grid(T * pieces, B, 4, 256, unless_one ? 2048 : 1ll << 40);
  const bool past = B * T * V * pf_dtype_size(dtype) >= PAST_BYTES;
#define CALL(DT)                                                                                                                                       \
  if (past) hipLaunchKernelGGL((token_gradient_kernel<DT, true>), grid, dim3(256), 0, (hipStream_t)stream, r, d, (const float2*)stats, coef, g_sb, g_st, scale, \
                               unless_one, (unsigned)pieces);                                                                                            \
  else hipLaunchKernelGGL((token_gradient_kernel<DT, false>), grid, dim3(256), 0, (hipStream_t)stream, r, d, (const float2*)stats, coef, g_sb, g_st, scale, \
                          unless_one, (unsigned)pieces)
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
#define CALL(DT, NV, ONE, LOOP) hipLaunchKernelGGL((token_logprob_kernel<DT, NV, ONE, LOOP, double>), grid, block, 0, (hipStream_t)stream, r, (int)b0, (int)t0, logprobs, (float2*)stats)
    PF_BY_ROW(dtype, V, R, B, false, PF_NO_OTHER);
#undef CALL
  }
  const PairArgs a = {logprobs, labels, R + shift, shift, ignore_index, ref, beta, label_smoothing, length_average, pairs, rewards, coef};
  // one workgroup saves a launch and reads less at a time: us of it / of the two, [2, 128] 4.3 / 6.1, [4, 2047] 5.5 / 6.9, [16, 1024] 7.1 / 7.9,
  // [32, 1024] 10.8 / 10.2, [64, 2048] 32 / 19
  if (B <= FEW_SEQUENCES && B * R <= 16384) {
    hipLaunchKernelGGL(preference_few_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a, loss);
  } else {
    hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)(pairs < 65536 ? pairs : 65536)), dim3(512), 0, (hipStream_t)stream, a, workspace);
    hipLaunchKernelGGL(sums_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, workspace, pairs, 1.0 / (double)pairs, loss, (float*)nullptr);
  }
  PF_CHECK_LAUNCH("pf_preference_loss");
  return PF_OK;
}

extern "C" int64_t pf_policy_workspace(int64_t B, int64_t T, int shift) { return B + 2 * B * (T > shift ? T - shift : 0); }

extern "C" int pf_policy_loss(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t sb, int64_t st, const int64_t* labels, int shift,
                              int64_t ignore_index, double temperature, const float* old_logprobs, const float* advantages, int64_t a_sb, int64_t a_st,
                              const float* ref_logprobs, double clip_low, double clip_high, double kl_coef, int by_sequence, double scale, float* loss, float* kl,
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
  const PolicyArgs a = {old_logprobs, ref_logprobs, advantages, a_sb, a_st, clip_low < 1.0 ? log1p(-clip_low) : -INFINITY, log1p(clip_high),
                        (float)(1.0 - clip_low), (float)(1.0 + clip_high), (float)kl_coef, scale};
  const int64_t R = T > shift ? T - shift : 0;
  double* terms = workspace ? workspace + B : nullptr;
  if (B * T > 0 && (R > 0 || dlogits)) {
    if (R > 0) hipLaunchKernelGGL(token_weights_kernel, dim3(1), dim3(1024), 0, s, r, by_sequence, workspace);
    const int64_t es = pf_dtype_size(dtype);
    const bool past = dlogits && B * T * V * es >= PAST_BYTES && pf_aligned(dlogits, 128) && V * es % 128 == 0 && d_sb * es % 128 == 0 && d_st * es % 128 == 0;
#define CALL(DT, NV, ONE, LOOP)                                                                                                                     \
  if (past) hipLaunchKernelGGL((policy_kernel<DT, NV, ONE, LOOP, true>), grid, block, 0, s, r, (int)b0, (int)t0, d, a, workspace, logprobs, (float2*)stats, coef, terms); \
  else hipLaunchKernelGGL((policy_kernel<DT, NV, ONE, LOOP, false>), grid, block, 0, s, r, (int)b0, (int)t0, d, a, workspace, logprobs, (float2*)stats, coef, terms)
    PF_BY_ROW(dtype, V, dlogits ? T : R, B, dlogits != nullptr, PF_FEW_OR_MANY);
#undef CALL
  }
  hipLaunchKernelGGL(sums_kernel, dim3(1), dim3(1024), 0, s, terms, B * R, 1.0, loss, kl);
  PF_CHECK_LAUNCH("pf_policy_loss");
  return PF_OK;
}
