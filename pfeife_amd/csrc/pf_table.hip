// Token table: lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale W[id_i];   dW[v] = scale * sum of dout_i over the i with id_i = v, in 32 bits, rounded once
//
// Text holds few tokens very often and most of the table not at all, so the gradient's work is dealt out by the tokens and not by
// the table's rows: the places are sorted by token (a stable radix sort of two digits, 2^18 rows; three beyond), a
// group of lanes adds up CHUNK neighbours of the sorted list, and a token whose run crosses chunks has its partial sums added
// in order by a last kernel.  Which lane adds what follows from the ids alone: the same ids give the same bits.  Rows that no token
// names are found by searching the sorted list and are zeroed by other workgroups of the same launch, so every byte of the
// gradient is written once.
#include "pf_common.h"

namespace {

constexpr int BINS = 512;        // of one digit
constexpr int SMALL = 4096;      // ids that one workgroup sorts by itself

__device__ __forceinline__ int key_of(int64_t id, int64_t vocab, int64_t padding) { return id >= 0 && id < vocab && id != padding ? (int)id : (int)vocab; }

// One digit's stable ranks: `wc[digit]` is where the wavefront's next key of the digit goes; -> where this lane's goes
__device__ __forceinline__ int rank_of(int digit, bool active, int bits, int* wc) {
  const int lane = threadIdx.x & 63;
  unsigned long long same = __ballot(active);
  for (int b = 0; b < bits; ++b) {
    const bool set = (digit >> b) & 1;
    const unsigned long long m = __ballot(set);
    same &= set ? m : ~m;
  }
  int at = 0;
  if (active) at = wc[digit];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (active && (same & ((1ull << lane) - 1)) == 0) wc[digit] = at + __popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return at + __popcll(same & ((1ull << lane) - 1));
}

// sums of BINS values before each, by the first BINS threads of a workgroup; every thread of it calls
__device__ __forceinline__ int scan_bins(int v, int* sm) {
  const int t = threadIdx.x, lane = t & 63;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63 && t < BINS) sm[t >> 6] = x;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < (t >> 6) && w < BINS / 64; ++w) before += sm[w];
  __syncthreads();
  return before + x - v;
}

// Up to SMALL ids sorted by one workgroup, in LDS
__global__ __launch_bounds__(1024) void table_sort_small_kernel(const int64_t* ids, int n, int64_t vocab, int64_t padding, int bits, int digits, int* keys, int* places) {
  extern __shared__ int lds[];
  auto kb = [&](int k) { return lds + k * SMALL; };
  auto pb = [&](int k) { return lds + (2 + k) * SMALL; };
  int* counts = lds + 4 * SMALL;      // [16][BINS]
  __shared__ int sm[BINS / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (n + 1023) / 1024 * 64;      // keys of a wavefront
  for (int i = t; i < n; i += 1024) {
    kb(0)[i] = key_of(ids[i], vocab, padding);
    pb(0)[i] = i;
  }
  for (int d = 0; d < digits; ++d) {
    const int *kin = kb(d & 1), *pin = pb(d & 1);
    int *kout = kb((d & 1) ^ 1), *pout = pb((d & 1) ^ 1);
    const int shift = d * bits, mask = (1 << bits) - 1;
    for (int i = t; i < 16 * BINS; i += 1024) counts[i] = 0;
    __syncthreads();
    for (int i = lane; i < per; i += 64)
      if (wave * per + i < n) atomicAdd(&counts[wave * BINS + ((kin[wave * per + i] >> shift) & mask)], 1);
    __syncthreads();
    int total = 0;
    if (t < BINS)
      for (int w = 0; w < 16; ++w) total += counts[w * BINS + t];
    int at = scan_bins(total, sm);
    if (t < BINS)
      for (int w = 0; w < 16; ++w) {
        const int c = counts[w * BINS + t];
        counts[w * BINS + t] = at;
        at += c;
      }
    __syncthreads();
    for (int i = lane; i < per; i += 64) {
      const bool active = wave * per + i < n;
      const int key = active ? kin[wave * per + i] : 0, place = active ? pin[wave * per + i] : 0;
      const int to = rank_of((key >> shift) & mask, active, bits, counts + wave * BINS);
      if (active) {
        kout[to] = key;
        pout[to] = place;
      }
    }
    __syncthreads();
  }
  for (int i = t; i < n; i += 1024) {
    keys[i] = kb(digits & 1)[i];
    places[i] = pb(digits & 1)[i];
  }
}

// How often each value of a digit occurs among a block's keys
template <int ITEMS>
__global__ __launch_bounds__(256) void table_count_kernel(const int64_t* ids, const int* keys, int64_t n, int64_t vocab, int64_t padding, int shift, int bits, int* counts) {
  __shared__ int c[BINS];
  const int t = threadIdx.x;
  for (int i = t; i < BINS; i += 256) c[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * ITEMS;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * 256 + t;
    if (at < n) atomicAdd(&c[((ids != nullptr ? key_of(ids[at], vocab, padding) : keys[at]) >> shift) & ((1 << bits) - 1)], 1);
  }
  __syncthreads();
  for (int i = t; i < BINS; i += 256) counts[(int64_t)blockIdx.x * BINS + i] = c[i];
}

// ... and the keys to their places.  A block finds out from all blocks' counts where its own begin.
template <int ITEMS>
__global__ __launch_bounds__(256) void table_place_kernel(const int64_t* ids, const int* keys, const int* places, int64_t n, int64_t vocab, int64_t padding, int shift,
                                                          int bits, const int* counts, int* keys_out, int* places_out) {
  __shared__ int wc[4][BINS];
  __shared__ int sm[8];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, mask = (1 << bits) - 1;
  for (int i = t; i < 4 * BINS; i += 256) (&wc[0][0])[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * ITEMS + wave * 64 * ITEMS;
  int key[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * 64 + lane;
    key[i] = at >= n ? 0 : ids != nullptr ? key_of(ids[at], vocab, padding) : keys[at];
    if (at < n) atomicAdd(&wc[wave][(key[i] >> shift) & mask], 1);
  }
  // thread t: digits 2 t and 2 t + 1
  int mine[2] = {0, 0}, all[2] = {0, 0};
  const int blocks = gridDim.x;
#pragma unroll 8
  for (int b = 0; b < blocks; ++b) {
    const int2 c = *(const int2*)(counts + (int64_t)b * BINS + 2 * t);
    all[0] += c.x;
    all[1] += c.y;
    if (b < (int)blockIdx.x) { mine[0] += c.x; mine[1] += c.y; }
  }
  int x = all[0] + all[1];
  const int own = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) sm[wave] = x;
  __syncthreads();
  int before = x - own;
  for (int w = 0; w < wave; ++w) before += sm[w];
  mine[0] += before;
  mine[1] += before + all[0];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int at = mine[k];
    for (int w = 0; w < 4; ++w) {
      const int c = wc[w][2 * t + k];
      wc[w][2 * t + k] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * 64 + lane;
    const bool active = at < n;
    const int to = rank_of((key[i] >> shift) & mask, active, bits, wc[wave]);
    if (active) {
      keys_out[to] = key[i];
      places_out[to] = places != nullptr ? places[at] : (int)at;
    }
  }
}

// Eight neighbouring elements that lie on 4 bytes, `left` of them inside the row
typedef uint32_t four_t __attribute__((ext_vector_type(4), aligned(4)));
template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t i, int64_t left, float (&v)[8]) {
  if (left >= 8) {
    if constexpr (DT == PF_F32) {
      const four_t a = *(const four_t*)((const float*)p + i), b = *(const four_t*)((const float*)p + i + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[k] = __uint_as_float(a[k]); v[4 + k] = __uint_as_float(b[k]); }
    } else {
      const four_t a = *(const four_t*)((const uint16_t*)p + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = DT == PF_BF16 ? __uint_as_float(a[k] << 16) : pf_f16_bits_to_f32((uint16_t)(a[k] & 0xffffu));
        v[2 * k + 1] = DT == PF_BF16 ? __uint_as_float(a[k] & 0xffff0000u) : pf_f16_bits_to_f32((uint16_t)(a[k] >> 16));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? Codec<DT>::load(p, i + k) : 0.f;
  }
}
template <int DT> __device__ __forceinline__ void store8(void* p, int64_t i, int64_t left, const float (&v)[8]) {
  if (left >= 8) {
    if constexpr (DT == PF_F32) {
      four_t a, b;
#pragma unroll
      for (int k = 0; k < 4; ++k) { a[k] = __float_as_uint(v[k]); b[k] = __float_as_uint(v[4 + k]); }
      *(four_t*)((float*)p + i) = a;
      *(four_t*)((float*)p + i + 4) = b;
    } else {
      four_t a;
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] = DT == PF_BF16 ? pf_pack2_bf16(v[2 * k], v[2 * k + 1]) : pf_pack2_f16(v[2 * k], v[2 * k + 1]);
      *(four_t*)((uint16_t*)p + i) = a;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) Codec<DT>::store(p, i + k, v[k]);
  }
}
// W = 8 where rows lie on 4 bytes, else 1
template <int DT, int W> __device__ __forceinline__ void load_row(const void* p, int64_t i, int64_t left, float (&v)[W]) {
  if constexpr (W == 8) load8<DT>(p, i, left, v);
  else v[0] = left > 0 ? Codec<DT>::load(p, i) : 0.f;
}
template <int DT, int W> __device__ __forceinline__ void store_row(void* p, int64_t i, int64_t left, const float (&v)[W]) {
  if constexpr (W == 8) store8<DT>(p, i, left, v);
  else if (left > 0) Codec<DT>::store(p, i, v[0]);
}

// out[i] = scale * W[ids[i]]; a group of 2^lg lanes takes a row
template <int DT, int W>
__global__ __launch_bounds__(256) void table_lookup_kernel(const void* table, const int64_t* ids, void* out, int64_t n, int64_t dim, int64_t vocab, float scale, int lg) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lg;
  if (i >= n) return;
  const int64_t id = ids[i];
  const bool ok = id >= 0 && id < vocab;
  const int64_t step = (int64_t)W << lg;
#pragma unroll 4
  for (int64_t c = (int64_t)(threadIdx.x & ((1 << lg) - 1)) * W; c < dim; c += step) {
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = NAN;      // (an id outside the table is visible, never a wild read)
    if (ok) load_row<DT, W>(table, id * dim + c, dim - c, v);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] *= scale;
    store_row<DT, W>(out, i * dim + c, dim - c, v);
  }
}

struct Sum {
  const void* dout;
  const int* keys;
  const int* places;
  void* dtable;
  float* partial;      // [chunks][2][dim]: of a run that comes from the chunk before, of one that goes on into the next
  int64_t n, dim, vocab, chunks;
  float scale;
  int lg, t_f32, accumulate;
};

template <int DT, int W>
__device__ __forceinline__ void put_row(const Sum& s, int64_t row, int64_t c, float (&v)[W]) {
  const int64_t left = s.dim - c, at = row * s.dim + c;
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] *= s.scale;
  if (s.accumulate) {
    float old[W];
    if (s.t_f32) load_row<PF_F32, W>(s.dtable, at, left, old);
    else load_row<DT, W>(s.dtable, at, left, old);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] += old[k];
  }
  if (s.t_f32) store_row<PF_F32, W>(s.dtable, at, left, v);
  else store_row<DT, W>(s.dtable, at, left, v);
}

// Workgroups of the first `sums` columns of the grid: a group of lanes adds up one chunk of the sorted list in one slice of the columns;
// runs that end inside it go to the table's gradient, the others' parts to `partial`.  The other workgroups: rows without a token.
template <int DT, int W, int CHUNK>
__global__ __launch_bounds__(256) void table_sum_kernel(const Sum s, int sums) {
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x >= sums) {
    // 64 rows to a wavefront, a lane looks for its own; then the rows that are not there, one by one
    const int64_t v0 = ((int64_t)((int)blockIdx.x - sums) * 4 + (threadIdx.x >> 6)) * 64;
    const int64_t v = v0 + lane;
    int64_t lo = 0, hi = s.n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (s.keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    unsigned long long missing = __ballot(v < s.vocab && !(lo < s.n && s.keys[lo] == v));
    const int64_t step = 64 * W;
    float zero[W];
#pragma unroll
    for (int k = 0; k < W; ++k) zero[k] = 0.f;
    while (missing) {
      const int b = __ffsll((long long)missing) - 1;
      missing &= missing - 1;
      for (int64_t c = lane * W; c < s.dim; c += step) {
        if (s.t_f32) store_row<PF_F32, W>(s.dtable, (v0 + b) * s.dim + c, s.dim - c, zero);
        else store_row<DT, W>(s.dtable, (v0 + b) * s.dim + c, s.dim - c, zero);
      }
    }
    return;
  }
  const int G = 1 << s.lg;
  const int64_t slices = (s.dim + (int64_t)G * W - 1) / ((int64_t)G * W);
  const int64_t unit = (int64_t)blockIdx.x * (256 >> s.lg) + (threadIdx.x >> s.lg);
  const int64_t chunk = unit / slices, c = (unit % slices) * G * W + (threadIdx.x & (G - 1)) * W;
  if (chunk >= s.chunks || c >= s.dim) return;
  const int64_t j0 = chunk * CHUNK, left = s.dim - c;
  const int count = (int)(s.n - j0 < CHUNK ? s.n - j0 : CHUNK);
  const int last_before = j0 > 0 ? s.keys[j0 - 1] : -1;
  const int first_after = j0 + count < s.n ? s.keys[j0 + count] : -1;
  float acc[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = 0.f;
  int run = -1;
  bool from_before = false;
  // a finished run: inside the chunk, or the part of one that began before it
  auto flush = [&](bool goes_on) {
    if (run < 0 || run >= s.vocab) return;
    if (from_before || goes_on) {
      float* to = s.partial + ((chunk * 2 + (from_before ? 0 : 1)) * s.dim);
      store_row<PF_F32, W>(to, c, left, acc);
    } else {
      put_row<DT, W>(s, run, c, acc);
    }
  };
  constexpr int AHEAD = 8;
  for (int b = 0; b < count; b += AHEAD) {
    int key[AHEAD];
    float v[AHEAD][W];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int64_t j = j0 + (b + q < count ? b + q : count - 1);
      key[q] = b + q < count ? s.keys[j] : -1;
      load_row<DT, W>(s.dout, (int64_t)s.places[j] * s.dim + c, left, v[q]);
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (b + q >= count) break;
      if (key[q] != run) {
        flush(false);
        from_before = b + q == 0 && key[q] == last_before;
        run = key[q];
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += v[q][k];
    }
  }
  flush(run == first_after);
}

// A run that begins in this chunk and goes on into others: their parts, in the list's order, TEAMS of them at once
template <int DT, int W, int CHUNK, int TEAMS>
__global__ __launch_bounds__(64 * TEAMS) void table_join_kernel(const Sum s) {
  __shared__ float part[TEAMS][64 * W];
  const int64_t chunk = blockIdx.x;
  const int lane = threadIdx.x & 63, team = threadIdx.x >> 6;
  const int64_t next = (chunk + 1) * CHUNK;
  if (next >= s.n) return;
  const int run = s.keys[next - 1];
  if (run >= s.vocab || s.keys[next] != run) return;
  if (s.keys[chunk * CHUNK] == run && chunk > 0 && s.keys[chunk * CHUNK - 1] == run) return;      // (it began before)
  // the last chunk that begins with the run
  int64_t lo = chunk + 1, hi = s.chunks - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (s.keys[mid * CHUNK] == run) lo = mid;
    else hi = mid - 1;
  }
  const int64_t many = lo - chunk;        // parts besides this chunk's own
  const int64_t c = (int64_t)blockIdx.y * 64 * W + lane * W, left = s.dim - c;
  const int64_t per = (many + TEAMS - 1) / TEAMS, a = chunk + 1 + team * per, b = a + per < lo + 1 ? a + per : lo + 1;
  float acc[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = 0.f;
  if (left > 0) {
    if (team == 0) load_row<PF_F32, W>(s.partial + (chunk * 2 + 1) * s.dim, c, left, acc);
#pragma unroll 4
    for (int64_t p = a; p < b; ++p) {
      float v[W];
      load_row<PF_F32, W>(s.partial + p * 2 * s.dim, c, left, v);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += v[k];
    }
  }
  if (team > 0) {
#pragma unroll
    for (int k = 0; k < W; ++k) part[team][lane * W + k] = acc[k];
  }
  __syncthreads();
  if (team > 0 || left <= 0) return;
  for (int w = 1; w < TEAMS && w * per < many; ++w) {
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k] += part[w][lane * W + k];
  }
  put_row<DT, W>(s, run, c, acc);
}

inline int64_t round_up(int64_t n, int64_t k) { return (n + k - 1) / k * k; }
inline int chunk_of(int64_t n) { return n <= 8192 ? 8 : 32; }
inline int items_of(int64_t n) { return n <= 65536 ? 8 : 16; }

struct Layout { int64_t keys[2], places[2], counts, partial, bytes; };
Layout layout_of(int64_t n, int64_t dim) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t p = at; at += round_up(bytes, 256); return p; };
  for (int k = 0; k < 2; ++k) { l.keys[k] = take(n * 4); l.places[k] = take(n * 4); }
  l.counts = take((n + 256 * items_of(n) - 1) / (256 * items_of(n)) * BINS * 4);
  l.partial = take((n + chunk_of(n) - 1) / chunk_of(n) * 2 * dim * 4);
  l.bytes = at;
  return l;
}

template <int DT, int W, int CHUNK>
void sum_launch(const Sum& s, hipStream_t st) {
  const int64_t slices = (s.dim + ((int64_t)W << s.lg) - 1) / ((int64_t)W << s.lg);
  const int64_t sums = (s.chunks * slices + (256 >> s.lg) - 1) / (256 >> s.lg);
  const int64_t zeros = s.accumulate ? 0 : (s.vocab + 255) / 256;
  if (sums + zeros > 0) hipLaunchKernelGGL((table_sum_kernel<DT, W, CHUNK>), dim3((unsigned)(sums + zeros)), dim3(256), 0, st, s, (int)sums);
  if (s.chunks > 1)
    hipLaunchKernelGGL((table_join_kernel<DT, W, CHUNK, 8>), dim3((unsigned)(s.chunks - 1), (unsigned)((s.dim + 64 * W - 1) / (64 * W))), dim3(512), 0, st, s);
}
template <int DT>
void sum_dispatch(const Sum& s, bool wide, hipStream_t st) {
  if (wide) {
    if (chunk_of(s.n) == 8) sum_launch<DT, 8, 8>(s, st);
    else sum_launch<DT, 8, 32>(s, st);
  } else {
    if (chunk_of(s.n) == 8) sum_launch<DT, 1, 8>(s, st);
    else sum_launch<DT, 1, 32>(s, st);
  }
}

// lanes that share a row: the power of two that covers it with W elements each, 64 at most
int lanes_of(int64_t dim, int W) {
  int lg = 0;
  while (lg < 6 && ((int64_t)W << lg) < dim) ++lg;
  return lg;
}

template <int ITEMS>
void sort_large(const int64_t* ids, int64_t n, int64_t vocab, int64_t padding, int bits, int digits, char* ws, const Layout& l, hipStream_t st) {
  const unsigned blocks = (unsigned)((n + 256 * ITEMS - 1) / (256 * ITEMS));
  int* counts = (int*)(ws + l.counts);
  for (int d = 0; d < digits; ++d) {
    const int64_t* from = d == 0 ? ids : nullptr;
    const int* kin = d == 0 ? nullptr : (const int*)(ws + l.keys[(d ^ digits) & 1]);
    const int* pin = d == 0 ? nullptr : (const int*)(ws + l.places[(d ^ digits) & 1]);
    int* kout = (int*)(ws + l.keys[(d + 1 + digits) & 1]);      // (the last digit's go to the first buffers)
    int* pout = (int*)(ws + l.places[(d + 1 + digits) & 1]);
    hipLaunchKernelGGL(table_count_kernel<ITEMS>, dim3(blocks), dim3(256), 0, st, from, kin, n, vocab, padding, d * bits, bits, counts);
    hipLaunchKernelGGL(table_place_kernel<ITEMS>, dim3(blocks), dim3(256), 0, st, from, kin, pin, n, vocab, padding, d * bits, bits, counts, kout, pout);
  }
}

}  // namespace

extern "C" int pf_embedding_scaled_fwd(const void* table, int dtype, const int64_t* ids, void* out, int64_t n_ids, int64_t dim, int64_t vocab, double scale, void* stream) {
  PF_REQUIRE(n_ids >= 0 && dim > 0 && vocab > 0 && pf_is_float_dtype(dtype), "pf_embedding_scaled_fwd: bad arguments");
  if (n_ids == 0) return PF_OK;
  PF_REQUIRE(table && ids && out, "pf_embedding_scaled_fwd: null pointer");
  PF_REQUIRE(n_ids < (1ll << 31), "pf_embedding_scaled_fwd: too many ids");
  const int size = pf_dtype_size(dtype);
  const bool wide = dim * size % 4 == 0 && pf_aligned(table, 4) && pf_aligned(out, 4);
  const int lg = lanes_of(dim, wide ? 8 : 1);
  const dim3 grid((unsigned)(((n_ids << lg) + 255) / 256));
  hipStream_t st = (hipStream_t)stream;
#define PF_TL(DT) \
  if (wide) hipLaunchKernelGGL((table_lookup_kernel<DT, 8>), grid, dim3(256), 0, st, table, ids, out, n_ids, dim, vocab, (float)scale, lg); \
  else hipLaunchKernelGGL((table_lookup_kernel<DT, 1>), grid, dim3(256), 0, st, table, ids, out, n_ids, dim, vocab, (float)scale, lg);
  if (dtype == PF_F32) { PF_TL(PF_F32) }
  else if (dtype == PF_F16) { PF_TL(PF_F16) }
  else { PF_TL(PF_BF16) }
#undef PF_TL
  PF_CHECK_LAUNCH("pf_embedding_scaled_fwd");
  return PF_OK;
}

extern "C" int64_t pf_embedding_sorted_workspace(int64_t n_ids, int64_t dim) { return n_ids <= 0 || dim <= 0 ? 256 : layout_of(n_ids, dim).bytes; }

extern "C" int pf_embedding_sorted_bwd(const void* dout, int d_dtype, const int64_t* ids, void* dtable, int t_dtype, int64_t n_ids, int64_t dim, int64_t vocab,
                                       int64_t padding_idx, double scale, int accumulate, void* workspace, void* stream) {
  const char* who = "pf_embedding_sorted_bwd";
  PF_REQUIRE(n_ids >= 0 && dim > 0 && vocab > 0 && pf_is_float_dtype(d_dtype) && (t_dtype == d_dtype || t_dtype == PF_F32), "%s: bad arguments", who);
  PF_REQUIRE(padding_idx >= -1 && padding_idx < vocab, "%s: padding_idx must be -1 (none) or a row", who);
  PF_REQUIRE(dtable && workspace && (n_ids == 0 || (dout && ids)), "%s: null pointer", who);
  PF_REQUIRE(n_ids <= (1ll << 27) && vocab < (1ll << 27) - 1 && dim < (1ll << 22), "%s: too many ids, rows or columns", who);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const Layout l = layout_of(n_ids > 0 ? n_ids : 1, dim);
  Sum s = {dout, (const int*)(ws + l.keys[0]), (const int*)(ws + l.places[0]), dtable, (float*)(ws + l.partial), n_ids, dim, vocab,
           (n_ids + chunk_of(n_ids) - 1) / chunk_of(n_ids), (float)scale, 0, t_dtype == PF_F32, accumulate != 0};
  if (n_ids > 0) {
    int need = 1;
    while ((vocab >> need) != 0) ++need;               // bits of the keys 0 .. vocab
    const int digits = (need + 8) / 9, bits = (need + digits - 1) / digits;
    if (n_ids <= SMALL) {
      const size_t lds = (4 * SMALL + 16 * BINS) * sizeof(int);
      const int rc = pf_allow_lds((const void*)table_sort_small_kernel, lds, who);
      if (rc != PF_OK) return rc;
      hipLaunchKernelGGL(table_sort_small_kernel, dim3(1), dim3(1024), lds, st, ids, (int)n_ids, vocab, padding_idx, bits, digits, (int*)(ws + l.keys[0]),
                         (int*)(ws + l.places[0]));
    } else if (items_of(n_ids) == 8) {
      sort_large<8>(ids, n_ids, vocab, padding_idx, bits, digits, ws, l, st);
    } else {
      sort_large<16>(ids, n_ids, vocab, padding_idx, bits, digits, ws, l, st);
    }
  }
  const int size = pf_dtype_size(d_dtype);
  const bool wide = dim * size % 4 == 0 && pf_aligned(dout, 4) && pf_aligned(dtable, 4);
  s.lg = lanes_of(dim, wide ? 8 : 1);
  if (d_dtype == PF_F32) sum_dispatch<PF_F32>(s, wide, st);
  else if (d_dtype == PF_F16) sum_dispatch<PF_F16>(s, wide, st);
  else sum_dispatch<PF_BF16>(s, wide, st);
  PF_CHECK_LAUNCH(who);
  return PF_OK;
}
