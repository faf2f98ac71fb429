// Token table: lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale W[id_i];   dW[v] = scale * sum of dout_i over the i with id_i = v, in 32 bits, rounded once
//
// Text holds few tokens very often and most of the table not at all, so the gradient's work is dealt out by the tokens and not by
// the table's rows: the places are sorted by token (up to MANY by counting what is smaller, beyond by a stable radix sort of two or three
// digits), a group of lanes adds up CHUNK neighbours of the sorted list, and a token whose run crosses chunks has its partial sums added
// in order by two last kernels.  Which lane adds what follows from the ids alone: the same ids give the same bits.
#include "pf_common.h"

namespace {

constexpr int BINS = 512;        // of one digit
constexpr int FEW_IDS = 256;     // ids that every workgroup looks through by itself
constexpr int PLACE_BITS = 11;
constexpr int BLOCK = 1 << PLACE_BITS;      // ids that are sorted among themselves first, key and place in one word
// ids up to which that is no slower than the radix sort (us of both sorts with sums of 256 columns: 1000 ids 20 / 39, 16384 30 / 49, 65536 56 / 63, 131072
// 92 / 80, 262144 213 / 92)
constexpr int MANY = 65536;

__device__ __forceinline__ int key_of(int64_t id, int64_t vocab, int64_t padding) { return id >= 0 && id < vocab && id != padding ? (int)id : (int)vocab; }

// One digit's stable ranks among the keys of a wavefront, which counts in `wc` (its own, zero before its first key): how many of the
// digit came before this lane's.  No atomics: a token that fills half of the list would queue all lanes at one counter.
template <typename C>
__device__ __forceinline__ int rank_of(int digit, bool active, int bits, C* wc) {
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
  const int before = __popcll(same & ((1ull << lane) - 1));
  if (active && before == 0) wc[digit] = (C)(at + __popcll(same));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return at + before;
}

// the sum of the values of the threads before this one, in workgroups of WAVES wavefronts
template <int WAVES>
__device__ __forceinline__ int sum_before(int v, int* sm) {
  const int t = threadIdx.x, lane = t & 63;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) sm[t >> 6] = x;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) before += w < (t >> 6) ? sm[w] : 0;
  __syncthreads();
  return before + x - v;
}

// Zeros to the whole of the table's gradient, by workgroups that would otherwise wait for the sort: what the sums write later
// they write over.  (Only the rows that no token names would be fewer bytes, but they are known when the sort is done.  16384 ids, 32000 x
// 2048, bf16: ranks and 131 MB of zeros take 20 us together, of which the ranks alone are 12.)
struct Zero { uint32_t* p; int64_t words, odd; };      // odd: a 16-bit value before / behind them, bits 0 and 1
__device__ __forceinline__ void zero_part(const Zero& z, int64_t block, int64_t blocks, int threads) {
  typedef uint32_t u4_t __attribute__((ext_vector_type(4), aligned(4)));
  const u4_t none = {0, 0, 0, 0};
  const int64_t n = z.words / 4;
  for (int64_t i = block * threads + threadIdx.x; i < n; i += blocks * threads) ((u4_t*)z.p)[i] = none;
  if (block == 0 && threadIdx.x < (z.words & 3)) z.p[n * 4 + threadIdx.x] = 0;
  if (block == 0 && threadIdx.x == 0 && (z.odd & 1)) ((uint16_t*)z.p)[-1] = 0;
  if (block == 0 && threadIdx.x == 0 && (z.odd & 2)) *(uint16_t*)(z.p + z.words) = 0;
}

// Up to MANY ids.  First BLOCK neighbours among themselves, by counting: a word's rank is the number of words below it (no two
// are alike), found by 16 wavefronts that each compare 64 of them with an eighth of a thousand.  2048 compares an id, but spread over
// the whole chip and without a dependence between them (50021 ids: 12 us).  The other workgroups write zeros.
__global__ __launch_bounds__(1024) void table_rank_kernel(const int64_t* ids, int n, int64_t vocab, int64_t padding, uint32_t* words, int* keys, int* places, int groups,
                                                          const Zero zero) {
  __shared__ __align__(16) uint32_t w[BLOCK];
  __shared__ int parts[16][64];
  if ((int)blockIdx.x >= groups) {
    zero_part(zero, (int)blockIdx.x - groups, (int)gridDim.x - groups, 1024);
    return;
  }
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int base = (int)blockIdx.x * 64 / BLOCK * BLOCK, mine = (int)blockIdx.x * 64 % BLOCK + lane;
#pragma unroll
  for (int i = 0; i < BLOCK / 1024; ++i) {
    const int at = base + i * 1024 + t;
    w[i * 1024 + t] = at < n ? (uint32_t)key_of(ids[at], vocab, padding) << PLACE_BITS | (uint32_t)(i * 1024 + t) : ~0u;
  }
  __syncthreads();
  const uint32_t word = w[mine];
  int below = 0;
#pragma unroll 8
  for (int j = wave * (BLOCK / 16); j < (wave + 1) * (BLOCK / 16); j += 4) {
    const uint4 o = *(const uint4*)(w + j);
    below += (o.x < word) + (o.y < word) + (o.z < word) + (o.w < word);
  }
  parts[wave][lane] = below;
  __syncthreads();
  if (wave > 0 || base + mine >= n) return;
  int rank = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) rank += parts[k][lane];
  if (n <= BLOCK) {
    keys[rank] = (int)(word >> PLACE_BITS);
    places[rank] = (int)(word & (BLOCK - 1));
  } else {
    words[base + rank] = word;
  }
}

// Then every sorted block's words to their places among all: as many as in each block before are not above it, in each behind below
// it.  Eight blocks at a time lie in LDS, and a thread's eight searches in them run side by side: 16384 ids 5.7 us, 50021 16.  (In
// memory a search's twelve steps are twelve round trips: 17 us and 57; in LDS with a branch at each step 9.6 and 28.)
__global__ __launch_bounds__(256) void table_merge_kernel(const uint32_t* words, int n, int* keys, int* places) {
  extern __shared__ __align__(16) uint32_t w[];      // [8][BLOCK]
  const int t = threadIdx.x, i = (int)blockIdx.x * 256 + t;
  const uint32_t word = i < n ? words[i] : 0;
  const int key = (int)(word >> PLACE_BITS), own = i / BLOCK, blocks = (n + BLOCK - 1) / BLOCK;
  int rank = i % BLOCK;
  for (int b0 = 0; b0 < blocks; b0 += 8) {
    uint4 v[8 * BLOCK / 1024];
#pragma unroll
    for (int k = 0; k < 8 * BLOCK / 1024; ++k) {
      const int at = b0 * BLOCK + (k * 256 + t) * 4;      // (what lies behind the last word is not looked at)
      v[k] = at < n ? *(const uint4*)(words + at) : make_uint4(~0u, ~0u, ~0u, ~0u);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8 * BLOCK / 1024; ++k) *(uint4*)(w + (k * 256 + t) * 4) = v[k];
    __syncthreads();
    int pos[8], size[8], limit[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      pos[q] = 0;
      const int left = n - (b0 + q) * BLOCK;
      size[q] = left < 0 ? 0 : left < BLOCK ? left : BLOCK;
      limit[q] = b0 + q < own ? key + 1 : key;
    }
#pragma unroll
    for (int step = BLOCK / 2; step > 0; step >>= 1) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {      // (no branch: eight reads on their way, not one)
        const int to = pos[q] + step, at = (int)(w[q * BLOCK + to - 1] >> PLACE_BITS);
        pos[q] = ((to <= size[q]) & (at < limit[q])) ? to : pos[q];
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int at = (int)(w[q * BLOCK + (pos[q] < BLOCK ? pos[q] : BLOCK - 1)] >> PLACE_BITS);
      pos[q] += (pos[q] < size[q]) & (at < limit[q]);      // (all of a block)
      if (b0 + q != own) rank += pos[q];
    }
  }
  if (i < n) {
    keys[rank] = key;
    places[rank] = own * BLOCK + (int)(word & (BLOCK - 1));
  }
}

// How often each value of a digit occurs among a block's keys
template <int ITEMS>
__global__ __launch_bounds__(256) void table_count_kernel(const int64_t* ids, const int* keys, int64_t n, int64_t vocab, int64_t padding, int shift, int bits, int* counts,
                                                          int blocks, const Zero zero) {
  __shared__ int wc[4][BINS];
  if ((int)blockIdx.x >= blocks) {
    zero_part(zero, (int)blockIdx.x - blocks, (int)gridDim.x - blocks, 256);
    return;
  }
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = t; i < 4 * BINS; i += 256) (&wc[0][0])[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * ITEMS + wave * 64 * ITEMS;
  int key[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * 64 + lane;
    key[i] = at >= n ? 0 : ids != nullptr ? key_of(ids[at], vocab, padding) : keys[at];
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) rank_of((key[i] >> shift) & ((1 << bits) - 1), base + i * 64 + lane < n, bits, wc[wave]);
  __syncthreads();
  for (int i = t; i < BINS; i += 256) counts[(int64_t)blockIdx.x * BINS + i] = wc[0][i] + wc[1][i] + wc[2][i] + wc[3][i];
}

// ... and the keys to their places.  A block finds out from all blocks' counts where its own begin.
template <int ITEMS>
__global__ __launch_bounds__(256) void table_place_kernel(const int64_t* ids, const int* keys, const int* places, int64_t n, int64_t vocab, int64_t padding, int shift,
                                                          int bits, const int* counts, int* keys_out, int* places_out) {
  __shared__ int wc[4][BINS];
  __shared__ int sm[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, mask = (1 << bits) - 1;
  for (int i = t; i < 4 * BINS; i += 256) (&wc[0][0])[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * ITEMS + wave * 64 * ITEMS;
  int key[ITEMS], rank[ITEMS], place[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * 64 + lane;
    key[i] = at >= n ? 0 : ids != nullptr ? key_of(ids[at], vocab, padding) : keys[at];
    place[i] = at >= n || places == nullptr ? (int)at : places[at];
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) rank[i] = rank_of((key[i] >> shift) & mask, base + i * 64 + lane < n, bits, wc[wave]);
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
  const int before = sum_before<4>(all[0] + all[1], sm);      // (its barriers: all wavefronts have counted)
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
    if (at >= n) continue;
    const int to = wc[wave][(key[i] >> shift) & mask] + rank[i];
    keys_out[to] = key[i];
    places_out[to] = place[i];
  }
}

constexpr int W = 8;      // neighbouring elements of a lane

// `left` of them inside the row, wherever that begins: 16 bytes at a time need no more than the element's own alignment
// (What is left of a row is converted behind the branch with 16 bits, inside it with 32: the other way about 16384 x 2048 in bf16 are
// summed in 35 us instead of 29, and 50021 x 769 in fp32 looked up in 57 instead of 47.)
typedef uint32_t four_t __attribute__((ext_vector_type(4), aligned(4)));
template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t i, int64_t left, float (&v)[W]) {
  typedef typename Codec<DT>::storage S;
  const S* from = (const S*)p + i;
  if constexpr (DT == PF_F32) {
    if (left >= W) {
      const four_t a = *(const four_t*)from, b = *(const four_t*)(from + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[k] = __uint_as_float(a[k]); v[4 + k] = __uint_as_float(b[k]); }
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = k < left ? from[k] : 0.f;
    }
  } else {
    uint4 a;
    if (left >= W) {
      __builtin_memcpy(&a, from, sizeof(a));
    } else {
      S e[W];
#pragma unroll
      for (int k = 0; k < W; ++k) e[k] = k < left ? from[k] : (S)0;
      __builtin_memcpy(&a, e, sizeof(a));
    }
    Vec8<DT>::load(&a, 0, v);
  }
}
template <int DT> __device__ __forceinline__ void store8(void* p, int64_t i, int64_t left, const float (&v)[W]) {
  if (left >= W) {
    if constexpr (DT == PF_F32) {
      four_t a, b;
#pragma unroll
      for (int k = 0; k < 4; ++k) { a[k] = __float_as_uint(v[k]); b[k] = __float_as_uint(v[4 + k]); }
      *(four_t*)((float*)p + i) = a;
      *(four_t*)((float*)p + i + 4) = b;
    } else {
      uint4 a;
      Vec8<DT>::store(&a, 0, v);
      __builtin_memcpy((uint16_t*)p + i, &a, sizeof(a));
    }
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (k < left) Codec<DT>::store(p, i + k, v[k]);
  }
}

// out[i] = scale * W[ids[i]]; a group of 2^lg lanes takes a row.  Bound by memory: 16384 x 2048, bf16: 27 us, 97 MB
template <int DT>
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
    if (ok) load8<DT>(table, id * dim + c, dim - c, v);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] *= scale;
    store8<DT>(out, i * dim + c, dim - c, v);
  }
}

struct Sum {
  const void* dout;
  const int* keys;
  const int* places;
  void* dtable;
  float* partial;      // [chunks][2][dim]: of a run that comes from the chunk before, of one that goes on into the next
  float* blocks;       // [chunks / FEW][dim]
  int64_t n, dim, vocab, chunks;
  float scale;
  int lg, t_f32, accumulate;
};

template <int DT>
__device__ __forceinline__ void put_row(const Sum& s, int64_t row, int64_t c, float (&v)[W]) {
  const int64_t left = s.dim - c, at = row * s.dim + c;
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] *= s.scale;
  if (s.accumulate) {
    float old[W];
    if (s.t_f32) load8<PF_F32>(s.dtable, at, left, old);
    else load8<DT>(s.dtable, at, left, old);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] += old[k];
  }
  if (s.t_f32) store8<PF_F32>(s.dtable, at, left, v);
  else store8<DT>(s.dtable, at, left, v);
}

// Up to FEW_IDS ids, in one launch: a workgroup owns `own` rows of the table's gradient, writes zeros to them, finds the ids that name
// one of them and adds up in the list's order, wide rows by its wavefronts side by side, else a wavefront to a row.  (The sort takes two launches
// more: 16 ids, 32000 x 2048, bf16: 24 us, most of them for the zeros, against 31.)
template <int DT>
__global__ __launch_bounds__(256) void table_few_kernel(const Sum s, const int64_t* ids, int64_t padding, int64_t own) {
  __shared__ int rows[FEW_IDS], at[FEW_IDS];
  __shared__ int before[5];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t v0 = (int64_t)blockIdx.x * own, v1 = v0 + own < s.vocab ? v0 + own : s.vocab;
  const int64_t id = t < s.n ? ids[t] : -1;
  if (!s.accumulate) {
    float zero[W];
#pragma unroll
    for (int k = 0; k < W; ++k) zero[k] = 0.f;
    const int64_t end = v1 * s.dim;
    for (int64_t i = v0 * s.dim + (int64_t)t * W; i < end; i += 256 * W) {
      if (s.t_f32) store8<PF_F32>(s.dtable, i, end - i, zero);
      else store8<DT>(s.dtable, i, end - i, zero);
    }
  }
  const bool hit = id >= v0 && id < v1 && id != padding;
  const unsigned long long mask = __ballot(hit);
  if (lane == 0) before[wave + 1] = __popcll(mask);
  __syncthreads();
  int first = 0;
  for (int w = 0; w < wave; ++w) first += before[w + 1];
  if (hit) {
    const int j = first + __popcll(mask & ((1ull << lane) - 1));
    rows[j] = (int)(id - v0);
    at[j] = t;
  }
  const int hits = before[1] + before[2] + before[3] + before[4];
  __syncthreads();      // (and the zeros are written)
  const int across = s.dim > 64 * W ? (s.dim > 2 * 64 * W ? 4 : 2) : 1;      // wavefronts to a row
  for (int j = wave / across; j < hits; j += 4 / across) {
    const int row = rows[j];
    bool earlier = false;
    for (int q = lane; q < j; q += 64) earlier |= rows[q] == row;
    if (__ballot(earlier) != 0) continue;
    for (int64_t c0 = wave % across * 64 * W; c0 < s.dim; c0 += across * 64 * W) {      // (no lane leaves before the others)
      const int64_t c = c0 + lane * W, left = s.dim - c;
      float acc[W];
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] = 0.f;
      for (int q0 = j & ~63; q0 < hits; q0 += 64) {
        const int q = q0 + lane;
        const int place = q < hits ? at[q] : 0;
        unsigned long long mine = __ballot(q < hits && rows[q < hits ? q : 0] == row);
        while (mine != 0) {      // the next eight of the row
          int n = 0, from[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            from[k] = mine != 0 ? __builtin_amdgcn_readlane(place, __ffsll((long long)mine) - 1) : 0;
            n += mine != 0;
            mine &= mine - 1;
          }
          float v[8][W];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < n) load8<DT>(s.dout, (int64_t)from[k] * s.dim + c, left, v[k]);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < n) {
#pragma unroll
              for (int e = 0; e < W; ++e) acc[e] += v[k][e];
            }
        }
      }
      put_row<DT>(s, v0 + row, c, acc);
    }
  }
}

// A group of lanes adds up one chunk of the sorted list in one slice of the columns; runs that end inside it go to the table's
// gradient, the others' parts to `partial`.  Bound by memory, and by the places' loads before dout's: 16384 x 2048, bf16: 29 us, 82 MB
template <int DT, int CHUNK>
__global__ __launch_bounds__(256) void table_sum_kernel(const Sum s) {
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
      store8<PF_F32>(to, c, left, acc);
    } else {
      put_row<DT>(s, run, c, acc);
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
      load8<DT>(s.dout, (int64_t)s.places[j] * s.dim + c, left, v[q]);
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

// Runs that cross chunks.  FEW neighbours from a multiple of FEW on are a block of chunks.  What is moved is small, each of the two
// launches waits for a few round trips: 7 us each at 16384 ids; 50021 with one of them a third of the list: 12 and 9 (50 without the
// blocks' sums).
constexpr int FEW = 64;

// The first `waves` wavefronts of each slice, one to a chunk: a run that begins in it and goes on over less than FEW others, their parts in the
// list's order.  The others, four to a block of chunks: where it lies inside one run, its parts' sum.
template <int DT, int CHUNK>
__global__ __launch_bounds__(256) void table_join_kernel(const Sum s, int joins) {
  __shared__ float part[4][64 * W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.y * 64 * W + lane * W, left = s.dim - c;
  float acc[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = 0.f;
  if ((int)blockIdx.x >= joins) {
    const int64_t block = (int)blockIdx.x - joins, first = block * FEW;
    const int64_t end = (first + FEW - 1) * CHUNK;
    if (first == 0 || end >= s.n) return;
    const int run = s.keys[end], before = s.keys[first * CHUNK - 1];
    if (run >= s.vocab || before != run) return;
    if (left > 0) {
#pragma unroll
      for (int p = 0; p < FEW / 4; ++p) {
        float v[W];
        load8<PF_F32>(s.partial + (first + wave * (FEW / 4) + p) * 2 * s.dim, c, left, v);
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] += v[k];
      }
    }
#pragma unroll
    for (int k = 0; k < W; ++k) part[wave][lane * W + k] = acc[k];
    __syncthreads();
    if (wave > 0 || left <= 0) return;
    for (int w = 1; w < 4; ++w) {
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += part[w][lane * W + k];
    }
    store8<PF_F32>(s.blocks + block * s.dim, c, left, acc);
    return;
  }
  const int64_t chunk = (int64_t)blockIdx.x * 4 + wave, next = (chunk + 1) * CHUNK;
  if (next >= s.n) return;
  // (all that decides on the way at once)
  const int64_t mine = next + (int64_t)lane * CHUNK;
  const int run = s.keys[next - 1], after = s.keys[next], first = s.keys[chunk * CHUNK], before = s.keys[chunk > 0 ? chunk * CHUNK - 1 : 0];
  const int there = s.keys[mine < s.n ? mine : s.n - 1];
  if (run >= s.vocab || after != run || (first == run && chunk > 0 && before == run)) return;      // (nothing goes on, or it began before)
  const unsigned long long on = __ballot(mine < s.n && there == run);
  if (on == ~0ull || left <= 0) return;                                                            // (of more chunks: below)
  const int many = __ffsll((long long)~on) - 1;      // chunks that begin with the run
  load8<PF_F32>(s.partial + (chunk * 2 + 1) * s.dim, c, left, acc);
#pragma unroll 4
  for (int p = 1; p <= many; ++p) {
    float v[W];
    load8<PF_F32>(s.partial + (chunk + p) * 2 * s.dim, c, left, v);
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k] += v[k];
  }
  put_row<DT>(s, run, c, acc);
}

// The smallest i in [lo, hi] with f(i), hi if there is none below it, f being false first and then true; a wavefront looks at 64 at a time
template <class F>
__device__ __forceinline__ int64_t wave_find(int64_t lo, int64_t hi, F f) {
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + (threadIdx.x & 63) * step;
    const unsigned long long yes = __ballot(at >= hi || f(at));
    const int k = yes != 0 ? __ffsll((long long)yes) - 1 : 64;
    const int64_t top = lo + k * step;
    lo = k > 0 ? lo + (k - 1) * step + 1 : lo;
    hi = top < hi ? top : hi;
  }
  return hi;
}

// Longer runs: each holds the first entry of a block of chunks.  The workgroup of the first such block finds the run's ends; its 16
// wavefronts each add a share of the parts, in the list's order: chunks up to a block, whole blocks, chunks after them.
template <int DT, int CHUNK>
__global__ __launch_bounds__(1024) void table_join_long_kernel(const Sum s) {
  __shared__ float part[16][64 * W];
  const int64_t mark = ((int64_t)blockIdx.x + 1) * FEW;
  const int lane = threadIdx.x & 63, team = threadIdx.x >> 6;
  if (mark >= s.chunks) return;
  const int run = s.keys[mark * CHUNK], before = s.keys[mark * CHUNK - 1];
  const int last = s.keys[(mark - FEW) * CHUNK], last_before = s.keys[mark > FEW ? (mark - FEW) * CHUNK - 1 : 0];
  if (run >= s.vocab || before != run || (mark > FEW && last == run && last_before == run)) return;      // (or a block before this one's)
  const int64_t first = wave_find(0, mark * CHUNK, [&](int64_t j) { return s.keys[j] >= run; }) / CHUNK;
  const int64_t lo = wave_find(mark + 1, s.chunks, [&](int64_t m) { return s.keys[m * CHUNK] > run; }) - 1;      // the last chunk that begins with it
  if (lo - first < FEW) return;
  const int64_t blocks = (lo + 1 - mark) / FEW, head = mark - first, rest = lo + 1 - mark - blocks * FEW, many = head + blocks + rest;
  const int64_t c = (int64_t)blockIdx.y * 64 * W + lane * W, left = s.dim - c;
  const int64_t per = (many + 15) / 16, a = team * per, b = a + per < many ? a + per : many;
  float acc[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = 0.f;
  if (left > 0) {
#pragma unroll 8
    for (int64_t p = a; p < b; ++p) {
      const float* from = p == 0 ? s.partial + (first * 2 + 1) * s.dim
                          : p < head ? s.partial + (first + p) * 2 * s.dim
                          : p < head + blocks ? s.blocks + (mark / FEW + p - head) * s.dim : s.partial + (mark + blocks * FEW + p - head - blocks) * 2 * s.dim;
      float v[W];
      load8<PF_F32>(from, c, left, v);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += v[k];
    }
  }
#pragma unroll
  for (int k = 0; k < W; ++k) part[team][lane * W + k] = acc[k];
  __syncthreads();
  if (team > 0 || left <= 0) return;
  for (int w = 1; w < 16 && w * per < many; ++w) {
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k] += part[w][lane * W + k];
  }
  put_row<DT>(s, run, c, acc);
}

inline int64_t round_up(int64_t n, int64_t k) { return (n + k - 1) / k * k; }
// Neighbours that a group of lanes adds up.  Few make more groups and more parts.  us of a gradient with 8 / 32, uniform ids, 32000 rows, bf16: 16384 x 128
// 28 / 36, 16384 x 2048 59 / 59, 65536 x 512 66 / 65, 131072 x 1024 189 / 160, 262144 x 2048 559 / 405
inline int chunk_of(int64_t n, int64_t dim) { return n * dim <= (1 << 25) ? 8 : 32; }
// Keys of a thread of the radix sort: 70000 ids 61 us with 8, 78 with 16, 262144 86 / 98, 1048576 169 / 155
inline int items_of(int64_t n) { return n <= (1 << 19) ? 8 : 16; }

struct Layout { int64_t keys[2], places[2], counts, partial, blocks, bytes; };
Layout layout_of(int64_t n, int64_t dim) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t p = at; at += round_up(bytes, 256); return p; };
  for (int k = 0; k < 2; ++k) { l.keys[k] = take(n * 4); l.places[k] = take(n * 4); }
  l.counts = take((n + 256 * items_of(n) - 1) / (256 * items_of(n)) * BINS * 4);
  l.partial = take((n + chunk_of(n, dim) - 1) / chunk_of(n, dim) * 2 * dim * 4);
  l.blocks = take((n + chunk_of(n, dim) - 1) / chunk_of(n, dim) / FEW * dim * 4);
  l.bytes = at;
  return l;
}

template <int DT, int CHUNK>
void sum_launch(const Sum& s, hipStream_t st) {
  const int64_t slices = (s.dim + ((int64_t)W << s.lg) - 1) / ((int64_t)W << s.lg);
  const int64_t sums = (s.chunks * slices + (256 >> s.lg) - 1) / (256 >> s.lg);
  hipLaunchKernelGGL((table_sum_kernel<DT, CHUNK>), dim3((unsigned)sums), dim3(256), 0, st, s);
  if (s.chunks < 2) return;
  const unsigned slices64 = (unsigned)((s.dim + 64 * W - 1) / (64 * W));
  const int64_t joins = (s.chunks + 3) / 4, blocks = s.chunks / FEW;
  hipLaunchKernelGGL((table_join_kernel<DT, CHUNK>), dim3((unsigned)(joins + blocks), slices64), dim3(256), 0, st, s, (int)joins);
  if (blocks > 0) hipLaunchKernelGGL((table_join_long_kernel<DT, CHUNK>), dim3((unsigned)blocks, slices64), dim3(1024), 0, st, s);
}
template <int DT>
void sum_dispatch(const Sum& s, hipStream_t st) {
  if (chunk_of(s.n, s.dim) == 8) sum_launch<DT, 8>(s, st);
  else sum_launch<DT, 32>(s, st);
}

// lanes that share a row: the power of two that covers it with W elements each, 64 at most
int lanes_of(int64_t dim) {
  int lg = 0;
  while (lg < 6 && ((int64_t)W << lg) < dim) ++lg;
  return lg;
}

template <int ITEMS>
void sort_large(const int64_t* ids, int64_t n, int64_t vocab, int64_t padding, int bits, int digits, char* ws, const Layout& l, const Zero& zero,
                int zero_blocks, hipStream_t st) {
  const unsigned blocks = (unsigned)((n + 256 * ITEMS - 1) / (256 * ITEMS));
  int* counts = (int*)(ws + l.counts);
  for (int d = 0; d < digits; ++d) {
    const int64_t* from = d == 0 ? ids : nullptr;
    const int* kin = d == 0 ? nullptr : (const int*)(ws + l.keys[(d ^ digits) & 1]);
    const int* pin = d == 0 ? nullptr : (const int*)(ws + l.places[(d ^ digits) & 1]);
    int* kout = (int*)(ws + l.keys[(d + 1 + digits) & 1]);      // (the last digit's go to the first buffers)
    int* pout = (int*)(ws + l.places[(d + 1 + digits) & 1]);
    hipLaunchKernelGGL(table_count_kernel<ITEMS>, dim3(blocks + (d == 0 ? (unsigned)zero_blocks : 0u)), dim3(256), 0, st, from, kin, n, vocab, padding, d * bits, bits,
                       counts, (int)blocks, zero);
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
  const int lg = lanes_of(dim);
  hipStream_t st = (hipStream_t)stream;
  constexpr int64_t MOST = 1ll << 25;      // ids of a launch, 2^31 threads at most
  for (int64_t i0 = 0; i0 < n_ids; i0 += MOST) {
    const int64_t n = n_ids - i0 < MOST ? n_ids - i0 : MOST;
    const int64_t* from = ids + i0;
    void* to = (char*)out + i0 * dim * size;
    const dim3 grid((unsigned)(((n << lg) + 255) / 256));
#define PF_TL(DT) \
    hipLaunchKernelGGL(table_lookup_kernel<DT>, grid, dim3(256), 0, st, table, from, to, n, dim, vocab, (float)scale, lg)
    if (dtype == PF_F32) PF_TL(PF_F32);
    else if (dtype == PF_F16) PF_TL(PF_F16);
    else PF_TL(PF_BF16);
#undef PF_TL
    PF_CHECK_LAUNCH("pf_embedding_scaled_fwd");
  }
  return PF_OK;
}

extern "C" int64_t pf_embedding_sorted_workspace(int64_t n_ids, int64_t dim) { return n_ids <= FEW_IDS || dim <= 0 ? 0 : layout_of(n_ids, dim).bytes; }

extern "C" int pf_embedding_sorted_bwd(const void* dout, int d_dtype, const int64_t* ids, void* dtable, int t_dtype, int64_t n_ids, int64_t dim, int64_t vocab,
                                       int64_t padding_idx, double scale, int accumulate, void* workspace, void* stream) {
  const char* who = "pf_embedding_sorted_bwd";
  PF_REQUIRE(n_ids >= 0 && dim > 0 && vocab > 0 && pf_is_float_dtype(d_dtype) && (t_dtype == d_dtype || t_dtype == PF_F32), "%s: bad arguments", who);
  PF_REQUIRE(padding_idx >= -1 && padding_idx < vocab, "%s: padding_idx must be -1 (none) or a row", who);
  PF_REQUIRE(dtable && (n_ids <= FEW_IDS || workspace) && (n_ids == 0 || (dout && ids)), "%s: null pointer", who);
  PF_REQUIRE(n_ids <= (1ll << 27) && vocab < (1ll << 27) - 1 && dim <= 65535 * 64, "%s: too many ids, rows or columns", who);
  PF_REQUIRE(pf_aligned(workspace, 16), "%s: the workspace lies on a boundary of 256 bytes", who);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const Layout l = layout_of(n_ids, dim);
  Sum s = {dout, (const int*)(ws + l.keys[0]), (const int*)(ws + l.places[0]), dtable, (float*)(ws + l.partial), (float*)(ws + l.blocks), n_ids, dim, vocab,
           (n_ids + chunk_of(n_ids, dim) - 1) / chunk_of(n_ids, dim), (float)scale, 0, t_dtype == PF_F32, accumulate != 0};
  s.lg = lanes_of(dim);
  if (n_ids <= FEW_IDS) {
    // (64 KB of zeros, and a thousand workgroups: 1000 x 128, bf16, 256 ids 89 us on four of them)
    int64_t own = 65536 / (dim * pf_dtype_size(t_dtype));
    own = own < vocab / 1024 ? own : vocab / 1024;
    own = own < 1 ? 1 : own > 1024 ? 1024 : own;
    const dim3 grid((unsigned)((vocab + own - 1) / own));
#define PF_TF(DT) \
    hipLaunchKernelGGL(table_few_kernel<DT>, grid, dim3(256), 0, st, s, ids, padding_idx, own)
    if (d_dtype == PF_F32) PF_TF(PF_F32);
    else if (d_dtype == PF_F16) PF_TF(PF_F16);
    else PF_TF(PF_BF16);
#undef PF_TF
    PF_CHECK_LAUNCH(who);
    return PF_OK;
  }
  // the gradient's bytes as words, and what is left of a 16-bit one at its ends
  Zero zero = {nullptr, 0, 0};
  int64_t zero_blocks = 0;
  if (!accumulate) {
    const int t_size = pf_dtype_size(t_dtype);
    int64_t bytes = vocab * dim * t_size;
    char* p = (char*)dtable;
    if (t_size == 2 && !pf_aligned(p, 4)) { zero.odd |= 1; p += 2; bytes -= 2; }
    if (bytes & 2) zero.odd |= 2;
    zero.p = (uint32_t*)p;
    zero.words = bytes / 4;
    zero_blocks = (zero.words + 16383) / 16384 < 2048 ? (zero.words + 16383) / 16384 : 2048;
    if (zero_blocks == 0) zero_blocks = 1;
  }
  int need = 1;
  while ((vocab >> need) != 0) ++need;               // bits of the keys 0 .. vocab
  const int digits = (need + 8) / 9, bits = (need + digits - 1) / digits;
  if (n_ids <= MANY && need <= 32 - PLACE_BITS) {
    const int groups = (int)((n_ids + 63) / 64);
    uint32_t* words = (uint32_t*)(ws + l.keys[1]);
    int *keys = (int*)(ws + l.keys[0]), *places = (int*)(ws + l.places[0]);
    if (groups + zero_blocks > 0)
      hipLaunchKernelGGL(table_rank_kernel, dim3((unsigned)(groups + zero_blocks)), dim3(1024), 0, st, ids, (int)n_ids, vocab, padding_idx, words, keys, places, groups, zero);
    if (n_ids > BLOCK)
      hipLaunchKernelGGL(table_merge_kernel, dim3((unsigned)((n_ids + 255) / 256)), dim3(256), 8 * BLOCK * 4, st, words, (int)n_ids, keys, places);
  } else if (items_of(n_ids) == 8) {
    sort_large<8>(ids, n_ids, vocab, padding_idx, bits, digits, ws, l, zero, (int)zero_blocks, st);
  } else {
    sort_large<16>(ids, n_ids, vocab, padding_idx, bits, digits, ws, l, zero, (int)zero_blocks, st);
  }
  PF_CHECK_LAUNCH(who);
  if (d_dtype == PF_F32) sum_dispatch<PF_F32>(s, st);
  else if (d_dtype == PF_F16) sum_dispatch<PF_F16>(s, st);
  else sum_dispatch<PF_BF16>(s, st);
  PF_CHECK_LAUNCH(who);
  return PF_OK;
}
