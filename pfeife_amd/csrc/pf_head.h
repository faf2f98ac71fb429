// The matrix products of the cross entropy from the last hidden state, one object file per 16-bit operand type.
#pragma once
#include "pf_common.h"

// Statistics of 64 x 2^n vocabulary rows for every token: largest logit, sum of exponentials beside it
struct PfHeadPart { float top, sum; };
// What turns a token's logits into their gradient: top, -log2(sum), the factor of the probabilities, that of the label
struct PfHeadColumn { float top, bias, f, g; };

// Rows of one of `splits` shares of a piece, the last one's may be fewer
__host__ __device__ inline int64_t pf_head_share(int64_t rows, int splits) { return splits > 1 ? ((rows + splits - 1) / splits + 63) / 64 * 64 : rows; }
// In how many shares of a piece's vocabulary rows the hidden state's gradient is summed: few tokens make few tiles, and what a round of 256 of
// them leaves over is idle.  by_count: the device decides for the tokens that take part, as many as fill a round of 256x256 tiles,
// `most` of them, and the sums lie [count][depth] behind each other, not [n_max][depth].  So many are all used by the first piece, of `first` rows, and
// by a piece of fewer no more.
struct PfHeadShares {
  int most, by_count;
  int64_t first;
  __host__ __device__ int of(int64_t count, int64_t depth) const {
    int s = most;
    if (by_count) {
      const int64_t tiles = (count + 255) / 256 * ((depth + 255) / 256), fill = tiles > 0 ? 256 / tiles : 1;
      s = fill < 1 ? 1 : fill < most ? (int)fill : most;
    }
    const int64_t share = pf_head_share(first, s);
    return (int)((first + share - 1) / share);
  }
  // bytes that the sums take
  int64_t bytes(int64_t n_max, int64_t depth) const {
    const int64_t one = n_max * depth * 4, round = 256ll * 256 * 256 * 4;      // (more than one share: no more than a round of tiles)
    if (!by_count) return one * most;
    return one > round ? one : one * most < round ? one * most : round;
  }
};

// Products over one piece of the vocabulary (rows `v0` .. `v0 + rows` of the weight).  `count` (in DEVICE memory) tokens take
// part; `hc` holds them as its first rows, followed by rows of zeros up to a multiple of 64 (at least 64), n_max at most.
struct PfHeadProduct {
  const void* w;             // first row of the piece
  int64_t ldw, v0, rows;
  int64_t depth;             // a multiple of 8, at least 64
  const void* hc;
  int64_t ldh, n_max;        // n_max a multiple of 64
  const int* count;
  const int* lab;            // [n_max] label of each token
  PfHeadPart* part;          // [blocks][n_max], see pf_head_blocks
  float* zl;                 // [n_max] the label's logit
  const PfHeadColumn* col;   // [n_max]
  void* dz;                  // [rows][n_max] gradient of the piece's logits
  const void* ht;            // [dim][n_max] the tokens' hidden state, transposed
  int64_t dim;               // columns of dw, the width of its rows a multiple of 8
  int64_t ldw_out;
  void* dw;                  // [rows][ldw_out] in the operands' type, on a boundary of 16 bytes
  float* dh;                 // a sum [n_max][depth] for each share of the piece's rows, accumulated where `add`
  int add;
  PfHeadShares shares;
  const float* unscale;      // both gradients are divided by this
};

// Tile of the logits' product (vocabulary rows x tokens) and the rows of one wavefront's block in it, which leaves one partial statistic.
// us of a forward pass, 2048 columns, 32000 classes, bf16, on 64x64 / 256x128 / 256x256: 64 tokens 39.7 / 42 / -, 128 48 / 43 / -, 256 73 / 48 / 61, 512 123 / 77 / 70
enum { PF_HEAD_64x64, PF_HEAD_256x128, PF_HEAD_256x256 };
inline int pf_head_tile(int64_t n_max, int64_t depth) {
  return n_max <= 64 ? PF_HEAD_64x64 : depth % 64 == 0 && n_max > 256 ? PF_HEAD_256x256 : PF_HEAD_256x128;
}
inline int64_t pf_head_blocks(int64_t rows, int64_t n_max, int64_t depth) {
  switch (pf_head_tile(n_max, depth)) {
    case PF_HEAD_64x64: return (rows + 63) / 64 * 2;
    case PF_HEAD_256x128: return (rows + 255) / 256 * 4;
    default: return (rows + 255) / 256 * 2;
  }
}
int pf_head_stats(int dtype, const PfHeadProduct& p, hipStream_t st);
int pf_head_dz(int dtype, const PfHeadProduct& p, hipStream_t st);
int pf_head_dh(int dtype, const PfHeadProduct& p, hipStream_t st);
int pf_head_dw(int dtype, const PfHeadProduct& p, hipStream_t st);
// us of such sums on 28672 vocabulary rows, 1024 columns, 3163 of 4662 tokens, fp16: two shares 282, three 208 (so many for 4662), four 178
PfHeadShares pf_head_shares(int dtype, int64_t n_max, int64_t depth, int64_t rows);
