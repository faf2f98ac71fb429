// The matrix products of the cross entropy from the last hidden state, one object file per 16-bit operand type.
#pragma once
#include "pf_common.h"

// Statistics of 64 x 2^n vocabulary rows for every token: largest logit, sum of exponentials beside it
struct PfHeadPart { float top, sum; };
// What turns a token's logits into their gradient: top, -log2(sum), the factor of the probabilities, that of the label
struct PfHeadColumn { float top, bias, f, g; };

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
  float* dh;                 // [splits][n_max][depth], accumulated where `add`
  int add, splits;           // the piece's rows in so many shares, a sum for each
  const float* unscale;      // both gradients are divided by this
};

// Tile of the logits' product (vocabulary rows x tokens) and the rows of one wavefront's block in it, which leaves one partial statistic
enum { PF_HEAD_64x64, PF_HEAD_256x128, PF_HEAD_256x256 };
inline int pf_head_tile(int64_t n_max, int64_t depth) {
  return n_max <= 64 ? PF_HEAD_64x64 : depth % 64 == 0 && n_max > 128 ? PF_HEAD_256x256 : PF_HEAD_256x128;
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
// Rows of one of `splits` shares of a piece, the last one's may be fewer
inline int64_t pf_head_share(int64_t rows, int splits) { return splits > 1 ? ((rows + splits - 1) / splits + 63) / 64 * 64 : rows; }
// In how many shares the hidden state's gradient is best summed over `rows` vocabulary rows: few tokens make few tiles, and what a round of
// 256 of them leaves over is idle.  So many are all used, by a piece of fewer rows no more.  (3163 of 4662 tokens, 1024 columns, 28672 rows, fp16:
// two shares 282 us, three 208.)
int pf_head_splits(int dtype, int64_t n_max, int64_t depth, int64_t rows);
