// What the kernels of the head's cross entropy are given.
#pragma once

#include "slab_gemm.h"

namespace mm {
namespace xent {

struct Loss {
  // given
  const void *x, *weight, *targets;
  int64_t rows, dim, vocab, x_ld, w_ld;   // elements
  int64_t ignore, dloss_stride;
  int32_t targets64, dtype, reduction;    // 0 none, 1 mean, 2 sum
  float* loss;
  float* lse;                             // (rows,)
  const float* dloss;
  void *dx, *dweight;
  // workspace
  int32_t* at;            // (rows,) a row's place among those that count, -1 for an ignored one
  int32_t* row;           // the row of each place
  int32_t* count;         // [0] how many count
  float* scalars;         // [0] what the sums of the pieces are multiplied by
  float* weights;         // by place: what multiplies a row's gradient, and
  float* lse_at;          // its lse
  int64_t* target_at;     // and target
  char* xc;               // rows that count, (rows, ld) with zeros behind dim
  char* wc;               // the weight laid out the same, where its rows are not aligned
  int64_t ld;             // bytes of their rows
  float* stats;           // (rows, tiles, 2): maximum and sum of exponentials of a tile of the vocabulary
  float* hit;             // by place: the target's logit
  float* row_loss;        // (rows,), where the loss is one number
  char* piece;            // dl of a piece of the vocabulary, (rows, piece_ld bytes)
  float* dx_part;         // (splits, rows, dim) sums of dx
  int64_t piece_ld, piece0, piece_n;      // bytes; this piece's tokens
  int64_t tiles, splits, split_k;         // of the vocabulary in stats; of dx's sums over a piece, and a split's tokens
  int32_t first_piece;
  uint32_t dx_tiles;                      // workgroups of dx, before dW's
  float* logit_part;      // (logit_splits, rows, logit_ld), where few tiles of logits are cut along their sums
  int64_t logit_splits, logit_k, logit_ld;
};

}  // namespace xent
}  // namespace mm
