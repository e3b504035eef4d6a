// Arguments of the norms around a block's gated residual: shared by the kernels (block_norm_*.hip)
// and their host side (block_norm_ops.cpp).
#pragma once

#include <stdint.h>

namespace st {

constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;
constexpr int kNormMaxWidth = 8192, kNormWaves = kNormMaxWidth / 512;

struct NormArgs {
  // forward: inputs; backward: what it recomputes the forward from
  const void* h;
  const void* res;      // null: no residual
  const void* gate;     // null, one value or one a column
  const void *w1, *b1;  // norm after the block; null w1: none
  const void *w2, *b2;  // norm before the next; null w2: none
  void* y;
  void* s;              // the new stream; backward: saved, in place of h and res (plain pre-norm)
  float* stats;         // [rows, 4]: mean, 1/std of h, mean, 1/std of s; null: not kept
  // backward
  const void *dy, *ds;  // null: zero
  void *dh, *dres;      // null: not wanted
  float* partial;       // column sums [blocks, arrays, width]; from the host: the workspace that holds them
  int64_t rows;
  int width;
  int layer;            // 0 RMS, 1 layer norm
  int gate_n;           // 0, 1 or width
  int w32;              // gate and weights are fp32, else of h's type
  float scale, eps;
};

}  // namespace st
