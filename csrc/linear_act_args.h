// Arguments of the matrix products with an epilogue, shared by the kernels (linear_act_*.hip) and
// their host side (linear_act_ops.cpp).
#pragma once

#include <stdint.h>

namespace st {

enum Act : int { kNoAct = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4 };

struct LinearEpi {
  const void* bias;  // 16-bit [N]; null: none
  const void* res;   // [M, N] of the output's type; null: none
  void* out;         // [M, N], rows ldo apart (z and res too)
  void* z;           // 16-bit, what the backward needs; null: not kept
  int64_t ldo;
  int act;
  int out_f32;
  int f16;           // the 16-bit type is fp16, else bf16
};

struct LinearArgs {
  const void *a, *b;  // 16-bit
  int64_t lda, ldb;   // elements between rows (kRow) or between k (kCol)
  int M, N, K;
  int vec;            // 16-byte loads and 4-column stores are aligned and end inside the operands
  float* ws;          // [splits, M, N] partial sums; null: one split
  int splits;
  LinearEpi epi;
};

}  // namespace st
