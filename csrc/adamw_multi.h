// The argument table of the many-tensor AdamW step, shared by its kernel (adamw_multi.hip) and
// its host side (adamw_multi_ops.cpp).
#pragma once

#include <stdint.h>

constexpr int kAdamBlock = 256;   // elements that share the scales of their 8-bit moments
constexpr int kAdamUnit = 16;     // blocks of one tensor that a workgroup updates
constexpr int kAdamTensors = 48;  // tensors a launch: the table stays under 4 KiB of kernel arguments

struct AdamTensor {
  void* param;       // fp32, or the 16-bit copy of `master`
  float* master;     // fp32 weights of a 16-bit parameter, else null
  void* grad;
  void* m;           // fp32, or e4m3 codes
  void* v;           // fp32 second moment, or e4m3 codes of its root
  float* scales;     // [blocks, 2]: of m, of the root (8-bit moments)
  int64_t n;         // elements
  int64_t blk_base;  // blocks of the call's tensors before this one
  float keep;        // 1 - lr * weight decay
  int vec;           // every pointer allows four elements at once
  int unit_end;      // units of this launch up to and including this tensor
  int pad;
};

struct AdamTable {
  AdamTensor t[kAdamTensors];
};

struct AdamScalars {
  const float* clip;  // factor of every gradient, on the device; null: one
  float lr, b1, c1, b2, c2, eps, inv_bc1, inv_sbc2;
  uint32_t key;       // of the step's rounding offsets
  int write_grads;    // leave the gradients multiplied by the clip factor
};
