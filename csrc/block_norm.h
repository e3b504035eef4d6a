// Norms around a block's gated residual (block_norm_fwd.hip, block_norm_bwd.hip): arguments, and
// what both directions share.
//
//   u = norm_post(h) w1 + b1 (or h),  s = residual + scale gate u,  y = norm_pre(s) w2 + b2
//
// with RMS or layer statistics of each row in fp32.  A row stays in registers, 8 elements a lane,
// spread over as many waves as its width needs (one up to 512 columns, 16 at 8192): few registers
// a lane, so that several rows are in flight on a SIMD, and all of a row's loads before its first
// sum.  Rows of up to 512 columns go four to a workgroup, a wave each, without a barrier.
// VEC = 8 (16-byte accesses) needs widths of a multiple of 8 and 16-byte aligned tensors; others
// are read element by element (VEC = 1), neighbouring lanes at neighbouring columns.
// The weights are combined once a workgroup (p1 = scale gate w1, p0 = scale gate b1), which then
// walks rows with a fixed stride.
#pragma once

#include "block_norm_args.h"
#include "row_io.h"

namespace st {

// a weight, the row type T or fp32 (the same for a whole launch); columns behind the row: 0
template <int VEC, typename T>
ST_DEVICE void ld_weight(const void* w, int f32, int lane, int lanes, int width, float (&f)[8]) {
  if (f32) ld_lane<VEC>((const float*)w, lane, lanes, width, f);
  else ld_lane<VEC>((const T*)w, lane, lanes, width, f);
}
template <typename T>
ST_DEVICE float ld_one(const void* w, int f32, int64_t i) {
  float f[1];
  if (f32) ld_row<1>((const float*)w + i, f);
  else ld_row<1>((const T*)w + i, f);
  return f[0];
}

// What a lane keeps of the weights for all its rows: p1 = scale gate w1 (w1 absent: 1), p0 = scale
// gate b1, w2, b2.
template <int VEC, typename T, bool BIAS>
ST_DEVICE void ld_weights(const NormArgs& a, int lane, int lanes, float (&p1)[8], float (&p0)[8], float (&w2)[8],
                          float (&b2)[8]) {
  const float gs = a.scale * (a.gate_n == 1 ? ld_one<T>(a.gate, a.w32, 0) : 1.f);
  float g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    g[i] = gs;
    p1[i] = 1.f;
    p0[i] = w2[i] = b2[i] = 0.f;
  }
  if (a.gate_n > 1) {
    ld_weight<VEC, T>(a.gate, a.w32, lane, lanes, a.width, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= gs;
  }
  if (a.w1) ld_weight<VEC, T>(a.w1, a.w32, lane, lanes, a.width, p1);
  if (BIAS && a.b1) ld_weight<VEC, T>(a.b1, a.w32, lane, lanes, a.width, p0);
  if (a.w2) ld_weight<VEC, T>(a.w2, a.w32, lane, lanes, a.width, w2);
  if (BIAS && a.b2) ld_weight<VEC, T>(a.b2, a.w32, lane, lanes, a.width, b2);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p1[i] *= g[i];
    if (BIAS) p0[i] *= g[i];
  }
}

// Sums over a row's lanes: its wave's, or, where several waves share the row, through LDS.  The
// sums take two buffers in turn, so that one barrier each is enough: who writes a buffer again has
// passed the barrier of the sum between, which every wave reaches after reading this one.
template <bool ONE>
struct RowSum {
  float2* red;  // [2][kNormWaves]
  int turn = 0;
  ST_DEVICE float2 two(float a, float b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (!ONE) {
      const int waves = blockDim.x >> 6;
      float2* r = red + turn * kNormWaves;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
      for (int i = 0; i < waves; ++i) {
        a += r[i].x;
        b += r[i].y;
      }
    }
    return make_float2(a, b);
  }
  ST_DEVICE float one(float a) { return two(a, 0.f).x; }
};

}  // namespace st
