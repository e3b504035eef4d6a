// Forward of the norms around a block's gated residual (formulas and layouts: block_norm.h).
//
// One pass: a row's h and residual are read once, both norms' statistics are taken from registers
// (mean first, then the squares of what is left: one pass over sums of squares would lose a large
// mean's digits), s and y are written once.  y comes from the unrounded s.  Bound by HBM: three or
// four streams of rows x width; the weights stay in L2.  Measured: 24576 x 4096 bf16, both norms and a
// channel gate, 156 us (5.2 TB/s); 16384 x 1280 LayerNorm with the residual add 36 us (4.6); 3001 x
// 1001 fp32, element by element, 17 us; 8 x 4096 4.6 us, a launch.  The grid of 16384 waves walks
// rows: a quarter of it took 390 us for forward and backward of the first instead of 373 (too few
// loads in flight), four times 381 (the weights are read and combined too often).
#include <algorithm>

#include "block_norm.h"

using namespace st;

namespace {

// ONE: a row is a wave's own, four rows a workgroup; else the workgroup's
template <typename T, typename S, int VEC, bool ONE, bool BIAS>
__global__ __launch_bounds__(ONE ? 256 : 1024) void block_norm_fwd_kernel(NormArgs a) {
  __shared__ float2 red[2 * kNormWaves];
  RowSum<ONE> sum{red};
  const int lanes = ONE ? 64 : (int)blockDim.x, t = ONE ? threadIdx.x & 63 : threadIdx.x;
  const int width = a.width;
  const float inv = 1.f / (float)width;
  bool in[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) in[i] = ((i / VEC) * lanes + t) * VEC < width;
  float p1[8], p0[8], w2[8], b2[8];
  ld_weights<VEC, T, BIAS>(a, t, lanes, p1, p0, w2, b2);
  // mean and 1/std of x; a column behind the row counts as nothing
  auto stats = [&](const float (&x)[8], float& mean, float& rstd) {
    mean = 0.f;
    if (a.layer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += in[i] ? x[i] : 0.f;
      mean = sum.one(s) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) q += in[i] ? (x[i] - mean) * (x[i] - mean) : 0.f;
    rstd = rsqrtf(sum.one(q) * inv + a.eps);
  };
  const int64_t step = (int64_t)gridDim.x * (ONE ? 4 : 1);
  for (int64_t row = ONE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x; row < a.rows; row += step) {
    const int64_t base = row * width;
    float x[8], r[8];
    ld_lane<VEC>((const T*)a.h + base, t, lanes, width, x);
    if (a.res) ld_lane<VEC>((const S*)a.res + base, t, lanes, width, r);
    float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
    if (a.w1) stats(x, m1, r1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = (x[i] - m1) * r1 * p1[i];
      if (BIAS) x[i] += p0[i];
      if (a.res) x[i] += r[i];
    }
    if (a.s) st_lane<VEC>((S*)a.s + base, t, lanes, width, x);
    if (a.w2) {
      stats(x, m2, r2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (x[i] - m2) * r2 * w2[i];
        if (BIAS) x[i] += b2[i];
      }
      st_lane<VEC>((T*)a.y + base, t, lanes, width, x);
    }
    if (a.stats && t == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, r1, m2, r2);
  }
}

template <typename T, typename S, int VEC, bool BIAS>
int launch(const NormArgs& a, hipStream_t st) {
  const int waves = (a.width + 511) / 512;
  if (waves == 1) {
    const int64_t grid = std::min<int64_t>((a.rows + 3) / 4, 4096);
    block_norm_fwd_kernel<T, S, VEC, true, BIAS><<<(unsigned)grid, 256, 0, st>>>(a);
  } else {
    const int64_t grid = std::min<int64_t>(a.rows, 16384 / waves);
    block_norm_fwd_kernel<T, S, VEC, false, BIAS><<<(unsigned)grid, 64 * waves, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}
template <typename T, typename S>
int launch(const NormArgs& a, int vec, hipStream_t st) {
  const bool bias = a.b1 || a.b2;
  if (vec) return bias ? launch<T, S, 8, true>(a, st) : launch<T, S, 8, false>(a, st);
  return bias ? launch<T, S, 1, true>(a, st) : launch<T, S, 1, false>(a, st);
}

}  // namespace

extern "C" {

// htype / stype: types of h, y and of the stream (residual, s): kF32, kBF16, kF16; the stream's is
// h's or fp32.  vec: width % 8 == 0 and every pointer 16-byte aligned.  -2: outside the kernel's.
int st_block_norm_fwd(const NormArgs* a, int htype, int stype, int vec, hipStream_t st) {
  if (a->rows <= 0 || a->width <= 0 || a->width > kNormMaxWidth || (vec && a->width % 8)) return -2;
  if (htype == kF32 && stype == kF32) return launch<float, float>(*a, vec, st);
  if (htype == kBF16 && stype == kBF16) return launch<bf16_t, bf16_t>(*a, vec, st);
  if (htype == kBF16 && stype == kF32) return launch<bf16_t, float>(*a, vec, st);
  if (htype == kF16 && stype == kF16) return launch<__half, __half>(*a, vec, st);
  if (htype == kF16 && stype == kF32) return launch<__half, float>(*a, vec, st);
  return -2;
}

}  // extern "C"
