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

#include "common.h"
#include "block_norm_args.h"
#include <hip/hip_fp16.h>

namespace st {

// VEC elements at p -> floats
template <int VEC>
ST_DEVICE void ld_row(const float* p, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    const float4 a = ld4f(p), b = ld4f(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    f[0] = *p;
  }
}
template <int VEC>
ST_DEVICE void ld_row(const bf16_t* p, float (&f)[VEC]) {
  if constexpr (VEC == 8) unpack8(ld8(p), f);
  else f[0] = bf2f(*p);
}
template <int VEC>
ST_DEVICE void ld_row(const __half* p, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    const BF8 v = ld8(reinterpret_cast<const bf16_t*>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __half2float(__ushort_as_half((unsigned short)(v.w[i >> 1] >> (16 * (i & 1)))));
  } else {
    f[0] = __half2float(*p);
  }
}
template <int VEC>
ST_DEVICE void st_row(float* p, const float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    st4f(p, make_float4(f[0], f[1], f[2], f[3]));
    st4f(p + 4, make_float4(f[4], f[5], f[6], f[7]));
  } else {
    *p = f[0];
  }
}
template <int VEC>
ST_DEVICE void st_row(bf16_t* p, const float (&f)[VEC]) {
  if constexpr (VEC == 8) st8(p, pack8(f));
  else *p = f2bf(f[0]);
}
template <int VEC>
ST_DEVICE void st_row(__half* p, const float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    BF8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v.w[i] = (uint32_t)__half_as_ushort(__float2half(f[2 * i])) |
               ((uint32_t)__half_as_ushort(__float2half(f[2 * i + 1])) << 16);
    st8(reinterpret_cast<bf16_t*>(p), v);
  } else {
    *p = __float2half(f[0]);
  }
}
// eight elements of a lane, as NCH = 8 / VEC chunks; a column behind the row reads as `pad`
template <int VEC, typename P>
ST_DEVICE void ld_lane(const P* p, int lane, int lanes, int width, float (&f)[8], float pad = 0.f) {
#pragma unroll
  for (int c = 0; c < 8 / VEC; ++c) {
    const int col = (c * lanes + lane) * VEC;
    float v[VEC];
    if (col < width) ld_row<VEC>(p + col, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[c * VEC + i] = col < width ? v[i] : pad;
  }
}
template <int VEC, typename P>
ST_DEVICE void st_lane(P* p, int lane, int lanes, int width, const float (&f)[8]) {
#pragma unroll
  for (int c = 0; c < 8 / VEC; ++c) {
    const int col = (c * lanes + lane) * VEC;
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = f[c * VEC + i];
    if (col < width) st_row<VEC>(p + col, v);
  }
}
// The same still as loaded, so that a row can be requested ahead of its use.
template <typename P>
struct LaneRaw {
  static constexpr int kWords = 8 * sizeof(P) / 4;
  uint32_t w[kWords];
};
template <int VEC, typename P>
ST_DEVICE void ld_raw(const P* p, int lane, int lanes, int width, LaneRaw<P>& r) {
  if constexpr (VEC == 8) {
    if (lane * 8 < width) {
#pragma unroll
      for (int i = 0; i < LaneRaw<P>::kWords / 4; ++i) {
        const u32x4 v = reinterpret_cast<const u32x4*>(p + lane * 8)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) r.w[4 * i + k] = v[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < LaneRaw<P>::kWords; ++i) r.w[i] = 0;
    }
  } else {
    uint32_t e[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int col = c * lanes + lane;
      e[c] = 0;
      if (col < width) {
        if constexpr (sizeof(P) == 4) e[c] = reinterpret_cast<const uint32_t*>(p)[col];
        else e[c] = reinterpret_cast<const uint16_t*>(p)[col];
      }
    }
#pragma unroll
    for (int i = 0; i < LaneRaw<P>::kWords; ++i)
      r.w[i] = sizeof(P) == 4 ? e[i] : e[(2 * i) & 7] | (e[(2 * i + 1) & 7] << 16);
  }
}
template <typename P>
ST_DEVICE void zero_raw(LaneRaw<P>& r) {
#pragma unroll
  for (int i = 0; i < LaneRaw<P>::kWords; ++i) r.w[i] = 0;
}
template <typename P>
ST_DEVICE void widen(const LaneRaw<P>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(P) == 4) f[i] = __uint_as_float(r.w[i]);
    else if constexpr (sizeof(P) == 2 && __is_same(P, bf16_t))
      f[i] = __uint_as_float((i & 1) ? r.w[i >> 1] & 0xffff0000u : r.w[i >> 1] << 16);
    else f[i] = __half2float(__ushort_as_half((unsigned short)(r.w[i >> 1] >> (16 * (i & 1)))));
  }
}

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
