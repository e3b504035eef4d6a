// A lane's part of a row: eight elements of fp32, bf16 or fp16, as 16-byte groups (VEC = 8: widths of
// a multiple of 8, aligned rows) or one by one with neighbouring lanes at neighbouring columns (VEC = 1).
#pragma once

#include "common.h"
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

}  // namespace st
