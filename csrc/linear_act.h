// Matrix products with an epilogue (linear_act_*.hip): arguments and what the kernels share.
//
//   forward   z = x W^T + b,  y = act(z) + residual
//   backward  dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum of dz over the rows
//
// One product C[m, n] = sum_k A(m, k) B(n, k) serves all three: an operand is stored with k
// contiguous ([rows, k], kRow) or with its rows contiguous ([k, rows], kCol):
//   y: x kRow, W kRow;   dx: dz kRow, W kCol;   dW: dz kCol, x kCol.
#pragma once

#include "linear_act_args.h"

#include "common.h"
#include <hip/hip_fp16.h>

namespace st {

typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 hx8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

typedef __amdgpu_buffer_rsrc_t rsrc_t;
// A lane's offset behind every range: loads give zero, stores go nowhere.  The range test subtracts the scalar
// offset from the range's size in 32 bits: with a scalar offset of up to the size the difference stays below
// 2^31 and kOut outside, with a larger one it can wrap to above kOut.  So scalar offsets stay inside the range.
constexpr uint32_t kOut = 0xffffffe0u;
ST_DEVICE uint32_t uni(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
ST_DEVICE rsrc_t rsrc_of(const void* base, uint32_t bytes) {  // of wave-uniform values
  const uint64_t a = (uint64_t)base;
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)uni((uint32_t)(a >> 32)) << 32) | uni((uint32_t)a)),
                                           (short)0, (int)uni(bytes), 0x00020000);
}

// 16-bit types travel as raw bits; F16 says which they are
ST_DEVICE float half_up(uint32_t h, bool f16) {
  return f16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
}
ST_DEVICE uint32_t half_down(float f, bool f16) {
  return f16 ? (uint32_t)__half_as_ushort(__float2half(f)) : (uint32_t)f2bf(f);
}
typedef __bf16 bfx2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
ST_DEVICE uint32_t pack2(float a, float b, bool f16) {
  if (f16) return half_down(a, true) | (half_down(b, true) << 16);
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bfx2));  // one v_cvt_pk_bf16_f32
}
ST_DEVICE u32x2 pack4(f32x4 v, bool f16) { return u32x2{pack2(v[0], v[1], f16), pack2(v[2], v[3], f16)}; }
ST_DEVICE f32x4 unpack4(u32x2 p, bool f16) {
  return f32x4{half_up(p[0] & 0xffffu, f16), half_up(p[0] >> 16, f16), half_up(p[1] & 0xffffu, f16),
               half_up(p[1] >> 16, f16)};
}

// The activations, from one exponential and one reciprocal each, in as few operations as can be: the
// epilogue of the wide kernel runs them with nothing beside it.  Their errors are relative to the result, so
// that the far tail of a 16-bit result is rounded rightly too: some 2^-22, and for the exponential 2^-23 of its
// exponent, 4e-6 at z = -8.  The normal distribution function's tail is Phi(-|z|) = exp(-z^2 / 2) t P(t) with
// t = 1 / (1 + 0.325 |z|): what is left beside the exponential, exp(z^2 / 2) erfc(|z| / sqrt(2)) / 2, falls as
// 1 / |z| does, so over t it is smooth on [0, 1], and P of degree 7 is its equal-ripple fit (least squares
// reweighted by the residual) of relative error 6.8e-7; 1e-6 with fp32 arithmetic.
ST_DEVICE float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
ST_DEVICE float rcp(float x) { return __builtin_amdgcn_rcpf(x); }
ST_DEVICE float sigmoid(float x) { return rcp(1.f + exp2_(x * -1.4426950408889634f)); }
// p, t and e = exp(-z^2 / 2) with Phi(-|z|) = t p e
ST_DEVICE float normal_poly(float z, float& e, float& t) {
  e = exp2_(z * (z * -0.72134752044448170f));
  t = rcp(__builtin_fmaf(__builtin_fabsf(z), 0.325f, 1.f));
  float p = __builtin_fmaf(t, 0.033816796f, -0.11351987f);
  p = __builtin_fmaf(t, p, 0.085308872f);
  p = __builtin_fmaf(t, p, 0.026046028f);
  p = __builtin_fmaf(t, p, 0.093516320f);
  p = __builtin_fmaf(t, p, 0.11550388f);
  p = __builtin_fmaf(t, p, 0.12967210f);
  return __builtin_fmaf(t, p, 0.12965615f);
}
constexpr float kTanhA = 1.5957691216057308f, kTanhB = 0.044715f;  // 2 sqrt(2 / pi): (1 + tanh(a)) / 2 = sigmoid(2 a)
constexpr float kLog2e = 1.4426950408889634f;

ST_DEVICE float act_of(float z, int act) {
  float e;
  switch (act) {
    case kRelu: return z < 0.f ? 0.f : z;
    case kGelu: {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|); an infinite |z| times a zero tail is kept out
      float t;
      const float p = normal_poly(z, e, t);
      return __builtin_fmaf(-__builtin_fminf(__builtin_fabsf(z), 1e30f), t * p * e, __builtin_fmaxf(z, 0.f));
    }
    case kGeluTanh: {
      const float s = z * __builtin_fmaf(z * z, -kTanhA * kTanhB * kLog2e, -kTanhA * kLog2e);
      return z * rcp(1.f + exp2_(s));
    }
    case kSilu: return z * sigmoid(z);
    default: return z;
  }
}
ST_DEVICE float act_slope(float z, int act) {
  // an fp16 z can have become infinite in storage: its slope is the limit, 0 or 1, not inf * 0
  z = __builtin_fabsf(z) > 1e30f ? __builtin_copysignf(1e30f, z) : z;
  switch (act) {
    case kRelu: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case kGelu: {
      float e, t;
      const float p = normal_poly(z, e, t), c = t * p * e;
      return (z < 0.f ? c : 1.f - c) + z * e * 0.39894228040143268f;
    }
    case kGeluTanh: {
      const float zz = __builtin_fminf(z * z, 1e6f);  // beyond: the slope is 0 or 1, and inf * 0 is kept out
      const float p = sigmoid(kTanhA * z * (1.f + kTanhB * zz));
      return p + z * p * (1.f - p) * kTanhA * (1.f + 3.f * kTanhB * zz);
    }
    case kSilu: {
      const float p = sigmoid(z), q = z * (1.f - p);
      return p + p * (p > 0.f ? q : 0.f);
    }
    default: return 1.f;
  }
}

ST_DEVICE void act4(f32x4& v, int act) {  // one choice for four values
  switch (act) {
    case kRelu:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of(v[i], kRelu);
      break;
    case kGelu:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of(v[i], kGelu);
      break;
    case kGeluTanh:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of(v[i], kGeluTanh);
      break;
    case kSilu:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of(v[i], kSilu);
      break;
    default: break;
  }
}

// The epilogue of four consecutive columns n .. n + 3 of row m (count of them inside the matrix;
// vec: all four, with aligned rows).
ST_DEVICE void epilogue4(const LinearEpi& e, int64_t m, int n, int count, bool vec, f32x4 v) {
  const int64_t at = m * e.ldo + n;
  if (vec && count >= 4) {
    if (e.bias) v += unpack4(*reinterpret_cast<const u32x2*>((const uint16_t*)e.bias + n), e.f16);
    if (e.z) *reinterpret_cast<u32x2*>((uint16_t*)e.z + at) = pack4(v, e.f16);
    act4(v, e.act);
    if (e.res)
      v += e.out_f32 ? *reinterpret_cast<const f32x4*>((const float*)e.res + at)
                     : unpack4(*reinterpret_cast<const u32x2*>((const uint16_t*)e.res + at), e.f16);
    if (e.out_f32) *reinterpret_cast<f32x4*>((float*)e.out + at) = v;
    else *reinterpret_cast<u32x2*>((uint16_t*)e.out + at) = pack4(v, e.f16);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= count) break;
    float x = v[i];
    if (e.bias) x += half_up(((const uint16_t*)e.bias)[n + i], e.f16);
    if (e.z) ((uint16_t*)e.z)[at + i] = (uint16_t)half_down(x, e.f16);
    x = act_of(x, e.act);
    if (e.res) x += e.out_f32 ? ((const float*)e.res)[at + i] : half_up(((const uint16_t*)e.res)[at + i], e.f16);
    if (e.out_f32) ((float*)e.out)[at + i] = x;
    else ((uint16_t*)e.out)[at + i] = (uint16_t)half_down(x, e.f16);
  }
}

}  // namespace st
