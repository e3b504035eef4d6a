// One AdamW step over many separate tensors, with the moments in 32 or in 8 bits:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr (m / bc1) / (sqrt(v / bc2) + eps).
// A tensor is cut into blocks of 256 elements, one wave a block (4 elements a lane); 16
// consecutive blocks of one tensor are a workgroup's unit.  The tensors' pointers travel in the
// kernel's arguments (48 tensors a launch), so a step neither copies a table to the device nor
// waits for one.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 codes (largest value 448) with an fp32 scale per block
// and moment, the block's largest |value| / 448.  The root and not v itself, because e4m3's 2^17.8
// of range then spans 2^35.6 of v, and the update divides by the root.  Codes are rounded
// STOCHASTICALLY: beta2 moves v by 0.1 % a step at 0.999, far below e4m3's step of 6-12 %, so
// round-to-nearest would never let a root move again; the offsets are hashed from the element's
// place in the call's blocks and the step, so a step's result is repeatable.  A root that is not
// zero is never rounded to zero: m / (0 + eps) would throw the weight far off.  Elements that
// are not finite keep a NaN code and stay out of their block's scale, so that they spoil
// themselves only, as with 32-bit moments.
//
// Bound by HBM: read p, g, m, r, write p, m, r (and the 16-bit copy): 16 B an element with fp32
// gradients and 8-bit moments, 28 B with 32-bit ones.  Measured on MI355X (a 2 GiB copy: 4.9 TB/s):
// 707M elements with bf16 copies, 8-bit moments and fp32 gradients written back 2.70 ms (5.8 TB/s),
// 302M in fp32 throughout 1.64 ms (5.9 TB/s), 51M with bf16 gradients and 8-bit moments 179 us (4.6
// TB/s); a model of 42 tensors and 0.1M elements 26 us, of it 7 on the GPU.  All loads of a wave's
// four blocks are issued before its first sum: two blocks a wave took 185 / 1670 us (51M / 302M)
// instead of 181 / 1649, eight 287 / 1774 (too few waves for their registers).
#include "adamw_multi.h"

#include "common.h"
#include <hip/hip_fp16.h>

using namespace st;

namespace {

constexpr int kBlk = kAdamBlock, kPerWave = kAdamUnit / 4;  // 4 waves a workgroup

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

ST_DEVICE uint32_t mix32(uint32_t x) {  // as csrc/adamw.hip; ops/adamw_multi.py mirrors it
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  x ^= x >> 16;
  return x;
}

ST_DEVICE uint32_t pack_half(float a, float b, bool f16) {
  if (!f16) return pack_bf16x2(a, b);
  return (uint32_t)__half_as_ushort(__float2half(a)) | ((uint32_t)__half_as_ushort(__float2half(b)) << 16);
}
ST_DEVICE float half_up(uint32_t h, bool f16) {
  return f16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
}

// element types of the gradients and of the 16-bit parameter copies
constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;

template <int GT>
ST_DEVICE f32x4 load_g(const void* g, int64_t i, int n, bool vec) {  // n valid elements at i
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if constexpr (GT == kF32) {
    const float* p = (const float*)g + i;
    if (vec && n >= 4) return __builtin_nontemporal_load((const f32x4*)p);
    for (int k = 0; k < 4; ++k)
      if (k < n) r[k] = p[k];
  } else {
    const uint16_t* p = (const uint16_t*)g + i;
    if (vec && n >= 4) {
      const u32x2_t v = __builtin_nontemporal_load((const u32x2_t*)p);
      for (int k = 0; k < 4; ++k) r[k] = half_up((v[k >> 1] >> (16 * (k & 1))) & 0xffffu, GT == kF16);
    } else {
      for (int k = 0; k < 4; ++k)
        if (k < n) r[k] = half_up(p[k], GT == kF16);
    }
  }
  return r;
}
ST_DEVICE void store_f(float* p, int64_t i, int n, bool vec, f32x4 v) {
  if (vec && n >= 4) {
    __builtin_nontemporal_store(v, (f32x4*)(p + i));
    return;
  }
  for (int k = 0; k < 4; ++k)
    if (k < n) p[i + k] = v[k];
}
// four 16-bit values, rounded
ST_DEVICE void store_h(uint16_t* p, int64_t i, int n, bool vec, f32x4 v, bool f16) {
  const uint32_t a = pack_half(v[0], v[1], f16), b = pack_half(v[2], v[3], f16);
  if (vec && n >= 4) {
    __builtin_nontemporal_store(u32x2_t{a, b}, (u32x2_t*)(p + i));
    return;
  }
  for (int k = 0; k < 4; ++k)
    if (k < n) p[i + k] = (uint16_t)((k < 2 ? a : b) >> (16 * (k & 1)));
}
ST_DEVICE uint32_t load_c(const uint8_t* p, int64_t i, int n, bool vec) {
  if (vec && n >= 4) return __builtin_nontemporal_load((const uint32_t*)(p + i));
  uint32_t r = 0;
  for (int k = 0; k < 4; ++k)
    if (k < n) r |= (uint32_t)p[i + k] << (8 * k);
  return r;
}
ST_DEVICE void store_c(uint8_t* p, int64_t i, int n, bool vec, uint32_t v) {
  if (vec && n >= 4) {
    __builtin_nontemporal_store(v, (uint32_t*)(p + i));
    return;
  }
  for (int k = 0; k < 4; ++k)
    if (k < n) p[i + k] = (uint8_t)(v >> (8 * k));
}
ST_DEVICE f32x4 decode(uint32_t c, float scale) {
  f32x4 r;
  r[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
  r[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
  r[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
  r[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
  return r * scale;
}

ST_DEVICE bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Four values of a block in 8 bits: |x| 448 / top, its low 20 mantissa bits rounded away with 16
// random ones.  Below 2^-6 e4m3's steps are equal (2^-9): adding 2^-6 brings such a value into the
// binade that has those steps.  `root`: what is not zero stays at least the smallest code.
ST_DEVICE uint32_t encode(f32x4 x, float top, bool root, const uint32_t (&r16)[4]) {
#pragma clang fp contract(off)
  const float inv = top > 0x1p-100f ? (1.f / top) * 448.f : 0.f;  // below: the moment is zero in fp32's own squares
  float q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = fminf(__builtin_fabsf(x[k]) * inv, 448.f);
    const float tiny = a < 0x1p-6f ? 0x1p-6f : 0.f;
    float t = __uint_as_float((__float_as_uint(a + tiny) + (r16[k] << 4)) & 0xfff00000u) - tiny;
    if (root && a > 0.f) t = fmaxf(t, 0x1p-9f);
    q[k] = finite(x[k]) ? __builtin_copysignf(t, x[k]) : __builtin_nanf("");
  }
  uint32_t c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
}

ST_DEVICE float top_of(f32x4 x) {
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) t = fmaxf(t, finite(x[k]) ? __builtin_fabsf(x[k]) : 0.f);
  return wave_max(t);
}

template <int GT, int PT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_multi_kernel(AdamTable tab, int count, AdamScalars h) {
#pragma clang fp contract(off)  // the sums below round as they are written, as the plain form does
  // the tensor that holds this unit: the first whose units end behind it
  const int unit = (int)blockIdx.x;
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].unit_end <= unit) lo = mid + 1; else hi = mid;
  }
  const AdamTensor& T = tab.t[lo];
  const int first = lo ? tab.t[lo - 1].unit_end : 0;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n = T.n;
  const int64_t blk0 = (int64_t)(unit - first) * kAdamUnit + wid * kPerWave;
  const bool vec = T.vec;
  const float clip = h.clip ? *h.clip : 1.f;
  const float keep = T.keep;
  float* pw = (float*)(PT == kF32 ? T.param : T.master);

  f32x4 p[kPerWave], g[kPerWave], m[kPerWave], v[kPerWave];
  uint32_t cm[kPerWave], cr[kPerWave];
  float2 sc[kPerWave];
  int left[kPerWave];
  // every load of the wave's four blocks is issued before the first sum
#pragma unroll
  for (int u = 0; u < kPerWave; ++u) {
    const int64_t i = (blk0 + u) * kBlk + lane * 4;
    left[u] = (int)(n - i < 4 ? (n - i < 0 ? 0 : n - i) : 4);
    const bool some = (blk0 + u) * kBlk < n;
    cm[u] = cr[u] = 0;
    sc[u] = make_float2(0.f, 0.f);
    p[u] = g[u] = m[u] = v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (left[u] > 0) {
      p[u] = load_g<kF32>(pw, i, left[u], vec);
      g[u] = load_g<GT>(T.grad, i, left[u], vec);
      if constexpr (EIGHT) {
        cm[u] = load_c((const uint8_t*)T.m, i, left[u], vec);
        cr[u] = load_c((const uint8_t*)T.v, i, left[u], vec);
      } else {
        m[u] = load_g<kF32>(T.m, i, left[u], vec);
        v[u] = load_g<kF32>(T.v, i, left[u], vec);
      }
    }
    if (EIGHT && some) sc[u] = reinterpret_cast<const float2*>(T.scales)[blk0 + u];
  }
#pragma unroll
  for (int u = 0; u < kPerWave; ++u) {
    if ((blk0 + u) * kBlk >= n) break;  // uniform over the wave
    const int64_t i = (blk0 + u) * kBlk + lane * 4;
    if constexpr (EIGHT) {
      m[u] = decode(cm[u], sc[u].x);
      const f32x4 r = decode(cr[u], sc[u].y);
      v[u] = r * r;
    }
    f32x4 root;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gk = g[u][k] * clip;
      g[u][k] = gk;
      m[u][k] = m[u][k] * h.b1 + gk * h.c1;
      v[u][k] = v[u][k] * h.b2 + gk * gk * h.c2;
      root[k] = __builtin_sqrtf(v[u][k]);
      const float upd = (m[u][k] * h.inv_bc1) / (root[k] * h.inv_sbc2 + h.eps);
      p[u][k] = p[u][k] * keep - upd * h.lr;
    }
    store_f(pw, i, left[u], vec, p[u]);
    if constexpr (PT != kF32) store_h((uint16_t*)T.param, i, left[u], vec, p[u], PT == kF16);
    if (h.write_grads) {
      if constexpr (GT == kF32) store_f((float*)T.grad, i, left[u], vec, g[u]);
      else store_h((uint16_t*)T.grad, i, left[u], vec, g[u], GT == kF16);
    }
    if constexpr (EIGHT) {
      const float tm = top_of(m[u]), tr = top_of(root);
      const uint64_t e = (uint64_t)((T.blk_base + blk0 + u) * kBlk + lane * 4);  // the element's place in the call
      const uint32_t hm = mix32((uint32_t)(e >> 32) ^ h.key);
      uint32_t rm[4], rr[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = mix32(((uint32_t)e + k) ^ hm);
        rm[k] = x & 0xffffu;
        rr[k] = x >> 16;
      }
      store_c((uint8_t*)T.m, i, left[u], vec, encode(m[u], tm, false, rm));
      store_c((uint8_t*)T.v, i, left[u], vec, encode(root, tr, true, rr));
      if (lane == 0)
        reinterpret_cast<float2*>(T.scales)[blk0 + u] = make_float2(tm * (1.f / 448.f), tr * (1.f / 448.f));
    } else {
      store_f((float*)T.m, i, left[u], vec, m[u]);
      store_f((float*)T.v, i, left[u], vec, v[u]);
    }
  }
}

template <int GT, int PT>
void launch(const AdamTable& tab, int count, int units, const AdamScalars& h, int eight, hipStream_t st) {
  if (eight)
    adamw_multi_kernel<GT, PT, true><<<(unsigned)units, 256, 0, st>>>(tab, count, h);
  else
    adamw_multi_kernel<GT, PT, false><<<(unsigned)units, 256, 0, st>>>(tab, count, h);
}

}  // namespace

extern "C" {

// gtype / ptype: 0 fp32, 1 bf16, 2 fp16.  0 on success, -2 for arguments outside the kernel's.
int st_adamw_multi(const AdamTable* tab, int count, const AdamScalars* h, int gtype, int ptype, int eight,
                   hipStream_t st) {
  if (count <= 0 || count > kAdamTensors || gtype < 0 || gtype > 2 || ptype < 0 || ptype > 2) return -2;
  const int units = tab->t[count - 1].unit_end;
  if (units <= 0) return -2;
  switch (gtype * 3 + ptype) {
    case 0: launch<0, 0>(*tab, count, units, *h, eight, st); break;
    case 1: launch<0, 1>(*tab, count, units, *h, eight, st); break;
    case 2: launch<0, 2>(*tab, count, units, *h, eight, st); break;
    case 3: launch<1, 0>(*tab, count, units, *h, eight, st); break;
    case 4: launch<1, 1>(*tab, count, units, *h, eight, st); break;
    case 5: launch<1, 2>(*tab, count, units, *h, eight, st); break;
    case 6: launch<2, 0>(*tab, count, units, *h, eight, st); break;
    case 7: launch<2, 1>(*tab, count, units, *h, eight, st); break;
    default: launch<2, 2>(*tab, count, units, *h, eight, st); break;
  }
  return (int)hipGetLastError();
}

}  // extern "C"
