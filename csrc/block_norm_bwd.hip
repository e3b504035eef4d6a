// Backward of the norms around a block's gated residual (formulas and layouts: block_norm.h).
//
// With shat, hhat the normalised rows, g2 = dy w2 and mean() over a row:
//   ds' = ds + r2 (g2 - shat mean(g2 shat) - mean(g2))        (the last mean: layer norm)
//   dres = ds',  du = scale gate ds',  g1 = du w1
//   dh = r1 (g1 - hhat mean(g1 hhat) - mean(g1))              (no norm after the block: dh = du)
//   dw2 = sum dy shat, db2 = sum dy, and from A = sum ds' hhat, B = sum ds' over the rows:
//   dw1 = scale gate A, db1 = scale gate B, dgate = scale (w1 A + b1 B)
// so two column sums serve the norm after the block and its gate, whatever the gate.
//
// Where there is a norm after the block or a gate, s is recomputed from h and the residual in
// fp32: that reads as much as s and h would, and s's rounding does not enter the gradients.  A
// plain pre-norm keeps s alone (one stream less).
//
// A workgroup walks rows with a fixed stride and keeps its column sums in registers; its partial
// sums are added up by the second kernel in a fixed order (no atomics: results repeat bit for bit).
// Bound by HBM: h, residual (or s), dy, ds in, dh, dres out.
#include "block_norm.h"

using namespace st;

namespace {

// GEN: a norm after the block or a gate (else s alone); BIAS: sums of dy / ds' are kept too
template <typename T, typename S, int VEC, bool ONE, bool GEN, bool BIAS>
__global__ __launch_bounds__(ONE ? 256 : 1024) void block_norm_bwd_kernel(NormArgs a) {
  constexpr int kArrays = (GEN ? 2 : 1) * (BIAS ? 2 : 1);
  constexpr int kA = 1, kDy = GEN ? 2 : 1, kB = 3;  // dy shat, [ds' hhat], [dy, [ds']]
  __shared__ float2 red[kNormWaves];
  const int lanes = ONE ? 64 : (int)blockDim.x, t = ONE ? threadIdx.x & 63 : threadIdx.x;
  const int width = a.width;
  const float inv = 1.f / (float)width;
  float p1[8], p0[8], w2[8], b2[8];
  ld_weights<VEC, T, BIAS>(a, t, lanes, p1, p0, w2, b2);
  float acc[kArrays][8];
#pragma unroll
  for (int k = 0; k < kArrays; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[k][i] = 0.f;
  const int64_t step = (int64_t)gridDim.x * (ONE ? 4 : 1);
  for (int64_t row = ONE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x; row < a.rows; row += step) {
    const int64_t base = row * width;
    float x[8], s[8], dy[8], d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s[i] = dy[i] = d[i] = 0.f;
    if constexpr (GEN) {
      ld_lane<VEC>((const T*)a.h + base, t, lanes, width, x);
      if (a.res) ld_lane<VEC>((const S*)a.res + base, t, lanes, width, s);
    } else if (a.dy) {
      ld_lane<VEC>((const S*)a.s + base, t, lanes, width, s);
    }
    if (a.dy) ld_lane<VEC>((const T*)a.dy + base, t, lanes, width, dy);
    if (a.ds) ld_lane<VEC>((const S*)a.ds + base, t, lanes, width, d);
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    if constexpr (GEN) {  // x: hhat, s: the stream
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (x[i] - st.x) * st.y;
        s[i] += x[i] * p1[i];
        if (BIAS) s[i] += p0[i];
      }
    }
    if (a.dy) {  // through the norm before the next block; behind the row, dy is zero
      float p = 0.f, q = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = (s[i] - st.z) * st.w;
        acc[0][i] += dy[i] * s[i];
        if (BIAS) acc[kDy][i] += dy[i];
        dy[i] *= w2[i];
        p += dy[i] * s[i];
        q += dy[i];
      }
      const float2 pq = row_sum2<ONE>(p, q, red);
      const float cp = pq.x * inv, cq = a.layer ? pq.y * inv : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] += st.w * (dy[i] - s[i] * cp - cq);
    }
    if (a.dres) st_lane<VEC>((S*)a.dres + base, t, lanes, width, d);
    float p = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (GEN) {
        acc[kA][i] += d[i] * x[i];
        if (BIAS) acc[kB][i] += d[i];
      }
      d[i] *= p1[i];  // zero behind the row where there is a w1
      p += d[i] * x[i];
      q += d[i];
    }
    if (GEN && a.w1) {
      const float2 pq = row_sum2<ONE>(p, q, red);
      const float cp = pq.x * inv, cq = a.layer ? pq.y * inv : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = st.y * (d[i] - x[i] * cp - cq);
    }
    if (a.dh) st_lane<VEC>((T*)a.dh + base, t, lanes, width, d);
  }
  if (!a.partial) return;
  __shared__ float fold[ONE ? 3 * 8 * 64 : 1];  // the other three rows' sums, added in order
  const int wid = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < kArrays; ++k) {
    if constexpr (ONE) {
      __syncthreads();
      if (wid)
#pragma unroll
        for (int i = 0; i < 8; ++i) fold[((wid - 1) * 8 + i) * 64 + t] = acc[k][i];
      __syncthreads();
      if (!wid)
        for (int w = 0; w < 3; ++w)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[k][i] += fold[(w * 8 + i) * 64 + t];
    }
    if (!ONE || !wid) st_lane<VEC>(a.partial + ((int64_t)blockIdx.x * kArrays + k) * width, t, lanes, width, acc[k]);
  }
}

struct FinishArgs {
  const float* partial;
  int blocks, arrays, width;
  int gen, bias;
  const void *gate, *w1, *b1;
  int gate_n, w32;
  float scale;
  void *dgate, *dw1, *db1, *dw2, *db2;  // null: not wanted
  int tgate, tw1, tb1, tw2, tb2;        // whether they are fp32, else T
  float* gate_part;                     // scalar gate: one sum a workgroup
};

template <typename T>
ST_DEVICE void put(void* p, int f32, int i, float v) {
  const float f[1] = {v};
  if (f32) st_row<1>((float*)p + i, f);
  else st_row<1>((T*)p + i, f);
}

// 32 columns a workgroup, 32 groups of partial rows each summed in order, then the groups in order
template <typename T>
__global__ __launch_bounds__(1024) void block_norm_finish_kernel(FinishArgs f) {
  __shared__ float red[4][32][33];
  const int q = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + q;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < f.width)
    for (int b = g; b < f.blocks; b += 32)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < f.arrays) s[k] += f.partial[((int64_t)b * f.arrays + k) * f.width + col];
#pragma unroll
  for (int k = 0; k < 4; ++k) red[k][g][q] = s[k];
  __syncthreads();
  if (g) return;
  for (int k = 0; k < 4; ++k) {
    s[k] = red[k][0][q];
    for (int i = 1; i < 32; ++i) s[k] += red[k][i][q];
  }
  float dg = 0.f;
  if (col < f.width) {
    const float A = s[1], dyb = s[f.gen ? 2 : 1], B = s[3];
    if (f.dw2) put<T>(f.dw2, f.tw2, col, s[0]);
    if (f.db2) put<T>(f.db2, f.tb2, col, dyb);
    if (f.gen) {
      const float w = f.w1 ? ld_one<T>(f.w1, f.w32, col) : 1.f, b = f.b1 ? ld_one<T>(f.b1, f.w32, col) : 0.f;
      const float k = f.scale * (f.gate_n ? ld_one<T>(f.gate, f.w32, f.gate_n > 1 ? col : 0) : 1.f);
      if (f.dw1) put<T>(f.dw1, f.tw1, col, k * A);
      if (f.db1) put<T>(f.db1, f.tb1, col, k * B);
      dg = f.scale * (w * A + (f.b1 ? b * B : 0.f));
      if (f.dgate && f.gate_n > 1) put<T>(f.dgate, f.tgate, col, dg);
    }
  }
  if (f.gate_part) {
    for (int o = 16; o > 0; o >>= 1) dg += __shfl_xor(dg, o, 32);
    if (q == 0) f.gate_part[blockIdx.x] = dg;
  }
}

template <typename T>
__global__ __launch_bounds__(64) void block_norm_gate_kernel(const float* __restrict__ part, int n, void* dgate,
                                                             int f32) {
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 64) s += part[i];
  s = wave_sum(s);
  if (threadIdx.x == 0) put<T>(dgate, f32, 0, s);
}

template <typename T, typename S, int VEC, bool GEN, bool BIAS>
int launch(const NormArgs& a, int blocks, hipStream_t st) {
  const int waves = (a.width + 511) / 512;
  if (waves == 1)
    block_norm_bwd_kernel<T, S, VEC, true, GEN, BIAS><<<(unsigned)blocks, 256, 0, st>>>(a);
  else
    block_norm_bwd_kernel<T, S, VEC, false, GEN, BIAS><<<(unsigned)blocks, 64 * waves, 0, st>>>(a);
  return (int)hipGetLastError();
}
template <typename T, typename S, int VEC>
int launch(const NormArgs& a, int gen, int bias, int blocks, hipStream_t st) {
  if (gen) return bias ? launch<T, S, VEC, true, true>(a, blocks, st) : launch<T, S, VEC, true, false>(a, blocks, st);
  return bias ? launch<T, S, VEC, false, true>(a, blocks, st) : launch<T, S, VEC, false, false>(a, blocks, st);
}
template <typename T, typename S>
int launch(const NormArgs& a, int gen, int bias, int blocks, int vec, hipStream_t st) {
  return vec ? launch<T, S, 8>(a, gen, bias, blocks, st) : launch<T, S, 1>(a, gen, bias, blocks, st);
}

template <typename T>
int finish(const FinishArgs& f, hipStream_t st) {
  const unsigned grid = (unsigned)((f.width + 31) / 32);
  block_norm_finish_kernel<T><<<grid, 1024, 0, st>>>(f);
  if (f.gate_part) block_norm_gate_kernel<T><<<1, 64, 0, st>>>(f.gate_part, (int)grid, f.dgate, f.tgate);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// Workgroups of a backward, hence rows of its partial sums.
int st_block_norm_bwd_blocks(int64_t rows, int width) {
  const int waves = (width + 511) / 512;
  const int64_t need = waves == 1 ? (rows + 3) / 4 : rows, most = waves == 1 ? 1024 : 4096 / waves;
  return (int)(need < most ? need : most);
}

int st_block_norm_bwd(const NormArgs* a, int gen, int bias, int blocks, int htype, int stype, int vec, hipStream_t st) {
  if (a->rows <= 0 || a->width <= 0 || a->width > kNormMaxWidth || (vec && a->width % 8) || blocks <= 0) return -2;
  if (htype == kF32 && stype == kF32) return launch<float, float>(*a, gen, bias, blocks, vec, st);
  if (htype == kBF16 && stype == kBF16) return launch<bf16_t, bf16_t>(*a, gen, bias, blocks, vec, st);
  if (htype == kBF16 && stype == kF32) return launch<bf16_t, float>(*a, gen, bias, blocks, vec, st);
  if (htype == kF16 && stype == kF16) return launch<__half, __half>(*a, gen, bias, blocks, vec, st);
  if (htype == kF16 && stype == kF32) return launch<__half, float>(*a, gen, bias, blocks, vec, st);
  return -2;
}

// The gradients of the weights and the gate from a's partial sums.  out: dgate, dw1, db1, dw2, db2
// (null: not wanted), out_f32: which of them are fp32 and not of h's type; gate_part: (width + 31) / 32
// floats for a scalar gate.
int st_block_norm_finish(const NormArgs* a, int gen, int bias, int blocks, void* const* out, const int* out_f32,
                         float* gate_part, int htype, hipStream_t st) {
  FinishArgs f{};
  f.partial = a->partial;
  f.blocks = blocks;
  f.arrays = (gen ? 2 : 1) * (bias ? 2 : 1);
  f.width = a->width;
  f.gen = gen;
  f.bias = bias;
  f.gate = a->gate;
  f.w1 = a->w1;
  f.b1 = bias ? a->b1 : nullptr;
  f.gate_n = a->gate_n;
  f.w32 = a->w32;
  f.scale = a->scale;
  f.dgate = out[0]; f.dw1 = out[1]; f.db1 = out[2]; f.dw2 = out[3]; f.db2 = out[4];
  f.tgate = out_f32[0]; f.tw1 = out_f32[1]; f.tb1 = out_f32[2]; f.tw2 = out_f32[3]; f.tb2 = out_f32[4];
  f.gate_part = a->gate_n == 1 && out[0] ? gate_part : nullptr;
  if (htype == kF32) return finish<float>(f, st);
  if (htype == kBF16) return finish<bf16_t>(f, st);
  return finish<__half>(f, st);
}

}  // extern "C"
