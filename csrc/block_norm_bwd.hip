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
// s is recomputed from h and the residual in fp32, so its rounding to 16 bits does not enter the
// gradients (from the rounded s, dw2 had 1.5 times the error of one rounding).  Where a norm after
// the block or a gate needs h anyway that reads no more; a plain pre-norm pays one stream for it,
// and keeps s alone where the stream is fp32 or s is h itself.
//
// A workgroup walks rows with a fixed stride and keeps its column sums in registers; its partial
// sums are added up by the second kernel in a fixed order (no atomics: results repeat bit for bit).
// Bound by HBM: h, residual (or s), dy, ds in, dh, dres out.  Measured: 24576 x 4096 bf16, both norms
// and a channel gate, 236-247 us (5.1-4.9 TB/s), and 10 us for its column sums; 16384 x 1280 LayerNorm
// 46 + 9 us; 3001 x 1001 fp32 with a scalar gate 18 + 12 us.  Without the next row's loads ahead the first took 301 us.  2048
// waves keep partial sums (512 workgroups where a wave has its own row): with half of them forward
// and backward took 515 us instead of 373, with twice as many 391.
#include "block_norm.h"

using namespace st;

namespace {

constexpr int kStream = 0, kPlain = 1, kFull = 2;

// MODE: from kStream s alone, from kPlain h and the residual, from kFull those with a norm after the
// block or a gate; BIAS: sums of dy / ds' are kept too
// MOST: the most threads of a workgroup, 256 where a wave has a row of its own; widths up to 4096 do
// with 512, which leaves a lane enough registers for the next row's loads
template <typename T, typename S, int VEC, int MOST, int MODE, bool BIAS>
__global__ __launch_bounds__(MOST) void block_norm_bwd_kernel(NormArgs a) {
  constexpr bool ONE = MOST == 256, GEN = MODE == kFull;
  constexpr int kArrays = (GEN ? 2 : 1) * (BIAS ? 2 : 1);
  constexpr int kA = 1, kDy = GEN ? 2 : 1, kB = 3;  // dy shat, [ds' hhat], [dy, [ds']]
  __shared__ float2 red[2 * kNormWaves];
  RowSum<ONE> sum{red};
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
  // the wave's next row is requested before this one's sums: two rows of loads in flight
  LaneRaw<T> nh, ndy;
  LaneRaw<S> ns, nds;
  float4 nst;
  zero_raw(nh);
  zero_raw(ns);
  zero_raw(ndy);
  zero_raw(nds);
  auto request = [&](int64_t row) {
    const int64_t base = row * width;
    if constexpr (MODE != kStream) {
      ld_raw<VEC>((const T*)a.h + base, t, lanes, width, nh);
      if (a.res) ld_raw<VEC>((const S*)a.res + base, t, lanes, width, ns);
    } else if (a.dy) {
      ld_raw<VEC>((const S*)a.s + base, t, lanes, width, ns);
    }
    if (a.dy) ld_raw<VEC>((const T*)a.dy + base, t, lanes, width, ndy);
    if (a.ds) ld_raw<VEC>((const S*)a.ds + base, t, lanes, width, nds);
    nst = reinterpret_cast<const float4*>(a.stats)[row];
  };
  const int64_t step = (int64_t)gridDim.x * (ONE ? 4 : 1);
  int64_t row = ONE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row < a.rows) request(row);
  for (; row < a.rows; row += step) {
    const int64_t base = row * width;
    float x[8], s[8], dy[8], d[8];
    widen(nh, x);
    widen(ns, s);
    widen(ndy, dy);
    widen(nds, d);
    const float4 st = nst;
    if (row + step < a.rows) request(row + step);
    if constexpr (MODE != kStream) {  // x: hhat, s: the stream
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
      const float2 pq = sum.two(p, q);
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
      const float2 pq = sum.two(p, q);
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

// The workgroups' partial sums [blocks][arrays][width] in kParts parts of blocks each: a wave 64
// columns, four waves a quarter of the part each, added in order.  From here on sums are held in 64
// bits: a scalar gate's gradient is one sum over all columns, in which the columns' sums cancel (in fp32
// that of 3001 x 1001 was off by up to 1e-6 of itself, as much as five times the rows' own sums are).
constexpr int kParts = 8;
__global__ __launch_bounds__(256) void block_norm_colsum_kernel(const float* __restrict__ partial, int blocks,
                                                                int arrays, int width, double* __restrict__ out) {
  __shared__ double red[4][64];
  const int q = threadIdx.x & 63, g = threadIdx.x >> 6, col = blockIdx.x * 64 + q;
  const int64_t line = (int64_t)arrays * width, at = (int64_t)blockIdx.y * width + col;
  const int per = (blocks + kParts - 1) / kParts, b1 = min(blocks, (int)(blockIdx.z + 1) * per);
  double s[4] = {0., 0., 0., 0.};
  if (col < width) {
    int b = blockIdx.z * per + g;
    for (; b + 12 < b1; b += 16)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += partial[(b + 4 * u) * line + at];
    for (; b < b1; b += 4) s[0] += partial[b * line + at];
  }
  red[g][q] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (!g && col < width) out[blockIdx.z * line + at] = (red[0][q] + red[1][q]) + (red[2][q] + red[3][q]);
}

int64_t sum_floats(int arrays, int width) { return (int64_t)kParts * arrays * width * 2; }  // whole 64 bytes

struct FinishArgs {
  const double* sums;  // [kParts][arrays][width]
  int arrays, width;
  int gen;
  const void *gate, *w1, *b1;
  int gate_n, w32;
  float scale;
  void *dgate, *dw1, *db1, *dw2, *db2;  // null: not wanted
  int tgate, tw1, tb1, tw2, tb2;        // whether they are fp32, else T
};

template <typename T>
ST_DEVICE void put(void* p, int f32, int i, float v) {
  const float f[1] = {v};
  if (f32) st_row<1>((float*)p + i, f);
  else st_row<1>((T*)p + i, f);
}

// One column a thread; with a scalar gate one workgroup takes all columns and adds up their gates.
template <typename T>
__global__ __launch_bounds__(1024) void block_norm_finish_kernel(FinishArgs f) {
  __shared__ double red[16];
  double total = 0.;
  for (int col = blockIdx.x * blockDim.x + threadIdx.x; col < f.width; col += gridDim.x * blockDim.x) {
    double s[4] = {0., 0., 0., 0.};
#pragma unroll
    for (int b = 0; b < kParts; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        s[k] += f.sums[((int64_t)b * f.arrays + (k < f.arrays ? k : 0)) * f.width + col];  // no branch: all in flight
    const double A = s[1], dyb = s[f.gen ? 2 : 1], B = s[3];
    if (f.dw2) put<T>(f.dw2, f.tw2, col, (float)s[0]);
    if (f.db2) put<T>(f.db2, f.tb2, col, (float)dyb);
    if (f.gen) {
      const double w = f.w1 ? ld_one<T>(f.w1, f.w32, col) : 1.f, b = f.b1 ? ld_one<T>(f.b1, f.w32, col) : 0.f;
      const double k = (double)f.scale * (f.gate_n ? ld_one<T>(f.gate, f.w32, f.gate_n > 1 ? col : 0) : 1.f);
      if (f.dw1) put<T>(f.dw1, f.tw1, col, (float)(k * A));
      if (f.db1) put<T>(f.db1, f.tb1, col, (float)(k * B));
      const double dg = f.scale * (w * A + (f.b1 ? b * B : 0.));
      if (f.dgate && f.gate_n > 1) put<T>(f.dgate, f.tgate, col, (float)dg);
      total += dg;
    }
  }
  if (f.gate_n != 1 || !f.dgate) return;
#pragma unroll
  for (int off = 32; off; off >>= 1) total += __shfl_xor(total, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) total += red[i];
    put<T>(f.dgate, f.tgate, 0, (float)total);
  }
}

template <typename T, typename S, int VEC, int MODE, bool BIAS>
int launch(const NormArgs& a, int blocks, hipStream_t st) {
  const int waves = (a.width + 511) / 512;
  if (waves == 1)
    block_norm_bwd_kernel<T, S, VEC, 256, MODE, BIAS><<<(unsigned)blocks, 256, 0, st>>>(a);
  else if (waves <= 8)
    block_norm_bwd_kernel<T, S, VEC, 512, MODE, BIAS><<<(unsigned)blocks, 64 * waves, 0, st>>>(a);
  else
    block_norm_bwd_kernel<T, S, VEC, 1024, MODE, BIAS><<<(unsigned)blocks, 64 * waves, 0, st>>>(a);
  return (int)hipGetLastError();
}
template <typename T, typename S, int VEC>
int launch(const NormArgs& a, int gen, int bias, int blocks, hipStream_t st) {
  if (gen) return bias ? launch<T, S, VEC, kFull, true>(a, blocks, st) : launch<T, S, VEC, kFull, false>(a, blocks, st);
  if constexpr (sizeof(S) == 2)  // an fp32 stream keeps s
    if (!a.s)
      return bias ? launch<T, S, VEC, kPlain, true>(a, blocks, st) : launch<T, S, VEC, kPlain, false>(a, blocks, st);
  return bias ? launch<T, S, VEC, kStream, true>(a, blocks, st) : launch<T, S, VEC, kStream, false>(a, blocks, st);
}
template <typename T, typename S>
int launch(const NormArgs& a, int gen, int bias, int blocks, int vec, hipStream_t st) {
  return vec ? launch<T, S, 8>(a, gen, bias, blocks, st) : launch<T, S, 1>(a, gen, bias, blocks, st);
}

template <typename T>
int finish(const FinishArgs& f, hipStream_t st) {
  const bool scalar = f.gate_n == 1 && f.dgate;
  const unsigned grid = scalar ? 1 : (unsigned)((f.width + 255) / 256);
  block_norm_finish_kernel<T><<<grid, scalar ? 1024 : 256, 0, st>>>(f);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// Workgroups of a backward, hence rows of its partial sums.
int st_block_norm_bwd_blocks(int64_t rows, int width) {
  const int waves = (width + 511) / 512;
  const int64_t need = waves == 1 ? (rows + 3) / 4 : rows, most = waves == 1 ? 512 : 2048 / waves;
  return (int)(need < most ? need : most);
}

int st_block_norm_bwd(const NormArgs* args, int gen, int bias, int blocks, int htype, int stype, int vec, hipStream_t st) {
  if (args->rows <= 0 || args->width <= 0 || args->width > kNormMaxWidth || (vec && args->width % 8) || blocks <= 0)
    return -2;
  if (!gen && !args->s && (stype == kF32 || !args->h)) return -2;
  NormArgs shifted = *args;
  if (shifted.partial) shifted.partial += sum_floats((gen ? 2 : 1) * (bias ? 2 : 1), args->width);
  const NormArgs* a = &shifted;
  if (htype == kF32 && stype == kF32) return launch<float, float>(*a, gen, bias, blocks, vec, st);
  if (htype == kBF16 && stype == kBF16) return launch<bf16_t, bf16_t>(*a, gen, bias, blocks, vec, st);
  if (htype == kBF16 && stype == kF32) return launch<bf16_t, float>(*a, gen, bias, blocks, vec, st);
  if (htype == kF16 && stype == kF16) return launch<__half, __half>(*a, gen, bias, blocks, vec, st);
  if (htype == kF16 && stype == kF32) return launch<__half, float>(*a, gen, bias, blocks, vec, st);
  return -2;
}

// Floats of a backward's workspace (NormArgs::partial) for `arrays` column sums: the parts' sums, then the
// workgroups'.
int64_t st_block_norm_bwd_floats(int64_t rows, int width, int arrays) {
  return sum_floats(arrays, width) + (int64_t)st_block_norm_bwd_blocks(rows, width) * arrays * width;
}

// The gradients of the weights and the gate from a's partial sums.  out: dgate, dw1, db1, dw2, db2
// (null: not wanted), out_f32: which of them are fp32 and not of h's type.
int st_block_norm_finish(const NormArgs* a, int gen, int bias, int blocks, void* const* out, const int* out_f32,
                         int htype, hipStream_t st) {
  FinishArgs f{};
  f.arrays = (gen ? 2 : 1) * (bias ? 2 : 1);
  double* sums = reinterpret_cast<double*>(a->partial);
  const float* partial = a->partial + sum_floats(f.arrays, a->width);
  const dim3 grid((unsigned)((a->width + 63) / 64), (unsigned)f.arrays, kParts);
  block_norm_colsum_kernel<<<grid, 256, 0, st>>>(partial, blocks, f.arrays, a->width, sums);
  f.sums = sums;
  f.width = a->width;
  f.gen = gen;
  f.gate = a->gate;
  f.w1 = a->w1;
  f.b1 = bias ? a->b1 : nullptr;
  f.gate_n = a->gate_n;
  f.w32 = a->w32;
  f.scale = a->scale;
  f.dgate = out[0]; f.dw1 = out[1]; f.db1 = out[2]; f.dw2 = out[3]; f.db2 = out[4];
  f.tgate = out_f32[0]; f.tw1 = out_f32[1]; f.tb1 = out_f32[2]; f.tw2 = out_f32[3]; f.tb2 = out_f32[4];
  if (htype == kF32) return finish<float>(f, st);
  if (htype == kBF16) return finish<bf16_t>(f, st);
  return finish<__half>(f, st);
}

}  // extern "C"
