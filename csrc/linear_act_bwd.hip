// dz = dy act'(z) and the bias gradient db = sum of dz over the rows (formulas: linear_act.h).
//
// One pass over dy and z: a workgroup takes 512 columns and a run of rows, its four waves every
// fourth row; each lane keeps its 8 columns' sums, which are folded in a fixed order and added up
// over the runs by the second kernel (no atomics: repeatable).  db sums the unrounded dz.  Bound by
// HBM: dy and z in, dz out: 24576 x 14336 bf16 404 us (5.2 TB/s), 8192 x 5120 53 us (4.8).
#include <algorithm>

#include "linear_act.h"
#include "row_io.h"

using namespace st;

namespace {

// P: dy's type; T: of z and dz.  z null: no activation (dz is dy).  dz null: only the sums.
template <typename P, typename T, int VEC>
__global__ __launch_bounds__(256) void linear_dz_kernel(const P* __restrict__ dy, const T* __restrict__ z,
                                                        T* __restrict__ dz, float* __restrict__ partial, int64_t rows,
                                                        int width, int64_t run, int act) {
  __shared__ float fold[3 * 8 * 64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c0 = blockIdx.x * 512, left = width - c0;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t r1 = min(rows, (int64_t)(blockIdx.y + 1) * run);
  LaneRaw<P> nd;
  LaneRaw<T> nz;
  zero_raw(nz);
  auto request = [&](int64_t r) {
    ld_raw<VEC>(dy + r * width + c0, lane, 64, left, nd);
    if (z) ld_raw<VEC>(z + r * width + c0, lane, 64, left, nz);
  };
  int64_t r = (int64_t)blockIdx.y * run + wid;
  if (r < r1) request(r);
  for (; r < r1; r += 4) {
    float d[8], s[8];
    widen(nd, d);
    widen(nz, s);
    if (r + 4 < r1) request(r + 4);
    if (z) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] *= act_slope(s[i], act);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += d[i];
    if (dz) st_lane<VEC>(dz + r * width + c0, lane, 64, left, d);
  }
  if (!partial) return;
  if (wid)
#pragma unroll
    for (int i = 0; i < 8; ++i) fold[((wid - 1) * 8 + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (wid) return;
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += fold[(w * 8 + i) * 64 + lane];
  st_lane<VEC>(partial + (int64_t)blockIdx.y * width + c0, lane, 64, left, acc);
}

// db from the runs' sums: 32 columns a workgroup at a time, 32 groups of runs
template <typename T>
__global__ __launch_bounds__(1024) void linear_db_kernel(const float* __restrict__ partial, int runs, int width,
                                                         T* __restrict__ db, float* __restrict__ db32) {
  __shared__ float red[32][33];
  const int q = threadIdx.x & 31, g = threadIdx.x >> 5;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < width; c0 += (int64_t)gridDim.x * 32) {
    const int64_t col = c0 + q;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < width) {
      int b = g;
      for (; b + 96 < runs; b += 128)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] += partial[(int64_t)(b + 32 * u) * width + col];
      for (; b < runs; b += 32) s[0] += partial[(int64_t)b * width + col];
    }
    red[g][q] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (!g && col < width) {
      float t = red[0][q];
      for (int i = 1; i < 32; ++i) t += red[i][q];
      const float f[1] = {t};
      if (db32) st_row<1>(db32 + col, f);
      else st_row<1>(db + col, f);
    }
    __syncthreads();
  }
}

template <typename P, typename T>
int launch(const void* dy, const void* z, void* dz, void* db, int db_f32, float* partial, int64_t rows, int width,
           int runs, int act, int vec, hipStream_t st) {
  const dim3 grid((unsigned)((width + 511) / 512), (unsigned)runs);
  const int64_t run = (rows + runs - 1) / runs;
  float* part = db ? partial : nullptr;
  if (vec)
    linear_dz_kernel<P, T, 8><<<grid, 256, 0, st>>>((const P*)dy, (const T*)z, (T*)dz, part, rows, width, run, act);
  else
    linear_dz_kernel<P, T, 1><<<grid, 256, 0, st>>>((const P*)dy, (const T*)z, (T*)dz, part, rows, width, run, act);
  if (db) {
    const unsigned blocks = (unsigned)std::min((width + 31) / 32, 1 << 21);  // a grid holds fewer than 2^32 threads
    linear_db_kernel<T><<<blocks, 1024, 0, st>>>(part, runs, width, db_f32 ? nullptr : (T*)db,
                                                 db_f32 ? (float*)db : nullptr);
  }
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// Runs of rows, hence rows of the partial sums.
int st_linear_dz_runs(int64_t rows, int width) {
  const int64_t cols = (width + 511) / 512, want = std::max<int64_t>(1, 1024 / cols);
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (rows + 15) / 16));
}

// dy [rows, width] fp32 (dy_f32) or 16-bit; z, dz 16-bit; db 16-bit or fp32; partial: runs * width
// floats where db is wanted.
int st_linear_dz(const void* dy, int dy_f32, const void* z, void* dz, void* db, int db_f32, float* partial,
                 int64_t rows, int width, int act, int f16, int vec, hipStream_t st) {
  if (rows <= 0 || width <= 0 || (vec && width % 8) || (db && !partial)) return -2;
  const int runs = st_linear_dz_runs(rows, width);
  if (f16)
    return dy_f32 ? launch<float, __half>(dy, z, dz, db, db_f32, partial, rows, width, runs, act, vec, st)
                  : launch<__half, __half>(dy, z, dz, db, db_f32, partial, rows, width, runs, act, vec, st);
  return dy_f32 ? launch<float, bf16_t>(dy, z, dz, db, db_f32, partial, rows, width, runs, act, vec, st)
                : launch<bf16_t, bf16_t>(dy, z, dz, db, db_f32, partial, rows, width, runs, act, vec, st);
}

}  // extern "C"
