// The forward product for few rows (up to 64): bound by reading the weight once.
//
// A workgroup owns 16 output columns, its four waves the quarters of k: every wave streams its part
// of the 16 weight rows straight into MFMA fragments (16 bytes a lane, eight loads in flight; no
// LDS), multiplies them with the rows of x, which come from L2, and the four partial tiles are added
// through LDS in order before the epilogue.  With 4096 x 14336 that is 896 workgroups of 32 steps:
// 26.3 us for one row, 4.5 TB/s of weight (a copy reaches 4.9; four and sixteen loads in flight
// instead of eight take 26.7 and 26.4).
#include "linear_act.h"

using namespace st;

namespace {

template <bool F16>
ST_DEVICE f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hx8, a), __builtin_bit_cast(hx8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfx8, a), __builtin_bit_cast(bfx8, b), c, 0, 0, 0);
}

// MB: groups of 16 rows of x
template <int MB, bool F16>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinearArgs p) {
  constexpr int U = MB <= 2 ? 8 : 4;  // steps of 32 k whose loads are in flight together
  __shared__ f32x4 part[3][MB][64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (int)blockIdx.x * 16, rl = lane & 15, g = lane >> 4;
  const int steps = (p.K + 31) / 32, s1 = (int)((int64_t)(wid + 1) * steps / 4);
  const bool nin = n0 + rl < p.N;
  const uint16_t* w = (const uint16_t*)p.b + (int64_t)(n0 + rl) * p.ldb + 8 * g;
  const uint16_t* x[MB];
  bool min_[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    min_[i] = 16 * i + rl < p.M;
    x[i] = (const uint16_t*)p.a + (int64_t)(16 * i + rl) * p.lda + 8 * g;
  }
  f32x4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u32x4 none = {0u, 0u, 0u, 0u};
  for (int s = (int)((int64_t)wid * steps / 4); s < s1; s += U) {
    u32x4 fw[U], fx[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (int64_t)(s + u) * 32;
      const bool kin = s + u < s1 && k + 8 * g < p.K;  // K % 8 == 0: the 8 are all in or all out
      fw[u] = none;
      if (kin && nin) fw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w + k));
#pragma unroll
      for (int i = 0; i < MB; ++i) fx[u][i] = kin && min_[i] ? *reinterpret_cast<const u32x4*>(x[i] + k) : none;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i] = mfma<F16>(fw[u], fx[u][i], acc[i]);
  }
  if (wid)
#pragma unroll
    for (int i = 0; i < MB; ++i) part[wid - 1][i][lane] = acc[i];
  __syncthreads();
  if (wid) return;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    f32x4 v = acc[i];
#pragma unroll
    for (int k = 0; k < 3; ++k) v += part[k][i][lane];
    const int m = 16 * i + rl, n = n0 + 4 * g;
    if (m < p.M && n < p.N) epilogue4(p.epi, m, n, p.N - n, true, v);
  }
}

template <int MB>
int launch(const LinearArgs& p, hipStream_t st) {
  const unsigned grid = (unsigned)((p.N + 15) / 16);
  if (p.epi.f16) linear_rows_kernel<MB, true><<<grid, 256, 0, st>>>(p);
  else linear_rows_kernel<MB, false><<<grid, 256, 0, st>>>(p);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// Forward products (both operands kRow) of up to 64 rows, vec.  -2: outside the kernel's.
int st_linear_rows(const LinearArgs* p, hipStream_t st) {
  if (p->M <= 0 || p->M > 64 || p->N <= 0 || p->K <= 0 || !p->vec || p->K % 8 || p->N % 4) return -2;
  if (p->N > 1 << 27) return -2;  // 2^32 threads is a grid's limit
  if (p->M <= 16) return launch<1>(*p, st);
  if (p->M <= 32) return launch<2>(*p, st);
  return launch<4>(*p, st);
}

}  // extern "C"
