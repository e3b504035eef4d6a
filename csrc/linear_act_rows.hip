// The forward product for up to 16 rows: bound by reading the weight once.
//
// A workgroup owns 16 or 32 output columns, its four waves the quarters of k: every wave streams its part
// of the weight rows straight into MFMA fragments (16 bytes a lane, two sets of loads in flight; no
// LDS), multiplies them with the rows of x, which come from L2, and the four partial tiles are added
// through LDS in order before the epilogue.  32 columns read x half as often, but have to be enough
// workgroups: 4096 -> 14336 one row 25.7 us (4.6 TB/s of weight; a copy reaches 4.9) against 27.1, sixteen
// rows 31 against 35; 4096 -> 4096 13 against 8.  With loads behind branches and one set of them it
// was 26.4 and 37, and 10.
#include <type_traits>

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

// NB: groups of 16 columns a wave
template <int NB, bool F16>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinearArgs p) {
  constexpr int U = 8 / NB;  // steps of 32 k whose loads are requested together, two such sets in flight
  __shared__ f32x4 part[3][NB][64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (int)blockIdx.x * 16 * NB, rl = lane & 15, g = lane >> 4;
  const int steps = (p.K + 31) / 32, s0 = (int)((int64_t)wid * steps / 4), s1 = (int)((int64_t)(wid + 1) * steps / 4);
  const int cols = min(16 * NB, p.N - n0);
  const rsrc_t rw = rsrc_of((const uint16_t*)p.b + (int64_t)n0 * p.ldb, (uint32_t)(((int64_t)(cols - 1) * p.ldb + p.K) * 2));
  const rsrc_t rx = rsrc_of(p.a, (uint32_t)(((int64_t)(p.M - 1) * p.lda + p.K) * 2));
  uint32_t ow[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) ow[b] = 16 * b + rl < cols ? (uint32_t)(((int64_t)(16 * b + rl) * p.ldb + 8 * g) * 2) : kOut;
  const uint32_t ox = rl < p.M ? (uint32_t)(((int64_t)rl * p.lda + 8 * g) * 2) : kOut;
  f32x4 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 fw[2][U][NB], fx[2][U];
  // steps behind the part's last read as zeros: no load is skipped, so the waits count the ones that follow
  auto request = [&](auto set, int s) {
    constexpr int h = decltype(set)::value;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = s + u < s1 && (s + u) * 32 + 8 * g < p.K;  // K % 8 == 0: the 8 are all in or all out
      const int k2 = min(s + u, steps - 1) * 64;  // inside both ranges: a scalar offset past a range's end would wrap the test of kOut
#pragma unroll
      for (int b = 0; b < NB; ++b)  // 2: non-temporal
        fw[h][u][b] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? ow[b] : kOut, k2, 2);
      fx[h][u] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? ox : kOut, k2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](auto set) {
    constexpr int h = decltype(set)::value;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = mfma<F16>(fw[h][u][b], fx[h][u], acc[b]);
    __builtin_amdgcn_sched_barrier(0);
  };
  typedef std::integral_constant<int, 0> S0;
  typedef std::integral_constant<int, 1> S1;
  request(S0(), s0);
  for (int s = s0; s < s1; s += 2 * U) {
    request(S1(), s + U);
    multiply(S0());
    request(S0(), s + 2 * U);
    multiply(S1());
  }
  if (wid)
#pragma unroll
    for (int b = 0; b < NB; ++b) part[wid - 1][b][lane] = acc[b];
  __syncthreads();
  if (wid) return;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f32x4 v = acc[b];
#pragma unroll
    for (int k = 0; k < 3; ++k) v += part[k][b][lane];
    const int n = n0 + 16 * b + 4 * g;
    if (rl < p.M && n < p.N) epilogue4(p.epi, rl, n, p.N - n, true, v);
  }
}

template <int NB>
int launch(const LinearArgs& p, hipStream_t st) {
  const unsigned grid = (unsigned)((p.N + 16 * NB - 1) / (16 * NB));
  if (p.epi.f16) linear_rows_kernel<NB, true><<<grid, 256, 0, st>>>(p);
  else linear_rows_kernel<NB, false><<<grid, 256, 0, st>>>(p);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// Forward products (both operands kRow) of up to 16 rows, vec.  -2: outside the kernel's.
int st_linear_rows(const LinearArgs* p, hipStream_t st) {
  if (p->M <= 0 || p->M > 16 || p->N <= 0 || p->K <= 0 || !p->vec || p->K % 8 || p->N % 4) return -2;
  if (p->N > 1 << 27) return -2;  // 2^32 threads is a grid's limit
  return p->N >= 8192 ? launch<2>(*p, st) : launch<1>(*p, st);  // 32 columns for each of 256 CUs
}

}  // extern "C"
