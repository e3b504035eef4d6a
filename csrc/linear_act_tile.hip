// The product with its epilogue for every shape: BM x BN tiles, 2 x 2 waves, k in steps of 64.
//
// A step's operands go global -> registers (16-byte loads, from any element where rows are not aligned),
// issued several steps ahead (a step of a small tile computes for 0.1 us, a load takes one), then to one of
// two LDS images, from which the waves read their MFMA fragments; one barrier a step.  kRow images are
// [rows][64 k], 16-byte chunk c of row r at c ^ ((r >> 1) & 7); kCol images [64 k][rows] in 256-byte
// (64-column tiles: 128-byte) rows, read with the transposing LDS read, chunk c of row k at c ^ swz(k).
// Chunks behind an operand's end are zeros.  Few tiles: k is split over workgroups, whose fp32 sums a second
// kernel adds up in order before the epilogue.
//
// Bound by a step's chain (LDS writes, barrier, fragments: 0.27 us for a 64 x 64 tile alone on its CU, of it
// 0.06 of matrix instructions) where there are few tiles, by the L1s where several share a CU.  Measured,
// bf16: 2048^3 33 us (520 TF/s; the library's product 26), its gradients 31 (28-30), 1024^3 9 us (21-25),
// 64 x 4096 x 14336 22 us (24), 777 x 1000 x 2504 with the epilogue 20 us (22 alone), 777 x 1001 x 2503 25 us,
// 24576 x 4096 x 14336 3.1 ms (930 TF/s).  With loads that some paths skip every fourth step of the loop
// waited for all of them: dx of 2048^3 took 33 us and not 29-31.
#include <algorithm>
#include <type_traits>

#include "linear_act.h"

using namespace st;

namespace {

constexpr int BK = 64, NT = 256;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;  // 16 bytes at any element
typedef __attribute__((address_space(3))) char lds_t;

template <bool F16>
ST_DEVICE f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hx8, a), __builtin_bit_cast(hx8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfx8, a), __builtin_bit_cast(bfx8, b), c, 0, 0, 0);
}

// One operand of a tile: R rows (m or n), layout COL.
//
// Loads never branch, so that several steps of them stay in flight (behind a branch the compiler
// waits for all of them).  VEC: through a buffer descriptor, lanes behind the operand's end at an
// offset that reads as zero.  Else: 16 bytes from any element, moved back where they would run past
// the operand's last one; the shift and the zeros follow when the chunk goes to LDS.
template <int R, bool COL, bool VEC>
struct Operand {
  static constexpr int kChunks = R * BK / 8 / NT;  // 16-byte chunks a thread moves
  static constexpr int kBytes = R * BK * 2;
  typedef u32x4 Regs[kChunks];  // one step's part of a thread
  const uint16_t* base;         // of the tile's first row
  int64_t ld, span;             // elements between rows (k), and from base to the operand's end
  int rows, K;                  // rows from the tile's first on, all of k

  ST_DEVICE static int swz(int k) {  // kCol: spreads the 16 k rows of a transposed read over the banks
    return R == 128 ? ((k & 3) << 2) | ((k >> 2) & 3) : ((k & 1) << 2) | ((k >> 1) & 3);
  }
  // row and k (within the step) of chunk i of this thread
  ST_DEVICE static int row_of(int i) {
    const int c = threadIdx.x + NT * i;
    return COL ? (c % (R / 8)) * 8 : c >> 3;
  }
  ST_DEVICE static int k_of(int i) {
    const int c = threadIdx.x + NT * i;
    return COL ? c / (R / 8) : (c & 7) * 8;
  }
  ST_DEVICE static int lds_at(int i) {  // its byte in the image
    const int r = row_of(i), k = k_of(i);
    return COL ? k * (R * 2) + 16 * ((r >> 3) ^ swz(k)) : r * 128 + 16 * ((k >> 3) ^ ((r >> 1) & 7));
  }
  ST_DEVICE int64_t at(int i, int k0) const {
    return COL ? (int64_t)(k0 + k_of(i)) * ld + row_of(i) : (int64_t)row_of(i) * ld + k0 + k_of(i);
  }
  ST_DEVICE int left(int i, int k0) const {  // elements of the chunk inside the operand; may be over 8 or below 0
    return COL ? (k0 + k_of(i) < K ? rows - row_of(i) : 0) : (row_of(i) < rows ? K - k0 - k_of(i) : 0);
  }
  ST_DEVICE void load(int k0, Regs& reg) const {
    if constexpr (VEC) {
      const int most = min(R, rows), so = COL || k0 >= K ? 0 : k0 * 2;  // the scalar offset: inside the range, as kOut's test needs
      const rsrc_t rs = COL ? rsrc_of(base + (int64_t)k0 * ld, k0 < K ? (uint32_t)(((int64_t)(min(BK, K - k0) - 1) * ld + most) * 2) : 0u)
                            : rsrc_of(base, (uint32_t)(((int64_t)(most - 1) * ld + K) * 2));
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const uint32_t off = (uint32_t)(((COL ? (int64_t)k_of(i) * ld + row_of(i) : (int64_t)row_of(i) * ld + k_of(i)) * 2));
        reg[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, left(i, k0) > 0 ? off : kOut, so, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int64_t a = left(i, k0) > 0 ? at(i, k0) : 0;
        reg[i] = *reinterpret_cast<const u32x4_any*>(base + min(a, span - 8));  // the operand has 8 elements or more
      }
    }
  }
  ST_DEVICE void store(lds_t* img, int k0, const Regs& reg) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      u32x4 v = reg[i];
      if constexpr (!VEC) {
        const int n = left(i, k0), d = n > 0 ? (int)max((int64_t)0, at(i, k0) - (span - 8)) : 0;
        uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
        if (d > 0) {  // the chunk was read d elements early
          lo = d >= 4 ? hi >> (16 * (d & 3)) : lo >> (16 * d) | hi << (64 - 16 * d);
          hi = d >= 4 ? 0 : hi >> (16 * d);
        }
        if (n < 8) {
          hi = n > 4 ? hi & ~(~0ull << (16 * (n - 4))) : 0;
          lo = n >= 4 ? lo : n > 0 ? lo & ~(~0ull << (16 * n)) : 0;
        }
        v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
      *reinterpret_cast<u32x4 __attribute__((address_space(3)))*>(img + lds_at(i)) = v;
    }
  }
  // fragment of rows r0 .. r0 + 15, k 32 ks .. + 31: lane (g = lane / 16) holds k 8 g .. 8 g + 7 of row lane % 16
  ST_DEVICE static u32x4 frag(const lds_t* img, int r0, int ks) {
    const int lane = threadIdx.x & 63;
    if constexpr (COL) {
      const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
      u32x2 h[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int k = 32 * ks + 8 * g + 4 * hf + q, col = r0 + 4 * p;
        const lds_t* at = img + k * (R * 2) + 16 * ((col >> 3) ^ swz(k)) + 2 * (col & 7);
        h[hf] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bfx4 __attribute__((address_space(3)))*)at));
      }
      return u32x4{h[0][0], h[0][1], h[1][0], h[1][1]};
    } else {
      const int r = r0 + (lane & 15), c = 4 * ks + (lane >> 4);
      return *reinterpret_cast<const u32x4 __attribute__((address_space(3)))*>(img + r * 128 +
                                                                              16 * (c ^ ((r >> 1) & 7)));
    }
  }
};

// AHEAD: steps whose loads are in flight in registers (even: the LDS image of a step is then known)
template <int BM, int BN, int AHEAD, bool ACOL, bool BCOL, bool VEC, bool F16>
__global__ __launch_bounds__(NT) void linear_tile_kernel(LinearArgs p) {
  constexpr int WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
  typedef Operand<BM, ACOL, VEC> OpA;
  typedef Operand<BN, BCOL, VEC> OpB;
  __shared__ __attribute__((aligned(16))) char smem_raw[2 * (OpA::kBytes + OpB::kBytes)];
  lds_t* smem = (lds_t*)smem_raw;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int nbn = (p.N + BN - 1) / BN, nbm = (p.M + BM - 1) / BM;
  const uint32_t wg = blockIdx.z * gridDim.x + blockIdx.x;  // launch: the tiles over x and z
  if (wg >= (uint32_t)(nbm * nbn)) return;
  const int vb = xcd_remap((int)wg, nbm * nbn);
  // groups of 8 row blocks: the tiles an XCD holds at once share operand slices in its L2
  const int per = 8 * nbn, grp = vb / per, in = vb % per, gsz = min(8, nbm - grp * 8);
  const int m0 = (grp * 8 + in % gsz) * BM, n0 = (in / gsz) * BN;
  // this workgroup's part of k, whole steps
  const int steps = (p.K + BK - 1) / BK, split = (int)blockIdx.y;
  const int s0 = (int)((int64_t)split * steps / p.splits), s1 = (int)((int64_t)(split + 1) * steps / p.splits);
  OpA A;
  OpB B;
  A.base = (const uint16_t*)p.a + (ACOL ? (int64_t)m0 : (int64_t)m0 * p.lda);
  B.base = (const uint16_t*)p.b + (BCOL ? (int64_t)n0 : (int64_t)n0 * p.ldb);
  A.ld = p.lda;
  B.ld = p.ldb;
  A.rows = p.M - m0;
  B.rows = p.N - n0;
  A.K = B.K = p.K;
  A.span = ACOL ? (int64_t)(p.K - 1) * p.lda + A.rows : (int64_t)(A.rows - 1) * p.lda + p.K;
  B.span = BCOL ? (int64_t)(p.K - 1) * p.ldb + B.rows : (int64_t)(B.rows - 1) * p.ldb + p.K;
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kStage = OpA::kBytes + OpB::kBytes;
  typename OpA::Regs ra[AHEAD];
  typename OpB::Regs rb[AHEAD];
  const int n = s1 - s0;
  // Steps behind the last are loaded too (zeros behind k's end, or the next part's values, which nothing
  // reads): where loads are skipped on some path the compiler waits as if none had followed.
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    A.load((s0 + j) * BK, ra[j]);
    B.load((s0 + j) * BK, rb[j]);
    __builtin_amdgcn_sched_barrier(0);  // in this order: the loop's waits count on it
  }
  // step i's operands from registers i % AHEAD to image i % 2, and the registers on to step i + AHEAD
  typedef std::true_type More;
  typedef std::false_type Last;
  auto stage = [&](auto j_c, auto more, int i) {
    constexpr int j = decltype(j_c)::value;
    A.store(smem + (j & 1) * kStage, (s0 + i) * BK, ra[j]);
    B.store(smem + (j & 1) * kStage + OpA::kBytes, (s0 + i) * BK, rb[j]);
    if constexpr (decltype(more)::value) {
      A.load((s0 + i + AHEAD) * BK, ra[j]);
      B.load((s0 + i + AHEAD) * BK, rb[j]);
    }
  };
  stage(std::integral_constant<int, 0>(), More(), 0);
  __syncthreads();
  auto step = [&](auto j_c, auto more, int i) {
    constexpr int j = decltype(j_c)::value;
    const lds_t* cur = smem + (j & 1) * kStage;
    // the other image was read a step ago, before the last barrier
    stage(std::integral_constant<int, (j + 1) % AHEAD>(), more, i + 1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 fa[FM], fb[FN];
#pragma unroll
      for (int q = 0; q < FM; ++q) fa[q] = OpA::frag(cur, wm * WM + 16 * q, ks);
#pragma unroll
      for (int q = 0; q < FN; ++q) fb[q] = OpB::frag(cur + OpA::kBytes, wn * WN + 16 * q, ks);
      // operands swapped: a lane holds 4 consecutive columns of one row
#pragma unroll
      for (int q = 0; q < FM; ++q)
#pragma unroll
        for (int r = 0; r < FN; ++r) acc[q][r] = mfma<F16>(fb[r], fa[q], acc[q][r]);
    }
    __syncthreads();
  };
  int i = 0;
  for (; i + AHEAD <= n; i += AHEAD) {  // one way through: a way out of its middle would count as skipped loads too
    step(std::integral_constant<int, 0>(), More(), i);
    step(std::integral_constant<int, 1>(), More(), i + 1);
    if constexpr (AHEAD > 2) {
      step(std::integral_constant<int, 2>(), More(), i + 2);
      step(std::integral_constant<int, 3>(), More(), i + 3);
    }
  }
  if (i < n) step(std::integral_constant<int, 0>(), Last(), i);
  if constexpr (AHEAD > 2) {
    if (i + 1 < n) step(std::integral_constant<int, 1>(), Last(), i + 1);
    if (i + 2 < n) step(std::integral_constant<int, 2>(), Last(), i + 2);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm * WM + 16 * i + (lane & 15);
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn * WN + 16 * j + 4 * (lane >> 4);
      if (n >= p.N) continue;
      if (p.splits > 1) {
        float* w = p.ws + ((int64_t)split * p.M + m) * p.N + n;
        if (VEC) {
          *reinterpret_cast<f32x4*>(w) = acc[i][j];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < p.N) w[r] = acc[i][j][r];
        }
      } else {
        epilogue4(p.epi, m, n, p.N - n, VEC, acc[i][j]);
      }
    }
  }
}

// The partial sums of the splits in order, then the epilogue; four columns a thread.
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs p) {
  const int quads = (p.N + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = id / quads;
  const int n = (int)(id % quads) * 4;
  if (m >= p.M) return;
  const float* w = p.ws + m * p.N + n;
  const int64_t step = (int64_t)p.M * p.N;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s, w += step) {
    if (p.vec) {
      v += *reinterpret_cast<const f32x4*>(w);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.N) v[r] += w[r];
    }
  }
  epilogue4(p.epi, m, n, p.N - n, p.vec != 0, v);
}

template <int BM, int BN, bool ACOL, bool BCOL, int AHEAD = BM + BN < 256 ? 4 : 2>
int launch(const LinearArgs& p, hipStream_t st) {
  const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles >= (1LL << 31)) return -2;
  const int64_t most = 1 << 23;  // a dimension of a grid holds fewer than 2^32 threads
  const dim3 grid((unsigned)std::min(tiles, most), (unsigned)p.splits, (unsigned)((tiles + most - 1) / most));
  if (p.vec) {
    if (p.epi.f16) linear_tile_kernel<BM, BN, AHEAD, ACOL, BCOL, true, true><<<grid, NT, 0, st>>>(p);
    else linear_tile_kernel<BM, BN, AHEAD, ACOL, BCOL, true, false><<<grid, NT, 0, st>>>(p);
  } else if constexpr (BM + BN == 128) {
    if (p.epi.f16) linear_tile_kernel<BM, BN, AHEAD, ACOL, BCOL, false, true><<<grid, NT, 0, st>>>(p);
    else linear_tile_kernel<BM, BN, AHEAD, ACOL, BCOL, false, false><<<grid, NT, 0, st>>>(p);
  }
  if (p.splits > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    const int64_t blocks = ((int64_t)p.M * ((p.N + 3) / 4) + 255) / 256;
    if (blocks >= (1LL << 31)) return -2;
    linear_join_kernel<<<(unsigned)blocks, 256, 0, st>>>(p);
  }
  return (int)hipGetLastError();
}

// Tile and splits of a product.  Measured, us, in 64 x 64 / 64 x 128 / 128 x 128 tiles:
//   y with bias and GELU: 2048 x 1536 x 2048 29 / 29 / 34, 3000 x 1024 x 3000 45 / 49 / 53, 4096 x 1024 x 4096
//     75 / 75 / 67 (a small tile's epilogue hides behind the other tiles of its CU);
//   dx: 2048 x 2304 x 768 23 / 21 / 30, 2048 x 2048 x 512 15 / 19 / 28, 2048^3 38 / 30 / 29;
//   dW: 2304 x 2048 x 768 27 / 23 / 29, 2048 x 2048 x 512 19 / 23 / 29, 2048^3 48 / 33 / 31.
// Splits (64 x 64; one, two, four): 512 x 4096 x 1024 21 / 16 / 17, 1000 x 4096 x 1000 22 / 24 / 26, 512 x 1024 x
// 1024 8 / 10 / 13; dW 768 x 4096 x 768 32 / 30 / 25 (three: 23), 256 x 2048 x 256 18 / 13 / 11.
struct Plan {
  int bm, bn, splits;
  double us;  // the time to expect
};
Plan plan(int M, int N, int K, int vec, int acol, int bcol) {
  auto tiles = [&](int bm, int bn) { return (int64_t)((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  Plan r{64, 64, 1, 1e30};
  if (vec) {  // shifted loads leave larger tiles no registers
    if (tiles(128, 128) >= (bcol ? 192 : 768)) r.bm = r.bn = 128;
    else if (bcol && tiles(64, 64) > 256) r.bn = 128;
  }
  // us of a step: 64 x 64 0.27 (0.42 with a transposed A, 0.8 with shifted loads), 64 x 128 0.5, 128 x 128 0.8;
  // several tiles on a CU take 0.85 (0.6) of their sum, epilogues of 128 x 128 2 a round, the second kernel 3 and
  // its sums at 4 TB/s.
  const int steps = (K + BK - 1) / BK;
  const double more = vec ? 0.85 : 0.6;
  const double step = !vec || r.bm == 128 ? 0.8 : r.bn == 128 ? 0.5 : acol ? 0.42 : 0.27;
  for (int s = 1; s <= 32 && (s == 1 || steps / s >= 4); ++s) {
    const double rounds = (double)((tiles(r.bm, r.bn) * s + 255) / 256);
    const double us = 4.0 + (steps + s - 1) / s * step * std::max(1.0, more * rounds) +
                      (r.bm == 128 && !bcol ? 2.0 * rounds : 0.0) + (s > 1 ? 3.0 + 2e-6 * s * M * N : 0.0);
    if (us < r.us) {
      r.us = us;
      r.splits = s;
    }
  }
  return r;
}

}  // namespace

extern "C" {

// The time in us that a product is expected to take here.
double st_linear_tile_us(int M, int N, int K, int vec, int acol, int bcol) { return plan(M, N, K, vec, acol, bcol).us; }

// fp32 workspace elements of a product.
int64_t st_linear_tile_ws(int M, int N, int K, int vec, int acol, int bcol) {
  const Plan r = plan(M, N, K, vec, acol, bcol);
  return r.splits > 1 ? (int64_t)r.splits * M * N : 0;
}

// C = A B^T with the epilogue; acol / bcol: the operand's rows are contiguous.  ws: st_linear_tile_ws
// floats.  -2: outside the kernel's.
int st_linear_tile(LinearArgs* p, int acol, int bcol, hipStream_t st) {
  if (p->M <= 0 || p->N <= 0 || p->K <= 0 || (acol && !bcol)) return -2;
  const Plan r = plan(p->M, p->N, p->K, p->vec, acol, bcol);
  p->splits = r.splits;
  if (r.splits > 1 && !p->ws) return -2;
  if (!bcol) return r.bm == 128 ? launch<128, 128, false, false>(*p, st) : launch<64, 64, false, false>(*p, st);
  if (r.bm == 128) return acol ? launch<128, 128, true, true>(*p, st) : launch<128, 128, false, true>(*p, st);
  if (r.bn == 128) return acol ? launch<64, 128, true, true>(*p, st) : launch<64, 128, false, true>(*p, st);
  return acol ? launch<64, 64, true, true>(*p, st) : launch<64, 64, false, true>(*p, st);
}

}  // extern "C"
