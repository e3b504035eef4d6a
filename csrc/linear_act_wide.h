// The product with its epilogue for large shapes (instances: linear_act_wide_*.hip): 256 x 256 tiles,
// one wave per SIMD, 128 x 128 a wave.
//
// Bound by the matrix instructions.  The schedule is csrc/gemm4w.hip's and csrc/wgrad4.hip's, for
// either layout of either operand: 64-k steps of both operands copied to LDS by DMA two steps
// ahead, a step's fragments of both 32-k halves in registers (128 VGPRs), 256 accumulators in AGPRs.
// A step runs its 128 MFMAs in a row; between them go the reads of the second half's fragments
// (MFMAs 0-31), a barrier at 20 that frees A's image for the copies of the step after next (21-56),
// one at 63 that frees B's and publishes the next step (copies 64-120), and the reads of the next
// step's first half (64-95).
//   kRow images: [256 rows][64 k], 16-byte chunk c of row r at c ^ ((r >> 1) & 7), read as b128.
//   kCol images: two of [64 k][128 rows], chunk c of row k at c ^ swz(k), read transposed.
// Rows of k behind a kCol operand's end arrive as zeros (the descriptor's range ends there); a kRow
// operand needs k in whole steps.  Rows of m and n behind the matrix compute values that are not stored.
// A lane holds 4 consecutive columns (operands swapped in the MFMA).
//
// Between two tiles: the next tile's first two steps are copied before this one's epilogue, so they
// arrive under it, and its first step does not wait for the epilogue's stores (vmcnt counts copies
// and stores in order).  The epilogue goes through buffer descriptors that end at the matrix, a row
// block of 16 at a time, so that nothing branches on the matrix' edge; the residual is requested two
// (fp32) or four row blocks ahead, in the registers that held the fragments.
//
// Where the tiles do not fill the last round of CUs, those left over are cut along k if that saves
// more steps than the fp32 sums' way through memory costs (linear_wide_plan); a second kernel adds
// the parts in order and runs their epilogue.
//
// Measured, bf16, kernel times of a trace of training passes, whose operands come from memory (ranges: cards
// differ by up to 4 %); in brackets the library's plain products in the same order.  24576 x 4096 x 14336 (2.89 TFLOP): y alone 2.36 ms (1.87),
// with bias, GELU and z 2.65, with tanh GELU, z and residual 2.75-2.79; dx 2.17-2.22 (2.12); dW 2.33-2.38 and 0.02
// for the sums of its cut tiles (2.87).  8192 x 1280 x 5120: y with bias, GELU and z 188 us (123), dx 135 (123), dW 117 and 17
// for the sums of its 100 cut tiles (141).  The chip holds its power limit here: the library's kernel keeps the
// matrix units 84 % busy at 1.75 GHz, this one 60 % at 1.93 and 50 % (epilogues) at 2.0, with no LDS conflicts
// and 16 % of the time in waits.  Lost to this schedule: both regions released at MFMA 40 and publication at 96
// (1-3 % slower), copies three MFMAs apart (6 %), other row groups (0-4 %), staggered workgroups (no change),
// 256 x 128 tiles with two workgroups a CU (1.0 PF/s).
#pragma once

#include <algorithm>
#include <type_traits>

#include "linear_act.h"

using namespace st;

namespace {

typedef __attribute__((address_space(3))) char lds_t;
typedef uint32_t srd_t __attribute__((ext_vector_type(4)));  // buffer descriptor, wave-uniform words

constexpr int BT = 256, BK = 64, NT = 256;
constexpr int IMG = BT * BK * 2;  // one operand of a step: 32 KiB
constexpr int STAGE = 2 * IMG;

ST_DEVICE int rsw(int r) { return (r >> 1) & 7; }
ST_DEVICE int swz(int k) { return ((k & 3) << 2) | ((k >> 2) & 3); }
ST_DEVICE void fence() { __builtin_amdgcn_sched_barrier(0); }

ST_DEVICE srd_t make_srd(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  srd_t w;
  w[0] = uni((uint32_t)a);
  w[1] = uni((uint32_t)(a >> 32)) & 0xffffu;
  w[2] = uni(bytes);
  w[3] = 0x00020000u;
  return w;
}

template <int B, int E, typename F>
ST_DEVICE void static_for(F&& f) {
  if constexpr (B < E) {
    f(std::integral_constant<int, B>());
    static_for<B + 1, E>(f);
  }
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: nothing else in this kernel uses it

// One operand: where a wave's 8 copies a step come from and go to, and where its fragments lie.
template <bool COL>
struct Side {
  uint32_t voff[8];          // of this lane's 16 bytes, from the descriptor's base
  int foff[COL ? 8 : 1][2];  // kCol: [fragment][half]; kRow: [0][32-k half]
  ST_DEVICE void init(int lane, int wid, int half, int64_t ld) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (COL) {  // copy i: image i / 4, rows of k 16 wid + 4 (i % 4) ..
        const int row = 16 * wid + 4 * (i & 3) + (lane >> 4), pos = lane & 15;
        voff[i] = (uint32_t)row * (uint32_t)(ld * 2) + (uint32_t)((i >> 2) * 256 + 16 * (pos ^ swz(row)));
      } else {  // copy i: rows (8 wid + i) 8 ..
        const int row = (wid * 8 + i) * 8 + (lane >> 3), pos = lane & 7;
        voff[i] = (uint32_t)row * (uint32_t)(ld * 2) + (uint32_t)(16 * (pos ^ rsw(row)));
      }
    }
    if constexpr (COL) {
      const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
#pragma unroll
      for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int k = 8 * g + 4 * hf + q;
          foff[f][hf] = half * (IMG / 2) + k * 256 + 16 * ((2 * f + (p >> 1)) ^ swz(k)) + 8 * (p & 1);
        }
    } else {
      const int q = lane >> 4, rl = lane & 15;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) foff[0][ks] = half * 128 * 128 + rl * 128 + (((4 * ks + q) ^ rsw(rl)) * 16);
    }
  }
  // LDS byte of copy i of this wave within the operand's image
  ST_DEVICE static uint32_t dst(int wid, int i) {
    return COL ? (uint32_t)((i >> 2) * (IMG / 2) + wid * 4096 + (i & 3) * 1024) : (uint32_t)(wid * 8192 + i * 1024);
  }
  ST_DEVICE u32x4 read(const lds_t* img, int ks, int f) const {
    if constexpr (COL) {
      u32x2 h[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        h[hf] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                              (bfx4 __attribute__((address_space(3)))*)(img + foff[f][hf] + ks * 32 * 256)));
      return u32x4{h[0][0], h[0][1], h[1][0], h[1][1]};
    } else {
      return *reinterpret_cast<const u32x4 __attribute__((address_space(3)))*>(img + f * 16 * 128 + foff[0][ks]);
    }
  }
  // descriptor and scalar offset of step kt: rows r0 .. of `rows`, K of k
  ST_DEVICE static void at(const uint16_t* base, int64_t ld, int r0, int rows, int K, int kt, srd_t& rs, uint32_t& so) {
    if constexpr (COL) {
      const int left = min(K - kt * BK, BK);
      rs = make_srd(base + (int64_t)kt * BK * ld + r0,
                    left > 0 ? (uint32_t)(((int64_t)(left - 1) * ld + min(BT, rows - r0)) * 2) : 0u);
      so = 0;
    } else {
      rs = make_srd(base + (int64_t)r0 * ld, (uint32_t)(((int64_t)(min(BT, rows - r0) - 1) * ld + K) * 2));
      so = uni((uint32_t)(kt * BK * 2));
    }
  }
};

template <bool ACOL, bool BCOL, bool F16, int ACT>
__global__ __launch_bounds__(NT, 1) void linear_wide_kernel(LinearArgs p, int gm, int nfull) {
  __shared__ __attribute__((aligned(16))) char smem_raw[2 * STAGE];
  lds_t* smem = (lds_t*)smem_raw;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int nbm = (p.M + BT - 1) / BT, nbn = (p.N + BT - 1) / BT, nv = nbm * nbn;
  const int KT = (p.K + BK - 1) / BK;
  const uint16_t* ga = (const uint16_t*)p.a;
  const uint16_t* gb = (const uint16_t*)p.b;
  Side<ACOL> sa;
  Side<BCOL> sb;
  sa.init(lane, wid, wm, p.lda);
  sb.init(lane, wid, wn, p.ldb);
  const uint32_t lbase = uni((uint32_t)(uintptr_t)smem);
  auto m0_of = [&](int buf, int i) {  // copy i < 8: A's, else B's
    return uni(lbase + buf * STAGE + (i < 8 ? Side<ACOL>::dst(wid, i) : IMG + Side<BCOL>::dst(wid, i - 8)));
  };
  auto set_m0 = [&](uint32_t v) { asm volatile("s_mov_b32 m0, %0" : : "s"(v) : "m0"); };
  struct Step {
    srd_t a, b;
    uint32_t soa, sob;
  };
  auto copy = [&](const Step& k, int i) {
    if (i < 8)
      asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(sa.voff[i]), "s"(k.a), "s"(k.soa) : "memory");
    else
      asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(sb.voff[i - 8]), "s"(k.b), "s"(k.sob) : "memory");
  };

  u32x4 fa[2][8], fb[2][8];
  auto read = [&](int buf, int ks, int r) {  // fragment r < 8: A's, else B's
    const lds_t* st = smem + buf * STAGE;
    if (r < 8) fa[ks][r] = sa.read(st, ks, r);
    else fb[ks][r - 8] = sb.read(st + IMG, ks, r - 8);
  };
  constexpr auto copy_slot = [](int m) constexpr -> int {
    if (m >= 21 && m <= 56 && (m - 21) % 5 == 0) return (m - 21) / 5;
    if (m >= 64 && m <= 120 && ((m - 64) & 7) == 0) return 8 + ((m - 64) >> 3);
    return -1;
  };

  // units of work: tiles 0 .. nfull - 1 whole, then the others as `splits` ranges of k each
  struct Unit {
    int m0, n0, kb, ke, part;  // part: of the workspace, -1 a whole tile
  };
  auto unit_of = [&](int u) {
    int vb = u;
    Unit r{0, 0, 0, KT, -1};
    if (u >= nfull) {
      const int t = u - nfull, tail = nv - nfull, sidx = t / tail;
      vb = nfull + t % tail;
      if (p.splits > 1) {
        r.kb = (int)((int64_t)sidx * KT / p.splits);
        r.ke = (int)((int64_t)(sidx + 1) * KT / p.splits);
        r.part = t;
      }
    }
    // XCD-aware: each XCD walks its own run of tiles, in groups of gm row blocks
    const int id = xcd_remap(vb, nv), per = gm * nbn, grp = id / per, in = id % per, gsz = min(gm, nbm - grp * gm);
    r.m0 = (grp * gm + in % gsz) * BT;
    r.n0 = (in / gsz) * BT;
    return r;
  };
  auto step_of = [&](const Unit& t, int kt) {
    Step s;
    Side<ACOL>::at(ga, p.lda, t.m0, p.M, p.K, kt, s.a, s.soa);
    Side<BCOL>::at(gb, p.ldb, t.n0, p.N, p.K, kt, s.b, s.sob);
    return s;
  };
  auto start = [&](const Unit& t) {  // its first two steps requested
    const Step s0 = step_of(t, t.kb);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      set_m0(m0_of(0, i));
      copy(s0, i);
    }
    if (t.ke - t.kb > 1) {
      const Step s1 = step_of(t, t.kb + 1);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        set_m0(m0_of(1, i));
        copy(s1, i);
      }
    }
  };
  const int nu = nfull + (nv - nfull) * p.splits;
  Unit cu = unit_of((int)blockIdx.x);
  start(cu);
  bool stores = false;  // at least 64 stores were issued after the copies of `start`
  for (int u = (int)blockIdx.x; u < nu; u += (int)gridDim.x) {
    f32x4 acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto mfma = [&](int ks, int idx) {
      const int i = idx >> 3, j = idx & 7;
      if constexpr (F16)
        asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(fb[ks][j]), "v"(fa[ks][i]));
      else
        asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(fb[ks][j]), "v"(fa[ks][i]));
    };
    const int steps = cu.ke - cu.kb;
    // the first step published, its first half's fragments read
    if (stores) asm volatile("s_waitcnt vmcnt(63)" ::: "memory");
    else if (steps > 1) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < 16; ++r) read(0, 0, r);
    auto step = [&](auto more_c, auto more2_c, int s) {  // s counts from the unit's first step
      constexpr bool more = decltype(more_c)::value, more2 = decltype(more2_c)::value;
      Step k2{};
      if constexpr (more2) k2 = step_of(cu, cu.kb + s + 2);
      const int cur = s & 1;
      __builtin_amdgcn_s_setprio(1);
      static_for<0, 128>([&](auto mc) {
        constexpr int m = decltype(mc)::value;
        mfma(m >> 6, m & 63);
        constexpr int now = copy_slot(m), soon = copy_slot(m + 2);
        if constexpr (m < 32 && (m & 1) == 0) {  // second half's fragment m / 2
          fence();
          read(cur, 1, m >> 1);
          fence();
        }
        if constexpr (m == 20 && more2) {  // A's 8 fragments read (B's first three may be in flight)
          fence();
          if constexpr (BCOL) asm volatile("s_waitcnt lgkmcnt(6)" ::: "memory");
          else asm volatile("s_waitcnt lgkmcnt(3)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          fence();
        }
        if constexpr (m == 63 && more) {
          fence();
          __builtin_amdgcn_s_setprio(0);
          if constexpr (more2) {
            // the next step's copies are older than A's 8 just issued -- and, in the first step behind
            // an epilogue, than its stores
            if (s == 0 && stores) asm volatile("s_waitcnt vmcnt(63) lgkmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
          } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          }
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_setprio(1);
          fence();
        }
        if constexpr (more2 && soon >= 0) {
          fence();
          set_m0(m0_of(cur, soon));
          fence();
        }
        if constexpr (more2 && now >= 0) {
          fence();
          copy(k2, now);
          fence();
        }
        if constexpr (more && m >= 64 && m < 96 && (m & 1) == 0) {  // next step's first half
          fence();
          read(cur ^ 1, 0, (m - 64) >> 1);
          fence();
        }
      });
      __builtin_amdgcn_s_setprio(0);
    };
    using T1 = std::true_type;
    using F0 = std::false_type;
    int s = 0;
    for (; s + 2 < steps; ++s) step(T1(), T1(), s);
    if (s + 1 < steps) step(T1(), F0(), s++);
    step(F0(), F0(), s);
    fence();
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");  // the last MFMAs' results
    fence();

    const Unit t = cu;
    const int next = u + (int)gridDim.x;
    if (next < nu) {
      // every wave has read its last fragments (its MFMAs took them): both stages are free
      __builtin_amdgcn_s_barrier();
      cu = unit_of(next);
      start(cu);
    }
    stores = true;
    if (t.part >= 0) {  // fp32 sums in the order of the registers; 64 stores
      f32x4* w = reinterpret_cast<f32x4*>(p.ws) + (int64_t)t.part * (BT * BT / 4) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) w[(i * 8 + j) * NT] = acc[i][j];
      continue;
    }
    const LinearEpi& e = p.epi;
    const int rl = lane & 15, q = lane >> 4, nc = t.n0 + wn * 128 + 4 * q;
    f32x4 bias[8];
    uint32_t at[8];  // byte of a lane's columns within 16 rows of 16-bit values; behind the matrix: out of range
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = nc + 16 * j < p.N;
      at[j] = in ? (uint32_t)(((int64_t)rl * e.ldo + nc + 16 * j) * 2) : kOut;
      bias[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (e.bias && in) bias[j] = unpack4(*reinterpret_cast<const u32x2*>((const uint16_t*)e.bias + nc + 16 * j), F16);
    }
    auto rows16 = [&](const void* base, int i, int size) {  // descriptor of row block i, ending with the matrix
      const int m = t.m0 + wm * 128 + 16 * i, left = max(0, min(16, p.M - m));
      return rsrc_of((const char*)base + (left ? (int64_t)m * e.ldo * size : 0), (uint32_t)((int64_t)left * e.ldo * size));
    };
    auto finish = [&](auto f32_c) {
      constexpr bool F32 = decltype(f32_c)::value;
      constexpr int AHEAD = F32 ? 2 : 4, W = F32 ? 4 : 2, SIZE = F32 ? 4 : 2;
      uint32_t res[AHEAD][8][W];
      auto request = [&](int i) {
        const rsrc_t rs = rows16(e.res, i, SIZE);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (F32) {
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, at[j] == kOut ? kOut : at[j] * 2, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) res[i % AHEAD][j][r] = v[r];
          } else {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, at[j], 0, 0);
            res[i % AHEAD][j][0] = v[0];
            res[i % AHEAD][j][1] = v[1];
          }
        }
      };
      if (e.res)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) request(i);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f32x4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[i][j] + bias[j];
        if (e.z) {
          const rsrc_t rs = rows16(e.z, i, 2);
#pragma unroll
          for (int j = 0; j < 8; ++j) __builtin_amdgcn_raw_buffer_store_b64(pack4(v[j], F16), rs, at[j], 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[j][r] = act_of(v[j][r], ACT);
        if (e.res) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (F32) {
#pragma unroll
              for (int r = 0; r < 4; ++r) v[j][r] += __uint_as_float(res[i % AHEAD][j][r]);
            } else {
              v[j] += unpack4(u32x2{res[i % AHEAD][j][0], res[i % AHEAD][j][1]}, F16);
            }
          }
          if (i + AHEAD < 8) request(i + AHEAD);
        }
        const rsrc_t rs = rows16(e.out, i, SIZE);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (F32)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[j]), rs, at[j] == kOut ? kOut : at[j] * 2,
                                                   0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b64(pack4(v[j], F16), rs, at[j], 0, 0);
        }
      }
    };
    if (e.out_f32) finish(T1());
    else finish(F0());
  }
}
#pragma clang diagnostic pop

// The parts of the cut tiles, in order, then their epilogue: an (i, j) block of a tile a workgroup.
// Neighbouring 16 x 16 blocks of a workgroup: it then writes whole 128-byte lines.  100 tiles of two parts (52 MB)
// take 17 us in a training pass; called again and again 13, and with one block each, whose lines belong to
// several XCDs, 27.
constexpr int kJoin = 4;
__global__ __launch_bounds__(NT) void linear_wide_join_kernel(LinearArgs p, int gm, int nfull) {
  const int nbm = (p.M + BT - 1) / BT, nbn = (p.N + BT - 1) / BT, nv = nbm * nbn, tail = nv - nfull;
  const int id = xcd_remap(nfull + (int)blockIdx.x, nv), per = gm * nbn, grp = id / per, in = id % per;
  const int gsz = min(gm, nbm - grp * gm);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int m0 = (grp * gm + in % gsz) * BT + (wid >> 1) * 128 + (lane & 15);
  const int n0 = (in / gsz) * BT + (wid & 1) * 128 + 4 * (lane >> 4);
  const int ij = (int)blockIdx.y * kJoin, m = m0 + 16 * (ij >> 3), n = n0 + 16 * (ij & 7);
  const f32x4* w = reinterpret_cast<const f32x4*>(p.ws) + (int64_t)blockIdx.x * (BT * BT / 4) + ij * NT + threadIdx.x;
  f32x4 part[8][kJoin];  // all requested before the first sum
#pragma unroll
  for (int s = 0; s < 8; ++s)
    if (s < p.splits)
#pragma unroll
      for (int j = 0; j < kJoin; ++j) part[s][j] = w[(int64_t)s * tail * (BT * BT / 4) + j * NT];
#pragma unroll
  for (int j = 0; j < kJoin; ++j) {
    f32x4 v = part[0][j];
#pragma unroll
    for (int s = 1; s < 8; ++s)
      if (s < p.splits) v += part[s][j];
    if (m < p.M && n + 16 * j < p.N) epilogue4(p.epi, m, n + 16 * j, p.N - n - 16 * j, true, v);
  }
}

int cu_count() {
  static int cache[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!cache[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

// Tiles that are done whole, the parts that each of the others is cut into, and the time to expect.
// Measured: a step of a tile takes some 1.6 us (24576 x 4096 x 14336), a round's epilogue 8, or 13 where
// it writes fp32 parts, the way to the first step 7; the second kernel reads the parts at some 4 TB/s and
// costs 6 us more.
constexpr int kGroup = 4;
struct WidePlan {
  int nfull, splits;
  double us;
};
WidePlan linear_wide_plan(int M, int N, int K) {
  const int cus = cu_count(), KT = (K + BK - 1) / BK;
  const int nv = ((M + BT - 1) / BT) * ((N + BT - 1) / BT), tail = nv % cus, rounds = (nv + cus - 1) / cus;
  WidePlan best{nv, 1, 7.0 + rounds * (8.0 + 1.6 * KT)};
  for (int s = 2; tail && s <= 8 && KT / s >= 4; ++s) {
    const int parts = (tail * s + cus - 1) / cus;
    const double us = 7.0 + (rounds - 1) * (8.0 + 1.6 * KT) + parts * (13.0 + 1.6 * ((KT + s - 1) / s)) + 6.0 + tail * s * 0.2621 / 4.0;
    if (us < best.us) best = WidePlan{nv - tail, s, us};
  }
  return best;
}

template <bool ACOL, bool BCOL, bool F16, int ACT>
int launch(const LinearArgs& p, hipStream_t st) {
  WidePlan w = linear_wide_plan(p.M, p.N, p.K);
  const int nv = ((p.M + BT - 1) / BT) * ((p.N + BT - 1) / BT);
  if (!p.ws) w = WidePlan{nv, 1, 0.0};
  LinearArgs q = p;
  q.splits = w.splits;
  const int nu = w.nfull + (nv - w.nfull) * w.splits;
  const unsigned grid = (unsigned)std::min(nu, cu_count());
  linear_wide_kernel<ACOL, BCOL, F16, ACT><<<grid, NT, 0, st>>>(q, kGroup, w.nfull);
  if (w.splits > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    linear_wide_join_kernel<<<dim3((unsigned)(nv - w.nfull), 64 / kJoin), NT, 0, st>>>(q, kGroup, w.nfull);
  }
  return (int)hipGetLastError();
}

}  // namespace
