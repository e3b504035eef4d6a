// The products of the backward of linear_act_wide.h, and the choice among all its instances.
#include "linear_act_wide.h"

namespace {

// vec, k in whole steps of 64 where an operand is kRow, an operand's 256 rows (kRow) or 64 rows of k
// (kCol) and 16 rows of C within 4 GiB, an activation only in the forward.
bool fits(const LinearArgs* p, int acol, int bcol) {
  if (p->M <= 0 || p->N <= 0 || p->K <= 0 || !p->vec || (acol && !bcol) || (bcol && p->epi.act)) return false;
  if ((!acol || !bcol) && p->K % BK) return false;
  const int64_t most = (int64_t)1 << 32, tiles = (int64_t)((p->M + BT - 1) / BT) * ((p->N + BT - 1) / BT);
  return tiles < 1 << 24 && p->epi.ldo * 64 + (int64_t)p->N * 4 < most &&
         (p->lda * (acol ? BK : BT) + (acol ? BT : p->K)) * 2 < most &&
         (p->ldb * (bcol ? BK : BT) + (bcol ? BT : p->K)) * 2 < most;
}

}  // namespace

extern "C" {

int st_linear_wide_bf16(const LinearArgs* p, hipStream_t st);
int st_linear_wide_f16(const LinearArgs* p, hipStream_t st);

// The time that a product would take here, in us; negative: outside the kernel's.
double st_linear_wide_us(const LinearArgs* p, int acol, int bcol) {
  if (!fits(p, acol, bcol)) return -1.0;
  return linear_wide_plan(p->M, p->N, p->K).us;
}

// fp32 workspace elements (p->ws) that a product uses; without them no tile is cut.
int64_t st_linear_wide_ws(const LinearArgs* p) {
  if (p->M <= 0 || p->N <= 0 || p->K <= 0) return 0;
  const WidePlan w = linear_wide_plan(p->M, p->N, p->K);
  const int nv = ((p->M + BT - 1) / BT) * ((p->N + BT - 1) / BT);
  return w.splits > 1 ? (int64_t)(nv - w.nfull) * w.splits * BT * BT : 0;
}

// C = A B^T with the epilogue, as st_linear_tile.  -2: outside the kernel's (fits).
int st_linear_wide(const LinearArgs* p, int acol, int bcol, hipStream_t st) {
  if (!fits(p, acol, bcol)) return -2;
  if (!bcol) return p->epi.f16 ? st_linear_wide_f16(p, st) : st_linear_wide_bf16(p, st);
  if (acol) return p->epi.f16 ? launch<true, true, true, 0>(*p, st) : launch<true, true, false, 0>(*p, st);
  return p->epi.f16 ? launch<false, true, true, 0>(*p, st) : launch<false, true, false, 0>(*p, st);
}

}  // extern "C"
