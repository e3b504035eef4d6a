// torch.ops.st_amd.block_norm_*: host side of the norms around a block's gated residual
// (csrc/block_norm_fwd.hip, csrc/block_norm_bwd.hip).
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_norm_args.h"

using st::NormArgs;

extern "C" {
int st_block_norm_fwd(const NormArgs* a, int htype, int stype, int vec, hipStream_t st);
int st_block_norm_bwd_blocks(int64_t rows, int width);
int st_block_norm_bwd(const NormArgs* a, int gen, int bias, int blocks, int htype, int stype, int vec, hipStream_t st);
int st_block_norm_finish(const NormArgs* a, int gen, int bias, int blocks, void* const* out, const int* out_f32,
                         float* gate_part, int htype, hipStream_t st);
}

namespace {

typedef c10::optional<at::Tensor> opt;

int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return st::kF32;
    case at::kBFloat16: return st::kBF16;
    case at::kHalf: return st::kF16;
    default: TORCH_CHECK(false, "block_norm: fp32, bf16 or fp16 tensors, got ", t.scalar_type());
  }
  return -1;
}

bool has(const opt& t) { return t.has_value() && t->defined(); }

// Fills what both directions share and checks it against the rows' tensor `ref` (of h's or y's shape).
struct Call {
  NormArgs a{};
  int htype, stype, vec = 1;
  const at::Tensor& ref;

  Call(const at::Tensor& r, at::ScalarType h, at::ScalarType s, bool layer, double scale, double eps) : ref(r) {
    TORCH_CHECK(ref.dim() >= 1 && ref.numel() > 0, "block_norm: empty rows");
    a.width = (int)std::min<int64_t>(ref.size(-1), INT32_MAX);
    TORCH_CHECK(ref.size(-1) <= st::kNormMaxWidth, "block_norm: rows of at most ", st::kNormMaxWidth,
                " columns, got ", ref.size(-1));
    a.rows = ref.numel() / ref.size(-1);
    a.layer = layer ? 1 : 0;
    a.scale = (float)scale;
    a.eps = (float)eps;
    htype = h == at::kFloat ? st::kF32 : h == at::kBFloat16 ? st::kBF16 : st::kF16;
    stype = s == at::kFloat ? st::kF32 : s == at::kBFloat16 ? st::kBF16 : st::kF16;
    TORCH_CHECK(stype == htype || stype == st::kF32, "block_norm: the residual stream has h's type or fp32");
    if (a.width % 8) vec = 0;
  }
  void* row(const at::Tensor& t, const char* what, bool stream) {
    TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), "block_norm: ", what, " must be on ", ref.device());
    TORCH_CHECK(type_code(t) == (stream ? stype : htype), "block_norm: ", what, " has type ", t.scalar_type());
    TORCH_CHECK(t.is_contiguous() && t.sizes() == ref.sizes(), "block_norm: ", what, " must be contiguous of shape ",
                ref.sizes(), ", got ", t.sizes());
    if ((uintptr_t)t.data_ptr() % 16) vec = 0;
    return t.data_ptr();
  }
  const void* weight(const opt& t, const char* what, bool gate = false) {
    if (!has(t)) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == ref.device(), "block_norm: ", what, " must be on ", ref.device());
    TORCH_CHECK(t->is_contiguous() && (t->numel() == a.width || (gate && t->numel() == 1)), "block_norm: ", what,
                " must be contiguous with ", a.width, " elements", gate ? " or one" : "", ", got ", t->sizes());
    const int c = type_code(*t);
    TORCH_CHECK(c == htype || c == st::kF32, "block_norm: ", what, " must have h's type or be fp32");
    TORCH_CHECK(!weights || (c == st::kF32) == (a.w32 != 0), "block_norm: gate and weights must have one type");
    a.w32 = c == st::kF32;
    weights = true;
    if (t->numel() > 1 && (uintptr_t)t->data_ptr() % 16) vec = 0;
    return t->data_ptr();
  }
  void take_weights(const opt& gate, const opt& w1, const opt& b1, const opt& w2, const opt& b2) {
    a.gate = weight(gate, "gate", true);
    a.gate_n = has(gate) ? (int)gate->numel() : 0;
    a.w1 = weight(w1, "post_weight");
    a.b1 = weight(b1, "post_bias");
    a.w2 = weight(w2, "pre_weight");
    a.b2 = weight(b2, "pre_bias");
    TORCH_CHECK((a.w1 || !a.b1) && (a.w2 || !a.b2), "block_norm: a bias needs its weight");
  }
  bool weights = false;
};

// -> y (undefined without pre_weight), s (undefined unless write_s), stats (undefined unless keep)
std::vector<at::Tensor> block_norm_fwd(const at::Tensor& h, const opt& residual, const opt& gate, const opt& w1,
                                       const opt& b1, const opt& w2, const opt& b2, bool layer, double scale,
                                       double eps, bool write_s, bool keep) {
  type_code(h);
  Call c(h, h.scalar_type(), has(residual) ? residual->scalar_type() : h.scalar_type(), layer, scale, eps);
  c.take_weights(gate, w1, b1, w2, b2);
  c10::hip::HIPGuardMasqueradingAsCUDA g(h.device());
  at::Tensor y, s, stats;
  c.a.h = c.row(h, "h", false);
  if (has(residual)) c.a.res = c.row(*residual, "residual", true);
  if (has(w2)) {
    y = at::empty_like(h);
    c.a.y = c.row(y, "y", false);
  }
  if (write_s) {
    s = at::empty_like(has(residual) ? *residual : h);
    c.a.s = c.row(s, "s", true);
  }
  if (keep) {
    stats = at::empty({c.a.rows, 4}, h.options().dtype(at::kFloat));
    c.a.stats = stats.data_ptr<float>();
  }
  const int rc = st_block_norm_fwd(&c.a, c.htype, c.stype, c.vec, c10::hip::getCurrentHIPStream().stream());
  TORCH_CHECK(rc == 0, "st_amd::block_norm_fwd launch failed with code ", rc);
  return {y, s, stats};
}

// want: dh, dres, dgate, dw1, db1, dw2, db2; want_f32: the last five in fp32 and not their weight's type.
// With a norm after the block or a gate h (and the residual) are given, else s.
std::vector<at::Tensor> block_norm_bwd(const opt& dy, const opt& ds, const opt& h, const opt& residual, const opt& s,
                                       const at::Tensor& stats, const opt& gate, const opt& w1, const opt& b1,
                                       const opt& w2, const opt& b2, bool layer, double scale, double eps,
                                       at::ArrayRef<int64_t> want, at::ArrayRef<int64_t> want_f32, at::ScalarType htype) {
  TORCH_CHECK(want.size() == 7 && want_f32.size() == 7, "block_norm_bwd: seven gradients");
  const bool gen = has(w1) || has(gate);
  TORCH_CHECK(gen ? has(h) : has(s), "block_norm_bwd: ", gen ? "h" : "s", " is needed");
  const at::Tensor& ref = gen ? *h : *s;
  const at::ScalarType stype = has(residual) ? residual->scalar_type() : gen ? htype : s->scalar_type();
  Call c(ref, htype, stype, layer, scale, eps);
  c.take_weights(gate, w1, b1, w2, b2);
  TORCH_CHECK(has(dy) || has(ds), "block_norm_bwd: no gradient comes in");
  TORCH_CHECK(!has(dy) || has(w2), "block_norm_bwd: dy without pre_weight");
  c10::hip::HIPGuardMasqueradingAsCUDA g(ref.device());
  if (gen) {
    c.a.h = c.row(*h, "h", false);
    if (has(residual)) c.a.res = c.row(*residual, "residual", true);
  } else {
    c.a.s = c.row(*s, "s", true);
  }
  if (has(dy)) c.a.dy = c.row(*dy, "dy", false);
  if (has(ds)) c.a.ds = c.row(*ds, "ds", true);
  TORCH_CHECK(stats.is_cuda() && stats.device() == ref.device() && stats.scalar_type() == at::kFloat &&
                  stats.is_contiguous() && stats.numel() == 4 * c.a.rows,
              "block_norm_bwd: stats");
  c.a.stats = stats.data_ptr<float>();
  std::vector<at::Tensor> out(7);
  if (want[0]) {
    out[0] = at::empty_like(ref, ref.options().dtype(htype));
    c.a.dh = c.row(out[0], "dh", false);
  }
  if (want[1]) {
    out[1] = at::empty_like(ref, ref.options().dtype(stype));
    c.a.dres = c.row(out[1], "dres", true);
  }
  const opt* ws[5] = {&gate, &w1, &b1, &w2, &b2};
  void* outp[5];
  int out32[5];
  bool sums = false;
  for (int i = 0; i < 5; ++i) {
    outp[i] = nullptr;
    out32[i] = 0;
    if (!want[2 + i] || !has(*ws[i])) continue;
    const at::ScalarType t = want_f32[2 + i] ? at::kFloat : (*ws[i])->scalar_type();
    // without dy the norm before the next block passes nothing on
    out[2 + i] = i >= 3 && !has(dy) ? at::zeros((*ws[i])->sizes(), ref.options().dtype(t))
                                    : at::empty((*ws[i])->sizes(), ref.options().dtype(t));
    if (i >= 3 && !has(dy)) continue;
    outp[i] = out[2 + i].data_ptr();
    out32[i] = t == at::kFloat;
    sums = true;
  }
  const bool bias = has(b1) || has(b2);
  const int blocks = st_block_norm_bwd_blocks(c.a.rows, c.a.width);
  at::Tensor ws_t, gp;
  if (sums) {
    ws_t = at::empty({blocks, (gen ? 2 : 1) * (bias ? 2 : 1), c.a.width}, ref.options().dtype(at::kFloat));
    c.a.partial = ws_t.data_ptr<float>();
  }
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  int rc = st_block_norm_bwd(&c.a, gen, bias, blocks, c.htype, c.stype, c.vec, stream);
  TORCH_CHECK(rc == 0, "st_amd::block_norm_bwd launch failed with code ", rc);
  if (sums) {
    if (c.a.gate_n == 1 && outp[0]) gp = at::empty({(c.a.width + 31) / 32}, ws_t.options());
    rc = st_block_norm_finish(&c.a, gen, bias, blocks, outp, out32, gp.defined() ? gp.data_ptr<float>() : nullptr,
                              c.htype, stream);
    TORCH_CHECK(rc == 0, "st_amd::block_norm_bwd column sums failed with code ", rc);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st_amd, m) {
  m.def("block_norm_fwd(Tensor h, Tensor? residual, Tensor? gate, Tensor? post_weight, Tensor? post_bias, "
        "Tensor? pre_weight, Tensor? pre_bias, bool layer, float scale, float eps, bool write_s, bool keep) -> Tensor[]");
  m.def("block_norm_bwd(Tensor? dy, Tensor? ds, Tensor? h, Tensor? residual, Tensor? s, Tensor stats, Tensor? gate, "
        "Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, bool layer, float scale, "
        "float eps, int[] want, int[] want_f32, ScalarType htype) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(st_amd, CUDA, m) {
  m.impl("block_norm_fwd", &block_norm_fwd);
  m.impl("block_norm_bwd", &block_norm_bwd);
}
