// torch.ops.st_amd.block_norm_*: host side of the norms around a block's gated residual
// (csrc/block_norm_fwd.hip, csrc/block_norm_bwd.hip).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_norm_args.h"
#include "capture_check.h"
#include "forward_grad_check.h"

using st::NormArgs;

extern "C" {
int st_block_norm_fwd(const NormArgs* a, int htype, int stype, int vec, hipStream_t st);
int st_block_norm_bwd_blocks(int64_t rows, int width);
int st_block_norm_bwd(const NormArgs* a, int gen, int bias, int blocks, int htype, int stype, int vec, hipStream_t st);
int st_block_norm_finish(const NormArgs* a, int gen, int bias, int blocks, void* const* out, const int* out_f32,
                         int htype, hipStream_t st);
int64_t st_block_norm_bwd_floats(int64_t rows, int width, int arrays);
}

namespace {

typedef c10::optional<at::Tensor> opt;

int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return st::kF32;
    case at::kBFloat16: return st::kBF16;
    case at::kHalf: return st::kF16;
    default: TORCH_CHECK_TYPE(false, "block_norm: fp32, bf16 or fp16 tensors, got ", t.scalar_type());
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
    TORCH_CHECK_VALUE(ref.size(-1) <= st::kNormMaxWidth, "block_norm: rows of at most ", st::kNormMaxWidth,
                " columns, got ", ref.size(-1));
    a.rows = ref.numel() / ref.size(-1);
    a.layer = layer ? 1 : 0;
    a.scale = (float)scale;
    a.eps = (float)eps;
    htype = h == at::kFloat ? st::kF32 : h == at::kBFloat16 ? st::kBF16 : st::kF16;
    stype = s == at::kFloat ? st::kF32 : s == at::kBFloat16 ? st::kBF16 : st::kF16;
    TORCH_CHECK_TYPE(stype == htype || stype == st::kF32, "block_norm: the residual has h's type (", h, ") or fp32, got ",
                     s);
    if (a.width % 8) vec = 0;
  }
  void* row(const at::Tensor& t, const char* what, bool stream) {
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == ref.device(), "block_norm: ", what, " must be on ", ref.device());
    TORCH_CHECK_TYPE(type_code(t) == (stream ? stype : htype), "block_norm: ", what, " has type ", t.scalar_type());
    TORCH_CHECK_VALUE(t.is_contiguous() && t.sizes() == ref.sizes(), "block_norm: ", what, " must be contiguous of shape ",
                ref.sizes(), ", got ", t.sizes());
    if ((uintptr_t)t.data_ptr() % 16) vec = 0;
    return t.data_ptr();
  }
  const void* weight(const opt& t, const char* what, bool gate = false) {
    if (!has(t)) return nullptr;
    TORCH_CHECK_VALUE(t->is_cuda() && t->device() == ref.device(), "block_norm: ", what, " must be on ", ref.device());
    TORCH_CHECK_VALUE(t->is_contiguous() && ((t->dim() == 1 && t->numel() == a.width) ||
                                             (gate && t->dim() <= 1 && t->numel() == 1)), "block_norm: ", what,
                " must be contiguous with ", a.width, " elements", gate ? " or one" : "", ", got ", t->sizes());
    const int c = type_code(*t);
    TORCH_CHECK_TYPE(c == htype || c == st::kF32, "block_norm: ", what, " must have h's type or be fp32");
    TORCH_CHECK_TYPE(!weights || (c == st::kF32) == (a.w32 != 0), "block_norm: gate and weights must have one type");
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
// h (and the residual) are given, or s where that is enough (keep_stream).
std::vector<at::Tensor> block_norm_bwd(const opt& dy, const opt& ds, const opt& h, const opt& residual, const opt& s,
                                       const at::Tensor& stats, const opt& gate, const opt& w1, const opt& b1,
                                       const opt& w2, const opt& b2, bool layer, double scale, double eps,
                                       at::ArrayRef<int64_t> want, at::ArrayRef<int64_t> want_f32, at::ScalarType htype) {
  TORCH_CHECK(want.size() == 7 && want_f32.size() == 7, "block_norm_bwd: seven gradients");
  const bool gen = has(w1) || has(gate);
  TORCH_CHECK(has(h) || (has(s) && !gen), "block_norm_bwd: h is needed");
  const at::Tensor& ref = has(h) ? *h : *s;
  const at::ScalarType stype = has(residual) ? residual->scalar_type() : has(h) ? htype : s->scalar_type();
  Call c(ref, htype, stype, layer, scale, eps);
  c.take_weights(gate, w1, b1, w2, b2);
  TORCH_CHECK(has(dy) || has(ds), "block_norm_bwd: no gradient comes in");
  TORCH_CHECK(!has(dy) || has(w2), "block_norm_bwd: dy without pre_weight");
  c10::hip::HIPGuardMasqueradingAsCUDA g(ref.device());
  if (has(h)) {
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
  at::Tensor ws_t;
  if (sums) {
    ws_t = at::empty({st_block_norm_bwd_floats(c.a.rows, c.a.width, (gen ? 2 : 1) * (bias ? 2 : 1))},
                     ref.options().dtype(at::kFloat));
    c.a.partial = ws_t.data_ptr<float>();
  }
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  int rc = st_block_norm_bwd(&c.a, gen, bias, blocks, c.htype, c.stype, c.vec, stream);
  TORCH_CHECK(rc == 0, "st_amd::block_norm_bwd launch failed with code ", rc);
  if (sums) {
    rc = st_block_norm_finish(&c.a, gen, bias, blocks, outp, out32, c.htype, stream);
    TORCH_CHECK(rc == 0, "st_amd::block_norm_bwd column sums failed with code ", rc);
  }
  return out;
}

void check_call(const at::Tensor& h, const opt& residual, const opt& w1, const opt& b1, const opt& w2, const opt& b2) {
  TORCH_CHECK_VALUE(h.dim() >= 1 && h.size(-1) >= 1, "block_norm: h needs rows of at least one column");
  TORCH_CHECK_VALUE(!has(residual) || residual->sizes() == h.sizes(), "block_norm: the residual must be h's ",
                    h.sizes(), ", got ", has(residual) ? residual->sizes() : h.sizes());
  TORCH_CHECK_VALUE((has(w1) || !has(b1)) && (has(w2) || !has(b2)), "block_norm: a bias needs its weight");
  type_code(h);
}

// Whether the backward reads s alone: no norm after the block, no gate, and s not rounded to 16 bits.
bool keep_stream(const at::Tensor& h, const opt& residual, const opt& gate, const opt& w1, bool write_s) {
  const auto type = has(residual) ? residual->scalar_type() : h.scalar_type();
  return !has(gate) && !has(w1) && (!write_s || type == at::kFloat);
}

// Whether the stream is h itself: nothing comes between the block and the next norm.
bool stream_is_h(const opt& residual, const opt& gate, const opt& w1, double scale) {
  return !has(residual) && !has(gate) && !has(w1) && scale == 1.0;
}

opt rows_of(const opt& t) { return has(t) ? opt(t->contiguous()) : opt(); }

// The operator and its gradient without a way through Python (a training pass of both spends some 10
// us here and several times that in a Python autograd function).
class BlockNorm : public torch::autograd::Function<BlockNorm> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& h,
                                                const opt& residual, const opt& gate, const opt& w1, const opt& b1,
                                                const opt& w2, const opt& b2, bool layer, double scale, double eps,
                                                bool write_s) {
    auto out = block_norm_fwd(h, residual, gate, w1, b1, w2, b2, layer, scale, eps, write_s, true);
    const bool alone = keep_stream(h, residual, gate, w1, write_s);
    auto get = [](const opt& t) { return has(t) ? *t : at::Tensor(); };
    // what the backward recomputes from (block_norm_bwd.hip): h and the residual, or s alone
    ctx->save_for_backward({alone ? at::Tensor() : h, alone ? at::Tensor() : get(residual),
                            !alone ? at::Tensor() : write_s ? out[1] : h, out[2], get(gate), get(w1), get(b1), get(w2),
                            get(b2)});
    const opt* in[6] = {&residual, &gate, &w1, &b1, &w2, &b2};
    int64_t need = h.requires_grad() ? 1 : 0;
    for (int i = 0; i < 6; ++i)
      if (has(*in[i]) && (*in[i])->requires_grad()) need |= int64_t(2) << i;
    ctx->saved_data["need"] = need;
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["htype"] = (int64_t)h.scalar_type();
    ctx->saved_data["rtype"] = has(residual) ? (int64_t)residual->scalar_type() : (int64_t)-1;
    ctx->saved_data["has_y"] = has(w2);
    ctx->set_materialize_grads(false);
    if (write_s && !(need & 31)) ctx->mark_non_differentiable({out[1]});  // nothing that s depends on wants a gradient
    torch::autograd::variable_list r;
    if (has(w2)) r.push_back(out[0]);
    if (write_s) r.push_back(out[1]);
    return r;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "block_norm: its gradient can't be differentiated again");
    torch::autograd::variable_list r(11);
    const bool has_y = ctx->saved_data["has_y"].toBool();
    opt dy, ds;
    if (has_y && grads[0].defined()) dy = grads[0].contiguous();
    const size_t at_s = has_y ? 1 : 0;
    if (grads.size() > at_s && grads[at_s].defined()) ds = grads[at_s].contiguous();
    if (!has(dy) && !has(ds)) return r;
    auto saved = ctx->get_saved_variables();
    auto o = [&](int i) { return saved[i].defined() ? opt(saved[i]) : opt(); };
    const int64_t need = ctx->saved_data["need"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t htype = ctx->saved_data["htype"].toInt(), rtype = ctx->saved_data["rtype"].toInt();
    const bool gen = saved[4].defined() || saved[5].defined();
    // without a norm after the block, gate or scale dh IS the residual's gradient
    const bool one = !gen && rtype == htype && scale == 1.0;
    int64_t want[7], f32[7] = {0, 0, 0, 0, 0, 0, 0};
    for (int i = 0; i < 7; ++i) want[i] = (need >> i) & 1;
    if (one) {
      want[1] |= want[0];
      want[0] = 0;
    }
    auto got = block_norm_bwd(dy, ds, o(0), o(1), o(2), saved[3], o(4), o(5), o(6), o(7), o(8),
                              ctx->saved_data["layer"].toBool(), scale, ctx->saved_data["eps"].toDouble(), want, f32,
                              (at::ScalarType)htype);
    if (one) got[0] = got[1];
    for (int i = 0; i < 7; ++i)
      if ((need >> i) & 1) r[i] = got[i];
    return r;
  }
};

// (y, s): y undefined without pre_weight; s is h itself where nothing comes between.
std::tuple<at::Tensor, at::Tensor> block_norm(const at::Tensor& h, const opt& residual, const opt& gate, const opt& w1,
                                              const opt& b1, const opt& w2, const opt& b2, bool layer, double scale,
                                              double eps) {
  check_call(h, residual, w1, b1, w2, b2);
  const bool same = stream_is_h(residual, gate, w1, scale);
  if (same && !has(w2)) return {at::Tensor(), h};
  auto hc = h.contiguous();
  auto out = block_norm_fwd(hc, rows_of(residual), rows_of(gate), rows_of(w1), rows_of(b1), rows_of(w2), rows_of(b2),
                            layer, scale, eps, !same, false);
  return {out[0], same ? h : out[1]};
}

std::tuple<at::Tensor, at::Tensor> block_norm_autograd(const at::Tensor& h, const opt& residual, const opt& gate,
                                                       const opt& w1, const opt& b1, const opt& w2, const opt& b2,
                                                       bool layer, double scale, double eps) {
  auto ptr = [](const opt& t) { return has(t) ? &*t : nullptr; };
  st::refuse_forward_grad({&h, ptr(residual), ptr(gate), ptr(w1), ptr(b1), ptr(w2), ptr(b2)}, "block_norm");
  bool grad = h.requires_grad();
  for (const opt* t : {&residual, &gate, &w1, &b1, &w2, &b2}) grad |= has(*t) && (*t)->requires_grad();
  if (!grad || !at::GradMode::is_enabled()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return block_norm(h, residual, gate, w1, b1, w2, b2, layer, scale, eps);
  }
  check_call(h, residual, w1, b1, w2, b2);
  const bool same = stream_is_h(residual, gate, w1, scale);
  if (same && !has(w2)) return {at::Tensor(), h};
  st::check_capture({&h, ptr(residual), ptr(gate), ptr(w1), ptr(b1), ptr(w2), ptr(b2)}, "block_norm");
  auto r = BlockNorm::apply(h.contiguous(), rows_of(residual), rows_of(gate), rows_of(w1), rows_of(b1), rows_of(w2),
                            rows_of(b2), layer, scale, eps, !same);
  at::Tensor y = has(w2) ? r[0] : at::Tensor();
  return {y, same ? h : r.back()};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st_amd, m) {
  m.def("block_norm(Tensor h, Tensor? residual, Tensor? gate, Tensor? post_weight, Tensor? post_bias, "
        "Tensor? pre_weight, Tensor? pre_bias, bool layer, float scale, float eps) -> (Tensor, Tensor)");
  m.def("block_norm_fwd(Tensor h, Tensor? residual, Tensor? gate, Tensor? post_weight, Tensor? post_bias, "
        "Tensor? pre_weight, Tensor? pre_bias, bool layer, float scale, float eps, bool write_s, bool keep) -> Tensor[]");
  m.def("block_norm_bwd(Tensor? dy, Tensor? ds, Tensor? h, Tensor? residual, Tensor? s, Tensor stats, Tensor? gate, "
        "Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, bool layer, float scale, "
        "float eps, int[] want, int[] want_f32, ScalarType htype) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(st_amd, CUDA, m) {
  m.impl("block_norm", &block_norm);
  m.impl("block_norm_fwd", &block_norm_fwd);
  m.impl("block_norm_bwd", &block_norm_bwd);
}

TORCH_LIBRARY_IMPL(st_amd, AutogradCUDA, m) { m.impl("block_norm", &block_norm_autograd); }
