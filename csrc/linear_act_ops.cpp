// torch.ops.st_amd.linear_act*: host side of the matrix products with an epilogue
// (csrc/linear_act_*.hip).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>

#include "capture_check.h"
#include "forward_grad_check.h"
#include "linear_act_args.h"

using st::LinearArgs;

extern "C" {
int64_t st_linear_tile_ws(int M, int N, int K, int vec, int acol, int bcol);
int st_linear_tile(LinearArgs* p, int acol, int bcol, hipStream_t st);
double st_linear_tile_us(int M, int N, int K, int vec, int acol, int bcol);
int st_linear_rows(const LinearArgs* p, hipStream_t st);
int64_t st_linear_wide_ws(const LinearArgs* p);
double st_linear_wide_us(const LinearArgs* p, int acol, int bcol);
int st_linear_wide(const LinearArgs* p, int acol, int bcol, hipStream_t st);
int st_linear_dz_runs(int64_t rows, int width);
int st_linear_dz(const void* dy, int dy_f32, const void* z, void* dz, void* db, int db_f32, float* partial,
                 int64_t rows, int width, int act, int f16, int vec, hipStream_t st);
}

namespace {

typedef c10::optional<at::Tensor> opt;

bool has(const opt& t) { return t.has_value() && t->defined(); }
hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
bool aligned(const at::Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0; }

// Rows of the last dimension with one stride between them, or a copy that has them.
at::Tensor rows_of(const at::Tensor& t) {
  auto m = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return m.stride(1) == 1 && (m.size(0) <= 1 || m.stride(0) >= m.size(1)) ? m : m.contiguous();
}
int64_t ld_of(const at::Tensor& m) { return m.size(0) <= 1 ? m.size(1) : m.stride(0); }

void check_dims(int64_t m, int64_t n, int64_t k) {
  const int64_t most = INT32_MAX - 511;  // rounding up to tiles stays in 32 bits
  TORCH_CHECK_VALUE(m <= most && n <= most && k <= most, "linear_act: dimensions of at most ", most);
}

// C [M, N] = A B^T with the epilogue e (its out set); A, B 2-D, acol / bcol: stored [k, rows].
void product(const at::Tensor& A, bool acol, const at::Tensor& B, bool bcol, st::LinearEpi e, int64_t M, int64_t N,
             int64_t K, bool vec) {
  check_dims(M, N, K);
  LinearArgs p{};
  p.lda = ld_of(A);
  p.ldb = ld_of(B);
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  e.ldo = N;
  e.f16 = A.scalar_type() == at::kHalf;
  p.epi = e;
  p.splits = 1;
  const int64_t ca = acol ? M : K, cb = bcol ? N : K;  // the contiguous dimension of each operand
  // an operand of fewer than 8 elements is read from a copy with room behind it
  auto roomy = [](const at::Tensor& t, int64_t ld) {
    if ((t.size(0) - 1) * ld + t.size(1) >= 8) return t;
    auto b = at::zeros({16}, t.options());
    b.as_strided(t.sizes(), {ld, 1}).copy_(t);
    return b;
  };
  const at::Tensor ka = roomy(A, p.lda), kb = roomy(B, p.ldb);
  p.a = ka.data_ptr();
  p.b = kb.data_ptr();
  const int64_t most = (int64_t)1 << 31;  // bytes that a descriptor of 128 rows spans
  p.vec = vec && (p.lda * 128 + K) * 2 < most && (p.ldb * 128 + K) * 2 < most && ca % 8 == 0 && cb % 8 == 0 &&
          N % 4 == 0 && p.lda % 8 == 0 && p.ldb % 8 == 0 && aligned(A) && aligned(B);
  int rc = -2;
  // Few rows stream the weight.  Measured, us, streamed / tiles: 4096 -> 14336 4 rows 27 / 25 (from memory 27 / 31),
  // 8 rows 28 / 21; 14336 -> 4096 8 rows 29 / 25; but 4096 -> 4096 8 rows 10 / 12, 16 rows 11 / 12; 1280 -> 5120 8 / 10.
  // Else whichever tiling is expected to be faster: smaller tiles / 256 x 256: y with GELU 8192 x 1024 x 1024 41 / 47,
  // 8192 x 1280 x 1280 57 / 52, 4096 x 1024 x 4096 67 / 52; dx 4096 x 4096 x 1024 50 / 66, 24576 x 1280 x 1280 107 / 98;
  // dW 4096 x 4096 x 1024 51 / 68, 1280 x 24576 x 1280 137 / 99.
  if (!acol && !bcol && (M <= 4 || (M <= 16 && N * K <= 1 << 24))) rc = st_linear_rows(&p, stream());
  if (rc == -2) {
    const double wide = st_linear_wide_us(&p, acol, bcol);
    const bool use_wide = wide >= 0.0 && wide < st_linear_tile_us(p.M, p.N, p.K, p.vec, acol, bcol);
    at::Tensor ws;
    if (const int64_t n = use_wide ? st_linear_wide_ws(&p) : st_linear_tile_ws(p.M, p.N, p.K, p.vec, acol, bcol)) {
      ws = at::empty({n}, A.options().dtype(at::kFloat));
      p.ws = ws.data_ptr<float>();
    }
    rc = use_wide ? st_linear_wide(&p, acol, bcol, stream()) : st_linear_tile(&p, acol, bcol, stream());
  }
  TORCH_CHECK(rc == 0, "st_amd::linear_act launch failed with code ", rc);
}

// x [..., K], weight [N, K] -> (y [..., N], z [rows, N] or undefined)
std::tuple<at::Tensor, at::Tensor> linear_act_fwd(const at::Tensor& x, const at::Tensor& w, const opt& bias,
                                                  const opt& residual, int64_t act, bool keep_z) {
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                   "linear_act: x must be bf16 or fp16 on the GPU, got ", x.scalar_type());
  TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type() && (!has(bias) || bias->scalar_type() == x.scalar_type()),
                   "linear_act: x, weight and bias must have one type, got ", x.scalar_type(), ", ", w.scalar_type(),
                   has(bias) ? ", " : "", has(bias) ? c10::toString(bias->scalar_type()) : "");
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1), "linear_act: weight ", w.sizes(),
                    " does not take x ", x.sizes());
  TORCH_CHECK_VALUE(act >= 0 && act <= st::kSilu, "linear_act: unknown activation");
  const int64_t N = w.size(0), K = w.size(1), M = K ? x.numel() / K : 0;
  TORCH_CHECK_VALUE(N > 0 && K > 0 && M > 0, "linear_act: empty product of x ", x.sizes(), " and weight ", w.sizes());
  auto oshape = x.sizes().vec();
  oshape.back() = N;
  TORCH_CHECK_VALUE(w.device() == x.device() && (!has(bias) || bias->device() == x.device()) &&
                        (!has(residual) || residual->device() == x.device()),
                    "linear_act: tensors on different devices");
  TORCH_CHECK_VALUE(!has(bias) || (bias->dim() == 1 && bias->size(0) == N), "linear_act: bias must have shape [", N, "]");
  c10::hip::HIPGuardMasqueradingAsCUDA g(x.device());
  at::Tensor xm = rows_of(x), wm = rows_of(w), bm, rm;
  st::LinearEpi e{};
  e.act = (int)act;
  bool vec = true;
  if (has(bias)) {
    bm = bias->contiguous();
    e.bias = bm.data_ptr();
    vec = vec && aligned(bm);
  }
  auto otype = x.scalar_type();
  if (has(residual)) {
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(oshape), "linear_act: the residual must have y's shape ",
                      at::IntArrayRef(oshape), ", got ", residual->sizes());
    otype = residual->scalar_type();
    TORCH_CHECK_TYPE(otype == x.scalar_type() || otype == at::kFloat, "linear_act: the residual has x's type or fp32, got ",
                     otype);
    rm = residual->contiguous();
    e.res = rm.data_ptr();
    vec = vec && aligned(rm);
  }
  e.out_f32 = otype == at::kFloat;
  auto y = at::empty(oshape, x.options().dtype(otype));
  e.out = y.data_ptr();
  at::Tensor z;
  if (keep_z) {
    z = at::empty({M, N}, x.options());
    e.z = z.data_ptr();
  }
  product(xm, false, wm, false, e, M, N, K, vec);
  return {y, z};
}

// dz [rows, N] (dy itself where z is not given and dy has its type) and db (undefined unless want_db)
std::tuple<at::Tensor, at::Tensor> linear_act_dz(const at::Tensor& dy, const opt& z, at::ScalarType type, int64_t act,
                                                 bool want_db, bool db_f32) {
  TORCH_CHECK(dy.is_cuda() && dy.dim() >= 1 && (type == at::kBFloat16 || type == at::kHalf) &&
                  (dy.scalar_type() == type || dy.scalar_type() == at::kFloat),
              "linear_act_dz: dy");
  c10::hip::HIPGuardMasqueradingAsCUDA g(dy.device());
  auto d = dy.reshape({-1, dy.size(-1)}).contiguous();
  const int64_t M = d.size(0), N = d.size(1);
  check_dims(M, N, 1);
  if (has(z))
    TORCH_CHECK(z->device() == dy.device() && z->scalar_type() == type && z->is_contiguous() && z->sizes() == d.sizes(),
                "linear_act_dz: z must be contiguous ", type, " of shape ", d.sizes());
  const bool same = !has(z) && d.scalar_type() == type;
  if (same && !want_db) return {d, at::Tensor()};
  at::Tensor dz = same ? d : at::empty({M, N}, d.options().dtype(type)), db, part;
  if (want_db) {
    db = at::empty({N}, d.options().dtype(db_f32 ? at::kFloat : type));
    part = at::empty({st_linear_dz_runs(M, (int)N), N}, d.options().dtype(at::kFloat));
  }
  const bool vec = N % 8 == 0 && aligned(d) && (!has(z) || aligned(*z));
  const int rc = st_linear_dz(d.data_ptr(), d.scalar_type() == at::kFloat, has(z) ? z->data_ptr() : nullptr,
                              same ? nullptr : dz.data_ptr(), want_db ? db.data_ptr() : nullptr, db_f32,
                              want_db ? part.data_ptr<float>() : nullptr, M, (int)N, (int)act, type == at::kHalf, vec,
                              stream());
  TORCH_CHECK(rc == 0, "st_amd::linear_act_dz launch failed with code ", rc);
  return {dz, db};
}

// dx [rows, K] = dz W
at::Tensor linear_act_dx(const at::Tensor& dz, const at::Tensor& w) {
  TORCH_CHECK(dz.is_cuda() && dz.dim() == 2 && w.dim() == 2 && dz.size(1) == w.size(0) && dz.device() == w.device() &&
                  dz.scalar_type() == w.scalar_type(),
              "linear_act_dx: dz ", dz.sizes(), ", weight ", w.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA g(dz.device());
  auto zm = rows_of(dz), wm = rows_of(w);
  auto dx = at::empty({dz.size(0), w.size(1)}, dz.options());
  st::LinearEpi e{};
  e.out = dx.data_ptr();
  product(zm, false, wm, true, e, dz.size(0), w.size(1), w.size(0), true);
  return dx;
}

// dW [N, K] = dz^T x, in dz's type
at::Tensor linear_act_dw(const at::Tensor& dz, const at::Tensor& x) {
  TORCH_CHECK(dz.is_cuda() && dz.dim() == 2 && x.dim() == 2 && dz.size(0) == x.size(0) && dz.device() == x.device() &&
                  dz.scalar_type() == x.scalar_type(),
              "linear_act_dw: dz ", dz.sizes(), ", x ", x.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA g(dz.device());
  auto zm = rows_of(dz), xm = rows_of(x);
  auto dw = at::empty({dz.size(1), x.size(1)}, dz.options());
  st::LinearEpi e{};
  e.out = dw.data_ptr();
  product(zm, true, xm, true, e, dz.size(1), x.size(1), dz.size(0), true);
  return dw;
}

// out [N, K] = dz^T x, or out + dz^T x: fp32, or dz's type.  Each element is read and written by one lane.
void linear_act_dw_(const at::Tensor& out, const at::Tensor& dz, const at::Tensor& x, bool accumulate) {
  TORCH_CHECK(dz.is_cuda() && dz.dim() == 2 && x.dim() == 2 && dz.size(0) == x.size(0) && dz.device() == x.device() &&
                  dz.scalar_type() == x.scalar_type(),
              "linear_act_dw_: dz ", dz.sizes(), ", x ", x.sizes());
  TORCH_CHECK(out.device() == dz.device() && out.is_contiguous() && out.dim() == 2 && out.size(0) == dz.size(1) &&
                  out.size(1) == x.size(1) && (out.scalar_type() == at::kFloat || out.scalar_type() == dz.scalar_type()),
              "linear_act_dw_: out must be contiguous [", dz.size(1), ", ", x.size(1), "], fp32 or ", dz.scalar_type(),
              ", got ", out.scalar_type(), " ", out.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA g(dz.device());
  auto zm = rows_of(dz), xm = rows_of(x);
  st::LinearEpi e{};
  e.out = out.data_ptr();
  e.out_f32 = out.scalar_type() == at::kFloat;
  if (accumulate) e.res = e.out;
  product(zm, true, xm, true, e, dz.size(1), x.size(1), dz.size(0), aligned(out));
}

class LinearAct : public torch::autograd::Function<LinearAct> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const opt& bias, const opt& residual, int64_t act) {
    int64_t need = (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0);
    if (has(bias) && bias->requires_grad()) need |= 4;
    if (has(residual) && residual->requires_grad()) need |= 8;
    auto [y, z] = linear_act_fwd(x, w, bias, residual, act, act != st::kNoAct && (need & 7) != 0);
    ctx->save_for_backward({(need & 2) ? x : at::Tensor(), (need & 1) ? w : at::Tensor(), z});
    ctx->saved_data["need"] = need;
    ctx->saved_data["act"] = act;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["xshape"] = x.sizes();
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_act: its gradient can't be differentiated again");
    torch::autograd::variable_list r(5);
    const auto& dy = grads[0];
    const int64_t need = ctx->saved_data["need"].toInt();
    auto saved = ctx->get_saved_variables();
    if (need & 8) r[3] = dy;
    if (need & 7) {
      auto [dz, db] = linear_act_dz(dy, saved[2].defined() ? opt(saved[2]) : opt(),
                                    (at::ScalarType)ctx->saved_data["type"].toInt(), ctx->saved_data["act"].toInt(),
                                    (need & 4) != 0, false);
      if (need & 1) r[0] = linear_act_dx(dz, saved[1]).view(ctx->saved_data["xshape"].toIntVector());
      if (need & 2) r[1] = linear_act_dw(dz, rows_of(saved[0]));
      if (need & 4) r[2] = db;
    }
    return r;
  }
};

at::Tensor linear_act(const at::Tensor& x, const at::Tensor& w, const opt& bias, const opt& residual, int64_t act) {
  return std::get<0>(linear_act_fwd(x, w, bias, residual, act, false));
}

void check_capture(at::TensorList inputs) {
  for (const auto& t : inputs) st::check_capture({&t}, "training call");
}

at::Tensor linear_act_autograd(const at::Tensor& x, const at::Tensor& w, const opt& bias, const opt& residual,
                               int64_t act) {
  auto ptr = [](const opt& t) { return has(t) ? &*t : nullptr; };
  st::refuse_forward_grad({&x, &w, ptr(bias), ptr(residual)}, "linear_act");
  const bool grad = x.requires_grad() || w.requires_grad() || (has(bias) && bias->requires_grad()) ||
                    (has(residual) && residual->requires_grad());
  if (!grad || !at::GradMode::is_enabled()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_act(x, w, bias, residual, act);
  }
  st::check_capture({&x, &w, ptr(bias), ptr(residual)}, "linear_act");
  return LinearAct::apply(x, w, bias, residual, act);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st_amd, m) {
  m.def("linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> Tensor");
  m.def("linear_act_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act, bool keep_z) -> (Tensor, Tensor)");
  m.def("linear_act_dz(Tensor dy, Tensor? z, ScalarType type, int act, bool want_db, bool db_f32) -> (Tensor, Tensor)");
  m.def("linear_act_dx(Tensor dz, Tensor weight) -> Tensor");
  m.def("linear_act_dw(Tensor dz, Tensor x) -> Tensor");
  m.def("linear_act_dw_(Tensor(a!) out, Tensor dz, Tensor x, bool accumulate) -> ()");
  m.def("check_capture(Tensor[] inputs) -> ()");
}

TORCH_LIBRARY_IMPL(st_amd, CUDA, m) {
  m.impl("linear_act", &linear_act);
  m.impl("linear_act_fwd", &linear_act_fwd);
  m.impl("linear_act_dz", &linear_act_dz);
  m.impl("linear_act_dx", &linear_act_dx);
  m.impl("linear_act_dw", &linear_act_dw);
  m.impl("linear_act_dw_", &linear_act_dw_);
  m.impl("check_capture", &check_capture);
}

TORCH_LIBRARY_IMPL(st_amd, AutogradCUDA, m) { m.impl("linear_act", &linear_act_autograd); }
