// torch.ops.st_amd.adamw_multi_: host side of the many-tensor AdamW step (csrc/adamw_multi.hip).
#include <torch/library.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "adamw_multi.h"
#include "capture_check.h"
#include "forward_grad_check.h"

extern "C" int st_adamw_multi(const AdamTable* tab, int count, const AdamScalars* h, int gtype, int ptype, int eight,
                              hipStream_t st);

namespace {

int type_code(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK(false, "adamw_multi: ", what, " must be fp32, bf16 or fp16, got ", t.scalar_type());
  }
  return -1;
}

struct Span {
  uintptr_t lo, hi;
  bool written;
};

uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

void adamw_multi_(at::TensorList params, at::TensorList grads, at::TensorList exp_avg, at::TensorList exp_avg_sq,
                  at::TensorList masters, at::TensorList scales, const c10::optional<at::Tensor>& clip_coef,
                  at::ArrayRef<double> weight_decay, double lr, double beta1, double beta2, double eps, int64_t step,
                  bool scale_grads) {
  const size_t N = params.size();
  TORCH_CHECK(grads.size() == N && exp_avg.size() == N && exp_avg_sq.size() == N && weight_decay.size() == N &&
                  (masters.empty() || masters.size() == N) && (scales.empty() || scales.size() == N),
              "adamw_multi: lists of different lengths");
  if (N == 0) return;
  TORCH_CHECK(step >= 1 && step <= UINT32_MAX, "adamw_multi: step counts from 1, got ", step);
  st::refuse_forward_grad({params, grads, exp_avg, exp_avg_sq, masters, scales}, "adamw_multi");
  const auto dev = params[0].device();
  TORCH_CHECK(dev.is_cuda(), "adamw_multi: param 0 must be on a GPU, got ", dev);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const auto current = c10::hip::getCurrentHIPStream();
  TORCH_CHECK(!st::is_capturing(current), "adamw_multi: the step number is the host's, so a captured step would repeat "
              "it; run the step outside the graph");
  auto check = [&](const at::Tensor& t, int64_t n, const char* what, size_t i) {
    TORCH_CHECK(t.is_cuda() && t.device() == dev, "adamw_multi: ", what, " ", i, " must be on ", dev, ", got ",
                t.device());
    TORCH_CHECK(t.is_contiguous(), "adamw_multi: ", what, " ", i, " must be contiguous");
    TORCH_CHECK(t.numel() == n, "adamw_multi: ", what, " ", i, " has ", t.numel(), " elements, not ", n);
  };
  AdamScalars h{};
  if (clip_coef.has_value() && clip_coef->defined()) {
    st::refuse_forward_grad({&*clip_coef}, "adamw_multi");
    check(*clip_coef, 1, "clip_coef", 0);
    TORCH_CHECK(clip_coef->scalar_type() == at::kFloat, "adamw_multi: clip_coef must be fp32");
    h.clip = clip_coef->data_ptr<float>();
  }
  h.write_grads = scale_grads && h.clip ? 1 : 0;
  h.lr = (float)lr;
  h.b1 = (float)beta1;
  h.c1 = (float)(1.0 - beta1);
  h.b2 = (float)beta2;
  h.c2 = (float)(1.0 - beta2);
  h.eps = (float)eps;
  h.inv_bc1 = (float)(1.0 / (1.0 - std::pow(beta1, (double)step)));
  h.inv_sbc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  h.key = mix32((uint32_t)step * 0x9e3779b9u);

  std::vector<Span> spans;
  spans.reserve(6 * N + 1);
  if (h.clip) spans.push_back({(uintptr_t)h.clip, (uintptr_t)h.clip + 4, false});
  std::vector<AdamTensor> all(N);
  std::vector<int> kind(N);  // (gradient type, parameter type, 8 bits); -1: empty
  int64_t blocks = 0;
  for (size_t i = 0; i < N; ++i) {
    const int64_t n = params[i].numel();
    AdamTensor& a = all[i];
    uintptr_t bits = 0;
    int at = 16;  // bytes that an access of four elements has to be aligned to, of the narrowest type at hand
    auto take = [&](const at::Tensor& t, const char* what, bool written, int64_t want) {
      check(t, want, what, i);
      const uintptr_t p = (uintptr_t)t.data_ptr();
      if (n) spans.push_back({p, p + (uintptr_t)t.nbytes(), written});
      return (void*)p;
    };
    auto align = [&](const void* p, int64_t bytes) { bits |= ((uintptr_t)p % bytes) ? 1 : 0; };
    a.param = take(params[i], "param", true, n);
    a.grad = take(grads[i], "grad", h.write_grads != 0, n);
    const int pt = type_code(params[i], "param"), gt = type_code(grads[i], "grad");
    TORCH_CHECK(grads[i].sizes() == params[i].sizes(), "adamw_multi: grad ", i, " has shape ", grads[i].sizes(),
                ", its param ", params[i].sizes());
    const bool has_master = !masters.empty() && masters[i].defined() && !(pt == 0 && masters[i].numel() == 0);
    TORCH_CHECK(has_master == (pt != 0), "adamw_multi: param ", i,
                pt ? " is 16 bits wide and needs an fp32 master" : " is fp32 and takes no master");
    a.master = nullptr;
    if (has_master) {
      TORCH_CHECK(masters[i].scalar_type() == at::kFloat, "adamw_multi: master ", i, " must be fp32");
      a.master = (float*)take(masters[i], "master", true, n);
      align(a.master, at);
    }
    a.m = take(exp_avg[i], "exp_avg", true, n);
    a.v = take(exp_avg_sq[i], "exp_avg_sq", true, n);
    const auto sd = exp_avg[i].scalar_type();
    TORCH_CHECK((sd == at::kFloat || sd == at::kFloat8_e4m3fn) && exp_avg_sq[i].scalar_type() == sd,
                "adamw_multi: exp_avg and exp_avg_sq ", i, " must both be fp32 or both float8_e4m3fn, got ", sd,
                " and ", exp_avg_sq[i].scalar_type());
    const bool eight = sd == at::kFloat8_e4m3fn;
    const int64_t nb = (n + kAdamBlock - 1) / kAdamBlock;
    a.scales = nullptr;
    if (eight) {
      TORCH_CHECK(!scales.empty() && scales[i].scalar_type() == at::kFloat,
                  "adamw_multi: 8-bit moments need fp32 scales [blocks, 2]");
      a.scales = (float*)take(scales[i], "scales", true, 2 * nb);
      TORCH_CHECK((uintptr_t)a.scales % 8 == 0, "adamw_multi: scales ", i, " must be 8-byte aligned");
    }
    align(a.param, pt ? 8 : 16);
    align(a.grad, gt ? 8 : 16);
    align(a.m, eight ? 4 : 16);
    align(a.v, eight ? 4 : 16);
    a.n = n;
    a.blk_base = blocks;
    a.keep = (float)(1.0 - lr * weight_decay[i]);
    a.vec = bits ? 0 : 1;
    blocks += nb;
    kind[i] = n ? (gt * 3 + pt) * 2 + (eight ? 1 : 0) : -1;
  }
  // a tensor given twice, or two that share memory, would be updated by two workgroups at once
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.lo < y.lo; });
  uintptr_t end_read = 0, end_written = 0;
  for (const Span& s : spans) {
    TORCH_CHECK(s.lo >= end_written && (!s.written || s.lo >= end_read),
                "adamw_multi: two of the tensors share memory (or one is given twice)");
    (s.written ? end_written : end_read) = std::max(s.written ? end_written : end_read, s.hi);
  }
  const hipStream_t stream = current.stream();
  AdamTable tab;
  for (int k = 0; k < 18; ++k) {
    int count = 0;
    int64_t units = 0;
    auto flush = [&]() {
      if (!count) return;
      const int rc = st_adamw_multi(&tab, count, &h, k / 6, (k / 2) % 3, k & 1, stream);
      TORCH_CHECK(rc == 0, "st_amd::adamw_multi_ launch failed with code ", rc);
      count = 0;
      units = 0;
    };
    for (size_t i = 0; i < N; ++i) {
      if (kind[i] != k) continue;
      const int64_t u = ((all[i].n + kAdamBlock - 1) / kAdamBlock + kAdamUnit - 1) / kAdamUnit;
      TORCH_CHECK(u <= INT32_MAX / 2, "adamw_multi: param ", i, " is too large");
      if (count == kAdamTensors || units + u > INT32_MAX / 2) flush();
      units += u;
      tab.t[count] = all[i];
      tab.t[count++].unit_end = (int)units;
    }
    flush();
  }
  // the kernel writes behind autograd's back: a graph that saved what it wrote has to notice
  for (const at::TensorList l : {params, exp_avg, exp_avg_sq, masters, scales})
    for (const auto& t : l)
      if (t.defined()) t.unsafeGetTensorImpl()->bump_version();
  if (h.write_grads)
    for (const auto& t : grads) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st_amd, m) {
  m.def("adamw_multi_(Tensor(a!)[] params, Tensor(f!)[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, "
        "Tensor(d!)[] masters, Tensor(e!)[] scales, Tensor? clip_coef, float[] weight_decay, float lr, float beta1, "
        "float beta2, float eps, int step, bool scale_grads) -> ()");
}

TORCH_LIBRARY_IMPL(st_amd, CUDA, m) { m.impl("adamw_multi_", &adamw_multi_); }
