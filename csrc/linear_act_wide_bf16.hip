// The forward products of linear_act_wide.h in bf16, one instance an activation.
#include "linear_act_wide.h"

extern "C" int st_linear_wide_bf16(const LinearArgs* p, hipStream_t st) {
  switch (p->epi.act) {
    case kNoAct: return launch<false, false, false, kNoAct>(*p, st);
    case kRelu: return launch<false, false, false, kRelu>(*p, st);
    case kGelu: return launch<false, false, false, kGelu>(*p, st);
    case kGeluTanh: return launch<false, false, false, kGeluTanh>(*p, st);
    case kSilu: return launch<false, false, false, kSilu>(*p, st);
    default: return -2;
  }
}
