// The forward products of linear_act_wide.h in f16, one instance an activation.
#include "linear_act_wide.h"

extern "C" int st_linear_wide_f16(const LinearArgs* p, hipStream_t st) {
  switch (p->epi.act) {
    case kNoAct: return launch<false, false, true, kNoAct>(*p, st);
    case kRelu: return launch<false, false, true, kRelu>(*p, st);
    case kGelu: return launch<false, false, true, kGelu>(*p, st);
    case kGeluTanh: return launch<false, false, true, kGeluTanh>(*p, st);
    case kSilu: return launch<false, false, true, kSilu>(*p, st);
    default: return -2;
  }
}
