// The many-row attention kernel's 4-bit forms.
#include "kv_attn_many.h"

namespace pp {

int kv_attn_many4(const AttnArgs& A, const AttnPlan& P, int D, int dtype, hipStream_t st) {
  return dtype == PP_F16 ? many_width<PP_KV_E2M1, IoF16>(A, P, D, st) : many_width<PP_KV_E2M1, IoBf16>(A, P, D, st);
}

}  // namespace pp
