// The many-row attention kernel's 8-bit forms.
#include "kv_attn_many.h"

namespace pp {

int kv_attn_many(const AttnArgs& A, const AttnPlan& P, int D, int codes, int dtype, hipStream_t st) {
  if (codes == PP_KV_E2M1) return kv_attn_many4(A, P, D, dtype, st);
  if (codes == PP_KV_INT8)
    return dtype == PP_F16 ? many_width<PP_KV_INT8, IoF16>(A, P, D, st) : many_width<PP_KV_INT8, IoBf16>(A, P, D, st);
  return dtype == PP_F16 ? many_width<PP_KV_E4M3, IoF16>(A, P, D, st) : many_width<PP_KV_E4M3, IoBf16>(A, P, D, st);
}

}  // namespace pp
