// tgs_attn_narrow8.hip -- tree attention of few query rows over an 8-bit cache
// (tgs_attn_narrow.h).
#include "tgs_attn_narrow.h"

namespace tgs {

hipError_t launch_attn_narrow8(const AttnArgs& a, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? attn::narrow_type<attn::BF16, true>(a, a.QB / 16, st) : attn::narrow_type<attn::F16, true>(a, a.QB / 16, st);
}
hipError_t set_attn_narrow8_lds() {
  const hipError_t e = attn::narrow_lds_type<attn::BF16, true>(), f = attn::narrow_lds_type<attn::F16, true>();
  return e != hipSuccess ? e : f;
}

}  // namespace tgs
