// tgs_attn_wide8.hip -- tree attention of many query rows over an 8-bit cache
// (tgs_attn_wide.h).
#include "tgs_attn_wide.h"

namespace tgs {

hipError_t launch_attn_wide8(const AttnArgs& a, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? attn::wide_type<attn::BF16, true>(a, a.QB / 32, st) : attn::wide_type<attn::F16, true>(a, a.QB / 32, st);
}
hipError_t set_attn_wide8_lds() {
  const hipError_t e = attn::wide_lds_type<attn::BF16, true>(), f = attn::wide_lds_type<attn::F16, true>();
  return e != hipSuccess ? e : f;
}

}  // namespace tgs
