// tgs_attn_wide.hip -- tree attention of many query rows over a 16-bit cache
// (tgs_attn_wide.h), and the choice between the kernels.
#include "tgs_attn_wide.h"

namespace tgs {

hipError_t launch_attn_wide(const AttnArgs& a, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? attn::wide_type<attn::BF16, false>(a, a.QB / 32, st) : attn::wide_type<attn::F16, false>(a, a.QB / 32, st);
}
hipError_t set_attn_wide_lds() {
  const hipError_t e = attn::wide_lds_type<attn::BF16, false>(), f = attn::wide_lds_type<attn::F16, false>();
  return e != hipSuccess ? e : f;
}

AttnPlan attn_plan(int M, int D, bool e8) {
  AttnPlan p;
  p.e8 = e8;
  // Narrow up to the 32 rows its waves hold in registers.  16 sequences of 1000
  // to 3000 tokens, 4 key heads, narrow against wide (us): 8 rows, D = 64 15 : 19,
  // 128 20 : 28, 256 21 : 52; 28 rows 20 : 23, 25 : 36, 35 : 60; one sequence of
  // 2000 tokens 11 : 18.
  if (M <= 32) {
    p.wide = 0;
    p.tile = e8 ? attn::Narrow8::TILE : attn::Narrow16::TILE;
    p.QB = M <= 16 ? 16 : 32;
    p.per_cu = D == 256 ? 1 : 2;
    p.least = 4;  // one per wave
    // 8-bit caches, one workgroup each against shares and a join (us): 1015 tokens, D =
    // 128, 1 sequence 10.6 : 12.8, 8 11.6 : 16.3, 64 26.2 : 30.8; 1527 13.6 : 13.0, 14.6 :
    // 15.9, 35.8 : 40.7; 100 to 1460 tokens, 17 sequences with 8 nodes 16.5 : 23.3, 128 54
    // : 73; D = 256, where a CU has one workgroup, 1000 tokens 18.1 : 16.2.  Where there
    // are several for each worker, a long one among short ones is hidden by the others:
    // 128 sequences of 100 to 4096 tokens, 8 nodes, 119 : 133, of 400 and one of 4096 49 :
    // 53, of 2500 with one node 103 : 110.  (A 16-bit cache's sums keep the order that
    // they have.)
    p.whole = e8 && D <= 128 ? 25 : 8;
    p.round = e8 && D <= 128 ? 33 : 0;
  } else {
    p.wide = 1;
    p.tile = attn::WideGeo::TILE;
    // (48 rows in 64: 43 us where in 128 they take 35; two groups of 128 a CU 98
    // where one of 256 takes 87)
    p.QB = D == 256 || M <= 128 ? 128 : 256;
    p.per_cu = D == 256 || p.QB == 256 ? 1 : 2;
    p.least = 4;
    p.whole = 8;
    p.round = 0;
  }
  p.nqb = (M + p.QB - 1) / p.QB;
  return p;
}

hipError_t launch_attn(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st) {
  if (p.e8) return p.wide ? launch_attn_wide8(a, dtype, st) : launch_attn_narrow8(a, dtype, st);
  return p.wide ? launch_attn_wide(a, dtype, st) : launch_attn_narrow(a, dtype, st);
}

hipError_t set_attn_lds() {
  for (hipError_t e : {set_attn_narrow_lds(), set_attn_wide_lds(), set_attn_narrow8_lds(), set_attn_wide8_lds()})
    if (e != hipSuccess) return e;
  return hipSuccess;
}

}  // namespace tgs
