// tgs_ctx.h -- the handle behind the C ABI and the helpers its entry points
// share (device guard, error returns).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/tgs_sampler.h"

struct tgs_ctx {
  int device = 0;
  int max_batch = 0, max_vocab = 0, max_hist = 0;
  int num_cu = 256;
  size_t lds_limit = 65536;
  unsigned long long* ws = nullptr;
  int* ws_cnt = nullptr;
  int ws_rows = 0;  // chunk lists of KMAX entries the workspace holds
  size_t ws_words = 0;  // its 8-byte words
  // one allocation, zeroed once, from k64_lists on
  unsigned long long* k64_lists = nullptr;  // fused kernel chunk lists, [max_batch * kMaxSplit][64]
  unsigned long long* k64_keys = nullptr;   // fused kernel bound-exchange keys, [max_batch][K64_KEYS]
  unsigned long long* tp_lines = nullptr;   // split-kernel exchange lines, [max_batch][TOPPS_LINE]
  unsigned* k64_cnt = nullptr;  // fused kernel exchange lines (arrival counter, epoch, count words), one per row
  uint32_t* mask_table = nullptr;
  int n_states = 0, mask_vocab = 0, mask_words = 0;
  void* mask_stage = nullptr;  // tgs_mask_table_update staging (grown on demand)
  size_t mask_stage_bytes = 0;
  float* spec_blk_m = nullptr;             // speculative workspace (tgs_reserve_spec)
  unsigned long long* spec_blk_q = nullptr;
  unsigned long long* spec_blk_w = nullptr;
  void* spec_state = nullptr;
  int spec_b = 0, spec_k = -1, spec_nbs = 0;
  std::string err;
};

namespace tgs {

// 8-byte words of workspace that tree attention's parts take when a launch
// fills the chip: two parts per CU of 256 rows of 128 values (128 rows of
// 256), a maximum and a sum each.
inline size_t attn_ws_words(int num_cu) { return (size_t)num_cu * 256 * (128 + 2); }

struct DeviceGuard {
  int prev = -1;
  bool ok = false;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    ok = hipSetDevice(dev) == hipSuccess;
  }
  ~DeviceGuard() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

inline int fail(tgs_ctx* h, int code, const std::string& msg) {
  if (h) h->err = msg;
  return code;
}

inline int hip_fail(tgs_ctx* h, hipError_t e, const char* what) {
  return fail(h, TGS_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace tgs
