// tgs_kv_write.h -- what the kernels that write new rows to a cache share: which
// rows they are, and whether they fit.
#pragma once

#include "tgs_device.h"
#include "tgs_kv.h"

namespace tgs {
namespace kv {

__device__ __forceinline__ unsigned div_by(unsigned x, FastDiv f) { return f.d == 1 ? x : __umulhi(x, f.m); }

struct WriteHead {
  int path[KV_MAX_NODES];
  int n;
};

// The accepted path of a tree by one wave, node j in lane j: from the root on,
// the lowest child whose drafted token is the one sampled at its parent.
// Children come after their parents, so each step moves to a higher node and
// the walk ends.  Returns the nodes taken, the root among them.
__device__ __forceinline__ int accept_walk(const int* parents, const int* draft, const int* sampled, int T, int* path) {
  const int lane = lane_id();
  const bool in = lane < T;
  const int par = in ? parents[lane] : -2, tok = in ? draft[lane] : 0, smp = in ? sampled[lane] : 0;
  int cur = 0, n = 0;
  while (true) {
    if (lane == n) path[n] = cur;
    n++;
    const int want = (int)readlane_u32((uint32_t)smp, cur);
    const u64 fits = __ballot(in && lane > cur && par == cur && tok == want);
    if (fits == 0) return n;
    cur = __ffsll((long long)fits) - 1;
  }
}

// How many rows follow sequence b's len tokens (COMMIT: those of s.path, found here by
// the whole workgroup).
template <bool COMMIT>
__device__ __forceinline__ int rows_of(const KvWriteArgs& a, WriteHead& s, int b) {
  if constexpr (!COMMIT) return a.counts ? a.counts[b] : a.T;
  const long long o = (long long)b * a.T;
  if (threadIdx.x < 64) {
    const int cnt = accept_walk(a.parents + o, a.draft + o, a.sampled + o, a.T, s.path);
    if (threadIdx.x == 0) s.n = cnt;
  }
  __syncthreads();
  return s.n;
}

// What does not fit is not written: a count outside [0, T], positions past the
// table, pages outside the pool (a thread looks at its share of them).
__device__ __forceinline__ bool past_table(const KvWriteArgs& a, int len, int n) {
  return n < 0 || n > a.T || len < 0 || (long long)len + n > ((long long)a.P << a.page_shift);
}
__device__ __forceinline__ bool outside_pool(const KvWriteArgs& a, const int* table, int len, int n) {
  int bad = 0;
  if (n > 0)
    for (int i = (len >> a.page_shift) + (int)threadIdx.x; i <= (len + n - 1) >> a.page_shift; i += (int)blockDim.x)
      bad |= (unsigned)table[i] >= (unsigned)a.c.n_pages;
  return bad;
}

// The outputs but the cache, by one workgroup.
template <bool COMMIT>
__device__ __forceinline__ void report(const KvWriteArgs& a, const WriteHead& s, int b, int len, int n, bool bad) {
  const int tid = threadIdx.x;
  if (tid == 0) {
    a.lens_out[b] = bad ? -1 : len + n;
    if (COMMIT) a.n_acc[b] = n - 1;
  }
  if (COMMIT && tid < a.T) {
    const long long o = (long long)b * a.T;
    a.path[o + tid] = tid < n ? s.path[tid] : -1;
    int t = -1;  // the accepted nodes' tokens, then the one sampled at the last
    if (tid < n - 1) t = a.draft[o + s.path[tid + 1]];
    if (tid == n - 1) t = a.sampled[o + s.path[tid]];
    a.tokens[o + tid] = t;
  }
}

}  // namespace kv
}  // namespace tgs
