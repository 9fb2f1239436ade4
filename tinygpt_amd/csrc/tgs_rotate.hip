// tgs_rotate.hip -- queries and keys of new nodes turned by their positions:
// lens[b] and the node's depth in its tree.  One read and one write of the rows;
// the cosines and sines of a token's position are found once for all its heads.
//
// Bound by bytes: 64 trees of 63 nodes, 32 query and 8 key heads of 128, 16.1 us (83 MB,
// 5.1 TB/s, a large copy's rate); by latency where nodes are few (8 of them 4.4 us).
#include "tgs_attn.h"
#include "tgs_e8.h"
#include "tgs_kv_write.h"

namespace tgs {
namespace rotate {

using kv::div_by;

constexpr int NT = 256;  // (a wave a token finds its depth: ROTATE_TOKENS of them at most)

struct Shared {
  alignas(16) e8::Turn cs[ROTATE_TOKENS][ROTARY_MAX / 2];
  uint32_t position[ROTATE_TOKENS];
};

__device__ __forceinline__ void store_row16(uint16_t* p, uint4 x) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef unsigned v4u __attribute__((ext_vector_type(4)));
  typedef v4u v4u_a2 __attribute__((aligned(2)));
  *(v4u_a2*)p = v4u{x.x, x.y, x.z, x.w};
#else
  __builtin_memcpy(p, &x, 16);
#endif
}

// Workgroup x takes tokens x, of all B T, `tokens` at a time; a thread takes units
// (16 dimensions that turn together) of their heads, both chunks of which it reads
// before it writes, so that a row may be written where it was read.
template <typename DT>
__global__ __launch_bounds__(NT) void rotate_kernel(RotateArgs a) {
  TGS_STATIC_SMEM(Shared, s);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long all = (long long)a.B * a.T, first = (long long)blockIdx.x * a.tokens;
  const int n = all - first < a.tokens ? (int)(all - first) : a.tokens;
  if (wave < n) {
    const int b = (int)((first + wave) / a.T), t = (int)(first + wave - (long long)b * a.T);
    int depth = t;
    if (a.parents) {
      int par = lane < a.T ? a.parents[(long long)b * a.T + lane] : -1;
      par = par < lane ? par : -1;
      const u64 line = attn::ancestors_of(par);
      depth = __popcll(attn::lane_bits(line, t)) - 1;
    }
    const int len = a.lens[b];
    if (lane == 0) s.position[wave] = (uint32_t)(len > 0 ? len : 0) + (uint32_t)depth;
  }
  __syncthreads();
  const int half = a.rot.dims >> 1;
  for (int e = tid; e < n * half; e += NT) {
    const int i = div_by((unsigned)e, a.turns), j = e - i * half;
    s.cs[i][j] = e8::turn(s.position[i], a.rot.freq[j]);
  }
  __syncthreads();
  const int U = e8::units(a.D), heads = a.q.heads + a.k.heads;
  for (int e = tid; e < n * heads * U; e += NT) {
    const unsigned row = div_by((unsigned)e, a.units), u = (unsigned)e - row * U;
    const int i = div_by(row, a.heads);
    int h = row - i * heads;
    const int b = (int)((first + i) / a.T);
    const long long t = first + i - (long long)b * a.T;
    const bool key = h >= a.q.heads;
    const tgs_rotate_rows& r = key ? a.k : a.q;
    if (key) h -= a.q.heads;
    const uint16_t* from = (const uint16_t*)r.x + b * r.x_seq + t * r.x_tok + h * r.x_head;
    uint16_t* to = (uint16_t*)r.out + b * r.out_seq + t * r.out_tok + h * r.out_head;
    const e8::Unit w = e8::unit_of((int)u, a.D, a.rot.dims, a.rot.pairs);
    if (w.angle < 0 && from == to) continue;
    const uint4 lo = load_row16<false>(from + w.a), hi = w.b >= 0 ? load_row16<false>(from + w.b) : lo;
    uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (w.angle >= 0) e8::turn_words<DT>(x, s.cs[i] + w.angle, a.rot.pairs);
    store_row16(to + w.a, make_uint4(x[0], x[1], x[2], x[3]));
    if (w.b >= 0) store_row16(to + w.b, make_uint4(x[4], x[5], x[6], x[7]));
  }
}

}  // namespace rotate

hipError_t launch_rotate(const RotateArgs& a, hipStream_t st) {
  const long long all = (long long)a.B * a.T;
  const dim3 grid((unsigned)((all + a.tokens - 1) / a.tokens));
  if (a.dtype == TGS_BF16)
    hipLaunchKernelGGL((rotate::rotate_kernel<e8::BF16>), grid, dim3(rotate::NT), 0, st, a);
  else
    hipLaunchKernelGGL((rotate::rotate_kernel<e8::F16>), grid, dim3(rotate::NT), 0, st, a);
  return hipGetLastError();
}

}  // namespace tgs
