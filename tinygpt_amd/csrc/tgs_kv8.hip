// tgs_kv8.hip -- new rows into a cache held in 8 bits, their keys turned by their
// positions on the way.
//
// Layout of a layer: keys [page][kv_head][token][D], values
// [page][kv_head][token / 16][D][16], scales [page][kv_head][token / 16][2]; the
// formulas are in tgs_e8.h.  Bound by bytes (a row is read in 16 bits and written
// in 8), or by latency for single tokens.
#include "tgs_device.h"
#include "tgs_e8.h"
#include "tgs_kv.h"
#include "tgs_kv_write.h"
#include "tgs_row.h"

namespace tgs {
namespace kv8 {

using kv::div_by;

constexpr int NT = 512;

struct Shared {
  kv::WriteHead head;
  e8::Turn cs[e8::BLOCK][ROTARY_MAX / 2];
};

// What is written to a block: tokens [lo, hi) of its 16 are new, those before are
// held already; what lies behind keeps its bytes.
struct Block {
  int lo, hi;
  uint8_t* scale;
};

// The block's scale from its new numbers' largest magnitude; `shrink`: what the held
// tokens' codes are multiplied by (1: they stay), `inv`: what new numbers are.
struct Scale {
  float inv, shrink;
};
template <typename DT>
__device__ __forceinline__ Scale rescale(const Block& k, float m, int old) {
  const int need = e8::need_byte<DT>(wave_maxf(m));
  const int now = k.lo > 0 && old > need ? old : need;
  if (lane_id() == 0 && (k.lo == 0 || now != old)) *k.scale = (uint8_t)now;
  return Scale{e8::inverse_of(now), k.lo > 0 ? e8::shrink(old, now) : 1.0f};
}

__device__ __forceinline__ uint2 reencode(uint2 w, float f) {
  float x[4], y[4];
  e8::decode4(w.x, x);
  e8::decode4(w.y, y);
  return make_uint2(e8::encode4(x[0] * f, x[1] * f, x[2] * f, x[3] * f), e8::encode4(y[0] * f, y[1] * f, y[2] * f, y[3] * f));
}
__device__ __forceinline__ uint2 encode8(const float* x, float f) {
  return make_uint2(e8::encode4(x[0] * f, x[1] * f, x[2] * f, x[3] * f), e8::encode4(x[4] * f, x[5] * f, x[6] * f, x[7] * f));
}

// Bytes [lo, hi) of eight.
__device__ __forceinline__ u64 bytes_of(int lo, int hi) {
  const u64 a = lo <= 0 ? 0ull : lo >= 8 ? ~0ull : (1ull << (8 * lo)) - 1;
  const u64 b = hi <= 0 ? 0ull : hi >= 8 ? ~0ull : (1ull << (8 * hi)) - 1;
  return b & ~a;
}

// Keys of a (block, head) by one wave: a lane takes NU of its 16 * D / 16 (token,
// unit)s.  row(i): the new row of token i of the block; to: the block's codes.
template <typename DT, int NU, class F>
__device__ __forceinline__ void put_keys(const KvWriteArgs& a, const Block& k, F row, const e8::Turn (*cs)[ROTARY_MAX / 2], uint8_t* to) {
  const int lane = lane_id(), D = a.c.head_dim, U = D >> 4;
  const int old = k.lo > 0 ? *k.scale : 0;
  float x[NU][16];
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < NU; n++) {
    const unsigned e = lane + 64 * n, i = div_by(e, a.units);
#pragma unroll
    for (int j = 0; j < 16; j++) x[n][j] = 0.0f;
    if ((int)i < k.lo || (int)i >= k.hi) continue;
    const e8::Unit w = e8::unit_of((int)(e - i * U), D, a.rot.dims, a.rot.pairs);
    const uint16_t* p = row((int)i);
    const uint4 lo = load_row16<false>(p + w.a), hi = load_row16<false>(p + w.b);
    e8::widen<DT>(lo, x[n]);
    e8::widen<DT>(hi, x[n] + 8);
    if (w.angle >= 0) e8::turn_unit(x[n], cs[i] + w.angle, a.rot.pairs);
#pragma unroll
    for (int j = 0; j < 16; j++) {
      x[n][j] = e8::taken<DT>(x[n][j]);
      m = e8::most(m, x[n][j]);
    }
  }
  const Scale s = rescale<DT>(k, m, old);
#pragma unroll
  for (int n = 0; n < NU; n++) {
    const unsigned e = lane + 64 * n, i = div_by(e, a.units);
    const e8::Unit w = e8::unit_of((int)(e - i * U), D, a.rot.dims, a.rot.pairs);
    uint8_t* p = to + (long long)i * D;
    if ((int)i >= k.lo && (int)i < k.hi) {
      *(uint2*)(p + w.a) = encode8(x[n], s.inv);
      *(uint2*)(p + w.b) = encode8(x[n] + 8, s.inv);
    } else if ((int)i < k.lo && s.shrink != 1.0f) {
      *(uint2*)(p + w.a) = reencode(*(const uint2*)(p + w.a), s.shrink);
      *(uint2*)(p + w.b) = reencode(*(const uint2*)(p + w.b), s.shrink);
    }
  }
}

// Values of a (block, head) by one wave: a lane takes NU of its D (eight tokens, two
// neighbouring dimensions)s, so that a wave reads 256 contiguous bytes of a row.
template <typename DT, int NU, class F>
__device__ __forceinline__ void put_values(const KvWriteArgs& a, const Block& k, F row, uint8_t* to) {
  const int lane = lane_id(), D = a.c.head_dim, D2 = D >> 1;
  const int old = k.lo > 0 ? *k.scale : 0;
  uint32_t raw[NU][8];
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < NU; n++) {
    const int e = lane + 64 * n, o = e >= D2 ? 8 : 0, d = 2 * (e - (o ? D2 : 0));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      raw[n][i] = 0;
      if (e < D && o + i >= k.lo && o + i < k.hi) __builtin_memcpy(&raw[n][i], row(o + i) + d, 4);
    }
  }
  float x[NU][16];
#pragma unroll
  for (int n = 0; n < NU; n++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[n][i] = e8::taken<DT>(e8::from16<DT>(raw[n][i] & 0xFFFFu));
      x[n][i + 8] = e8::taken<DT>(e8::from16<DT>(raw[n][i] >> 16));
      m = e8::most(e8::most(m, x[n][i]), x[n][i + 8]);
    }
  const Scale s = rescale<DT>(k, m, old);
#pragma unroll
  for (int n = 0; n < NU; n++) {
    const int e = lane + 64 * n, o = e >= D2 ? 8 : 0, d = 2 * (e - (o ? D2 : 0));
    if (e >= D) continue;
    const u64 fresh = bytes_of(k.lo - o, k.hi - o), held = bytes_of(0, k.lo - o);
    if (fresh == 0 && (held == 0 || s.shrink == 1.0f)) continue;
    uint8_t* p = to + d * e8::BLOCK + o;
#pragma unroll
    for (int c = 0; c < 2; c++, p += e8::BLOCK) {
      uint2 w = encode8(x[n] + 8 * c, s.inv);
      if (fresh != ~0ull) {
        const uint2 was = *(const uint2*)p;
        uint2 kept = was;
        if (s.shrink != 1.0f) kept = reencode(was, s.shrink);
        auto join = [](uint32_t f, uint32_t h, uint32_t neu, uint32_t kp, uint32_t rest) {
          return (neu & f) | (kp & h) | (rest & ~(f | h));
        };
        w.x = join((uint32_t)fresh, (uint32_t)held, w.x, kept.x, was.x);
        w.y = join((uint32_t)(fresh >> 32), (uint32_t)(held >> 32), w.y, kept.y, was.y);
      }
      *(uint2*)p = w;
    }
  }
}

// Workgroup (x, sequence b, layer l) over the 16-token blocks x, x + nblk, ... of
// the positions that b's new rows take; a wave takes the keys or the values of a
// head of a block, whose largest magnitude is then one reduction over the wave.
template <typename DT, int NU, bool COMMIT>
__global__ __launch_bounds__(NT) void write_kernel(KvWriteArgs a) {
  TGS_STATIC_SMEM(Shared, sh);
  kv::WriteHead& s = sh.head;
  const int x = blockIdx.x % a.nblk, bl = blockIdx.x / a.nblk, b = bl % a.B, l = bl / a.B;
  const int tid = threadIdx.x;
  int len, n;
  if (!kv::write_head<COMMIT>(a, s, b, l == 0 && x == 0, len, n)) return;
  const int* table = a.tables + (long long)b * a.P;
  const int D = a.c.head_dim, H = a.c.kv_heads, page = 1 << a.page_shift;
  const uint16_t* kn = (const uint16_t*)a.r.k + l * a.r.k_layer + b * a.r.k_seq;
  const uint16_t* vn = (const uint16_t*)a.r.v + l * a.r.v_layer + b * a.r.v_seq;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
  const int last = (len + n - 1) >> 4;
  for (int blk = (len >> 4) + x; blk <= last; blk += a.nblk) {
    const int pos0 = blk << 4;
    Block k;
    k.lo = len > pos0 ? len - pos0 : 0;
    k.hi = len + n < pos0 + e8::BLOCK ? len + n - pos0 : e8::BLOCK;
    const long long pg = table[pos0 >> a.page_shift];
    const int in_page = pos0 & (page - 1);
    if (a.rot.freq) {
      const int half = a.rot.dims >> 1;
      __syncthreads();  // (the block before is done with the table)
      for (int e = tid; e < (k.hi - k.lo) * half; e += (int)blockDim.x) {
        const int i = e / half, j = e - i * half;
        sh.cs[k.lo + i][j] = e8::turn((uint32_t)(pos0 + k.lo + i), a.rot.freq[j]);
      }
      __syncthreads();
    }
    for (int t = wave; t < 2 * H; t += waves) {
      const int h = t >> 1;
      k.scale = a.scales + l * a.s_layer + pg * a.s_page + ((((long long)h << a.page_shift) + in_page) >> 4) * 2 + (t & 1);
      const long long at = (((long long)h << a.page_shift) + in_page) * D;  // (keys and values alike)
      auto node = [&](int i) { return COMMIT ? s.path[pos0 + i - len] : pos0 + i - len; };
      if (t & 1)
        put_values<DT, NU>(a, k, [&](int i) { return vn + node(i) * a.r.v_tok + h * a.r.v_head; },
                           (uint8_t*)a.c.v + l * a.c.v_layer + pg * a.c.v_page + at);
      else
        put_keys<DT, NU>(a, k, [&](int i) { return kn + node(i) * a.r.k_tok + h * a.r.k_head; }, sh.cs,
                         (uint8_t*)a.c.k + l * a.c.k_layer + pg * a.c.k_page + at);
    }
  }
}

template <typename DT, bool COMMIT>
hipError_t run(const KvWriteArgs& a, hipStream_t st) {
  const dim3 grid(a.nblk * a.B * a.c.layers);
  const int waves = 2 * a.c.kv_heads < NT / 64 ? 2 * a.c.kv_heads : NT / 64;
  if (a.c.head_dim <= 64)
    hipLaunchKernelGGL((write_kernel<DT, 1, COMMIT>), grid, dim3(64 * waves), 0, st, a);
  else if (a.c.head_dim <= 128)
    hipLaunchKernelGGL((write_kernel<DT, 2, COMMIT>), grid, dim3(64 * waves), 0, st, a);
  else
    hipLaunchKernelGGL((write_kernel<DT, 4, COMMIT>), grid, dim3(64 * waves), 0, st, a);
  return hipGetLastError();
}

}  // namespace kv8

hipError_t launch_kv8_append(const KvWriteArgs& a, hipStream_t st) {
  return a.c.dtype == TGS_BF16 ? kv8::run<e8::BF16, false>(a, st) : kv8::run<e8::F16, false>(a, st);
}
hipError_t launch_kv8_commit(const KvWriteArgs& a, hipStream_t st) {
  return a.c.dtype == TGS_BF16 ? kv8::run<e8::BF16, true>(a, st) : kv8::run<e8::F16, true>(a, st);
}

}  // namespace tgs
