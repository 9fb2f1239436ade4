// tgs_attn.h -- attention of drafted nodes over a paged cache: what the two
// kernels (tgs_attn_narrow.hip, tgs_attn_wide.hip) and the join share.
//
//   out[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]
// over j in the cache's len tokens and in node i's ancestors and itself.  The
// G query heads of a key head and the T nodes are M = T G rows that read the
// same keys and values.
//
// Both products run transposed on the matrix units, S^T = K Q^T and
// O^T = V^T P^T, so that a lane's scores belong to one query row and are, as
// they stand, the second product's operand: the tokens that the first
// product's rows stand for are permuted such that a lane ends with eight
// consecutive tokens, which is also one 16-byte vector of the values' layout.
// No score goes through LDS or another lane.  The running maximum and sum are
// 32-bit; P is rounded to the inputs' 16 bits (half a step of a weight in
// [0, 1], the precision of the values it multiplies), O accumulates in 32.
//
// Work is cut by an even share of tiles per worker, not by sequence: worker w
// of N takes tiles [w U / N, (w + 1) U / N) of the U tiles of all sequences
// and key heads in order, whatever the lengths are.  A (sequence, key head)
// that lies in one worker's range is written at once; the parts of the others
// go to the workspace and are joined by a second launch in a fixed order.
#pragma once

#include "tgs_device.h"
#include "tgs_kv.h"
#include "tgs_row.h"

namespace tgs {
namespace attn {

typedef float f32x4 __attribute__((vector_size(16)));
typedef float f32x16 __attribute__((vector_size(64)));
typedef uint32_t Vec __attribute__((vector_size(16)));  // eight 16-bit values
__device__ __forceinline__ Vec vec16(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return Vec{a, b, c, d}; }
// At any alignment of the values.
__device__ __forceinline__ Vec load16(const uint16_t* p) {
  typedef Vec Vec2 __attribute__((aligned(2)));
  return *(const Vec2*)p;
}

struct BF16 {};
struct F16 {};

#if defined(__HIP_DEVICE_COMPILE__)
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#endif

// c + a b, 16 x 16 with 32 products each: lane l holds a's row (b's column)
// l % 16, k = 8 (l / 16) .. + 7, and c's rows 4 (l / 16) .. + 3 of column l % 16.
template <typename DT>
__device__ __forceinline__ f32x4 mfma16(Vec a, Vec b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (__is_same(DT, BF16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#elif defined(TGS_HOST_MFMA)
  return hipcpu_mfma<16, __is_same(DT, BF16)>(a, b, c);
#else
  (void)a, (void)b;
  return c;
#endif
}

// The same for 32 x 32 with 16 products: row or column l % 32, k = 8 (l / 32)
// .. + 7; c's element i is row 8 (i / 4) + 4 (l / 32) + i % 4.
template <typename DT>
__device__ __forceinline__ f32x16 mfma32(Vec a, Vec b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (__is_same(DT, BF16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#elif defined(TGS_HOST_MFMA)
  return hipcpu_mfma<32, __is_same(DT, BF16)>(a, b, c);
#else
  (void)a, (void)b;
  return c;
#endif
}

// Two floats to 16 bits, to the nearest, ties to even: the first in the low half.
template <typename DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  const f32x2v x = {lo, hi};
  if constexpr (__is_same(DT, BF16))
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
#elif defined(TGS_HOST_MFMA)
  return hipcpu_pack2<__is_same(DT, BF16)>(lo, hi);
#else
  (void)lo, (void)hi;
  return 0;
#endif
}

// 2^x by the hardware instruction: results below 2^-126 are 0, weights that
// no sum of at least 1 shows.
__device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);
#else
  return exp2f(x);
#endif
}

// No instruction moves across it.
__device__ __forceinline__ void sched_fence() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// A workgroup barrier for LDS alone: requests to memory stay on their way
// (__syncthreads may wait for them).
__device__ __forceinline__ void lds_barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
#elif defined(TGS_HOST_MFMA)
  __syncthreads();
#endif
}

constexpr int NTILE = 32, WTILE = 64;  // tokens of a tile of the narrow and of the wide kernel
constexpr float NEG = -__builtin_inff();

// A query row's running state (maximum in units of log2, scaled) grows only
// when a score passes it by more than SLACK: weights up to 2^SLACK keep their
// relative precision in 16 bits and 32-bit sums, and most tiles skip the
// exchange between lanes and the scaling of O.
constexpr float SLACK = 6.0f;

// ------------------------------------------------------------------ shares

// A value that every lane of the wave holds, for the scalar unit: what loops,
// branches and addresses derive from it takes no vector registers.
__device__ __forceinline__ int uniform(int x) { return (int)__builtin_amdgcn_readfirstlane((unsigned)x); }

__device__ __forceinline__ int clamp_len(const AttnArgs& a, int n) {
  const long long cap = (long long)a.P << a.page_shift;
  return n < 0 ? 0 : n > cap ? (int)cap : n;
}
__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) { return uniform(clamp_len(a, a.lens[b])); }
template <int TILE>
__device__ __forceinline__ int cache_tiles(const AttnArgs& a, int b) {
  return (seq_len(a, b) + TILE - 1) / TILE;
}
template <int TILE>  // (a sequence per lane)
__device__ __forceinline__ int lane_tiles(const AttnArgs& a, int b) {
  return (clamp_len(a, a.lens[b]) + TILE - 1) / TILE;
}

// Tiles of sequences before b (of one key head), and of all: by one wave.
template <int TILE>
__device__ __forceinline__ void tiles_before(const AttnArgs& a, int b, int& before, int& all) {
  const int tree = (a.T + TILE - 1) / TILE;
  int x = 0, y = 0;
  for (int i = lane_id(); i < a.B; i += 64) {
    const int n = lane_tiles<TILE>(a, i) + tree;
    y += n;
    if (i < b) x += n;
  }
  before = uniform(wave_sum(x));
  all = uniform(wave_sum(y));
}

// The sequence that holds tile t of one key head's tiles in order, and the tiles before it: by one wave.
template <int TILE>
__device__ __forceinline__ void find_tile(const AttnArgs& a, long long t, int heads, int& b, long long& before) {
  const int tree = (a.T + TILE - 1) / TILE, lane = lane_id();
  before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? lane_tiles<TILE>(a, b0 + lane) + tree : 0;
    const int incl = wave_incl_scan(n);
    const u64 ends = __ballot(b0 + lane < a.B && before + (long long)incl * heads > t);
    if (ends) {
      const int at = __ffsll((long long)ends) - 1;
      b = b0 + at;
      const int prev = (int)readlane_u32((uint32_t)incl, at) - (int)readlane_u32((uint32_t)n, at);
      before += (long long)prev * heads;
      return;
    }
    before += (long long)(int)readlane_u32((uint32_t)incl, 63) * heads;
  }
  b = a.B;
}

__device__ __forceinline__ long long share_start(long long U, int N, int w) { return U * w / N; }

// ------------------------------------------------------------------ the tree

// Ancestors of each node, itself among them, as bits: by one wave, node in
// lane.  A parent that is not an earlier node makes a root.
__device__ __forceinline__ u64 ancestors(const AttnArgs& a, int b) {
  const int lane = lane_id();
  if (!a.parents) return lane == 63 ? ~0ull : (2ull << lane) - 1;
  int par = lane < a.T ? a.parents[(long long)b * a.T + lane] : -1;
  if (par >= lane) par = -1;
  u64 m = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; i++) {  // paths double
    const int from = par < 0 ? lane : par;
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)m, from, 64), hi = (uint32_t)__shfl((int)(m >> 32), from, 64);
    const int up = __shfl(par, from, 64);
    if (par >= 0) {
      m |= ((u64)hi << 32) | lo;
      par = up;
    }
  }
  return m;
}

// Of the eight 16-bit values of x those with index < n stay (n <= 0: none), the others become 0.
__device__ __forceinline__ Vec keep_first(Vec x, int n) {
  auto word = [&](uint32_t w, int i) { return n >= i + 2 ? w : n == i + 1 ? w & 0xFFFFu : 0u; };
  return vec16(word(x[0], 0), word(x[1], 2), word(x[2], 4), word(x[3], 6));
}

// 8 x 8 16-bit values, rows x[j], turned: x[i] becomes the i-th of every row.
__device__ __forceinline__ void transpose8(Vec (&x)[8]) {
  uint32_t w[8][4];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    for (int i = 0; i < 4; i++) w[j][i] = x[j][i];
  }
  auto lo = [&](int i, int j) { return (w[j][i] & 0xFFFFu) | (w[j + 1][i] << 16); };
  auto hi = [&](int i, int j) { return (w[j][i] >> 16) | (w[j + 1][i] & 0xFFFF0000u); };
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = vec16(lo(i, 0), lo(i, 2), lo(i, 4), lo(i, 6));
    x[2 * i + 1] = vec16(hi(i, 0), hi(i, 2), hi(i, 4), hi(i, 6));
  }
}

// Eight tokens' values of one d, tok .. tok + 7 of the drafted nodes; past the last 0.
__device__ __forceinline__ Vec tree_values(const uint16_t* v, long long stride, int tok, int T) {
  uint32_t x[8];
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = tok + j < T ? v[(tok + j) * stride] : 0u;
  return vec16(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
}

// ------------------------------------------------------------------ results

template <typename DT>
__device__ __forceinline__ void store4(uint16_t* p, f32x4 x) {
  uint2 w;
  w.x = pack2<DT>(x[0], x[1]);
  w.y = pack2<DT>(x[2], x[3]);
  *(uint2*)p = w;
}

// Natural logsumexp from the maximum (log2 units) and the sum.
__device__ __forceinline__ float row_lse(float m, float l) {
  return (float)(((double)m + (double)log2f(l)) * 0.69314718055994530942);
}

// Sum over the wave, the same in every lane.
__device__ __forceinline__ float wave_sumf(float x) {
  x += xor_lane<32>(x);
  x += xor_lane<16>(x);
  x += xor_lane<8>(x);
  x += xor_lane<4>(x);
  x += xor_lane<2>(x);
  return x + xor_lane<1>(x);
}

// Joins the parts of (sequence, key head)s that several workers hold: a wave
// per output row, in the workers' order.
template <typename DT, int TILE>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  const int lane = lane_id();
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b, h, query row)
  if (row >= (long long)a.B * a.Hkv * a.M) return;
  const int i = (int)(row % a.M), bh = (int)(row / a.M), h = bh % a.Hkv, b = bh / a.Hkv;
  int before, all;
  tiles_before<TILE>(a, b, before, all);
  const int nt = cache_tiles<TILE>(a, b) + (a.T + TILE - 1) / TILE;
  const long long U = (long long)all * a.Hkv, s0 = (long long)before * a.Hkv + (long long)h * nt, s1 = s0 + nt;
  const int N = a.nwg;
  const int w0 = (int)(((s0 + 1) * N - 1) / U), w1 = (int)((s1 * N - 1) / U);
  if (w0 == w1) return;
  // A lane per part (64 at a time): its place, maximum and sum.  A worker's
  // second part is the one that starts past its share's first tile.
  const int qb = i / a.QB, r = i - qb * a.QB;
  auto part_of = [&](int w) -> int {
    if (w > w1) return -1;
    const long long from = share_start(U, N, w);
    if (from == share_start(U, N, w + 1)) return -1;
    return ((qb * N + w) * 2 + (from < s0)) * a.QB + r;
  };
  float m = NEG;
  for (int w = w0; w <= w1; w += 64) {
    const int p = part_of(w + lane);
    m = fmaxf(m, p < 0 ? NEG : a.part_ml[2ll * p]);
  }
  m = wave_maxf(m);
  float l = 0.0f;
  float o[4] = {0, 0, 0, 0};
  for (int w = w0; w <= w1; w += 64) {
    int p = part_of(w + lane);
    const float f = p < 0 ? 0.0f : exp2_hw(a.part_ml[2ll * p] - m);
    l += p < 0 ? 0.0f : f * a.part_ml[2ll * p + 1];
    p = p < 0 ? 0 : p;  // (its factor is 0)
    const int n = w1 - w + 1 < 64 ? w1 - w + 1 : 64;
    for (int j = 0; j < n; j += 4) {
      float x[4][4];
#pragma unroll
      for (int y = 0; y < 4; y++) {  // (past the last part: part 0's values, not used)
        const long long at = (long long)(int)readlane_u32((uint32_t)p, j + y < n ? j + y : j) * a.D;
#pragma unroll
        for (int z = 0; z < 4; z++) x[y][z] = z * 64 + lane < a.D ? a.part_o[at + z * 64 + lane] : 0.0f;
      }
#pragma unroll
      for (int y = 0; y < 4; y++) {
        const float g = j + y < n ? readlane_f32(f, j + y < n ? j + y : j) : 0.0f;
#pragma unroll
        for (int z = 0; z < 4; z++) o[z] += g == 0.0f ? 0.0f : g * x[y][z];
      }
    }
  }
  l = wave_sumf(l);
  const int t = i / a.G, hq = h * a.G + i % a.G;
  const long long out = ((long long)b * a.T + t) * a.Hq + hq;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = j * 64 + lane;
    if (d < a.D) ((uint16_t*)a.out)[out * a.D + d] = (uint16_t)pack2<DT>(o[j] / l, 0.0f);
  }
  if (a.lse && lane == 0) a.lse[out] = row_lse(m, l);
}

}  // namespace attn

hipError_t launch_attn_narrow(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st);
hipError_t launch_attn_wide(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st);
hipError_t set_attn_narrow_lds(size_t bytes);

}  // namespace tgs
