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
// 32-bit; P is rounded to the inputs' 16 bits (half a step of each weight, the
// precision of the values it multiplies), O accumulates in 32.  O is divided by
// the sum of the rounded weights, so that what they are off by together cancels
// (fp16, 217 tokens: the error against 64 bits, over that of 32-bit weights, from
// 1.21 to 1.11 in the mean and from 1.55 to 1.21 at worst); the logsumexp is
// that of the unrounded ones.  The second sum costs nothing that shows below 32
// rows and 1 to 2 % above.
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

// c plus the products of the two 16-bit values of x and those of y, in 32 bits.
template <typename DT>
__device__ __forceinline__ float dot2(uint32_t x, uint32_t y, float c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (__is_same(DT, BF16))
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, y), c, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), __builtin_bit_cast(f16x2, y), c, false);
#elif defined(TGS_HOST_MFMA)
  auto value = [](uint32_t u) { return hipcpu_to_float((uint16_t)u, __is_same(DT, BF16)); };
  return c + value(x) * value(y) + value(x >> 16) * value(y >> 16);
#else
  (void)x, (void)y;
  return c;
#endif
}
template <typename DT>
__device__ __forceinline__ float add2(uint32_t x, float c) {
  return dot2<DT>(x, __is_same(DT, BF16) ? 0x3F803F80u : 0x3C003C00u, c);
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

// The length by which an append, a commit or a fork reports that rows did not
// fit: such a sequence's rows become NaN.
constexpr int FAILED = -1;

// A query row's running state (maximum in units of log2, scaled) grows only
// when a score passes it by more than SLACK: weights up to 2^SLACK keep their
// relative precision in 16 bits and 32-bit sums, and most tiles skip the
// exchange between lanes and the scaling of O.
constexpr float SLACK = 6.0f;

// fp16 holds numbers below 2^-14 with fewer bits and none below 2^-25.  Its
// weights are therefore relative to a maximum 2^9 lower: they reach 2^(9 + SLACK),
// half of its largest number, and down to 2^-23 of the row's largest they
// keep their precision.
template <typename DT>
constexpr float lift() { return __is_same(DT, BF16) ? 0.0f : 9.0f; }

// ------------------------------------------------------------------ shares

// A value that every lane of the wave holds, for the scalar unit: what loops,
// branches and addresses derive from it takes no vector registers.
__device__ __forceinline__ int uniform(int x) { return (int)__builtin_amdgcn_readfirstlane((unsigned)x); }

__device__ __forceinline__ int clamp_len(const AttnArgs& a, int n) {
  const long long cap = (long long)a.P << a.page_shift;
  return n < 0 ? 0 : n > cap ? (int)cap : n;
}
template <int TILE>
__device__ __forceinline__ int cache_tiles(const AttnArgs& a, int b) {
  return (uniform(clamp_len(a, a.lens[b])) + TILE - 1) / TILE;
}
template <int TILE>  // (a sequence per lane)
__device__ __forceinline__ int lane_tiles(const AttnArgs& a, int b) {
  return (clamp_len(a, a.lens[b]) + TILE - 1) / TILE;
}

// What a (sequence, key head) costs beyond its tiles (queries, the first
// tile's latency, the result), counted in tiles when shares are cut: a worker
// whose share lies in short sequences would else end last (32 sequences of 100
// to 4096 tokens, 8 key heads of 128: 86 us without, 63 with 4 or more).
template <int TILE>
constexpr int extra() { return TILE == NTILE ? 8 : 4; }

// Tiles of sequences before b (of one key head), and of all: by one wave.
template <int TILE>
__device__ __forceinline__ void tiles_before(const AttnArgs& a, int b, int& before, int& all) {
  const int tree = (a.T + TILE - 1) / TILE + extra<TILE>();
  int x = 0, y = 0;
  for (int i = lane_id(); i < a.B; i += 64) {
    const int n = lane_tiles<TILE>(a, i) + tree;
    y += n;
    if (i < b) x += n;
  }
  before = uniform(wave_sum(x));
  all = uniform(wave_sum(y));
}

// First tile of worker w's share: floor(U w / N), in 32 bits where U allows
// (w < N <= 2^16: with U = q N + r it is w q + floor(w r / N)).
__device__ __forceinline__ long long share_start(long long U, int N, int w) {
  if (U >> 31) return U * w / N;
  const unsigned q = (unsigned)U / (unsigned)N, r = (unsigned)U - q * (unsigned)N;
  return (long long)w * q + (unsigned)w * r / (unsigned)N;
}

// A worker's place: its share [u0, u1), and of tile u0 the sequence, key head
// and tile in them, with the tiles of that sequence (drafted nodes and the
// extra ones, behind which nothing lies, included).
struct Place {
  long long u0, u1;
  int b, h, at, nt;
};
template <int TILE>
__device__ __forceinline__ Place find_place(const AttnArgs& a, int w) {
  const int tree = (a.T + TILE - 1) / TILE + extra<TILE>(), lane = lane_id();
  const int mine = lane < a.B ? lane_tiles<TILE>(a, lane) + tree : 0;  // (of the first 64 sequences)
  int y = mine;
  for (int i = lane + 64; i < a.B; i += 64) y += lane_tiles<TILE>(a, i) + tree;
  const long long U = (long long)uniform(wave_sum(y)) * a.Hkv;
  Place p{share_start(U, a.nwg, w), share_start(U, a.nwg, w + 1), 0, 0, 0, 0};
  if (p.u0 == p.u1) return p;
  long long before = 0;
  for (int b0 = 0;; b0 += 64) {
    const int n = b0 == 0 ? mine : b0 + lane < a.B ? lane_tiles<TILE>(a, b0 + lane) + tree : 0;
    const int incl = wave_incl_scan(n);
    const u64 ends = __ballot(b0 + lane < a.B && before + (long long)incl * a.Hkv > p.u0);
    if (ends) {
      const int at = __ffsll((long long)ends) - 1;
      p.b = b0 + at;
      p.nt = (int)readlane_u32((uint32_t)n, at);
      before += (long long)((int)readlane_u32((uint32_t)incl, at) - p.nt) * a.Hkv;
      const long long in = p.u0 - before;
      p.h = in >> 31 ? (int)(in / p.nt) : (int)((unsigned)in / (unsigned)p.nt);
      p.at = (int)(in - (long long)p.h * p.nt);
      return p;
    }
    before += (long long)(int)readlane_u32((uint32_t)incl, 63) * a.Hkv;
  }
}

// ------------------------------------------------------------------ the tree

// The parent of node `lane` of sequence b: an earlier node, or -1.
__device__ __forceinline__ int parent_of(const AttnArgs& a, int b) {
  const int lane = lane_id();
  if (!a.parents) return lane - 1;
  const int par = lane < a.T ? a.parents[(long long)b * a.T + lane] : -1;
  return par < lane ? par : -1;
}

// Ancestors of each node, itself among them, as bits, from its parent: by one
// wave, node in lane.
__device__ __forceinline__ u64 ancestors(const AttnArgs& a, int par) {
  const int lane = lane_id();
  if (!a.parents) return lane == 63 ? ~0ull : (2ull << lane) - 1;
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

// Lane `from`'s 64 bits.
__device__ __forceinline__ u64 lane_bits(u64 m, int from) {
  return ((u64)(uint32_t)__shfl((int)(m >> 32), from, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)m, from, 64);
}

// A mask of the first n of eight 16-bit values (n <= 0: none).
__device__ __forceinline__ Vec first_of(int n) {
  const u64 lo = n >= 4 ? ~0ull : n <= 0 ? 0ull : (1ull << (16 * n)) - 1;
  const u64 hi = n >= 8 ? ~0ull : n <= 4 ? 0ull : (1ull << (16 * n - 64)) - 1;
  return vec16((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// A mask of the i-th of eight 16-bit values (i = 8: of none).
__device__ __forceinline__ Vec only(int i) {
  const uint32_t m = i & 1 ? 0xFFFF0000u : 0xFFFFu;
  return vec16(i >> 1 == 0 ? m : 0u, i >> 1 == 1 ? m : 0u, i >> 1 == 2 ? m : 0u, i >> 1 == 3 ? m : 0u);
}

// A drafted value that is no finite number would reach the rows that do not see
// its node as well, since 0 times it is NaN.  Where a drafted tile has such
// values they are taken out of it and added to the rows that see them.
// Of two 16-bit values: bits 15 and 31 of those that are not finite (a step of
// the exponent carries out of it when all its bits are set).
template <typename DT>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  constexpr bool B = __is_same(DT, BF16);
  return ((w & (B ? 0x7F807F80u : 0x7C007C00u)) + (B ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// c where all eight values are finite, else NaN (0 times each is added; code
// that every launch meets cold, so that few instructions count).
template <typename DT>
__device__ __forceinline__ float finite_or_nan(Vec x, float c) {
#pragma unroll
  for (int i = 0; i < 4; i++) c = dot2<DT>(x[i], 0u, c);
  return c;
}
// Those values, and 0 for the others.
template <typename DT>
__device__ __forceinline__ Vec odd_of(Vec x) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t m = odd_bits<DT>(x[i]) >> 15;
    x[i] &= (m << 16) - m;
  }
  return x;
}
template <typename DT>
__device__ __forceinline__ bool is_nan(uint32_t u) {
  return odd_bits<DT>(u) != 0 && (u & (__is_same(DT, BF16) ? 0x7Fu : 0x3FFu)) != 0;
}
// Elements d .. d + 3 of (b, h)'s drafted values: the sum of what is not finite
// in the nodes of `sees`, 0 where all is.
template <typename DT>
__device__ __forceinline__ f32x4 odd_sum(const AttnArgs& a, int b, int h, u64 sees, int d) {
  const uint16_t* p = (const uint16_t*)a.v_new + b * a.vn_b + h * a.vn_h + d;
  f32x4 s = {0, 0, 0, 0};
  for (int j = 0; j < a.T; j++, p += a.vn_t) {
    if (!(sees >> j & 1)) continue;
#pragma unroll
    for (int z = 0; z < 4; z++) {
      const uint32_t u = p[z];
      if (odd_bits<DT>(u)) s[z] += tg_u2f((u & 0x8000u) << 16 | 0x7F800000u | (is_nan<DT>(u) ? 0x400000u : 0u));
    }
  }
  return s;
}

// x where bit i of bits is set, else -inf.
__device__ __forceinline__ float seen(float x, uint32_t bits, int i) {
  const uint32_t m = (uint32_t)((int)(bits << (31 - i)) >> 31);
  return tg_u2f((tg_f2u(x) & m) | (0xFF800000u & ~m));
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

// Joins the parts of (sequence, key head)s that several workers hold.  A
// workgroup takes R rows of one (sequence, key head): with R = 1 its four
// waves share the row's parts (few rows, many parts), with R = 16 each takes
// four rows (the places of the parts are found once for them).  Every sum runs
// in an order that the lengths alone fix.
//
// A part's sums lie as its kernel holds them: the narrow kernel's row by row,
// the wide kernel's by 32 rows, [D / 8][half][row][4], a lane's four next to the
// neighbouring rows' (its stores are 1 KB each; 64-byte pieces took 5 us more
// of 16 sequences' 63 nodes).
template <int TILE>
__device__ __forceinline__ int part_at(int D, int row, int d) {
  if (TILE == NTILE) return row * D + d;
  return (row >> 5) * 32 * D + ((d >> 3) * 64 + ((d >> 2) & 1) * 32 + (row & 31)) * 4 + (d & 3);
}

struct JoinShared {
  int part[1024];  // of this (sequence, key head)
  int n;
  float o[4][256];
  float ml[4][2];
};
constexpr int JOIN_NT = 256;

// Row i of (b, h): its sums over its weights' sum; d = 64 z + lane.
template <typename DT>
__device__ __forceinline__ void write_row(const AttnArgs& a, int b, int h, int i, const float (&o)[4], float m, float l) {
  const int lane = lane_id(), t = i / a.G, hq = h * a.G + i - t * a.G;
  const long long out = ((long long)b * a.T + t) * a.Hq + hq;
  const float rl = 1.0f / l;
#pragma unroll
  for (int z = 0; z < 4; z++)
    if (z * 64 + lane < a.D) ((uint16_t*)a.out)[out * a.D + z * 64 + lane] = (uint16_t)pack2<DT>(o[z] * rl, 0.0f);
  if (a.lse && lane == 0) a.lse[out] = row_lse(m, l);
}

// Row i of (b, h) from n parts, a quarter of them a wave.
template <typename DT, int TILE>
__device__ __forceinline__ void join_one(const AttnArgs& a, JoinShared& s, int b, int h, int i, int n) {
  const int r = i % a.QB, part = a.QB * a.D;
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
  const int j0 = n * wave / 4, j1 = n * (wave + 1) / 4;
  float m = NEG;
  for (int j = j0 + lane; j < j1; j += 64) m = fmaxf(m, a.part_ml[2ll * (s.part[j] * a.QB + r)]);
  m = wave_maxf(m);
  float l = 0.0f, o[4] = {0, 0, 0, 0};
  for (int c = j0; c < j1; c += 64) {
    float f = 0.0f;
    if (c + lane < j1) {
      const long long p = s.part[c + lane] * a.QB + r;
      const float pm = a.part_ml[2 * p];
      f = pm == NEG ? 0.0f : exp2_hw(pm - m);
      l += f * a.part_ml[2 * p + 1];
    }
    const int cn = j1 - c < 64 ? j1 - c : 64;
    for (int j = 0; j < cn; j += 8) {
      float x[8][4];
#pragma unroll
      for (int y = 0; y < 8; y++) {  // (past the last part: the last one's, not used)
        const long long at = (long long)s.part[j + y < cn ? c + j + y : c + cn - 1] * part;
#pragma unroll
        for (int z = 0; z < 4; z++)
          x[y][z] = z * 64 + lane < a.D ? a.part_o[at + part_at<TILE>(a.D, r, z * 64 + lane)] : 0.0f;
      }
#pragma unroll
      for (int y = 0; y < 8; y++) {
        if (j + y >= cn) break;
        const float fy = readlane_f32(f, j + y);
#pragma unroll
        for (int z = 0; z < 4; z++) o[z] += fy * x[y][z];
      }
    }
  }
  l = wave_sumf(l);
  s.ml[wave][0] = m;
  s.ml[wave][1] = l;
#pragma unroll
  for (int z = 0; z < 4; z++) s.o[wave][z * 64 + lane] = o[z];
  __syncthreads();
  if (wave > 0) return;
  float top = NEG;
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, s.ml[w][0]);
  l = 0.0f;
#pragma unroll
  for (int z = 0; z < 4; z++) o[z] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float f = s.ml[w][0] == NEG ? 0.0f : exp2_hw(s.ml[w][0] - top);
    l += f * s.ml[w][1];
#pragma unroll
    for (int z = 0; z < 4; z++) o[z] += f * s.o[w][z * 64 + lane];
  }
  write_row<DT>(a, b, h, i, o, top, l);
}

template <typename DT, int TILE, int R>
__global__ __launch_bounds__(JOIN_NT) void join_kernel(AttnArgs a, int groups) {
  TGS_STATIC_SMEM(JoinShared, s);
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
  const int g = blockIdx.x % groups, bh = blockIdx.x / groups, h = bh % a.Hkv, b = bh / a.Hkv;
  int before, all;
  tiles_before<TILE>(a, b, before, all);
  const int nt = cache_tiles<TILE>(a, b) + (a.T + TILE - 1) / TILE;
  const long long U = (long long)all * a.Hkv, s0 = (long long)before * a.Hkv + (long long)h * (nt + extra<TILE>()), s1 = s0 + nt;
  const int N = a.nwg;
  const int w0 = (int)(((s0 + 1) * N - 1) / U), w1 = (int)((s1 * N - 1) / U);
  if (w0 == w1) return;
  const int i0 = g * R;  // (R divides QB: the rows lie in one row group)
  const int qb = i0 / a.QB, r0 = i0 - qb * a.QB;
  if (wave == 0) {
    // a worker's second part is the one that starts past its share's first
    // tile; a worker whose share is empty has none
    int n = 0;
    for (int w = w0 + lane; w - lane <= w1; w += 64) {
      long long from = 0;
      bool has = w <= w1;
      if (has) {
        from = share_start(U, N, w);
        has = from != share_start(U, N, w + 1);
      }
      const u64 m = __ballot(has);
      if (has) s.part[n + lanes_below(m)] = (qb * N + w) * 2 + (from < s0);
      n += __popcll(m);
    }
    if (lane == 0) s.n = n;
  }
  __syncthreads();
  const int n = s.n;
  if constexpr (R == 1) {
    join_one<DT, TILE>(a, s, b, h, i0, n);
    return;
  }
  // A lane takes one row and, of the row's D / 4 fours, every sixteenth.
  const int i = i0 + (lane & 15), r = r0 + (lane & 15), sub = wave * 4 + (lane >> 4);
  const long long part = (long long)a.QB * a.D;
  float m = NEG;
  for (int j = 0; j < n; j++) m = fmaxf(m, a.part_ml[2ll * (s.part[j] * a.QB + r)]);
  float l = 0.0f;
  f32x4 o[4] = {};
  for (int j = 0; j < n; j += 2) {
    f32x4 x[2][4];
    float f[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int p = s.part[j + k < n ? j + k : j];  // (past the last part: not used)
      const float pm = a.part_ml[2ll * (p * a.QB + r)], pl = a.part_ml[2ll * (p * a.QB + r) + 1];
#pragma unroll
      for (int z = 0; z < 4; z++)
        if ((sub + 16 * z) * 4 < a.D) x[k][z] = *(const f32x4*)(a.part_o + p * part + part_at<TILE>(a.D, r, (sub + 16 * z) * 4));
      f[k] = j + k >= n || pm == NEG ? 0.0f : exp2_hw(pm - m);
      if (j + k < n) l += pm == NEG ? pl : f[k] * pl;  // (a part without weights has the sum 0, or NaN)
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      if (j + k >= n) break;
#pragma unroll
      for (int z = 0; z < 4; z++)
        if ((sub + 16 * z) * 4 < a.D) o[z] += x[k][z] * f[k];
    }
  }
  if (i >= a.M) return;
  const int t = i / a.G;
  const long long out = ((long long)b * a.T + t) * a.Hq + h * a.G + (i - t * a.G);
  const float rl = 1.0f / l;
#pragma unroll
  for (int z = 0; z < 4; z++)
    if ((sub + 16 * z) * 4 < a.D) store4<DT>((uint16_t*)a.out + out * a.D + (sub + 16 * z) * 4, o[z] * rl);
  if (a.lse && sub == 0) a.lse[out] = row_lse(m, l);
}

// Few rows: one a workgroup, so that their parts are read by many.  The whole
// call, one row a workgroup against 16, 8 key heads of 128 (us): one sequence of
// 131,000 tokens and 160 rows 103 : 135; of 2,000 to 4,000 tokens 8 with 1,024
// rows 26.6 : 29.7, 16 with 2,048 50.3 : 49.5, 16 with 4,096 59.5 : 52.8.  The wide
// kernel's rows, which lie apart in fewer parts, gain from 16 earlier (one
// sequence of 30,000, 1,280 rows 65.7 : 54.6), which this rule leaves.
template <typename DT, int TILE>
hipError_t launch_join(const AttnArgs& a, hipStream_t st) {
  if ((long long)a.B * a.Hkv * a.M <= 2048)
    hipLaunchKernelGGL((join_kernel<DT, TILE, 1>), dim3(a.B * a.Hkv * a.M), dim3(JOIN_NT), 0, st, a, a.M);
  else {
    const int groups = (a.M + 15) / 16;
    hipLaunchKernelGGL((join_kernel<DT, TILE, 16>), dim3(a.B * a.Hkv * groups), dim3(JOIN_NT), 0, st, a, groups);
  }
  return hipGetLastError();
}

}  // namespace attn

hipError_t launch_attn_narrow(const AttnArgs& a, int dtype, hipStream_t st);
hipError_t launch_attn_wide(const AttnArgs& a, int dtype, hipStream_t st);
hipError_t set_attn_narrow_lds();

}  // namespace tgs
