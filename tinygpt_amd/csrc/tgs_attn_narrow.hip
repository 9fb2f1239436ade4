// tgs_attn_narrow.hip -- tree attention where a key head has at most 32 query
// rows: the cache is read once and the reading bounds it.
//
// Each wave owns whole tiles of 32 tokens and loads their keys and values from
// the cache straight into the matrix units' operand registers; nothing is
// shared while tiles are read, so no wave waits for another.  The next tile's
// keys are requested as soon as this tile's are used, and so the values: with
// eight waves a CU has about 100 KB on the way.  The waves' states join
// through LDS at the end of a (sequence, key head).
//
// 16-bit, D = 128, 8 key heads: one sequence of 131,000 tokens 96 us (537 MB,
// 5.6 TB/s; a plain read reaches 6.2); 32 sequences of 100 to 4096 tokens 62 us
// (280 MB, 4.5 TB/s), where a worker starts and ends about 1.5 of the
// (sequence, key head) pairs.
#include "tgs_attn.h"

namespace tgs {
namespace attn {

constexpr int NARROW_WAVES = 4;

template <typename DT, int D, int QT, int NW>
struct Narrow {
  static constexpr int KK = D / 32, DT16 = D / 16;
  static constexpr int ROWS = 16 * QT;
  struct Shared {
    f32x4 o[NW][DT16 * QT][64];
    float ml[NW][ROWS][2];
    float tot[ROWS][2];
  };

  const AttnArgs& a;
  const int lane, wave, col, grp;
  // the tiles in progress
  int b, h, len, nc;
  const int* table;
  bool bad;

  __device__ __forceinline__ Narrow(const AttnArgs& a_)
      : a(a_), lane(lane_id()), wave((int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), col(lane & 15), grp(lane >> 4), b(0), h(0), len(0), nc(0),
        table(nullptr), bad(false) {}

  struct State {
    f32x4 o[QT][DT16];
    float m[QT], l[QT], r[QT];  // (l, r: of the lane's tokens alone; r: of the rounded weights)
  };

  // Page entries of cache tile i for the lane's key block and value block.
  __device__ __forceinline__ int2 entries(int i) const {
    const int kb = i * NTILE + (col >> 2) * 8, vb = i * NTILE + grp * 8;
    const int last = len - 1;
    return make_int2(table[(kb < last ? kb : last) >> a.page_shift], table[(vb < last ? vb : last) >> a.page_shift]);
  }
  __device__ __forceinline__ long long page_of(int e) {
    if ((unsigned)e >= (unsigned)a.n_pages) {
      bad = true;  // (its sequence's rows become NaN)
      return 0;
    }
    return e;
  }

  // Keys of cache tile i: product row r = 4 g + j of half t is token 8 g + 4 t + j.
  __device__ __forceinline__ void load_keys(int i, int entry, Vec (&k)[2][KK]) {
    const uint16_t* base = (const uint16_t*)a.k + page_of(entry) * a.k_page + (((long long)h * D) << a.page_shift) + grp * 8;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      int p = i * NTILE + (col >> 2) * 8 + (col & 3) + 4 * t;
      p = (p < len ? p : len - 1) & ((1 << a.page_shift) - 1);
#pragma unroll
      for (int kk = 0; kk < KK; kk++) k[t][kk] = *(const Vec*)(base + p * D + kk * 32);
    }
  }
  __device__ __forceinline__ void load_values(int i, int entry, Vec (&v)[DT16]) {
    const int blk = i * NTILE + grp * 8, last = (len - 1) & ~7;
    const int p = (blk < last ? blk : last) & ((1 << a.page_shift) - 1);
    const uint16_t* base = (const uint16_t*)a.v + page_of(entry) * a.v_page + (((long long)h * D) << a.page_shift) +
                           (long long)p * D + col * 8;
#pragma unroll
    for (int d = 0; d < DT16; d++) v[d] = *(const Vec*)(base + d * 128);
  }

  // The same of the drafted nodes (T <= NTILE: one tile).  Their values come
  // row by row, 16 chunks a go, and turn into blocks of eight tokens in
  // registers and through `turn`, the wave's own 4 D vectors of LDS.
  static constexpr int GO = (D / 8 + 15) / 16;
  __device__ __forceinline__ void load_tree_values(Vec (&x)[GO][8]) const {
    const uint16_t* vb = (const uint16_t*)a.v_new + b * a.vn_b + h * a.vn_h;
#pragma unroll
    for (int n = 0; n < GO; n++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int c = n * 16 + col, p = grp * 8 + j;
        x[n][j] = vec16(0, 0, 0, 0);
        if (p < a.T && c < D / 8) x[n][j] = load16(vb + p * a.vn_t + c * 8);
      }
  }
  __device__ __forceinline__ void load_tree_keys(Vec (&k)[2][KK]) const {
    const uint16_t* kb = (const uint16_t*)a.k_new + b * a.kn_b + h * a.kn_h + grp * 8;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      int p = (col >> 2) * 8 + (col & 3) + 4 * t;
      p = p < a.T ? p : a.T - 1;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) k[t][kk] = load16(kb + p * a.kn_t + kk * 32);
    }
  }
  __device__ __forceinline__ void turn_tree(Vec* turn, Vec (&x)[GO][8], Vec (&v)[DT16]) const {
#pragma unroll
    for (int n = 0; n < GO; n++) {
      transpose8(x[n]);
      if (n * 16 + col < D / 8)
#pragma unroll
        for (int j = 0; j < 8; j++) turn[grp * D + (n * 16 + col) * 8 + j] = x[n][j];
    }
    wave_lds_sync();
#pragma unroll
    for (int d = 0; d < DT16; d++) v[d] = turn[grp * D + d * 16 + col];
  }

  __device__ __forceinline__ void scores(const Vec (&k)[2][KK], const Vec (&q)[QT][KK], f32x4 (&sc)[QT][2]) const {
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        sc[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; kk++) sc[t][x] = mfma16<DT>(k[x][kk], q[t][kk], sc[t][x]);
      }
  }

  __device__ __forceinline__ void weights(const f32x4 (&sc)[QT][2], State& s, Vec (&p)[QT]) const {
#pragma unroll
    for (int t = 0; t < QT; t++) {
      float top = sc[t][0][0];
#pragma unroll
      for (int j = 1; j < 8; j++) top = fmaxf(top, sc[t][j >> 2][j & 3]);
      top = top * a.scale_log2 - lift<DT>();
      if (__ballot(top > s.m[t] + SLACK)) {
        top = fmaxf(top, xor_lane<16>(top));
        top = fmaxf(top, xor_lane<32>(top));
        const float now = fmaxf(s.m[t], top);
        const float f = s.m[t] == NEG ? 0.0f : exp2_hw(s.m[t] - now);
        s.m[t] = now;
        s.l[t] *= f;
        s.r[t] *= f;
#pragma unroll
        for (int d = 0; d < DT16; d++) s.o[t][d] *= f;
      }
      const float base = s.m[t] == NEG ? 0.0f : s.m[t];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        w[j] = exp2_hw(__builtin_fmaf(sc[t][j >> 2][j & 3], a.scale_log2, -base));
        s.l[t] += w[j];
      }
      p[t] = vec16(pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7]));
#pragma unroll
      for (int j = 0; j < 4; j++) s.r[t] = add2<DT>(p[t][j], s.r[t]);
    }
  }

  __device__ __forceinline__ void add(const Vec (&v)[DT16], const Vec (&p)[QT], State& s) const {
#pragma unroll
    for (int d = 0; d < DT16; d++)
#pragma unroll
      for (int t = 0; t < QT; t++) s.o[t][d] = mfma16<DT>(v[d], p[t], s.o[t][d]);
  }

  // Takes what is not finite out of the drafted tile's values, and adds it node
  // by node to the rows that see the node.
  __device__ __forceinline__ void add_odd(Vec (&v)[DT16], const Vec (&p)[QT], u64 anc, State& s) const {
    u64 sees[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) sees[t] = lane_bits(anc, t * 16 + col < a.M ? (t * 16 + col) / a.G : 0);
    for (int j = 0; j < a.T; j++) {
      const Vec one = only(grp == j >> 3 ? j & 7 : 8);
#pragma unroll
      for (int d = 0; d < DT16; d++) {
        const Vec x = odd_of<DT>(v[d]) & one;
        if (__ballot((x[0] | x[1] | x[2] | x[3]) != 0) == 0) continue;
#pragma unroll
        for (int t = 0; t < QT; t++) {
          const f32x4 y = mfma16<DT>(x, p[t], f32x4{0, 0, 0, 0});
#pragma unroll
          for (int z = 0; z < 4; z++) s.o[t][d][z] += sees[t] >> j & 1 ? y[z] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT16; d++) v[d] ^= odd_of<DT>(v[d]);
  }

  // Tiles [t0, t1) of (b, h); full: they are all of it.  part: the workspace's rows otherwise.
  __device__ __forceinline__ void segment(Shared& s, int t0, int t1, bool full, long long part) {
    const int given = uniform(a.lens[b]);
    len = clamp_len(a, given);
    nc = (len + NTILE - 1) / NTILE;
    table = a.tables + (long long)b * a.P;
    bad = given == FAILED;
    const int par = t1 > nc ? parent_of(a, b) : -1;
    Vec q[QT][KK];
#pragma unroll
    for (int t = 0; t < QT; t++) {
      const int i = t * 16 + col;
      const int node = i < a.M ? i / a.G : 0, hg = i < a.M ? i - node * a.G : 0;
      const uint16_t* p = (const uint16_t*)a.q + b * a.q_b + node * a.q_t + (long long)(h * a.G + hg) * a.q_h + grp * 8;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) q[t][kk] = load16(p + kk * 32);
    }
    State st;
#pragma unroll
    for (int t = 0; t < QT; t++) {
      st.m[t] = NEG;
      st.l[t] = 0.0f;
      st.r[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT16; d++) st.o[t][d] = f32x4{0, 0, 0, 0};
    }
    Vec k[2][KK], v[DT16], p[QT];
    f32x4 sc[QT][2];
    int i = t0 + wave;
    const int tc = t1 < nc ? t1 : nc;  // the end of the cache's tiles
    if (i < tc) {
      // Requests complete in order: a tile's keys, the entries of the tile
      // after the next, then its values, each waited for with what follows it
      // still on the way.  Only the last tile can end inside.
      int2 e = entries(i);
      load_keys(i, e.x, k);
      sched_fence();
      int2 next = entries(i + NW < tc ? i + NW : i);
      sched_fence();
      load_values(i, e.y, v);
      sched_fence();
      for (; i + NW < tc; i += NW) {
        scores(k, q, sc);
        e = next;
        load_keys(i + NW, e.x, k);
        sched_fence();
        next = entries(i + 2 * NW < tc ? i + 2 * NW : i);
        sched_fence();
        weights(sc, st, p);
        add(v, p, st);
        load_values(i + NW, e.y, v);
        sched_fence();
      }
      scores(k, q, sc);
      const int left = len - i * NTILE - grp * 8;  // of the lane's eight tokens
      if ((i + 1) * NTILE > len) {
        const uint32_t bits = left >= 8 ? 0xFFu : left <= 0 ? 0u : (1u << left) - 1;
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int j = 0; j < 8; j++) sc[t][j >> 2][j & 3] = seen(sc[t][j >> 2][j & 3], bits, j);
        // what lies past the end is not 0 (it may be anything, NaN too)
        const Vec keep = first_of(left);
#pragma unroll
        for (int d = 0; d < DT16; d++) v[d] &= keep;
      }
      i += NW;
      weights(sc, st, p);
      add(v, p, st);
    }
    if (i < t1) {
      Vec x[GO][8];
      load_tree_values(x);
      load_tree_keys(k);
      const u64 anc = ancestors(a, par);  // of node `lane`
      float odd = 0.0f;  // NaN: not all values are finite
      if (a.T > 1) {  // (one node: every row sees it)
#pragma unroll
        for (int n = 0; n < GO; n++)
#pragma unroll
          for (int j = 0; j < 8; j++) odd = finite_or_nan<DT>(x[n][j], odd);
      }
      scores(k, q, sc);
      turn_tree((Vec*)s.o[wave], x, v);
#pragma unroll
      for (int t = 0; t < QT; t++) {
        const int node = t * 16 + col < a.M ? (t * 16 + col) / a.G : 0;
        const u64 sees = lane_bits(anc, node);
        const uint32_t in = (uint32_t)(sees >> (grp * 8));
#pragma unroll
        for (int j = 0; j < 8; j++) sc[t][j >> 2][j & 3] = seen(sc[t][j >> 2][j & 3], in, j);
      }
      weights(sc, st, p);
      if (__ballot(odd != 0.0f)) add_odd(v, p, anc, st);
      add(v, p, st);
    }
    // the waves' states
    const bool any_bad = __ballot(bad) != 0;
#pragma unroll
    for (int t = 0; t < QT; t++) {
      st.l[t] += xor_lane<16>(st.l[t]);
      st.l[t] += xor_lane<32>(st.l[t]);
      st.r[t] += xor_lane<16>(st.r[t]);
      st.r[t] += xor_lane<32>(st.r[t]);
      st.r[t] = st.r[t] > 0.0f ? st.l[t] / st.r[t] : 1.0f;
      if (any_bad) st.l[t] = __builtin_nanf("");
      if (grp == 0) {
        s.ml[wave][t * 16 + col][0] = st.m[t];
        s.ml[wave][t * 16 + col][1] = st.l[t];
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < QT; t++) {
      float top = NEG, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; w++) top = fmaxf(top, s.ml[w][t * 16 + col][0]);
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float mw = s.ml[w][t * 16 + col][0];
        sum += s.ml[w][t * 16 + col][1] * (mw == NEG ? 1.0f : exp2_hw(mw - top));
      }
      const float f = st.m[t] == NEG ? 0.0f : exp2_hw(st.m[t] - top) * st.r[t];
#pragma unroll
      for (int d = 0; d < DT16; d++) s.o[wave][d * QT + t][lane] = st.o[t][d] * f;
      if (wave == 0 && grp == 0) {
        s.tot[t * 16 + col][0] = top;
        s.tot[t * 16 + col][1] = sum;
      }
    }
    __syncthreads();
    for (int e = wave; e < DT16 * QT; e += NW) {
      f32x4 x = s.o[0][e][lane];
#pragma unroll
      for (int w = 1; w < NW; w++) x += s.o[w][e][lane];
      const int t = e % QT, d = e / QT * 16 + grp * 4, i = t * 16 + col;
      if (i >= a.M) continue;
      if (full) {
        const int node = i / a.G;
        const long long row = ((long long)b * a.T + node) * a.Hq + h * a.G + (i - node * a.G);
        const float r = 1.0f / s.tot[i][1];
        store4<DT>((uint16_t*)a.out + row * D + d, x * r);
        if (a.lse && e < QT && grp == 0) a.lse[row] = row_lse(s.tot[i][0], s.tot[i][1]);
      } else {
        *(f32x4*)(a.part_o + (part + i) * D + d) = x;
        if (e < QT && grp == 0) {
          a.part_ml[(part + i) * 2] = s.tot[i][0];
          a.part_ml[(part + i) * 2 + 1] = s.tot[i][1];
        }
      }
    }
    __syncthreads();
  }
};

template <typename DT, int D, int QT, int NW>
__global__ __launch_bounds__(NW * 64, D == 256 ? 1 : 2) void narrow_kernel(AttnArgs a) {
  typedef Narrow<DT, D, QT, NW> K;
  TGS_DYN_SMEM(dyn);
  typename K::Shared& s = *(typename K::Shared*)dyn;
  K n(a);
  const int tree = (a.T + NTILE - 1) / NTILE;
  if (a.nwg == 0) {
    n.b = blockIdx.x / a.Hkv;
    n.h = blockIdx.x % a.Hkv;
    n.segment(s, 0, cache_tiles<NTILE>(a, n.b) + tree, true, 0);
    return;
  }
  const Place at0 = find_place<NTILE>(a, blockIdx.x);
  const long long u0 = at0.u0, u1 = at0.u1;
  int b = at0.b, h = at0.h, at = at0.at, nt = at0.nt;
  for (long long u = u0; u < u1;) {
    const int end = nt - at < u1 - u ? nt : at + (int)(u1 - u);
    const int real = nt - extra<NTILE>();
    if (at < real) {
      n.b = b;
      n.h = h;
      n.segment(s, at, end < real ? end : real, at == 0 && end >= real, ((long long)blockIdx.x * 2 + (u != u0)) * a.QB);
    }
    u += end - at;
    at = 0;
    if (++h == a.Hkv) {
      h = 0;
      if (++b < a.B) nt = cache_tiles<NTILE>(a, b) + tree + extra<NTILE>();
    }
  }
}

template <typename DT, int D, int QT>
hipError_t narrow_run(const AttnArgs& a, hipStream_t st) {
  constexpr int NW = NARROW_WAVES;
  typedef Narrow<DT, D, QT, NW> K;
  const int grid = a.nwg ? a.nwg : a.B * a.Hkv;
  hipLaunchKernelGGL((narrow_kernel<DT, D, QT, NW>), dim3(grid), dim3(NW * 64), sizeof(typename K::Shared), st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nwg == 0) return e;
  return launch_join<DT, NTILE>(a, st);
}
template <typename DT, int D, int QT>
hipError_t narrow_lds() {
  constexpr int NW = NARROW_WAVES;
  return hipFuncSetAttribute((const void*)narrow_kernel<DT, D, QT, NW>, hipFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sizeof(typename Narrow<DT, D, QT, NW>::Shared));
}

template <typename DT>
hipError_t narrow_type(const AttnArgs& a, int qt, hipStream_t st) {
  switch (a.D * 2 + qt - 1) {
    case 128: return narrow_run<DT, 64, 1>(a, st);
    case 129: return narrow_run<DT, 64, 2>(a, st);
    case 192: return narrow_run<DT, 96, 1>(a, st);
    case 193: return narrow_run<DT, 96, 2>(a, st);
    case 256: return narrow_run<DT, 128, 1>(a, st);
    case 257: return narrow_run<DT, 128, 2>(a, st);
    case 512: return narrow_run<DT, 256, 1>(a, st);
    case 513: return narrow_run<DT, 256, 2>(a, st);
  }
  return hipErrorInvalidValue;
}
template <typename DT>
hipError_t narrow_lds_type() {
  hipError_t e = hipSuccess;
  auto take = [&](hipError_t x) { e = x != hipSuccess ? x : e; };
  take(narrow_lds<DT, 64, 1>());
  take(narrow_lds<DT, 64, 2>());
  take(narrow_lds<DT, 96, 1>());
  take(narrow_lds<DT, 96, 2>());
  take(narrow_lds<DT, 128, 1>());
  take(narrow_lds<DT, 128, 2>());
  take(narrow_lds<DT, 256, 1>());
  take(narrow_lds<DT, 256, 2>());
  return e;
}

}  // namespace attn

hipError_t launch_attn_narrow(const AttnArgs& a, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? attn::narrow_type<attn::BF16>(a, a.QB / 16, st) : attn::narrow_type<attn::F16>(a, a.QB / 16, st);
}
hipError_t set_attn_narrow_lds() {
  const hipError_t e = attn::narrow_lds_type<attn::BF16>(), f = attn::narrow_lds_type<attn::F16>();
  return e != hipSuccess ? e : f;
}

}  // namespace tgs
