// tgs_attn_narrow.h -- tree attention where a key head has at most 32 query
// rows: the cache is read once and the reading bounds it.
//
// Each wave owns whole tiles, 32 tokens of a 16-bit cache or 64 of an 8-bit one
// (E8), and loads their keys and values from the cache straight into registers;
// nothing is shared while tiles are read, so no wave waits for another.  The next
// tile's keys are requested as soon as this tile's are used, and so the values:
// with eight waves a CU has about 100 KB on the way.  The waves' states join
// through LDS at the end of a (sequence, key head).
//
// 16-bit numbers are the matrix units' operands as they lie in the cache.  8-bit
// ones become operands by one conversion of two numbers, which takes the block's
// scale along, when they are used: the lane's sixteen tokens are one block of
// values, and the rows that it brings to the first product are one block of keys.
//
// 16-bit, D = 128, 8 key heads, whole calls: one sequence of 131,000 tokens 94 us
// (537 MB, 5.7 TB/s; a plain read reaches 6.2); 32 sequences of 100 to 4096 tokens 64 us
// (280 MB, 4.4 TB/s), where a worker starts and ends about 1.5 of the (sequence, key
// head) pairs.  8-bit: the one sequence 58 us (269 MB, 4.6 TB/s), the 32 46 us
// (143 MB, 3.1 TB/s; 39 where three such caches take turns, whose keys stay in the
// memory-side cache).  What is not reading is about 15 us a call, as with 16 bits: the first requests' chain
// (length, entry, tile), the joining of waves, and 6 to 7 us of the parts' launch.
// Requesting the drafted rows before the last tiles are done costs more registers
// than there are (spills: 51 us for the 32), wave priorities change nothing.
#pragma once

#include <type_traits>

#include "tgs_attn.h"

namespace tgs {
namespace attn {

constexpr int NARROW_WAVES = 4;

template <typename DT, int D, int QT, int NW, bool E8>
struct Narrow {
  typedef std::conditional_t<E8, Narrow8, Narrow16> GEO;
  static constexpr int KK = D / 32, DT16 = D / 16;
  static constexpr int ROWS = 16 * QT;
  static constexpr int XB = GEO::TILE / 16;  // products of 16 tokens in a tile
  static constexpr int PER = GEO::TILE / 4;  // tokens of a lane in it, consecutive ones
  // What is read once takes no place in the caches: values, and keys of rows of at least
  // 256 bytes (a shorter row's lines are asked for again by the requests that follow).
  // Caches of 10 and more calls in turn, all plain / values / both (us): 32 sequences of
  // 100 to 4096 tokens, D = 128, 8 bits 46.8 / 45.7 / 47.6, 16 bits 70.7 / 66.2 / 63.8;
  // 131,000 tokens 62.0 / 57.9 / 61.8, 103 / 93.4 / 94.1; 64 sequences of 3000 to 9000,
  // 16 rows of 256, 89.5 / 82.5 / 81.2, 165 / 161 / 139; of 96 43.3 / 40.9 / 41.9,
  // 75.9 / 72.0 / 75.5.
  static constexpr bool ROWS_NT = D * (E8 ? 1 : 2) >= 256;
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
    const int kb = i * GEO::TILE + (col >> 2) * PER, vb = i * GEO::TILE + grp * PER;
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

  // First of the lane's eight dimensions in step kk of the first product.  An 8-bit
  // row's vectors of 16 bytes hold those of two steps; 96 dimensions end with half a one.
  __device__ __forceinline__ int dim_of(int kk) const {
    if constexpr (!E8) return kk * 32 + grp * 8;
    return kk < D / 64 * 2 ? (kk >> 1) * 64 + grp * 16 + (kk & 1) * 8 : (kk >> 1) * 64 + grp * 8;
  }

  // Operands of a cache tile as they lie in the cache.  Product row r = 4 g + j of
  // product x is token PER g + 4 x + j; the lane's values are those of its PER tokens.
  struct Keys16 {
    Vec k[XB][KK];
    __device__ __forceinline__ Vec operand(int x, int kk) const { return k[x][kk]; }
  };
  struct Keys8 {
    Vec k[XB][(KK + 1) / 2];
    uint32_t scale;  // (of the block that the lane's row lies in in every product)
    __device__ __forceinline__ Vec operand(int x, int kk) const {
      const Vec& w = k[x][kk >> 1];
      return kk & 1 ? decode8<DT>(w[2], w[3], e8::scale_of(scale)) : decode8<DT>(w[0], w[1], e8::scale_of(scale));
    }
  };
  struct Values16 {
    Vec v[DT16];
    __device__ __forceinline__ Vec operand(int d, int) const { return v[d]; }
  };
  struct Values8 {
    Vec v[DT16];
    uint32_t scale;
    __device__ __forceinline__ Vec operand(int d, int y) const {
      return y ? decode8<DT>(v[d][2], v[d][3], e8::scale_of(scale)) : decode8<DT>(v[d][0], v[d][1], e8::scale_of(scale));
    }
  };
  typedef std::conditional_t<E8, Keys8, Keys16> Keys;
  typedef std::conditional_t<E8, Values8, Values16> Values;

  // The scale of position p's block, of keys (0) or values (1).
  __device__ __forceinline__ uint32_t scale_at(long long page, int p, int which) const {
    return a.scales[page * a.s_page + ((((long long)h << a.page_shift) + p) >> 4) * 2 + which];
  }

  __device__ __forceinline__ void load_keys(int i, int entry, Keys& k) {
    const long long page = page_of(entry), at = page * a.k_page + (((long long)h * D) << a.page_shift);
    const int kb = i * GEO::TILE + (col >> 2) * PER, last = len - 1, in = (1 << a.page_shift) - 1;
    if constexpr (E8) k.scale = scale_at(page, (kb < last ? kb : last) & in, 0);
#pragma unroll
    for (int x = 0; x < XB; x++) {
      int p = kb + (col & 3) + 4 * x;
      p = (p < last ? p : last) & in;
      if constexpr (E8) {
        const uint8_t* base = (const uint8_t*)a.k + at + p * D;
#pragma unroll
        for (int c = 0; c < D / 64; c++) k.k[x][c] = load_once<ROWS_NT>(base + c * 64 + grp * 16);
        if constexpr (D % 64 != 0) {
          const uint2 w = *(const uint2*)(base + D / 64 * 64 + grp * 8);
          k.k[x][D / 64] = vec16(w.x, w.y, 0, 0);
        }
      } else {
        const uint16_t* base = (const uint16_t*)a.k + at + grp * 8;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) k.k[x][kk] = load_once<ROWS_NT>(base + p * D + kk * 32);
      }
    }
  }
  __device__ __forceinline__ void load_values(int i, int entry, Values& v) {
    const int blk = i * GEO::TILE + grp * PER, last = (len - 1) & ~(PER - 1);
    const int p = (blk < last ? blk : last) & ((1 << a.page_shift) - 1);
    const long long page = page_of(entry);
    const long long at = page * a.v_page + (((long long)h * D) << a.page_shift) + (long long)p * D + col * PER;
    if constexpr (E8) {
      v.scale = scale_at(page, p, 1);
#pragma unroll
      for (int d = 0; d < DT16; d++) v.v[d] = load_once<true>((const uint8_t*)a.v + at + d * 256);
    } else {
#pragma unroll
      for (int d = 0; d < DT16; d++) v.v[d] = load_once<true>((const uint16_t*)a.v + at + d * 128);
    }
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
  struct TreeKeys {
    Vec k[2][KK];
    __device__ __forceinline__ Vec operand(int x, int kk) const { return k[x][kk]; }
  };
  __device__ __forceinline__ void load_tree_keys(TreeKeys& k) const {
    const uint16_t* kb = (const uint16_t*)a.k_new + b * a.kn_b + h * a.kn_h;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      int p = (col >> 2) * 8 + (col & 3) + 4 * t;
      p = p < a.T ? p : a.T - 1;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) k.k[t][kk] = load16(kb + p * a.kn_t + dim_of(kk));
    }
  }
  __device__ __forceinline__ void turn_tree(Vec* turn, Vec (&x)[GO][8], Values16& v) const {
#pragma unroll
    for (int n = 0; n < GO; n++) {
      transpose8(x[n]);
      if (n * 16 + col < D / 8)
#pragma unroll
        for (int j = 0; j < 8; j++) turn[grp * D + (n * 16 + col) * 8 + j] = x[n][j];
    }
    wave_lds_sync();
#pragma unroll
    for (int d = 0; d < DT16; d++) v.v[d] = turn[grp * D + d * 16 + col];
  }

  // N products of 16 tokens.
  template <int N, class K>
  __device__ __forceinline__ void scores(const K& k, const Vec (&q)[QT][KK], f32x4 (&sc)[QT][N]) const {
    if constexpr (!E8) {
#pragma unroll
      for (int t = 0; t < QT; t++)
#pragma unroll
        for (int x = 0; x < N; x++) {
          sc[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < KK; kk++) sc[t][x] = mfma16<DT>(k.operand(x, kk), q[t][kk], sc[t][x]);
        }
    } else {  // (an operand is decoded once for all rows)
#pragma unroll
      for (int x = 0; x < N; x++) {
#pragma unroll
        for (int t = 0; t < QT; t++) sc[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
          const Vec y = k.operand(x, kk);
#pragma unroll
          for (int t = 0; t < QT; t++) sc[t][x] = mfma16<DT>(y, q[t][kk], sc[t][x]);
        }
      }
    }
  }

  // Of the lane's 4 N tokens, eight to an operand of the second product.
  template <int N>
  __device__ __forceinline__ void weights(const f32x4 (&sc)[QT][N], State& s, Vec (&p)[QT][N / 2]) const {
#pragma unroll
    for (int t = 0; t < QT; t++) {
      float top = sc[t][0][0];
#pragma unroll
      for (int j = 1; j < 4 * N; j++) top = fmaxf(top, sc[t][j >> 2][j & 3]);
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
#pragma unroll
      for (int y = 0; y < N / 2; y++) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          w[j] = exp2_hw(__builtin_fmaf(sc[t][2 * y + (j >> 2)][j & 3], a.scale_log2, -base));
          s.l[t] += w[j];
        }
        p[t][y] = vec16(to16<DT>(w[0], w[1]), to16<DT>(w[2], w[3]), to16<DT>(w[4], w[5]), to16<DT>(w[6], w[7]));
#pragma unroll
        for (int j = 0; j < 4; j++) s.r[t] = add2<DT>(p[t][y][j], s.r[t]);
      }
    }
  }

  template <int N, class V>
  __device__ __forceinline__ void add(const V& v, const Vec (&p)[QT][N], State& s) const {
#pragma unroll
    for (int d = 0; d < DT16; d++)
#pragma unroll
      for (int y = 0; y < N; y++) {
        const Vec x = v.operand(d, y);
#pragma unroll
        for (int t = 0; t < QT; t++) s.o[t][d] = mfma16<DT>(x, p[t][y], s.o[t][d]);
      }
  }

  // Takes what is not finite out of the drafted tile's values, and adds it node
  // by node to the rows that see the node.
  __device__ __forceinline__ void add_odd(Values16& v, const Vec (&p)[QT][1], u64 anc, State& s) const {
    u64 sees[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) sees[t] = lane_bits(anc, t * 16 + col < a.M ? (t * 16 + col) / a.G : 0);
    for (int j = 0; j < a.T; j++) {
      const Vec one = only(grp == j >> 3 ? j & 7 : 8);
#pragma unroll
      for (int d = 0; d < DT16; d++) {
        const Vec x = odd_of<DT>(v.v[d]) & one;
        if (__ballot((x[0] | x[1] | x[2] | x[3]) != 0) == 0) continue;
#pragma unroll
        for (int t = 0; t < QT; t++) {
          const f32x4 y = mfma16<DT>(x, p[t][0], f32x4{0, 0, 0, 0});
#pragma unroll
          for (int z = 0; z < 4; z++) s.o[t][d][z] += sees[t] >> j & 1 ? y[z] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT16; d++) v.v[d] ^= odd_of<DT>(v.v[d]);
  }

  // Tiles [t0, t1) of (b, h), a sequence of the length `given`; full: they are all of
  // it.  part: the workspace's rows otherwise.
  __device__ __forceinline__ void segment(Shared& s, int given, int t0, int t1, bool full, long long part) {
    len = clamp_len(a, given);
    nc = (len + GEO::TILE - 1) / GEO::TILE;
    table = a.tables + (long long)b * a.P;
    bad = given == FAILED;
    const int par = t1 > nc ? parent_of(a, b) : -1;
    Vec q[QT][KK];
#pragma unroll
    for (int t = 0; t < QT; t++) {
      const int i = t * 16 + col;
      const int node = i < a.M ? i / a.G : 0, hg = i < a.M ? i - node * a.G : 0;
      const uint16_t* p = (const uint16_t*)a.q + b * a.q_b + node * a.q_t + (long long)(h * a.G + hg) * a.q_h;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) q[t][kk] = load16(p + dim_of(kk));
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
    int i = t0 + wave;
    const int tc = t1 < nc ? t1 : nc;  // the end of the cache's tiles
    if (i < tc) {
      Keys k;
      Values v;
      Vec p[QT][XB / 2];
      f32x4 sc[QT][XB];
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
      const int left = len - i * GEO::TILE - grp * PER;  // of the lane's tokens
      if ((i + 1) * GEO::TILE > len) {
        const uint32_t bits = left >= PER ? (1u << PER) - 1 : left <= 0 ? 0u : (1u << left) - 1;
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int j = 0; j < PER; j++) sc[t][j >> 2][j & 3] = seen(sc[t][j >> 2][j & 3], bits, j);
        // what lies past the end is not 0 (it may be anything, NaN too)
        const Vec keep = first_of<128 / PER>(left);
#pragma unroll
        for (int d = 0; d < DT16; d++) v.v[d] &= keep;
      }
      i += NW;
      weights(sc, st, p);
      add(v, p, st);
    }
    if (i < t1) {
      TreeKeys k;
      Values16 v;
      Vec p[QT][1];
      f32x4 sc[QT][2];
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

// SPLIT: workers with their shares of all tiles; else one workgroup per (sequence, key
// head).  (With both in one kernel a single short sequence takes 5.2 us, so 4.9.)
template <typename DT, int D, int QT, int NW, bool E8, bool SPLIT>
__global__ __launch_bounds__(NW * 64, D == 256 ? 1 : 2) void narrow_kernel(AttnArgs a) {
  typedef Narrow<DT, D, QT, NW, E8> K;
  typedef typename K::GEO GEO;
  TGS_DYN_SMEM(dyn);
  typename K::Shared& s = *(typename K::Shared*)dyn;
  K n(a);
  const int tree = (a.T + GEO::TILE - 1) / GEO::TILE;
  if constexpr (!SPLIT) {
    n.b = blockIdx.x / a.Hkv;
    n.h = blockIdx.x % a.Hkv;
    const int given = uniform(a.lens[n.b]);
    n.segment(s, given, 0, cache_tiles<GEO>(a, given) + tree, true, 0);
    return;
  }
  Place p = find_place<GEO>(a, blockIdx.x);
  for (long long u = p.u0; u < p.u1;) {
    const int end = p.nt - p.at < p.u1 - u ? p.nt : p.at + (int)(p.u1 - u);
    const int real = p.nt - GEO::EXTRA;
    if (p.at < real) {
      n.b = p.b;
      n.h = p.h;
      n.segment(s, p.given, p.at, end < real ? end : real, p.at == 0 && end >= real, ((long long)blockIdx.x * 2 + (u != p.u0)) * a.QB);
    }
    u += end - p.at;
    p.at = 0;
    if (++p.h == a.Hkv) {
      p.h = 0;
      if (++p.b < a.B) {
        p.given = uniform(a.lens[p.b]);
        p.nt = cache_tiles<GEO>(a, p.given) + tree + GEO::EXTRA;
      }
    }
  }
}

template <typename DT, int D, int QT, bool E8>
hipError_t narrow_run(const AttnArgs& a, hipStream_t st) {
  constexpr int NW = NARROW_WAVES;
  typedef Narrow<DT, D, QT, NW, E8> K;
  if (a.nwg)
    hipLaunchKernelGGL((narrow_kernel<DT, D, QT, NW, E8, true>), dim3(a.nwg), dim3(NW * 64), sizeof(typename K::Shared), st, a);
  else
    hipLaunchKernelGGL((narrow_kernel<DT, D, QT, NW, E8, false>), dim3(a.B * a.Hkv), dim3(NW * 64), sizeof(typename K::Shared), st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nwg == 0) return e;
  return launch_join<DT, typename K::GEO>(a, st);
}
template <typename DT, int D, int QT, bool E8>
hipError_t narrow_lds() {
  constexpr int NW = NARROW_WAVES;
  const int lds = (int)sizeof(typename Narrow<DT, D, QT, NW, E8>::Shared);
  const hipError_t e = hipFuncSetAttribute((const void*)narrow_kernel<DT, D, QT, NW, E8, false>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  return hipFuncSetAttribute((const void*)narrow_kernel<DT, D, QT, NW, E8, true>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename DT, bool E8>
hipError_t narrow_type(const AttnArgs& a, int qt, hipStream_t st) {
  switch (a.D * 2 + qt - 1) {
    case 128: return narrow_run<DT, 64, 1, E8>(a, st);
    case 129: return narrow_run<DT, 64, 2, E8>(a, st);
    case 192: return narrow_run<DT, 96, 1, E8>(a, st);
    case 193: return narrow_run<DT, 96, 2, E8>(a, st);
    case 256: return narrow_run<DT, 128, 1, E8>(a, st);
    case 257: return narrow_run<DT, 128, 2, E8>(a, st);
    case 512: return narrow_run<DT, 256, 1, E8>(a, st);
    case 513: return narrow_run<DT, 256, 2, E8>(a, st);
  }
  return hipErrorInvalidValue;
}
template <typename DT, bool E8>
hipError_t narrow_lds_type() {
  hipError_t e = hipSuccess;
  auto take = [&](hipError_t x) { e = x != hipSuccess ? x : e; };
  take(narrow_lds<DT, 64, 1, E8>());
  take(narrow_lds<DT, 64, 2, E8>());
  take(narrow_lds<DT, 96, 1, E8>());
  take(narrow_lds<DT, 96, 2, E8>());
  take(narrow_lds<DT, 128, 1, E8>());
  take(narrow_lds<DT, 128, 2, E8>());
  take(narrow_lds<DT, 256, 1, E8>());
  take(narrow_lds<DT, 256, 2, E8>());
  return e;
}

}  // namespace attn
}  // namespace tgs
