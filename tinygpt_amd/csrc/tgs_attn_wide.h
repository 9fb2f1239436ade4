// tgs_attn_wide.h -- tree attention where a key head has more than 32 query
// rows: a tile's keys and values go through LDS, where every wave of the
// workgroup, each with 32 rows of its own, reads them.
//
// Tiles of 64 tokens, two in LDS and one or two more on their way to
// registers, one barrier a tile.  Keys lie in LDS row by row with the 16-byte chunks of a
// row permuted by the row's number, so that the 16 lanes served together take
// 16 different chunks; values lie as in the cache, where a lane's operands
// are neighbours already.  Tiles of an 8-bit cache (E8) become 16-bit numbers on
// their way from registers to LDS, by one conversion of two numbers that takes the
// block's scale along; everything behind is the same.
//
// 16 sequences of 2000 to 6000 tokens, 63 nodes, 4 key heads with 8 query heads
// each, D = 128: 87 us for 66.6 GFLOP, 0.8 PFLOP/s (59 us at a large library
// product's rate).  28 us of it are not in the tile loop.  In the loop a tile's
// LDS reads, products and weights follow each other in both waves of a SIMD;
// 64 rows a wave would halve the reads but need copies between the register
// files and scratch (165 us).  Of an 8-bit cache the same 88 to 94 us: half the bytes
// do not help, as reading does not bound it, and the conversions come on top (matrix
// units are busy 43 % of the waves' time, vector ones 48 %, mostly in turn).
#pragma once

#include <type_traits>

#include "tgs_attn.h"

namespace tgs {
namespace attn {

template <typename DT, int D, int QW, bool E8>
struct Wide {
  static constexpr int NTHR = QW * 64, KK = D / 16, DT32 = D / 32, C = D / 8;
  static constexpr int BT = E8 ? 16 : 8;  // tokens of a block of the cache
  static constexpr int CM = D / BT;       // 16-byte chunks of a cached row (and of BT values each, of a block's values by BT)
  static constexpr int NCH = (WTILE * CM + NTHR - 1) / NTHR;  // chunks a thread moves, of keys and of values
  static constexpr bool EVEN = WTILE * CM % NTHR == 0;
  static constexpr bool MIXED = D % 64 != 0;      // the chunks of a wave may belong to two blocks
  static constexpr int AHEAD = NCH <= 2 ? 2 : 1;  // tiles on their way (a tile takes 8 NCH registers)
  struct Shared {
    Vec k[2][WTILE * C];
    Vec v[2][WTILE * C];
    int odd[QW];  // whether what a wave brings of the drafted tile's values is not all finite
  };

  const AttnArgs& a;
  const int tid, lane, wave, col, half;
  int b, h, qb, len, nc;
  const int* table;
  bool bad;
  int odd;  // whether a drafted tile so far had values that are not finite

  __device__ __forceinline__ Wide(const AttnArgs& a_)
      : a(a_), tid((int)threadIdx.x), lane(lane_id()), wave((int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), col(lane & 31), half(lane >> 5), b(0), h(0), qb(0),
        len(0), nc(0), table(nullptr), bad(false), odd(0) {}

  // Where chunk ch of row tok lies.
  static __device__ __forceinline__ int at_key(int tok, int ch) {
    if constexpr (C % 16 == 0) return tok * C + (ch ^ (tok & 15));
    else if constexpr (C == 8) return tok * C + (ch ^ ((tok >> 1) & 7));
    else {  // 12 chunks: rows 4 apart start at the same banks; turned by 0 .. 3 they differ
      const int x = ch + ((tok >> 2) & 3);
      return tok * C + (x < C ? x : x - C);
    }
  }

  // Pages of the blocks from cache tile i on, one a lane (WTILE / BT a tile); of a
  // block past the end, the last one's.
  __device__ __forceinline__ int entries(int i) const {
    const int blk = i * WTILE + lane * BT, last = len - 1;
    return table[(blk < last ? blk : last) >> a.page_shift];
  }
  static constexpr int HOLDS = 64 / (WTILE / BT);  // tiles whose entries it holds

  // The place of block blk of tile i: its page and its first token there.
  // The chunks of a wave belong to one block (but for rows of 96), so this is
  // scalar arithmetic.
  struct Spot {
    long long page;
    int in;
  };
  __device__ __forceinline__ Spot spot_of(int i, int blk, int entry, int off) const {
    const int last = (len - 1) / BT, x = i * (WTILE / BT) + blk;
    Spot s;
    s.in = ((x < last ? x : last) * BT) & ((1 << a.page_shift) - 1);
    if constexpr (MIXED)
      s.page = __shfl(entry, off * (WTILE / BT) + blk, 64);
    else
      s.page = (int)readlane_u32((uint32_t)entry, off * (WTILE / BT) + blk);
    return s;
  }
  // Where it lies in its pool, in elements.
  __device__ __forceinline__ long long place(const Spot& s, long long page) const {
    return s.page * page + (((long long)h * D) << a.page_shift) + (long long)s.in * D;
  }
  __device__ __forceinline__ uint32_t scale_at(const Spot& s, int which) const {
    return a.scales[s.page * a.s_page + ((((long long)h << a.page_shift) + s.in) >> 4) * 2 + which];
  }
  // A chunk's index, its wave's for the block's sake.
  __device__ __forceinline__ int chunk(int n) const {
    const int c = n * NTHR + tid;
    return EVEN || c < WTILE * CM ? c : 0;
  }
  template <int PER>  // chunks of a block of tokens
  __device__ __forceinline__ int block_of(int n) const {
    if constexpr (MIXED) return chunk(n) / PER;
    return (n * NTHR + wave * 64) / PER;
  }

  // Chunks on their way, and of an 8-bit cache their blocks' scales.
  struct Moved16 {
    Vec x[NCH];
  };
  struct Moved8 {
    Vec x[NCH];
    uint32_t scale[NCH];
  };
  typedef std::conditional_t<E8, Moved8, Moved16> Moved;

  // Tile i; entry: entries(i - off).
  __device__ __forceinline__ void load(int i, int entry, int off, Moved& k, Moved& v) {
    if ((unsigned)entry >= (unsigned)a.n_pages) {
      bad = true;  // (its sequence's rows become NaN)
      entry = 0;
    }
    typedef std::conditional_t<E8, uint8_t, uint16_t> T;
#pragma unroll
    for (int n = 0; n < NCH; n++) {
      const Spot s = spot_of(i, block_of<BT * CM>(n), entry, off);
      if constexpr (E8) k.scale[n] = scale_at(s, 0);
      k.x[n] = *(const Vec*)((const T*)a.k + place(s, a.k_page) + chunk(n) % (BT * CM) * BT);
    }
#pragma unroll
    for (int n = 0; n < NCH; n++) {
      const Spot s = spot_of(i, block_of<D>(n), entry, off);
      if constexpr (E8) v.scale[n] = scale_at(s, 1);
      v.x[n] = *(const Vec*)((const T*)a.v + place(s, a.v_page) + chunk(n) % D * BT);
    }
  }

  // To buffer f; what lies past the sequence's end is not 0 there (it may be
  // anything, NaN too), and is 0 here.
  __device__ __forceinline__ void store(Shared& s, int f, int i, const Moved& k, Moved& v) {
    if ((i + 1) * WTILE > len) {
#pragma unroll
      for (int n = 0; n < NCH; n++) v.x[n] &= first_of<128 / BT>(len - i * WTILE - block_of<D>(n) * BT);
    }
#pragma unroll
    for (int n = 0; n < NCH; n++) {
      const int c = n * NTHR + tid;
      if (!EVEN && c >= WTILE * CM) continue;
      if constexpr (E8) {
        const float ks = e8::scale_of(k.scale[n]), vs = e8::scale_of(v.scale[n]);
        s.k[f][at_key(c / CM, c % CM * 2)] = decode8<DT>(k.x[n][0], k.x[n][1], ks);
        s.k[f][at_key(c / CM, c % CM * 2 + 1)] = decode8<DT>(k.x[n][2], k.x[n][3], ks);
        Vec* to = s.v[f] + c / D * (2 * D) + c % D;
        to[0] = decode8<DT>(v.x[n][0], v.x[n][1], vs);
        to[D] = decode8<DT>(v.x[n][2], v.x[n][3], vs);
      } else {
        s.k[f][at_key(c / CM, c % CM)] = k.x[n];
        s.v[f][c] = v.x[n];
      }
    }
  }

  // The drafted nodes' tile, from their own rows, to buffer 1 (T <= WTILE: one
  // tile).  Values come row by row and turn into blocks of eight tokens.
  static constexpr int TURN = (8 * C + NTHR - 1) / NTHR;  // (block, chunk)s a thread turns
  static constexpr int NCT = (WTILE * C + NTHR - 1) / NTHR;  // chunks of keys a thread moves
  __device__ __forceinline__ void load_tree(Vec (&k)[NCT], Vec (&v)[TURN][8]) const {
    const uint16_t* kb = (const uint16_t*)a.k_new + b * a.kn_b + h * a.kn_h;
    const uint16_t* vb = (const uint16_t*)a.v_new + b * a.vn_b + h * a.vn_h;
#pragma unroll
    for (int n = 0; n < NCT; n++) {
      const int x = n * NTHR + tid, c = x < WTILE * C ? x : 0, p = c / C;
      k[n] = load16(kb + (p < a.T ? p : a.T - 1) * a.kn_t + c % C * 8);
    }
#pragma unroll
    for (int n = 0; n < TURN; n++) {
      const int c = n * NTHR + tid;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int p = c / C * 8 + j;
        v[n][j] = vec16(0, 0, 0, 0);
        if (c < 8 * C && p < a.T) v[n][j] = load16(vb + p * a.vn_t + c % C * 8);
      }
    }
  }
  __device__ __forceinline__ void store_tree(Shared& s, const Vec (&k)[NCT], Vec (&v)[TURN][8]) const {
#pragma unroll
    for (int n = 0; n < NCT; n++) {
      const int c = n * NTHR + tid;
      if (c < WTILE * C) s.k[1][at_key(c / C, c % C)] = k[n];
    }
    int odd = 0;
    if (a.T > 1) {  // (one node: every row sees it)
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < TURN; n++)
#pragma unroll
        for (int j = 0; j < 8; j++) sum = finite_or_nan<DT>(v[n][j], sum);
      odd = __ballot(sum != 0.0f) != 0;
      if (odd) {
#pragma unroll
        for (int n = 0; n < TURN; n++)
#pragma unroll
          for (int j = 0; j < 8; j++) v[n][j] ^= odd_of<DT>(v[n][j]);
      }
    }
    if (lane == 0) s.odd[wave] = odd;
#pragma unroll
    for (int n = 0; n < TURN; n++) {
      const int c = n * NTHR + tid;
      transpose8(v[n]);
      if (c < 8 * C)
#pragma unroll
        for (int j = 0; j < 8; j++) s.v[1][c / C * D + c % C * 8 + j] = v[n][j];
    }
  }

  struct State {
    f32x16 o[DT32];
    float m, l, r;  // r: the sum of the rounded weights
  };

  // S^T of the tile in buffer f: element j of half x is token 32 x + 16 (j / 8) + 8 half + j % 8.
  __device__ __forceinline__ void scores(const Shared& s, int f, const Vec (&q)[KK], f32x16 (&sc)[2]) const {
    // product row r = 8 x + 4 y + j (j < 4, y < 2) of a half tile is its token 16 (x / 2) + 8 y + 4 (x % 2) + j
    const int tok = (col >> 4) * 16 + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int j = 0; j < 16; j++) sc[x][j] = 0.0f;
    // four operands ahead of the products
    constexpr int N = 2 * KK;
    Vec x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = s.k[f][at_key(j % 2 * 32 + tok, j / 2 * 2 + half)];
#pragma unroll
    for (int j = 0; j < N; j++) {
      sched_fence();
      sc[j % 2] = mfma32<DT>(x[j % 4], q[j / 2], sc[j % 2]);
      if (j + 4 < N) x[j % 4] = s.k[f][at_key(j % 2 * 32 + tok, (j + 4) / 2 * 2 + half)];
    }
    sched_fence();
  }

  // Scores of tokens whose bit (16 x + j) is clear become -inf.
  static __device__ __forceinline__ void mask(f32x16 (&sc)[2], uint32_t bits) {
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int j = 0; j < 16; j++) sc[x][j] = seen(sc[x][j], bits, 16 * x + j);
  }

  __device__ __forceinline__ void add(const Shared& s, int f, const f32x16 (&sc)[2], State& st) const {
    float top = sc[0][0];
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int j = 0; j < 16; j++) top = fmaxf(top, sc[x][j]);
    top = top * a.scale_log2 - lift<DT>();
    if (__ballot(top > st.m + SLACK)) {
      top = fmaxf(top, xor_lane<32>(top));
      const float now = fmaxf(st.m, top);
      const float g = st.m == NEG ? 0.0f : exp2_hw(st.m - now);
      st.m = now;
      st.l *= g;
      st.r *= g;
#pragma unroll
      for (int d = 0; d < DT32; d++) st.o[d] *= g;
    }
    const float base = st.m == NEG ? 0.0f : st.m;
    // Two neighbouring tokens' weights: word i of the 16 tokens 16 y ...
    auto word = [&](int y, int i) {
      const float u = exp2_hw(__builtin_fmaf(sc[y >> 1][(y & 1) * 8 + 2 * i], a.scale_log2, -base));
      const float w = exp2_hw(__builtin_fmaf(sc[y >> 1][(y & 1) * 8 + 2 * i + 1], a.scale_log2, -base));
      st.l += u + w;
      const uint32_t x = to16<DT>(u, w);
      st.r = add2<DT>(x, st.r);
      return x;
    };
    // each product runs beside the weights and the operand of the next 16 tokens'
    Vec x[DT32];
#pragma unroll
    for (int d = 0; d < DT32; d++) x[d] = s.v[f][half * D + d * 32 + col];
    Vec p = vec16(word(0, 0), word(0, 1), word(0, 2), word(0, 3));
#pragma unroll
    for (int y = 0; y < 4; y++) {
      Vec next = p;
#pragma unroll
      for (int d = 0; d < DT32; d++) {
        sched_fence();
        st.o[d] = mfma32<DT>(x[d], p, st.o[d]);
        if (y < 3) {
          x[d] = s.v[f][((y + 1) * 2 + half) * D + d * 32 + col];
#pragma unroll
          for (int i = d * 4 / DT32; i < (d + 1) * 4 / DT32; i++) next[i] = word(y + 1, i);
        }
      }
      p = next;
    }
    sched_fence();
  }

  __device__ __forceinline__ void segment(Shared& s, int given, int t0, int t1, bool full, long long part) {
    len = clamp_len(a, given);
    nc = (len + WTILE - 1) / WTILE;
    table = a.tables + (long long)b * a.P;
    bad = given == FAILED;
    const int row0 = qb * a.QB + wave * 32;  // of the M
    const bool work = row0 < a.M;
    const int i = row0 + col;
    const int node = i < a.M ? i / a.G : 0, hg = i < a.M ? i - node * a.G : 0;
    // Requests first: page entries, queries, the drafted nodes' tile (a worker
    // that has it starts with it), the first tile.
    const int tc = t1 < nc ? t1 : nc;  // the end of the cache's tiles
    auto cut = [&](int t) { return t < tc ? t : tc - 1; };
    const bool cached = t0 < tc, drafted = t1 > nc;
    int e = 0, next = 0;
    if (cached) e = entries(t0);  // (of the first HOLDS tiles)
    int par = -1;
    if (drafted) par = parent_of(a, b);
    Vec q[KK];
    {
      const uint16_t* p = (const uint16_t*)a.q + b * a.q_b + node * a.q_t + (long long)(h * a.G + hg) * a.q_h + half * 8;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) q[kk] = load16(p + kk * 16);
    }
    State st;
    st.m = NEG;
    st.l = st.r = 0.0f;
#pragma unroll
    for (int d = 0; d < DT32; d++)
#pragma unroll
      for (int x = 0; x < 16; x++) st.o[d][x] = 0.0f;
    f32x16 sc[2];
    Moved k0, v0, k1, v1;
    if (drafted) {
      Vec kt[NCT], vt[TURN][8];
      load_tree(kt, vt);
      if (cached) load(t0, e, 0, k0, v0);
      sched_fence();
      lds_barrier();  // (the buffers are free)
      store_tree(s, kt, vt);
    } else {
      load(t0, e, 0, k0, v0);
      sched_fence();
      lds_barrier();
    }
    if (cached) {
      // Tile t is worked on in one buffer while t + 1 goes to the other and
      // the next AHEAD ones are on their way to registers; requests past the
      // last tile ask for it again, so that the number in flight is known.
      store(s, 0, t0, k0, v0);
      next = entries(cut(t0 + 1 + AHEAD));
      sched_fence();
      load(cut(t0 + 1), e, cut(t0 + 1) - t0, k0, v0);
      sched_fence();
      if constexpr (AHEAD == 2) {
        load(cut(t0 + 2), e, cut(t0 + 2) - t0, k1, v1);
        sched_fence();
      }
    }
    lds_barrier();
    if (drafted) {
      int any = 0;
#pragma unroll
      for (int w = 0; w < QW; w++) any |= s.odd[w];
      odd |= uniform(any);
      if (work) {
        const u64 sees = lane_bits(ancestors(a, par), node);
        scores(s, 1, q, sc);
        const u64 in = sees >> (8 * half);
        uint32_t bits = 0;
#pragma unroll
        for (int y = 0; y < 4; y++) bits |= ((uint32_t)(in >> (16 * y)) & 0xFFu) << (8 * y);
        mask(sc, bits);
        add(s, 1, sc, st);
      }
      lds_barrier();
    }
    if (cached) {
      auto step = [&](int t, int f, Moved& ks, Moved& vs) {
        store(s, f ^ 1, cut(t + 1), ks, vs);
        e = next;
        next = entries(cut(t + 2 + AHEAD));
        sched_fence();
        load(cut(t + 1 + AHEAD), e, 0, ks, vs);
        sched_fence();
        if (work) {
          scores(s, f, q, sc);
          if ((t + 1) * WTILE > len) {
            const int left = len - t * WTILE - 8 * half;
            uint32_t bits = 0;
#pragma unroll
            for (int y = 0; y < 4; y++) {
              const int n = left - 16 * y;
              bits |= (n >= 8 ? 0xFFu : n <= 0 ? 0u : (1u << n) - 1) << (8 * y);
            }
            mask(sc, bits);
          }
          add(s, f, sc, st);
        }
        lds_barrier();
      };
      int t = t0;
      for (; t + 1 < tc; t += 2) {  // (an exit between the two would merge their requests' order)
        step(t, 0, k0, v0);
        if constexpr (AHEAD == 2)
          step(t + 1, 1, k1, v1);
        else
          step(t + 1, 1, k0, v0);
      }
      if (t < tc) step(t, 0, k0, v0);
    }
    float m = st.m, l = st.l, lr = st.r;
    const f32x16(&o)[DT32] = st.o;
    l += xor_lane<32>(l);
    lr += xor_lane<32>(lr);
    if (__ballot(bad)) l = __builtin_nanf("");  // (every wave read every entry)
    if (i >= a.M) return;  // (a part's rows past M are not read)
    if (full) {
      const long long row = ((long long)b * a.T + node) * a.Hq + h * a.G + hg;
      const float r = (l > 0.0f ? 1.0f : l) / lr;
#pragma unroll
      for (int d = 0; d < DT32; d++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const f32x4 y = {o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
          store4<DT>((uint16_t*)a.out + row * D + d * 32 + x * 8 + half * 4, y * r);
        }
      if (a.lse && half == 0) a.lse[row] = row_lse(m, l);
    } else {
      float* to = a.part_o + part * D + wave * 32 * D + lane * 4;
      const float r = lr > 0.0f ? l / lr : 1.0f;
#pragma unroll
      for (int d = 0; d < DT32; d++)
#pragma unroll
        for (int x = 0; x < 4; x++)
          *(f32x4*)(to + (d * 4 + x) * 256) = f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]} * r;
      if (half == 0) {
        const long long row = part + wave * 32 + col;
        a.part_ml[row * 2] = m;
        a.part_ml[row * 2 + 1] = l;
      }
    }
  }

  // Puts the drafted values that are not finite (the product had 0 for them)
  // where a row that sees them has its results: no weight or addend that is
  // finite changes them.  A lane writes what it wrote before.
  __device__ __forceinline__ void put_odd(bool full, long long part) const {
    const int i = qb * a.QB + wave * 32 + col;
    const int node = i < a.M ? i / a.G : 0, hg = i < a.M ? i - node * a.G : 0;
    const u64 sees = lane_bits(ancestors(a, parent_of(a, b)), node);
    if (i >= a.M) return;
    __threadfence();  // (behind the stores of the segment, whose types are others)
    uint16_t* out = (uint16_t*)a.out + (((long long)b * a.T + node) * a.Hq + h * a.G + hg) * D;
#pragma nounroll
    for (int d = half * 4; d < D; d += 8) {
      const f32x4 y = odd_sum<DT>(a, b, h, sees, d);
#pragma unroll
      for (int z = 0; z < 4; z++) {
        if (y[z] == 0.0f) continue;
        if (!full)
          a.part_o[part * D + part_at<WideGeo>(D, wave * 32 + col, d + z)] = y[z];
        else if (!is_nan<DT>(out[d + z]))  // (a row of NaN stays one)
          out[d + z] = (uint16_t)to16<DT>(y[z], 0.0f);
      }
    }
  }
};

template <typename DT, int D, int QW, bool E8>
__global__ __launch_bounds__(QW * 64, D == 256 ? 1 : 2) void wide_kernel(AttnArgs a) {
  typedef Wide<DT, D, QW, E8> K;
  TGS_DYN_SMEM(dyn);
  typename K::Shared& s = *(typename K::Shared*)dyn;
  K n(a);
  const int tree = (a.T + WTILE - 1) / WTILE;
  if (a.nwg == 0) {
    const int seg = blockIdx.x / a.nqb;
    n.qb = blockIdx.x % a.nqb;
    n.b = seg / a.Hkv;
    n.h = seg % a.Hkv;
    const int given = uniform(a.lens[n.b]);
    n.segment(s, given, 0, cache_tiles<WideGeo>(a, given) + tree, true, 0);
    if (n.odd) n.put_odd(true, 0);
    return;
  }
  // the row groups that read the same tiles run at the same time on one XCD
  // (workgroups are dealt out to the 8 XCDs in turn)
  const int x = blockIdx.x;
  const int w = a.nwg % 8 == 0 ? x / (8 * a.nqb) * 8 + x % 8 : x / a.nqb;
  n.qb = a.nwg % 8 == 0 ? x / 8 % a.nqb : x % a.nqb;
  const Place at0 = find_place<WideGeo>(a, w);
  const long long u0 = at0.u0, u1 = at0.u1;
  auto walk = [&](auto f) {
    int b = at0.b, h = at0.h, at = at0.at, nt = at0.nt, given = at0.given;
    for (long long u = u0; u < u1;) {
      const int end = nt - at < u1 - u ? nt : at + (int)(u1 - u);
      const int real = nt - WideGeo::EXTRA;
      if (at < real) {
        n.b = b;
        n.h = h;
        f(given, at, end < real ? end : real, real, at == 0 && end >= real, ((long long)(n.qb * a.nwg + w) * 2 + (u != u0)) * a.QB);
      }
      u += end - at;
      at = 0;
      if (++h == a.Hkv) {
        h = 0;
        if (++b < a.B) {
          given = uniform(a.lens[b]);
          nt = cache_tiles<WideGeo>(a, given) + tree + WideGeo::EXTRA;
        }
      }
    }
  };
  walk([&](int given, int t0, int t1, int, bool full, long long part) { n.segment(s, given, t0, t1, full, part); });
  // (Behind everything: code to jump over in a segment costs 1 us of 33, for 16
  // sequences of 1000 to 3000 tokens and 48 rows of 128.)
  if (n.odd) walk([&](int, int, int t1, int real, bool full, long long part) {
    if (t1 == real) n.put_odd(full, part);
  });
}

template <typename DT, int D, int QW, bool E8>
hipError_t wide_run(const AttnArgs& a, hipStream_t st) {
  typedef Wide<DT, D, QW, E8> K;
  const int grid = (a.nwg ? a.nwg : a.B * a.Hkv) * a.nqb;
  hipLaunchKernelGGL((wide_kernel<DT, D, QW, E8>), dim3(grid), dim3(QW * 64), sizeof(typename K::Shared), st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nwg == 0) return e;
  return launch_join<DT, WideGeo>(a, st);
}

template <typename DT, int D, bool E8>
hipError_t wide_dim(const AttnArgs& a, int qw, hipStream_t st) {
  if (qw == 4) return wide_run<DT, D, 4, E8>(a, st);
  if constexpr (D <= 128)
    if (qw == 8) return wide_run<DT, D, 8, E8>(a, st);
  return hipErrorInvalidValue;
}
template <typename DT, int D, int QW, bool E8>
hipError_t wide_lds() {
  return hipFuncSetAttribute((const void*)wide_kernel<DT, D, QW, E8>, hipFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sizeof(typename Wide<DT, D, QW, E8>::Shared));
}
template <typename DT, bool E8>
hipError_t wide_lds_type() {
  hipError_t e = hipSuccess;
  auto take = [&](hipError_t x) { e = x != hipSuccess ? x : e; };
  take(wide_lds<DT, 64, 4, E8>());
  take(wide_lds<DT, 64, 8, E8>());
  take(wide_lds<DT, 96, 4, E8>());
  take(wide_lds<DT, 96, 8, E8>());
  take(wide_lds<DT, 128, 4, E8>());
  take(wide_lds<DT, 128, 8, E8>());
  take(wide_lds<DT, 256, 4, E8>());
  return e;
}
template <typename DT, bool E8>
hipError_t wide_type(const AttnArgs& a, int qw, hipStream_t st) {
  switch (a.D) {
    case 64: return wide_dim<DT, 64, E8>(a, qw, st);
    case 96: return wide_dim<DT, 96, E8>(a, qw, st);
    case 128: return wide_dim<DT, 128, E8>(a, qw, st);
    case 256: return wide_dim<DT, 256, E8>(a, qw, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace attn
}  // namespace tgs
