// tgs_kv8.hip -- new rows into a cache held in 8 bits, their keys turned by their
// positions on the way.
//
// Layout of a layer: keys [page][kv_head][token][D], values
// [page][kv_head][token / 16][D][16], scales [page][kv_head][token / 16][2]; the
// formulas are in tgs_e8.h.  Bound by bytes (a row is read in 16 bits and written
// in 8), or by latency for single tokens.
//
// A wave takes the keys or the values of a head of a block, so that the block's
// largest magnitude is one reduction over the wave.  Numbers stay in 16 bits, two to
// an instruction, from the load to the conversion (magnitudes compare as integers);
// only keys that turn become floats.
//
// 16 layers, 8 key heads of 128: prompts of 300 to 2048 tokens, keys turned, 145 to 147
// us (692 MB, 4.7 TB/s; with floats from the load on and a thread to a number's unit
// 359); single tokens of 8 sequences 5.1 (latency); 32 layers, 64 trees of 63 nodes, up
// to 8 taken, 43 us (first 101).  There the bytes that have to move are 57 MB, but the
// values of a few tokens lie in whole sectors of other tokens', read and written.
#include <type_traits>

#include "tgs_device.h"
#include "tgs_e8.h"
#include "tgs_kv.h"
#include "tgs_kv_write.h"
#include "tgs_row.h"

namespace tgs {
namespace kv8 {

using kv::div_by;

constexpr int NT = 512;  // (64 trees 45 us, with 256 53, with 1024 58)

template <bool ROT>
struct Shared {
  alignas(16) e8::Turn cs[e8::BLOCK][ROTARY_MAX / 2];
  kv::WriteHead head;
};
template <>
struct Shared<false> {
  kv::WriteHead head;
};

// What is written to a block: tokens [lo, hi) of its 16 are new, those before are
// held already; what lies behind keeps its bytes.
struct Block {
  int lo, hi;
};

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  x = step(x, xor_lane<32>(x));
  x = step(x, xor_lane<16>(x));
  x = step(x, xor_lane<8>(x));
  x = step(x, xor_lane<4>(x));
  x = step(x, xor_lane<2>(x));
  return step(x, xor_lane<1>(x));
}

// The block's scale from its new numbers' largest magnitude m (its wave's): the byte,
// its value, and by how much it has grown (1: the held tokens' codes stay).
struct Scale {
  int byte;
  float of, grown;
};
template <typename DT>
__device__ __forceinline__ Scale rescale(const Block& k, float m, int old, uint8_t* at) {
  const int need = e8::need_byte<DT>(m);
  const int now = k.lo > 0 && old > need ? old : need;
  if (lane_id() == 0 && (k.lo == 0 || now != old)) *at = (uint8_t)now;
  return Scale{now, e8::scale_of((uint32_t)now), k.lo > 0 ? e8::growth(old, now) : 1.0f};
}

// Bytes [lo, hi) of eight.
__device__ __forceinline__ u64 bytes_of(int lo, int hi) {
  const u64 a = lo <= 0 ? 0ull : lo >= 8 ? ~0ull : (1ull << (8 * lo)) - 1;
  const u64 b = hi <= 0 ? 0ull : hi >= 8 ? ~0ull : (1ull << (8 * hi)) - 1;
  return b & ~a;
}
// Eight tokens' codes of a dimension: the new ones of x where `fresh`, the held ones'
// over `grown` where `held`, else what was there.
__device__ __forceinline__ uint2 merged(uint2 x, uint2 was, u64 fresh, u64 held, float grown) {
  auto join = [&](uint32_t f, uint32_t h, uint32_t neu, uint32_t old) { return (neu & f) | (((e8::recode4(old, grown) & h) | (old & ~h)) & ~f); };
  return make_uint2(join((uint32_t)fresh, (uint32_t)held, x.x, was.x), join((uint32_t)(fresh >> 32), (uint32_t)(held >> 32), x.y, was.y));
}

// A lane's part of a (block, head): NU units of sixteen 16-bit numbers, two to a word.
// Of keys a (new token, unit of dimensions), of values (eight tokens, two neighbouring
// dimensions), so that a wave reads 256 contiguous bytes of a row.  WHOLE: all sixteen
// tokens are new.
//
// Instructions bound these kernels before bytes do (a block of 128 dimensions gives a
// lane 32 numbers), so that what a wave has in common is left to the scalar unit: the
// tokens of its values, with their rows' addresses.
template <typename DT, int NU, bool ROT, bool WHOLE>
struct Part {
  static constexpr int H = NU == 1 ? 1 : 2;  // units of a lane that are halves of the same dimensions' blocks
  const KvWriteArgs& a;
  const Block k;
  uint32_t w[NU][8];
  uint2 was[WHOLE ? 1 : NU][2];  // of values: what a unit's two dimensions hold
  int D, U;

  __device__ __forceinline__ Part(const KvWriteArgs& args, const Block& b) : a(args), k(b), D(args.c.head_dim), U(args.c.head_dim >> 4) {}

  struct KeyUnit {
    int token;
    e8::Unit u;
    bool fresh;
  };
  __device__ __forceinline__ KeyUnit key_unit(int n) const {
    const unsigned e = lane_id() + 64 * n, i = div_by(e, a.units);
    const int t = (WHOLE ? 0 : k.lo) + (int)i, end = WHOLE ? e8::BLOCK : k.hi;
    return KeyUnit{t < end ? t : end - 1, e8::unit_of((int)(e - i * U), D, ROT ? a.rot.dims : 0, ROT && a.rot.pairs), t < end};
  }
  // Whether any lane has a live unit n: a block that is filled in has few.
  __device__ __forceinline__ bool live(int n) const { return WHOLE || 64 * n < (k.hi - k.lo) * U; }
  struct ValueUnit {
    int first, d;  // of the tokens and of the dimensions
    bool in;
  };
  __device__ __forceinline__ ValueUnit value_unit(int n) const {
    const int lane = lane_id(), D2 = D >> 1;
    const int p = NU == 1 ? (lane < D2 ? lane : lane - D2) : lane + 64 * (n >> 1);
    const int first = NU == 1 ? (lane < D2 ? 0 : 8) : (n & 1) * 8;
    return ValueUnit{first, 2 * (p < D2 ? p : D2 - 1), p < D2};  // (past the last: the last one again, not written)
  }
  // A token, or where it is not new its neighbour among those: no branch among the requests.
  __device__ __forceinline__ int near(int t) const { return WHOLE ? t : t < k.lo ? k.lo : t < k.hi ? t : k.hi - 1; }

  // row(i): the new row of token i of the block.
  template <class F>
  __device__ __forceinline__ void load_keys(F row) {
#pragma unroll
    for (int n = 0; n < NU; n++) {
      if (!live(n)) break;
      const KeyUnit x = key_unit(n);
      const uint16_t* p = row(x.token);
      const uint4 lo = load_row16<true>(p + x.u.a), hi = load_row16<true>(p + x.u.b);
      w[n][0] = lo.x, w[n][1] = lo.y, w[n][2] = lo.z, w[n][3] = lo.w;
      w[n][4] = hi.x, w[n][5] = hi.y, w[n][6] = hi.z, w[n][7] = hi.w;
    }
  }
  // from: row 0 of the new ones; base: the number among them of the block's token 0.
  __device__ __forceinline__ void load_values(const uint16_t* from, long long tok, int base) {
    const ValueUnit x = value_unit(0);
    const uint16_t* p = from + (base + near(x.first)) * tok;
#pragma unroll
    for (int h = 0; h < H; h++) {
      if (!any_new(h)) continue;
#pragma unroll
      for (int i = 0; i < 8; i++) {
#pragma unroll
        for (int n = 0; n < NU; n += H) __builtin_memcpy(&w[n + h][i], p + value_unit(n).d, 4);
        const int t = x.first + 8 * h + i;
        p += WHOLE || (t >= k.lo && t < k.hi - 1) ? tok : 0;
      }
    }
  }
  // The same where path gives the rows' numbers.
  __device__ __forceinline__ void load_values(const uint16_t* from, long long tok, int base, const int* path) {
    if constexpr (NU == 1) {
      const ValueUnit x = value_unit(0);
#pragma unroll
      for (int i = 0; i < 8; i++) __builtin_memcpy(&w[0][i], from + path[base + near(x.first + i)] * tok + x.d, 4);
    } else {
      const int mine = path[base + near(lane_id() & 15)];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (!any_new(h)) continue;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint16_t* p = from + (int)readlane_u32((uint32_t)mine, 8 * h + i) * tok;
#pragma unroll
          for (int n = 0; n < NU; n += 2) __builtin_memcpy(&w[n + h][i], p + value_unit(n).d, 4);
        }
      }
    }
  }
  // Whether unit n of the values has new tokens: of a block that is filled in, often
  // only one half does (a lane has units of both where it has one alone).
  __device__ __forceinline__ bool any_new(int n) const { return WHOLE || NU == 1 || (k.lo < (n & 1) * 8 + 8 && k.hi > (n & 1) * 8); }
  __device__ __forceinline__ bool any_held(int n) const { return NU == 1 || k.lo > (n & 1) * 8; }
  __device__ __forceinline__ void load_held(const uint8_t* from, int n) {
    const ValueUnit x = value_unit(n);
#pragma unroll
    for (int d = 0; d < 2; d++) was[n][d] = *(const uint2*)(from + (x.d + d) * e8::BLOCK + x.first);
  }
  __device__ __forceinline__ void load_held(const uint8_t* from) {
    if constexpr (!WHOLE) {
#pragma unroll
      for (int n = 0; n < NU; n++)
        if (any_new(n)) load_held(from, n);
    }
  }

  // Words of tokens that are not new count as 0.
  __device__ __forceinline__ void select_values() {
    if constexpr (!WHOLE) {
#pragma unroll
      for (int n = 0; n < NU; n++) {
        const ValueUnit x = value_unit(n);
#pragma unroll
        for (int i = 0; i < 8; i++) w[n][i] &= x.first + i >= k.lo && x.first + i < k.hi ? ~0u : 0u;
      }
    }
  }

  static __device__ __forceinline__ uint32_t both(uint32_t m) { return wave_max(m >> 16 > (m & 0xFFFFu) ? m >> 16 : m & 0xFFFFu); }
  // The largest magnitude of all lanes, of the units that count; where it passes the
  // cap, the numbers are capped, and NaN where they are not finite.
  template <class F>
  __device__ __forceinline__ float largest(F counts) {
    uint32_t m = 0;
#pragma unroll
    for (int n = 0; n < NU; n++) {
      if (!counts(n)) continue;
#pragma unroll
      for (int i = 0; i < 8; i++) m = e8::max2(m, w[n][i] & 0x7FFF7FFFu);
    }
    uint32_t top = both(m);
    if (__builtin_expect(top > e8::cap_bits<DT>(), 0)) {
      m = 0;
#pragma unroll
      for (int n = 0; n < NU; n++) {
        if (!counts(n)) continue;
#pragma unroll
        for (int i = 0; i < 8; i++) w[n][i] = e8::taken2<DT>(w[n][i], m);
      }
      top = both(m);
    }
    return e8::from16<DT>(top);
  }

  // The held tokens' keys, whose rows lie one behind the other, over what the scale
  // has grown by.
  __device__ __forceinline__ void regrow(uint8_t* to, float grown) const {
    if (WHOLE || grown == 1.0f) return;
#pragma nounroll
    for (int i = lane_id() * 8; i < k.lo * D; i += 512) {
      const uint2 x = *(const uint2*)(to + i);
      *(uint2*)(to + i) = make_uint2(e8::recode4(x.x, grown), e8::recode4(x.y, grown));
    }
  }
  __device__ __forceinline__ void put_key(const KeyUnit& x, uint8_t* to, uint2 lo, uint2 hi) const {
    if (!x.fresh) return;
    uint8_t* p = to + x.token * D;
    tg_store_nt(p + x.u.a, lo);
    tg_store_nt(p + x.u.b, hi);
  }
  // A scale of NaN, which another program has written, makes NaN of what is added too.
  static __device__ __forceinline__ uint32_t code(uint32_t c, int byte) { return !WHOLE && byte == 255 ? 0x7F7F7F7Fu : c; }

  __device__ __forceinline__ void put_keys(uint8_t* to, int old, uint8_t* scale) {
    const Scale s = rescale<DT>(k, largest([&](int n) { return live(n); }), old, scale);
#pragma unroll
    for (int n = 0; n < NU; n++) {
      if (!live(n)) break;
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; i++) c[i] = code(e8::encode4<DT>(w[n][2 * i], w[n][2 * i + 1], s.of), s.byte);
      put_key(key_unit(n), to, make_uint2(c[0], c[1]), make_uint2(c[2], c[3]));
    }
    regrow(to, s.grown);
  }

  __device__ __forceinline__ void put_turned_keys(const e8::Turn (*cs)[ROTARY_MAX / 2], uint8_t* to, int old, uint8_t* scale) {
    float x[NU][16];
    float top = 0.0f;
    uint32_t m = 0;
#pragma unroll
    for (int n = 0; n < NU; n++) {
      if (!live(n)) break;
      const KeyUnit u = key_unit(n);
      if (a.rot.pairs) e8::take_apart(w[n]);
      e8::widen<DT>(w[n], x[n]);
      if (u.u.angle >= 0) e8::turn_unit(x[n], cs[u.token] + u.u.angle);
#pragma unroll
      for (int i = 0; i < 8; i++) m = e8::max2(m, w[n][i] & 0x7FFF7FFFu);
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, fabsf(x[n][i]));
    }
    top = wave_maxf(top);
    auto put = [&]() {
      const Scale s = rescale<DT>(k, top, old, scale);
#pragma unroll
      for (int n = 0; n < NU; n++) {
        if (!live(n)) break;
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = code(e8::encode4(x[n][4 * i], x[n][4 * i + 1], x[n][4 * i + 2], x[n][4 * i + 3], s.of), s.byte);
        if (a.rot.pairs) e8::put_together(c);
        put_key(key_unit(n), to, make_uint2(c[0], c[1]), make_uint2(c[2], c[3]));
      }
      regrow(to, s.grown);
    };
    // (a NaN shows in no maximum, but in the rows)
    if (__builtin_expect(top <= e8::cap<DT>() && !__ballot((m & 0xFFFFu) >= e8::inf_bits<DT>() || m >> 16 >= e8::inf_bits<DT>()), 1)) {
      put();
      return;
    }
    top = 0.0f;
#pragma unroll
    for (int n = 0; n < NU; n++) {
      if (!live(n)) break;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        x[n][i] = e8::taken<DT>(x[n][i]);
        top = fmaxf(top, fabsf(x[n][i]));
      }
    }
    top = wave_maxf(top);
    put();
  }

  // The codes of unit n's two dimensions, eight tokens each.
  __device__ __forceinline__ void codes(int n, const Scale& s, uint2 (&c)[2]) const {
    uint32_t p[4];  // two tokens' two codes
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = code(e8::encode4<DT>(w[n][2 * i], w[n][2 * i + 1], s.of), s.byte);
    c[0] = make_uint2(e8::every_second<false>(p[0], p[1]), e8::every_second<false>(p[2], p[3]));
    c[1] = make_uint2(e8::every_second<true>(p[0], p[1]), e8::every_second<true>(p[2], p[3]));
  }

  __device__ __forceinline__ void put_values(uint8_t* to, int old, uint8_t* scale) {
    select_values();
    const Scale s = rescale<DT>(k, largest([&](int n) { return any_new(n); }), old, scale);
    if constexpr (WHOLE) {
#pragma unroll
      for (int n = 0; n < NU; n += H) {
        uint2 c[H][2];
#pragma unroll
        for (int h = 0; h < H; h++) codes(n + h, s, c[h]);
        const ValueUnit x = value_unit(n);
        if (!x.in) continue;
        uint8_t* p = to + x.d * e8::BLOCK + x.first;
#pragma unroll
        for (int d = 0; d < 2; d++, p += e8::BLOCK) {
          if constexpr (H == 2) tg_store_nt(p, make_uint4(c[0][d].x, c[0][d].y, c[1][d].x, c[1][d].y));
          else tg_store_nt(p, c[0][d]);
        }
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < NU; n++) {
      const ValueUnit x = value_unit(n);
      uint8_t* p = to + x.d * e8::BLOCK + x.first;
      uint2 c[2];
      if (any_new(n)) {
        codes(n, s, c);
#pragma unroll
        for (int d = 0; d < 2; d++) c[d] = merged(c[d], was[n][d], bytes_of(k.lo - x.first, k.hi - x.first), bytes_of(0, k.lo - x.first), s.grown);
      } else if (s.grown != 1.0f && any_held(n)) {
        load_held(to, n);
#pragma unroll
        for (int d = 0; d < 2; d++) c[d] = merged(c[d], was[n][d], 0, ~0ull, s.grown);
      } else {
        continue;
      }
      if (!x.in) continue;
#pragma unroll
      for (int d = 0; d < 2; d++) *(uint2*)(p + d * e8::BLOCK) = c[d];
    }
  }
};

// Workgroup (sequence b, x, layers from l0 on, keys or values) over the 16-token blocks
// x, x + step, ... of the positions that b's new rows take.  An append's values come
// behind all keys, so that what runs together reads and writes the same pools (prompts
// 152 us where they alternate 160; a commit, of few workgroups, alternates: one tree
// 6.0 where keys first take 6.4).  The layers of a workgroup
// share the look at the sequence and the cosines and sines of a block's positions.
template <typename DT, int NU, bool COMMIT, bool ROT>
__global__ __launch_bounds__(NT) void write_kernel(KvWriteArgs a, int per, int step, FastDiv heads) {
  TGS_STATIC_SMEM(Shared<ROT>, sh);
  kv::WriteHead& s = sh.head;
  const int b = blockIdx.x, half = gridDim.y >> 1;
  const bool values = COMMIT ? blockIdx.y & 1 : (int)blockIdx.y >= half;
  const int y = COMMIT ? blockIdx.y >> 1 : blockIdx.y - (values ? half : 0), g = y / step, x = y - g * step, l0 = g * per;
  const int tid = threadIdx.x;
  const int len = a.lens[b], n = kv::rows_of<COMMIT>(a, s, b);
  const int* table = a.tables + (long long)b * a.P;
  int bad = kv::past_table(a, len, n);
  if (!bad) bad = kv::outside_pool(a, table, len, n);
  bad = __syncthreads_or(bad);
  if (blockIdx.y == 0) kv::report<COMMIT>(a, s, b, len, n, bad);
  if (bad || n == 0) return;
  const int H = a.c.kv_heads, page = 1 << a.page_shift;
  const int tasks = H * (a.c.layers - l0 < per ? a.c.layers - l0 : per);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
  const int first = (len >> 4) + x, last = (len + n - 1) >> 4;
  auto block = [&](int blk) {
    const int lo = len - (blk << 4), hi = len + n - (blk << 4);
    return Block{lo > 0 ? lo : 0, hi < e8::BLOCK ? hi : e8::BLOCK};
  };
  // (layer, head) t: f(layer, its scale, its codes' place in a layer's pool)
  auto each = [&](int blk, const Block& k, long long page_bytes, auto f) {
    const long long pg = table[blk << 4 >> a.page_shift];
    const int in_page = (blk << 4) & (page - 1);
#pragma nounroll
    for (int t = wave; t < tasks; t += waves) {
      const int dl = div_by((unsigned)t, heads), l = l0 + dl, h = t - dl * H;
      const long long slot = ((long long)h << a.page_shift) + in_page;
      uint8_t* scale = a.scales + l * a.s_layer + pg * a.s_page + (slot >> 4) * 2 + values;
      f(l, h, scale, k.lo > 0 ? *scale : 0, pg * page_bytes + slot * a.c.head_dim);
    }
  };
  if (values) {
    for (int blk = first; blk <= last; blk += step) {
      const Block k = block(blk);
      const int base = (blk << 4) - len;
      auto go = [&](auto whole) {
        each(blk, k, a.c.v_page, [&](int l, int h, uint8_t* scale, int old, long long at) {
          Part<DT, NU, ROT, decltype(whole)::value> p(a, k);
          const uint16_t* from = (const uint16_t*)a.r.v + l * a.r.v_layer + b * a.r.v_seq + h * a.r.v_head;
          uint8_t* to = (uint8_t*)a.c.v + l * a.c.v_layer + at;
          if constexpr (COMMIT) p.load_values(from, a.r.v_tok, base, s.path);
          else p.load_values(from, a.r.v_tok, base);
          p.load_held(to);
          p.put_values(to, old, scale);
        });
      };
      if (k.lo == 0 && k.hi == e8::BLOCK) go(std::true_type{});
      else go(std::false_type{});
    }
    return;
  }
  for (int blk = first; blk <= last; blk += step) {
    const Block k = block(blk);
    const int base = (blk << 4) - len;
    if constexpr (ROT) {
      const int half = a.rot.dims >> 1;
      __syncthreads();  // (the block before is done with the table)
      for (int e = tid; e < (k.hi - k.lo) * half; e += (int)blockDim.x) {
        const int i = div_by((unsigned)e, a.turns), j = e - i * half;
        sh.cs[k.lo + i][j] = e8::turn((uint32_t)((blk << 4) + k.lo + i), a.rot.freq[j]);
      }
      __syncthreads();
    }
    auto go = [&](auto whole) {
      each(blk, k, a.c.k_page, [&](int l, int h, uint8_t* scale, int old, long long at) {
        Part<DT, NU, ROT, decltype(whole)::value> p(a, k);
        const uint16_t* from = (const uint16_t*)a.r.k + l * a.r.k_layer + b * a.r.k_seq + h * a.r.k_head;
        uint8_t* to = (uint8_t*)a.c.k + l * a.c.k_layer + at;
        p.load_keys([&](int i) { return from + (COMMIT ? s.path[base + i] : base + i) * a.r.k_tok; });
        if constexpr (ROT) p.put_turned_keys(sh.cs, to, old, scale);
        else p.put_keys(to, old, scale);
      });
    };
    if (k.lo == 0 && k.hi == e8::BLOCK) go(std::true_type{});
    else go(std::false_type{});
  }
}

// ------------------------------------------------------------------ single tokens

// One new row a sequence and layer: a thread takes sixteen dimensions of a head, of
// its key or of its value, and the largest magnitude of each goes by integer maxima
// in LDS.  A value's codes are single bytes of their blocks.  In the kernel above a
// wave would work on sixteen tokens of which one is new (16 layers, 8 sequences, 8
// heads of 128: 4.9 us, there 9 to 13).
constexpr int STEP_NT = 256;
constexpr int STEP_HEADS = STEP_NT / 2;  // of a round at most (a head has at least one unit of its key)

struct StepShared {
  alignas(16) e8::Turn cs[ROTARY_MAX / 2];
  uint32_t top[STEP_HEADS][2];  // bits of the largest magnitude
  int grown[STEP_HEADS][2];     // bytes that the scale has grown by
};

template <typename DT, bool ROT>
__global__ __launch_bounds__(STEP_NT) void step_kernel(KvWriteArgs a, int round) {
  TGS_STATIC_SMEM(StepShared, s);
  const int b = blockIdx.x, rounds = (a.c.kv_heads + round - 1) / round, l = blockIdx.y / rounds, z = blockIdx.y - l * rounds, tid = threadIdx.x;
  const int D = a.c.head_dim, U = D >> 4;
  const int len = a.lens[b], n = a.counts ? a.counts[b] : 1;
  const bool past = kv::past_table(a, len, n);
  const int entry = past || n == 0 ? 0 : a.tables[(long long)b * a.P + (len >> a.page_shift)];
  const bool bad = past || (unsigned)entry >= (unsigned)a.c.n_pages;
  if (blockIdx.y == 0 && tid == 0) a.lens_out[b] = bad ? -1 : len + n;
  if (bad || n == 0) return;
  // heads of this workgroup's round: unit u of which, key or value, is this thread's
  const int h0 = z * round, heads = a.c.kv_heads - h0 < round ? a.c.kv_heads - h0 : round;
  const bool work = tid < 2 * heads * U;
  const int hv = work ? (int)div_by((unsigned)tid, a.units) : 0, u = tid - hv * U;
  const bool value = hv >= heads;
  const int hl = value ? hv - heads : hv, h = h0 + hl;
  const e8::Unit w = e8::unit_of(u, D, ROT && !value ? a.rot.dims : 0, ROT && a.rot.pairs);
  uint32_t words[8];
  if (work) {
    const uint16_t* p = value ? (const uint16_t*)a.r.v + l * a.r.v_layer + b * a.r.v_seq + h * a.r.v_head
                              : (const uint16_t*)a.r.k + l * a.r.k_layer + b * a.r.k_seq + h * a.r.k_head;
    const uint4 lo = load_row16<true>(p + w.a), hi = load_row16<true>(p + w.b);
    words[0] = lo.x, words[1] = lo.y, words[2] = lo.z, words[3] = lo.w;
    words[4] = hi.x, words[5] = hi.y, words[6] = hi.z, words[7] = hi.w;
  }
  const bool turns = ROT && w.angle >= 0, apart = turns && a.rot.pairs;
  float x[16];
  const int in_page = len & ((1 << a.page_shift) - 1), at = in_page & 15;
  const long long slot = ((long long)h << a.page_shift) + (in_page & ~15);
  uint8_t* scale = a.scales + l * a.s_layer + entry * a.s_page + (slot >> 4) * 2 + value;
  uint8_t* to = value ? (uint8_t*)a.c.v + l * a.c.v_layer + entry * a.c.v_page + slot * D
                      : (uint8_t*)a.c.k + l * a.c.k_layer + entry * a.c.k_page + slot * D;
  int old = 0;
  if (work && at) old = *scale;
  if (tid < 2 * heads) (&s.top[0][0])[tid] = 0;
  if constexpr (ROT)
    for (int j = tid; j < a.rot.dims >> 1; j += STEP_NT) s.cs[j] = e8::turn((uint32_t)len, a.rot.freq[j]);
  __syncthreads();
  if (work) {
    if (apart) e8::take_apart(words);
    e8::widen<DT>(words, x);
    if (turns) e8::turn_unit(x, s.cs + w.angle);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      x[i] = e8::taken<DT>(x[i]);
      top = fmaxf(top, fabsf(x[i]));
    }
    atomicMax(&s.top[hl][value], tg_f2u(top));
  }
  __syncthreads();
  if (work) {
    const int need = e8::need_byte<DT>(tg_u2f(s.top[hl][value]));
    const int now = at && old > need ? old : need;
    const float of = e8::scale_of((uint32_t)now);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      c[i] = e8::encode4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], of);
      if (now == 255) c[i] = 0x7F7F7F7Fu;  // (a scale of NaN, which another program has written)
    }
    if (apart) e8::put_together(c);
    if (u == 0) {
      s.grown[hl][value] = at ? now - old : 0;
      if (!at || now != old) *scale = (uint8_t)now;
    }
    if (!value) {
      *(uint2*)(to + at * D + w.a) = make_uint2(c[0], c[1]);
      *(uint2*)(to + at * D + w.b) = make_uint2(c[2], c[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) to[(w.a + i) * e8::BLOCK + at] = (uint8_t)(c[i >> 2] >> 8 * (i & 3));
    }
  }
  if (at == 0) return;
  __syncthreads();
  // the held tokens' codes of a head whose scale has grown, eight bytes a thread
#pragma nounroll
  for (int g = 0; g < 2 * heads; g++) {
    const int by = (&s.grown[0][0])[g];
    if (by == 0) continue;
    const float of = e8::growth(0, by);
    const bool val = g & 1;
    const long long first = (((long long)(h0 + (g >> 1)) << a.page_shift) + (in_page & ~15)) * D;
    uint8_t* p = val ? (uint8_t*)a.c.v + l * a.c.v_layer + entry * a.c.v_page + first : (uint8_t*)a.c.k + l * a.c.k_layer + entry * a.c.k_page + first;
    const int chunks = (val ? e8::BLOCK : at) * D >> 3;
#pragma nounroll
    for (int i = tid; i < chunks; i += STEP_NT) {
      const u64 held = val ? bytes_of(0, at - 8 * (i & 1)) : ~0ull;
      const uint2 o = ((const uint2*)p)[i];
      ((uint2*)p)[i] = merged(make_uint2(0, 0), o, 0, held, of);
    }
  }
}

template <typename DT, bool COMMIT, bool ROT>
hipError_t run(const KvWriteArgs& a, int num_cu, hipStream_t st) {
  // Layers to a workgroup: as many as leave eight workgroups a CU (half of them for
  // blocks that are not there, as a rule), and at most four (layer, head)s to a wave.  One
  // always, this rule, eight always (us): 64 trees of 32 layers, 8 heads of 128, 71, 45,
  // 53; prompts of 16 layers 217, 148, 157; one tree of 16 layers 5.9, 5.9, 15.5.
  const long long all = 2ll * a.nblk * a.B * a.c.layers;
  int per = (int)(all / (8ll * num_cu));
  const int most = 4 * NT / 64 / a.c.kv_heads;
  per = per < most ? per : most;
  per = per < 1 ? 1 : per;
  per = per < a.c.layers ? per : a.c.layers;
  const int groups = (a.c.layers + per - 1) / per, tasks = a.c.kv_heads * per;
  if (groups > 32767) return hipErrorInvalidValue;
  const int step = a.nblk < 32767 / groups ? a.nblk : 32767 / groups;
  const dim3 grid(a.B, 2 * step * groups), block(64 * (tasks < NT / 64 ? tasks : NT / 64));
  const FastDiv heads = fast_div(a.c.kv_heads);
  if (a.c.head_dim <= 64)
    hipLaunchKernelGGL((write_kernel<DT, 1, COMMIT, ROT>), grid, block, 0, st, a, per, step, heads);
  else if (a.c.head_dim <= 128)
    hipLaunchKernelGGL((write_kernel<DT, 2, COMMIT, ROT>), grid, block, 0, st, a, per, step, heads);
  else
    hipLaunchKernelGGL((write_kernel<DT, 4, COMMIT, ROT>), grid, block, 0, st, a, per, step, heads);
  return hipGetLastError();
}

template <typename DT>
hipError_t step(const KvWriteArgs& a, hipStream_t st) {
  const int most = STEP_NT / (2 * (a.c.head_dim >> 4)), round = a.c.kv_heads < most ? a.c.kv_heads : most;
  const long long y = (long long)a.c.layers * ((a.c.kv_heads + round - 1) / round);
  if (y > 65535) return hipErrorInvalidValue;
  const dim3 grid(a.B, (unsigned)y);
  if (a.rot.freq)
    hipLaunchKernelGGL((step_kernel<DT, true>), grid, dim3(STEP_NT), 0, st, a, round);
  else
    hipLaunchKernelGGL((step_kernel<DT, false>), grid, dim3(STEP_NT), 0, st, a, round);
  return hipGetLastError();
}

}  // namespace kv8

hipError_t launch_kv8_append(const KvWriteArgs& a, int num_cu, hipStream_t st) {
  if (a.T == 1) return a.c.dtype == TGS_BF16 ? kv8::step<e8::BF16>(a, st) : kv8::step<e8::F16>(a, st);
  if (a.rot.freq) return a.c.dtype == TGS_BF16 ? kv8::run<e8::BF16, false, true>(a, num_cu, st) : kv8::run<e8::F16, false, true>(a, num_cu, st);
  return a.c.dtype == TGS_BF16 ? kv8::run<e8::BF16, false, false>(a, num_cu, st) : kv8::run<e8::F16, false, false>(a, num_cu, st);
}
hipError_t launch_kv8_commit(const KvWriteArgs& a, int num_cu, hipStream_t st) {
  return a.c.dtype == TGS_BF16 ? kv8::run<e8::BF16, true, false>(a, num_cu, st) : kv8::run<e8::F16, true, false>(a, num_cu, st);
}

}  // namespace tgs
