// tgs_e8.h -- numbers of the 8-bit cache, and the position rotation.
//
// A block is 16 tokens of one head, its keys or its values: e4m3 codes and one
// power of two 2^e (stored as the byte e + 127).  With e the smallest exponent,
// not below the type's floor, with which the block's largest magnitude stays
// within 448, every number of the block is code * 2^e, and that is exact in the
// 16-bit type that the rows had: a code has 4 significant bits, and the floors
// (2^-100 in bf16, 2^-15 in fp16: code steps of 2^-109 and 2^-24) and caps keep
// it inside the type's range.  So attention multiplies what the cache stands
// for, and a block whose scale grows by 2^n loses nothing but the n last bits
// of the codes below 2^-6 2^n.
#pragma once

#include "tgs_device.h"
#include "tgs_kv.h"

namespace tgs {
namespace e8 {

constexpr int BLOCK = 16;

struct BF16 {};
struct F16 {};

#if defined(__HIP_DEVICE_COMPILE__)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#endif

// The 16-bit number in the low half of u.
template <typename DT>
__device__ __forceinline__ float from16(uint32_t u) {
  if constexpr (__is_same(DT, BF16)) return tg_u2f(u << 16);
#if defined(__HIP_DEVICE_COMPILE__)
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
#elif defined(TGS_HOST_MFMA)
  else return hipcpu_to_float((uint16_t)u, false);
#else
  else return 0.0f;
#endif
}
// Two floats to 16 bits, to the nearest, ties to even: the first in the low half.
template <typename DT>
__device__ __forceinline__ uint32_t to16(float lo, float hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  const f32x2 x = {lo, hi};
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

// 2^e of a scale's byte (255 is NaN, and so is what it scales).
__device__ __forceinline__ float scale_of(uint32_t byte) { return tg_u2f(byte << 23); }

// Two e4m3 codes, the low or the high two of w, times the scale s, in 16 bits.
template <bool BF, bool HI>
__device__ __forceinline__ uint32_t decode16(uint32_t w, float s) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, HI));
#elif defined(TGS_HOST_MFMA)
  const uint32_t x = HI ? w >> 16 : w;
  return hipcpu_pack2<BF>(hipcpu_from_e4m3((uint8_t)x) * hipcpu_scale(s), hipcpu_from_e4m3((uint8_t)(x >> 8)) * hipcpu_scale(s));
#else
  (void)w, (void)s;
  return 0;
#endif
}

// The four codes of w as numbers.
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
#elif defined(TGS_HOST_MFMA)
  for (int i = 0; i < 4; i++) x[i] = hipcpu_from_e4m3((uint8_t)(w >> 8 * i));
#else
  (void)w;
  x[0] = x[1] = x[2] = x[3] = 0.0f;
#endif
}
// Codes of four numbers over the scale s, whose magnitudes are at most 448 then (or
// NaN), to the nearest, ties to even.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float s) {
#if defined(__HIP_DEVICE_COMPILE__)
  const s16x2 none = {0, 0};
  const s16x2 w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(none, a, b, s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, s, true));
#elif defined(TGS_HOST_MFMA)
  s = hipcpu_scale(s);
  return hipcpu_to_e4m3(a / s) | (uint32_t)hipcpu_to_e4m3(b / s) << 8 | (uint32_t)hipcpu_to_e4m3(c / s) << 16 | (uint32_t)hipcpu_to_e4m3(d / s) << 24;
#else
  (void)a, (void)b, (void)c, (void)d, (void)s;
  return 0;
#endif
}

// Codes of the four 16-bit numbers of two words over the scale s; four codes whose
// numbers are multiplied by 1 / s (a power of two; they stay where it is 1).
template <typename DT>
__device__ __forceinline__ uint32_t encode4(uint32_t lo, uint32_t hi, float s) {
#if defined(__HIP_DEVICE_COMPILE__)
  s16x2 w = {0, 0};
  if constexpr (__is_same(DT, BF16)) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, lo), s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, hi), s, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, lo), s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, hi), s, true);
  }
  return __builtin_bit_cast(uint32_t, w);
#elif defined(TGS_HOST_MFMA)
  s = hipcpu_scale(s);
  auto one = [&](uint32_t u, int i) { return (uint32_t)hipcpu_to_e4m3(from16<DT>(u & 0xFFFFu) / s) << i; };
  return one(lo, 0) | one(lo >> 16, 8) | one(hi, 16) | one(hi >> 16, 24);
#else
  (void)lo, (void)hi, (void)s;
  return 0;
#endif
}
__device__ __forceinline__ uint32_t recode4(uint32_t w, float s) {  // (a code is exact in bf16)
  return encode4<BF16>(decode16<true, false>(w, 1.0f), decode16<true, true>(w, 1.0f), s);
}

#if defined(__HIP_DEVICE_COMPILE__)
#define TGS_HALVES(op, x, y) __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)))
// Of each half of two words the larger one, and the smaller one.
__device__ __forceinline__ uint32_t max2(uint32_t x, uint32_t y) { return TGS_HALVES(__builtin_elementwise_max, x, y); }
__device__ __forceinline__ uint32_t min2(uint32_t x, uint32_t y) { return TGS_HALVES(__builtin_elementwise_min, x, y); }
#undef TGS_HALVES
#else
template <class F>
__device__ inline uint32_t halves(uint32_t x, uint32_t y, F f) { return f(x & 0xFFFFu, y & 0xFFFFu) | f(x >> 16, y >> 16) << 16; }
__device__ inline uint32_t max2(uint32_t x, uint32_t y) { return halves(x, y, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
__device__ inline uint32_t min2(uint32_t x, uint32_t y) { return halves(x, y, [](uint32_t a, uint32_t b) { return a < b ? a : b; }); }
#endif
// The low (high with HIGH) halves of x and y, in this order.
template <bool HIGH>
__device__ __forceinline__ uint32_t halves_of(uint32_t x, uint32_t y) {
  return HIGH ? x >> 16 | (y & 0xFFFF0000u) : (x & 0xFFFFu) | y << 16;
}
// Bytes 0, 1 (2, 3 with HIGH) of x between those of y: x0 y0 x1 y1.
template <bool HIGH>
__device__ __forceinline__ uint32_t mixed(uint32_t x, uint32_t y) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_perm(y, x, HIGH ? 0x07030602u : 0x05010400u);
#else
  if (HIGH) x >>= 16, y >>= 16;
  return (x & 0xFFu) | (y & 0xFFu) << 8 | (x >> 8 & 0xFFu) << 16 | (y >> 8 & 0xFFu) << 24;
#endif
}
// Bytes 0, 2 of x and 0, 2 of y (1, 3 with ODD), in this order.
template <bool ODD>
__device__ __forceinline__ uint32_t every_second(uint32_t x, uint32_t y) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_perm(y, x, ODD ? 0x07050301u : 0x06040200u);
#else
  if (ODD) x >>= 8, y >>= 8;
  return (x & 0xFFu) | (x >> 8 & 0xFF00u) | (y & 0xFFu) << 16 | (y << 8 & 0xFF000000u);
#endif
}

// The largest magnitude kept: with the largest scale (2^120, 2^8) the next code
// would not be finite in the type.  fp16 numbers from 61,440 to 65,504 are off by
// at most 2^-4 so, as by rounding; bf16 ones past 1.875 2^127 likewise.
template <typename DT>
constexpr float cap() { return __is_same(DT, BF16) ? 0x1.Ep127f : 61440.0f; }
// Byte of the smallest scale.
template <typename DT>
constexpr int floor_byte() { return __is_same(DT, BF16) ? 27 : 112; }

// The bits of the cap in its type, and of infinity.
template <typename DT>
constexpr uint32_t cap_bits() { return __is_same(DT, BF16) ? 0x7F70u : 0x7B80u; }
template <typename DT>
constexpr uint32_t inf_bits() { return __is_same(DT, BF16) ? 0x7F80u : 0x7C00u; }

// A number as a block takes it: within the cap, NaN where it is not finite.
template <typename DT>
__device__ __forceinline__ float taken(float x) {
  const float y = fminf(fmaxf(x, -cap<DT>()), cap<DT>());
  return (tg_f2u(x) & 0x7F800000u) == 0x7F800000u ? __builtin_nanf("") : y;
}
// The same of the two 16-bit numbers of a word; and the largest magnitudes' bits with
// theirs (NaN counts as 0).
template <typename DT>
__device__ __forceinline__ uint32_t taken2(uint32_t w, uint32_t& most) {
  const uint32_t m = w & 0x7FFF7FFFu;
  const uint32_t over = (m + (0x8000u - inf_bits<DT>()) * 0x10001u) & 0x80008000u;  // (no carry between the halves)
  const uint32_t odd = over - (over >> 15);
  const uint32_t y = min2(m, cap_bits<DT>() * 0x10001u);
  most = max2(most, y & ~odd);
  return (w & 0x80008000u) | y | odd;
}

// Byte of the smallest scale for the largest magnitude m: 448 = 1.75 2^8, so it
// is m's exponent - 8, one more where m's significand passes 1.75 (the addition
// carries then).
template <typename DT>
__device__ __forceinline__ int need_byte(float m) {
  const int e = (int)((tg_f2u(m) + 0x1FFFFFu) >> 23) - 8;
  return e > floor_byte<DT>() ? e : floor_byte<DT>();
}
// 2^(to - from) of bytes from <= to (beyond 2^127, which leaves nothing of a code: that).
__device__ __forceinline__ float growth(int from, int to) { return tg_u2f((uint32_t)(127 + (to - from < 127 ? to - from : 127)) << 23); }

// ------------------------------------------------------------------ rotation

// Cosine and sine of position * freq: the product and its quarter turn in 64
// bits (a position near 2^17 leaves a 32-bit product 2^-7 off), what is left of
// it, at most pi / 4, by the Taylor polynomials of degree 9 and 10, whose first
// left out terms are below 2^-29.
struct alignas(8) Turn {
  float c, s;
};
__device__ __forceinline__ Turn turn(uint32_t position, float freq) {
  const double r = (double)position * (double)freq * 0.15915494309189533577;  // turns
  const double q = __builtin_rint(4.0 * r);
  const float x = (float)((r - 0.25 * q) * 6.28318530717958647693), y = x * x;
  float p = __builtin_fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  p = __builtin_fmaf(y, p, 8.3333333e-3f);
  p = __builtin_fmaf(y, p, -1.6666667e-1f);
  const float sx = __builtin_fmaf(y * x, p, x);
  p = __builtin_fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  p = __builtin_fmaf(y, p, -1.3888889e-3f);
  p = __builtin_fmaf(y, p, 4.1666667e-2f);
  p = __builtin_fmaf(y, p, -0.5f);
  const float cx = __builtin_fmaf(y, p, 1.0f);
  // q mod 4, from -2 to 2 before the mask (any quarter where it is no number: x is NaN then)
  const int k = (int)fmin(fmax(q - 4.0 * __builtin_rint(0.25 * q), -2.0), 2.0) & 3;
  Turn t{k & 1 ? sx : cx, k & 1 ? cx : sx};
  if (k == 1 || k == 2) t.c = -t.c;
  if (k >= 2) t.s = -t.s;
  return t;
}

// A row of D dimensions, R of them rotated, falls into units of two chunks of
// eight: unit u of the first R / 16 turns as pairs, halves (8u .. 8u + 7 with
// those R / 2 further) or neighbours (16u .. 16u + 15); the units behind hold
// the dimensions that do not turn, the last of them one chunk where D - R is no
// multiple of 16.
struct Unit {
  int a, b;    // first dimension of each chunk (b < 0: none)
  int angle;   // index of its first of eight angles, -1: it does not turn
};
__device__ __forceinline__ Unit unit_of(int u, int D, int R, bool pairs) {
  if (u < R >> 4) return pairs ? Unit{16 * u, 16 * u + 8, 8 * u} : Unit{8 * u, 8 * u + (R >> 1), 8 * u};
  const int a = 16 * u;
  return Unit{a, a + 8 < D ? a + 8 : -1, -1};
}
__device__ __forceinline__ int units(int D) { return (D + 15) >> 4; }

// Turns the unit's pairs (x[i], x[i + 8]); cs: its eight cosines and sines.
__device__ __forceinline__ void turn_unit(float (&x)[16], const Turn* cs) {
  typedef float Two __attribute__((vector_size(16)));  // two of them
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const Two t = *(const Two*)(cs + i);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float lo = x[i + j], hi = x[i + j + 8];
      x[i + j] = __builtin_fmaf(lo, t[2 * j], -(hi * t[2 * j + 1]));
      x[i + j + 8] = __builtin_fmaf(hi, t[2 * j], lo * t[2 * j + 1]);
    }
  }
}

// A unit's sixteen 16-bit numbers in eight words; neighbours' pairs are taken apart
// (numbers 2 i to place i, 2 i + 1 to place i + 8), and put together again.
template <typename W>
__device__ __forceinline__ void take_apart(W& w) {
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[i] = halves_of<false>(w[2 * i], w[2 * i + 1]);
    x[i + 4] = halves_of<true>(w[2 * i], w[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = x[i];
}
template <typename W>
__device__ __forceinline__ void put_together(W& w) {
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = halves_of<false>(w[i], w[i + 4]);
    x[2 * i + 1] = halves_of<true>(w[i], w[i + 4]);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = x[i];
}
// The same of sixteen codes in four words.
__device__ __forceinline__ void put_together(uint32_t (&c)[4]) {
  const uint32_t x[4] = {mixed<false>(c[0], c[2]), mixed<true>(c[0], c[2]), mixed<false>(c[1], c[3]), mixed<true>(c[1], c[3])};
#pragma unroll
  for (int i = 0; i < 4; i++) c[i] = x[i];
}

// The words' numbers as floats, and back.
template <typename DT>
__device__ __forceinline__ void widen(const uint32_t (&w)[8], float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    x[2 * i] = from16<DT>(w[i] & 0xFFFFu);
    x[2 * i + 1] = from16<DT>(w[i] >> 16);
  }
}
template <typename DT>
__device__ __forceinline__ void narrow(const float (&x)[16], uint32_t (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = to16<DT>(x[2 * i], x[2 * i + 1]);
}

// A unit of a 16-bit row, turned.
template <typename DT>
__device__ __forceinline__ void turn_words(uint32_t (&w)[8], const Turn* cs, bool pairs) {
  float x[16];
  if (pairs) take_apart(w);
  widen<DT>(w, x);
  turn_unit(x, cs);
  narrow<DT>(x, w);
  if (pairs) put_together(w);
}

}  // namespace e8
}  // namespace tgs
