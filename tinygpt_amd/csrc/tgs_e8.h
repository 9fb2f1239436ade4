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
// Four numbers of at most 448 (or NaN) to codes, to the nearest, ties to even.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#elif defined(TGS_HOST_MFMA)
  return hipcpu_to_e4m3(a) | (uint32_t)hipcpu_to_e4m3(b) << 8 | (uint32_t)hipcpu_to_e4m3(c) << 16 | (uint32_t)hipcpu_to_e4m3(d) << 24;
#else
  (void)a, (void)b, (void)c, (void)d;
  return 0;
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

__device__ __forceinline__ bool finite(float x) { return (tg_f2u(x) & 0x7F800000u) != 0x7F800000u; }

// A number as a block takes it: within the cap, NaN where it is not finite.
template <typename DT>
__device__ __forceinline__ float taken(float x) {
  const float y = fminf(fmaxf(x, -cap<DT>()), cap<DT>());
  return finite(x) ? y : __builtin_nanf("");
}
// The larger of m and a taken number's magnitude (NaN: m).
__device__ __forceinline__ float most(float m, float x) { return fmaxf(m, fabsf(x)); }

// Byte of the smallest scale for the largest magnitude m: 448 = 1.75 2^8, so it
// is m's exponent - 8, one more where m's significand passes 1.75 (the addition
// carries then).
template <typename DT>
__device__ __forceinline__ int need_byte(float m) {
  const int e = (int)((tg_f2u(m) + 0x1FFFFFu) >> 23) - 8;
  return e > floor_byte<DT>() ? e : floor_byte<DT>();
}
// 2^-e of a byte.
__device__ __forceinline__ float inverse_of(int byte) {
  return tg_u2f(byte < 254 ? (uint32_t)(254 - byte) << 23 : byte == 254 ? 0x400000u : 0x7FC00000u);
}
// 2^(from - to) of bytes from <= to (below 2^-126, which leaves nothing of a code: 0).
__device__ __forceinline__ float shrink(int from, int to) { return to - from < 127 ? tg_u2f((uint32_t)(127 + from - to) << 23) : 0.0f; }

// ------------------------------------------------------------------ rotation

// Cosine and sine of position * freq: the product and its quarter turn in 64
// bits (a position near 2^17 leaves a 32-bit product 2^-7 off), what is left of
// it, at most pi / 4, by the Taylor polynomials of degree 9 and 10, whose first
// left out terms are below 2^-29.
struct Turn {
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

// Turns the unit's sixteen numbers x (two chunks of eight); cs: its eight cosines
// and sines.
__device__ __forceinline__ void turn_unit(float (&x)[16], const Turn* cs, bool pairs) {
  auto two = [](float& a, float& b, Turn t) {
    const float lo = a, hi = b;
    a = __builtin_fmaf(lo, t.c, -(hi * t.s));
    b = __builtin_fmaf(hi, t.c, lo * t.s);
  };
  if (pairs) {
#pragma unroll
    for (int i = 0; i < 8; i++) two(x[2 * i], x[2 * i + 1], cs[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) two(x[i], x[i + 8], cs[i]);
  }
}

// A chunk's eight 16-bit numbers as floats, and back.
template <typename DT>
__device__ __forceinline__ void widen(uint4 w, float* x) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = from16<DT>(u[i] & 0xFFFFu);
    x[2 * i + 1] = from16<DT>(u[i] >> 16);
  }
}
template <typename DT>
__device__ __forceinline__ uint4 narrow(const float* x) {
  return make_uint4(to16<DT>(x[0], x[1]), to16<DT>(x[2], x[3]), to16<DT>(x[4], x[5]), to16<DT>(x[6], x[7]));
}

}  // namespace e8
}  // namespace tgs
