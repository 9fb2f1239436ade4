// hip_runtime.h -- the CPU simulation's shim (../cpu_sim/hip) with what the
// cache, beam and attention kernels use beyond it: 16-byte integer vectors,
// memory fences and the matrix instructions.  TEST INFRASTRUCTURE ONLY.
#pragma once

#include "../../cpu_sim/hip/hip_runtime.h"

#include <cmath>

struct alignas(16) int4 {
  int x, y, z, w;
};
static inline int4 make_int4(int a, int b, int c, int d) { return {a, b, c, d}; }
inline void __threadfence() { __atomic_thread_fence(__ATOMIC_SEQ_CST); }

// ---- matrix instructions: the operands of a wave's lanes lie in one buffer
// per wave of the block (blocks run one after another), between two barriers.
#define TGS_HOST_MFMA 1
inline float hipcpu_to_float(uint16_t x, bool bf16) {
  if (bf16) return __uint_as_float((uint32_t)x << 16);
  const int e = (x >> 10) & 31, m = x & 1023;
  const float s = x & 0x8000 ? -1.0f : 1.0f;
  if (e == 31) return m ? NAN : s * INFINITY;
  return s * (e ? std::ldexp((float)(1024 + m), e - 25) : std::ldexp((float)m, -24));
}
inline uint16_t hipcpu_from_float(float f, bool bf16) {
  const uint32_t u = __float_as_uint(f);
  if (f != f) return bf16 ? 0x7FC0 : 0x7E00;
  if (bf16) return (uint16_t)((u + 0x7FFF + ((u >> 16) & 1)) >> 16);
  const uint16_t s = (uint16_t)(u >> 16 & 0x8000);
  const float a = std::fabs(f);
  if (a >= 65520.0f) return s | 0x7C00;
  int e;
  std::frexp(a, &e);  // a in [2^(e-1), 2^e)
  if (a == 0.0f) return s;
  const int q = e - 11 < -24 ? -24 : e - 11;  // exponent of a step
  const float steps = std::nearbyint(std::ldexp(a, -q));
  const uint32_t n = (uint32_t)steps;
  return s | (uint16_t)(q == -24 ? n : ((uint32_t)(q + 24) << 10) + n);
}
template <bool BF16>
inline uint32_t hipcpu_pack2(float lo, float hi) {
  return hipcpu_from_float(lo, BF16) | (uint32_t)hipcpu_from_float(hi, BF16) << 16;
}
struct hipcpu_ops {
  uint16_t a[64][8], b[64][8];
};
template <int N, bool BF16, typename A, typename V>
inline V hipcpu_mfma(const A& a, const A& b, V c) {
  static hipcpu_ops ops[16];
  hipcpu_ops& o = ops[hipcpu::t_thread.x / 64];
  const int l = hipcpu::lane();
  std::memcpy(o.a[l], &a, 16);
  std::memcpy(o.b[l], &b, 16);
  hipcpu::wave().bar->arrive_and_wait();
  constexpr int PER = N * N / 64, GROUPS = 64 / N;
  for (int i = 0; i < PER; i++) {
    const int row = N == 16 ? 4 * (l / 16) + i : 8 * (i / 4) + 4 * (l / 32) + i % 4;
    float s = c[i];
    for (int g = 0; g < GROUPS; g++)
      for (int k = 0; k < 8; k++)
        s += hipcpu_to_float(o.a[g * N + row][k], BF16) * hipcpu_to_float(o.b[g * N + l % N][k], BF16);
    c[i] = s;
  }
  hipcpu::wave().bar->arrive_and_wait();
  return c;
}
