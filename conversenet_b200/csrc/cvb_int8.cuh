// Quantisation of tokens to 8-bit integers, shared by the kernels of k_int8.cu and k_int8_planes.cu.
//
// q = the integer nearest to 127 x / a, a the token's largest magnitude, an even one where two are as near, decided exactly: with
// r = fp32(127 / a), fma(x, r, 1.5 . 2^23) rounds the exact product to an integer, whose bits end in it; that product is off by
// less than 127 . 2^-24 = 7.6e-6.  Where it lies nearer than 2e-5 to a half (4 in 100000 values) 254 |x| and (2 m + 1) a are
// compared, both exact in 64 bits.  So the integers do not depend on the route, the layout or the device.
// Rounding each value by rintf and a conversion, and comparing where it stood, took 3 times as long (33.6 M bf16 values: 47 us).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cvb {
namespace i8 {

// the larger magnitude of three; a NaN stays
__device__ __forceinline__ float largest(float m, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ float largest(float m, float a) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(a)));
  return r;
}

static __device__ __noinline__ uint32_t quantise4_exactly(float x0, float x1, float x2, float x3, float a) {
  const float up = a < 0x1p-100f ? 0x1p100f : 1.f, top = a * up, r = __fdiv_rn(127.f, top);          // 127 / a stays finite
  const float x[4] = {x0, x1, x2, x3};
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float t = fabsf(x[j] * up) * r;
    int n = (int)rintf(t);
    const int m = (int)floorf(t);
    if (fabsf(t - (float)m - 0.5f) < 1e-4f) {
      const double d = 254.0 * (double)fabsf(x[j] * up) - (2.0 * (double)m + 1.0) * (double)top;
      n = d > 0 || (d == 0 && (m & 1)) ? m + 1 : m;
    }
    w |= (uint32_t)((x[j] < 0.f ? -n : n) & 255) << (8 * j);
  }
  return w;
}

struct Quantiser {
  float a, r;
  bool hard;
  __device__ __forceinline__ explicit Quantiser(float largest_magnitude) : a(largest_magnitude) {
    const bool none = !(a < INFINITY) || a == 0.f;          // (an infinity or NaN among the values: the scale says so)
    hard = !none && a < 0x1p-100f;
    r = none || hard ? 0.f : __fdiv_rn(127.f, a);
  }
  __device__ __forceinline__ float scale() const { return a < INFINITY ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu); }
  // four values as bytes, the first one lowest
  __device__ __forceinline__ uint32_t four(float x0, float x1, float x2, float x3) const {
    constexpr float M = 12582912.f;
    if (!(a < INFINITY)) return 0;
    const float u0 = fmaf(x0, r, M), u1 = fmaf(x1, r, M), u2 = fmaf(x2, r, M), u3 = fmaf(x3, r, M);
    const bool near = fabsf(fmaf(x0, r, M - u0)) > 0.49998f || fabsf(fmaf(x1, r, M - u1)) > 0.49998f ||
                      fabsf(fmaf(x2, r, M - u2)) > 0.49998f || fabsf(fmaf(x3, r, M - u3)) > 0.49998f;
    if (near || hard) return quantise4_exactly(x0, x1, x2, x3, a);
    const uint32_t lo = __byte_perm(__float_as_uint(u0), __float_as_uint(u1), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(u2), __float_as_uint(u3), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
};

}  // namespace i8
}  // namespace cvb
