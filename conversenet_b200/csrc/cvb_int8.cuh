// Quantisation of tokens to 8-bit integers, shared by the kernels of k_int8.cu and k_int8_planes.cu.
//
// q = the integer nearest to t = 127 x / a, a the token's largest magnitude, an even one where two are as near, decided exactly, so
// that the integers do not depend on the route, the layout or the device.  fma(x, r, 1.5 . 2^23), r about 127 / a, rounds the
// exact product x r to an integer, to an even one from a half, and its bits end in it.
//
// fp32: r is 127 / a rounded to nearest, and x r off by less than 127 . 2^-24 = 7.6e-6.  Where it lies nearer than 2e-5 to a half,
// m + 1/2 (4 values in 100000), the sign of 254 |x| - (2 m + 1) a decides, each product as a sum of two fp32 numbers.  So that 254 a is
// an fp32 number and no product loses digits, x and a are multiplied by a power of two first where a lies outside [2^-100, 2^100].
//
// bf16: r is rounded up, and that is enough.  With x = X 2^p, a = A 2^q, X, A integers up to 255, e = p - q <= 0: unless t is a half
// it is at least 2^e / (2 A) >= 2^e / 510 away from one, while x r exceeds t by less than t 2^-23 <= 255 . 2^e . 2^-23.  If t is
// the half m + 1/2, 254 X 2^e = (2 m + 1) A: 127 divides 2 m + 1, so m = 63 and the even integer is the upper one, as x r >= t has
// it; or 127 divides A, and then r is exact.  (Halves are common here: 2 in 1000 values of a wide token are half of its
// largest.  With fp32's way of deciding, 8192 x 4096 values took 41 us.)
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cvb {
namespace i8 {

// the two halves of pdl_start (cvb_tma.cuh)
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*(const uint64_t*)&a), "l"(*(const uint64_t*)&b), "l"(*(const uint64_t*)&c));
  return *(float2*)&d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(const uint64_t*)&a), "l"(*(const uint64_t*)&b));
  return *(float2*)&d;
}

__device__ __forceinline__ uint32_t low_bytes(float2 u, float2 v) {
  const uint32_t lo = __byte_perm(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
constexpr float kRounder = 12582912.f;
// Four fp32 values as bytes, the first one lowest.  `left`: set to `hard` (the caller does them another way)
__device__ __forceinline__ uint32_t nearest_bytes(float x0, float x1, float x2, float x3, float a, float r, bool hard, bool& left) {
  const float2 x = make_float2(x0, x1), y = make_float2(x2, x3), rr = make_float2(r, r), mm = make_float2(kRounder, kRounder);
  float2 u = fma2(x, rr, mm), v = fma2(y, rr, mm);
  // minus the integers, exact
  const float2 nu = add2(mm, make_float2(-u.x, -u.y)), nv = add2(mm, make_float2(-v.x, -v.y));
  const float2 d = fma2(x, rr, nu), e = fma2(y, rr, nv);
  const bool near = (fabsf(d.x) > 0.49998f) | (fabsf(d.y) > 0.49998f) | (fabsf(e.x) > 0.49998f) | (fabsf(e.y) > 0.49998f) | hard;
  left = false;
  if (near) {
    left = hard;
    const float xs[4] = {x0, x1, x2, x3}, ns[4] = {-nu.x, -nu.y, -nv.x, -nv.y}, ds[4] = {d.x, d.y, e.x, e.y};
    float out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float n = fabsf(ns[j]), ax = fabsf(xs[j]);
      const float m = fmaf(ax, r, -n) > 0.f ? n : n - 1.f, k = fmaf(2.f, m, 1.f);
      const float p = 254.f * ax, q = k * a;
      const float s = (p - q) + (fmaf(254.f, ax, -p) - fmaf(k, a, -q));
      const bool up = s > 0.f || (s == 0.f && ((int)m & 1));
      out[j] = kRounder + (fabsf(ds[j]) > 0.49998f ? copysignf(up ? m + 1.f : m, xs[j]) : ns[j]);
    }
    u = make_float2(out[0], out[1]);
    v = make_float2(out[2], out[3]);
  }
  return low_bytes(u, v);
}
// Tokens of very small or very large values, scaled by 2^100 or 2^-100, which leaves every integer as it is: exact, but for values of
// a large token that leave fp32's range below, which are 0.  0 where an infinity or a NaN is among the values.
static __device__ __noinline__ uint32_t nearest_bytes_scaled(float x0, float x1, float x2, float x3, float a) {
  if (!(a < INFINITY)) return 0;
  const float by = a < 1.f ? 0x1p100f : 0x1p-100f, top = a * by;
  bool left;
  return nearest_bytes(x0 * by, x1 * by, x2 * by, x3 * by, top, __fdiv_rn(127.f, top), false, left);
}

template <bool BF16>
struct Quantiser {
  float a, r;
  bool hard;          // 127 / a or 254 a may be no fp32 number; or an infinity or a NaN among the values (0, the scale says so)
  __device__ __forceinline__ explicit Quantiser(float largest_magnitude) : a(largest_magnitude) {
    hard = !(a <= (BF16 ? 0x1.fffffep127f : 0x1p100f)) || (a < 0x1p-100f && a != 0.f);          // (bf16 forms no 254 a)
    r = hard || a == 0.f ? 0.f : BF16 ? __fdiv_ru(127.f, a) : __fdiv_rn(127.f, a);
  }
  __device__ __forceinline__ float scale() const { return a < INFINITY ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu); }
  __device__ __forceinline__ uint32_t four(float x0, float x1, float x2, float x3) const {
    if (BF16) {
      if (hard) return nearest_bytes_scaled(x0, x1, x2, x3, a);
      const float2 rr = make_float2(r, r), mm = make_float2(kRounder, kRounder);
      return low_bytes(fma2(make_float2(x0, x1), rr, mm), fma2(make_float2(x2, x3), rr, mm));
    }
    bool left;
    const uint32_t w = nearest_bytes(x0, x1, x2, x3, a, r, hard, left);
    return left ? nearest_bytes_scaled(x0, x1, x2, x3, a) : w;
  }
};

}  // namespace i8
}  // namespace cvb
