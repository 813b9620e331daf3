// The seam between two branches of a block, forward and backward.  With N an affine LayerNorm or RMS norm over the channels of
// a token (N = identity without weights) and s(g) the gate, itself or its sigmoid:
//     p = N_post(branch),  y = x + a . s(g) . p,  z = N_pre(y)
// and, with h = the normalised branch, k = the normalised y, r their 1 / spread:
//     d  = dy + r_k ( dz w_pre - mean(dz w_pre) - k mean(dz w_pre k) )               dx = d      (RMS norm: without mean(.))
//     dp = d a s(g),  dbranch = r_h ( dp w_post - mean(dp w_post) - h mean(dp w_post h) ),  dg = d a p s'(g)
//     dw_pre = sum dz k,  db_pre = sum dz;  with A = sum d s(g) h and B = sum d s(g) over tokens:
//     dw_post = a A,  db_post = a B,  da = w_post A + b_post B;  a gate per image and channel: a (w_post A_i + b_post B_i) s'(g)
//     with A_i, B_i the sums over the image's tokens without s(g), and A = sum_i s(g_i) A_i.
// So every parameter's gradient follows from four sums for each channel (for each image and channel where the gate is).
//
// All of it is bound by bytes: each tensor is read and written once, the values of a token stay in registers between its
// norms.  channels_first (B,C,HW): a warp holds 32 VEC pixels, its threads CPT channels of them each, and the warps of a block the
// other channels; a token's sums meet in shared memory, once for each norm (each thread brings its own mean and the squares
// around it, which are joined exactly).  channels_last (T,C): the threads that share a token hold vectors of its channels; sums
// meet by shuffles, and through shared memory where a token has more than a warp.  Backward: blocks walk over tokens with the
// four sums of their channels in registers and leave one partial result each; a second kernel adds them in order, in 64 bits.
// Means, spreads and sums are held in 32 bits or more; z comes from y before y is rounded to the tensors' type.
//
// A spread's reciprocal is rsqrtf's, good to 2 units.  With one to three channels the normalised values are near 1 and -1 and what a norm's
// gradient keeps is their difference from that, so that a weight's gradient, summed over tokens of both signs, lies 3 to 6 times as far
// from 64 bits as with a square root and a division (33 x 31 tokens of one channel: 4.4e-6 of it, and 9.5e-7).
//
// 8 x 64 x 256 x 256 fp32 with both norms: forward 89 us (82 at the measured copy rate), gradients 134 (123).  On the way: 145 us with
// every thread adding up all warps' sums and vectors read from global memory (120 instructions an element); gradients 280 us with a
// tile's loads waited for at its beginning, 194 with two pixels a thread instead of four.  bf16 tokens with a gate (65472 x 1024): 211 us
// (102), gradients 281 (164; 1.4 % more since a gate's slope keeps its digits), at present bound by instructions: conversions, the gate's exponential and two norms' sums of 8 values a thread.
#include "../../include/converse_b200.h"
#include "cvb_internal.h"
#include "cvb_seam.h"

namespace cvb {
namespace seam {

// ------------------------------------------------------------------ values
template <typename IO, int V>
struct Vec;
template <>
struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) { v[0] = ((const float*)p)[i]; }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) { ((float*)p)[i] = v[0]; }
};
template <>
struct Vec<float, 2> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const float2 a = *(const float2*)((const float*)p + i);
    v[0] = a.x; v[1] = a.y;
  }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) { *(float2*)((float*)p + i) = make_float2(v[0], v[1]); }
};
template <>
struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const float4 a = *(const float4*)((const float*)p + i);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec<__nv_bfloat16, 1> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) { v[0] = __bfloat162float(((const __nv_bfloat16*)p)[i]); }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) { ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v[0]); }
};
template <>
struct Vec<__nv_bfloat16, 2> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const unsigned a = *(const unsigned*)((const __nv_bfloat16*)p + i);
    v[0] = __uint_as_float(a << 16); v[1] = __uint_as_float(a & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) {
    *(__nv_bfloat162*)((__nv_bfloat16*)p + i) = __floats2bfloat162_rn(v[0], v[1]);
  }
};
template <>
struct Vec<__nv_bfloat16, 4> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const uint2 a = *(const uint2*)((const __nv_bfloat16*)p + i);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) {
    __nv_bfloat162 a[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
    *(uint2*)((__nv_bfloat16*)p + i) = *(const uint2*)a;
  }
};
template <>
struct Vec<__nv_bfloat16, 8> {
  static __device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const uint4 a = *(const uint4*)((const __nv_bfloat16*)p + i);
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(void* p, long long i, const float* v) {
    __nv_bfloat162 a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    *(uint4*)((__nv_bfloat16*)p + i) = *(const uint4*)a;
  }
};

// Asynchronous copies of a thread's own values to its own shared memory, which it alone reads: no barrier, and the loads of the
// next token are in flight while this one is worked on without a register held for them.  Zeros where `on` is false.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool on) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(on ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES), "r"(on ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy_pieces(void* to, const void* from, int bytes) {          // 16 bytes or fewer, zeros behind
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A gate of each element: its sigmoid s = 1 / (1 + e), e = exp(-g) = 2^(-g log2 e).  fp32: with what the product and the constant lose,
// which would be |g| 2^-24 of e: the product's rounding error is itself an fma, and 2^(h + c) = 2^h (1 + c ln 2) for so small a c (g kept
// where that is a number; NaN stays).  ex2.approx is good to 2^-22, the reciprocal to a unit.
// bf16: without, 1e-6 of s at |g| = 10 or a thousandth of the type's rounding.  Neither keeps numbers below 2^-126.
// (expf and a division took 4 to 12 % more of the fp32 kernels' times forward and 5 to 26 % of the gradients'; this takes 0 to 3 and 0 to
// 5 % more than s from __expf and s (1 - s) did, 8 x 96 x 128 x 128 fp32 gradients 118 -> 124 us the most.)
template <typename IO>
__device__ __forceinline__ float gate_exp(float g) {
  constexpr double kLn2 = 0.693147180559945309417;
  constexpr float log2e = (float)(1 / kLn2), rest = (float)(1 / kLn2 - (double)log2e), ln2 = (float)kLn2;
  float e;
  if (sizeof(IO) == 2) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -log2e));
    return e;
  }
  asm("min.NaN.f32 %0, %0, 0f42D00000;" : "+f"(g));          // 104
  asm("max.NaN.f32 %0, %0, 0fC2B00000;" : "+f"(g));          // -88
  const float h = g * -log2e, c = fmaf(g, -rest, fmaf(g, -log2e, -h));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(h));
  return fmaf(e * c, ln2, e);
}
__device__ __forceinline__ float reciprocal(float v) {
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v));
  return v;
}
// For the gradient it is held as the smaller of s and 1 - s, negative where it is 1 - s: so the slope s (1 - s) keeps all its digits (s
// by itself has none of 1 - s from g = 17 on).  sigmoid_hold gives s and leaves that in g; gate_factor gives s from it, but for the last
// place the same (`one`: the bits of 1, or 0 where the gate is taken as it is; -0 gives 1).  A forward kernel takes s the way that the
// gradients' does.
template <typename IO>
__device__ __forceinline__ float sigmoid_hold(float& g) {
  const float e = gate_exp<IO>(g), s = reciprocal(1.f + e);
  g = g > 0.f ? -(e * s) : s;
  return s;
}
__device__ __forceinline__ float gate_factor(float f, int one) { return f + __int_as_float((__float_as_int(f) >> 31) & one); }
__device__ __forceinline__ float gate_slope(float f, bool act) { return act ? fmaf(-fabsf(f), fabsf(f), fabsf(f)) : 1.f; }
constexpr int kOne = 0x3f800000;
// channels_first
template <typename IO>
__device__ __forceinline__ float cf_gate_of(float g, int act) { return act ? reciprocal(1.f + gate_exp<IO>(g)) : g; }
// channels_last
template <typename IO>
__device__ __forceinline__ float cl_gate_of(float g, int act) {
  if (!act) return g;
  sigmoid_hold<IO>(g);
  return gate_factor(g, kOne);
}
// the gate of an image, of which there are few: to the last place
__device__ __forceinline__ float image_gate_of(float g, int act) { return act ? 1.f / (1.f + expf(-g)) : g; }
__device__ __forceinline__ float image_gate_slope(float g, int act) {
  const float e = expf(-fabsf(g)), s = 1.f / (1.f + e);
  return act ? s * (e * s) : 1.f;
}

// ------------------------------------------------------------------ channels_first, forward
// The VEC pixels of a thread: neighbours, read and written as vectors (ALONG), where rows are aligned to them; else 32 apart.
// `live`: bit j for a pixel j inside the image (neighbours: all or none).
template <int VEC, bool ALONG>
struct Pixels {
  long long first;
  unsigned live;
  __device__ __forceinline__ Pixels(unsigned tile, int lane, long long HW) {
    first = (long long)tile * (32 * VEC) + (ALONG ? lane * VEC : lane);
    if (ALONG) {
      live = first < HW ? (1u << VEC) - 1 : 0u;
    } else {
      live = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) live |= (first + 32 * j < HW ? 1u : 0u) << j;
    }
  }
  // zeros outside
  template <typename IO>
  __device__ __forceinline__ void load(const void* p, long long at, float* v, bool on = true) const {
    if (ALONG) {
      if (live && on) {
        Vec<IO, VEC>::load(p, at, v);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[j] = 0.f;
        if (on && (live >> j & 1)) Vec<IO, 1>::load(p, at + 32 * j, v + j);
      }
    }
  }
  // The same through shared memory: `fetch` begins it, `fetched` reads it.  Vectors and 4-byte values: a thread's own, which it alone
  // reads.  Else, 2 bytes being too few for a copy, the warp's pixels of the row in the 16-byte pieces that they lie in (the warp
  // meets before it reads them and before the next ones come).  `row`: the tile's first pixel; of the bytes before it only those
  // inside the tensor, from `all` on, are read.
  template <typename IO>
  static constexpr bool kOwn = sizeof(IO) == 4 || (ALONG && VEC * sizeof(IO) >= 4);
  template <typename IO>
  static constexpr int kSlot = kOwn<IO> ? 32 * VEC * (int)sizeof(IO) : 32 * VEC * (int)sizeof(IO) + 16;          // bytes of a warp
  template <typename IO>
  __device__ __forceinline__ void fetch(char* slot, const IO* all, const IO* row, long long HW) const {
    const int lane = threadIdx.x & 31, tile_first = ALONG ? lane * VEC : lane;
    if constexpr (kOwn<IO> && ALONG) {
      copy_async<VEC * sizeof(IO)>(slot + tile_first * sizeof(IO), live ? row + tile_first : row, live);
    } else if constexpr (kOwn<IO>) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool on = live >> j & 1;
        copy_async<4>(slot + (lane + 32 * j) * 4, on ? row + lane + 32 * j : row, on);
      }
    } else {
      const long long left = HW - (first - tile_first);
      const int count = left < 32 * VEC ? (int)left : 32 * VEC, shift = (int)((size_t)row & 15);
      const int bytes = shift + count * (int)sizeof(IO);
      const char* from = (const char*)row - shift;
#pragma unroll
      for (int k = 0; k < (32 * VEC * (int)sizeof(IO) + 16) / 512 + 1; ++k) {
        const int at = (k * 32 + lane) * 16;
        if (at >= bytes) continue;
        if (from + at >= (const char*)all) {
          copy_pieces(slot + at, from + at, bytes - at < 16 ? bytes - at : 16);
        } else {
          for (int j = shift; j < 16 && j < bytes; j += sizeof(IO)) *(IO*)(slot + j) = *(const IO*)(from + j);
        }
      }
    }
  }
  template <typename IO>
  __device__ __forceinline__ void fetched(const char* slot, const IO* row, float* v) const {
    const int lane = threadIdx.x & 31;
    if constexpr (kOwn<IO> && ALONG) {
      Vec<IO, VEC>::load(slot, lane * VEC, v);
    } else if constexpr (kOwn<IO>) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) Vec<IO, 1>::load(slot, lane + 32 * j, v + j);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[j] = 0.f;
        if (live >> j & 1) Vec<IO, 1>::load(slot + ((size_t)row & 15), (ALONG ? lane * VEC + j : lane + 32 * j), v + j);
      }
    }
  }
  template <typename IO>
  __device__ __forceinline__ void store(void* p, long long at, const float* v) const {
    if (ALONG) {
      if (live) Vec<IO, VEC>::store(p, at, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (live >> j & 1) Vec<IO, 1>::store(p, at + 32 * j, v + j);
    }
  }
};
// block: 32 x S threads; thread (lane, s) holds channels s CPT .. of its pixels of the tile (of 32 VEC)
// Shared memory: vectors of the channels, padded to CPT; a pair of sums of each warp for each pixel; a pair for each pixel.
__host__ __device__ inline size_t cf_smem(int S, int CPT, int VEC, int vectors) {
  return (size_t)vectors * S * CPT * sizeof(float) + (S > 1 ? (size_t)(S + 1) * 32 * VEC * sizeof(float2) : 0);
}
// What a branch's normalised value is multiplied by and what is added to it on the way to y (without a gate for each element):
// scale . s(gate of the image) . (post_w, post_b).  Behind the last channel 0.
__device__ __forceinline__ float2 branch_factors(const Params& P, int c, long long image) {
  if (c >= P.C) return make_float2(0.f, 0.f);
  float a = P.scale ? P.scale[c] : 1.f;
  if (P.gate_kind == kGateImage) a *= image_gate_of(((const float*)P.gate)[image * P.C + c], P.act);
  return make_float2(P.post_w ? a * P.post_w[c] : a, P.post_b ? a * P.post_b[c] : 0.f);
}
__device__ __forceinline__ void four_of(const float* v, float (&out)[4]) {
  const float4 q = *(const float4*)v;
  out[0] = q.x; out[1] = q.y; out[2] = q.z; out[3] = q.w;
}
// Mean and 1 / spread of each pixel.  A thread brings the sum of its channels and the squares around their own mean; joined,
// M2 = sum (M2_i + (sum_i - n_i mean)^2 / n_i).  Values behind the last channel are 0.
template <int CPT, int VEC>
__device__ __forceinline__ void cf_stats(const float (&v)[CPT][VEC], int n, const Params& P, float2* red, float (&mean)[VEC],
                                         float (&rstd)[VEC]) {
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5;
  const float inv = 1.f / (float)P.C;
  float m[VEC], q[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) m[j] = q[j] = 0.f;
  if (!P.rms) {
    const float own = 1.f / (float)n;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) m[j] += v[i][j];
      const float c = m[j] * own;
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        if (i < n) q[j] = fmaf(v[i][j] - c, v[i][j] - c, q[j]);
      if (S == 1) m[j] = c;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
#pragma unroll
      for (int i = 0; i < CPT; ++i) q[j] = fmaf(v[i][j], v[i][j], q[j]);
  }
  if (S == 1) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) mean[j] = m[j], rstd[j] = rsqrtf(fmaf(q[j], inv, P.eps));
    return;
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) red[(s * VEC + j) * 32 + lane] = make_float2(m[j], q[j]);
  __syncthreads();
  float2* joined = red + S * VEC * 32;
  for (int p = threadIdx.x; p < 32 * VEC; p += blockDim.x) {
    float t = 0.f, u = 0.f;
    for (int r = 0; r < S; ++r) {
      const float2 o = red[r * VEC * 32 + p];
      t += o.x;
      u += o.y;
    }
    t *= inv;
    if (!P.rms) {
      for (int r = 0; r < S - 1; ++r) {
        const float d = fmaf(-(float)CPT, t, red[r * VEC * 32 + p].x);
        u = fmaf(d * d, 1.f / (float)CPT, u);
      }
      const float k = (float)(P.C - (S - 1) * CPT), d = fmaf(-k, t, red[(S - 1) * VEC * 32 + p].x);
      u += d * d / k;
    }
    joined[p] = make_float2(t, rsqrtf(fmaf(u, inv, P.eps)));
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float2 o = joined[j * 32 + lane];
    mean[j] = o.x;
    rstd[j] = o.y;
  }
}

template <typename IO, int CPT, int VEC, bool ALONG, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cf_fwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  extern __shared__ __align__(16) float cf_shared[];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5, padded = S * CPT;
  float *wy = cf_shared, *oy = wy + padded, *pw = oy + padded, *po = pw + padded;
  float2* red = (float2*)(po + padded);
  const int c0 = s * CPT, n = min(CPT, P.C - c0);
  const long long b = blockIdx.x / P.tiles;
  const Pixels<VEC, ALONG> px(blockIdx.x - b * P.tiles, lane, P.HW);
  const long long base = (b * P.C + c0) * P.HW + px.first, token = b * P.HW + px.first;
  float v[CPT][VEC], x[CPT][VEC];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    px.template load<IO>(P.branch, base + i * P.HW, v[i], i < n);
    px.template load<IO>(P.x, base + i * P.HW, x[i], i < n);
  }
  for (int c = threadIdx.x; c < padded; c += blockDim.x) {
    const float2 f = branch_factors(P, c, b);
    wy[c] = f.x;
    oy[c] = f.y;
    pw[c] = P.pre_w && c < P.C ? P.pre_w[c] : 0.f;
    po[c] = P.pre_b && c < P.C ? P.pre_b[c] : 0.f;
  }
  float mean[VEC], rstd[VEC], w[4], o[4];
  if (P.post_w) {
    if (S == 1) __syncthreads();
    cf_stats<CPT, VEC>(v, n, P, red, mean, rstd);
    if (P.stats && s == 0) {
      px.template store<float>(P.stats, token, mean);
      px.template store<float>(P.stats + P.tokens, token, rstd);
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = (v[i][j] - mean[j]) * rstd[j];
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (i % 4 == 0) four_of(wy + c0 + i, w), four_of(oy + c0 + i, o);
    if (P.gate_kind == kGateFull) {
      float g[VEC];
      px.template load<IO>(P.gate, base + i * P.HW, g, i < n);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(fmaf(v[i][j], w[i & 3], o[i & 3]), cf_gate_of<IO>(g[j], P.act), x[i][j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(v[i][j], w[i & 3], x[i][j] + o[i & 3]);
    }
    if (i < n) {
      px.template store<IO>(P.y, base + i * P.HW, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    }
  }
  if (!P.pre_w) return;
  cf_stats<CPT, VEC>(v, n, P, red, mean, rstd);
  if (P.stats && s == 0) {
    px.template store<float>(P.stats + 2 * P.tokens, token, mean);
    px.template store<float>(P.stats + 3 * P.tokens, token, rstd);
  }
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (i % 4 == 0) four_of(pw + c0 + i, w), four_of(po + c0 + i, o);
    if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf((v[i][j] - mean[j]) * rstd[j], w[i & 3], o[i & 3]);
      px.template store<IO>(P.z, base + i * P.HW, v[i]);
    }
  }
}

// Any number of channels: the values are read again for every step (from the L2 cache) instead of being kept.  32 warps.
template <typename IO>
__device__ __forceinline__ float cf_sum_value(const Params& P, long long at, int c, long long b, float mean, float rstd) {
  float v, x, g;
  Vec<IO, 1>::load(P.branch, at, &v);
  Vec<IO, 1>::load(P.x, at, &x);
  if (P.post_w) v = fmaf((v - mean) * rstd, P.post_w[c], P.post_b ? P.post_b[c] : 0.f);
  float a = P.scale ? P.scale[c] : 1.f;
  if (P.gate_kind == kGateImage) a *= image_gate_of(((const float*)P.gate)[b * P.C + c], P.act);
  if (P.gate_kind == kGateFull) {
    Vec<IO, 1>::load(P.gate, at, &g);
    v *= cf_gate_of<IO>(g, P.act);
  }
  return fmaf(v, a, x);
}
// the warps' sums of two values for each of the 32 pixels, in every thread
__device__ __forceinline__ float2 cf_join2(float2 own, float2* red, int S) {
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  __syncthreads();          // the values before are read
  red[s * 32 + lane] = own;
  __syncthreads();
  float2 r = make_float2(0.f, 0.f);
  for (int t = 0; t < S; ++t) r.x += red[t * 32 + lane].x, r.y += red[t * 32 + lane].y;
  return r;
}
template <typename IO>
__global__ void __launch_bounds__(1024) cf_fwd_wide_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ float2 red[32 * 32];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  const long long b = blockIdx.x / P.tiles, px = (long long)(blockIdx.x - b * P.tiles) * 32 + lane;
  const bool live = px < P.HW;
  const long long base = b * P.C * P.HW + (live ? px : P.HW - 1), token = b * P.HW + px;
  const float inv = 1.f / (float)P.C;
  float mean = 0.f, rstd = 1.f;
  if (P.post_w) {
    if (!P.rms) {
      float m = 0.f, v;
      for (int c = s; c < P.C; c += 32) {
        Vec<IO, 1>::load(P.branch, base + c * P.HW, &v);
        m += v;
      }
      mean = cf_join2(make_float2(m, 0.f), red, 32).x * inv;
    }
    float q = 0.f, v;
    for (int c = s; c < P.C; c += 32) {
      Vec<IO, 1>::load(P.branch, base + c * P.HW, &v);
      q = fmaf(v - mean, v - mean, q);
    }
    rstd = rsqrtf(fmaf(cf_join2(make_float2(q, 0.f), red, 32).x, inv, P.eps));
    if (P.stats && live && s == 0) P.stats[token] = mean, P.stats[P.tokens + token] = rstd;
  }
  // y, and its sum around its first channel
  float m = 0.f, q = 0.f;
  const float first = P.rms ? 0.f : cf_sum_value<IO>(P, base, 0, b, mean, rstd);
  for (int c = s; c < P.C; c += 32) {
    const float y = cf_sum_value<IO>(P, base + c * P.HW, c, b, mean, rstd);
    if (live) Vec<IO, 1>::store(P.y, base + c * P.HW, &y);
    m += y - first;
  }
  if (!P.pre_w) return;
  // (x is read again: y may not be kept in x's place)
  const float mean2 = P.rms ? 0.f : fmaf(cf_join2(make_float2(m, 0.f), red, 32).x, inv, first);
  for (int c = s; c < P.C; c += 32) {
    const float d = cf_sum_value<IO>(P, base + c * P.HW, c, b, mean, rstd) - mean2;
    q = fmaf(d, d, q);
  }
  const float rstd2 = rsqrtf(fmaf(cf_join2(make_float2(q, 0.f), red, 32).x, inv, P.eps));
  if (P.stats && live && s == 0) P.stats[2 * P.tokens + token] = mean2, P.stats[3 * P.tokens + token] = rstd2;
  for (int c = s; c < P.C; c += 32) {
    const float y = cf_sum_value<IO>(P, base + c * P.HW, c, b, mean, rstd);
    const float z = fmaf((y - mean2) * rstd2, P.pre_w[c], P.pre_b ? P.pre_b[c] : 0.f);
    if (live) Vec<IO, 1>::store(P.z, base + c * P.HW, &z);
  }
}

// ------------------------------------------------------------------ channels_first, backward
// The sums over the warps of two values for each pixel
template <int VEC>
__device__ __forceinline__ void cf_join(float (&a)[VEC], float (&b)[VEC], float2* red, int S) {
  if (S == 1) return;
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < VEC; ++j) red[(s * VEC + j) * 32 + lane] = make_float2(a[j], b[j]);
  __syncthreads();
  float2* joined = red + S * VEC * 32;
  for (int p = threadIdx.x; p < 32 * VEC; p += blockDim.x) {
    float2 t = red[p];
    for (int r = 1; r < S; ++r) {
      const float2 o = red[r * VEC * 32 + p];
      t.x += o.x;
      t.y += o.y;
    }
    joined[p] = t;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float2 o = joined[j * 32 + lane];
    a[j] = o.x;
    b[j] = o.y;
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// `parts` blocks walk over all images' tiles, or over those of an image where the gate has a value for each image
template <typename IO, int CPT, int VEC, bool ALONG, bool GATED, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cf_bwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  extern __shared__ __align__(16) float cf_shared[];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5, padded = S * CPT;
  float *wy = cf_shared, *oy = wy + padded, *pw = oy + padded;
  float2* red = (float2*)(pw + padded);
  using Px = Pixels<VEC, ALONG>;
  // dz, x, branch, the gate of an element, dy of the next tile: CPT slots each; its means and spreads: four (fp32)
  constexpr int TENSORS = GATED ? 5 : 4, DY = TENSORS - 1;
  constexpr int SLOT = Px::template kSlot<IO>, STAT = Px::template kSlot<float>;
  char* const slots = (char*)(red + (S > 1 ? (S + 1) * 32 * VEC : 0)) + s * (TENSORS * CPT * SLOT + 4 * STAT);          // this warp's
  char* const stats = slots + TENSORS * CPT * SLOT;
  const int c0 = s * CPT, n = min(CPT, P.C - c0);
  const float inv = 1.f / (float)P.C;
  float sa[CPT], sb[CPT], sw[CPT], so[CPT];       // sums A, B; dz k, dz
#pragma unroll
  for (int i = 0; i < CPT; ++i) sa[i] = sb[i] = sw[i] = so[i] = 0.f;
  const bool image = P.gate_kind == kGateImage, act = GATED && P.act;
  const int one = act ? kOne : 0;
  const unsigned of = image ? blockIdx.x / P.parts : 0, first = of * P.tiles, last = image ? first + P.tiles : (unsigned)(P.tiles * P.B);
  for (int c = threadIdx.x; c < padded; c += blockDim.x) {
    const float2 f = branch_factors(P, c, of);
    wy[c] = f.x;
    oy[c] = f.y;
    pw[c] = P.pre_w && c < P.C ? P.pre_w[c] : 0.f;
  }
  __syncthreads();
  auto begin = [&](unsigned tile, int from, int to) {
    if (tile >= last) return;
    const unsigned b = tile / (unsigned)P.tiles;
    const Px px(tile - b * P.tiles, lane, P.HW);
    const long long at = ((long long)b * P.C + c0) * P.HW + (long long)(tile - b * P.tiles) * (32 * VEC);
    const void* all[5] = {P.dz, P.dz ? P.x : nullptr, P.branch, GATED ? P.gate : P.dy, P.dy};
    __syncwarp();          // (pieces: what was there is read)
#pragma unroll
    for (int a = 0; a < TENSORS; ++a)
      if (a >= from && a < to && all[a]) {
        const IO* row = (const IO*)all[a] + at;
#pragma unroll
        for (int i = 0; i < CPT; ++i)
          if (i < n) {
            px.template fetch<IO>(slots + (a * CPT + i) * SLOT, (const IO*)all[a], row, P.HW);
            row += P.HW;
          }
      }
    if (from == 0 && P.stats) {
      const float* row = P.stats + (long long)b * P.HW + (long long)(tile - b * P.tiles) * (32 * VEC);
#pragma unroll
      for (int a = 0; a < 4; ++a)
        if (a < 2 ? P.post_w != nullptr : P.dz != nullptr) px.template fetch<float>(stats + a * STAT, P.stats, row + a * P.tokens, P.HW);
    }
  };
  auto get = [&](const Px& px, int a, int i, const void* p, long long row, float (&v)[VEC]) {
    if (!p || i >= n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    } else {
      px.template fetched<IO>(slots + (a * CPT + i) * SLOT, (const IO*)p + row, v);
    }
  };
  auto stat = [&](const Px& px, int a, long long row, float (&v)[VEC]) {
    px.template fetched<float>(stats + a * STAT, P.stats + a * P.tokens + row, v);
  };
  begin(first + blockIdx.x % P.parts, 0, TENSORS);
  for (unsigned tile = first + blockIdx.x % P.parts; tile < last; tile += P.parts) {
    const unsigned b = tile / (unsigned)P.tiles;
    const Px px(tile - b * P.tiles, lane, P.HW);
    const long long tile_at = (long long)(tile - b * P.tiles) * (32 * VEC), row = ((long long)b * P.C + c0) * P.HW + tile_at;
    const long long base = ((long long)b * P.C + c0) * P.HW + px.first, token_row = (long long)b * P.HW + tile_at;
    float d[CPT][VEC], k[CPT][VEC], h[CPT][VEC], f[GATED ? CPT : 1][VEC];          // f: the gate of an element
    float mean[VEC], rstd[VEC], u[VEC], w[VEC], vec[4], add[4];
    copies_done();
    if (!Px::template kOwn<IO>) __syncwarp();
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      get(px, 0, i, P.dz, row + i * P.HW, d[i]);
      get(px, 1, i, P.dz ? P.x : nullptr, row + i * P.HW, k[i]);
      get(px, 2, i, P.branch, row + i * P.HW, h[i]);
      if constexpr (GATED) get(px, 3, i, P.gate, row + i * P.HW, f[i]);
    }
    float mk[VEC], rk[VEC];
    if (P.dz) {
      stat(px, 2, token_row, mk);
      stat(px, 3, token_row, rk);
    }
    if (P.post_w) {
      stat(px, 0, token_row, mean);
      stat(px, 1, token_row, rstd);
    }
    begin(tile + P.parts, 0, DY);
    if (P.post_w) {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = i < n ? (h[i][j] - mean[j]) * rstd[j] : 0.f;
    }
    if (P.dz) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        if (i % 4 == 0) four_of(wy + c0 + i, vec), four_of(oy + c0 + i, add);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {        // y again, as it was before it was rounded
          if constexpr (GATED) k[i][j] = fmaf(fmaf(h[i][j], vec[i & 3], add[i & 3]), act ? sigmoid_hold<IO>(f[i][j]) : f[i][j], k[i][j]) - mk[j];
          else k[i][j] = fmaf(h[i][j], vec[i & 3], k[i][j] + add[i & 3]) - mk[j];
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[j] = w[j] = 0.f;
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        if (i % 4 == 0) four_of(pw + c0 + i, vec);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {        // (dz is 0 behind the last pixel and channel, and so are the sums)
          k[i][j] *= rk[j];
          so[i] += d[i][j];
          sw[i] = fmaf(d[i][j], k[i][j], sw[i]);
          d[i][j] *= vec[i & 3];
          u[j] += d[i][j];
          w[j] = fmaf(d[i][j], k[i][j], w[j]);
        }
      }
      cf_join<VEC>(u, w, red, S);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u[j] = P.rms ? 0.f : u[j] * inv;
        w[j] *= inv;
      }
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[i][j] = rk[j] * (d[i][j] - fmaf(k[i][j], w[j], u[j]));
    } else if (GATED && act) {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sigmoid_hold<IO>(f[GATED ? i : 0][j]);
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      if (P.dy) {
        float e[VEC];
        get(px, DY, i, P.dy, row + i * P.HW, e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[i][j] += e[j];
      }
      if (i < n) {
        if (P.dx) px.template store<IO>(P.dx, base + i * P.HW, d[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[i][j] = 0.f;
      }
    }
    begin(tile + P.parts, DY, TENSORS);
    if (!P.branch) continue;
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        if (i % 4 == 0) four_of(wy + c0 + i, vec), four_of(oy + c0 + i, add);
        if (i < n && P.dgate) {
          float dg[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) dg[j] = d[i][j] * fmaf(h[i][j], vec[i & 3], add[i & 3]) * gate_slope(f[i][j], act);
          px.template store<IO>(P.dgate, base + i * P.HW, dg);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[i][j] *= gate_factor(f[i][j], one);
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[j] = w[j] = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      if (i % 4 == 0) four_of(wy + c0 + i, vec);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {          // (an image's sums are without its gate, which is in vec)
        sb[i] += d[i][j];
        sa[i] = fmaf(d[i][j], h[i][j], sa[i]);
        d[i][j] *= vec[i & 3];
        u[j] += d[i][j];
        w[j] = fmaf(d[i][j], h[i][j], w[j]);
      }
    }
    if (!P.dbranch) continue;
    if (P.post_w) {
      cf_join<VEC>(u, w, red, S);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u[j] = P.rms ? 0.f : u[j] * inv;
        w[j] *= inv;
      }
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (i < n) {
        if (P.post_w) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) d[i][j] = rstd[j] * (d[i][j] - fmaf(h[i][j], w[j], u[j]));
        }
        px.template store<IO>(P.dbranch, base + i * P.HW, d[i]);
      }
  }
  copies_done();
  if (!P.partial) return;
  float* out = P.partial + (long long)blockIdx.x * 4 * P.C;
#pragma unroll
  for (int i = 0; i < CPT; ++i)
    if (i < n) {        // (the same for the whole warp)
      const float q0 = warp_sum(sa[i]), q1 = warp_sum(sb[i]), q2 = warp_sum(sw[i]), q3 = warp_sum(so[i]);
      const float q = lane == 0 ? q0 : lane == 1 ? q1 : lane == 2 ? q2 : q3;
      if (lane < 4) out[lane * P.C + c0 + i] = q;
    }
}

// Any number of channels: values are read again for every step, a warp's sums over its 32 pixels are added to shared memory
// (4 C floats: each channel belongs to one warp), tile after tile.
template <typename IO>
__global__ void __launch_bounds__(1024) cf_bwd_wide_kernel(const __grid_constant__ Params P) {
  pdl_start();
  extern __shared__ float2 red[];
  float* sums = (float*)(red + 32 * 32);
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  const float inv = 1.f / (float)P.C;
  for (int i = threadIdx.x; i < 4 * P.C; i += 1024) sums[i] = 0.f;
  __syncthreads();
  const bool image = P.gate_kind == kGateImage;
  const long long first = image ? (long long)(blockIdx.x / P.parts) * P.tiles : 0, last = image ? first + P.tiles : (long long)P.tiles * P.B;
  for (long long tile = first + blockIdx.x % P.parts; tile < last; tile += P.parts) {
    const long long b = tile / P.tiles, px = (tile - b * P.tiles) * 32 + lane;
    const bool live = px < P.HW;
    const long long base = b * P.C * P.HW + (live ? px : P.HW - 1), token = b * P.HW + (live ? px : P.HW - 1);
    float mk = 0.f, rk = 1.f, mh = 0.f, rh = 1.f, v;
    float2 pre = make_float2(0.f, 0.f), post = make_float2(0.f, 0.f);
    if (P.post_w) mh = P.stats[token], rh = P.stats[P.tokens + token];
    // the normalised y, from y as it was before it was rounded
    auto normed = [&](int c) { return (cf_sum_value<IO>(P, base + c * P.HW, c, b, mh, rh) - mk) * rk; };
    if (P.dz) {
      mk = P.stats[2 * P.tokens + token];
      rk = P.stats[3 * P.tokens + token];
      for (int c = s; c < P.C; c += 32) {
        Vec<IO, 1>::load(P.dz, base + c * P.HW, &v);
        const float k = normed(c), t = v * P.pre_w[c];
        pre.x += t;
        pre.y = fmaf(t, k, pre.y);
        const float q0 = warp_sum(live ? v * k : 0.f), q1 = warp_sum(live ? v : 0.f);
        if (lane == 0) sums[2 * P.C + c] += q0, sums[3 * P.C + c] += q1;
      }
      pre = cf_join2(pre, red, 32);
      pre.x = P.rms ? 0.f : pre.x * inv;
      pre.y *= inv;
    }
    auto total = [&](int c) {          // dL/dy
      float d = 0.f;
      if (P.dz) {
        float v;
        Vec<IO, 1>::load(P.dz, base + c * P.HW, &v);
        d = rk * (v * P.pre_w[c] - pre.x - normed(c) * pre.y);
      }
      if (P.dy) {
        float e;
        Vec<IO, 1>::load(P.dy, base + c * P.HW, &e);
        d += e;
      }
      return d;
    };
    auto factor = [&](int c, float g) {    // what takes it to the normalised branch
      float a = P.scale ? P.scale[c] : 1.f;
      if (image) a *= image_gate_of(((const float*)P.gate)[b * P.C + c], P.act);
      if (P.gate_kind == kGateFull) a *= g;
      return P.post_w ? a * P.post_w[c] : a;
    };
    for (int c = s; c < P.C; c += 32) {
      const float d = total(c);
      if (live && P.dx) Vec<IO, 1>::store(P.dx, base + c * P.HW, &d);
      if (!P.branch) continue;
      float h, g = 1.f;
      Vec<IO, 1>::load(P.branch, base + c * P.HW, &h);
      h = (h - mh) * rh;
      if (P.gate_kind == kGateFull) {
        Vec<IO, 1>::load(P.gate, base + c * P.HW, &g);
        float held = g;
        if (P.act) g = sigmoid_hold<IO>(held);
        if (live && P.dgate) {
          const float pw = P.post_w ? P.post_w[c] : 1.f, pb = P.post_b ? P.post_b[c] : 0.f;
          const float dg = d * (P.scale ? P.scale[c] : 1.f) * fmaf(h, pw, pb) * gate_slope(held, P.act);
          Vec<IO, 1>::store(P.dgate, base + c * P.HW, &dg);
        }
      }
      const float q0 = warp_sum(live ? d * g * h : 0.f), q1 = warp_sum(live ? d * g : 0.f);
      if (lane == 0) sums[c] += q0, sums[P.C + c] += q1;
      const float t = d * factor(c, g);
      post.x += t;
      post.y = fmaf(t, h, post.y);
    }
    if (!P.branch || !P.dbranch) continue;
    if (P.post_w) {
      post = cf_join2(post, red, 32);
      post.x = P.rms ? 0.f : post.x * inv;
      post.y *= inv;
    }
    for (int c = s; c < P.C; c += 32) {
      float g = 1.f, h;
      if (P.gate_kind == kGateFull) {
        Vec<IO, 1>::load(P.gate, base + c * P.HW, &g);
        g = cf_gate_of<IO>(g, P.act);
      }
      float t = total(c) * factor(c, g);
      if (P.post_w) {
        Vec<IO, 1>::load(P.branch, base + c * P.HW, &h);
        t = rh * (t - post.x - (h - mh) * rh * post.y);
      }
      if (live) Vec<IO, 1>::store(P.dbranch, base + c * P.HW, &t);
    }
  }
  if (!P.partial) return;
  __syncthreads();
  float* out = P.partial + (long long)blockIdx.x * 4 * P.C;
  for (int i = threadIdx.x; i < 4 * P.C; i += 1024) out[i] = sums[i];
}

// ------------------------------------------------------------------ channels_last
// `tpr` threads (a power of two) share a token: thread t holds the vectors t, t + tpr, ... of its channels.
// Sums over the token's threads.  Tokens of more than a warp meet in `red` (twice 32 values of the block): `buf` alternates, since
// the values of the sum before the last have been read by everybody who arrived at the last one.
template <int N>
__device__ __forceinline__ void cl_sum(float (&v)[N], int tpr, float2* red, int& buf) {
  if (tpr >= 32) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
  } else {
    for (int o = tpr >> 1; o; o >>= 1)
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
  }
  if (tpr <= 32) return;
  float2* r = red + 32 * buf;
  buf ^= 1;
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = make_float2(v[0], v[N - 1]);
  __syncthreads();
  r += (threadIdx.x & ~(tpr - 1)) >> 5;
  float2 t = r[0];
  for (int j = 1; j < (tpr >> 5); ++j) t.x += r[j].x, t.y += r[j].y;
  v[0] = t.x;
  if (N == 2) v[1] = t.y;
}
template <int NV, int V>
__device__ __forceinline__ void cl_stats(const float (&v)[NV][V], const Params& P, int tpr, int t, float2* red, int& buf, float& mean,
                                         float& rstd) {
  const float inv = 1.f / (float)P.C;
  float m = 0.f, q = 0.f;
  mean = 0.f;
  if (!P.rms) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) m += v[i][j];          // (zeros behind the last channel)
    float all[1] = {m};
    cl_sum(all, tpr, red, buf);
    mean = all[0] * inv;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * tpr + t) * V < P.C) {
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(v[i][j] - mean, v[i][j] - mean, q);
    }
  float all[1] = {q};
  cl_sum(all, tpr, red, buf);
  rstd = rsqrtf(fmaf(all[0], inv, P.eps));
}
template <int V>
__device__ __forceinline__ void cl_vector(const float* p, int c, float other, float (&v)[V]) {
  if (p) {
    if constexpr (V == 8) {
      Vec<float, 4>::load(p, c, v);
      Vec<float, 4>::load(p, c + 4, v + 4);
    } else {
      Vec<float, V>::load(p, c, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = other;
  }
}

// the factors of branch_factors for V channels (a gate of each image apart)
template <int V>
__device__ __forceinline__ void cl_factors(const Params& P, int c, float (&w)[V], float (&o)[V]) {
  float a[V];
  cl_vector<V>(P.scale, c, 1.f, a);
  cl_vector<V>(P.post_w, c, 1.f, w);
  cl_vector<V>(P.post_b, c, 0.f, o);
#pragma unroll
  for (int j = 0; j < V; ++j) w[j] *= a[j], o[j] *= a[j];
}

// Blocks walk over tokens with the vectors of their channels in registers; the next token's values are loaded before this one's
// norms are known.
template <typename IO, int NV, int V, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cl_fwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ float2 red[64];
  int buf = 0;
  const int tpr = P.tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x / tpr;
  float wy[NV][V], oy[NV][V], pw[NV][V], po[NV][V], v[NV][V], x[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) wy[i][j] = oy[i][j] = pw[i][j] = po[i][j] = 0.f;
    if (c >= P.C) continue;
    cl_factors<V>(P, c, wy[i], oy[i]);
    if (P.pre_w) {
      cl_vector<V>(P.pre_w, c, 1.f, pw[i]);
      cl_vector<V>(P.pre_b, c, 0.f, po[i]);
    }
  }
  auto fetch = [&](long long token) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (token < P.tokens && c < P.C) {
        Vec<IO, V>::load(P.branch, token * P.C + c, v[i]);
        Vec<IO, V>::load(P.x, token * P.C + c, x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = x[i][j] = 0.f;
      }
    }
  };
  const long long step = (long long)gridDim.x * rows;
  long long start = (long long)blockIdx.x * rows;
  fetch(start + threadIdx.x / tpr);
  for (; start < P.tokens; start += step) {
    const long long token = start + threadIdx.x / tpr, base = token * P.C;
    const bool live = token < P.tokens;
    float mean = 0.f, rstd = 1.f, y[NV][V];
    if (P.post_w) {
      cl_stats<NV, V>(v, P, tpr, t, red, buf, mean, rstd);
      if (P.stats && live && t == 0) P.stats[token] = mean, P.stats[P.tokens + token] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c < P.C && live) {
        // (each way as the backward forms y again: where a token has one channel, y - mean has to be 0 there too)
        float g[V];
        if (P.gate_kind == kGateImage) {
          cl_vector<V>((const float*)P.gate + token / P.HW * P.C, c, 0.f, g);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            g[j] = image_gate_of(g[j], P.act);
            y[i][j] = fmaf((v[i][j] - mean) * rstd, wy[i][j] * g[j], oy[i][j] * g[j]) + x[i][j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] = 1.f;
          if (P.gate_kind == kGateFull) {
            Vec<IO, V>::load(P.gate, base + c, g);
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = cl_gate_of<IO>(g[j], P.act);
          }
#pragma unroll
          for (int j = 0; j < V; ++j) y[i][j] = fmaf(fmaf((v[i][j] - mean) * rstd, wy[i][j], oy[i][j]), g[j], x[i][j]);
        }
        Vec<IO, V>::store(P.y, base + c, y[i]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) y[i][j] = 0.f;
      }
    }
    fetch(token + step);
    if (!P.pre_w) continue;
    cl_stats<NV, V>(y, P, tpr, t, red, buf, mean, rstd);
    if (!live) continue;
    if (P.stats && t == 0) P.stats[2 * P.tokens + token] = mean, P.stats[3 * P.tokens + token] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c >= P.C) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) y[i][j] = fmaf((y[i][j] - mean) * rstd, pw[i][j], po[i][j]);
      Vec<IO, V>::store(P.z, base + c, y[i]);
    }
  }
}

template <typename IO, int NV, int V>
__host__ __device__ constexpr bool cl_async() { return V * sizeof(IO) >= 4 && NV * V * sizeof(IO) <= 32; }

template <typename IO, int NV, int V, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cl_bwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  int buf = 0;
  // 64 pairs for the sums; dz, x, branch, gate, dy of the next token, in the end 4 C floats for each warp, or each token of more than a
  // warp
  extern __shared__ __align__(16) char cl_dynamic[];
  float2* const red = (float2*)cl_dynamic;
  char* const cl_shared = cl_dynamic + 64 * sizeof(float2);
  constexpr int BYTES = V * sizeof(IO), SLOT = MAXT * BYTES;
  constexpr bool ASYNC = cl_async<IO, NV, V>();
  const int tpr = P.tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x / tpr, row = threadIdx.x / tpr;
  const float inv = 1.f / (float)P.C;
  const bool image = P.gate_kind == kGateImage;
  const bool act = P.gate_kind == kGateFull && P.act;
  const int one = act ? kOne : 0;
  const long long of = blockIdx.x / P.parts, first = image ? of * P.HW : 0, last = image ? first + P.HW : P.tokens;
  float sa[NV][V], sb[NV][V], sw[NV][V], so[NV][V], wy[NV][V], oy[NV][V], pw[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) sa[i][j] = sb[i][j] = sw[i][j] = so[i][j] = wy[i][j] = oy[i][j] = pw[i][j] = 0.f;
    if (c >= P.C) continue;
    cl_factors<V>(P, c, wy[i], oy[i]);
    if (P.pre_w) cl_vector<V>(P.pre_w, c, 1.f, pw[i]);
    if (image) {
      float g[V];
      cl_vector<V>((const float*)P.gate + of * P.C, c, 0.f, g);
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = image_gate_of(g[j], P.act), wy[i][j] *= g[j], oy[i][j] *= g[j];
    }
  }
  const long long step = (long long)P.parts * rows;
  long long start = first + (long long)(blockIdx.x % P.parts) * rows;
  float stat[4];          // means and spreads of the next token
  auto begin = [&](long long token) {
    const bool live = token < last;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      stat[a] = a & 1 ? 1.f : 0.f;
      if (live && (a < 2 ? P.post_w != nullptr : P.dz != nullptr)) stat[a] = P.stats[a * P.tokens + token];
    }
    if constexpr (ASYNC) {
      const void* all[5] = {P.dz, P.dz ? P.x : nullptr, P.branch, P.gate_kind == kGateFull ? P.gate : nullptr, P.dy};
#pragma unroll
      for (int a = 0; a < 5; ++a)
        if (all[a]) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + t) * V;
            const bool on = live && c < P.C;
            copy_async<BYTES>(cl_shared + (a * NV + i) * SLOT + threadIdx.x * BYTES, (const IO*)all[a] + (on ? token * P.C + c : 0), on);
          }
        }
    }
  };
  auto get = [&](int a, int i, const void* p, long long at, bool on, float (&v)[V]) {
    if (!p || !on) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
    } else if constexpr (ASYNC) {
      Vec<IO, V>::load(cl_shared + (a * NV + i) * SLOT, threadIdx.x * V, v);
    } else {
      Vec<IO, V>::load(p, at, v);
    }
  };
  begin(start + row);
  for (; start < last; start += step) {
    const long long token = start + row;
    const bool live = token < last;
    const long long base = token * P.C;
    float d[NV][V], k[NV][V], h[NV][V], f[NV][V], e[NV][V];          // f: the gate; e: dy
    const float mean = stat[0], rstd = stat[1], mk = stat[2], rk = stat[3];
    if (ASYNC) copies_done();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      const bool on = live && c < P.C;
      get(0, i, P.dz, base + c, on, d[i]);
      get(1, i, P.dz ? P.x : nullptr, base + c, on, k[i]);
      get(2, i, P.branch, base + c, on, h[i]);
      get(4, i, P.dy, base + c, on, e[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] = on ? (h[i][j] - mean) * rstd : 0.f, f[i][j] = 1.f;
      if (P.gate_kind == kGateFull) {
        get(3, i, P.gate, base + c, on, f[i]);
        if (act) {
#pragma unroll
          for (int j = 0; j < V; ++j) sigmoid_hold<IO>(f[i][j]);
        }
      }
    }
    begin(token + step);
    if (P.dz) {
      float u[2] = {0.f, 0.f};
      // y again, as it was before it was rounded
      if (act) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) k[i][j] = fmaf(fmaf(h[i][j], wy[i][j], oy[i][j]), gate_factor(f[i][j], one), k[i][j]);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) k[i][j] = fmaf(fmaf(h[i][j], wy[i][j], oy[i][j]), f[i][j], k[i][j]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {          // (dz is 0 behind the last token and channel, and so are the sums)
          k[i][j] = (k[i][j] - mk) * rk;
          so[i][j] += d[i][j];
          sw[i][j] = fmaf(d[i][j], k[i][j], sw[i][j]);
          d[i][j] *= pw[i][j];
          u[0] += d[i][j];
          u[1] = fmaf(d[i][j], k[i][j], u[1]);
        }
      cl_sum(u, tpr, red, buf);
      u[0] = P.rms ? 0.f : u[0] * inv;
      u[1] *= inv;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = rk * (d[i][j] - u[0] - k[i][j] * u[1]);
    }
    float u[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c >= P.C || !live) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) d[i][j] += e[i][j];
      if (P.dx) Vec<IO, V>::store(P.dx, base + c, d[i]);
      if (!P.branch) continue;
      if (P.gate_kind == kGateFull) {
        if (P.dgate) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = d[i][j] * fmaf(h[i][j], wy[i][j], oy[i][j]) * gate_slope(f[i][j], act);
          Vec<IO, V>::store(P.dgate, base + c, o);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] *= gate_factor(f[i][j], one);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {          // (an image's sums are without its gate, which is in wy)
        sb[i][j] += d[i][j];
        sa[i][j] = fmaf(d[i][j], h[i][j], sa[i][j]);
        d[i][j] *= wy[i][j];
        u[0] += d[i][j];
        u[1] = fmaf(d[i][j], h[i][j], u[1]);
      }
    }
    if (!P.dbranch) continue;
    if (P.post_w) {
      cl_sum(u, tpr, red, buf);
      u[0] = P.rms ? 0.f : u[0] * inv;
      u[1] *= inv;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c >= P.C || !live) continue;
      if (P.post_w) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = rstd * (d[i][j] - u[0] - h[i][j] * u[1]);
      }
      Vec<IO, V>::store(P.dbranch, base + c, d[i]);
    }
  }
  if (!P.partial) return;
  float* out = P.partial + (long long)blockIdx.x * 4 * P.C;
  const int slots = blockDim.x / (tpr > 32 ? tpr : 32);
  float* const joined = (float*)cl_shared;
  float* own = slots > 1 ? joined + (threadIdx.x / (tpr > 32 ? tpr : 32)) * 4 * P.C : out;
  if (ASYNC) copies_done();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int o = 16; o >= tpr; o >>= 1) {          // the warp's other tokens
        sa[i][j] += __shfl_xor_sync(0xffffffffu, sa[i][j], o);
        sb[i][j] += __shfl_xor_sync(0xffffffffu, sb[i][j], o);
        sw[i][j] += __shfl_xor_sync(0xffffffffu, sw[i][j], o);
        so[i][j] += __shfl_xor_sync(0xffffffffu, so[i][j], o);
      }
      if (c + j < P.C && (tpr > 32 || (threadIdx.x & 31) < tpr)) {
        own[c + j] = sa[i][j];
        own[P.C + c + j] = sb[i][j];
        own[2 * P.C + c + j] = sw[i][j];
        own[3 * P.C + c + j] = so[i][j];
      }
    }
  }
  if (slots == 1) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * P.C; i += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < slots; ++w) v += joined[w * 4 * P.C + i];
    out[i] = v;
  }
}

// ------------------------------------------------------------------ the parameters' gradients from the partial sums
// grid: (groups of 32 channels, 2): the sums A, B and what follows from them; the sums of dz
__global__ void __launch_bounds__(1024) finish_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ double red[32][33][2];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  int c = blockIdx.x * 32 + lane;
  const bool pre = blockIdx.y == 1;
  const int images = P.gate_kind == kGateImage ? (int)P.B : 1;
  float a = P.scale && c < P.C ? P.scale[c] : 1.f, w = P.post_w && c < P.C ? P.post_w[c] : 1.f;
  float o = P.post_b && c < P.C ? P.post_b[c] : 0.f;
  // `share` of the 32 rows of threads add up an image, the others other images
  int share = 32;
  while (share > 1 && images > 32 / share) share >>= 1;
  double t0 = 0, t1 = 0;
  for (int round = 0; round < images; round += 32 / share) {
    const int b = round + s / share;
    double u0 = 0, u1 = 0;
    if (c < P.C && b < images) {
      const float* from = P.partial + (long long)b * P.parts * 4 * P.C + (pre ? 2 * P.C : 0) + c;
#pragma unroll 4
      for (int r = s % share; r < P.parts; r += share) {
        u0 += (double)from[(long long)r * 4 * P.C];
        u1 += (double)from[(long long)r * 4 * P.C + P.C];
      }
    }
    if (share > 1) {
      red[s][lane][0] = u0;
      red[s][lane][1] = u1;
      __syncthreads();
      if (s % share == 0)
        for (int r = 1; r < share; ++r) u0 += red[s + r][lane][0], u1 += red[s + r][lane][1];
      __syncthreads();
      if (s % share) u0 = u1 = 0;
    }
    if (P.gate_kind == kGateImage && !pre && c < P.C && b < images && s % share == 0) {
      const float held = ((const float*)P.gate)[(long long)b * P.C + c], g = image_gate_of(held, P.act);
      if (P.dgate) ((float*)P.dgate)[(long long)b * P.C + c] = (float)(a * (w * u0 + o * u1) * image_gate_slope(held, P.act));
      u0 *= g;
      u1 *= g;
    }
    t0 += u0;
    t1 += u1;
  }
  // warp s finishes channel s of the 32
  red[s][lane][0] = t0;
  red[s][lane][1] = t1;
  __syncthreads();
  t0 = red[lane][s][0];
  t1 = red[lane][s][1];
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    t0 += __shfl_xor_sync(0xffffffffu, t0, m);
    t1 += __shfl_xor_sync(0xffffffffu, t1, m);
  }
  c = blockIdx.x * 32 + s;
  if (lane != 0 || c >= P.C) return;
  a = P.scale ? P.scale[c] : 1.f;
  w = P.post_w ? P.post_w[c] : 1.f;
  o = P.post_b ? P.post_b[c] : 0.f;
  if (pre) {
    if (P.dpre_w) P.dpre_w[c] = (float)t0;
    if (P.dpre_b) P.dpre_b[c] = (float)t1;
  } else {
    if (P.dpost_w) P.dpost_w[c] = (float)(a * t0);
    if (P.dpost_b) P.dpost_b[c] = (float)(a * t1);
    if (P.dscale) P.dscale[c] = (float)(w * t0 + o * t1);
  }
}

// ------------------------------------------------------------------ launches
static bool aligned(const Params& P, size_t to) {
  const void* all[] = {P.x, P.branch, P.gate_kind == kGateFull ? P.gate : nullptr, P.y, P.z, P.dy, P.dz, P.dx, P.dbranch,
                       P.gate_kind == kGateFull ? P.dgate : nullptr};
  for (const void* p : all)
    if ((size_t)p % to) return false;
  return true;
}
// pixels of a thread as vectors of each tensor, and of the means and spreads
template <typename IO>
static bool pixels_aligned(const Params& P, int pixels) {
  return P.HW % pixels == 0 && aligned(P, pixels * sizeof(IO)) && (size_t)P.stats % (pixels * sizeof(float)) == 0;
}
static bool vectors_aligned(const Params& P) {
  const void* all[] = {P.scale, P.post_w, P.post_b, P.pre_w, P.pre_b, P.gate_kind == kGateImage ? P.gate : nullptr};
  for (const void* p : all)
    if ((size_t)p % 16) return false;
  return true;
}
static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

template <typename IO, int CPT, int VEC, bool ALONG, int MAXT, int MINB>
static int cf_fwd(Params& P, cudaStream_t st) {
  const int S = ceil_div(P.C, CPT);
  P.tiles = ceil_div(P.HW, 32 * VEC);
  const size_t smem = cf_smem(S, CPT, VEC, 4);
  const int rc = allow_smem(cf_fwd_kernel<IO, CPT, VEC, ALONG, MAXT, MINB>, smem);
  if (rc != CVB_OK) return rc;
  return launch_chained(cf_fwd_kernel<IO, CPT, VEC, ALONG, MAXT, MINB>, dim3((unsigned)(P.tiles * P.B)), 32 * S, smem, st, P);
}
template <typename IO>
static int cf_fwd_any(Params& P, int sms, cudaStream_t st) {
  // Several pixels a thread where that still gives half of the SMs a block, as vectors where rows allow it; else one.  Four of up
  // to 64 channels (two blocks an SM).  Up to 96 two, with two blocks of 384 threads (4 x 96 x 65536 fp32: 79 us, four pixels 92);
  // up to 128 four as vectors (118 us, two 114; bf16 102 and 107), two where they are 32 apart (bf16 120 us, four 161).
  const bool several = P.tokens >= (long long)64 * sms;
  const bool along2 = pixels_aligned<IO>(P, 2), along4 = pixels_aligned<IO>(P, 4);
  if (P.C <= 64 && several) return along4 ? cf_fwd<IO, 8, 4, true, 256, 2>(P, st) : cf_fwd<IO, 8, 4, false, 256, 2>(P, st);
  if (P.C <= 96 && several) return along2 ? cf_fwd<IO, 8, 2, true, 384, 2>(P, st) : cf_fwd<IO, 8, 2, false, 384, 2>(P, st);
  if (P.C <= 128 && several) return along4 ? cf_fwd<IO, 8, 4, true, 512, 1>(P, st) : cf_fwd<IO, 8, 2, false, 512, 2>(P, st);
  // Up to 256 sixteen channels a thread: two pixels as vectors (4 x 256 x 16384 fp32 66 us; one pixel in two blocks of 512 threads 78;
  // eight channels in one block of 1024 99), or one where rows allow none (5 x 184 x 18221 bf16 97 us, two pixels 118, eight channels 130)
  if (P.C <= 256 && several) return along2 ? cf_fwd<IO, 16, 2, true, 512, 1>(P, st) : cf_fwd<IO, 16, 1, true, 512, 2>(P, st);
  if (P.C <= 256) return cf_fwd<IO, 8, 1, true, 1024, 1>(P, st);
  if (P.C <= 1024) return cf_fwd<IO, 32, 1, true, 1024, 1>(P, st);
  P.tiles = ceil_div(P.HW, 32);
  return launch_chained(cf_fwd_wide_kernel<IO>, dim3((unsigned)(P.tiles * P.B)), 1024, 0, st, P);
}
template <typename IO, int NV, int V, int MAXT, int MINB>
static int cl_fwd(Params& P, int sms, cudaStream_t st) {
  int tpr = 4;
  while (tpr * NV * V < P.C) tpr *= 2;
  const int threads = tpr > 256 ? tpr : 256;
  P.tpr = tpr;
  const int blocks = ceil_div(P.tokens, threads / tpr);
  return launch_chained(cl_fwd_kernel<IO, NV, V, MAXT, MINB>, dim3((unsigned)min(blocks, MINB * sms)), threads, 0, st, P);
}
// Elements that a thread reads and writes at once: 16 bytes, pairs, or single ones, as rows and addresses allow
template <typename IO>
static int cl_width(const Params& P) {
  constexpr int V = 16 / (int)sizeof(IO);
  if (P.C % V == 0 && aligned(P, 16) && vectors_aligned(P)) return V;
  return P.C % 2 == 0 && aligned(P, 2 * sizeof(IO)) && vectors_aligned(P) ? 2 : 1;
}
template <typename IO, int V>
static int cl_fwd_by_size(Params& P, int sms, cudaStream_t st) {
  if (P.C <= 2048) return cl_fwd<IO, 8 / V, V, 256, sizeof(IO) == 2 && V == 8 ? 4 : 3>(P, sms, st);
  if (P.C <= 4096) return cl_fwd<IO, 8 / V, V, 512, 1>(P, sms, st);
  return cl_fwd<IO, 16 / V, V, 1024, 1>(P, sms, st);
}
template <typename IO>
static int cl_fwd_any(Params& P, int sms, cudaStream_t st) {
  const int width = cl_width<IO>(P);
  return width == 1 ? cl_fwd_by_size<IO, 1>(P, sms, st)
         : width == 2 ? cl_fwd_by_size<IO, 2>(P, sms, st)
                      : cl_fwd_by_size<IO, 16 / (int)sizeof(IO)>(P, sms, st);
}

int run_fwd(Params& P, int io, int sms, cudaStream_t st) {
  if (P.first) return io == CVB_F32 ? cf_fwd_any<float>(P, sms, st) : cf_fwd_any<__nv_bfloat16>(P, sms, st);
  return io == CVB_F32 ? cl_fwd_any<float>(P, sms, st) : cl_fwd_any<__nv_bfloat16>(P, sms, st);
}

// Blocks of the backward kernel that add into sums of their own, for each image where the gate has a value for each image.
static int parts_of(const Params& P, long long units, int resident) {
  const long long images = P.gate_kind == kGateImage ? P.B : 1;
  long long n = (resident + images - 1) / images;
  const long long each = P.gate_kind == kGateImage ? units : units * (P.first ? P.B : 1);
  if (n > each) n = each;
  return (int)(n < 1 ? 1 : n);
}
constexpr int kWideChannels = 4096;       // channels_first: 64 KB of sums

template <typename K>
static int bwd_launch(K kernel, Params& P, int threads, size_t smem, long long units, int per_sm, int sms, cudaStream_t st) {
  const int rc = allow_smem(kernel, smem);
  if (rc != CVB_OK) return rc;
  P.parts = parts_of(P, units, per_sm * sms);
  if (P.parts > P.max_parts) P.parts = P.max_parts;
  const dim3 grid((unsigned)(P.parts * (P.gate_kind == kGateImage ? P.B : 1)));
  return launch_chained(kernel, grid, threads, smem, st, P);
}
template <typename IO, int VEC, bool ALONG, bool GATED, int MAXT, int MINB>
static int cf_bwd(Params& P, int sms, cudaStream_t st) {
  const int S = ceil_div(P.C, 8);
  P.tiles = ceil_div(P.HW, 32 * VEC);
  using Px = Pixels<VEC, ALONG>;
  const size_t slots = (size_t)S * ((GATED ? 5 : 4) * 8 * Px::template kSlot<IO> + 4 * Px::template kSlot<float>);
  return bwd_launch(cf_bwd_kernel<IO, 8, VEC, ALONG, GATED, MAXT, MINB>, P, 32 * S, cf_smem(S, 8, VEC, 3) + slots, P.tiles, MINB, sms,
                    st);
}
template <typename IO, bool GATED>
static int cf_bwd_any(Params& P, int sms, cudaStream_t st) {
  // as the forward: four pixels a thread (registers for 64 channels in a block of 256), or two
  const bool four = P.tokens >= (long long)64 * sms, along4 = pixels_aligned<IO>(P, 4);
  const bool along = pixels_aligned<IO>(P, 2);
  if (P.C <= 64 && four) return along4 ? cf_bwd<IO, 4, true, GATED, 256, 1>(P, sms, st) : cf_bwd<IO, 4, false, GATED, 256, 1>(P, sms, st);
  if (P.C <= 128) return along ? cf_bwd<IO, 2, true, GATED, 512, 1>(P, sms, st) : cf_bwd<IO, 2, false, GATED, 512, 1>(P, sms, st);
  return cf_bwd<IO, 1, true, GATED, 1024, 1>(P, sms, st);
}
template <typename IO, int NV, int V, int MAXT, int MINB>
static int cl_bwd(Params& P, int sms, cudaStream_t st) {
  int tpr = 4;
  while (tpr * NV * V < P.C) tpr *= 2;
  const int threads = tpr > 256 ? tpr : 256;
  P.tpr = tpr;
  const long long per = P.gate_kind == kGateImage ? P.HW : P.tokens;
  const int slots = threads / (tpr > 32 ? tpr : 32);
  const size_t joined = slots > 1 ? (size_t)slots * 16 * P.C : 0, ahead = cl_async<IO, NV, V>() ? (size_t)5 * NV * MAXT * V * sizeof(IO) : 0;
  return bwd_launch(cl_bwd_kernel<IO, NV, V, MAXT, MINB>, P, threads, 64 * sizeof(float2) + (joined > ahead ? joined : ahead),
                    ceil_div(per, threads / tpr), MINB, sms, st);
}
template <typename IO, int V>
static int cl_bwd_by_size(Params& P, int sms, cudaStream_t st) {
  if (P.C <= 2048) return cl_bwd<IO, 8 / V, V, 256, 2>(P, sms, st);
  if (P.C <= 4096) return cl_bwd<IO, 8 / V, V, 512, 1>(P, sms, st);
  return cl_bwd<IO, 16 / V, V, 1024, 1>(P, sms, st);
}
template <typename IO>
static int bwd_any(Params& P, int sms, cudaStream_t st) {
  if (P.first) {
    if (P.C <= 256) return P.gate_kind == kGateFull ? cf_bwd_any<IO, true>(P, sms, st) : cf_bwd_any<IO, false>(P, sms, st);
    P.tiles = ceil_div(P.HW, 32);
    return bwd_launch(cf_bwd_wide_kernel<IO>, P, 1024, 32 * 32 * sizeof(float2) + (size_t)16 * P.C, P.tiles, 1, sms, st);
  }
  const int width = cl_width<IO>(P);
  return width == 1 ? cl_bwd_by_size<IO, 1>(P, sms, st)
         : width == 2 ? cl_bwd_by_size<IO, 2>(P, sms, st)
                      : cl_bwd_by_size<IO, 16 / (int)sizeof(IO)>(P, sms, st);
}

int run_bwd(Params& P, int io, int sms, cudaStream_t st) {
  const int rc = io == CVB_F32 ? bwd_any<float>(P, sms, st) : bwd_any<__nv_bfloat16>(P, sms, st);
  if (rc != CVB_OK || !P.partial) return rc;
  return launch_chained(finish_kernel, dim3((unsigned)ceil_div(P.C, 32), 2), 1024, 0, st, P);
}

// Partial sums for each image (or for all): as many as blocks are launched
int most_parts(int C, long long B, int gate_kind, int sms) {
  const long long n = (long long)(C <= 256 ? 4 : C <= 2048 ? 2 : 1) * sms;
  return gate_kind == kGateImage ? (int)((n + B - 1) / B) : (int)n;
}

bool takes(int C, bool first, bool backward) { return C >= 1 && C <= (first && backward ? kWideChannels : 16384); }

}  // namespace seam
}  // namespace cvb
