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

// The gate's factor.  ex2.approx and the approximate reciprocal are good to 2 units in the last place; the product before them
// loses |g| . 2^-24, so a sigmoid is off by 1e-6 of itself at |g| = 10.
__device__ __forceinline__ float gate_of(float g, int act) { return act ? __fdividef(1.f, 1.f + __expf(-g)) : g; }
// its derivative, from the factor
__device__ __forceinline__ float gate_slope(float s, int act) { return act ? s * (1.f - s) : 1.f; }

// ------------------------------------------------------------------ channels_first, forward
// block: 32 x S threads; thread (lane, s) holds channels s CPT .. of pixels 32 VEC tile + VEC lane ..
// `red`: 2 x S x 32 VEC pairs
template <int CPT, int VEC>
__device__ __forceinline__ void cf_stats(const float (&v)[CPT][VEC], int n, const Params& P, float2* red, float (&mean)[VEC],
                                         float (&rstd)[VEC]) {
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5;
  // this thread's mean and squares around it; joined: M2 = sum (M2_i + n_i (m_i - mean)^2)
  float2 own[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float m = 0.f, q = 0.f;
    if (!P.rms) {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        if (i < n) m += v[i][j];
      m = n ? m / (float)n : 0.f;
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (i < n) q = fmaf(v[i][j] - m, v[i][j] - m, q);
    own[j] = make_float2(m, q);
  }
  const float inv = 1.f / (float)P.C;
  if (S == 1) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) mean[j] = own[j].x, rstd[j] = rsqrtf(fmaf(own[j].y, inv, P.eps));
    return;
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) red[(s * VEC + j) * 32 + lane] = own[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float m = 0.f, q = 0.f;
    if (!P.rms) {
      for (int t = 0; t < S; ++t) m = fmaf(red[(t * VEC + j) * 32 + lane].x, (float)min(CPT, P.C - t * CPT), m);
      m *= inv;
    }
    for (int t = 0; t < S; ++t) {
      const float2 o = red[(t * VEC + j) * 32 + lane];
      q += o.y;
      if (!P.rms) q = fmaf((o.x - m) * (o.x - m), (float)min(CPT, P.C - t * CPT), q);
    }
    mean[j] = m;
    rstd[j] = rsqrtf(fmaf(q, inv, P.eps));
  }
}

template <typename IO, int CPT, int VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) cf_fwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  extern __shared__ float2 red[];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5;
  const int c0 = s * CPT, n = min(CPT, P.C - c0);
  const long long b = blockIdx.x / P.tiles, px = ((long long)(blockIdx.x - b * P.tiles) * 32 + lane) * VEC;
  const bool live = px < P.HW;
  const long long base = ((long long)b * P.C + c0) * P.HW + px, token = b * P.HW + px;
  float v[CPT][VEC], x[CPT][VEC];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (live && i < n) {
      Vec<IO, VEC>::load(P.branch, base + i * P.HW, v[i]);
      Vec<IO, VEC>::load(P.x, base + i * P.HW, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = x[i][j] = 0.f;
    }
  }
  float mean[VEC], rstd[VEC];
  if (P.post_w) {
    cf_stats<CPT, VEC>(v, n, P, red, mean, rstd);
    if (P.stats && live && s == 0) {
      Vec<float, VEC>::store(P.stats, token, mean);
      Vec<float, VEC>::store(P.stats + P.tokens, token, rstd);
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (i < n) {
        const float w = P.post_w[c0 + i], o = P.post_b ? P.post_b[c0 + i] : 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = fmaf((v[i][j] - mean[j]) * rstd[j], w, o);
      }
  }
  if (P.gate_kind == kGateFull && live) {
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (i < n) {
        float g[VEC];
        Vec<IO, VEC>::load(P.gate, base + i * P.HW, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= gate_of(g[j], P.act);
      }
  }
#pragma unroll
  for (int i = 0; i < CPT; ++i)
    if (i < n) {
      float a = P.scale ? P.scale[c0 + i] : 1.f;
      if (P.gate_kind == kGateImage) a *= gate_of(((const float*)P.gate)[b * P.C + c0 + i], P.act);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(v[i][j], a, x[i][j]);
      if (live) Vec<IO, VEC>::store(P.y, base + i * P.HW, v[i]);
    }
  if (!P.pre_w) return;
  cf_stats<CPT, VEC>(v, n, P, red + S * 32 * VEC, mean, rstd);
  if (P.stats && live && s == 0) {
    Vec<float, VEC>::store(P.stats + 2 * P.tokens, token, mean);
    Vec<float, VEC>::store(P.stats + 3 * P.tokens, token, rstd);
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < CPT; ++i)
    if (i < n) {
      const float w = P.pre_w[c0 + i], o = P.pre_b ? P.pre_b[c0 + i] : 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf((v[i][j] - mean[j]) * rstd[j], w, o);
      Vec<IO, VEC>::store(P.z, base + i * P.HW, v[i]);
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
  if (P.gate_kind == kGateImage) a *= gate_of(((const float*)P.gate)[b * P.C + c], P.act);
  if (P.gate_kind == kGateFull) {
    Vec<IO, 1>::load(P.gate, at, &g);
    v *= gate_of(g, P.act);
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
// The sums over the warps of two values for each pixel.  `buf` alternates: the values of the reduction before the last are read
// by everybody who arrived at the last one.
template <int VEC>
__device__ __forceinline__ void cf_join(float (&a)[VEC], float (&b)[VEC], float2* red, int S, int& buf) {
  if (S == 1) return;
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  float2* r = red + buf * S * 32 * VEC;
  buf ^= 1;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r[(s * VEC + j) * 32 + lane] = make_float2(a[j], b[j]);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    a[j] = b[j] = 0.f;
    for (int t = 0; t < S; ++t) {
      const float2 o = r[(t * VEC + j) * 32 + lane];
      a[j] += o.x;
      b[j] += o.y;
    }
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// `parts` blocks walk over all images' tiles, or over those of an image where the gate has a value for each image
template <typename IO, int CPT, int VEC, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cf_bwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  extern __shared__ float2 red[];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5;
  const int c0 = s * CPT, n = min(CPT, P.C - c0);
  const float inv = 1.f / (float)P.C;
  float sa[CPT], sb[CPT], sw[CPT], so[CPT];       // sums A, B; dz k, dz
#pragma unroll
  for (int i = 0; i < CPT; ++i) sa[i] = sb[i] = sw[i] = so[i] = 0.f;
  int buf = 0;
  const bool image = P.gate_kind == kGateImage;
  const long long first = image ? (long long)(blockIdx.x / P.parts) * P.tiles : 0, last = image ? first + P.tiles : (long long)P.tiles * P.B;
  for (long long tile = first + blockIdx.x % P.parts; tile < last; tile += P.parts) {
    const long long b = tile / P.tiles, px = ((tile - b * P.tiles) * 32 + lane) * VEC;
    const bool live = px < P.HW;
    const long long base = (b * P.C + c0) * P.HW + px, token = b * P.HW + px;
    float d[CPT][VEC], k[CPT][VEC], h[CPT][VEC], f[CPT][VEC];          // f: the gate
    float mean[VEC], rstd[VEC], u[VEC], w[VEC];
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const bool on = live && i < n;
#pragma unroll
      for (int j = 0; j < VEC; ++j) d[i][j] = h[i][j] = k[i][j] = 0.f, f[i][j] = 1.f;
      if (on && P.dz) {
        Vec<IO, VEC>::load(P.dz, base + i * P.HW, d[i]);
        Vec<IO, VEC>::load(P.x, base + i * P.HW, k[i]);
      }
      if (on && P.branch) Vec<IO, VEC>::load(P.branch, base + i * P.HW, h[i]);
      if (on && P.branch && P.gate_kind == kGateFull) {
        Vec<IO, VEC>::load(P.gate, base + i * P.HW, f[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[i][j] = gate_of(f[i][j], P.act);
      } else if (image && i < n) {
        const float g = gate_of(((const float*)P.gate)[b * P.C + c0 + i], P.act);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[i][j] = g;
      }
    }
    if (P.post_w) {
      if (live) {
        Vec<float, VEC>::load(P.stats, token, mean);
        Vec<float, VEC>::load(P.stats, P.tokens + token, rstd);
#pragma unroll
        for (int i = 0; i < CPT; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] = (h[i][j] - mean[j]) * rstd[j];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) rstd[j] = 1.f;
      }
    }
    if (P.dz) {
      float mk[VEC], rk[VEC];
      if (live) {
        Vec<float, VEC>::load(P.stats, 2 * P.tokens + token, mk);
        Vec<float, VEC>::load(P.stats, 3 * P.tokens + token, rk);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) mk[j] = 0.f, rk[j] = 1.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[j] = w[j] = 0.f;
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        if (live && i < n) {
          const float a = P.scale ? P.scale[c0 + i] : 1.f, pw = P.post_w ? P.post_w[c0 + i] : 1.f;
          const float pb = P.post_b ? P.post_b[c0 + i] : 0.f, g = P.pre_w[c0 + i];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            // y again, as it was before it was rounded
            k[i][j] = (fmaf(fmaf(h[i][j], pw, pb) * f[i][j], a, k[i][j]) - mk[j]) * rk[j];
            so[i] += d[i][j];
            sw[i] = fmaf(d[i][j], k[i][j], sw[i]);
            d[i][j] *= g;
            u[j] += d[i][j];
            w[j] = fmaf(d[i][j], k[i][j], w[j]);
          }
        }
      cf_join<VEC>(u, w, red, S, buf);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u[j] = P.rms ? 0.f : u[j] * inv;
        w[j] *= inv;
      }
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[i][j] = rk[j] * (d[i][j] - u[j] - k[i][j] * w[j]);
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (live && i < n) {
        if (P.dy) {
          float e[VEC];
          Vec<IO, VEC>::load(P.dy, base + i * P.HW, e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) d[i][j] += e[j];
        }
        if (P.dx) Vec<IO, VEC>::store(P.dx, base + i * P.HW, d[i]);
      }
    if (!P.branch) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[j] = w[j] = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (live && i < n) {
        const float a = P.scale ? P.scale[c0 + i] : 1.f, pw = P.post_w ? P.post_w[c0 + i] : 1.f;
        if (P.gate_kind == kGateFull && P.dgate) {
          const float pb = P.post_b ? P.post_b[c0 + i] : 0.f;
          float dg[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) dg[j] = d[i][j] * a * fmaf(h[i][j], pw, pb) * gate_slope(f[i][j], P.act);
          Vec<IO, VEC>::store(P.dgate, base + i * P.HW, dg);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (!image) d[i][j] *= f[i][j];          // (an image's sums are without its gate)
          sb[i] += d[i][j];
          sa[i] = fmaf(d[i][j], h[i][j], sa[i]);
          d[i][j] *= image ? a * pw * f[i][j] : a * pw;
          u[j] += d[i][j];
          w[j] = fmaf(d[i][j], h[i][j], w[j]);
        }
      }
    if (!P.dbranch) continue;
    if (P.post_w) {
      cf_join<VEC>(u, w, red, S, buf);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u[j] = P.rms ? 0.f : u[j] * inv;
        w[j] *= inv;
      }
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (live && i < n) {
        if (P.post_w) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) d[i][j] = rstd[j] * (d[i][j] - u[j] - h[i][j] * w[j]);
        }
        Vec<IO, VEC>::store(P.dbranch, base + i * P.HW, d[i]);
      }
  }
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
      if (image) a *= gate_of(((const float*)P.gate)[b * P.C + c], P.act);
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
        g = gate_of(g, P.act);
        if (live && P.dgate) {
          const float pw = P.post_w ? P.post_w[c] : 1.f, pb = P.post_b ? P.post_b[c] : 0.f;
          const float dg = d * (P.scale ? P.scale[c] : 1.f) * fmaf(h, pw, pb) * gate_slope(g, P.act);
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
        g = gate_of(g, P.act);
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
// Sum over the token's threads; `red`: the block's, for tokens of more than a warp.
__device__ __forceinline__ float cl_sum(float v, int tpr, float* red) {
  for (int o = (tpr < 32 ? tpr : 32) >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  __syncthreads();          // the values before are read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  const int w0 = (threadIdx.x & ~(tpr - 1)) >> 5;
  for (int j = 0; j < (tpr >> 5); ++j) v += red[w0 + j];
  return v;
}
__device__ __forceinline__ float2 cl_sum2(float2 v, int tpr, float2* red) {
  for (int o = (tpr < 32 ? tpr : 32) >> 1; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (tpr <= 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = make_float2(0.f, 0.f);
  const int w0 = (threadIdx.x & ~(tpr - 1)) >> 5;
  for (int j = 0; j < (tpr >> 5); ++j) v.x += red[w0 + j].x, v.y += red[w0 + j].y;
  return v;
}
template <int NV, int V>
__device__ __forceinline__ void cl_stats(const float (&v)[NV][V], const Params& P, int tpr, int t, float* red, float& mean,
                                         float& rstd) {
  const float inv = 1.f / (float)P.C;
  float m = 0.f, q = 0.f;
  mean = 0.f;
  if (!P.rms) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) m += v[i][j];          // (zeros behind the last channel)
    mean = cl_sum(m, tpr, red) * inv;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * tpr + t) * V < P.C) {
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(v[i][j] - mean, v[i][j] - mean, q);
    }
  rstd = rsqrtf(fmaf(cl_sum(q, tpr, red), inv, P.eps));
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

template <typename IO, int NV, int V, int MAXT>
__global__ void __launch_bounds__(MAXT) cl_fwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ float red[32];
  const int tpr = P.tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x / tpr;
  const long long token = (long long)blockIdx.x * rows + threadIdx.x / tpr;
  const bool live = token < P.tokens;
  const long long base = token * P.C, b = live ? token / P.HW : 0;
  float v[NV][V], x[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
    if (live && c < P.C) {
      Vec<IO, V>::load(P.branch, base + c, v[i]);
      Vec<IO, V>::load(P.x, base + c, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = x[i][j] = 0.f;
    }
  }
  float mean = 0.f, rstd = 1.f;
  if (P.post_w) {
    cl_stats<NV, V>(v, P, tpr, t, red, mean, rstd);
    if (P.stats && live && t == 0) P.stats[token] = mean, P.stats[P.tokens + token] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
    if (c >= P.C || !live) continue;
    float w[V], o[V];
    if (P.post_w) {
      cl_vector<V>(P.post_w, c, 1.f, w);
      cl_vector<V>(P.post_b, c, 0.f, o);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = fmaf((v[i][j] - mean) * rstd, w[j], o[j]);
    }
    if (P.gate_kind) {
      if (P.gate_kind == kGateFull) Vec<IO, V>::load(P.gate, base + c, w);
      else cl_vector<V>((const float*)P.gate + b * P.C, c, 0.f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= gate_of(w[j], P.act);
    }
    cl_vector<V>(P.scale, c, 1.f, w);
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = fmaf(v[i][j], w[j], x[i][j]);
    Vec<IO, V>::store(P.y, base + c, v[i]);
  }
  if (!P.pre_w) return;
  cl_stats<NV, V>(v, P, tpr, t, red, mean, rstd);
  if (!live) return;
  if (P.stats && t == 0) P.stats[2 * P.tokens + token] = mean, P.stats[3 * P.tokens + token] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + t) * V;
    if (c >= P.C) continue;
    float w[V], o[V];
    cl_vector<V>(P.pre_w, c, 1.f, w);
    cl_vector<V>(P.pre_b, c, 0.f, o);
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = fmaf((v[i][j] - mean) * rstd, w[j], o[j]);
    Vec<IO, V>::store(P.z, base + c, v[i]);
  }
}

template <typename IO, int NV, int V, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) cl_bwd_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ float2 red[32];
  extern __shared__ float2 joined[];          // 4 C floats for each warp, or each token of more than a warp
  const int tpr = P.tpr, t = threadIdx.x & (tpr - 1), rows = blockDim.x / tpr, row = threadIdx.x / tpr;
  const float inv = 1.f / (float)P.C;
  const bool image = P.gate_kind == kGateImage;
  const long long of = blockIdx.x / P.parts, first = image ? of * P.HW : 0, last = image ? first + P.HW : P.tokens;
  float sa[NV][V], sb[NV][V], sw[NV][V], so[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sa[i][j] = sb[i][j] = sw[i][j] = so[i][j] = 0.f;
  for (long long start = first + (long long)(blockIdx.x % P.parts) * rows; start < last; start += (long long)P.parts * rows) {
    const long long token = start + row;
    const bool live = token < last;
    const long long base = token * P.C;
    float d[NV][V], k[NV][V], h[NV][V], f[NV][V];          // f: the gate
    float mean = 0.f, rstd = 1.f;
    if (P.post_w && live) mean = P.stats[token], rstd = P.stats[P.tokens + token];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      const bool on = live && c < P.C;
#pragma unroll
      for (int j = 0; j < V; ++j) d[i][j] = k[i][j] = h[i][j] = 0.f, f[i][j] = 1.f;
      if (on && P.dz) {
        Vec<IO, V>::load(P.dz, base + c, d[i]);
        Vec<IO, V>::load(P.x, base + c, k[i]);
      }
      if (on && P.branch) {
        Vec<IO, V>::load(P.branch, base + c, h[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (h[i][j] - mean) * rstd;
      }
      if (on && P.branch && P.gate_kind) {
        if (image) cl_vector<V>((const float*)P.gate + of * P.C, c, 0.f, f[i]);
        else Vec<IO, V>::load(P.gate, base + c, f[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) f[i][j] = gate_of(f[i][j], P.act);
      }
    }
    if (P.dz) {
      const float mk = live ? P.stats[2 * P.tokens + token] : 0.f, rk = live ? P.stats[3 * P.tokens + token] : 1.f;
      float2 u = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * tpr + t) * V;
        if (c >= P.C || !live) continue;
        float w[V], a[V], pw[V], pb[V];
        cl_vector<V>(P.pre_w, c, 1.f, w);
        cl_vector<V>(P.scale, c, 1.f, a);
        cl_vector<V>(P.post_w, c, 1.f, pw);
        cl_vector<V>(P.post_b, c, 0.f, pb);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          // y again, as it was before it was rounded
          k[i][j] = (fmaf(fmaf(h[i][j], pw[j], pb[j]) * f[i][j], a[j], k[i][j]) - mk) * rk;
          so[i][j] += d[i][j];
          sw[i][j] = fmaf(d[i][j], k[i][j], sw[i][j]);
          d[i][j] *= w[j];
          u.x += d[i][j];
          u.y = fmaf(d[i][j], k[i][j], u.y);
        }
      }
      u = cl_sum2(u, tpr, red);
      u.x = P.rms ? 0.f : u.x * inv;
      u.y *= inv;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = rk * (d[i][j] - u.x - k[i][j] * u.y);
    }
    float2 u = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c >= P.C || !live) continue;
      if (P.dy) {
        float w[V];
        Vec<IO, V>::load(P.dy, base + c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] += w[j];
      }
      if (P.dx) Vec<IO, V>::store(P.dx, base + c, d[i]);
      if (!P.branch) continue;
      float a[V], pw[V];
      cl_vector<V>(P.scale, c, 1.f, a);
      cl_vector<V>(P.post_w, c, 1.f, pw);
      if (P.gate_kind == kGateFull && P.dgate) {
        float o[V];
        cl_vector<V>(P.post_b, c, 0.f, o);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = d[i][j] * a[j] * fmaf(h[i][j], pw[j], o[j]) * gate_slope(f[i][j], P.act);
        Vec<IO, V>::store(P.dgate, base + c, o);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!image) d[i][j] *= f[i][j];          // (an image's sums are without its gate)
        sb[i][j] += d[i][j];
        sa[i][j] = fmaf(d[i][j], h[i][j], sa[i][j]);
        d[i][j] *= image ? a[j] * pw[j] * f[i][j] : a[j] * pw[j];
        u.x += d[i][j];
        u.y = fmaf(d[i][j], h[i][j], u.y);
      }
    }
    if (!P.dbranch) continue;
    if (P.post_w) {
      u = cl_sum2(u, tpr, red);
      u.x = P.rms ? 0.f : u.x * inv;
      u.y *= inv;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * V;
      if (c >= P.C || !live) continue;
      if (P.post_w) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = rstd * (d[i][j] - u.x - h[i][j] * u.y);
      }
      Vec<IO, V>::store(P.dbranch, base + c, d[i]);
    }
  }
  if (!P.partial) return;
  float* out = P.partial + (long long)blockIdx.x * 4 * P.C;
  const int slots = blockDim.x / (tpr > 32 ? tpr : 32);
  float* own = slots > 1 ? (float*)joined + (threadIdx.x / (tpr > 32 ? tpr : 32)) * 4 * P.C : out;
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
    for (int w = 0; w < slots; ++w) v += ((float*)joined)[w * 4 * P.C + i];
    out[i] = v;
  }
}

// ------------------------------------------------------------------ the parameters' gradients from the partial sums
// grid: (groups of 32 channels, 2): the sums A, B and what follows from them; the sums of dz
__global__ void __launch_bounds__(1024) finish_kernel(const __grid_constant__ Params P) {
  pdl_start();
  __shared__ double red[32][32][2];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const bool pre = blockIdx.y == 1;
  const int images = P.gate_kind == kGateImage ? (int)P.B : 1;
  const float a = P.scale && c < P.C ? P.scale[c] : 1.f, w = P.post_w && c < P.C ? P.post_w[c] : 1.f;
  const float o = P.post_b && c < P.C ? P.post_b[c] : 0.f;
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
      const float g = gate_of(((const float*)P.gate)[(long long)b * P.C + c], P.act);
      if (P.dgate) ((float*)P.dgate)[(long long)b * P.C + c] = (float)(a * (w * u0 + o * u1) * gate_slope(g, P.act));
      u0 *= g;
      u1 *= g;
    }
    t0 += u0;
    t1 += u1;
  }
  red[s][lane][0] = t0;
  red[s][lane][1] = t1;
  __syncthreads();
  if (s == 0)
    for (int r = 1; r < 32; ++r) t0 += red[r][lane][0], t1 += red[r][lane][1];
  if (s != 0 || c >= P.C) return;
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
static bool vectors_aligned(const Params& P) {
  const void* all[] = {P.scale, P.post_w, P.post_b, P.pre_w, P.pre_b, P.gate_kind == kGateImage ? P.gate : nullptr};
  for (const void* p : all)
    if ((size_t)p % 16) return false;
  return true;
}
static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

template <typename IO, int CPT, int VEC, int MAXT>
static int cf_fwd(Params& P, cudaStream_t st) {
  const int S = ceil_div(P.C, CPT);
  P.tiles = ceil_div(P.HW, 32 * VEC);
  const size_t smem = S > 1 ? (size_t)2 * S * 32 * VEC * sizeof(float2) : 0;
  const int rc = allow_smem(cf_fwd_kernel<IO, CPT, VEC, MAXT>, smem);
  if (rc != CVB_OK) return rc;
  return launch_chained(cf_fwd_kernel<IO, CPT, VEC, MAXT>, dim3((unsigned)(P.tiles * P.B)), 32 * S, smem, st, P);
}
template <typename IO>
static int cf_fwd_any(Params& P, int sms, cudaStream_t st) {
  // four pixels a thread where rows allow it and still give every SM two blocks; else one, which also takes odd rows
  const bool four = P.HW % 4 == 0 && aligned(P, 4 * sizeof(IO)) && P.tokens >= (long long)2 * sms * 128;
  if (P.C <= 128 && four) return cf_fwd<IO, 8, 4, 512>(P, st);
  if (P.C <= 256) return cf_fwd<IO, 8, 1, 1024>(P, st);
  if (P.C <= 1024) return cf_fwd<IO, 32, 1, 1024>(P, st);
  P.tiles = ceil_div(P.HW, 32);
  return launch_chained(cf_fwd_wide_kernel<IO>, dim3((unsigned)(P.tiles * P.B)), 1024, 0, st, P);
}
template <typename IO, int NV, int V, int MAXT>
static int cl_fwd(Params& P, cudaStream_t st) {
  int tpr = 4;
  while (tpr * NV * V < P.C) tpr *= 2;
  const int threads = tpr > 256 ? tpr : 256;
  P.tpr = tpr;
  return launch_chained(cl_fwd_kernel<IO, NV, V, MAXT>, dim3((unsigned)ceil_div(P.tokens, threads / tpr)), threads, 0, st, P);
}
template <typename IO>
static int cl_fwd_any(Params& P, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(IO);
  const bool vec = P.C % V == 0 && aligned(P, 16) && vectors_aligned(P);
  if (P.C <= 2048) return vec ? cl_fwd<IO, 8 / V, V, 256>(P, st) : cl_fwd<IO, 8, 1, 256>(P, st);
  return vec ? cl_fwd<IO, 16 / V, V, 1024>(P, st) : cl_fwd<IO, 16, 1, 1024>(P, st);
}

int run_fwd(Params& P, int io, int sms, cudaStream_t st) {
  if (P.first) return io == CVB_F32 ? cf_fwd_any<float>(P, sms, st) : cf_fwd_any<__nv_bfloat16>(P, sms, st);
  return io == CVB_F32 ? cl_fwd_any<float>(P, st) : cl_fwd_any<__nv_bfloat16>(P, st);
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
template <typename IO, int VEC, int MAXT, int MINB>
static int cf_bwd(Params& P, int sms, cudaStream_t st) {
  const int S = ceil_div(P.C, 8);
  P.tiles = ceil_div(P.HW, 32 * VEC);
  const int per_sm = MINB;
  return bwd_launch(cf_bwd_kernel<IO, 8, VEC, MAXT, MINB>, P, 32 * S, S > 1 ? (size_t)2 * S * 32 * VEC * sizeof(float2) : 0, P.tiles,
                    per_sm, sms, st);
}
template <typename IO, int NV, int V, int MAXT, int MINB>
static int cl_bwd(Params& P, int sms, cudaStream_t st) {
  int tpr = 4;
  while (tpr * NV * V < P.C) tpr *= 2;
  const int threads = tpr > 256 ? tpr : 256;
  P.tpr = tpr;
  const long long per = P.gate_kind == kGateImage ? P.HW : P.tokens;
  const int slots = threads / (tpr > 32 ? tpr : 32);
  return bwd_launch(cl_bwd_kernel<IO, NV, V, MAXT, MINB>, P, threads, slots > 1 ? (size_t)slots * 16 * P.C : 0,
                    ceil_div(per, threads / tpr), MINB, sms, st);
}
template <typename IO>
static int bwd_any(Params& P, int sms, cudaStream_t st) {
  if (P.first) {
    if (P.C <= 64 && P.HW % 2 == 0 && aligned(P, 2 * sizeof(IO)) && P.tokens >= (long long)2 * sms * 64)
      return cf_bwd<IO, 2, 256, 2>(P, sms, st);
    if (P.C <= 64) return cf_bwd<IO, 1, 256, 3>(P, sms, st);
    if (P.C <= 128) return cf_bwd<IO, 1, 512, 1>(P, sms, st);
    if (P.C <= 256) return cf_bwd<IO, 1, 1024, 1>(P, sms, st);
    P.tiles = ceil_div(P.HW, 32);
    return bwd_launch(cf_bwd_wide_kernel<IO>, P, 1024, 32 * 32 * sizeof(float2) + (size_t)16 * P.C, P.tiles, 1, sms, st);
  }
  constexpr int V = 16 / (int)sizeof(IO);
  const bool vec = P.C % V == 0 && aligned(P, 16) && vectors_aligned(P);
  if (P.C <= 2048) return vec ? cl_bwd<IO, 8 / V, V, 256, 2>(P, sms, st) : cl_bwd<IO, 8, 1, 256, 2>(P, sms, st);
  return vec ? cl_bwd<IO, 16 / V, V, 1024, 1>(P, sms, st) : cl_bwd<IO, 16, 1, 1024, 1>(P, sms, st);
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
