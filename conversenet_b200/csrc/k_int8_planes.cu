// 1x1 product in 8-bit integers over channels_first tensors, quantised on the way: out (B,N,HW) from x (B,K,HW), K up to 128.
// Bound by the bytes of x and out, which are all it reads and writes beside the weights.
//
// A pixel belongs to two threads from its loads to its stores, half of the channels each.  A group of 256 threads works on 128
// pixels: the threads of a pixel find its largest magnitude, quantise their channels and write them to their lane of tensor memory,
// four bytes a column, where the MMAs (kind::i8, M = 128) read them; the weights stay in shared memory.  The sums come back to
// the same lanes, so the pixel's scale is at hand, and 32 pixels of an output channel are stored by a warp.  The next tile's
// values are loaded to registers between the MMAs and the stores.  Two groups share an SM, so that one's arithmetic
// covers the other's waits.  Tensor memory of a group (256 columns): sums [0,128), values [128,192).
// Every wait is bounded; after a time-out a thread stops working but keeps meeting the group's barriers.
//
// 8 x 64 -> 128 x 256 x 256 fp32: 75 us, 0.81 of the bytes' time at the measured copy rate (a quantising kernel and a product behind it:
// 49 + 134); what is left is 60 % of the issue slots, loads, conversions and stores of single values.  1 x 128 -> 64 x 321 x 481
// bf16: 30 us, floor 9: five rounds of tiles where 4.1 would do, and 64 loads of 2 bytes a thread for each.
#include "../../include/converse_b200.h"
#include "cvb_int8.cuh"
#include "cvb_internal.h"
#include "cvb_tc.cuh"

namespace cvb {
namespace i8 {

constexpr int kPlaneTile = 128, kPlaneThreads = 256, kPlaneGroups = 2, kPlaneWait = 1 << 20;
constexpr int kPlaneCols = 128;                        // output channels of a pass
constexpr size_t kPlaneWeights = 160 * 1024;           // bytes of shared memory for the weights

struct PlaneParams {
  const void* x;
  const signed char* w;
  const float *w_scale, *bias;
  void* out;
  long long ldw, HW, tiles;
  int K, N, image_tiles;
  int* status;
};

__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "n"(kPlaneThreads) : "memory"); }
__device__ __forceinline__ void plane_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t elected) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void plane_commit(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t"
      ".reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void plane_st4(uint32_t t, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(t), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void plane_ld16(uint32_t t, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void plane_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void plane_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// CH channels of a pixel, a register each, as they were loaded: nothing waits for them before they are used.  (bf16 values packed in
// pairs were waited for at once, before the stores that should cover the loads: 1 x 128 -> 64 x 321 x 481 took 72 us.)
template <typename IO, int CH>
struct Values;
template <int CH>
struct Values<float, CH> {
  uint32_t raw[CH];
  __device__ __forceinline__ uint32_t at(const float* p) const { return __float_as_uint(*p); }
  __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(raw[i]); }
};
template <int CH>
struct Values<__nv_bfloat16, CH> {
  uint32_t raw[CH];
  __device__ __forceinline__ uint32_t at(const __nv_bfloat16* p) const { return *(const unsigned short*)p; }
  __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(raw[i] << 16); }
};

template <typename IO, int CH>
__global__ void __launch_bounds__(kPlaneThreads* kPlaneGroups, 1) planes_kernel(const __grid_constant__ PlaneParams P) {
  // The wait comes before tensor memory is taken, and the next kernel is let in behind it: a block that held tensor memory while it
  // waited for a kernel whose blocks still have to take theirs would wait for ever.
  pdl_wait();
  extern __shared__ __align__(16) unsigned char weights[];
  __shared__ float red[kPlaneGroups][2][kPlaneTile];
  __shared__ uint64_t bars[kPlaneGroups];
  __shared__ uint32_t tmem_base;
  const int np = (P.N + 15) & ~15, kc = (P.K + 31) / 32 * 2, groups = blockDim.x / kPlaneThreads;
  float* vec = (float*)(weights + (size_t)kc * np * 16);          // np scales, np biases
  const int g = threadIdx.x / kPlaneThreads, warp = (threadIdx.x >> 5) & 7, lane = threadIdx.x & 31;
  const int quadrant = warp & 3, half = warp >> 2, r = quadrant * 32 + lane;
  // weights: rows of 16 bytes of K, all output channels of the same 16 side by side
  for (int i = threadIdx.x; i < kc * np; i += blockDim.x) {
    const int c = i / np, n = i - c * np, k = 16 * c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n < P.N && k < P.K) {
      const signed char* from = P.w + n * P.ldw + k;
      if (k + 16 <= P.K) {
        v = *(const uint4*)from;
      } else {
        uint32_t b[4] = {0, 0, 0, 0};
        for (int j = 0; j < P.K - k; ++j) b[j >> 2] |= (uint32_t)(unsigned char)from[j] << (8 * (j & 3));
        v = make_uint4(b[0], b[1], b[2], b[3]);
      }
    }
    *(uint4*)(weights + (size_t)i * 16) = v;
  }
  for (int i = threadIdx.x; i < 2 * np; i += blockDim.x) {
    const int n = i < np ? i : i - np;
    vec[i] = n >= P.N ? 0.f : i < np ? P.w_scale[n] : P.bias ? P.bias[n] : 0.f;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < groups; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();
  }
  __syncwarp();
  if (threadIdx.x < 32) tc::tmem_alloc(&tmem_base, groups == 1 ? 256 : 512);
  tc::fence_proxy_async();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_let_next();
  const uint32_t tmem = tmem_base + g * 256, lanes = tmem + ((uint32_t)(quadrant * 32) << 16);
  const uint32_t elected = tc::elect_one();
  uint32_t phase = 0;
  bool alive = true;

  const long long step = (long long)gridDim.x * groups;
  long long tile = (long long)blockIdx.x * groups + g;
  Values<IO, CH> v;
  auto fetch = [&](long long t) {
    const long long b = t / P.image_tiles, px = (t - b * P.image_tiles) * kPlaneTile + r;
    const IO* p = (const IO*)P.x + (b * P.K + half * CH) * P.HW + px;
    const int n = t < P.tiles && px < P.HW ? P.K - half * CH : 0;
    if (n >= CH) {
#pragma unroll
      for (int i = 0; i < CH; ++i, p += P.HW) v.raw[i] = v.at(p);
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i, p += P.HW) v.raw[i] = i < n ? v.at(p) : 0u;
    }
  };
  fetch(tile);
  for (; tile < P.tiles; tile += step) {
    const long long b = tile / P.image_tiles, px = (tile - b * P.image_tiles) * kPlaneTile + r;
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < CH; i += 2) a = largest(a, v[i], v[i + 1]);
    red[g][half][r] = a;
    group_sync(g);
    const Quantiser<sizeof(IO) == 2> q(largest(a, red[g][half ^ 1][r]));
    const float scale = q.scale();
#pragma unroll
    for (int i = 0; i < CH / 16; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = q.four(v[16 * i + 4 * j], v[16 * i + 4 * j + 1], v[16 * i + 4 * j + 2], v[16 * i + 4 * j + 3]);
      __syncwarp();          // (a value next to a border took some lanes another way; the store is one of the whole warp)
      plane_st4(lanes + 128 + half * (CH / 4) + 4 * i, w[0], w[1], w[2], w[3]);
    }
    tc::tmem_wait_st();
    for (int n0 = 0; n0 < np; n0 += kPlaneCols) {
      const int cols = np - n0 < kPlaneCols ? np - n0 : kPlaneCols;
      tc::fence_before_sync();
      group_sync(g);          // the values are written, and the sums before are read
      if (warp == 0 && alive) {
        tc::fence_after_sync();
        const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | (8u << 24);
        for (int k = 0; k < kc / 2; ++k)
          plane_mma(tmem, tmem + 128 + 8 * k, tc::smem_desc(weights + ((size_t)2 * k * np + n0) * 16, 16 * np, 128), idesc, k != 0, elected);
        plane_commit(&bars[g], elected);
      }
      if (n0 == 0) fetch(tile + step);
      if (alive) alive = __all_sync(0xffffffffu, mbar_wait_bounded(&bars[g], phase, kPlaneWait));
      phase ^= 1;
      if (!alive) continue;
      tc::fence_after_sync();
      IO* out = (IO*)P.out + (b * P.N + n0) * P.HW + px;
      for (int c = 16 * half; c < cols; c += 32) {
        int s[16];
        __syncwarp();          // (lanes behind the last pixel store nothing, and the load is one of the whole warp)
        plane_ld16(lanes + c, s);
        tc::tmem_wait_ld();
        IO* to = out + c * P.HW;
        if (px >= P.HW) continue;
        const int left = P.N - n0 - c;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (j >= left) break;
          const float4 w = *(const float4*)(vec + n0 + c + j), o = *(const float4*)(vec + np + n0 + c + j);
          const float ws[4] = {w.x, w.y, w.z, w.w}, os[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // the integer as fp32 (its magnitude is below 128 . 127 . 128 < 2^22) without the conversion unit
            const float t = __int_as_float(s[j + i] + 0x4b400000) - 12582912.f;
            const float y = fmaf(t * ws[i], scale, os[i]);          // (tokens are of any size, weights of ordinary ones)
            if (i == 0 || j + i < left) plane_store(to, y);
            to += P.HW;
          }
        }
      }
      __syncwarp();
    }
  }
  if (!alive && lane == 0 && P.status) *P.status = 1;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (threadIdx.x < 32) tc::tmem_dealloc(tmem_base, groups == 1 ? 256 : 512);
}

static size_t plane_weight_bytes(int K, int N) { return (size_t)((K + 31) / 32 * 32) * ((N + 15) / 16 * 16); }

// K that two threads hold in 64 registers each; weights that fit shared memory; few pixels with many output channels go to the
// kernels that share the channels out to all multiprocessors
bool planes_take(long long B, long long HW, int K, int N, int io, int sms) {
  const long long tiles = B * ((HW + kPlaneTile - 1) / kPlaneTile);
  (void)io;
  return K <= 128 && plane_weight_bytes(K, N) <= kPlaneWeights && (N <= 256 || tiles >= sms);
}

template <typename IO, int CH>
static int launch(const PlaneParams& P, int sms, cudaStream_t st) {
  const size_t smem = plane_weight_bytes(P.K, P.N) + (size_t)(P.N + 15) / 16 * 16 * 8;
  CVB_CUDA(cudaFuncSetAttribute(planes_kernel<IO, CH>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
  const int groups = P.tiles > sms ? kPlaneGroups : 1;
  const long long blocks = (P.tiles + groups - 1) / groups;
  return launch_chained(planes_kernel<IO, CH>, dim3((unsigned)(blocks < sms ? blocks : sms)), kPlaneThreads * groups, smem, st, P);
}

int run_planes(const void* x, const signed char* w, long long ldw, const float* w_scale, const float* bias, void* out, long long B,
               long long HW, int K, int N, int io, int sms, int* status, cudaStream_t st) {
  PlaneParams P;
  P.x = x; P.w = w; P.ldw = ldw; P.w_scale = w_scale; P.bias = bias; P.out = out; P.HW = HW; P.K = K; P.N = N; P.status = status;
  P.image_tiles = (int)((HW + kPlaneTile - 1) / kPlaneTile);
  P.tiles = B * P.image_tiles;
  if (io == CVB_F32) return K <= 64 ? launch<float, 32>(P, sms, st) : launch<float, 64>(P, sms, st);
  return K <= 64 ? launch<__nv_bfloat16, 32>(P, sms, st) : launch<__nv_bfloat16, 64>(P, sms, st);
}

}  // namespace i8
}  // namespace cvb
