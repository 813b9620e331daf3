// 1x1 products in 8-bit integers: tokens quantised by their largest channel, weights by output channel.
//
// The product: D = L R^T on tcgen05 (kind::i8, sums exact in 32 bits).  The operand whose rows become lanes of tensor memory
// is the one whose index is contiguous in the output: pixels in channels_first, output channels in channels_last.  So a warp
// stores 32 neighbours of a row whichever layout it is, straight from its registers.  Both operands are K-major in global
// memory; TMA brings boxes of 128 bytes of K by 128 (L) or NT (R) rows to shared memory (128-byte swizzle), zeros behind the
// last K and the last row.  One block a multiprocessor walks over tiles of 128 x NT: a warp that copies, a warp that issues the
// MMAs, eight warps that scale and store; two accumulators, so that a tile is stored while the next one is computed.
// Every wait is bounded; a role that gives up sets the status word and ends, and the others follow.
//
// What bounds it: the tensor pipe where K is long (8192 x 4096 -> 4096: 91 us, the pipe active 80 % of the cycles, 3.0 POP/s);
// bytes and the epilogue's conversions and stores where it is short (192360 x 117 -> 16 fp32: 21 us; 55 with the columns' scales
// passed by shuffles and an address multiplied out for every store).
#include <cuda.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "../../include/converse_b200.h"
#include "cvb_int8.cuh"
#include "cvb_internal.h"
#include "cvb_tc.cuh"

namespace cvb {
namespace i8 {

// ------------------------------------------------------------------ quantisation
struct QuantParams {
  const void* x;
  signed char* q;
  float* scale;
  long long B, HW, tokens, ldq;
  int K, tiles, tpr;
};

template <typename IO>
__device__ __forceinline__ float load1(const void* p, long long i);
template <>
__device__ __forceinline__ float load1<float>(const void* p, long long i) { return ((const float*)p)[i]; }
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const void* p, long long i) { return __bfloat162float(((const __nv_bfloat16*)p)[i]); }

// channels_first: 32 pixels a block, warp s takes channels 32 s .. of each group of 32 S; more than one group is read twice.  (Of
// 4 x 3460 x 2550 bf16 with 8 warps a block the quantising took 260 us.)
constexpr int kQuantWarps = 32;
template <typename IO, int MAXT>
__global__ void __launch_bounds__(MAXT) quant_first_kernel(const __grid_constant__ QuantParams P) {
  pdl_start();
  __shared__ float red[kQuantWarps][32];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, S = blockDim.x >> 5;
  const long long b = blockIdx.x / P.tiles, px = (long long)(blockIdx.x - b * P.tiles) * 32 + lane;
  const bool live = px < P.HW;
  const IO* x = (const IO*)P.x + b * P.K * P.HW + (live ? px : P.HW - 1);
  const long long token = b * P.HW + px;
  float v[32], a = 0.f;
  auto fetch = [&](int c0) {
    const IO* p = x + c0 * P.HW;
    if (c0 + 32 <= P.K) {
#pragma unroll
      for (int i = 0; i < 32; ++i, p += P.HW) v[i] = load1<IO>(p, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i, p += P.HW) v[i] = c0 + i < P.K ? load1<IO>(p, 0) : 0.f;
    }
  };
  for (int c0 = 32 * s; c0 < P.K; c0 += 32 * S) {
    fetch(c0);
#pragma unroll
    for (int i = 0; i < 32; i += 2) a = largest(a, v[i], v[i + 1]);
  }
  if (S > 1) {
    red[s][lane] = a;
    __syncthreads();
    for (int t = 0; t < S; ++t) a = largest(a, red[t][lane]);
  }
  if (!live) return;
  const Quantiser<sizeof(IO) == 2> q(a);
  if (s == 0) P.scale[token] = q.scale();
  for (int c0 = 32 * s; c0 < P.K; c0 += 32 * S) {
    if (P.K > 32 * S) fetch(c0);
    signed char* to = P.q + token * P.ldq + c0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = q.four(v[16 * h + 4 * i], v[16 * h + 4 * i + 1], v[16 * h + 4 * i + 2], v[16 * h + 4 * i + 3]);
      if (c0 + 16 * h < P.K) *(uint4*)(to + 16 * h) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// channels_last: a warp a token, or fewer threads of it (tpr) where that is enough for one piece each.  A row is read in the 16-byte
// pieces of memory that it lies in, wherever it begins: the bytes that a piece gives belong `shift` places further to the left, so
// a thread joins its own with its neighbour's before it stores them.  NV pieces of a thread stay in registers as they were loaded;
// rows of more than 32 NV pieces are read twice.  (Element by element, rows of odd lengths took 228 us for 30456 x 1796 bf16.  With
// 256 threads a token of 4096 channels most of the work was what a thread does once: 41 us for 8192 tokens.)
__device__ __forceinline__ float half_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// the first or the last piece of a row, element by element (a function: it would be part of every load)
template <typename IO>
static __device__ __noinline__ uint4 edge_piece(const char* p, const char* from, const char* to) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(IO); ++j) {
    const char* q = p + j * (int)sizeof(IO);
    if (q < from || q >= to) continue;
    if (sizeof(IO) == 4) w[j & 3] = *(const uint32_t*)q;
    else w[(j >> 1) & 3] |= (uint32_t)*(const unsigned short*)q << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename IO>
struct Piece {
  static constexpr int V = 16 / (int)sizeof(IO);
  using Bytes = std::conditional_t<V == 4, uint32_t, uint64_t>;
  uint4 v;
  __device__ __forceinline__ float top(float a) const {
    if (sizeof(IO) == 4)
      return largest(largest(a, __uint_as_float(v.x), __uint_as_float(v.y)), __uint_as_float(v.z), __uint_as_float(v.w));
    a = largest(largest(a, half_lo(v.x), half_hi(v.x)), half_lo(v.y), half_hi(v.y));
    return largest(largest(a, half_lo(v.z), half_hi(v.z)), half_lo(v.w), half_hi(v.w));
  }
  // its V integers, the first one lowest
  __device__ __forceinline__ Bytes bytes(const Quantiser<sizeof(IO) == 2>& q) const {
    if constexpr (V == 4) {
      return q.four(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    } else {
      const uint32_t lo = q.four(half_lo(v.x), half_hi(v.x), half_lo(v.y), half_hi(v.y));
      const uint32_t hi = q.four(half_lo(v.z), half_hi(v.z), half_lo(v.w), half_hi(v.w));
      return (uint64_t)hi << 32 | lo;
    }
  }
};

// EVEN: every row begins with a piece and ends with one
template <typename IO, int NV, bool EVEN>
__global__ void __launch_bounds__(256, NV == 16 ? 2 : 3) quant_last_kernel(const __grid_constant__ QuantParams P) {
  pdl_start();
  using Bytes = typename Piece<IO>::Bytes;
  constexpr int V = Piece<IO>::V;
  const int tpr = P.tpr, t = threadIdx.x & (tpr - 1);
  const long long token = (long long)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  const bool live = token < P.tokens;
  const int K = live ? P.K : 0;
  const IO* row = (const IO*)P.x + (live ? token : 0) * P.K;
  const int shift = EVEN ? 0 : (int)((size_t)row & 15) / (int)sizeof(IO);          // values of the first piece that lie before the row
  const char* first = (const char*)(row - shift);
  const int pieces = (K + shift + V - 1) / V, whole_from = shift != 0, whole_to = (K + shift) / V;
  const int rounds = (pieces + NV * tpr - 1) / (NV * tpr);
  Piece<IO> v[NV];
  auto fetch = [&](int round) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = (round * NV + i) * tpr + t;
      if (p >= whole_from && p < whole_to) v[i].v = *(const uint4*)(first + (long long)p * 16);
      else if (EVEN || p >= pieces) v[i].v = make_uint4(0, 0, 0, 0);
      else v[i].v = edge_piece<IO>(first + (long long)p * 16, (const char*)row, (const char*)(row + K));
    }
  };
  float a = 0.f;
  for (int r = 0; r < rounds; ++r) {
    fetch(r);
#pragma unroll
    for (int i = 0; i < NV; ++i) a = v[i].top(a);
  }
  for (int o = tpr >> 1; o; o >>= 1) a = largest(a, __shfl_xor_sync(0xffffffffu, a, o));
  const Quantiser<sizeof(IO) == 2> q(a);
  if (t == 0 && live) P.scale[token] = q.scale();
  signed char* out = P.q + token * P.ldq;
  // Every lane of the warp takes part in the shuffles, with as many rounds as any of its rows; from the rows' ends to their
  // beginnings, for the bytes behind a thread's own are needed first.
  int most = rounds;
  for (int o = 16; o >= tpr; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  Bytes behind = 0;          // of the first of the tpr pieces behind
  for (int r = most - 1; r >= 0; --r) {
    if (most > 1) fetch(r);
#pragma unroll
    for (int i = NV - 1; i >= 0; --i) {
      Bytes w = v[i].bytes(q);
      if (!EVEN) {
        const Bytes own = w, beside = __shfl_down_sync(0xffffffffu, own, 1, tpr), next = t == tpr - 1 ? behind : beside;
        if (NV > 1 || most > 1) behind = __shfl_sync(0xffffffffu, own, 0, tpr);
        if (shift) w = own >> (8 * shift) | next << (8 * (V - shift));
      }
      const int c = ((r * NV + i) * tpr + t) * V;
      if (c < K) *(Bytes*)(out + c) = w;          // (behind the last channel zeros: rows are that long)
    }
  }
}

// ------------------------------------------------------------------ product
constexpr int kM = 128, kBK = 128;                     // rows of L in a tile; bytes of K in a stage
constexpr int kMostK = 131072;                         // sums from -127 . 128 . 2^17 to 2^31
constexpr int kEpilogueWarps = 8, kThreads = 32 * (4 + kEpilogueWarps);
constexpr int kPolls = 1 << 20;

struct ProductParams {
  const float *l_scale, *r_scale, *l_bias, *r_bias;    // by row of L (of all images), by row of R
  void* out;
  long long images, rows, cols;        // of each image: rows of L, and of R
  long long image_stride, ldc;         // elements of the output
  int K, row_tiles, col_tiles;
  long long tiles;
  int* status;
};

__host__ __device__ constexpr int stages_of(int NT) { return NT == 256 ? 4 : NT == 128 ? 6 : 8; }
__host__ __device__ constexpr int stage_bytes(int NT) { return (kM + NT) * kBK; }

__device__ __forceinline__ uint64_t swizzled_desc(const void* p) {
  uint64_t d = (uint64_t)((smem_u32(p) >> 4) & 0x3FFF);
  d |= (uint64_t)1 << 16;                              // (not read for swizzled K-major operands)
  d |= (uint64_t)(1024 >> 4) << 32;                    // eight rows of 128 bytes
  d |= (uint64_t)1 << 46;                              // version
  d |= (uint64_t)2 << 61;                              // 128-byte swizzle
  return d;
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t elected) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t"
      ".reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tmem_ld32i(uint32_t taddr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// every lane waits, and all of them learn the same
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, kPolls));
}

struct Tile {
  long long image;
  int row, col;          // first row of L in the image, first row of R
  __device__ __forceinline__ Tile(const ProductParams& P, long long t, int NT) {
    const unsigned r = (unsigned)t / (unsigned)P.col_tiles, b = r / (unsigned)P.row_tiles;
    col = ((unsigned)t - r * P.col_tiles) * NT;
    image = b;
    row = (r - b * P.row_tiles) * kM;
  }
};

__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// LAST: the rows of L are output channels, else pixels.  The sum is multiplied by the weights' scale first: a token's may be of any
// size, and its product with a large sum no fp32 number although the result is one.
template <typename IO, int NT, bool LAST>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap mapL, const __grid_constant__ CUtensorMap mapR,
               const __grid_constant__ ProductParams P) {
  constexpr int ST = stages_of(NT);
  extern __shared__ unsigned char dynamic[];
  unsigned char* const ring = dynamic + (-smem_u32(dynamic) & 1023);       // the swizzle counts from 1024-byte boundaries
  __shared__ uint64_t full[ST], empty[ST], done[2], free_[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) float columns[kEpilogueWarps][LAST ? NT / 2 : NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The wait comes before tensor memory is taken, and the next kernel is let in behind it: a block that held tensor memory while it
  // waited for a kernel whose blocks still have to take theirs would wait for ever.
  pdl_wait();
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&done[i], 1), mbar_init(&free_[i], kEpilogueWarps);
    mbar_init(&drained, 1);
    mbar_fence_init();
  }
  if (warp == 2) tc::tmem_alloc(&tmem_base, 2 * NT);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_let_next();
  const uint32_t tmem = tmem_base;
  const int kblocks = (P.K + kBK - 1) / kBK;
  bool ok = true;
  if (warp == 0) {
    // copies
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      long long issued = 0;
      for (long long t = blockIdx.x; t < P.tiles && ok; t += gridDim.x) {
        const Tile tile(P, t, NT);
        const int row = (int)(tile.image * P.rows) + tile.row;
        for (int k = 0; k < kblocks; ++k) {
          ok = mbar_wait_bounded(&empty[st], ph ^ 1, kPolls);
          if (!ok) break;
          unsigned char* at = ring + st * stage_bytes(NT);
          mbar_expect_tx(&full[st], stage_bytes(NT));
          tma_2d(at, &mapL, k * kBK, row, &full[st]);
          tma_2d(at + kM * kBK, &mapR, k * kBK, tile.col, &full[st]);
          ++issued;
          if (++st == ST) st = 0, ph ^= 1;
        }
      }
      if (!ok) {
        // no copy may be in flight when the block ends
        for (int i = 0; i < ST; ++i) {
          const long long uses = issued > i ? (issued - 1 - i) / ST + 1 : 0;
          if (uses) mbar_wait_bounded(&full[i], (uint32_t)((uses - 1) & 1), kPolls);
        }
      }
    }
  } else if (warp == 1) {
    // MMAs
    const uint32_t elected = tc::elect_one();
    const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
    int st = 0, acc = 0;
    uint32_t ph = 0, aph = 0;
    for (long long t = blockIdx.x; t < P.tiles && ok; t += gridDim.x) {
      ok = warp_wait(&free_[acc], aph ^ 1);
      if (!ok) break;
      tc::fence_after_sync();
      for (int k = 0; k < kblocks; ++k) {
        ok = warp_wait(&full[st], ph);
        if (!ok) break;
        tc::fence_after_sync();
        const unsigned char* at = ring + st * stage_bytes(NT);
        const uint64_t a = swizzled_desc(at), b = swizzled_desc(at + kM * kBK);
        const int steps = min(kBK / 32, (P.K - k * kBK + 31) / 32);
        for (int s = 0; s < steps; ++s) mma_i8(tmem + acc * NT, a + 2 * s, b + 2 * s, idesc, (k | s) != 0, elected);
        commit(&empty[st], elected);
        if (++st == ST) st = 0, ph ^= 1;
      }
      if (!ok) break;
      commit(&done[acc], elected);
      if (acc) aph ^= 1;
      acc ^= 1;
    }
    commit(&drained, elected);
    if (!warp_wait(&drained, 0)) ok = false;
  } else if (warp >= 4) {
    // lane r of quadrant w & 3; the two warps of a quadrant take half of the columns each.  The columns' scales (and biases) lie in
    // the warp's shared memory, loaded before the sums are waited for.
    const int quadrant = warp & 3, half = (warp - 4) >> 2;
    float* const rs = columns[warp - 4];
    float* const rb = rs + NT / 2;
    int acc = 0;
    uint32_t aph = 0;
    for (long long t = blockIdx.x; t < P.tiles; t += gridDim.x) {
      const Tile tile(P, t, NT);
      const int r = tile.row + quadrant * 32 + lane;
      const bool live = r < P.rows;
      const float ls = live ? P.l_scale[tile.image * P.rows + r] : 0.f, lb = LAST && live && P.l_bias ? P.l_bias[r] : 0.f;
      const int c0 = tile.col + half * (NT / 2), left = (int)(P.cols - c0 < NT / 2 ? P.cols - c0 : NT / 2);
      __syncwarp();          // the tile's before are read
#pragma unroll
      for (int c = 0; c < NT / 2; c += 32) {
        const bool in = c + lane < left;
        rs[c + lane] = in ? P.r_scale[c0 + c + lane] : 0.f;
        if (!LAST) rb[c + lane] = in && P.r_bias ? P.r_bias[c0 + c + lane] : 0.f;
      }
      __syncwarp();
      ok = warp_wait(&done[acc], aph);
      if (!ok) break;
      tc::fence_after_sync();
      if (__any_sync(0xffffffffu, live)) {
        IO* out = (IO*)P.out + tile.image * P.image_stride + (long long)c0 * P.ldc + r;
        for (int c = 0; c < left; c += 32) {
          int v[32];
          __syncwarp();          // (not every lane has stored what is before)
          tmem_ld32i(tmem + acc * NT + half * (NT / 2) + c + ((uint32_t)(quadrant * 32) << 16), v);
          if (P.K == kMostK) {          // 2^31 = 131072 . 128 . 128 came out as -2^31, which no other sum is: 2^31 - 1 is 2^31 in fp32
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = v[j] == INT_MIN ? INT_MAX : v[j];
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *(const float4*)(rs + c + j);
            const float s[4] = {s4.x, s4.y, s4.z, s4.w};
            float o[4] = {lb, lb, lb, lb};
            if (!LAST) {
              const float4 o4 = *(const float4*)(rb + c + j);
              o[0] = o4.x; o[1] = o4.y; o[2] = o4.z; o[3] = o4.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float y = LAST ? fmaf((float)v[j + i] * ls, s[i], o[i]) : fmaf((float)v[j + i] * s[i], ls, o[i]);
              if (live && c + j + i < left) store1(out, y);
              out += P.ldc;
            }
          }
        }
      }
      __syncwarp();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&free_[acc]);
      if (acc) aph ^= 1;
      acc ^= 1;
    }
  }
  if (!ok && lane == 0 && P.status) *P.status = 1;
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 2) tc::tmem_dealloc(tmem, 2 * NT);
}

// ------------------------------------------------------------------ launches
static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static int encode_tiled(EncodeTiled* out) {
  static std::atomic<EncodeTiled> known{nullptr};          // (looked up twice at worst)
  EncodeTiled fn = known.load(std::memory_order_acquire);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    CVB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !p) return CVB_ERR_CUDA;
    fn = (EncodeTiled)p;
    known.store(fn, std::memory_order_release);
  }
  *out = fn;
  return CVB_OK;
}
// rows x K bytes, boxes of 128 bytes x box_rows
static int row_map(CUtensorMap* m, const signed char* p, long long rows, int K, long long ld, int box_rows) {
  EncodeTiled encode;
  const int rc = encode_tiled(&encode);
  if (rc != CVB_OK) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows}, step[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)p, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? CVB_OK : CVB_ERR_BAD_ARGUMENT;
}

template <typename IO>
static int quantize_last(QuantParams& P, cudaStream_t st) {
  constexpr int V = Piece<IO>::V;
  const bool even = P.K % V == 0 && (size_t)P.x % 16 == 0;          // every row begins with a piece
  const int pieces = (P.K + (even ? 0 : V - 1) + V - 1) / V;
  P.tpr = 1;
  while (P.tpr < 32 && P.tpr < pieces) P.tpr *= 2;
  const dim3 grid((unsigned)ceil_div(P.tokens, 256 / P.tpr));
  const int each = ceil_div(pieces, P.tpr);
  auto go = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    return even ? launch_chained(quant_last_kernel<IO, NV, true>, grid, 256, 0, st, P)
                : launch_chained(quant_last_kernel<IO, NV, false>, grid, 256, 0, st, P);
  };
  return each == 1   ? go(std::integral_constant<int, 1>())
         : each == 2 ? go(std::integral_constant<int, 2>())
         : each <= 4 ? go(std::integral_constant<int, 4>())
                     : go(std::integral_constant<int, 16>());
}
template <typename IO>
static int quantize(QuantParams& P, bool last, cudaStream_t st) {
  if (!last) {
    P.tiles = ceil_div(P.HW, 32);
    const int S = min(kQuantWarps, ceil_div(P.K, 32));
    const dim3 grid((unsigned)(P.tiles * P.B));
    return S <= 8 ? launch_chained(quant_first_kernel<IO, 256>, grid, 32 * S, 0, st, P)
                  : launch_chained(quant_first_kernel<IO, 1024>, grid, 32 * S, 0, st, P);
  }
  return quantize_last<IO>(P, st);
}

template <typename IO, int NT, bool LAST>
static int product(ProductParams& P, const signed char* l, long long lrows, long long ldl, const signed char* r, long long rrows,
                   long long ldr, int sms, cudaStream_t st) {
  CUtensorMap mapL, mapR;
  int rc = row_map(&mapL, l, lrows, P.K, ldl, kM);
  if (rc == CVB_OK) rc = row_map(&mapR, r, rrows, P.K, ldr, NT);
  if (rc != CVB_OK) return rc;
  P.row_tiles = ceil_div(P.rows, kM);
  P.col_tiles = ceil_div(P.cols, NT);
  P.tiles = P.images * P.row_tiles * P.col_tiles;
  if (P.tiles > 0x7fffffffll) return CVB_ERR_TOO_LARGE;
  const size_t smem = (size_t)stages_of(NT) * stage_bytes(NT) + 1024;
  CVB_CUDA(cudaFuncSetAttribute(product_kernel<IO, NT, LAST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_chained(product_kernel<IO, NT, LAST>, dim3((unsigned)(P.tiles < sms ? P.tiles : sms)), kThreads, smem, st, mapL, mapR, P);
}
template <typename IO>
static int product_any(const signed char* q, long long ldq, const float* scale, const signed char* w, long long ldw,
                       const float* w_scale, const float* bias, void* out, long long B, long long HW, int K, int N, bool last,
                       int sms, int* status, cudaStream_t st) {
  ProductParams P;
  memset(&P, 0, sizeof(P));
  P.out = out; P.K = K; P.status = status;
  const long long tokens = B * HW;
  if (last) {
    P.l_scale = w_scale; P.l_bias = bias; P.r_scale = scale;
    P.images = 1; P.rows = N; P.cols = tokens; P.ldc = N;
  } else {
    P.l_scale = scale; P.r_scale = w_scale; P.r_bias = bias;
    P.images = B; P.rows = HW; P.cols = N; P.ldc = HW; P.image_stride = (long long)N * HW;
  }
  const signed char *l = last ? w : q, *r = last ? q : w;
  const long long lrows = last ? N : tokens, rrows = last ? tokens : N, ldl = last ? ldw : ldq, ldr = last ? ldq : ldw;
  // the widest tile that leaves a tile for every multiprocessor
  auto tiles = [&](int NT) { return P.images * ceil_div(P.rows, kM) * ceil_div(P.cols, NT); };
  const int NT = P.cols > 128 && tiles(256) >= sms ? 256 : P.cols > 64 && tiles(128) >= sms ? 128 : 64;
  auto go = [&](auto nt, auto l_last) {
    return product<IO, decltype(nt)::value, decltype(l_last)::value>(P, l, lrows, ldl, r, rrows, ldr, sms, st);
  };
  auto by_width = [&](auto l_last) {
    return NT == 256   ? go(std::integral_constant<int, 256>(), l_last)
           : NT == 128 ? go(std::integral_constant<int, 128>(), l_last)
                       : go(std::integral_constant<int, 64>(), l_last);
  };
  return last ? by_width(std::true_type()) : by_width(std::false_type());
}

int run_quantize(const void* x, signed char* q, float* scale, long long B, long long HW, int K, long long ldq, bool last, int io,
                 cudaStream_t st) {
  QuantParams P;
  P.x = x; P.q = q; P.scale = scale; P.B = B; P.HW = HW; P.tokens = B * HW; P.ldq = ldq; P.K = K; P.tiles = P.tpr = 0;
  return io == CVB_F32 ? quantize<float>(P, last, st) : quantize<__nv_bfloat16>(P, last, st);
}
int run_product(const signed char* q, long long ldq, const float* scale, const signed char* w, long long ldw, const float* w_scale,
                const float* bias, void* out, long long B, long long HW, int K, int N, bool last, int io, int sms, int* status,
                cudaStream_t st) {
  return io == CVB_F32 ? product_any<float>(q, ldq, scale, w, ldw, w_scale, bias, out, B, HW, K, N, last, sms, status, st)
                       : product_any<__nv_bfloat16>(q, ldq, scale, w, ldw, w_scale, bias, out, B, HW, K, N, last, sms, status, st);
}
// where x is quantised on the way there is no workspace
size_t workspace(long long B, long long HW, int K, int N, bool last, int io, int sms) {
  const long long tokens = B * HW;
  if (!last && planes_take(B, HW, K, N, io, sms)) return 0;
  return ((size_t)tokens * ((K + 15) / 16 * 16) + 255) / 256 * 256 + (size_t)tokens * sizeof(float);
}
int run_pointwise(const void* x, const signed char* w, long long ldw, const float* w_scale, const float* bias, void* out,
                  long long B, long long HW, int K, int N, bool last, int io, void* ws, int sms, int* status, cudaStream_t st) {
  if (!last && planes_take(B, HW, K, N, io, sms))
    return run_planes(x, w, ldw, w_scale, bias, out, B, HW, K, N, io, sms, status, st);
  const long long ldq = (K + 15) / 16 * 16, tokens = B * HW;
  signed char* q = (signed char*)ws;
  float* scale = (float*)((char*)ws + ((size_t)tokens * ldq + 255) / 256 * 256);
  const int rc = run_quantize(x, q, scale, B, HW, K, ldq, last, io, st);
  return rc != CVB_OK ? rc : run_product(q, ldq, scale, w, ldw, w_scale, bias, out, B, HW, K, N, last, io, sms, status, st);
}

}  // namespace i8
}  // namespace cvb
