// The norm of many tensors together, and the tensors scaled so that it does not exceed a largest value:
//     norm = ( sum over tensors and elements of |g|^p )^(1/p),  p = 1, 2 or infinity (the largest magnitude)
//     out  = g . min(1, max_norm / (norm + 1e-6))
// Two kernels.  The first leaves a partial result for each of its blocks, in 64 bits; every block of the second reduces all of
// them, in the same order, and scales its share: no atomics, no counters to clear, the same bits at every run.
//
// The tensors' addresses travel in the kernels' parameters (up to 31 KB of them), so nothing is copied to the device and a
// captured graph holds its own table.  Work is cut into chunks of kChunk elements that belong to one tensor; a block finds the
// tensor of a chunk by bisection.
//
// Squares of fp32 numbers leave fp32's range (1e20 squared).  A thread adds the squares of eight elements in fp32 where their
// largest magnitude lies between 2^-40 and 2^50 (what is then lost to underflow is below 2^-60 of the sum), else it squares
// them in 64 bits; each sum of eight goes into a 64-bit one.
//
// 48 tensors, 64 M fp32 values, outputs at odd places: 43 us for the norm, 138 for both (78 if every value were read once; the norm has
// to be known before the first store).  The scaling kernel goes backwards, from what is still in the L2 cache; outputs are stored from
// 128-byte boundaries on (from anywhere: 150 us).  284 tensors, 0.56 M values: 13 us on the device.
#include "../../include/converse_b200.h"
#include "cvb_internal.h"

namespace cvb {

constexpr int kClipThreads = 256, kClipPer = 16, kChunk = kClipThreads * kClipPer;   // elements of a chunk
constexpr int kClipBlocksPerSm = 8;
constexpr int kClipTensors = 960;          // of one launch
// chunks that the second kernel may find in the L2 cache: measured for fp32, 75 MB.  (Of bf16 they are 38 MB, and more of them might stay;
// not measured.)
constexpr unsigned kClipKept = 4600;

struct ClipItem {
  const void* in;
  void* out;
  unsigned first;          // its first chunk in the launch
  unsigned n_low;
  unsigned short n_high, types;      // elements: n_high . 2^32 + n_low; types: bit 0 in bf16, bit 1 out bf16, bit 2 vectors
  unsigned ahead;          // elements that its first chunk lacks, so that the others begin at 16 bytes of in, or 128 of out
};
static_assert(sizeof(ClipItem) == 32, "");
template <int N>
struct ClipParams {
  double* partial;         // of this launch's blocks (first kernel); of all (second)
  float* norm;
  double max_norm;
  int partials;            // second kernel: how many
  int count;
  unsigned chunks;
  unsigned passing;        // first kernel: chunks read as used for the last time
  int kind;                // 1, 2, or 0 for the largest magnitude
  int writes_norm;
  ClipItem item[N];
};

__device__ __forceinline__ float2 clip_bf2(unsigned v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// eight elements from `i` on (all inside the tensor)
template <bool BF16, bool LAST_USE>
__device__ __forceinline__ void clip_load8(const void* p, long long i, float (&v)[8]) {
  if (BF16) {
    const uint4* q = (const uint4*)((const unsigned short*)p + i);
    const uint4 u = LAST_USE ? __ldcs(q) : *q;
    const float2 a = clip_bf2(u.x), b = clip_bf2(u.y), c = clip_bf2(u.z), d = clip_bf2(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  } else {
    const float4* q = (const float4*)((const float*)p + i);
    const float4 a = LAST_USE ? __ldcs(q) : *q, b = LAST_USE ? __ldcs(q + 1) : q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}
template <bool BF16, bool LAST_USE>
__device__ __forceinline__ float clip_load1(const void* p, long long i) {
  if (BF16) {
    const unsigned short* q = (const unsigned short*)p + i;
    return __uint_as_float((unsigned)(LAST_USE ? __ldcs(q) : *q) << 16);
  }
  const float* q = (const float*)p + i;
  return LAST_USE ? __ldcs(q) : *q;
}

// NaN stays
__device__ __forceinline__ double clip_join(double a, double b, int kind) {
  if (kind) return a + b;
  return a > b || a != a ? a : b;
}
__device__ __forceinline__ void clip_add8(const float (&v)[8], double& acc, int kind) {
  if (kind == 2) {
    float m = 0.f, s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m = fmaxf(m, fabsf(v[j]));
      s = fmaf(v[j], v[j], s);
    }
    if (m > 9.1e-13f && m < 1.1e15f && s == s) {
      acc += (double)s;
    } else if (m > 0.f || s != s) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc = fma((double)v[j], (double)v[j], acc);
    }
  } else if (kind == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc += (double)fabsf(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = clip_join(acc, (double)fabsf(v[j]), 0);
  }
}

// sum (or largest) over the block, in every thread
__device__ __forceinline__ double clip_block_join(double v, int kind) {
  __shared__ double part[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = clip_join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int j = 1; j < kClipThreads / 32; ++j) v = clip_join(v, part[j], kind);
  return v;
}

template <int N>
__device__ __forceinline__ int clip_find(const ClipParams<N>& P, unsigned chunk, int lo) {
  int hi = P.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (P.item[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// the elements of a chunk: [begin, end) of the tensor
__device__ __forceinline__ void clip_range(const ClipItem& t, unsigned chunk, long long& begin, long long& end) {
  const long long n = ((long long)t.n_high << 32) + t.n_low;
  begin = (long long)(chunk - t.first) * kChunk - t.ahead;
  end = begin + kChunk < n ? begin + kChunk : n;
  if (begin < 0) begin = 0;
}

template <bool BF16, bool LAST_USE>
__device__ __forceinline__ void clip_chunk_norm(const ClipItem& t, long long begin, long long end, double& acc, int kind) {
  const int tid = threadIdx.x;
  if (end - begin == kChunk && ((size_t)((const char*)t.in + begin * (BF16 ? 2 : 4)) & 15) == 0) {
    float v[kClipPer / 8][8];
#pragma unroll
    for (int j = 0; j < kClipPer / 8; ++j) clip_load8<BF16, LAST_USE>(t.in, begin + 8 * (j * kClipThreads + tid), v[j]);
#pragma unroll
    for (int j = 0; j < kClipPer / 8; ++j) clip_add8(v[j], acc, kind);
    return;
  }
#pragma unroll
  for (int h = 0; h < kClipPer / 8; ++h) {
    float v[8];
    const long long at = begin + (long long)h * 8 * kClipThreads + tid;
    if (begin + (long long)h * 8 * kClipThreads >= end) break;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at + j * kClipThreads < end ? clip_load1<BF16, LAST_USE>(t.in, at + j * kClipThreads) : 0.f;
    clip_add8(v, acc, kind);
  }
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipParams<N> P) {
  pdl_start();
  double acc = 0;
  int at = 0;
  for (unsigned c = blockIdx.x; c < P.chunks; c += gridDim.x) {
    at = clip_find(P, c, at);
    const ClipItem& t = P.item[at];
    long long begin, end;
    clip_range(t, c, begin, end);
    // what will not be in the L2 cache any more when the second kernel comes to it makes room for what will
    if (c < P.passing) {
      if (t.types & 1) clip_chunk_norm<true, true>(t, begin, end, acc, P.kind);
      else clip_chunk_norm<false, true>(t, begin, end, acc, P.kind);
    } else {
      if (t.types & 1) clip_chunk_norm<true, false>(t, begin, end, acc, P.kind);
      else clip_chunk_norm<false, false>(t, begin, end, acc, P.kind);
    }
  }
  acc = clip_block_join(acc, P.kind);
  if (threadIdx.x == 0) P.partial[blockIdx.x] = acc;
}

template <bool INBF, bool OUTBF>
__device__ __forceinline__ void clip_chunk_scale(const ClipItem& t, long long begin, long long end, float c) {
  const int tid = threadIdx.x;
  if (end - begin == kChunk && (t.types & 4)) {
    float v[kClipPer / 8][8];
#pragma unroll
    for (int j = 0; j < kClipPer / 8; ++j) clip_load8<INBF, true>(t.in, begin + 8 * (j * kClipThreads + tid), v[j]);
#pragma unroll
    for (int j = 0; j < kClipPer / 8; ++j) {
      const long long i = begin + 8 * (j * kClipThreads + tid);
      if (OUTBF) {
        __nv_bfloat162 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __floats2bfloat162_rn(v[j][2 * e] * c, v[j][2 * e + 1] * c);
        __stcs((uint4*)((__nv_bfloat16*)t.out + i), *(const uint4*)w);
      } else {
        __stcs((float4*)((float*)t.out + i), make_float4(v[j][0] * c, v[j][1] * c, v[j][2] * c, v[j][3] * c));
        __stcs((float4*)((float*)t.out + i + 4), make_float4(v[j][4] * c, v[j][5] * c, v[j][6] * c, v[j][7] * c));
      }
    }
    return;
  }
  // not both at vectors: neighbouring threads take neighbouring elements, all of them in flight at once; out's lines are whole
  float v[kClipPer];
#pragma unroll
  for (int j = 0; j < kClipPer; ++j) {
    const long long i = begin + j * kClipThreads + tid;
    v[j] = i < end ? clip_load1<INBF, true>(t.in, i) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kClipPer; ++j) {
    const long long i = begin + j * kClipThreads + tid;
    if (i >= end) continue;
    if (OUTBF) ((__nv_bfloat16*)t.out)[i] = __float2bfloat16_rn(v[j] * c);
    else ((float*)t.out)[i] = v[j] * c;
  }
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_scale_kernel(const __grid_constant__ ClipParams<N> P) {
  pdl_start();
  double acc = 0;
  for (int j = threadIdx.x; j < P.partials; j += kClipThreads) acc = clip_join(acc, P.partial[j], P.kind);
  acc = clip_block_join(acc, P.kind);
  const double norm = P.kind == 2 ? sqrt(acc) : acc;
  if (P.writes_norm && blockIdx.x == 0 && threadIdx.x == 0) *P.norm = (float)norm;
  const double ratio = P.max_norm / (norm + 1e-6);
  const float c = ratio >= 1.0 ? 1.f : (float)ratio;           // NaN stays
  // the chunks that the first kernel read last are the ones still in the L2 cache
  for (unsigned k = blockIdx.x; k < P.chunks; k += gridDim.x) {
    const unsigned chunk = P.chunks - 1 - k;
    const ClipItem& t = P.item[clip_find(P, chunk, 0)];
    if (c == 1.f && t.in == t.out) continue;                   // nothing to change
    long long begin, end;
    clip_range(t, chunk, begin, end);
    switch (t.types & 3) {
      case 0: clip_chunk_scale<false, false>(t, begin, end, c); break;
      case 1: clip_chunk_scale<true, false>(t, begin, end, c); break;
      case 2: clip_chunk_scale<false, true>(t, begin, end, c); break;
      default: clip_chunk_scale<true, true>(t, begin, end, c); break;
    }
  }
}

static int clip_blocks(unsigned chunks, int sms) {
  const unsigned most = (unsigned)(kClipBlocksPerSm * sms);
  return (int)(chunks < most ? chunks : most);
}

// one launch of either kernel for the tensors [from, to)
template <int N>
static int clip_launch(const cvb_span* spans, int from, int to, bool scale, const ClipParams<1>& base, int& blocks, int sms,
                       cudaStream_t st) {
  static thread_local ClipParams<N> P;
  P.partial = base.partial; P.norm = base.norm; P.max_norm = base.max_norm; P.partials = base.partials; P.kind = base.kind;
  P.writes_norm = base.writes_norm;
  unsigned long long all = 0;
  unsigned chunks = 0;
  int count = 0;
  for (int i = from; i < to; ++i) {
    const cvb_span& s = spans[i];
    if (s.n == 0) continue;
    ClipItem& t = P.item[count++];
    t.in = s.in; t.out = s.out; t.first = chunks;
    const int in_size = s.in_type == CVB_BF16 ? 2 : 4, out_size = s.out_type == CVB_BF16 ? 2 : 4;
    t.ahead = scale ? (unsigned)((size_t)s.out % 128 / out_size) : (unsigned)((size_t)s.in % 16 / in_size);
    t.n_low = (unsigned)s.n; t.n_high = (unsigned short)(s.n >> 32);
    const bool vectors = (((size_t)s.in - t.ahead * in_size) & 15) == 0 && (((size_t)s.out - t.ahead * out_size) & 15) == 0;
    t.types = (unsigned short)((s.in_type == CVB_BF16) | (s.out_type == CVB_BF16) << 1 | vectors << 2);
    all += (unsigned long long)(s.n + t.ahead + kChunk - 1) / kChunk;
    if (all > 0x7fffffffull) return CVB_ERR_TOO_LARGE;
    chunks = (unsigned)all;
  }
  P.count = count;
  P.chunks = chunks;
  // about what the L2 cache holds beside the outputs (4600 chunks of fp32 are 75 MB)
  P.passing = chunks > kClipKept ? chunks - kClipKept : 0;
  blocks = clip_blocks(chunks, sms);
  if (!scale && !chunks) return CVB_OK;
  return launch_chained(scale ? clip_scale_kernel<N> : clip_norm_kernel<N>, dim3(blocks ? blocks : 1), kClipThreads, 0, st, P);
}
static int clip_launch_any(const cvb_span* spans, int from, int to, bool scale, const ClipParams<1>& base, int& blocks, int sms,
                           cudaStream_t st) {
  // the parameters are copied at every launch: no more room than the tensors need
  const int n = to - from;
  if (n <= 16) return clip_launch<16>(spans, from, to, scale, base, blocks, sms, st);
  if (n <= 128) return clip_launch<128>(spans, from, to, scale, base, blocks, sms, st);
  if (n <= 384) return clip_launch<384>(spans, from, to, scale, base, blocks, sms, st);
  return clip_launch<kClipTensors>(spans, from, to, scale, base, blocks, sms, st);
}

size_t clip_workspace(int count, int sms) {
  const size_t launches = count > 0 ? ((size_t)count + kClipTensors - 1) / kClipTensors : 1;
  return launches * kClipBlocksPerSm * sms * sizeof(double);
}

int run_clip(const cvb_span* spans, int count, int kind, double max_norm, bool scale, float* norm, void* workspace, int sms,
             cudaStream_t st) {
  ClipParams<1> base;
  memset(&base, 0, sizeof(base));
  base.partial = (double*)workspace; base.norm = norm; base.max_norm = max_norm; base.kind = kind;
  int total = 0, blocks = 0;
  for (int from = 0; from < count; from += kClipTensors) {
    base.partial = (double*)workspace + total;
    const int rc = clip_launch_any(spans, from, from + kClipTensors < count ? from + kClipTensors : count, false, base, blocks, sms, st);
    if (rc != CVB_OK) return rc;
    total += blocks;
  }
  base.partial = (double*)workspace;
  base.partials = total;
  base.writes_norm = 1;
  if (!scale || !count) return clip_launch_any(spans, 0, 0, true, base, blocks, sms, st);
  for (int from = 0; from < count; from += kClipTensors) {
    const int rc = clip_launch_any(spans, from, from + kClipTensors < count ? from + kClipTensors : count, true, base, blocks, sms, st);
    if (rc != CVB_OK) return rc;
    base.writes_norm = 0;
  }
  return CVB_OK;
}

}  // namespace cvb
