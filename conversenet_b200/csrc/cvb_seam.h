// What the kernels of the residual seam (k_seam.cu) are told.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

namespace cvb {
namespace seam {

enum { kGateNone = 0, kGateFull = 1, kGateImage = 2 };

struct Params {
  const void *x, *branch;
  const void* gate;              // kGateFull: like branch; kGateImage: (B,C) fp32
  void *y, *z;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;       // (C); null: 1, no norm, 0
  float* stats;                  // 4 x tokens: mean and 1 / spread of branch, of y; null: not kept
  const void *dy, *dz;           // null: 0
  void *dx, *dbranch, *dgate;    // null: not wanted
  float *dscale, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
  float* partial;                // [images or 1][parts][4][C]; null: no sums wanted
  long long B, HW, tokens;       // tokens = B HW
  int C, first, rms, gate_kind, act;
  float eps;
  int tiles;                     // channels_first: groups of pixels of an image
  int tpr;                       // channels_last: threads that share a token
  int parts, max_parts;
};

int run_fwd(Params& P, int io, int sms, cudaStream_t st);
int run_bwd(Params& P, int io, int sms, cudaStream_t st);
int most_parts(int C, long long B, int gate_kind, int sms);
bool takes(int C, bool first, bool backward);

}  // namespace seam
}  // namespace cvb
