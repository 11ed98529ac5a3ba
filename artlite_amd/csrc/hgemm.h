// The large tiles: dense fp16 products with fp32 sums (hgemm.hip).
#pragma once

#include "common.h"

namespace artlite {

enum HEpilogue { H_STORE = 0, H_GLU = 1, H_DGLU = 2 };

// out[m][n] = sum over the segments and K of a[m][k] b[n][k]; a, b fp16 rows of lda, ldb values (K a multiple of 64; both
// multiples of 8). A segment names its operands: planes of split values, or parts of a longer sum.
constexpr int H_SEGS = 6;
struct HGemm {
  const uint16_t* a[H_SEGS];
  const uint16_t* b[H_SEGS];
  const uint16_t* b2[H_SEGS];  // (gated: the second matrix)
  int segs;
  int64_t lda, ldb;
  int64_t M, N, K;
  int epilogue;
  // scales: the sums of row m are worth 2^(e + row_e[m] + *e0 + *e1) (row_e, e0, e1 may be null); gated: e2 the second's
  const int32_t* row_e;
  const int32_t *e0, *e1;
  int e, e2;
  // H_STORE: y[m][n] = the sum + bias[n], bf16 or fp32; or (y16) fp16 scaled by 2^-out_e[m] in `planes` planes
  const float* bias;
  void* y;
  int64_t y_stride;
  int dtype;
  // H_GLU: h = act(g) u as fp16 planes of rows of h_stride values, times 2^-out_e[m]; columns N .. h_stride zeros
  // H_DGLU: from dh (fp32, rows of h_stride values): dg and du likewise (2^-out_e[m]), and (h set) h times 2^-h_e[m]
  int act;
  const int32_t *out_e, *h_e;
  const float* dh;
  uint16_t *h, *dg, *du;
  int64_t h_stride, h_plane;
  int planes;
};
int launch_hgemm(const HGemm& g, hipStream_t s);

}  // namespace artlite
