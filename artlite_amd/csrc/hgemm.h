// The large tiles: dense fp16 products with fp32 sums (hgemm.hip).
#pragma once

#include "common.h"

struct artlite_matrix;

namespace artlite {

// what becomes of the sums: H_STORE y (bf16 or fp32); H_ROWS fp16 rows; H_GLU h of a gated pair; H_DGLU its gradients
enum HEpilogue { H_STORE = 0, H_ROWS = 1, H_GLU = 2, H_DGLU = 3 };

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
  // scales: the sums of row m are worth 2^(e + row_e[m]) (row_e may be null); gated: e2 the second's
  const int32_t* row_e;
  int e, e2;
  // H_STORE: y[m][n] = the sum + bias[n], bf16 or fp32
  const float* bias;
  void* y;
  int64_t y_stride;
  int dtype;
  // the others: fp16 planes of rows of h_stride values (a multiple of 64), times 2^-out_e[m]; columns N .. h_stride zeros.
  // H_ROWS: h; H_GLU: h = act(g) u; H_DGLU: from dh (planes as these, worth 2^dh_e[m]) dg and du, and (h set) h times 2^-h_e[m]
  int act;
  const int32_t *out_e, *h_e, *dh_e;
  const uint16_t* dh;
  uint16_t *h, *dg, *du;
  int64_t h_stride, h_plane;
  int64_t h_cols;  // (set by the launch: the columns of the planes from the first on)
  int planes;
  // scratch for sums in parts: hgemm_parts_bytes of it
  float* parts;
};
// the scratch that a product may take (gated: N columns of each matrix)
size_t hgemm_parts_bytes(int64_t M, int64_t N, int64_t K, int segs, bool gated);
int launch_hgemm(const HGemm& g, hipStream_t s);
// up to three H_STORE products of as many 128 x 128 tiles each, in one launch without parts: short sums of many outputs
int launch_hgemms(const HGemm* g, int count, hipStream_t s);
// out = x W^T with W (gated, H_GLU and H_DGLU: and W2, alike) in its blocks, values times 2^-g.e (2^-g.e2): a as one segment of
// one plane, no b
bool qgemm_fits(int64_t M, const artlite_matrix* w, bool gated);  // (by its shape; the matrices have to be `direct` besides)
size_t qgemm_parts_bytes(int64_t M, const artlite_matrix* w, bool gated);
int launch_qgemm(HGemm g, const artlite_matrix* w, const artlite_matrix* w2, hipStream_t s);
// what becomes of sums that are there already, in parts of M rows of pad64(N) values (gated: both matrices' side by side)
int launch_join(const HGemm& g, int parts, hipStream_t s);

}  // namespace artlite
