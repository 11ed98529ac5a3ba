// The dense operators' calls: one matrix's product and the gated feed-forward block, forward and backward, on device memory
// (the C entry points artlite_linear*, artlite_ffn*), and the passes over activations that the large tiles need.
//
// Up to FEW_ROWS rows go through k_few (linear.hip; backward also k_few_t), straight from the blocks. More rows go through the
// large tiles (hgemm.hip), over fp16 operands made for the call in its workspace, or, some hundreds of bf16 rows, through tiles
// that make the weights' operands from the blocks (k_qgemm):
//   x, dy: each row times the power of two that brings its largest value into [2^14, 2^15): bf16 values convert exactly
//     (those above 2^-29 of their row's largest; smaller ones keep 2^-39 of it), fp32 ones as two planes (hi + lo, 2^-22);
//   weights: each value times the matrix's power of two, rounded once to fp16 (2^-11; fp32 calls: two planes, 2^-22), an
//     eighth of the rounding of a bf16 output;
//   h, dg, du: in fp32 from the sums, then fp16 (fp32 calls: two planes) scaled by a row's power of two from bounds:
//     |g| <= |x| max |gate row| in the 2-norm, |act(g)| <= |g|, |act'| < 2, |dh| <= |dy| max |down| sqrt(H); typical values lie
//     some 2^14 below their bound, fp16 holds 2^29 below it in full.
// Products of two planes are three sums (hi hi + hi lo + lo hi). The weights' gradients sum over rows, so their operands are
// turned, and the rows' powers of two go into one of the two: each of its turned rows, a row of the output, takes the power that
// brings its own largest term's factor into [2^14, 2^15), so that what a row of x and of dy adds counts by what the two come to
// together (k_top reads dg, du and dy once more for that: 37 us of the 2110 that all gradients of 4096 rows of 4096 x 8192 take).
#include "hgemm.h"
#include "matrix.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace artlite {

namespace {

// the exponent of nothing but zeros, below those of all rows
constexpr int NO_TOP = -(1 << 24);

// A launch of k_rows16: x, or x and dy, and the exponents of their rows (and of h, dh, dg and du, from the rows' 2-norms and
// the matrices' bounds)
struct Rows16 {
  const void* x[2];
  int64_t stride[2];
  uint16_t* out[2];
  int32_t *e[2];            // (their values are times 2^-e)
  int arrays;
  int64_t K, Kp, plane;
  int32_t *he, *dhe, *de;   // (those that are wanted)
  int lg, lu, ld;           // gate's, up's and down's bounds
  int32_t* top;             // (wanted) `tops` exponents to set to NO_TOP
  int64_t tops;
};

__device__ __forceinline__ float finite(float v) { return fabsf(v) < __builtin_inff() ? v : 0.0f; }

// a row a workgroup -> fp16 planes of Kp values. The exponents are those of its finite values: a row with an infinite one
// keeps the others' bits, which a gradient of the weights sums apart from it.
template <bool BF16>
__global__ __launch_bounds__(256) void k_rows16(const Rows16 a) {
  __shared__ float red[4];
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  for (int64_t i = m * 256 + threadIdx.x; i < a.tops; i += int64_t(gridDim.x) * 256) a.top[i] = NO_TOP;
  auto all = [&](float v, bool add) {
    for (int o = 32; o; o >>= 1) {
      const float u = __shfl_xor(v, o);
      v = add ? v + u : fmaxf(v, u);
    }
    __syncthreads();
    if (lane == 0) red[wv] = v;
    __syncthreads();
    return add ? red[0] + red[1] + red[2] + red[3] : fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  };
  int norm[2] = {0, 0};
  for (int i = 0; i < a.arrays; i++) {
    auto load = [&](int64_t k, float(&v)[8]) {  // (at any address: rows need not be aligned)
      if constexpr (BF16) {
        uint16_t b[8];
        __builtin_memcpy(b, static_cast<const uint16_t*>(a.x[i]) + m * a.stride[i] + k, 16);
        for (int j = 0; j < 8; j++) v[j] = bf16_to_f32(b[j]);
      } else {
        __builtin_memcpy(v, static_cast<const float*>(a.x[i]) + m * a.stride[i] + k, 32);
      }
    };
    float mx = 0.0f;
    for (int64_t k = threadIdx.x * 8; k < a.K; k += 2048) {
      float v[8];
      load(k, v);
      for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(finite(v[j])));
    }
    mx = all(mx, false);
    const int e = exp_above(mx);
    float ss = 0.0f;
    uint16_t* out = a.out[i] + m * a.Kp;
    for (int64_t k = threadIdx.x * 8; k < a.Kp; k += 2048) {
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (k < a.K) load(k, v);
      uint16_t hi[8], lo[8];
      for (int j = 0; j < 8; j++) {
        const float r = __builtin_amdgcn_ldexpf(v[j], -e), s = __builtin_amdgcn_ldexpf(r, 15);
        ss = __builtin_fmaf(finite(r), finite(r), ss);
        const _Float16 h = _Float16(s);
        hi[j] = __builtin_bit_cast(uint16_t, h);
        // (an infinite value is its first plane)
        lo[j] = __builtin_bit_cast(uint16_t, _Float16(__builtin_isinf(s) ? 0.0f : s - float(h)));
      }
      __builtin_memcpy(__builtin_assume_aligned(out + k, 16), hi, 16);
      if (!BF16) __builtin_memcpy(__builtin_assume_aligned(out + a.plane + k, 16), lo, 16);
    }
    // (|x| < 2^e sqrt(ss); ss is at most K and its fp32 sum off by less than the step to the next exponent)
    ss = all(ss, true);
    norm[i] = e + exp_above(sqrtf(ss) * 1.01f);
    if (threadIdx.x == 0) a.e[i][m] = e - 15;
  }
  if (threadIdx.x == 0) {
    // (h is act(g) times u over 2^he, which is below 2^127 that way: where g is below 2^-112, h has no value but 0 in fp32)
    if (a.he) a.he[m] = max(norm[0] + a.lg, -112) + norm[0] + a.lu - 15;
    if (a.dhe) a.dhe[m] = norm[1] + a.ld - 15;
    if (a.de) a.de[m] = norm[1] + a.ld + norm[0] + max(a.lg, a.lu) + 1 - 15;  // (1 for the derivative)
  }
}

// An fp16 value's place among those worth 2^e: its bits with the exponent put in, in the order of sizes (an infinite one comes
// last: all of its output row is no number), nothing for 0; and the exponent that brings it into [2^14, 2^15) (or less: a
// subnormal one counts as 2^-14)
__device__ __forceinline__ int top_key(uint32_t h, int e) {
  const int b = int(h & 0x7FFFu);
  return b ? b + e * 1024 : NO_TOP;
}
__device__ __forceinline__ int top_exp(int key) { return key == NO_TOP ? NO_TOP : (key >> 10) - 29; }

// Tops of a launch: of each of C columns of T rows of fp16 values (ld apart, row t worth 2^(e[t] + e2[t])), the exponent that
// brings its largest value into [2^14, 2^15) (out: set to NO_TOP before; integer maxima, so any order is the same).
// 128 rows of 512 columns a workgroup, read once.
constexpr int TOP_ROWS = 128, TOP_COLS = 512;
struct Top {
  const uint16_t* in;
  int64_t ld, C;
  const int32_t *e, *e2;
  int32_t* out;
};
struct Tops {
  Top t[3];
  int64_t T;
};
__global__ __launch_bounds__(256) void k_top(const Tops a) {
  __shared__ __attribute__((aligned(16))) int red[4][TOP_COLS];
  const Top& j = a.t[blockIdx.z];
  const int64_t c0 = int64_t(blockIdx.x) * TOP_COLS, t0 = int64_t(blockIdx.y) * TOP_ROWS;
  if (c0 >= j.C) return;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int top[8];
#pragma unroll
  for (int k = 0; k < 8; k++) top[k] = NO_TOP;
  if (c0 + 8 * lane < j.ld) {  // (ld is a multiple of 64)
    constexpr int AT_ONCE = 8;  // (rows of a wave in flight)
    const int64_t end = min(t0 + TOP_ROWS, a.T);
    for (int64_t t = t0 + wv; t < end; t += 4 * AT_ONCE) {
      uint4 v[AT_ONCE];
      int e[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) {  // (past the last row the last again: the largest stays)
        const int64_t r = min(t + 4 * i, end - 1);
        v[i] = *reinterpret_cast<const uint4*>(j.in + r * j.ld + c0 + 8 * lane);
        e[i] = j.e[r] + j.e2[r];
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 8; k++) top[k] = max(top[k], top_key(w[k >> 1] >> (16 * (k & 1)), e[i]));
      }
    }
  }
  for (int k = 0; k < 8; k++) red[wv][8 * lane + k] = top[k];
  __syncthreads();
  for (int c = threadIdx.x; c < TOP_COLS; c += 256) {
    const int v = max(max(red[0][c], red[1][c]), max(red[2][c], red[3][c]));
    if (c0 + c < j.C && v > NO_TOP) atomicMax(j.out + c0 + c, top_exp(v));
  }
}

// Turns of a launch: rows of C fp16 values (ld apart) into C rows of Tp values, zeros past T; as they are, or (top) those of
// row t worth 2^(e[t] + e2[t]) into those of row c worth 2^top[c]. Up to TURN_ROWS rows are a workgroup's (ONE): it finds `top`
// by itself, a launch less (45 rows of 1024 x 2816, fp32, all gradients: 81 us, 86 with k_top)
constexpr int TURN_ROWS = 64;
struct Turn {
  const uint16_t* in;
  int64_t ld, C;
  const int32_t *e, *e2;
  int32_t* top;
  uint16_t* out;
};
struct Turns {
  Turn t[5];
  int64_t T, Tp;
  int planes;
};
template <bool ONE>
__global__ __launch_bounds__(256) void k_turn(const Turns a) {
  __shared__ __attribute__((aligned(16))) uint16_t t[64][72];
  const Turn& j = a.t[blockIdx.z / a.planes];
  const int64_t c0 = int64_t(blockIdx.x) * 64, t0 = int64_t(blockIdx.y) * 64;
  if (c0 >= j.C) return;
  const int64_t pl = blockIdx.z % a.planes;
  const uint16_t* in = j.in + pl * a.T * j.ld;
  uint16_t* out = j.out + pl * j.C * a.Tp;
  const int c = 8 * (threadIdx.x & 7);
  int top[8] = {0, 0, 0, 0, 0, 0, 0, 0}, e[2] = {0, 0};
  uint16_t v[2][8] = {};
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int64_t r = t0 + (threadIdx.x >> 3) + 32 * q;
    if (r < a.T && c0 + c < j.ld) {  // (ld is a multiple of 64: the row's padding is read at most)
      __builtin_memcpy(v[q], __builtin_assume_aligned(in + r * j.ld + c0 + c, 16), 16);
      if (j.top) e[q] = j.e[r] + j.e2[r];
    }
  }
  if (ONE && j.top) {
    __shared__ int most[64];
    if (threadIdx.x < 64) most[threadIdx.x] = NO_TOP;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; q++) {
      uint16_t h[8] = {0, 0, 0, 0, 0, 0, 0, 0};  // (the first plane's: the second's come with its exponents)
      const int64_t r = (threadIdx.x >> 3) + 32 * q;
      if (r < a.T && c0 + c < j.ld) __builtin_memcpy(h, __builtin_assume_aligned(j.in + r * j.ld + c0 + c, 16), 16);
#pragma unroll
      for (int k = 0; k < 8; k++) atomicMax(&most[c + k], top_key(h[k], e[q]));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; k++) top[k] = top_exp(most[c + k]);
    if (pl == 0 && threadIdx.x < 64 && c0 + threadIdx.x < j.C) j.top[c0 + threadIdx.x] = top_exp(most[threadIdx.x]);
  } else if (j.top && c0 + c < j.C) {  // (C is a multiple of 32)
    __builtin_memcpy(top, __builtin_assume_aligned(j.top + c0 + c, 16), 32);
  }
#pragma unroll
  for (int q = 0; q < 2; q++)
#pragma unroll
    for (int k = 0; k < 8; k++)
      t[c + k][(threadIdx.x >> 3) + 32 * q] = __builtin_bit_cast(
          uint16_t, _Float16(__builtin_amdgcn_ldexpf(float(__builtin_bit_cast(_Float16, v[q][k])), e[q] - top[k])));
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 8; i += 256) {
    const int c = i >> 3, r = 8 * (i & 7);
    if (c0 + c < j.C) *reinterpret_cast<uint4*>(out + (c0 + c) * a.Tp + t0 + r) = *reinterpret_cast<const uint4*>(&t[c][r]);
  }
}

__global__ __launch_bounds__(256) void k_zero(uint16_t* p, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) p[i] = 0;
}

int rows16(const Rows16& a, int dtype, int64_t M, hipStream_t s) {
  if (dtype == ARTLITE_X_BF16)
    k_rows16<true><<<unsigned(M), 256, 0, s>>>(a);
  else
    k_rows16<false><<<unsigned(M), 256, 0, s>>>(a);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

// Products' operand pairs as segments: of one plane each, or of two lo hi + hi lo, then hi hi: the small sums first, so that
// only the last ones' additions are rounded at the result's size.
struct Pair {
  const uint16_t* a;
  int64_t ap;  // (values from a plane to the next)
  const uint16_t* b;
  int64_t bp;
  const uint16_t* b2 = nullptr;
};
void segments(HGemm& g, std::initializer_list<Pair> pairs, int planes) {
  const auto add = [&](const Pair& p, int pa, int pb) {
    g.a[g.segs] = p.a + pa * p.ap;
    g.b[g.segs] = p.b + pb * p.bp;
    g.b2[g.segs] = p.b2 ? p.b2 + pb * p.bp : nullptr;
    g.segs++;
  };
  if (planes == 2)
    for (const Pair& p : pairs) add(p, 1, 0), add(p, 0, 1);
  for (const Pair& p : pairs) add(p, 0, 0);
}

// the most rows of a call of the large tiles (their launches' grids and a workspace's sizes stay in range)
constexpr int64_t MOST_ROWS = int64_t(1) << 21;

// ---- one matrix's product

struct LinearPlan {
  bool few, direct = false;
  uint16_t* planes = nullptr;                 // few rows: x as planes, where it is not read as it is
  uint16_t *x16 = nullptr, *w16 = nullptr;    // else
  int32_t* xe = nullptr;
  float* parts = nullptr;
};
LinearPlan linear_layout(Carve& c, const artlite_matrix* w, int dtype, int64_t n, bool direct) {
  LinearPlan p;
  const int few_pl = dtype == ARTLITE_X_BF16 ? 1 : 3;
  const bool apart = few_apart(w, few_pl, false, n);
  const bool large = direct && w->tiles * w->units > FEW_LARGE && qgemm_fits(n, w, false);
  p.few = apart || n <= (dtype != ARTLITE_X_BF16 ? FEW_ROWS_F32 : large ? FEW_ROWS_LARGE : FEW_ROWS);
  if (p.few) {
    const int pl = few_pl;
    if (pl == 3 && !apart) p.planes = c.take<uint16_t>(3 * size_t(n) * w->K);
    p.parts = c.take<float>(few_parts_bytes(w, pl, false, n) / 4);
  } else {
    const int pl = dtype == ARTLITE_X_BF16 ? 1 : 2;
    const int64_t Kp = pad64(w->K);
    p.x16 = c.take<uint16_t>(size_t(pl) * n * Kp);
    p.direct = direct && pl == 1 && qgemm_fits(n, w, false);
    if (p.direct) {
      p.xe = c.take<int32_t>(n);
      p.parts = c.take<float>(qgemm_parts_bytes(n, w, false) / 4);
      return p;
    }
    p.w16 = c.take<uint16_t>(size_t(pl) * w->N * Kp);
    p.xe = c.take<int32_t>(n);
    p.parts = c.take<float>(hgemm_parts_bytes(n, w->N, Kp, pl == 2 ? 3 : 1, false) / 4);
  }
  return p;
}

// (the same bytes whatever the matrix holds: a workspace outlives its values)
LinearPlan linear_plan(Carve& c, const artlite_matrix* w, int dtype, int64_t n) {
  Carve other(nullptr);
  (void)linear_layout(other, w, dtype, n, !w->direct);
  const LinearPlan p = linear_layout(c, w, dtype, n, w->direct);
  c.at = std::max(c.at, other.at);
  return p;
}

int check_matrix(const artlite_matrix* m, const char* what) {
  if (!m) return fail(ARTLITE_EINVAL, "%s: null matrix", what);
  if (!m->have) return fail(ARTLITE_EINVAL, "%s: matrix not uploaded", what);
  return ARTLITE_OK;
}
int check_dtype(int dtype, const char* what) {
  if (dtype != ARTLITE_X_F32 && dtype != ARTLITE_X_BF16) return fail(ARTLITE_EINVAL, "%s: dtype %d", what, dtype);
  return ARTLITE_OK;
}
int check_rows(int64_t n, const char* what) {
  if (n < 0 || n > MOST_ROWS) return fail(ARTLITE_EINVAL, "%s: %lld rows", what, (long long)n);
  return ARTLITE_OK;
}
// rows of `cols` values that a call reads (stride at least 0) or writes (at least cols)
int check_array(const void* p, int64_t n, int64_t cols, int64_t stride, bool written, int dtype, int device,
                const char* what) {
  if (n > 1 && (stride < (written ? cols : 0) || stride > (int64_t(1) << 40)))
    return fail(ARTLITE_EINVAL, "%s: rows of %lld values %lld apart", what, (long long)cols, (long long)stride);
  if (reinterpret_cast<uintptr_t>(p) % (dtype == ARTLITE_X_BF16 ? 2 : 4))
    return fail(ARTLITE_EINVAL, "%s: address not aligned to its values", what);
  return check_device(p, device, what);
}

// x as a launch over few rows takes it: bf16 as it is, fp32 too where the blocks of rows are apart, else as planes
int few_x(FewArgs& a, const void* x, int dtype, int64_t n, int64_t K, int64_t stride, uint16_t* planes, hipStream_t s) {
  a.planes = dtype == ARTLITE_X_BF16 ? 1 : 3;
  a.x32 = dtype == ARTLITE_X_F32 && !planes;
  a.x = x, a.x_stride = stride;
  if (!planes) return ARTLITE_OK;
  a.x = planes, a.x_stride = K, a.x_plane = n * K;
  return launch_planes(static_cast<const float*>(x), n, K, stride, planes, s);
}

int linear(const artlite_matrix* w, const void* x, int dtype, int64_t n, int64_t x_stride, void* y, int64_t y_stride,
           char* base, hipStream_t s) {
  Carve c(base);
  const LinearPlan p = linear_plan(c, w, dtype, n);
  if (p.few) {
    FewArgs a{};
    a.w = w;
    ART_TRY(few_x(a, x, dtype, n, w->K, x_stride, p.planes, s));
    a.M = n;
    a.y = y, a.y_stride = y_stride, a.dtype = dtype;
    a.parts = p.parts;
    return launch_few(a, s);
  }
  const int pl = dtype == ARTLITE_X_BF16 ? 1 : 2, e = p.direct ? qexp16(w) : wexp16(w);
  const int64_t Kp = pad64(w->K);
  Rows16 r{};
  r.x[0] = x, r.stride[0] = x_stride, r.out[0] = p.x16, r.e[0] = p.xe;
  r.arrays = 1, r.K = w->K, r.Kp = Kp, r.plane = n * Kp;
  ART_TRY(rows16(r, dtype, n, s));
  HGemm g{};
  if (p.direct) {
    g.a[0] = p.x16, g.segs = 1;
  } else {
    ART_TRY(launch_unpack(w, nullptr, false, e, 0, p.w16, nullptr, Kp, w->N * Kp, pl, s));
    segments(g, {{p.x16, n * Kp, p.w16, w->N * Kp}}, pl);
  }
  g.lda = g.ldb = g.K = Kp;
  g.M = n, g.N = w->N;
  g.row_e = p.xe, g.e = e;
  g.bias = w->has_bias ? w->bias.as<float>() : nullptr;
  g.y = y, g.y_stride = y_stride, g.dtype = dtype;
  g.parts = p.parts;
  return p.direct ? launch_qgemm(g, w, nullptr, s) : launch_hgemm(g, s);
}

// ---- the gated block

struct Ffn {
  const artlite_matrix *gate, *up, *down;
  int act;
  int64_t H, F, Hp, Fp;
};
int check_ffn(const artlite_ffn* f, Ffn& o, const char* what) {
  if (!f) return fail(ARTLITE_EINVAL, "%s: null", what);
  for (const artlite_matrix* m : {f->gate, f->up, f->down}) {
    ART_TRY(check_matrix(m, what));
    if (m->has_bias) return fail(ARTLITE_EINVAL, "%s: a matrix with a bias", what);
    if (m->device != f->gate->device)
      return fail(ARTLITE_EINVAL, "%s: matrices of devices %d and %d", what, m->device, f->gate->device);
  }
  if (f->act != ARTLITE_ACT_SILU && f->act != ARTLITE_ACT_GELU_TANH)
    return fail(ARTLITE_EINVAL, "%s: activation %d", what, f->act);
  const artlite_matrix *g = f->gate, *u = f->up, *d = f->down;
  if (g->N != u->N || g->K != u->K || g->t != u->t || d->N != g->K || d->K != g->N)
    return fail(ARTLITE_EINVAL, "%s: gate %lld x %lld (%s), up %lld x %lld (%s), down %lld x %lld", what, (long long)g->N,
                (long long)g->K, g->t->name, (long long)u->N, (long long)u->K, u->t->name, (long long)d->N, (long long)d->K);
  o = Ffn{g, u, d, f->act, g->K, g->N, pad64(g->K), pad64(g->N)};
  return ARTLITE_OK;
}

struct FfnPlan {
  bool few, direct, gated;  // (direct: down from its blocks, gated: gate and up from theirs, k_qgemm)
  uint16_t *planes = nullptr, *hp = nullptr;  // few rows: x as planes (where it is not read as it is), h as planes
  uint16_t *x16, *w16, *u16, *d16, *h16;      // else: x, the unpacked matrices, h
  int32_t *xe, *he;
  float* parts;
};
FfnPlan ffn_layout(Carve& c, const Ffn& f, int dtype, int64_t n, bool direct, bool gated) {
  FfnPlan p{};
  const bool b = dtype == ARTLITE_X_BF16, apart = few_apart(f.gate, b ? 1 : 3, true, n);
  const bool made = b && direct && gated && qgemm_fits(n, f.gate, true) && qgemm_fits(n, f.down, false);
  p.few = n <= (made ? FEW_ROWS_FFN_DIRECT : FEW_ROWS_FFN) || (apart && few_apart(f.down, b ? 2 : 3, false, n));
  if (p.few) {
    if (!b && !apart) p.planes = c.take<uint16_t>(3 * size_t(n) * f.H);
    p.hp = c.take<uint16_t>(size_t(b ? 2 : 3) * n * f.F);
    p.parts = c.take<float>(
        std::max(few_parts_bytes(f.gate, b ? 1 : 3, true, n), few_parts_bytes(f.down, b ? 2 : 3, false, n)) / 4);
    return p;
  }
  const size_t pl = b ? 1 : 2;
  p.x16 = c.take<uint16_t>(pl * n * f.Hp);
  p.gated = gated && b && qgemm_fits(n, f.gate, true);
  if (!p.gated) {
    p.w16 = c.take<uint16_t>(pl * f.F * f.Hp);
    p.u16 = c.take<uint16_t>(pl * f.F * f.Hp);
  }
  p.direct = direct && b && qgemm_fits(n, f.down, false);
  if (!p.direct) p.d16 = c.take<uint16_t>(pl * f.H * f.Fp);
  p.h16 = c.take<uint16_t>(pl * n * f.Fp);
  p.xe = c.take<int32_t>(n);
  p.he = c.take<int32_t>(n);
  const int sg = b ? 1 : 3;
  const size_t gate = p.gated ? qgemm_parts_bytes(n, f.gate, true) : hgemm_parts_bytes(n, f.F, f.Hp, sg, true);
  const size_t down = p.direct ? qgemm_parts_bytes(n, f.down, false) : hgemm_parts_bytes(n, f.H, f.Fp, sg, false);
  p.parts = c.take<float>(std::max(gate, down) / 4);
  return p;
}

FfnPlan ffn_plan(Carve& c, const Ffn& f, int dtype, int64_t n) {
  size_t most = 0;
  for (int i = 0; i < 4; i++) {
    Carve any(nullptr);
    (void)ffn_layout(any, f, dtype, n, i & 1, i & 2);
    most = std::max(most, any.at);
  }
  const FfnPlan p = ffn_layout(c, f, dtype, n, f.down->direct, f.gate->direct && f.up->direct);
  c.at = most;
  return p;
}

int ffn_forward(const Ffn& f, const void* x, int dtype, int64_t n, int64_t x_stride, void* y, int64_t y_stride, char* base,
                hipStream_t s) {
  Carve c(base);
  const bool b = dtype == ARTLITE_X_BF16;
  const FfnPlan p = ffn_plan(c, f, dtype, n);
  if (p.few) {
    FewArgs a{};
    a.w = f.gate, a.up = f.up, a.act = f.act;
    ART_TRY(few_x(a, x, dtype, n, f.H, x_stride, p.planes, s));
    a.M = n;
    a.h = p.hp, a.h_stride = f.F, a.h_plane = n * f.F, a.h_planes = b ? 2 : 3;
    a.parts = p.parts;
    ART_TRY(launch_few(a, s));
    FewArgs d{};
    d.w = f.down;
    d.planes = a.h_planes;
    d.x = p.hp, d.x_stride = f.F, d.x_plane = n * f.F;
    d.M = n;
    d.y = y, d.y_stride = y_stride, d.dtype = dtype;
    d.parts = p.parts;
    return launch_few(d, s);
  }
  const int pl = b ? 1 : 2;
  Rows16 r{};
  r.x[0] = x, r.stride[0] = x_stride, r.out[0] = p.x16, r.e[0] = p.xe;
  r.arrays = 1, r.K = f.H, r.Kp = f.Hp, r.plane = n * f.Hp;
  r.he = p.he, r.lg = f.gate->row_exp, r.lu = f.up->row_exp;
  ART_TRY(rows16(r, dtype, n, s));
  const int eg = p.gated ? qexp16(f.gate) : wexp16(f.gate), eu = p.gated ? qexp16(f.up) : wexp16(f.up);
  if (!p.gated) ART_TRY(launch_unpack(f.gate, f.up, false, eg, eu, p.w16, p.u16, f.Hp, f.F * f.Hp, pl, s));
  if (!p.direct) ART_TRY(launch_unpack(f.down, nullptr, false, wexp16(f.down), 0, p.d16, nullptr, f.Fp, f.H * f.Fp, pl, s));
  HGemm g{};
  if (p.gated)
    g.a[0] = p.x16, g.segs = 1;
  else
    segments(g, {{p.x16, n * f.Hp, p.w16, f.F * f.Hp, p.u16}}, pl);
  g.lda = g.ldb = g.K = f.Hp;
  g.M = n, g.N = f.F;
  g.epilogue = H_GLU;
  g.row_e = p.xe, g.e = eg, g.e2 = eu;
  g.act = f.act;
  g.out_e = p.he, g.h = p.h16, g.h_stride = f.Fp, g.h_plane = n * f.Fp, g.planes = pl;
  g.parts = p.parts;
  ART_TRY(p.gated ? launch_qgemm(g, f.gate, f.up, s) : launch_hgemm(g, s));
  HGemm d{};
  if (p.direct)
    d.a[0] = p.h16, d.segs = 1;
  else
    segments(d, {{p.h16, n * f.Fp, p.d16, f.H * f.Fp}}, pl);
  d.lda = d.ldb = d.K = f.Fp;
  d.M = n, d.N = f.H;
  d.row_e = p.he, d.e = p.direct ? qexp16(f.down) : wexp16(f.down);
  d.y = y, d.y_stride = y_stride, d.dtype = dtype;
  d.parts = p.parts;
  return p.direct ? launch_qgemm(d, f.down, nullptr, s) : launch_hgemm(d, s);
}

// Rows up to which the gradients' products run from the blocks (dx alone, 2048 x 8192 Q4_K: 192 rows 122 us against 121 by
// the large tiles, 256 rows 141 against 126, fp32 260 against 262 and 327 against 281; 4096 x 11008 Q4_0: 192 rows 276 against
// 363, 256 rows 297 against 372; one row 52 against 103 and 65 against 241)
constexpr int FEW_ROWS_GRAD = 192;
// Rows (a multiple of 64) up to which the weights' gradients are one launch of small tiles: what they write bounds them, and a
// launch's start (all gradients of 1024 x 2816 IQ4_NL, 45 rows of fp32: 85 us in three launches, 82 in one; 4096 x 11008
// Q4_0, 1 row 187 and 161, fp32 332 and 251, 256 rows 1136 and 1065; 2048 x 8192 Q4_K, 256 rows of bf16, 187 and 189; all
// before k_top, which is as much for both: the last is 195 with it)
constexpr int64_t SHORT_SUMS = 256;
struct GradPlan {
  bool few, gated;  // (gated: g and u from the blocks, k_qgemm)
  uint16_t* planes = nullptr;                    // few rows: x as planes, where it is not read as it is
  uint16_t *x16, *dy16, *a16, *b16, *c16;        // x, dy; gate and up, later their transposes; down's transpose
  uint16_t *h16, *dh16, *dg16, *du16;
  uint16_t *xt, *dyt, *ht, *dgt, *dut;           // (weights' gradients) turned
  int32_t *xe, *ye, *he, *dhe, *de;
  int32_t* top;                                  // (weights' gradients) the exponents of rows of dgate, dup and ddown
  float* parts;
};
GradPlan grad_plan(Carve& c, const Ffn& f, int dtype, int64_t n, bool weights) {
  GradPlan p{};
  const size_t pl = dtype == ARTLITE_X_BF16 ? 1 : 2;
  const size_t w = pl * size_t(f.F * f.Hp > f.H * f.Fp ? f.F * f.Hp : f.H * f.Fp);
  p.few = n <= FEW_ROWS_GRAD;
  const bool fits = !p.few && pl == 1 && qgemm_fits(n, f.gate, true);
  p.gated = fits && f.gate->direct && f.up->direct;
  p.x16 = c.take<uint16_t>(pl * n * f.Hp);
  p.dy16 = c.take<uint16_t>(pl * n * f.Hp);
  if (!p.few) {
    p.a16 = c.take<uint16_t>(w);
    p.b16 = c.take<uint16_t>(w);
    p.c16 = c.take<uint16_t>(pl * f.F * f.Hp);
  } else if (pl == 2 && !few_apart(f.gate, 3, true, n)) {
    p.planes = c.take<uint16_t>(3 * size_t(n) * f.H);
  }
  p.dg16 = c.take<uint16_t>(pl * n * f.Fp);
  p.du16 = c.take<uint16_t>(pl * n * f.Fp);
  p.dh16 = c.take<uint16_t>(pl * n * f.Fp);
  p.xe = c.take<int32_t>(n);
  p.ye = c.take<int32_t>(n);
  p.he = c.take<int32_t>(n);
  p.dhe = c.take<int32_t>(n);
  p.de = c.take<int32_t>(n);
  if (weights) {
    const int64_t Tp = pad64(n);
    p.h16 = c.take<uint16_t>(pl * n * f.Fp);
    p.xt = c.take<uint16_t>(pl * f.H * Tp);
    p.dyt = c.take<uint16_t>(pl * f.H * Tp);
    p.ht = c.take<uint16_t>(pl * f.F * Tp);
    p.dgt = c.take<uint16_t>(pl * f.F * Tp);
    p.dut = c.take<uint16_t>(pl * f.F * Tp);
    p.top = c.take<int32_t>(2 * f.F + f.H);
  }
  const int sg = pl == 2 ? 3 : 1;
  size_t parts = 0;
  if (p.few)
    parts = std::max({few_t_bytes(f.down, 1, int(pl), n), few_t_bytes(f.gate, 2, int(pl), n),
                      size_t(few_raw_parts(f.gate, pl == 2 ? 3 : 1, n)) * n * 2 * f.Fp * 4});
  else
    parts = std::max({hgemm_parts_bytes(n, f.F, f.Hp, sg, false), hgemm_parts_bytes(n, f.F, f.Hp, sg, true),
                           hgemm_parts_bytes(n, f.H, f.Fp, 2 * sg, false)});
  if (weights)
    parts = std::max({parts, hgemm_parts_bytes(f.F, f.H, pad64(n), sg, false), hgemm_parts_bytes(f.H, f.F, pad64(n), sg, false)});
  if (fits) parts = std::max(parts, qgemm_parts_bytes(n, f.gate, true));
  p.parts = c.take<float>(parts / 4);
  return p;
}

int ffn_backward(const Ffn& f, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int dtype, int64_t n,
                 void* dx, int64_t dx_stride, void* dgate, void* dup, void* ddown, char* base, hipStream_t s) {
  const bool weights = dgate || dup || ddown;
  Carve c(base);
  const GradPlan p = grad_plan(c, f, dtype, n, weights);
  const int pl = dtype == ARTLITE_X_BF16 ? 1 : 2;
  Rows16 r{};
  r.x[0] = x, r.stride[0] = x_stride, r.out[0] = p.x16, r.e[0] = p.xe;
  r.x[1] = dy, r.stride[1] = dy_stride, r.out[1] = p.dy16, r.e[1] = p.ye;
  r.arrays = 2, r.K = f.H, r.Kp = f.Hp, r.plane = n * f.Hp;
  r.he = p.he, r.dhe = p.dhe, r.de = p.de;
  r.lg = f.gate->row_exp, r.lu = f.up->row_exp;
  r.ld = f.down->max_exp + int(std::ceil(0.5 * std::log2(double(f.H))));
  if (weights && n > TURN_ROWS) r.top = p.top, r.tops = 2 * f.F + f.H;
  ART_TRY(rows16(r, dtype, n, s));
  // (gate and up share a scale: dx sums over both)
  const int e = wexp16(f.gate) > wexp16(f.up) ? wexp16(f.gate) : wexp16(f.up), ed = wexp16(f.down);
  if (!p.few) {
    if (!p.gated) ART_TRY(launch_unpack(f.gate, f.up, false, e, e, p.a16, p.b16, f.Hp, f.F * f.Hp, pl, s));
    ART_TRY(launch_unpack(f.down, nullptr, true, ed, 0, p.c16, nullptr, f.Hp, f.F * f.Hp, pl, s));
  }
  HGemm d{};
  if (!p.few) segments(d, {{p.dy16, n * f.Hp, p.c16, f.F * f.Hp}}, pl);
  d.lda = d.ldb = d.K = f.Hp;
  d.M = n, d.N = f.F;
  d.epilogue = H_ROWS;
  d.row_e = p.ye, d.e = ed;
  d.out_e = p.dhe, d.h = p.dh16, d.h_stride = f.Fp, d.h_plane = n * f.Fp, d.planes = pl;
  d.parts = p.parts;
  if (p.few) {
    ART_TRY(launch_few_t(FewTArgs{{f.down}, {p.dy16}, 1, f.Hp, n * f.Hp, pl, ed, n, p.parts}, s));
    ART_TRY(launch_join(d, few_t_parts(f.down, 1, pl, n), s));
  } else {
    ART_TRY(launch_hgemm(d, s));
  }
  HGemm g{};
  if (!p.few && !p.gated) segments(g, {{p.x16, n * f.Hp, p.a16, f.F * f.Hp, p.b16}}, pl);
  g.lda = g.ldb = g.K = f.Hp;
  g.M = n, g.N = f.F;
  g.epilogue = H_DGLU;
  g.row_e = p.xe, g.e = g.e2 = e;
  g.act = f.act;
  g.dh = p.dh16, g.dh_e = p.dhe;
  g.out_e = p.de, g.h_e = p.he;
  g.dg = p.dg16, g.du = p.du16, g.h = p.h16;
  g.h_stride = f.Fp, g.h_plane = n * f.Fp, g.planes = pl;
  g.parts = p.parts;
  if (p.few) {
    FewArgs a{};
    a.w = f.gate, a.up = f.up;
    ART_TRY(few_x(a, x, dtype, n, f.H, x_stride, p.planes, s));
    a.M = n;
    a.parts = p.parts;
    a.raw = few_raw_parts(f.gate, a.planes, n);
    ART_TRY(launch_few(a, s));
    g.row_e = nullptr, g.e = g.e2 = 0;  // (sums of the values themselves)
    ART_TRY(launch_join(g, a.raw, s));
  } else if (p.gated) {
    g.a[0] = p.x16, g.segs = 1;
    g.e = qexp16(f.gate), g.e2 = qexp16(f.up);
    ART_TRY(launch_qgemm(g, f.gate, f.up, s));
  } else {
    ART_TRY(launch_hgemm(g, s));
  }
  if (dx) {
    if (!p.few) ART_TRY(launch_unpack(f.gate, f.up, true, e, e, p.a16, p.b16, f.Fp, f.H * f.Fp, pl, s));
    HGemm x2{};
    if (!p.few) segments(x2, {{p.dg16, n * f.Fp, p.a16, f.H * f.Fp}, {p.du16, n * f.Fp, p.b16, f.H * f.Fp}}, pl);
    x2.lda = x2.ldb = x2.K = f.Fp;
    x2.M = n, x2.N = f.H;
    x2.row_e = p.de, x2.e = e;
    x2.y = dx, x2.y_stride = dx_stride, x2.dtype = dtype;
    x2.parts = p.parts;
    if (p.few) {
      ART_TRY(launch_few_t(FewTArgs{{f.gate, f.up}, {p.dg16, p.du16}, 2, f.Fp, n * f.Fp, pl, e, n, p.parts}, s));
      ART_TRY(launch_join(x2, few_t_parts(f.gate, 2, pl, n), s));
    } else {
      ART_TRY(launch_hgemm(x2, s));
    }
  }
  if (!weights) return ARTLITE_OK;
  // Sums over rows t of a[t][m] b[t][k]: a (dg, du, dy) takes both rows' powers of two, and an output row one of its own, from
  // what its terms come to; b (x, h) stays as it is.
  const int64_t Tp = pad64(n);
  int32_t *const ge = p.top, *const ue = ge + f.F, *const ddowne = ue + f.F;
  Tops o{};
  o.T = n;
  Turns t{};
  t.T = n, t.Tp = Tp, t.planes = pl;
  HGemm w[3] = {};
  int turns = 0, count = 0;
  const auto grad = [&](const uint16_t* a, uint16_t* at, int64_t M, int64_t Mp, const int32_t* ea, const uint16_t* bt, int64_t N,
                        const int32_t* eb, int32_t* top, void* out) {
    if (!out) return;
    o.t[count] = Top{a, Mp, M, ea, eb, top};
    t.t[turns++] = Turn{a, Mp, M, ea, eb, top, at};
    HGemm& g = w[count++];
    segments(g, {{at, M * Tp, bt, N * Tp}}, pl);
    g.lda = g.ldb = g.K = Tp;
    g.M = M, g.N = N;
    g.row_e = top;
    g.y = out, g.y_stride = N, g.dtype = dtype;
    g.parts = p.parts;
  };
  grad(p.dg16, p.dgt, f.F, f.Fp, p.de, p.xt, f.H, p.xe, ge, dgate);
  grad(p.du16, p.dut, f.F, f.Fp, p.de, p.xt, f.H, p.xe, ue, dup);
  grad(p.dy16, p.dyt, f.H, f.Hp, p.ye, p.ht, f.F, p.he, ddowne, ddown);
  if (dgate || dup) t.t[turns++] = Turn{p.x16, f.Hp, f.H, nullptr, nullptr, nullptr, p.xt};
  if (ddown) t.t[turns++] = Turn{p.h16, f.Fp, f.F, nullptr, nullptr, nullptr, p.ht};
  const int64_t widest = std::max(f.H, f.F);
  if (n > TURN_ROWS) {
    const dim3 grid(unsigned((widest + TOP_COLS - 1) / TOP_COLS), unsigned((n + TOP_ROWS - 1) / TOP_ROWS), unsigned(count));
    k_top<<<grid, 256, 0, s>>>(o);
    ART_HIP(hipGetLastError());
  }
  (n > TURN_ROWS ? k_turn<false> : k_turn<true>)<<<dim3(unsigned((widest + 63) / 64), unsigned(Tp / 64), unsigned(turns * pl)),
                                                   256, 0, s>>>(t);
  ART_HIP(hipGetLastError());
  if (Tp <= SHORT_SUMS) return launch_hgemms(w, count, s);
  for (int i = 0; i < count; i++) ART_TRY(launch_hgemm(w[i], s));
  return ARTLITE_OK;
}

}  // namespace

}  // namespace artlite

using namespace artlite;

extern "C" int artlite_linear_workspace(const artlite_matrix* w, int dtype, int64_t n, size_t* nbytes) {
  if (!w || !nbytes) return fail(ARTLITE_EINVAL, "linear: null");
  ART_TRY(check_dtype(dtype, "linear"));
  ART_TRY(check_rows(n, "linear"));
  Carve c(nullptr);
  if (n) (void)linear_plan(c, w, dtype, n);
  *nbytes = c.at;
  return ARTLITE_OK;
}

extern "C" int artlite_linear(const artlite_matrix* w, const void* x, int dtype, int64_t n, int64_t x_stride, void* y,
                              int64_t y_stride, artlite_workspace* work, void* stream) {
  ART_TRY(check_matrix(w, "linear"));
  ART_TRY(check_dtype(dtype, "linear"));
  ART_TRY(check_rows(n, "linear"));
  if (n == 0) return ARTLITE_OK;
  ART_TRY(check_array(x, n, w->K, x_stride, false, dtype, w->device, "linear: x"));
  ART_TRY(check_array(y, n, w->N, y_stride, true, dtype, w->device, "linear: y"));
  Carve c(nullptr);
  (void)linear_plan(c, w, dtype, n);
  if (c.at && work && work->w.device != w->device)
    return fail(ARTLITE_EINVAL, "linear: a workspace of device %d, not %d", work->w.device, w->device);
  OnDevice on;
  ART_TRY(on.set(w->device));
  WorkScope ws;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  ART_TRY(ws.begin(work ? &work->w : nullptr, c.at, s, "linear"));
  return linear(w, x, dtype, n, x_stride, y, y_stride, work ? work->w.p : nullptr, s);
}

extern "C" int artlite_ffn_workspace(const artlite_ffn* d, int dtype, int64_t n, int backward, size_t* nbytes) {
  Ffn f;
  ART_TRY(check_ffn(d, f, "ffn"));
  if (!nbytes) return fail(ARTLITE_EINVAL, "ffn: null");
  ART_TRY(check_dtype(dtype, "ffn"));
  ART_TRY(check_rows(n, "ffn"));
  Carve c(nullptr);
  if (n && backward) {
    (void)grad_plan(c, f, dtype, n, backward == 2);
  } else if (n) {
    (void)ffn_plan(c, f, dtype, n);
  }
  *nbytes = c.at;
  return ARTLITE_OK;
}

extern "C" int artlite_ffn_forward(const artlite_ffn* d, const void* x, int dtype, int64_t n, int64_t x_stride, void* y,
                                   int64_t y_stride, artlite_workspace* work, void* stream) {
  Ffn f;
  ART_TRY(check_ffn(d, f, "ffn"));
  ART_TRY(check_dtype(dtype, "ffn"));
  ART_TRY(check_rows(n, "ffn"));
  if (n == 0) return ARTLITE_OK;
  const int dev = f.gate->device;
  ART_TRY(check_array(x, n, f.H, x_stride, false, dtype, dev, "ffn: x"));
  ART_TRY(check_array(y, n, f.H, y_stride, true, dtype, dev, "ffn: y"));
  Carve c(nullptr);
  (void)ffn_plan(c, f, dtype, n);
  if (work && work->w.device != dev) return fail(ARTLITE_EINVAL, "ffn: a workspace of device %d, not %d", work->w.device, dev);
  OnDevice on;
  ART_TRY(on.set(dev));
  WorkScope ws;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  ART_TRY(ws.begin(work ? &work->w : nullptr, c.at, s, "ffn"));
  return ffn_forward(f, x, dtype, n, x_stride, y, y_stride, work->w.p, s);
}

extern "C" int artlite_ffn_backward(const artlite_ffn* d, const void* x, int64_t x_stride, const void* dy,
                                    int64_t dy_stride, int dtype, int64_t n, void* dx, int64_t dx_stride, void* dgate,
                                    void* dup, void* ddown, artlite_workspace* work, void* stream) {
  Ffn f;
  ART_TRY(check_ffn(d, f, "ffn backward"));
  ART_TRY(check_dtype(dtype, "ffn backward"));
  ART_TRY(check_rows(n, "ffn backward"));
  const int dev = f.gate->device;
  const bool weights = dgate || dup || ddown;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (void* p : {dgate, dup, ddown})
    if (p) ART_TRY(check_array(p, 1, 0, 0, true, dtype, dev, "ffn backward: a weight's gradient"));
  OnDevice on;
  if (n == 0) {  // (sums of nothing)
    ART_TRY(on.set(dev));
    for (void* p : {dgate, dup, ddown})
      if (p) k_zero<<<1024, 256, 0, s>>>(static_cast<uint16_t*>(p), f.F * f.H * (dtype == ARTLITE_X_BF16 ? 1 : 2));
    ART_HIP(hipGetLastError());
    return ARTLITE_OK;
  }
  ART_TRY(check_array(x, n, f.H, x_stride, false, dtype, dev, "ffn backward: x"));
  ART_TRY(check_array(dy, n, f.H, dy_stride, false, dtype, dev, "ffn backward: dy"));
  if (dx) ART_TRY(check_array(dx, n, f.H, dx_stride, true, dtype, dev, "ffn backward: dx"));
  if (!dx && !weights) return ARTLITE_OK;
  Carve c(nullptr);
  (void)grad_plan(c, f, dtype, n, weights);
  if (work && work->w.device != dev)
    return fail(ARTLITE_EINVAL, "ffn backward: a workspace of device %d, not %d", work->w.device, dev);
  ART_TRY(on.set(dev));
  WorkScope ws;
  ART_TRY(ws.begin(work ? &work->w : nullptr, c.at, s, "ffn backward"));
  return ffn_backward(f, x, x_stride, dy, dy_stride, dtype, n, dx, dx_stride, dgate, dup, ddown, work->w.p, s);
}
