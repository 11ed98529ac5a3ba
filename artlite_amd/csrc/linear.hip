// Dense products over few rows: y = x W^T (+ bias) and the gated h = act(x W^T) (x U^T) for W, U in 4-bit blocks (matrix.h's
// tile layout), 1 to 64 rows of x a pass over the weights, on the bf16 MFMA (16x16x32) over the blocks' codes.
//
// Mathematics. Values come in groups of 32 with one scale s and offset o: w = s c - o. A group's share of an output is
// s sum(c x) - o sum(x): one MFMA takes sum(c x) of 16 rows of x and 16 weight rows over the group's 32 values, exact
// products of bf16 codes and bf16 x summed in fp32, and the scale is applied to the sum, so no weight is ever rounded. fp32 x
// goes as three planes of bf16 (x = hi + mid + lo to 2^-24), the gated launch's h as two (bf16 calls: 2^-17, far below the
// output's own rounding of 2^-8) or three.
//   One or two planes: the codes as 128 + c (the bits 0x4300 | c: 7 instructions for 8 codes) and 128 (or 136, Q4_0's zero
//   point) times sum(x) taken off through the C input, one MFMA against a constant that serves all of a wave's weight rows.
//   The sums of 128 x cost about 5 bits of the 24: nothing to bf16 outputs, too much for fp32 ones.
//   Three planes, and IQ4's values: the codes' own bf16 values from a table of 16 in registers (byte permutes, 24
//   instructions for 8 codes).
//
// Shape. A workgroup takes a tile of 16 weight rows (gated: the same rows of both matrices, so that h forms in a thread) and
// its waves share K, unit by unit in turn; their sums meet in LDS and are added in wave order. A wave's loads of a unit are
// contiguous (2 KiB of codes, the 16 headers) and go to registers, the next unit's in flight while one computes; x comes from
// L2, only the rows that there are. What bounds it: the weights' bytes from HBM, for a small matrix the latency of a launch
// and two dependent round trips.
#include "matrix.h"

namespace artlite {

namespace {

constexpr uint32_t bf16_of(int v) { return __builtin_bit_cast(uint32_t, float(v)) >> 16; }

// 16 values as byte tables of their bf16 halves
struct Lut16 {
  uint32_t lo[4], hi[4];
};
constexpr Lut16 make_lut(int kind) {  // 0: IQ4's values, 1: c - 8, 2: c
  constexpr int V[16] = {-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113};
  Lut16 t{};
  for (int i = 0; i < 16; i++) {
    const uint32_t b = bf16_of(kind == 0 ? V[i] : kind == 1 ? i - 8 : i);
    t.lo[i / 4] |= (b & 0xFF) << (8 * (i % 4));
    t.hi[i / 4] |= (b >> 8) << (8 * (i % 4));
  }
  return t;
}
template <int KIND>
__device__ __forceinline__ void lut_bytes(uint32_t c, uint32_t& lo, uint32_t& hi) {
  constexpr Lut16 T = make_lut(KIND);
  const uint32_t s = c & 0x07070707u;
  // bytes of ones where the code's bit 3 is set (selectors 8 .. 11: the sign of bytes 1, 3 of the second and first source)
  const uint32_t m = __builtin_amdgcn_perm(c << 4, c << 12, 0x0B090A08u);
  lo = (__builtin_amdgcn_perm(T.lo[3], T.lo[2], s) & m) | (__builtin_amdgcn_perm(T.lo[1], T.lo[0], s) & ~m);
  hi = (__builtin_amdgcn_perm(T.hi[3], T.hi[2], s) & m) | (__builtin_amdgcn_perm(T.hi[1], T.hi[0], s) & ~m);
}

// the operand of a code dword: 128 + c, or by table the codes' own values
template <int KIND>
__device__ __forceinline__ u32x4 operand(uint32_t w) {
  if constexpr (KIND < 0) {
    return u32x4{(w & 0x000F000Fu) | 0x43004300u, ((w >> 4) & 0x000F000Fu) | 0x43004300u,
                 ((w >> 8) & 0x000F000Fu) | 0x43004300u, ((w >> 12) & 0x000F000Fu) | 0x43004300u};
  } else {
    uint32_t l0, h0, l1, h1;  // (nibbles 0, 2, 4, 6 and 1, 3, 5, 7)
    lut_bytes<KIND>(w & 0x0F0F0F0Fu, l0, h0);
    lut_bytes<KIND>((w >> 4) & 0x0F0F0F0Fu, l1, h1);
    return u32x4{__builtin_amdgcn_perm(h0, l0, 0x06020400u), __builtin_amdgcn_perm(h1, l1, 0x06020400u),
                 __builtin_amdgcn_perm(h0, l0, 0x07030501u), __builtin_amdgcn_perm(h1, l1, 0x07030501u)};
  }
}

template <int QT, int P>
constexpr int code_kind() {
  return iq4<QT> ? 0 : P < 3 ? -1 : QT == ARTLITE_Q4_0 ? 1 : 2;
}

struct FewK {
  const uint8_t *w, *up;
  int units;
  int64_t N, K, M;
  const uint16_t* x;
  int64_t x_stride, x_plane;
  const float* bias;
  void* y;
  int64_t y_stride;
  int dtype, act;
  uint16_t* h;
  int64_t h_stride, h_plane;
  int h_planes;
};

__device__ __forceinline__ void store_planes(uint16_t* p, int64_t plane, int planes, float v) {
  for (int i = 0; i < planes; i++) {
    const uint32_t b = f32_to_bf16(v);
    p[i * plane] = uint16_t(b);
    // (an infinite value is its first plane; the difference would be none)
    v = __builtin_isinf(v) ? 0.0f : v - bf16_to_f32(b);
  }
}

template <int QT, int P, int NC, bool GLU>
__global__ __launch_bounds__(P* NC == 1 ? 1024 : 512) void k_few(const FewK a) {
  constexpr int RB = GLU ? 2 : 1, KIND = code_kind<QT, P>(), UB = unit_bytes<QT>();
  constexpr bool CIN = KIND < 0 || has_offset<QT>;  // (sum(x) times a constant is wanted)
  constexpr float CC = KIND < 0 ? (QT == ARTLITE_Q4_0 ? -136.0f : -128.0f) : -1.0f;
  constexpr uint32_t CB = bf16_of(int(CC)) * 0x10001u;
  constexpr int XG = P * NC <= 2 ? 4 : P * NC <= 4 ? 2 : 1;  // (groups whose x is loaded together: registers)
  extern __shared__ f32x4 red[];  // [wave][block][lane]
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6,
            lg = lane >> 4, lr = lane & 15;
  const int64_t tile = blockIdx.x, m0 = int64_t(blockIdx.y) * (16 * NC);
  const int64_t tb = tile * a.units * UB;
  const uint8_t* wp[2] = {a.w + tb, GLU ? a.up + tb : nullptr};
  const uint16_t* xp[NC];
  bool live[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const int64_t m = m0 + 16 * c + lr;
    live[c] = m < a.M;
    xp[c] = a.x + (live[c] ? m : 0) * a.x_stride + 8 * lg;
  }
  f32x4 acc[RB][NC];
#pragma unroll
  for (int b = 0; b < RB; b++)
#pragma unroll
    for (int c = 0; c < NC; c++) acc[b][c] = f32x4{0, 0, 0, 0};

  uint4 code[RB][2];
  TileHdr<QT> hd[RB];
  auto load = [&](int u) {
#pragma unroll
    for (int b = 0; b < RB; b++) {
      const uint8_t* p = wp[b] + int64_t(u) * UB;
#pragma unroll
      for (int h = 0; h < 2; h++) code[b][h] = *reinterpret_cast<const uint4*>(p + 1024 * h + 16 * lane);
      hd[b].load(p + 2048 + hdr_bytes<QT>() * lr);
    }
  };
  if (wv < a.units) load(wv);
  for (int u = wv; u < a.units; u += W) {
    uint4 cur[RB][2];
    TileHdr<QT> hc[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) {
      cur[b][0] = code[b][0], cur[b][1] = code[b][1];
      hc[b] = hd[b];
    }
    if (u + W < a.units) load(u + W);
    const int64_t k0 = int64_t(u) * UNIT;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      u32x4 x[XG][NC][P];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int g = 4 * h + j;
        if (j % XG == 0)
#pragma unroll
          for (int i = 0; i < XG; i++)
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
              for (int p = 0; p < P; p++) {
                const int64_t k = k0 + 32 * (g + i);
                x[i][c][p] = u32x4{0, 0, 0, 0};
                if (live[c] && k < a.K) x[i][c][p] = *reinterpret_cast<const u32x4*>(xp[c] + p * a.x_plane + k);
              }
        const u32x4 cst{CB, CB, CB, CB};
        f32x4 cin[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) {
          cin[c] = f32x4{0, 0, 0, 0};
          if constexpr (CIN)
#pragma unroll
            for (int p = P - 1; p >= 0; p--) cin[c] = mfma(x[j % XG][c][p], cst, cin[c]);
        }
#pragma unroll
        for (int b = 0; b < RB; b++) {
          const uint32_t w = j == 0 ? cur[b][h].x : j == 1 ? cur[b][h].y : j == 2 ? cur[b][h].z : cur[b][h].w;
          const u32x4 q = operand<KIND>(w);
          const float s = hc[b].scale(g);
          float o = 0.0f;
          if constexpr (has_offset<QT>) o = hc[b].offset(g) * (KIND < 0 ? 1.0f / 128.0f : 1.0f);
#pragma unroll
          for (int c = 0; c < NC; c++) {
            f32x4 d = KIND < 0 ? cin[c] : f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = P - 1; p >= 0; p--) d = mfma(x[j % XG][c][p], q, d);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              acc[b][c][i] = __builtin_fmaf(s, d[i], acc[b][c][i]);
              if constexpr (has_offset<QT>) acc[b][c][i] = __builtin_fmaf(o, cin[c][i], acc[b][c][i]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int b = 0; b < RB; b++)
#pragma unroll
    for (int c = 0; c < NC; c++) red[(wv * (RB * NC) + b * NC + c) * WAVE + lane] = acc[b][c];
  __syncthreads();
  // the waves' sums, in wave order; thread t takes block t / 64 (of a gated launch both matrices')
  for (int c = wv; c < NC; c += W) {
    f32x4 s[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) {
      s[b] = red[(b * NC + c) * WAVE + lane];
      for (int w = 1; w < W; w++) s[b] += red[(w * (RB * NC) + b * NC + c) * WAVE + lane];
    }
    const int64_t n = tile * TROWS + lr;
    if (n >= a.N) continue;
    const float bias = !GLU && a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t m = m0 + 16 * c + 4 * lg + i;
      if (m >= a.M) continue;
      const float v = s[0][i] + bias;
      if constexpr (GLU) {
        store_planes(a.h + m * a.h_stride + n, a.h_plane, a.h_planes, gate_act(a.act, v) * s[1][i]);
      } else if (a.dtype == ARTLITE_X_BF16) {
        static_cast<uint16_t*>(a.y)[m * a.y_stride + n] = uint16_t(f32_to_bf16(v));
      } else {
        static_cast<float*>(a.y)[m * a.y_stride + n] = v;
      }
    }
  }
}

__global__ __launch_bounds__(256) void k_planes(const void* __restrict__ x, int bf16, int64_t K, int64_t stride,
                                                uint16_t* __restrict__ out, int64_t Kp, int64_t plane, int planes) {
  const int64_t m = blockIdx.y, k = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (k >= Kp) return;
  float v = 0.0f;
  if (k < K)
    v = bf16 ? bf16_to_f32(static_cast<const uint16_t*>(x)[m * stride + k]) : static_cast<const float*>(x)[m * stride + k];
  store_planes(out + m * Kp + k, plane, planes, v);
}

// Waves of a workgroup: 16 to share K where the tiles alone leave the device's waves few (2048 x 2048, one row: the whole
// matrix in one round of loads), 4 where there are enough of them, never more than units.
int few_waves(int64_t groups, int units, bool wide) {
  int w = 4;
  while (w < (wide ? 16 : 8) && groups * w < 8192) w *= 2;
  return int(units < w ? units : w);
}

template <int QT, int P, int NC, bool GLU>
int launch_few_t(const FewK& k, int64_t tiles, hipStream_t s) {
  const int64_t mb = (k.M + 16 * NC - 1) / (16 * NC);
  const int W = few_waves(tiles * mb, k.units, P * NC == 1);
  const size_t lds = size_t(W) * (GLU ? 2 : 1) * NC * WAVE * 16;
  k_few<QT, P, NC, GLU><<<dim3(unsigned(tiles), unsigned(mb)), 64 * W, lds, s>>>(k);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

template <int QT, int P, bool GLU>
int launch_few_p(const FewK& k, int64_t tiles, hipStream_t s) {
  if (k.M <= 16) return launch_few_t<QT, P, 1, GLU>(k, tiles, s);
  if (k.M <= 32) return launch_few_t<QT, P, 2, GLU>(k, tiles, s);
  return launch_few_t<QT, P, 4, GLU>(k, tiles, s);
}

template <int QT>
int launch_few_q(const FewArgs& a, const FewK& k, hipStream_t s) {
  const int64_t t = a.w->tiles;
  if (a.up) return a.planes == 1 ? launch_few_p<QT, 1, true>(k, t, s) : launch_few_p<QT, 3, true>(k, t, s);
  return a.planes == 1   ? launch_few_p<QT, 1, false>(k, t, s)
         : a.planes == 2 ? launch_few_p<QT, 2, false>(k, t, s)
                         : launch_few_p<QT, 3, false>(k, t, s);
}

}  // namespace

int launch_few(const FewArgs& a, hipStream_t s) {
  if (a.M <= 0) return ARTLITE_OK;
  if (a.M > int64_t(65535) * 16) return fail(ARTLITE_EINVAL, "dense rows: %lld rows", (long long)a.M);
  FewK k{};
  k.w = a.w->w.as<uint8_t>();
  k.up = a.up ? a.up->w.as<uint8_t>() : nullptr;
  k.units = a.w->units;
  k.N = a.w->N, k.K = a.w->K, k.M = a.M;
  k.x = a.x, k.x_stride = a.x_stride, k.x_plane = a.x_plane;
  k.bias = a.w->has_bias ? a.w->bias.as<float>() : nullptr;
  k.y = a.y, k.y_stride = a.y_stride, k.dtype = a.dtype, k.act = a.act;
  k.h = a.h, k.h_stride = a.h_stride, k.h_plane = a.h_plane, k.h_planes = a.h_planes;
#define ART_F(QT) return launch_few_q<QT>(a, k, s)
  ART_TILE_QTYPES(a.w->t->id, ART_F)
#undef ART_F
}

int launch_planes(const void* x, int dtype, int64_t M, int64_t K, int64_t stride, uint16_t* out, int64_t Kp, int64_t plane,
                  int planes, hipStream_t s) {
  if (M <= 0) return ARTLITE_OK;
  for (int64_t m = 0; m < M; m += 65535) {
    const int64_t rows = M - m < 65535 ? M - m : 65535;
    const int es = dtype == ARTLITE_X_BF16 ? 2 : 4;
    k_planes<<<dim3(unsigned((Kp + 255) / 256), unsigned(rows)), 256, 0, s>>>(
        static_cast<const char*>(x) + m * stride * es, dtype == ARTLITE_X_BF16, K, stride, out + m * Kp, Kp, plane, planes);
    ART_HIP(hipGetLastError());
  }
  return ARTLITE_OK;
}

}  // namespace artlite
