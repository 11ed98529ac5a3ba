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

#include <algorithm>
#include <utility>

namespace artlite {

namespace {

// the constants of a code dword's operand in registers: an and-or takes them so, literals make it two instructions
struct Nibbles {
  uint32_t mask = 0x000F000Fu, top = 0x43004300u;
  __device__ __forceinline__ Nibbles() { asm("" : "+s"(mask), "+v"(top)); }
};
// the operand of a code dword: 128 + c, or by table the codes' own values
template <int KIND>
__device__ __forceinline__ u32x4 operand(uint32_t w, const Nibbles& n) {
  if constexpr (KIND < 0) {
    return u32x4{(w & n.mask) | n.top, ((w >> 4) & n.mask) | n.top, ((w >> 8) & n.mask) | n.top, ((w >> 12) & n.mask) | n.top};
  } else {
    return lut_operand<KIND>(w);
  }
}

template <int QT, int P>
constexpr int code_kind() {
  return iq4<QT> ? 0 : P < 3 ? -1 : QT == ARTLITE_Q4_0 ? 1 : 2;
}

struct FewK {
  const uint8_t *w, *up;
  int64_t tiles;
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
  float* parts;
  int64_t part_row, part_up;  // (values of a row of the parts; where the second matrix's begin)
};

__device__ __forceinline__ void store_planes(uint16_t* p, int64_t plane, int planes, float v) {
  for (int i = 0; i < planes; i++) {
    const uint32_t b = f32_to_bf16(v);
    p[i * plane] = uint16_t(b);
    // (an infinite value is its first plane; the difference would be none)
    v = __builtin_isinf(v) ? 0.0f : v - bf16_to_f32(b);
  }
}

// eight fp32 values (a, b) -> their planes: two values' bf16 in a dword each, x = hi + mid + lo to 2^-24
__device__ __forceinline__ void split3(const u32x4& a, const u32x4& b, u32x4& hi, u32x4& mid, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float u = __uint_as_float(i < 2 ? a[2 * i] : b[2 * i - 4]), v = __uint_as_float(i < 2 ? a[2 * i + 1] : b[2 * i - 3]);
    hi[i] = bf16_pair(u, v);
    u -= __uint_as_float(hi[i] << 16), v -= __uint_as_float(hi[i] & 0xFFFF0000u);
    mid[i] = bf16_pair(u, v);
    u -= __uint_as_float(mid[i] << 16), v -= __uint_as_float(mid[i] & 0xFFFF0000u);
    lo[i] = bf16_pair(u, v);
  }
}

__device__ __forceinline__ void store_row(const FewK& a, int64_t m, int64_t n, float v) {
  if (a.dtype == ARTLITE_X_BF16)
    static_cast<uint16_t*>(a.y)[m * a.y_stride + n] = uint16_t(f32_to_bf16(v));
  else
    static_cast<float*>(a.y)[m * a.y_stride + n] = v;
}
// an output of row m, column n from its sum (gated: and the second matrix's)
template <bool GLU>
__device__ __forceinline__ void few_out(const FewK& a, int64_t m, int64_t n, float s, float u) {
  if constexpr (GLU) {
    store_planes(a.h + m * a.h_stride + n, a.h_plane, a.h_planes, gate_act(a.act, s) * u);
  } else {
    store_row(a, m, n, s + (a.bias ? a.bias[n] : 0.0f));
  }
}

// A launch's shape: tiles of a workgroup (each wave takes its units of all of them, so that an x operand serves them all),
// most waves (registers: 128 a lane of 16 waves)
constexpr int few_tiles(int nc, bool glu) { return nc == 2 ? (glu ? 2 : 4) : nc == 4 ? (glu ? 1 : 2) : 1; }
constexpr int few_most(int planes, int nc, bool glu) { return nc == 1 && planes <= 2 && !glu ? 16 : 8; }

// whether x goes by way of LDS: past 4 rows (1 row's operand loads take few cache accesses; 5 rows of 4096 x 4096 5.7 us as
// operands, 5.0 through LDS), of fp32 past 8 (5 rows of 1536 x 2880 8.4 us as operands, 9.1 through LDS)
constexpr bool few_stage(int ri, bool x32) { return ri > (x32 ? 2 : 1); }

// x's slot of a wave: NC blocks of 16 rows, CG groups of them (8 KiB or so: registers hold the next chunk), by planes
template <int P, int NC, bool X32>
struct FewStage {
  static constexpr int PL = X32 ? 1 : P, SIZE = X32 ? 128 : 64;  // (planes; bytes of a row's group in one)
  static constexpr int CG = NC * PL * SIZE <= 64 ? 8 : NC * PL * SIZE <= 128 ? 4 : NC * PL * SIZE <= 384 ? 2 : 1;
  static constexpr int PIECES = CG * SIZE / 16;                  // (of a row in a plane)
  static constexpr int PLANE = NC * 16 * CG * SIZE, BYTES = PL * PLANE, LOADS = BYTES / 1024;
  static_assert(PIECES % 4 == 0 && 64 % PIECES == 0, "pieces");
  __device__ static int turn(int r) { return PIECES >= 8 ? r & 7 : (r >> 1) & 3; }
};

// P planes of x, NC blocks of 16 rows, RI rows of a block a lane: block row 4 g + i is x's row g + 4 i, so that up to 4 rows
// are in each lane's first sum (RI 1) and up to 8 in its first two, and the others take no scaling. The units in gridDim.z
// parts (PART: their sums into a.parts, for k_few_join). X32: x is fp32, split into its planes as it is used.
template <int QT, int P, int NC, int RI, bool GLU, bool PART, bool X32>
__global__ __launch_bounds__(few_most(P, NC, GLU) * 64) void k_few(const FewK a) {
  constexpr int TB = few_tiles(NC, GLU), RB = GLU ? 2 * TB : TB, KIND = code_kind<QT, P>(), UB = unit_bytes<QT>();
  constexpr bool CIN = KIND < 0 || has_offset<QT>;  // (sum(x) times a constant is wanted)
  constexpr float CC = KIND < 0 ? (QT == ARTLITE_Q4_0 ? -136.0f : -128.0f) : -1.0f;
  constexpr uint32_t CB = bf16_of(int(CC)) * 0x10001u;
  constexpr float OM = KIND < 0 ? 1.0f / 128.0f : 1.0f;
  const Nibbles nib;
  // groups whose x is in flight, whether the next unit's codes are (registers)
  constexpr int XD = X32 ? 2 : P > 1 || GLU ? 4 : 8;
  constexpr bool AHEAD = NC == 1;
  using S = FewStage<P, NC, X32>;
  constexpr bool STAGE = few_stage(RI, X32);
  extern __shared__ __attribute__((aligned(16))) float red[];  // x's slots; then [wave][tile of a matrix][block][row][lane]
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6,
            lg = lane >> 4, lr = lane & 15;
  const int64_t t0 = int64_t(blockIdx.x) * TB, m0 = int64_t(blockIdx.y) * (16 * NC);
  const int first = PART ? int(int64_t(a.units) * blockIdx.z / gridDim.z) : 0;
  const int end = PART ? int(int64_t(a.units) * (blockIdx.z + 1) / gridDim.z) : a.units;
  const uint8_t* wp[RB];  // (a tile past the last: the last one's, unused)
#pragma unroll
  for (int b = 0; b < RB; b++)
    wp[b] = (GLU && b >= TB ? a.up : a.w) + min(t0 + b % TB, a.tiles - 1) * a.units * UB;
  // rows that there are not take row 0: each row of the products is its own
  constexpr int XE = X32 ? 4 : 2, PL = X32 ? 1 : P;  // (bytes of a value of x; its planes in memory)
  const auto xrow = [&](int r) __attribute__((always_inline)) {  // (row r of the NC blocks)
    const int64_t m = m0 + 16 * (r >> 4) + ((r & 15) >> 2) + 4 * (r & 3);
    return reinterpret_cast<const uint8_t*>(a.x) + (m < a.M ? m : 0) * a.x_stride * XE;
  };
  float acc[RB][NC][RI];
#pragma unroll
  for (int b = 0; b < RB; b++)
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int i = 0; i < RI; i++) acc[b][c][i] = 0.0f;

  uint4 code[RB][2];
  TileHdr<QT> hd[RB];
  auto load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; b++) {
      const uint8_t* p = wp[b] + int64_t(u) * UB;
#pragma unroll
      for (int h = 0; h < 2; h++) code[b][h] = *reinterpret_cast<const uint4*>(p + 1024 * h + 16 * lane);
      hd[b].load(p + 2048 + hdr_bytes<QT>() * lr);
    }
  };
  // Up to 4 rows: x of a group as its operand, loaded so. Past the last group of K the last one's (the scales there are 0).
  constexpr int XP = X32 ? 2 : P;  // (a group's loads: its planes, or 8 fp32 values in two)
  u32x4 x[STAGE ? 1 : XD][XP];
  const uint8_t* const xd = xrow(lr) + 8 * XE * lg;
  const int klast = int(a.K) - 32;
  auto load_x = [&](int j, int u, int g) __attribute__((always_inline)) {
    const int64_t k = min(u * UNIT + 32 * g, klast);
#pragma unroll
    for (int p = 0; p < XP; p++)  // (at any address: rows need not be aligned)
      __builtin_memcpy(&x[j][p], xd + (X32 ? 4 * k + 16 * p : 2 * (p * a.x_plane + k)), 16);
  };
  // More rows: x a chunk of CG groups at a time by way of the wave's own slot in LDS, in lines' order (an operand's own order
  // has 16 rows in a quarter of a wave: 64 cache accesses a load against 16, which bound 77 rows of 4096 x 4096 at 13 of 21
  // us), the next chunk's loads in flight while one is used. 16-byte pieces swizzled by row.
  uint8_t* const slot = reinterpret_cast<uint8_t*>(red) + wv * S::BYTES;
  u32x4 st[STAGE ? S::LOADS : 1];
  const uint8_t* sp[STAGE ? S::LOADS : 1];
  uint32_t sk = 0, sl[STAGE ? S::LOADS : 1];
  if constexpr (STAGE) {
#pragma unroll
    for (int i = 0; i < S::LOADS; i++) {
      const int q = (i % (S::LOADS / PL)) * 64 + lane, r = q / S::PIECES, c = q % S::PIECES;
      sp[i] = xrow(r) + 2 * int64_t(X32 ? 0 : i / (S::LOADS / PL)) * a.x_plane;
      sl[i] = (i / (S::LOADS / PL)) * S::PLANE + r * (16 * S::PIECES) + ((c ^ S::turn(r)) << 4);
      sk = 16 * c;  // (the same of every load: 64 is a multiple of PIECES)
    }
  }
  auto load_chunk = [&](int u, int g) __attribute__((always_inline)) {
    const int64_t at = min(int64_t(u * UNIT + 32 * g) * XE + sk, a.K * XE - 16);
#pragma unroll
    for (int i = 0; i < S::LOADS; i++) __builtin_memcpy(&st[i], sp[i] + at, 16);
  };
  if (first + wv < end) {
    if (AHEAD) load(first + wv);
    if constexpr (STAGE) {
      load_chunk(first + wv, 0);
    } else {
#pragma unroll
      for (int g = 0; g < XD; g++) load_x(g, first + wv, g);
    }
  }
  for (int u = first + wv; u < end; u += W) {
    const bool more = u + W < end;
    const int un = more ? u + W : u;  // (past the last unit x's loads are its own again, unread)
    uint4 cur[RB][2];
    TileHdr<QT> hc[RB];
    if (!AHEAD) load(u);
#pragma unroll
    for (int b = 0; b < RB; b++) {
      cur[b][0] = code[b][0], cur[b][1] = code[b][1];
      hc[b] = hd[b];
    }
    if (AHEAD && more) load(u + W);
    const auto half = [&](auto hv) __attribute__((always_inline)) {
      constexpr int H = decltype(hv)::value;
      float s[RB][4], o[RB][4];
#pragma unroll
      for (int b = 0; b < RB; b++) hc[b].template fields<H>(s[b], o[b], OM);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int g = 4 * H + j;
        const u32x4 cst{CB, CB, CB, CB};
        u32x4 xo[NC][P];
        if constexpr (STAGE) {
          if (g % S::CG == 0) {  // (the chunk's loads to the slot; the next chunk's go out)
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) *reinterpret_cast<u32x4*>(slot + sl[i]) = st[i];
            load_chunk(g + S::CG < 8 ? u : un, (g + S::CG) % 8);
          }
#pragma unroll
          for (int c = 0; c < NC; c++) {
            const uint8_t* r = slot + (16 * c + lr) * (16 * S::PIECES);
            const int piece = (g % S::CG) * (X32 ? 8 : 4);
            if constexpr (X32)
              split3(*reinterpret_cast<const u32x4*>(r + (((piece + 2 * lg) ^ S::turn(lr)) << 4)),
                     *reinterpret_cast<const u32x4*>(r + (((piece + 2 * lg + 1) ^ S::turn(lr)) << 4)), xo[c][0],
                     xo[c][P > 1 ? 1 : 0], xo[c][P - 1]);
            else
#pragma unroll
              for (int p = 0; p < P; p++)
                xo[c][p] = *reinterpret_cast<const u32x4*>(r + p * S::PLANE + (((piece + lg) ^ S::turn(lr)) << 4));
          }
        } else if constexpr (X32) {
          split3(x[g % XD][0], x[g % XD][XP - 1], xo[0][0], xo[0][P > 1 ? 1 : 0], xo[0][P - 1]);
        } else {
#pragma unroll
          for (int p = 0; p < P; p++) xo[0][p] = x[g % XD][p];
        }
        f32x4 cin[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) {
          cin[c] = f32x4{0, 0, 0, 0};
          if constexpr (CIN)
#pragma unroll
            for (int p = P - 1; p >= 0; p--) cin[c] = mfma(xo[c][p], cst, cin[c]);
        }
#pragma unroll
        for (int b = 0; b < RB; b++) {
          const uint4& cc = cur[b][H];
          const u32x4 q = operand<KIND>(j == 0 ? cc.x : j == 1 ? cc.y : j == 2 ? cc.z : cc.w, nib);
#pragma unroll
          for (int c = 0; c < NC; c++) {
            f32x4 d = KIND < 0 ? cin[c] : f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = P - 1; p >= 0; p--) d = mfma(xo[c][p], q, d);
#pragma unroll
            for (int i = 0; i < RI; i++) {
              acc[b][c][i] = __builtin_fmaf(s[b][j], d[i], acc[b][c][i]);
              if constexpr (has_offset<QT>)
                acc[b][c][i] = __builtin_fmaf(o[b][j], cin[c][i], acc[b][c][i]);
            }
          }
        }
        if constexpr (!STAGE) load_x(g % XD, g + XD < 8 ? u : un, (g + XD) % 8);
        if (P * NC > 1) __builtin_amdgcn_sched_barrier(0);  // (the groups' sums in turn: registers)
      }
    };
    half(std::integral_constant<int, 0>{});
    half(std::integral_constant<int, 1>{});
  }
  constexpr int ACC = NC * RI;
  if constexpr (STAGE) __syncthreads();  // (the slots' place)
#pragma unroll
  for (int b = 0; b < RB; b++)
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int i = 0; i < RI; i++) red[((wv * RB + b) * ACC + c * RI + i) * WAVE + lane] = acc[b][c][i];
  __syncthreads();
  // the waves' sums, in wave order: 64 outputs a wave at a time
  for (int q = wv; q < TB * ACC; q += W) {
    const int b = q / ACC, ci = q % ACC;
    float s = red[(b * ACC + ci) * WAVE + lane], v = GLU ? red[((b + TB) * ACC + ci) * WAVE + lane] : 0.0f;
    for (int w = 1; w < W; w++) {
      s += red[((w * RB + b) * ACC + ci) * WAVE + lane];
      if (GLU) v += red[((w * RB + b + TB) * ACC + ci) * WAVE + lane];
    }
    const int64_t n = (t0 + b) * TROWS + lr, m = m0 + 16 * (ci / RI) + lg + 4 * (ci % RI);
    if (n >= a.N || m >= a.M) continue;
    if constexpr (PART) {
      float* o = a.parts + (blockIdx.z * a.M + m) * a.part_row + n;
      o[0] = s;
      if (GLU) o[a.part_up] = v;
    } else {
      few_out<GLU>(a, m, n, s, v);
    }
  }
}

// the parts' sums, in order
template <bool GLU>
__global__ __launch_bounds__(256) void k_few_join(const FewK a, int parts) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x, m = i / a.N, n = i % a.N;
  if (m >= a.M) return;
  const float* p = a.parts + m * a.part_row + n;
  float s = 0.0f, u = 0.0f;
  for (int k = 0; k < parts; k++, p += a.M * a.part_row) {
    s += p[0];
    if (GLU) u += p[a.part_up];
  }
  few_out<GLU>(a, m, n, s, u);
}

__global__ __launch_bounds__(256) void k_planes(const float* __restrict__ x, int64_t K, int64_t stride,
                                                uint16_t* __restrict__ out, int64_t plane) {
  const int64_t m = blockIdx.y, k = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (k < K) store_planes(out + m * K + k, plane, 3, x[m * stride + k]);
}

// Tall matrices, up to 16 rows of x: a workgroup a CU; the tiles shared out among workgroups, a workgroup's units, tile after
// tile, evenly among its waves, so that a wave reads one run of memory from beginning to end with the next units in flight and
// leaves a sum only at a tile's end. x (as its planes) and the workgroup's biases are in LDS. A tile that several waves share:
// the one that begins it adds the others' shares, in order. What bounds it: the weights' bytes, and nearly as much the
// instructions (about 120 a unit and wave for one bf16 row).
constexpr int TALL_WAVES = 16, TALL_WGS = 256;
// From 1024 tiles of together 32768 units on (Q4_K, one row: 131072 x 2048 32 us against k_few's 39, 32768 x 4096 18.6
// against 21.9, 16384 x 12288 25 against 33; 16384 x 4096 13.2 against 10.4, 65536 x 1024 11.5 against 9.9). 16 rows of 131072
// x 2048: 41 us against 57; 3 rows of fp32: 59 against 89.
constexpr int64_t TALL_TILES = 1024, TALL_UNITS = 32768;

template <int QT, int P, int RI, bool X32>
__global__ __launch_bounds__(TALL_WAVES * 64) void k_tall(const FewK a) {
  constexpr int KIND = code_kind<QT, P>(), UB = unit_bytes<QT>(), D = 3;  // (units in flight)
  constexpr bool CIN = KIND < 0 || has_offset<QT>;
  constexpr float CC = KIND < 0 ? (QT == ARTLITE_Q4_0 ? -136.0f : -128.0f) : -1.0f;
  constexpr uint32_t CB = bf16_of(int(CC)) * 0x10001u;
  constexpr float OM = KIND < 0 ? 1.0f / 128.0f : 1.0f;
  const Nibbles nib;
  extern __shared__ __attribute__((aligned(16))) float red[];  // [wave][RI][lane]; x: [plane][row][units 256 + 8]; biases
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
  uint8_t* const xs = reinterpret_cast<uint8_t*>(red) + TALL_WAVES * RI * WAVE * 4;
  const int K = int(a.K), pitch = 2 * a.units * UNIT + 16, rows = int(a.M), plane = rows * pitch;
  float* const bias = reinterpret_cast<float*>(xs + P * plane);
  const int64_t t0 = a.tiles * blockIdx.x / gridDim.x, t1 = a.tiles * (blockIdx.x + 1) / gridDim.x;
  const int64_t all = (t1 - t0) * a.units;
  if (all == 0) return;
  const int64_t first = all * wv / TALL_WAVES, end = all * (wv + 1) / TALL_WAVES;
  const uint8_t* const last = a.w + (t1 * a.units - 1) * UB;

  u32x4 code[D][2];
  TileHdr<QT> hd[D];
  const uint8_t* next = a.w + (t0 * a.units + first) * UB;
  auto load = [&](auto sv) __attribute__((always_inline)) {
    constexpr int S = decltype(sv)::value;
    const uint8_t* p = next < last ? next : last;  // (past the run: unread)
#pragma unroll
    for (int h = 0; h < 2; h++) code[S][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 1024 * h + 16 * lane));
    hd[S].load(p + 2048 + hdr_bytes<QT>() * lr);
    next += UB;
  };
  load(std::integral_constant<int, 0>{});
  load(std::integral_constant<int, 1>{});
  load(std::integral_constant<int, 2>{});
  for (int m = 0; m < rows; m++)
    for (int k = 8 * threadIdx.x; k < a.units * UNIT; k += 8 * TALL_WAVES * 64) {
      u32x4 v[P];
#pragma unroll
      for (int i = 0; i < P; i++) v[i] = u32x4{0, 0, 0, 0};
      if (k < K) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.x) + (m * a.x_stride + k) * (X32 ? 4 : 2);
        if constexpr (X32) {
          u32x4 u[2];
          __builtin_memcpy(u, p, 32);
          split3(u[0], u[1], v[0], v[P > 1 ? 1 : 0], v[P - 1]);
        } else {
          __builtin_memcpy(v, p, 16);
        }
      }
#pragma unroll
      for (int i = 0; i < P; i++) *reinterpret_cast<u32x4*>(xs + i * plane + m * pitch + 2 * k) = v[i];
    }
  for (int64_t n = t0 * TROWS + threadIdx.x; n < t1 * TROWS; n += TALL_WAVES * 64)
    bias[n - t0 * TROWS] = a.bias && n < a.N ? a.bias[n] : 0.0f;
  __syncthreads();

  const int xr = (lr >> 2) + 4 * (lr & 3);
  const uint8_t* const x0 = xs + (xr < rows ? xr : 0) * pitch + 16 * lg;
  float acc[RI];
#pragma unroll
  for (int i = 0; i < RI; i++) acc[i] = 0.0f;
  int t = int(first / a.units), u = int(first - int64_t(t) * a.units);  // (the workgroup's tile)
  bool begun = u == 0;                                                // (the wave has the tile's first unit)
  const auto put = [&]() __attribute__((always_inline)) {
    const int64_t n = (t0 + t) * TROWS + lr;
    const float b = bias[t * TROWS + lr];
#pragma unroll
    for (int i = 0; i < RI; i++)
      if (n < a.N && lg + 4 * i < rows) store_row(a, lg + 4 * i, n, acc[i] + b);
  };
  const auto leave = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RI; i++) red[(wv * RI + i) * WAVE + lane] = acc[i];
  };
  const auto step = [&](auto sv) __attribute__((always_inline)) {
    constexpr int S = decltype(sv)::value;
    const uint8_t* const xu = x0 + 2 * UNIT * u;
    const auto half = [&](auto hv) __attribute__((always_inline)) {
      constexpr int H = decltype(hv)::value;
      float s[4], o[4];
      hd[S].template fields<H>(s, o, OM);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const u32x4 cst{CB, CB, CB, CB};
        u32x4 xo[P];
#pragma unroll
        for (int p = 0; p < P; p++) xo[p] = *reinterpret_cast<const u32x4*>(xu + p * plane + 64 * (4 * H + j));
        f32x4 cin{0, 0, 0, 0};
        if constexpr (CIN)
#pragma unroll
          for (int p = P - 1; p >= 0; p--) cin = mfma(xo[p], cst, cin);
        const u32x4 q = operand<KIND>(code[S][H][j], nib);
        f32x4 d = KIND < 0 ? cin : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int p = P - 1; p >= 0; p--) d = mfma(xo[p], q, d);
#pragma unroll
        for (int i = 0; i < RI; i++) {
          acc[i] = __builtin_fmaf(s[j], d[i], acc[i]);
          if constexpr (has_offset<QT>) acc[i] = __builtin_fmaf(o[j], cin[i], acc[i]);
        }
      }
    };
    half(std::integral_constant<int, 0>{});
    half(std::integral_constant<int, 1>{});
    load(sv);
    if (++u == a.units) {
      if (begun)
        put();
      else
        leave();
#pragma unroll
      for (int i = 0; i < RI; i++) acc[i] = 0.0f;
      u = 0, t++, begun = true;
    }
  };
  int64_t n = end - first;
  for (; n >= D; n -= D) {
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
  }
  if (n > 0) step(std::integral_constant<int, 0>{});
  if (n > 1) step(std::integral_constant<int, 1>{});
  if (!begun) leave();  // (a share with neither of the tile's ends, or none)
  __syncthreads();
  if (begun && u) {
    const int64_t until = int64_t(t + 1) * a.units;
    for (int w = wv + 1; w < TALL_WAVES && all * w / TALL_WAVES < until; w++)
#pragma unroll
      for (int i = 0; i < RI; i++) acc[i] += red[(w * RI + i) * WAVE + lane];
    put();
  }
}

size_t tall_lds(const FewK& k, int planes, int ri) {
  return size_t(TALL_WAVES) * ri * WAVE * 4 + size_t(planes) * size_t(k.M) * (size_t(k.units) * UNIT * 2 + 16) +
         size_t((k.tiles + TALL_WGS - 1) / TALL_WGS) * TROWS * 4;
}
template <int QT, int P, int RI, bool X32>
int launch_tall_t(const FewK& k, hipStream_t s) {
  static DeviceOnce set;
  if (!set.lds(reinterpret_cast<const void*>(k_tall<QT, P, RI, X32>), LDS_BYTES))
    return fail(ARTLITE_EHIP, "dense rows: kernel set-up failed");
  k_tall<QT, P, RI, X32><<<TALL_WGS, TALL_WAVES * 64, tall_lds(k, P, RI), s>>>(k);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

// How a product is shared out: the units of K in `parts` workgroups (where the groups of tiles leave half the CUs idle and a
// part has 4 units at least: 32 rows of 4096 x 4096, 64 groups, 13.8 us in one part, 12.8 in 4; 64 rows, 128 groups, 14.6 in
// one, 13.3 in 2; 77 rows, 256 groups, 14.8 in one, 21.2 in 2), a part's units among `waves` waves: up to 16 of them where the
// workgroups leave the device's waves few (16 rows of 4096 x 4096, 256 workgroups, in 16: 5.5 us, in 8 6.2; of 4608 x 8192,
// 288 workgroups, which are no longer all there at once, 14.5 and 12.5), 4 where they are enough, each with the same number
// of units but for the last.
struct FewCut {
  int64_t groups, blocks;
  int parts, waves;
};
// Blocks of 16 rows a workgroup's pass takes. More than one shares the weights' expansion and x's loads among tiles, but leaves
// few workgroups, which then take parts and a launch more (about 4 us): one where the products are few. 16384 unit products of
// one plane (4096 x 4096 Q4_K: 24 rows 12.1 us in passes of 32, 8.0 in blocks apart; 64 rows 13.1 and 12.3; 96 rows 15 and 17;
// 2048 x 2048, 64 rows, 10.7 and 5.2), half as many of more (2048 x 8192, two planes: 24 rows 14.3 and 14.3, 48 rows 16.5 and
// 22; 4096 x 4096, three: 24 rows 17.1 and 13.3, 48 rows 19.4 and 19.1).
constexpr int64_t FEW_APART = 16384;
int few_nc(int64_t tiles, int units, int64_t M, int planes, bool glu) {
  if (M <= 16 || tiles * units * (glu ? 2 : 1) * ((M + 15) / 16) <= FEW_APART / (planes > 1 ? 2 : 1)) return 1;
  return M <= 32 ? 2 : 4;
}
FewCut few_cut(int64_t tiles, int units, int64_t M, int planes, bool glu) {
  const int nc = few_nc(tiles, units, M, planes, glu), tb = few_tiles(nc, glu), most = few_most(planes, nc, glu);
  FewCut c{(tiles + tb - 1) / tb, (M + 16 * nc - 1) / (16 * nc), 1, 4};
  const int64_t wgs = c.groups * c.blocks;
  if (nc > 1)
    while (wgs * c.parts * 2 <= 256 && units / (2 * c.parts) >= 4) c.parts *= 2;
  const int own = (units + c.parts - 1) / c.parts;
  while (c.waves < (wgs > 256 ? 8 : most) && wgs * c.parts * c.waves < (nc > 1 ? 2048 : 4096)) c.waves *= 2;
  const int each = (own + c.waves - 1) / c.waves;
  c.waves = (own + each - 1) / each;
  return c;
}

template <int QT, int P, int NC, int RI, bool GLU, bool X32>
int launch_few_nc(const FewK& k, int raw, hipStream_t s) {
  constexpr int RED = (GLU ? 2 : 1) * few_tiles(NC, GLU) * NC * RI * WAVE * 4;
  constexpr int SLOT = few_stage(RI, X32) ? FewStage<P, NC, X32>::BYTES : 0;
  constexpr int WAVE_LDS = RED > SLOT ? RED : SLOT, LDS = few_most(P, NC, GLU) * WAVE_LDS;
  static_assert(LDS <= LDS_BYTES, "LDS");
  const FewCut c = few_cut(k.tiles, k.units, k.M, P, GLU);
  const size_t lds = size_t(c.waves) * WAVE_LDS;
  const dim3 grid(unsigned(c.groups), unsigned(c.blocks), unsigned(c.parts));
  constexpr bool PARTS = NC > 1 || GLU;
  static DeviceOnce set, set_part;
  if (!set.lds(reinterpret_cast<const void*>(k_few<QT, P, NC, RI, GLU, false, X32>), LDS) ||
      (PARTS && !set_part.lds(reinterpret_cast<const void*>(k_few<QT, P, NC, RI, GLU, PARTS, X32>), LDS)))
    return fail(ARTLITE_EHIP, "dense rows: kernel set-up failed");
  if (raw && (!PARTS || raw != c.parts)) return fail(ARTLITE_EINVAL, "dense rows: %d parts", raw);
  if (PARTS && (raw || c.parts > 1)) {
    if (!k.parts) return fail(ARTLITE_EINVAL, "dense rows: no scratch for parts");
    if constexpr (PARTS) k_few<QT, P, NC, RI, GLU, true, X32><<<grid, 64 * c.waves, lds, s>>>(k);
    ART_HIP(hipGetLastError());
    if (raw) return ARTLITE_OK;
    k_few_join<GLU><<<unsigned((k.M * k.N + 255) / 256), 256, 0, s>>>(k, c.parts);
  } else {
    k_few<QT, P, NC, RI, GLU, false, X32><<<grid, 64 * c.waves, lds, s>>>(k);
  }
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

template <int QT, int P, bool GLU, bool X32 = false>
int launch_few_p(const FewK& k, int raw, hipStream_t s) {
  if constexpr (!GLU && (P == 1 || X32))
    if (k.M <= 16 && k.tiles >= TALL_TILES && k.tiles * k.units >= TALL_UNITS && tall_lds(k, P, 4) <= size_t(LDS_BYTES))
      return k.M <= 4   ? launch_tall_t<QT, P, 1, X32>(k, s)
             : k.M <= 8 ? launch_tall_t<QT, P, 2, X32>(k, s)
                        : launch_tall_t<QT, P, 4, X32>(k, s);
  if (k.M <= 4) return launch_few_nc<QT, P, 1, 1, GLU, X32>(k, raw, s);
  if (k.M <= 8) return launch_few_nc<QT, P, 1, 2, GLU, X32>(k, raw, s);
  if (X32 || few_nc(k.tiles, k.units, k.M, P, GLU) == 1) return launch_few_nc<QT, P, 1, 4, GLU, X32>(k, raw, s);
  if (k.M <= 32) return launch_few_nc<QT, P, 2, 4, GLU, false>(k, raw, s);
  return launch_few_nc<QT, P, 4, 4, GLU, false>(k, raw, s);
}

template <int QT>
int launch_few_q(const FewArgs& a, const FewK& k, hipStream_t s) {
  if (a.x32) return a.up ? launch_few_p<QT, 3, true, true>(k, a.raw, s) : launch_few_p<QT, 3, false, true>(k, 0, s);
  if (a.up) return a.planes == 1 ? launch_few_p<QT, 1, true>(k, a.raw, s) : launch_few_p<QT, 3, true>(k, a.raw, s);
  return a.planes == 1   ? launch_few_p<QT, 1, false>(k, 0, s)
         : a.planes == 2 ? launch_few_p<QT, 2, false>(k, 0, s)
                         : launch_few_p<QT, 3, false>(k, 0, s);
}

// ---- the transposed product: out[m][k] = sum_n x[m][n] W[n][k], for few rows
//
// Mathematics. W's values as fp16 times 2^-e, rounded once (fp32 calls: two planes), as the large tiles have them; x fp16 rows
// scaled by rows. The MFMA sums over what lies in a lane's registers, and there a tile has 8 values of one row n, so the codes
// are turned first, by the MFMA itself: codes (bf16, exact) times a matrix of ones and zeros that picks 16 of the group's 32
// columns give c[n][k] in fp32 with 4 rows n in a lane, whose scales and offsets make them values, which are rounded and are
// then an operand of 32 rows (4 and 4 of two tiles) as they are. No weight goes through memory or LDS.
//
// Shape. A workgroup takes a unit (256 columns; past 32 rows of x half of one) and a part of the tiles, its waves pairs of
// tiles in turn; their sums meet in LDS, the parts' in k_join. The scales go to lanes by way of the wave's slot in LDS. What
// bounds it: about 4 instructions a weight and lane, and the launch.
struct FewTK {
  const uint8_t* w[2];
  const uint16_t* x[2];
  int pairs;
  int64_t tiles;
  int units;
  int64_t M, ld, x_plane;
  int e;
  float* parts;
  int64_t part_row;
};
constexpr int FEW_T_WAVES = 8;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// PL planes of x and W, NC blocks of 16 rows of x, HU halves of a unit
template <int QT, int PL, int NC, int HU>
__global__ __launch_bounds__(FEW_T_WAVES * 64) void k_few_t(const FewTK a) {
  constexpr int KIND = iq4<QT> ? 0 : -1, UB = unit_bytes<QT>(), G = 4 * HU, CB = 2 * G;
  constexpr float CC = KIND < 0 ? (QT == ARTLITE_Q4_0 ? -136.0f : -128.0f) : 0.0f;
  constexpr int RED = 4 * NC * 4 * WAVE;  // (a wave's sums of four blocks of 16 columns)
  extern __shared__ __attribute__((aligned(16))) float red[];  // [wave][RED]; in the loop the scales: [tile][2][group][row]
  const Nibbles nib;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
  const int u = HU == 2 ? blockIdx.x : blockIdx.x >> 1, h0 = HU == 2 ? 0 : blockIdx.x & 1;
  const int64_t m0 = int64_t(blockIdx.y) * (16 * NC);
  const int each = int(a.tiles / 2), all = each * a.pairs;  // (pairs of tiles)
  const int first = int(int64_t(all) * blockIdx.z / gridDim.z), end = int(int64_t(all) * (blockIdx.z + 1) / gridDim.z);
  float* const slot = red + wv * RED;
  static_assert(RED >= 2 * 2 * G * TROWS, "the scales' slot");

  // ones that pick column 16 i + lr of a group's 32
  u32x4 pick[2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int d = 0; d < 4; d++)
      pick[i][d] = lg == 2 * i + (lr >> 3) && d == ((lr & 7) >> 1) ? (lr & 1 ? 0x3F800000u : 0x3F80u) : 0u;
  int64_t xp[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) {  // (rows that there are not take the block's first)
    const int64_t m = m0 + 16 * c + (lr >> 2) + 4 * (lr & 3);
    xp[c] = (m < a.M ? m : m0) * a.ld + 4 * lg;
  }
  f32x4 acc[CB][NC];
#pragma unroll
  for (int b = 0; b < CB; b++)
#pragma unroll
    for (int c = 0; c < NC; c++) acc[b][c] = f32x4{0, 0, 0, 0};

  uint4 code[2][HU];
  TileHdr<QT> hd;
  uint2 x[NC][PL][2];
  // (lane group lg has the header of tile lg % 2)
  const auto load = [&](int p) __attribute__((always_inline)) {
    const int sg = p >= each ? 1 : 0, t = 2 * (p - sg * each);
    const uint8_t* w = (sg ? a.w[1] : a.w[0]) + (int64_t(t) * a.units + u) * UB;
    const uint8_t* const wt[2] = {w, w + int64_t(a.units) * UB};
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int h = 0; h < HU; h++) code[b][h] = *reinterpret_cast<const uint4*>(wt[b] + 1024 * (h0 + h) + 16 * lane);
    hd.load((lg & 1 ? wt[1] : wt[0]) + 2048 + hdr_bytes<QT>() * lr);
    const uint16_t* xs = (sg ? a.x[1] : a.x[0]) + 16 * t;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int q = 0; q < PL; q++)
#pragma unroll
        for (int b = 0; b < 2; b++)
          x[c][q][b] = *reinterpret_cast<const uint2*>(xs + xp[c] + q * a.x_plane + 16 * b);
  };
  if (first + wv < end) load(first + wv);
  for (int p = first + wv; p < end; p += FEW_T_WAVES) {
    uint4 cur[2][HU];
    f16x8 xo[NC][PL];
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int h = 0; h < HU; h++) cur[b][h] = code[b][h];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int q = 0; q < PL; q++)
        xo[c][q] = __builtin_bit_cast(f16x8, u32x4{x[c][q][0].x, x[c][q][0].y, x[c][q][1].x, x[c][q][1].y});
    {
      // the scales of half h of the tile's row lr: of a unit, lane groups 0, 1 have the first half's, 2, 3 the second's
      float s[4], o[4] = {0, 0, 0, 0}, s1[4], o1[4] = {0, 0, 0, 0};
      hd.template fields<0>(s, o);
      hd.template fields<1>(s1, o1);
      const bool second = HU == 2 ? lg >= 2 : h0 == 1;
      float* const at = slot + ((lg & 1) * 2 * G + (HU == 2 && second ? 4 : 0)) * TROWS + lr;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        at[j * TROWS] = __builtin_amdgcn_ldexpf(second ? s1[j] : s[j], -a.e);
        if constexpr (has_offset<QT>) at[(G + j) * TROWS] = __builtin_amdgcn_ldexpf(second ? o1[j] : o[j], -a.e);
      }
    }
    load(p + FEW_T_WAVES < end ? p + FEW_T_WAVES : p);
    __builtin_amdgcn_wave_barrier();  // (the wave's own slot: its writes come before its reads)
#pragma unroll
    for (int g = 0; g < G; g++) {
      u32x4 q[2];
      f32x4 s[2], o[2];
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const uint4& cc = cur[b][g / 4];
        q[b] = operand<KIND>(g % 4 == 0 ? cc.x : g % 4 == 1 ? cc.y : g % 4 == 2 ? cc.z : cc.w, nib);
        s[b] = *reinterpret_cast<const f32x4*>(slot + (b * 2 * G + g) * TROWS + 4 * lg);
        if constexpr (has_offset<QT>) o[b] = *reinterpret_cast<const f32x4*>(slot + ((b * 2 + 1) * G + g) * TROWS + 4 * lg);
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        f16x8 hi, lo;
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const f32x4 c = mfma(q[b], pick[i], f32x4{CC, CC, CC, CC});
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float v = has_offset<QT> ? __fsub_rn(__fmul_rn(s[b][r], c[r]), o[b][r]) : s[b][r] * c[r];
            hi[4 * b + r] = _Float16(v);
            if constexpr (PL == 2) lo[4 * b + r] = _Float16(v - float(hi[4 * b + r]));
          }
        }
#pragma unroll
        for (int c = 0; c < NC; c++) {
          f32x4& d = acc[2 * g + i][c];
          if constexpr (PL == 2) {
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(xo[c][PL - 1], hi, d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(xo[c][0], lo, d, 0, 0, 0);
          }
          d = __builtin_amdgcn_mfma_f32_16x16x32_f16(xo[c][0], hi, d, 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (the groups in turn: registers)
    }
    __builtin_amdgcn_wave_barrier();
  }
  // the waves' sums, in wave order, four blocks of 16 columns at a time: block row 4 g + i is x's row g + 4 i
#pragma unroll
  for (int f = 0; f < CB; f += 4) {
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (m0 + 16 * c + 4 * i < a.M) slot[((b * NC + c) * 4 + i) * WAVE + lane] = acc[f + b][c][i];
    __syncthreads();
    for (int j = wv; j < 16 * NC; j += FEW_T_WAVES) {
      const int64_t m = m0 + 16 * (j / 4 % NC) + 4 * (j % 4) + lg, k = u * UNIT + h0 * (UNIT / 2) + 16 * (f + j / (4 * NC)) + lr;
      if (m >= a.M || k >= a.part_row) continue;
      float s = 0.0f;
      for (int w = 0; w < FEW_T_WAVES; w++) s += red[w * RED + j * WAVE + lane];
      a.parts[(blockIdx.z * a.M + m) * a.part_row + k] = s;
    }
  }
}

struct FewTCut {
  int nc, cols, parts;
};
// blocks of 16 rows and halves of a unit by what registers hold; one workgroup a CU, each wave a pair of tiles at least
constexpr int few_t_halves(int nc, int planes) { return nc * planes <= 2 ? 2 : 1; }
FewTCut few_t_cut(int64_t tiles, int units, int pairs, int planes, int64_t M) {
  FewTCut c{M <= 16 ? 1 : M <= 32 || planes == 2 ? 2 : 4, units, 1};
  c.cols = units * (3 - few_t_halves(c.nc, planes));
  const int64_t wgs = c.cols * ((M + 16 * c.nc - 1) / (16 * c.nc)), all = tiles / 2 * pairs;
  c.parts = int(std::max<int64_t>(1, std::min<int64_t>(256 / wgs, (all + FEW_T_WAVES - 1) / FEW_T_WAVES)));
  return c;
}
template <int QT, int PL, int NC, int HU>
int launch_few_t_nc(const FewTK& k, const FewTCut& c, hipStream_t s) {
  constexpr int LDS = FEW_T_WAVES * 4 * NC * 4 * WAVE * 4;
  static DeviceOnce set;
  if (!set.lds(reinterpret_cast<const void*>(k_few_t<QT, PL, NC, HU>), LDS))
    return fail(ARTLITE_EHIP, "dense rows: kernel set-up failed");
  k_few_t<QT, PL, NC, HU><<<dim3(unsigned(c.cols), unsigned((k.M + 16 * NC - 1) / (16 * NC)), unsigned(c.parts)),
                            FEW_T_WAVES * 64, LDS, s>>>(k);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}
template <int QT, int PL>
int launch_few_t_p(const FewTK& k, hipStream_t s) {
  const FewTCut c = few_t_cut(k.tiles, k.units, k.pairs, PL, k.M);
  if (c.nc == 1) return launch_few_t_nc<QT, PL, 1, few_t_halves(1, PL)>(k, c, s);
  if (PL == 2 || c.nc == 2) return launch_few_t_nc<QT, PL, 2, few_t_halves(2, PL)>(k, c, s);
  return launch_few_t_nc<QT, PL, PL == 1 ? 4 : 2, 1>(k, c, s);
}

}  // namespace

bool few_apart(const artlite_matrix* w, int planes, bool gated, int64_t M) {
  return few_nc(w->tiles, w->units, M, planes, gated) == 1;
}

size_t few_parts_bytes(const artlite_matrix* w, int planes, bool gated, int64_t M) {
  if (few_apart(w, planes, gated, M)) return 0;
  const FewCut c = few_cut(w->tiles, w->units, M, planes, gated);
  return c.parts > 1 ? size_t(c.parts) * M * w->N * (gated ? 2 : 1) * 4 : 0;
}

int few_raw_parts(const artlite_matrix* w, int planes, int64_t M) {
  return few_cut(w->tiles, w->units, M, planes, true).parts;
}

int launch_few(const FewArgs& a, hipStream_t s) {
  if (a.M <= 0) return ARTLITE_OK;
  if (a.x32 && !few_apart(a.w, 3, a.up != nullptr, a.M))
    return fail(ARTLITE_EINVAL, "dense rows: %lld fp32 rows", (long long)a.M);
  if (a.M > int64_t(65535) * 16) return fail(ARTLITE_EINVAL, "dense rows: %lld rows", (long long)a.M);
  FewK k{};
  k.w = a.w->w.as<uint8_t>();
  k.up = a.up ? a.up->w.as<uint8_t>() : nullptr;
  k.tiles = a.w->tiles, k.units = a.w->units;
  k.N = a.w->N, k.K = a.w->K, k.M = a.M;
  k.x = static_cast<const uint16_t*>(a.x), k.x_stride = a.x_stride, k.x_plane = a.x_plane;
  k.bias = a.w->has_bias ? a.w->bias.as<float>() : nullptr;
  k.y = a.y, k.y_stride = a.y_stride, k.dtype = a.dtype, k.act = a.act;
  k.h = a.h, k.h_stride = a.h_stride, k.h_plane = a.h_plane, k.h_planes = a.h_planes;
  k.parts = a.parts;
  k.part_up = a.raw ? pad64(k.N) : k.N, k.part_row = (a.up ? 2 : 1) * k.part_up;
#define ART_F(QT) return launch_few_q<QT>(a, k, s)
  ART_TILE_QTYPES(a.w->t->id, ART_F)
#undef ART_F
}

int few_t_parts(const artlite_matrix* w, int pairs, int planes, int64_t M) {
  return few_t_cut(w->tiles, w->units, pairs, planes, M).parts;
}
size_t few_t_bytes(const artlite_matrix* w, int pairs, int planes, int64_t M) {
  return size_t(few_t_parts(w, pairs, planes, M)) * M * pad64(w->K) * 4;
}

int launch_few_t(const FewTArgs& a, hipStream_t s) {
  if (a.M <= 0) return ARTLITE_OK;
  const artlite_matrix *w = a.w[0], *v = a.pairs == 2 ? a.w[1] : w;
  if (a.pairs < 1 || a.pairs > 2 || v->N != w->N || v->K != w->K || v->t != w->t || w->N % 32 || a.ld % 64 || a.ld < w->N ||
      a.planes < 1 || a.planes > 2 || !a.parts || a.M > int64_t(65535) * 16)
    return fail(ARTLITE_EINVAL, "dense rows, transposed: %lld rows of %lld", (long long)a.M, (long long)a.ld);
  FewTK k{};
  for (int i = 0; i < a.pairs; i++) k.w[i] = a.w[i]->w.as<uint8_t>(), k.x[i] = a.x[i];
  k.pairs = a.pairs, k.tiles = w->tiles, k.units = w->units, k.M = a.M;
  k.ld = a.ld, k.x_plane = a.x_plane, k.e = a.e;
  k.parts = a.parts, k.part_row = pad64(w->K);
#define ART_T(QT) return a.planes == 1 ? launch_few_t_p<QT, 1>(k, s) : launch_few_t_p<QT, 2>(k, s)
  ART_TILE_QTYPES(w->t->id, ART_T)
#undef ART_T
}

int launch_planes(const float* x, int64_t M, int64_t K, int64_t stride, uint16_t* out, hipStream_t s) {
  for (int64_t m = 0; m < M; m += 65535) {
    const int64_t rows = M - m < 65535 ? M - m : 65535;
    k_planes<<<dim3(unsigned((K + 255) / 256), unsigned(rows)), 256, 0, s>>>(x + m * stride, K, stride, out + m * K, M * K);
    ART_HIP(hipGetLastError());
  }
  return ARTLITE_OK;
}

}  // namespace artlite
