// The large tiles: out = A B^T over fp16 rows with fp32 sums, on the MFMA (16x16x32), with the epilogues of the dense
// products (a scaled store, the gated activation, its backward).
//
// Shape. A workgroup of 4 waves takes a tile of TM x TM outputs, a wave a quarter of it ((16 MB)^2: 128 x 128 of the large
// tile, its 256 sums a lane in the accumulation registers, one wave a SIMD; 64 x 64 of the small one, two workgroups a CU).
// K streams in steps of 32 values through a ring of 4 LDS slots filled by DMA (global_load_lds by asm, so that the compiler
// does not wait for it), three steps ahead; operands go from LDS to registers a step ahead of the MFMAs that use them, so one
// barrier a step is all that a wave waits for. At its barrier a step's successor has landed (every wave has waited for its
// own loads) and the slot that is filled next has been read (a step before the last).
// Rows of a slot are 64 bytes, four 16-byte chunks, chunk c of row r at c ^ (r / 2 % 4): the 16 rows that a lane group reads
// take all banks. Rows past the matrices' ends repeat the last one, their outputs are not stored.
// The weights' block is the MFMA's first operand, so a lane holds four consecutive columns of one output row.
// Tiles are dealt so that the workgroups that run on an XCD at a time share rows and columns (its L2 holds them).
#include "hgemm.h"

#include "matrix.h"

#include <utility>

namespace artlite {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int N>
__device__ __forceinline__ void hg_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
__device__ __forceinline__ void hg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ uint32_t hg_lds_addr(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}
// a pointer that every lane has alike, in scalar registers
__device__ __forceinline__ const uint16_t* hg_uniform(const uint16_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return reinterpret_cast<const uint16_t*>(uint64_t(hi) << 32 | lo);
}
// one DMA of 16 bytes a lane from base (uniform) + off (the lane's) into LDS at lds (uniform) + 16 lane
__device__ __forceinline__ void hg_dma(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
               : "memory");
}
__device__ __forceinline__ f32x4 hg_mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename F, int... I>
__device__ __forceinline__ void hg_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void hg_for(F&& f) {
  hg_for_impl(f, std::make_integer_sequence<int, N>{});
}

constexpr int BK = 32;

template <int MB>
struct HT {
  static constexpr int TM = 32 * MB;                 // rows and columns of a tile
  static constexpr int HALF = TM * BK * 2;           // bytes of an operand's step
  static constexpr int SLOT = 2 * HALF;
  static constexpr int RING = MB == 8 ? 4 : 5;       // (all of LDS, or half: two small tiles a CU)
  static constexpr int LPW = SLOT / 1024 / 4;        // DMAs of a wave a step
  static constexpr int LDS = RING * SLOT;
  static_assert(LDS <= (MB == 8 ? LDS_BYTES : LDS_BYTES / 2), "LDS");
};

// eight values as fp16 at p, and with a second plane what their rounding left
template <bool TWO>
__device__ __forceinline__ void store16(uint16_t* p, int64_t plane, const float (&v)[8]) {
  f16x8 a, b;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    a[i] = _Float16(v[i]);
    if constexpr (TWO) b[i] = _Float16(v[i] - float(a[i]));
  }
  *reinterpret_cast<f16x8*>(p) = a;
  if constexpr (TWO) *reinterpret_cast<f16x8*>(p + plane) = b;
}
// eight fp16 values, the sum of two planes where there are
template <bool TWO>
__device__ __forceinline__ void load16(const uint16_t* p, int64_t plane, float (&v)[8]) {
  const f16x8 a = *reinterpret_cast<const f16x8*>(p);
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = float(a[k]);
  if constexpr (TWO) {
    const f16x8 b = *reinterpret_cast<const f16x8*>(p + plane);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] += float(b[k]);
  }
}

// a row's exponents: of its sums, of what is written, of h beside dg and du, of dh
struct RowExp {
  int sum, out, h, dh;
};

// columns n .. n + 8 of row m of the planes from their sums v (gated: and the second matrix's u); the exponents of what is
// written go into its factors, so that each value takes one scaling
template <int EPI, bool TWO>
__device__ __forceinline__ void finish16(const HGemm& g, int es, const RowExp& r, int64_t m, int64_t n, float (&v)[8],
                                         float (&u)[8]) {
  const int64_t at = m * g.h_stride + n;
  const int ev = es + r.sum, eu = es - g.e + g.e2 + r.sum;
  const int there = int(max(int64_t(0), min(int64_t(8), g.N - n)));  // (columns that there are)
  float d[8], h[8];
  if constexpr (EPI == H_DGLU) load16<TWO>(g.dh + at, g.h_plane, d);
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if constexpr (EPI == H_ROWS) {
      v[k] = __builtin_amdgcn_ldexpf(v[k], ev - r.out);
    } else if constexpr (EPI == H_GLU) {
      v[k] = gate_act<TWO>(g.act, __builtin_amdgcn_ldexpf(v[k], ev)) * __builtin_amdgcn_ldexpf(u[k], eu - r.out);
    } else {
      const float uv = __builtin_amdgcn_ldexpf(u[k], eu), dh = __builtin_amdgcn_ldexpf(d[k], r.dh - r.out);
      float a, da;
      gate_act_grad<TWO>(g.act, __builtin_amdgcn_ldexpf(v[k], ev), a, da);
      h[k] = a * __builtin_amdgcn_ldexpf(u[k], eu - r.h);
      v[k] = dh * uv * da;
      u[k] = dh * a;
    }
  }
  if (there < 8) {
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k >= there) v[k] = u[k] = h[k] = 0.0f;
  }
  if constexpr (EPI == H_DGLU) {
    store16<TWO>(g.dg + at, g.h_plane, v);
    store16<TWO>(g.du + at, g.h_plane, u);
    if (g.h) store16<TWO>(g.h + at, g.h_plane, h);
  } else {
    store16<TWO>(g.h + at, g.h_plane, v);
  }
}

// columns n .. n + 8 of row m from their sums v (gated: and the second matrix's u)
template <int EPI>
__device__ __forceinline__ void finish(const HGemm& g, int es, const RowExp& r, int64_t m, int64_t n, float (&v)[8],
                                       float (&u)[8], const float (&bias)[8]) {
  if constexpr (EPI == H_STORE) {
    const int there = int(max(int64_t(0), min(int64_t(8), g.N - n)));  // (columns that there are)
    if (there == 0) return;
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = __builtin_amdgcn_ldexpf(v[k], es + r.sum);
    if (g.bias)
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] += bias[k];
    const int64_t at = m * g.y_stride + n;
    if (g.dtype == ARTLITE_X_BF16) {
      uint16_t* y = static_cast<uint16_t*>(g.y) + at;
      if (there == 8 && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = bf16_pair(v[2 * k], v[2 * k + 1]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(y));
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k < there) y[k] = uint16_t(f32_to_bf16(v[k]));
      }
    } else {
      float* y = static_cast<float*>(g.y) + at;
      if (there == 8 && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(y));
        __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(y + 4));
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k < there) y[k] = v[k];
      }
    }
  } else {
    if (n >= g.h_cols) return;
    if (g.planes == 2)
      finish16<EPI, true>(g, es, r, m, n, v, u);
    else
      finish16<EPI, false>(g, es, r, m, n, v, u);
  }
}

template <int EPI>
constexpr bool gated = EPI == H_GLU || EPI == H_DGLU;
template <int EPI>
__device__ __forceinline__ RowExp row_exp(const HGemm& g, int64_t m) {
  return RowExp{g.row_e ? g.row_e[m] : 0, EPI != H_STORE ? g.out_e[m] : 0, EPI == H_DGLU && g.h ? g.h_e[m] : 0,
                EPI == H_DGLU ? g.dh_e[m] : 0};
}
// a part's sums: rows of pad64(N) floats, of a gated pair both matrices' side by side
template <int EPI>
__host__ __device__ __forceinline__ int64_t part_row(const HGemm& g) {
  return (gated<EPI> ? 2 : 1) * pad64(g.N);
}

// gm x gn tiles from column 0 on; K in gridDim.y parts (PART: their sums into g.parts, for k_join)
template <int MB, int EPI, bool PART>
__global__ __launch_bounds__(256, MB == 8 ? 1 : 2) void k_hgemm(const HGemm g, int gm, int gn) {
  using T = HT<MB>;
  constexpr int TM = T::TM, RING = T::RING;
  constexpr bool GATED = gated<EPI>;
  constexpr int TN = GATED ? TM / 2 : TM;  // output columns of a tile
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
  const int wm = wv >> 1, wn = wv & 1;

  // ---- the tile: the workgroups of an XCD (every eighth) take a run of tiles, in columns of 4 tile rows
  int mt, nt;
  {
    const int total = gm * gn, per = total / 8, rest = total % 8;
    const int x = int(blockIdx.x) & 7, i = int(blockIdx.x) >> 3;
    const int t = x * per + (x < rest ? x : rest) + i;
    constexpr int GR = 4;
    const int band = t / (GR * gn), in = t % (GR * gn), rows = min(GR, gm - band * GR);
    mt = __builtin_amdgcn_readfirstlane(band * GR + in % rows);
    nt = __builtin_amdgcn_readfirstlane(in / rows);
  }
  const int64_t m0 = int64_t(mt) * TM, n0 = int64_t(nt) * TN;
  const int mv = int(min(int64_t(TM), g.M - m0)), nv = int(min(int64_t(TN), g.N - n0));  // (rows, columns that there are)

  // ---- the issue side: a wave's DMAs of a step take 16 rows each, HPW of A's and HPW of B's (a wave's columns of a gated
  // tile are its rows of the first matrix, then the same of the second: every second wave loads the second's)
  constexpr int HPW = T::LPW / 2;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(hg_lds_addr(lds));
  uint32_t offa[HPW], offb[HPW];
#pragma unroll
  for (int i = 0; i < HPW; i++) {
    const int r = 16 * (HPW * wv + i) + (lane >> 2), c = (lane & 3) ^ ((r >> 1) & 3);
    const int rb = GATED ? r / (TM / 2) * (TM / 4) + r % (TM / 4) : r;
    offa[i] = uint32_t(min(r, mv - 1)) * uint32_t(g.lda) * 2 + 16 * c;
    offb[i] = uint32_t(min(rb, nv - 1)) * uint32_t(g.ldb) * 2 + 16 * c;
  }
  // K in pairs of steps (64 values), a part of them; pair j's first values at (pa, pb): a segment's, then the next one's,
  // past the last pair its own again (loads into slots that are not read: the counts stay)
  const int pairs_seg = int(g.K / (2 * BK)), all = pairs_seg * g.segs;
  const int first = PART ? int(int64_t(all) * blockIdx.y / gridDim.y) : 0;
  const int pairs = PART ? int(int64_t(all) * (blockIdx.y + 1) / gridDim.y) - first : all;
  int iseg = PART ? first / pairs_seg : 0, ipair = PART ? first % pairs_seg : 0;
  const uint16_t *pa, *pb;
  auto open_seg = [&]() {
    pa = hg_uniform(g.a[iseg] + m0 * g.lda + ipair * (2 * BK));
    pb = hg_uniform((GATED && (wv & 1) ? g.b2[iseg] : g.b[iseg]) + n0 * g.ldb + ipair * (2 * BK));
  };
  auto next_pair = [&]() {
    if (++ipair < pairs_seg) {
      pa += 2 * BK, pb += 2 * BK;
    } else if (iseg + 1 < g.segs) {
      ipair = 0, iseg++;
      open_seg();
    } else {
      ipair = pairs_seg - 1;
    }
  };
  // DMA i of a step at (a, b) into slot
  auto dma = [&](int i, const uint16_t* a, const uint16_t* b, int slot) __attribute__((always_inline)) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(lds0 + slot * T::SLOT + (HPW * wv + (i >> 1)) * 1024);
    if (i & 1)
      hg_dma(hg_uniform(b), offb[i >> 1], d + T::HALF);
    else
      hg_dma(hg_uniform(a), offa[i >> 1], d);
  };

  f32x4 acc[MB][MB];
  hg_for<MB>([&](auto i) {
    hg_for<MB>([&](auto j) { acc[i][j] = f32x4{0, 0, 0, 0}; });
  });
  const uint32_t lo = lr * 64 + ((lg ^ ((lr >> 1) & 3)) << 4);
  const uint8_t* const la = lds + wm * (TM / 2) * 64 + lo;
  const uint8_t* const lb = lds + T::HALF + wn * (TM / 2) * 64 + lo;
  // B's operands of a step, and the next step's as they are read; A's in a window of 4, read two blocks ahead. Each block's
  // products stay behind its loads and reads (sched_barrier: the scheduler would gather the reads before their uses).
  u32x4 fa[4], fb[2][MB];
  auto ld = [](const uint8_t* p) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4*>(p); };
  // a step of a pair (SET: which of its two) on the slot `slot`, its successor in the next one; loads from (a, b) into the
  // slot before it
  int slot = 0;
  auto step = [&](auto set, const uint16_t* a, const uint16_t* b) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
    const int nslot = slot + 1 < RING ? slot + 1 : 0, islot = slot > 0 ? slot - 1 : RING - 1;
    hg_wait<(RING - 3) * T::LPW>();
    hg_barrier();
    const uint8_t *sa = la + slot * T::SLOT, *na = la + nslot * T::SLOT, *nb = lb + nslot * T::SLOT;
    hg_for<MB>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      fb[1 - S][i] = ld(nb + 1024 * i);
      fa[(i + 2) % 4] = i + 2 < MB ? ld(sa + 1024 * (i + 2)) : ld(na + 1024 * (i + 2 - MB));
      dma(i, a, b, islot);
      hg_for<MB>([&](auto j) __attribute__((always_inline)) { acc[i][j] = hg_mfma(fb[S][j], fa[i % 4], acc[i][j]); });
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = nslot;
  };
  static_assert(T::LPW == MB && (RING == 4 || RING == 5), "a DMA a block; 3 or 4 steps ahead");
  open_seg();
  for (int i = 0; i < MB; i++) dma(i, pa, pb, 0);
  for (int i = 0; i < MB; i++) dma(i, pa + BK, pb + BK, 1);
  next_pair();
  for (int i = 0; i < MB; i++) dma(i, pa, pb, 2);
  if constexpr (RING == 5)
    for (int i = 0; i < MB; i++) dma(i, pa + BK, pb + BK, 3);
  hg_wait<(RING - 2) * T::LPW>();
  hg_barrier();
  hg_for<MB>([&](auto j) { fb[0][j] = ld(lb + 1024 * decltype(j)::value); });
  fa[0] = ld(la);
  fa[1] = ld(la + 1024);
  // pair p's two steps; loaded meanwhile the steps RING - 1 after them: the second of pair p + 1 and the first of pair p + 2,
  // or both of pair p + 2
  for (int p = 0; p < pairs; p++) {
    const uint16_t *a1 = pa + BK, *b1 = pb + BK;
    next_pair();
    step(std::integral_constant<int, 0>{}, RING == 4 ? a1 : pa, RING == 4 ? b1 : pb);
    step(std::integral_constant<int, 1>{}, RING == 4 ? pa : pa + BK, RING == 4 ? pb : pb + BK);
  }
  hg_wait<0>();  // (every load of the workgroup has landed: the sums take its LDS)
  hg_barrier();

  // (the rows' exponents, so that no load is waited for row by row)
  RowExp* const rows_e = reinterpret_cast<RowExp*>(lds + T::LDS - TM * sizeof(RowExp));
  if constexpr (!PART) {
    for (int r = threadIdx.x; r < TM; r += 256) rows_e[r] = row_exp<EPI>(g, m0 + min(r, mv - 1));
    __syncthreads();
  }

  // ---- outputs, 32 of the wave's rows at a time by way of its own part of LDS, from where a lane takes 8 columns of a row
  constexpr int LROW = 16 * MB + 4;                    // (a row's floats and 4 more: banks)
  constexpr int COLS = GATED ? 8 * MB : 16 * MB;       // the wave's output columns
  constexpr int LPR = COLS / 8, RPI = 64 / LPR;        // lanes a row, rows an iteration
  float* const buf = reinterpret_cast<float*>(lds) + wv * 32 * LROW;
  static_assert(4 * 32 * LROW * 4 + TM * sizeof(RowExp) <= T::LDS, "LDS");
  const int es = PART ? 0 : g.e + (g.e0 ? *g.e0 : 0) + (g.e1 ? *g.e1 : 0);
  const int64_t n = n0 + wn * COLS + 8 * (lane % LPR);
  const float* const from = buf + (lane / LPR) * LROW + 8 * (lane % LPR);
  const auto get = [](const float* p, float(&v)[8]) __attribute__((always_inline)) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = a[k], v[4 + k] = b[k];
  };
  float bias[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (EPI == H_STORE && !PART && g.bias)
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (n + k < g.N) bias[k] = g.bias[n + k];
  auto put = [&](auto pc) __attribute__((always_inline)) {
    hg_for<2>([&](auto ic) __attribute__((always_inline)) {
      hg_for<MB>([&](auto jc) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
        *reinterpret_cast<f32x4*>(buf + (16 * i + lr) * LROW + 16 * j + 4 * lg) = acc[2 * decltype(pc)::value + i][j];
      });
    });
  };
  // (one copy of the rows' code: instructions that run once come from memory)
#pragma unroll 1
  for (int P = 0; P < MB / 2; P++) {
    if (P == 0)
      put(std::integral_constant<int, 0>{});
    else if (P == 1)
      put(std::integral_constant<int, 1>{});
    else if (P == 2)
      put(std::integral_constant<int, (MB > 4 ? 2 : 0)>{});
    else
      put(std::integral_constant<int, (MB > 4 ? 3 : 0)>{});
#pragma unroll 2
    for (int r = 0; r < 32; r += RPI) {
      const int row = wm * (TM / 2) + 32 * P + r + lane / LPR;
      const int64_t m = m0 + row;
      if (m >= g.M) continue;
      const float* p = from + r * LROW;
      float v[8], u[8];
      get(p, v);
      if constexpr (GATED) get(p + 8 * MB, u);
      if constexpr (PART) {
        const int64_t pr = part_row<EPI>(g);
        float* o = g.parts + (int64_t(blockIdx.y) * g.M + m) * pr + n;
        if (n < pad64(g.N)) {
          *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
          if constexpr (GATED) {
            *reinterpret_cast<f32x4*>(o + pr / 2) = f32x4{u[0], u[1], u[2], u[3]};
            *reinterpret_cast<f32x4*>(o + pr / 2 + 4) = f32x4{u[4], u[5], u[6], u[7]};
          }
        }
      } else {
        finish<EPI>(g, es, rows_e[row], m, n, v, u, bias);
      }
    }
  }
}

// the parts' sums, in order, and what becomes of them: 8 columns a thread
template <int EPI>
__global__ __launch_bounds__(256) void k_join(const HGemm g, int parts) {
  const int64_t cols = pad64(g.N) / 8, i = int64_t(blockIdx.x) * 256 + threadIdx.x, m = i / cols, n = 8 * (i % cols);
  if (m >= g.M) return;
  const int64_t pr = part_row<EPI>(g);
  const float* p = g.parts + m * pr + n;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, u[8] = {0, 0, 0, 0, 0, 0, 0, 0}, bias[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 8
  for (int k = 0; k < parts; k++, p += g.M * pr)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + 4 * h);
#pragma unroll
      for (int c = 0; c < 4; c++) v[4 * h + c] += a[c];
      if constexpr (gated<EPI>) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(p + pr / 2 + 4 * h);
#pragma unroll
        for (int c = 0; c < 4; c++) u[4 * h + c] += b[c];
      }
    }
  if (EPI == H_STORE && g.bias)
    for (int k = 0; k < 8; k++)
      if (n + k < g.N) bias[k] = g.bias[n + k];
  finish<EPI>(g, g.e + (g.e0 ? *g.e0 : 0) + (g.e1 ? *g.e1 : 0), row_exp<EPI>(g, m), m, n, v, u, bias);
}

// How a product is cut: `gn` columns of tiles, big (256 x 256) or small (128 x 128), K in `parts`; columns past them are cut
// anew. The choice goes by what a product takes as measured on the card (us; a step is 32 values of K):
//   a round of 256 big tiles: 0.76 a step and 18 for its start and its outputs;
//   a round of 512 small ones, two a CU: 0.53 a step and 10; with one a CU 0.31 a step;
//   parts: the sums written and read again at 4 TB/s, and 5 for the launch that joins them.
// (3001 x 4096 of 11008 values, 192 big tiles: 283 us, 366 in small ones; 2048 x 2048 of 16384, 64 big tiles: 4 parts 130 us,
// 256 small ones in 2 parts 170; 1000 x 6144 of 2048: 96 big 66 us, 384 small 39.)
struct Cut {
  bool big;
  int64_t gn;
  int parts;
  double us;
};
constexpr int CUS = 256;
double round_us(int64_t tiles, bool big, double steps) {
  if (big) return double((tiles + CUS - 1) / CUS) * (0.76 * steps + 18);
  const int64_t left = tiles % (2 * CUS);
  return double(tiles / (2 * CUS)) * (0.53 * steps + 10) + (left ? (left > CUS ? 0.53 : 0.31) * steps + 10 : 0);
}
Cut best_cut(int64_t M, int64_t cols, int64_t K, int segs, bool mixed) {
  const int64_t pairs = K / (2 * BK) * segs;
  Cut best{false, 0, 0, 1e30};
  const auto size = [](int64_t v, bool big) { return (v + (big ? 255 : 127)) / (big ? 256 : 128); };
  for (int big = 0; big < 2; big++)
    for (int parts = 1; parts <= (big ? 4 : 16); parts *= 2) {
      if (parts > 1 && pairs / parts < 4) break;
      const int64_t gn = size(cols, big);
      double us = round_us(size(M, big) * gn * parts, big, 2.0 * double(pairs) / parts);
      if (parts > 1) us += 5 + 2.0 * 4 * parts * double(M) * double(cols) / 4e6;
      if (us < best.us) best = Cut{big != 0, gn, parts, us};
    }
  const int64_t gm = size(M, true), tiles = gm * size(cols, true), keep = tiles / CUS * CUS / gm;
  if (mixed && tiles > CUS && keep >= 1 && keep < size(cols, true)) {  // (whole rounds big, the columns left as is best for them)
    const double us = round_us(gm * keep, true, 2.0 * double(pairs)) + 2 + best_cut(M, cols - 256 * keep, K, segs, false).us;
    if (us < best.us) best = Cut{true, keep, 1, us};
  }
  return best;
}

template <int MB, int EPI, bool PART>
int launch_t(const HGemm& g, int64_t gn, int parts, hipStream_t s) {
  using T = HT<MB>;
  static DeviceOnce set;
  if (!set.lds(reinterpret_cast<const void*>(k_hgemm<MB, EPI, PART>), T::LDS))
    return fail(ARTLITE_EHIP, "large tiles: kernel set-up failed");
  const int64_t gm = (g.M + T::TM - 1) / T::TM;
  if (gm * gn > (int64_t(1) << 30)) return fail(ARTLITE_EINVAL, "large tiles: %lld tiles", (long long)(gm * gn));
  k_hgemm<MB, EPI, PART><<<dim3(unsigned(gm * gn), unsigned(parts)), 256, T::LDS, s>>>(g, int(gm), int(gn));
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

template <int EPI>
int join(const HGemm& g, int parts, hipStream_t s) {
  const int64_t threads = g.M * (pad64(g.N) / 8);
  k_join<EPI><<<unsigned((threads + 255) / 256), 256, 0, s>>>(g, parts);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

template <int EPI>
int launch_e(HGemm g, bool mixed, hipStream_t s) {
  const int64_t cols = gated<EPI> ? 2 * g.N : g.N;
  const Cut c = best_cut(g.M, cols, g.K, g.segs, mixed);
  if (c.parts > 1) {
    if (!g.parts) return fail(ARTLITE_EINVAL, "large tiles: no scratch for parts");
    if (c.big)
      ART_TRY((launch_t<8, EPI, true>(g, c.gn, c.parts, s)));
    else
      ART_TRY((launch_t<4, EPI, true>(g, c.gn, c.parts, s)));
    return join<EPI>(g, c.parts, s);
  }
  if (c.big)
    ART_TRY((launch_t<8, EPI, false>(g, c.gn, 1, s)));
  else
    ART_TRY((launch_t<4, EPI, false>(g, c.gn, 1, s)));
  const int64_t done = c.gn * (c.big ? 256 : 128);
  if (done >= cols) return ARTLITE_OK;
  // the columns left, as a product of their own
  const int64_t n = gated<EPI> ? done / 2 : done;
  for (int i = 0; i < g.segs; i++) {
    g.b[i] += n * g.ldb;
    if (gated<EPI>) g.b2[i] += n * g.ldb;
  }
  g.N -= n;
  if (EPI == H_STORE) {
    if (g.bias) g.bias += n;
    g.y = static_cast<char*>(g.y) + n * (g.dtype == ARTLITE_X_BF16 ? 2 : 4);
  } else {
    g.h_cols -= n;
    for (uint16_t** p : {&g.h, &g.dg, &g.du})
      if (*p) *p += n;
    if (g.dh) g.dh += n;
  }
  return launch_e<EPI>(g, false, s);
}

}  // namespace

size_t hgemm_parts_bytes(int64_t M, int64_t N, int64_t K, int segs, bool gate) {
  size_t most = 0;
  for (int64_t cols = gate ? 2 * N : N, mixed = 1; cols > 0; mixed = 0) {
    const Cut c = best_cut(M, cols, K, segs, mixed);
    const int64_t n = gate ? (cols + 1) / 2 : cols;
    if (c.parts > 1) most = size_t(c.parts) * M * (gate ? 2 : 1) * pad64(n) * 4;
    cols -= c.gn * (c.big ? 256 : 128);
  }
  return most;
}

int launch_hgemm(const HGemm& g, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return ARTLITE_OK;
  if (g.segs < 1 || g.segs > H_SEGS || g.K < 64 || g.K % 64 || g.lda < g.K || g.ldb < g.K || g.lda % 8 || g.ldb % 8 ||
      g.lda > (int64_t(1) << 22) || g.ldb > (int64_t(1) << 22) || g.K * g.segs / BK >= (int64_t(1) << 30))
    return fail(ARTLITE_EINVAL, "large tiles: K %lld of rows of %lld and %lld", (long long)g.K, (long long)g.lda,
                (long long)g.ldb);
  HGemm h = g;
  h.h_cols = g.h_stride;
  return g.epilogue == H_STORE  ? launch_e<H_STORE>(h, true, s)
         : g.epilogue == H_ROWS ? launch_e<H_ROWS>(h, true, s)
         : g.epilogue == H_GLU  ? launch_e<H_GLU>(h, true, s)
                                : launch_e<H_DGLU>(h, true, s);
}

int launch_join(const HGemm& g, int parts, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return ARTLITE_OK;
  HGemm h = g;
  h.h_cols = g.h_stride;
  return g.epilogue == H_STORE  ? join<H_STORE>(h, parts, s)
         : g.epilogue == H_ROWS ? join<H_ROWS>(h, parts, s)
         : g.epilogue == H_GLU  ? join<H_GLU>(h, parts, s)
                                : join<H_DGLU>(h, parts, s);
}

}  // namespace artlite
