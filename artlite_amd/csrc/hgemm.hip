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
               : "memory", "m0");
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
__device__ __forceinline__ void finish16(const HGemm& g, const RowExp& r, int64_t m, int64_t n, float (&v)[8], float (&u)[8]) {
  const int64_t at = m * g.h_stride + n;
  const int ev = g.e + r.sum, eu = g.e2 + r.sum;
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
      // (act(g) and u over 2^ga, which is above both: no factor passes fp32's range, however small or large the row)
      const int ga = r.out - r.dh;
      float a, da;
      gate_act_grad<TWO>(g.act, __builtin_amdgcn_ldexpf(v[k], ev), a, da);
      a = __builtin_amdgcn_ldexpf(a, -ga);
      h[k] = a * __builtin_amdgcn_ldexpf(u[k], eu + ga - r.h);
      v[k] = d[k] * __builtin_amdgcn_ldexpf(u[k], eu - ga) * da;
      u[k] = d[k] * a;
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
__device__ __forceinline__ void finish(const HGemm& g, const RowExp& r, int64_t m, int64_t n, float (&v)[8],
                                       float (&u)[8], const float (&bias)[8]) {
  if constexpr (EPI == H_STORE) {
    const int there = int(max(int64_t(0), min(int64_t(8), g.N - n)));  // (columns that there are)
    if (there == 0) return;
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = __builtin_amdgcn_ldexpf(v[k], g.e + r.sum);
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
      finish16<EPI, true>(g, r, m, n, v, u);
    else
      finish16<EPI, false>(g, r, m, n, v, u);
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

// the tile of a workgroup: those of an XCD (every eighth) take a run of tiles, in columns of 4 tile rows
__device__ __forceinline__ void deal_tile(int gm, int gn, int& mt, int& nt) {
  const int total = gm * gn, per = total / 8, rest = total % 8;
  const int x = int(blockIdx.x) & 7, i = int(blockIdx.x) >> 3;
  const int t = x * per + (x < rest ? x : rest) + i;
  constexpr int GR = 4;
  const int band = t / (GR * gn), in = t % (GR * gn), rows = min(GR, gm - band * GR);
  mt = __builtin_amdgcn_readfirstlane(band * GR + in % rows);
  nt = __builtin_amdgcn_readfirstlane(in / rows);
}

// gm x gn tiles from column 0 on; K in gridDim.y parts (PART: their sums into g.parts, for k_join)
template <int MB, int EPI, bool PART>
__device__ __forceinline__ void hgemm_tile(const HGemm& g, int gm, int gn) {
  using T = HT<MB>;
  constexpr int TM = T::TM, RING = T::RING;
  constexpr bool GATED = gated<EPI>;
  constexpr int TN = GATED ? TM / 2 : TM;  // output columns of a tile
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
  const int wm = wv >> 1, wn = wv & 1;

  int mt, nt;
  deal_tile(gm, gn, mt, nt);
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
        finish<EPI>(g, rows_e[row], m, n, v, u, bias);
      }
    }
  }
}

template <int MB, int EPI, bool PART>
__global__ __launch_bounds__(256, MB == 8 ? 1 : 2) void k_hgemm(const HGemm g, int gm, int gn) {
  hgemm_tile<MB, EPI, PART>(g, gm, gn);
}
// up to three products of as many small tiles each
struct HGemms {
  HGemm g[3];
  int gm[3], gn[3];
};
__global__ __launch_bounds__(256, 2) void k_hgemms(const HGemms all) {
  const int i = blockIdx.z;
  hgemm_tile<4, H_STORE, false>(all.g[i], all.gm[i], all.gn[i]);
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
  finish<EPI>(g, row_exp<EPI>(g, m), m, n, v, u, bias);
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


// ---- the same product with W in its blocks, for hundreds of rows: y = x W^T, x as fp16 rows, W's values made of the codes in
// registers, as the MFMA's operands
//
// A workgroup of 4 waves takes 128 rows of x and 256 of W, a wave 64 of W's and all of x's. x goes through an LDS ring as
// above; a wave's codes (and headers) go through its own part of LDS by the same DMAs, whose counts then stay one queue, and
// are values when they are operands: code to fp16 (exact), times its group's scale less its offset in fp16 (both rounded to
// fp16 from fp32 products: a value is off by 2^-11 of its product and of its offset, at most 8 times its group's largest value
// where `direct` says so, 3 times it where the codes span their range; the large tiles' are by 2^-11 of themselves). That
// saves the unpacked matrix's way through memory and most of an operand's traffic from L2, which bounds the small tiles; one
// wave a SIMD does the values' instructions (15 to 28 for 8 of them) between the MFMAs of the step before. A step (32 values
// of K) takes 0.55 us with one workgroup a CU and 0.95 with two, which is neither the ring's depth (8 slots: the same), the
// barriers (every second step: the same) nor the operands' latency (read 5 blocks ahead: the same): 1.1 to 1.3 PFLOP/s where
// the large tiles have 1.4. 1000 rows of 4096 x 4096 Q4_K: 46 us and 7 to join 2 parts; of 6144 x 2048 IQ4_NL 44.
constexpr int Q_TM = 128, Q_TN = 256, Q_RING = 4, Q_SLOT = Q_TM * BK * 2;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// the fp16 values of a code dword, with its scale and offset (twice in a word each)
template <int QT>
__device__ __forceinline__ u32x4 q_values(uint32_t w, uint32_t s, uint32_t o, uint32_t mask, uint32_t top) {
  const f16x2 sc = __builtin_bit_cast(f16x2, s);
  u32x4 r;
  if constexpr (iq4<QT>) {
    r = lut_operand<3>(w);
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, uint32_t(r[i])) * sc);
  } else {
    constexpr _Float16 Z = QT == ARTLITE_Q4_0 ? _Float16(-1032.0f) : _Float16(-1024.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f16x2 c = __builtin_bit_cast(f16x2, ((w >> (4 * i)) & mask) | top) + f16x2{Z, Z};  // (1024 + c)
      f16x2 v;
      if constexpr (has_offset<QT>)
        v = __builtin_elementwise_fma(c, sc, __builtin_bit_cast(f16x2, o));
      else
        v = c * sc;
      r[i] = __builtin_bit_cast(uint32_t, v);
    }
  }
  return r;
}

// gated: a wave's 64 rows are 32 of W and the same 32 of the second matrix
template <int QT, int EPI, bool PART>
__global__ __launch_bounds__(256, 1) void k_qgemm(const HGemm g, const uint8_t* __restrict__ w, const uint8_t* __restrict__ w2,
                                                  int64_t tiles, int units, int gm, int gn) {
  constexpr bool GATED = gated<EPI>;
  constexpr int TN = GATED ? Q_TN / 2 : Q_TN, WT = TN / 4 / TROWS;  // (output columns; a wave's tiles of a matrix)
  constexpr int UB = unit_bytes<QT>(), HB = hdr_bytes<QT>(), HD = GATED || HB == 32 ? 2 : 1;  // (header DMAs a unit)
  constexpr int CODES = Q_RING * Q_SLOT, HDRS = CODES + 4 * 8192, LDS = HDRS + 4 * 2048;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
  int mt, nt;
  deal_tile(gm, gn, mt, nt);
  const int64_t m0 = int64_t(mt) * Q_TM, n0 = int64_t(nt) * TN;
  const int mv = int(min(int64_t(Q_TM), g.M - m0));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(hg_lds_addr(lds));
  uint32_t mask = 0x000F000Fu, top = 0x64006400u;
  asm("" : "+s"(mask), "+v"(top));

  uint32_t offa[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = 16 * (2 * wv + i) + (lane >> 2), c = (lane & 3) ^ ((r >> 1) & 3);
    offa[i] = uint32_t(min(r, mv - 1)) * uint32_t(g.lda) * 2 + 16 * c;
  }
  // (tiles past the last: the last again, their columns are not stored)
  const int64_t tw = n0 / TROWS + WT * wv, t0 = min(tw, tiles - 1);
  uint32_t tile_at[4], offh[HD];
#pragma unroll
  for (int j = 0; j < 4; j++)
    tile_at[j] = __builtin_amdgcn_readfirstlane(uint32_t(min(tw + j % WT, tiles - 1) - t0) * uint32_t(units) * UB);
  {
    constexpr int LT = TROWS * HB / 16;  // lanes of a tile's headers
#pragma unroll
    for (int d = 0; d < HD; d++) {
      const int j = GATED ? (lane / LT) & 1 : (lane / LT + d * (64 / LT)) & 3;  // (gated: a DMA a matrix)
      offh[d] = uint32_t(min(tw + j, tiles - 1) - t0) * uint32_t(units) * UB + 16 * (lane % LT);
    }
  }
  const uint8_t* const wbase = w + t0 * units * UB;
  const uint8_t* const wbase2 = GATED ? w2 + t0 * units * UB : nullptr;
  const int steps_all = int(g.K / BK);
  const int u0 = PART ? int(int64_t(units) * blockIdx.y / gridDim.y) : 0;
  const int u1 = PART ? int(int64_t(units) * (blockIdx.y + 1) / gridDim.y) : units;
  const int steps = min(8 * u1, steps_all);  // (of K)
  const uint16_t* const abase = g.a[0] + m0 * g.lda;
  auto dma_a = [&](int i, int t) __attribute__((always_inline)) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(lds0 + (t & (Q_RING - 1)) * Q_SLOT + (2 * wv + i) * 1024);
    hg_dma(hg_uniform(abase + int64_t(min(t, steps - 1)) * BK), offa[i], d);
  };
  auto dma_code = [&](int j, int h, int u) __attribute__((always_inline)) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(lds0 + CODES + wv * 8192 + (h * 4 + j) * 1024);
    const uint8_t* p = (j < WT ? wbase : wbase2) + int64_t(min(u, u1 - 1)) * UB + tile_at[j] + 1024 * h;
    hg_dma(hg_uniform(reinterpret_cast<const uint16_t*>(p)), 16 * lane, d);
  };
  auto dma_hdr = [&](int d, int u) __attribute__((always_inline)) {
    const uint8_t* p = (GATED && d ? wbase2 : wbase) + int64_t(min(u, u1 - 1)) * UB + 2048;
    hg_dma(hg_uniform(reinterpret_cast<const uint16_t*>(p)), offh[d],
           __builtin_amdgcn_readfirstlane(lds0 + HDRS + wv * 2048 + d * 1024));
  };

  f32x4 acc[8][4];
  hg_for<8>([&](auto i) {
    hg_for<4>([&](auto j) { acc[i][j] = f32x4{0, 0, 0, 0}; });
  });
  const uint32_t lo = lr * 64 + ((lg ^ ((lr >> 1) & 3)) << 4);
  auto ld = [](const uint8_t* p) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4*>(p); };
  u32x4 fa[4], fb[2][4], code[4], code2[4];
  uint32_t sc[4][4], of[4][4], sc2[4][4], of2[4][4];
  TileHdr<QT> hd[4];
  const uint8_t* const mycodes = lds + CODES + wv * 8192 + 16 * lane;
  const uint8_t* const myhdrs = lds + HDRS + wv * 2048 + HB * lr;
  auto read_hdrs = [&]() __attribute__((always_inline)) {
    hg_for<4>([&](auto j) { hd[j].load(myhdrs + (GATED ? (j / 2) * 1024 + (j % 2) * TROWS * HB : j * TROWS * HB)); });
  };
  auto read_codes = [&](int h) __attribute__((always_inline)) {
    hg_for<4>([&](auto j) { code2[j] = ld(mycodes + (4 * h + decltype(j)::value) * 1024); });
  };
  // a tile's scales of half H
  auto scales = [&](auto jc, auto hc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value, H = decltype(hc)::value;
    float s[4], o[4] = {0, 0, 0, 0};
    hd[j].template fields<H>(s, o);
    const int e = j < WT ? g.e : g.e2;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const _Float16 a = _Float16(__builtin_amdgcn_ldexpf(s[k], -e)), b = _Float16(-__builtin_amdgcn_ldexpf(o[k], -e));
      sc2[j][k] = __builtin_bit_cast(uint32_t, f16x2{a, a});
      if constexpr (has_offset<QT>) of2[j][k] = __builtin_bit_cast(uint32_t, f16x2{b, b});
    }
  };
  auto next_half = [&]() __attribute__((always_inline)) {
    hg_for<4>([&](auto jc) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      code[j] = code2[j];
      hg_for<4>([&](auto k) { sc[j][k] = sc2[j][k], of[j][k] = has_offset<QT> ? of2[j][k] : 0; });
    });
  };
  // operand j of the group gi of the half at hand
  auto values = [&](auto jc, auto gc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value, gi = decltype(gc)::value;
    return q_values<QT>(code[j][gi], sc[j][gi], of[j][gi], mask, top);
  };

  const int s0 = 8 * u0;
  for (int d = 0; d < HD; d++) dma_hdr(d, u0);
  for (int j = 0; j < 4; j++) dma_code(j, 0, u0);
  for (int t = 0; t < 2; t++)
    for (int i = 0; i < 2; i++) dma_a(i, s0 + t);
  for (int j = 0; j < 4; j++) dma_code(j, 1, u0);
  for (int i = 0; i < 2; i++) dma_a(i, s0 + 2);
  hg_wait<6>();
  hg_barrier();
  read_hdrs();
  read_codes(0);
  hg_for<4>([&](auto j) { scales(j, std::integral_constant<int, 0>{}); });
  next_half();
  hg_for<4>([&](auto j) { fb[0][j] = values(j, std::integral_constant<int, 0>{}); });
  fa[0] = ld(lds + lo);
  fa[1] = ld(lds + lo + 1024);

  // Step t = 8 u + J on ring slot t % 4: its operands of W are there; the next step's are made meanwhile. Loads issued in it:
  // a tile's codes of the same half of unit u + 1, at J = 0 its headers, x of step t + 3. At its barrier all that was issued
  // up to step t - 2 has landed: x of step t + 1, the other half's codes (read into registers at J = 2 and 6, a step before
  // their first use), the next unit's headers.
  auto step = [&](auto jc, int u) __attribute__((always_inline)) {
    constexpr int J = decltype(jc)::value, S = J & 1;
    const int t = 8 * u + J;
    hg_wait<(J == 1 ? 3 + HD : 3)>();
    hg_barrier();
    const uint8_t *sa = lds + (t & 3) * Q_SLOT + lo, *na = lds + ((t + 1) & 3) * Q_SLOT + lo;
    if constexpr (J == 6) read_hdrs();
    if constexpr (J == 2) read_codes(1);
    if constexpr (J == 6) read_codes(0);
    hg_for<8>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      fa[(i + 2) % 4] = i + 2 < 8 ? ld(sa + 1024 * (i + 2)) : ld(na + 1024 * (i + 2 - 8));
      if constexpr (i == 0) dma_code(J & 3, J >> 2, u + 1);
      if constexpr (i == 1 && J == 0)
        for (int d = 0; d < HD; d++) dma_hdr(d, u + 1);
      if constexpr (i == 2 || i == 3) dma_a(i - 2, t + 3);
      if constexpr (i % 2 == 1 && J % 4 == 2) scales(std::integral_constant<int, i / 2>{}, std::integral_constant<int, J == 2>{});
      if constexpr (i == 0 && J % 4 == 3) next_half();
      if constexpr (i % 2 == 0)
        fb[1 - S][i / 2] = values(std::integral_constant<int, i / 2>{}, std::integral_constant<int, (J + 1) % 4>{});
      hg_for<4>([&](auto j) __attribute__((always_inline)) { acc[i][j] = hg_mfma(fb[S][j], fa[i % 4], acc[i][j]); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  for (int u = u0; u < u1; u++)
    hg_for<4>([&](auto pc) __attribute__((always_inline)) {
      constexpr int P = decltype(pc)::value;
      if (P == 0 || 8 * u + 2 * P < steps) {  // (K is a multiple of 64)
        step(std::integral_constant<int, 2 * P>{}, u);
        step(std::integral_constant<int, 2 * P + 1>{}, u);
      }
    });
  hg_wait<0>();
  hg_barrier();

  // ---- outputs, as above
  RowExp* const rows_e = reinterpret_cast<RowExp*>(lds + LDS - Q_TM * sizeof(RowExp));
  if constexpr (!PART) {
    for (int r = threadIdx.x; r < Q_TM; r += 256) rows_e[r] = row_exp<EPI>(g, m0 + min(r, mv - 1));
    __syncthreads();
  }
  constexpr int LROW = 64 + 4, LPR = TN / 4 / 8, RPI = 64 / LPR;  // (lanes a row, rows an iteration)
  float* const buf = reinterpret_cast<float*>(lds) + wv * 32 * LROW;
  static_assert(4 * 32 * LROW * 4 + Q_TM * sizeof(RowExp) <= LDS, "LDS");
  const int64_t n = n0 + TN / 4 * wv + 8 * (lane % LPR);
  const float* const from = buf + (lane / LPR) * LROW + 8 * (lane % LPR);
  float bias[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (EPI == H_STORE && !PART && g.bias)
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (n + k < g.N) bias[k] = g.bias[n + k];
  hg_for<4>([&](auto pc) __attribute__((always_inline)) {
    constexpr int P = decltype(pc)::value;
    hg_for<2>([&](auto i) __attribute__((always_inline)) {
      hg_for<4>([&](auto j) __attribute__((always_inline)) {
        *reinterpret_cast<f32x4*>(buf + (16 * i + lr) * LROW + 16 * j + 4 * lg) = acc[2 * P + decltype(i)::value][j];
      });
    });
#pragma unroll 1
    for (int r = 0; r < 32; r += RPI) {
      const int row = 32 * P + r + lane / LPR;
      const int64_t m = m0 + row;
      if (m >= g.M) continue;
      f32x4 a[GATED ? 4 : 2];
#pragma unroll
      for (int k = 0; k < (GATED ? 4 : 2); k++)
        a[k] = *reinterpret_cast<const f32x4*>(from + r * LROW + (k / 2) * 32 + (k % 2) * 4);
      if constexpr (PART) {
        const int64_t pr = part_row<EPI>(g);
        float* o = g.parts + (int64_t(blockIdx.y) * g.M + m) * pr + n;
        if (n < pad64(g.N)) {
#pragma unroll
          for (int k = 0; k < (GATED ? 4 : 2); k++) *reinterpret_cast<f32x4*>(o + (k / 2) * (pr / 2) + (k % 2) * 4) = a[k];
        }
      } else {
        float v[8] = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]}, u[8];
        if constexpr (GATED)
#pragma unroll
          for (int k = 0; k < 4; k++) u[k] = a[2][k], u[4 + k] = a[3][k];
        finish<EPI>(g, rows_e[row], m, n, v, u, bias);
      }
    }
  });
}

int64_t q_groups(int64_t M, const artlite_matrix* w, bool gate) {
  const int tn = gate ? Q_TN / 2 : Q_TN;
  return (M + Q_TM - 1) / Q_TM * ((w->N + tn - 1) / tn);
}
template <int QT, int EPI>
int launch_q(const HGemm& g, const artlite_matrix* w, const artlite_matrix* w2, int parts, hipStream_t s) {
  constexpr int LDS = Q_RING * Q_SLOT + 4 * 8192 + 4 * 2048;
  const int64_t gm = (g.M + Q_TM - 1) / Q_TM, gn = q_groups(g.M, w, gated<EPI>) / gm;
  static DeviceOnce set, set_part;
  if (!set.lds(reinterpret_cast<const void*>(k_qgemm<QT, EPI, false>), LDS) ||
      !set_part.lds(reinterpret_cast<const void*>(k_qgemm<QT, EPI, true>), LDS))
    return fail(ARTLITE_EHIP, "dense tiles: kernel set-up failed");
  const dim3 grid(unsigned(gm * gn), unsigned(parts));
  const uint8_t *a = w->w.as<uint8_t>(), *b = w2 ? w2->w.as<uint8_t>() : nullptr;
  if (parts == 1) {
    k_qgemm<QT, EPI, false><<<grid, 256, LDS, s>>>(g, a, b, w->tiles, w->units, int(gm), int(gn));
    ART_HIP(hipGetLastError());
    return ARTLITE_OK;
  }
  k_qgemm<QT, EPI, true><<<grid, 256, LDS, s>>>(g, a, b, w->tiles, w->units, int(gm), int(gn));
  ART_HIP(hipGetLastError());
  return join<EPI>(g, parts, s);
}
template <int QT>
int launch_q_e(const HGemm& g, const artlite_matrix* w, const artlite_matrix* w2, int parts, hipStream_t s) {
  return g.epilogue == H_STORE ? launch_q<QT, H_STORE>(g, w, w2, parts, s)
         : g.epilogue == H_GLU ? launch_q<QT, H_GLU>(g, w, w2, parts, s)
                               : launch_q<QT, H_DGLU>(g, w, w2, parts, s);
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

namespace {
int check_hgemm(const HGemm& g) {
  if (g.segs < 1 || g.segs > H_SEGS || g.K < 64 || g.K % 64 || g.lda < g.K || g.ldb < g.K || g.lda % 8 || g.ldb % 8 ||
      g.lda > (int64_t(1) << 22) || g.ldb > (int64_t(1) << 22) || g.K * g.segs / BK >= (int64_t(1) << 30))
    return fail(ARTLITE_EINVAL, "large tiles: K %lld of rows of %lld and %lld", (long long)g.K, (long long)g.lda,
                (long long)g.ldb);
  return ARTLITE_OK;
}
}  // namespace

int launch_hgemm(const HGemm& g, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return ARTLITE_OK;
  ART_TRY(check_hgemm(g));
  HGemm h = g;
  h.h_cols = g.h_stride;
  return g.epilogue == H_STORE  ? launch_e<H_STORE>(h, true, s)
         : g.epilogue == H_ROWS ? launch_e<H_ROWS>(h, true, s)
         : g.epilogue == H_GLU  ? launch_e<H_GLU>(h, true, s)
                                : launch_e<H_DGLU>(h, true, s);
}

int launch_hgemms(const HGemm* g, int count, hipStream_t s) {
  using T = HT<4>;
  HGemms all{};
  int64_t tiles = 0;
  if (count > 3) return fail(ARTLITE_EINVAL, "large tiles: %d products", count);
  for (int i = 0; i < count; i++) {
    ART_TRY(check_hgemm(g[i]));
    const int64_t gm = (g[i].M + T::TM - 1) / T::TM, gn = (g[i].N + T::TM - 1) / T::TM;
    if (g[i].epilogue != H_STORE || gm < 1 || gn < 1 || gm * gn > (int64_t(1) << 30) || (i && gm * gn != tiles))
      return fail(ARTLITE_EINVAL, "large tiles: products that are not alike");
    all.g[i] = g[i], all.gm[i] = int(gm), all.gn[i] = int(gn);
    tiles = gm * gn;
  }
  static DeviceOnce set;
  if (!set.lds(reinterpret_cast<const void*>(k_hgemms), T::LDS)) return fail(ARTLITE_EHIP, "large tiles: kernel set-up failed");
  if (count) k_hgemms<<<dim3(unsigned(tiles), 1, unsigned(count)), 256, T::LDS, s>>>(all);
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
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

// Where it is the faster way (against unpacking W and the tiles above): for what is one workgroup a CU at most (4096 x 4096 Q4_K,
// 257 rows 36 us against 42, 2048 rows, 256 workgroups, 80 against 95, 3000 rows, 384, 125 against 115; 4096 x 12288 Q4_0, 512
// rows 75 against 105, 2048 rows 198 against 225; 12288 x 4096 IQ4_XS, 512 rows 88 against 101, 700 rows, 288, 137 against
// 118), and where the unpacking is most of the work (32768 x 2048 Q4_K, 512 rows, 512 workgroups, 77 against 98). A gated pair,
// two matrices to unpack, to four a CU (a block's forward, 4096 x 11008 Q4_0: 1000 rows, 688 workgroups, 266 against 326, 1300
// rows, 946, 359 against 445; 2048 x 8192 Q4_K, 2048 rows, 1024, 213 against 231; 3584 x 9472 IQ4_XS, 1000 rows, 592, 282
// against 278).
bool qgemm_fits(int64_t M, const artlite_matrix* w, bool gate) {
  return int64_t(4) * w->units * w->ub < (int64_t(1) << 32) && (M <= 512 || q_groups(M, w, gate) <= (gate ? 4 : 1) * CUS);
}
// the parts of K: as long as they fill CUs and a part has two units
int qgemm_parts(int64_t M, const artlite_matrix* w, bool gate) {
  const int64_t wgs = q_groups(M, w, gate);
  int parts = 1;
  while (wgs * parts * 2 <= CUS && w->units / (2 * parts) >= 2) parts *= 2;
  return parts;
}
size_t qgemm_parts_bytes(int64_t M, const artlite_matrix* w, bool gate) {
  const int parts = qgemm_parts(M, w, gate);
  return parts > 1 ? size_t(parts) * M * (gate ? 2 : 1) * pad64(w->N) * 4 : 0;
}

int launch_qgemm(HGemm g, const artlite_matrix* w, const artlite_matrix* w2, hipStream_t s) {
  if (g.M <= 0) return ARTLITE_OK;
  const bool gate = g.epilogue != H_STORE;
  const int parts = qgemm_parts(g.M, w, gate);
  g.h_cols = g.h_stride;
  if (g.K != pad64(w->K) || g.lda < g.K || g.lda % 8 || g.lda > (int64_t(1) << 22) || g.N != w->N || g.segs != 1 ||
      !w->direct || !qgemm_fits(g.M, w, gate) || g.epilogue == H_ROWS || (gate && g.planes != 1) || gate != (w2 != nullptr) ||
      (w2 && (!w2->direct || w2->t != w->t || w2->N != w->N || w2->K != w->K)) || (parts > 1 && !g.parts))
    return fail(ARTLITE_EINVAL, "dense tiles: K %lld of rows of %lld", (long long)g.K, (long long)g.lda);
#define ART_Q(QT) return launch_q_e<QT>(g, w, w2, parts, s)
  ART_TILE_QTYPES(w->t->id, ART_Q)
#undef ART_Q
}

}  // namespace artlite
