// The large tiles: out = A B^T over fp16 rows with fp32 sums, on the MFMA (16x16x32), with the epilogues of the dense
// products (a scaled store, the gated activation, its backward).
//
// Shape. A workgroup of 4 waves takes a tile of TM x TM outputs, a wave a quarter of it ((16 MB)^2: 128 x 128 of the large
// tile, its 256 sums a lane in the accumulation registers, one wave a SIMD; 64 x 64 of the small one, two workgroups a CU).
// K streams in steps of 32 values through a ring of 4 LDS slots filled by DMA (global_load_lds by asm, so that the compiler
// does not wait for it), three steps ahead; operands go from LDS to registers a step ahead of the MFMAs that use them, so one
// barrier a step is all that a wave waits for. At its barrier a step's successor has landed (every wave has waited for its
// own loads) and the slot that is filled next has been read (a step before the last).
// Rows of a slot are 64 bytes, four 16-byte chunks, chunk c of row r at c ^ (r / 4 % 4): the 16 rows that a lane group reads
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

constexpr int BK = 32, RING = 4;

template <int MB>
struct HT {
  static constexpr int TM = 32 * MB;                 // rows and columns of a tile
  static constexpr int HALF = TM * BK * 2;           // bytes of an operand's step
  static constexpr int SLOT = 2 * HALF;
  static constexpr int LPW = SLOT / 1024 / 4;        // DMAs of a wave a step
  static constexpr int LDS = RING * SLOT;
  static_assert(LDS <= LDS_BYTES, "LDS");
};

__device__ __forceinline__ uint16_t f16_bits(float v) { return __builtin_bit_cast(uint16_t, _Float16(v)); }

// four fp16 values times 2^-e at p, and with a second plane what their rounding left
__device__ __forceinline__ void store16(uint16_t* p, int64_t plane, int planes, const float (&v)[4], int e) {
  uint16_t a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float x = ldexpf(v[i], -e);
    const _Float16 hi = _Float16(x);
    a[i] = __builtin_bit_cast(uint16_t, hi);
    b[i] = f16_bits(x - float(hi));
  }
  __builtin_memcpy(__builtin_assume_aligned(p, 8), a, 8);
  if (planes == 2) __builtin_memcpy(__builtin_assume_aligned(p + plane, 8), b, 8);
}

template <int MB, int EPI>
__global__ __launch_bounds__(256, MB == 8 ? 1 : 2) void k_hgemm(const HGemm g, int gm, int gn) {
  using T = HT<MB>;
  constexpr int TM = T::TM;
  constexpr int TN = EPI == H_STORE ? TM : TM / 2;  // output columns of a tile
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
    const int r = 16 * (HPW * wv + i) + (lane >> 2), c = (lane & 3) ^ ((r >> 2) & 3);
    const int rb = EPI == H_STORE ? r : r / (TM / 2) * (TM / 4) + r % (TM / 4);
    offa[i] = uint32_t(min(r, mv - 1)) * uint32_t(g.lda) * 2 + 16 * c;
    offb[i] = uint32_t(min(rb, nv - 1)) * uint32_t(g.ldb) * 2 + 16 * c;
  }
  const int steps_seg = int(g.K / BK), steps = steps_seg * g.segs;
  int iseg = 0, ik = 0, islot = 0;
  const uint16_t *pa, *pb;
  auto open_seg = [&]() {
    pa = g.a[iseg] + m0 * g.lda;
    pb = (EPI != H_STORE && (wv & 1) ? g.b2[iseg] : g.b[iseg]) + n0 * g.ldb;
  };
  open_seg();
  auto issue = [&]() {
    const uint32_t d = __builtin_amdgcn_readfirstlane(lds0 + islot * T::SLOT + HPW * wv * 1024);
    const uint16_t *ua = hg_uniform(pa), *ub = hg_uniform(pb);
#pragma unroll
    for (int i = 0; i < HPW; i++) {
      hg_dma(ua, offa[i], d + 1024 * i);
      hg_dma(ub, offb[i], d + T::HALF + 1024 * i);
    }
    islot = (islot + 1) % RING;
    // (past the last step its loads are made again, into slots that are not read: the counts stay)
    if (++ik < steps_seg) {
      pa += BK, pb += BK;
    } else if (iseg + 1 < g.segs) {
      ik = 0;
      iseg++;
      open_seg();
    } else {
      ik = steps_seg - 1;
    }
  };

  f32x4 acc[MB][MB];
  hg_for<MB>([&](auto i) {
    hg_for<MB>([&](auto j) { acc[i][j] = f32x4{0, 0, 0, 0}; });
  });
  const uint32_t lo = lr * 64 + ((lg ^ ((lr >> 2) & 3)) << 4);
  const uint8_t* const la = lds + wm * (TM / 2) * 64 + lo;
  const uint8_t* const lb = lds + T::HALF + wn * (TM / 2) * 64 + lo;
  // B's operands of a step, and the next step's as they are read; A's in a window of 4, read two blocks ahead
  u32x4 fa[4], fb[2][MB];
  int rslot = 0;
  auto ld = [](const uint8_t* p) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4*>(p); };
  auto step = [&](auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
    hg_wait<T::LPW>();
    hg_barrier();
    issue();
    const int nslot = (rslot + 1) % RING;
    const uint8_t *a = la + rslot * T::SLOT, *an = la + nslot * T::SLOT, *bn = lb + nslot * T::SLOT;
    rslot = nslot;
    hg_for<MB>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      fb[1 - S][i] = ld(bn + 1024 * i);
      fa[(i + 2) % 4] = i + 2 < MB ? ld(a + 1024 * (i + 2)) : ld(an + 1024 * (i + 2 - MB));
      hg_for<MB>([&](auto j) __attribute__((always_inline)) { acc[i][j] = hg_mfma(fb[S][j], fa[i % 4], acc[i][j]); });
    });
  };
  issue();
  issue();
  issue();
  hg_wait<2 * T::LPW>();
  hg_barrier();
  hg_for<MB>([&](auto j) { fb[0][j] = ld(lb + 1024 * decltype(j)::value); });
  fa[0] = ld(la);
  fa[1] = ld(la + 1024);
  for (int s = 0; s < steps; s += 2) {  // (K is a multiple of 64: an even number of steps)
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
  }
  hg_wait<0>();  // (no load may land after the workgroup's LDS is another's)

  // ---- outputs: block (i, j), lane: row m0 + wm TM / 2 + 16 i + lr, four columns from 16 j + 4 lg of the wave's
  const int es = g.e + (g.e0 ? *g.e0 : 0) + (g.e1 ? *g.e1 : 0);
  hg_for<MB>([&](auto ic) {
    constexpr int i = decltype(ic)::value;
    const int64_t m = m0 + wm * (TM / 2) + 16 * i + lr;
    if (m >= g.M) return;
    const int re = g.row_e ? g.row_e[m] : 0;
    if constexpr (EPI == H_STORE) {
      hg_for<MB>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int64_t n = n0 + wn * (TM / 2) + 16 * j + 4 * lg;
        if (n >= g.N) return;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
          v[k] = ldexpf(acc[i][j][k], es + re) + (g.bias && n + k < g.N ? g.bias[n + k] : 0.0f);
        const int64_t at = m * g.y_stride + n;
        if (g.dtype == ARTLITE_X_BF16) {
          uint16_t* y = static_cast<uint16_t*>(g.y) + at;
          if (n + 3 < g.N && (reinterpret_cast<uintptr_t>(y) & 7) == 0) {
            *reinterpret_cast<uint2*>(y) = uint2{f32_to_bf16(v[0]) | f32_to_bf16(v[1]) << 16,
                                                 f32_to_bf16(v[2]) | f32_to_bf16(v[3]) << 16};
          } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (n + k < g.N) y[k] = uint16_t(f32_to_bf16(v[k]));
          }
        } else {
          float* y = static_cast<float*>(g.y) + at;
          if (n + 3 < g.N && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
            *reinterpret_cast<float4*>(y) = float4{v[0], v[1], v[2], v[3]};
          } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (n + k < g.N) y[k] = v[k];
          }
        }
      });
    } else {
      const int oe = g.out_e[m], he = EPI == H_DGLU && g.h ? g.h_e[m] : 0;
      hg_for<MB / 2>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int64_t n = n0 + wn * (TM / 4) + 16 * j + 4 * lg;
        if (n >= g.h_stride) return;
        const int64_t at = m * g.h_stride + n;
        float h[4], dg[4], du[4];
        float4 dh = {0, 0, 0, 0};
        if constexpr (EPI == H_DGLU) dh = *reinterpret_cast<const float4*>(g.dh + at);
        const float d[4] = {dh.x, dh.y, dh.z, dh.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const bool there = n + k < g.N;
          const float gv = ldexpf(acc[i][j][k], g.e + re), uv = ldexpf(acc[i][j + MB / 2][k], g.e2 + re);
          const float a = gate_act(g.act, gv);
          h[k] = there ? a * uv : 0.0f;
          if constexpr (EPI == H_DGLU) {
            dg[k] = there ? d[k] * uv * gate_act_grad(g.act, gv) : 0.0f;
            du[k] = there ? d[k] * a : 0.0f;
          }
        }
        if constexpr (EPI == H_GLU) {
          store16(g.h + at, g.h_plane, g.planes, h, oe);
        } else {
          store16(g.dg + at, g.h_plane, g.planes, dg, oe);
          store16(g.du + at, g.h_plane, g.planes, du, oe);
          if (g.h) store16(g.h + at, g.h_plane, g.planes, h, he);
        }
      });
    }
  });
}

template <int MB, int EPI>
int launch_t(const HGemm& g, hipStream_t s) {
  using T = HT<MB>;
  constexpr int TN = EPI == H_STORE ? T::TM : T::TM / 2;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(k_hgemm<MB, EPI>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS) == hipSuccess;
  if (!ok) return fail(ARTLITE_EHIP, "large tiles: kernel set-up failed");
  const int64_t gm = (g.M + T::TM - 1) / T::TM, gn = (g.N + TN - 1) / TN;
  if (gm * gn > (int64_t(1) << 30)) return fail(ARTLITE_EINVAL, "large tiles: %lld tiles", (long long)(gm * gn));
  k_hgemm<MB, EPI><<<unsigned(gm * gn), 256, T::LDS, s>>>(g, int(gm), int(gn));
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

template <int EPI>
int launch_e(const HGemm& g, hipStream_t s) {
  const int64_t cols = EPI == H_STORE ? g.N : 2 * g.N;
  const int64_t big = ((g.M + 255) / 256) * ((cols + 255) / 256);
  return big >= 256 ? launch_t<8, EPI>(g, s) : launch_t<4, EPI>(g, s);
}

}  // namespace

int launch_hgemm(const HGemm& g, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return ARTLITE_OK;
  if (g.segs < 1 || g.segs > H_SEGS || g.K < 64 || g.K % 64 || g.lda < g.K || g.ldb < g.K || g.lda % 8 || g.ldb % 8 ||
      g.lda > (int64_t(1) << 22) || g.ldb > (int64_t(1) << 22) || g.K * g.segs / BK >= (int64_t(1) << 30))
    return fail(ARTLITE_EINVAL, "large tiles: K %lld of rows of %lld and %lld", (long long)g.K, (long long)g.lda,
                (long long)g.ldb);
  return g.epilogue == H_STORE ? launch_e<H_STORE>(g, s)
         : g.epilogue == H_GLU ? launch_e<H_GLU>(g, s)
                               : launch_e<H_DGLU>(g, s);
}

}  // namespace artlite
