// A matrix of 4-bit GGUF blocks in HBM (matrix.hip) and what the dense operators share: its tile layout and the decode of
// it, workspaces, the checks of device arguments, the launches of the dense products.
#pragma once

#include <atomic>
#include <mutex>

#include "codes.h"
#include "common.h"

// The tile layout. A matrix of N rows of K values is cut into tiles of 16 rows and units of 256 values (rows and values past
// its end are zeros: scales of 0). A unit of a tile is 2048 bytes of codes, then 16 headers of HB bytes, one a row:
//   codes: half h (128 values), lane l = 16 lg + lr: 16 bytes at 1024 h + 16 l, dword j those of row lr's values
//     32 (4 h + j) + 8 lg .. + 8, value 2 p in nibble p and value 2 p + 1 in nibble p + 4 (p < 4), so that
//     (dword >> 4 p) & 0x000F000F are the codes of values 2 p and 2 p + 1: one 16-bit operand dword of the MFMA;
//   header: Q4_0, IQ4_NL: the 8 groups' fp16 scales; Q4_1: their (scale, min) pairs; Q4_K: the block's 16 bytes before its
//     codes (d, dmin, the 6-bit scales and mins); IQ4_XS: its 8 (d and the 6-bit scales).
// The bytes are the file's (but for the padding and the scales of Q4_0's blocks of zeros), in the order in which a wave reads
// them: 1 KiB of codes a load, contiguous.
namespace artlite {

constexpr int UNIT = 256;   // values of a unit
constexpr int TROWS = 16;   // rows of a tile

template <int QT>
constexpr int hdr_bytes() {
  return QT == ARTLITE_Q4_1 ? 32 : QT == ARTLITE_IQ4_XS ? 8 : 16;
}
template <int QT>
constexpr int unit_bytes() {
  return 2048 + TROWS * hdr_bytes<QT>();
}

// whether a format has the tile layout, and its bytes a unit (0: none)
int tile_unit_bytes(int qtype);

// a switch over the formats of the tile layout
#define ART_TILE_QTYPES(qtype, X)            \
  switch (qtype) {                           \
    case ARTLITE_Q4_0: X(ARTLITE_Q4_0);      \
    case ARTLITE_Q4_1: X(ARTLITE_Q4_1);      \
    case ARTLITE_Q4_K: X(ARTLITE_Q4_K);      \
    case ARTLITE_IQ4_NL: X(ARTLITE_IQ4_NL);  \
    default: X(ARTLITE_IQ4_XS);              \
  }

// A row's header of a unit in registers, and the scale s and offset o of group g (of 8) from it: a value is s c - o with c
// the code (Q4_1, Q4_K), c - 8 (Q4_0) or IQ4[c] (o = 0), exact in fp32 but for that last product and difference.
template <int QT>
struct TileHdr {
  static constexpr int DW = hdr_bytes<QT>() / 4;
  uint32_t h[DW];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (DW == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      h[0] = v.x, h[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < DW; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
        h[i] = v.x, h[i + 1] = v.y, h[i + 2] = v.z, h[i + 3] = v.w;
      }
    }
  }
  // s and o (times om, a power of two) of groups 4 H .. + 4; K-quants' 6-bit fields four at a time, as the bytes of a word
  template <int H>
  __device__ __forceinline__ void fields(float (&s)[4], float (&o)[4], float om = 1.0f) const {
    if constexpr (QT == ARTLITE_Q4_0 || QT == ARTLITE_IQ4_NL) {
#pragma unroll
      for (int g = 0; g < 4; g++) s[g] = h2f((h[2 * H + (g >> 1)] >> (16 * (g & 1))) & 0xFFFFu);
    } else if constexpr (QT == ARTLITE_Q4_1) {
#pragma unroll
      for (int g = 0; g < 4; g++) s[g] = h2f(h[4 * H + g] & 0xFFFFu), o[g] = -om * h2f(h[4 * H + g] >> 16);
    } else if constexpr (QT == ARTLITE_Q4_K) {
      const float d = h2f(h[0] & 0xFFFFu), dm = om * h2f(h[0] >> 16);
      uint32_t sc = H == 0 ? h[1] & 0x3F3F3F3Fu : (h[3] & 0x0F0F0F0Fu) | ((h[1] >> 2) & 0x30303030u);
      uint32_t mn = H == 0 ? h[2] & 0x3F3F3F3Fu : ((h[3] >> 4) & 0x0F0F0F0Fu) | ((h[2] >> 2) & 0x30303030u);
      asm("" : "+v"(sc), "+v"(mn));  // (else a field is taken out of its word by an instruction of its own)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        s[g] = __fmul_rn(d, float((sc >> (8 * g)) & 0xFFu));
        o[g] = __fmul_rn(dm, float((mn >> (8 * g)) & 0xFFu));
      }
    } else {
      const float d = h2f(h[0] & 0xFFFFu);
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int k = 4 * H + g;
        s[g] = __fmul_rn(d, float((int((h[1] >> (4 * k)) & 15) | (int((h[0] >> (16 + 2 * k)) & 3) << 4)) - 32));
      }
    }
  }
};

template <int QT>
constexpr bool has_offset = QT == ARTLITE_Q4_1 || QT == ARTLITE_Q4_K;
template <int QT>
constexpr bool iq4 = QT == ARTLITE_IQ4_NL || QT == ARTLITE_IQ4_XS;

constexpr uint32_t bf16_of(int v) { return __builtin_bit_cast(uint32_t, float(v)) >> 16; }
constexpr uint32_t f16_of(int v) { return __builtin_bit_cast(uint16_t, _Float16(v)); }

// 16 values as byte tables of their 16-bit forms' halves
struct Lut16 {
  uint32_t lo[4], hi[4];
};
constexpr Lut16 make_lut(int kind) {  // 0: IQ4's values, 1: c - 8, 2: c (bf16), 3: IQ4's values in fp16
  constexpr int V[16] = {-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113};
  Lut16 t{};
  for (int i = 0; i < 16; i++) {
    const uint32_t b = kind == 3 ? f16_of(V[i]) : bf16_of(kind == 0 ? V[i] : kind == 1 ? i - 8 : i);
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

// a code dword's 8 values by table, as MFMA operand dwords
template <int KIND>
__device__ __forceinline__ u32x4 lut_operand(uint32_t w) {
  uint32_t l0, h0, l1, h1;  // (nibbles 0, 2, 4, 6 and 1, 3, 5, 7)
  lut_bytes<KIND>(w & 0x0F0F0F0Fu, l0, h0);
  lut_bytes<KIND>((w >> 4) & 0x0F0F0F0Fu, l1, h1);
  return u32x4{__builtin_amdgcn_perm(h0, l0, 0x06020400u), __builtin_amdgcn_perm(h1, l1, 0x06020400u),
               __builtin_amdgcn_perm(h0, l0, 0x07030501u), __builtin_amdgcn_perm(h1, l1, 0x07030501u)};
}

// the 8 values of a code dword as fp32, in order (dequantized as the file's: rows of artlite_dequant_rows)
template <int QT>
__device__ __forceinline__ void tile_values(uint32_t w, float s, float o, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const uint32_t c = (w >> (4 * p)) & 0x000F000Fu;
    float a, b;
    if constexpr (iq4<QT>) {
      const uint32_t t = iq4_int8((c | (c >> 8)) & 0x0F0Fu);
      a = float(int8_t(t & 0xFFu)), b = float(int8_t((t >> 8) & 0xFFu));
    } else {
      a = float(c & 0xFFFFu), b = float(c >> 16);
      if constexpr (QT == ARTLITE_Q4_0) a -= 8.0f, b -= 8.0f;
    }
    v[2 * p] = has_offset<QT> ? __fsub_rn(__fmul_rn(s, a), o) : __fmul_rn(s, a);
    v[2 * p + 1] = has_offset<QT> ? __fsub_rn(__fmul_rn(s, b), o) : __fmul_rn(s, b);
  }
}

// two fp32 -> two bf16, rounded to nearest even (one instruction)
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// 1 / (1 + e^-v). EXACT: to about 2 ulp, e^-v as 2^t with t = -v log2 e in two parts (the product's rounding, put back to
// first order), the hardware's 2^t and reciprocal, the latter with a step of Newton's. Else without either correction, for
// results of 11 bits: off by |v| 2^-24 and 2 ulp (a fourth of the instructions, two of them the quarter-rate ones).
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float v) {
  constexpr float L2E = 1.44269504f, L2E_LO = 1.92596303e-8f;  // (log2 e and what its rounding leaves)
  const float t = v * -L2E;
  if constexpr (!EXACT) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
  const float r = __builtin_fmaf(v, -L2E, -t) - v * L2E_LO;
  const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(r, 0.69314718f, 1.0f);
  const float d = 1.0f + e;
  float q = __builtin_amdgcn_rcpf(d);
  q = __builtin_fmaf(__builtin_fmaf(-d, q, 1.0f), q, q);
  return t > 126.0f ? 0.0f : v > 100.0f ? 1.0f : q;
}
// the gated block's activation a and its derivative da at g (artlite_act); gelu's (1 + tanh z) / 2 is sigmoid(2 z)
template <bool EXACT = true>
__device__ __forceinline__ float gate_act(int act, float g) {
  if (act == ARTLITE_ACT_SILU) return g * sigmoid<EXACT>(g);
  return g * sigmoid<EXACT>(1.5957691216f * __builtin_fmaf(0.044715f * g * g, g, g));
}
template <bool EXACT = true>
__device__ __forceinline__ void gate_act_grad(int act, float g, float& a, float& da) {
  const float c = 0.044715f * g * g;
  const float s = sigmoid<EXACT>(act == ARTLITE_ACT_SILU ? g : 1.5957691216f * __builtin_fmaf(c, g, g));
  a = g * s;
  // (0 where s is 0 or 1: nothing times a large slope stays nothing)
  const float w = s * (1.0f - s), k = act == ARTLITE_ACT_SILU ? 1.0f : 1.5957691216f * __builtin_fmaf(3.0f, c, 1.0f);
  da = w > 0.0f ? __builtin_fmaf(a * (1.0f - s), k, s) : s;
}

// the least e with |v| < 2^e of a finite v (0 and what is no number: a very small one)
__host__ __device__ __forceinline__ int exp_above(float v) {
  if (!(v > 0.0f)) return -200;
  if (v > 3.0e38f) return 129;
  int e;
  (void)frexpf(v, &e);
  return e;
}

// A workspace: device memory that calls carve their scratch from. Calls on one stream follow each other; a call on another
// stream than the last one's waits for that one's end.
struct Work {
  int device = -1;
  char* p = nullptr;
  size_t n = 0;
  std::mutex mu;
  hipEvent_t done = nullptr;
  hipStream_t last = nullptr;
  bool used = false, eager = false;
};
// Around the launches of a call that uses a workspace: `begin` locks it, checks its size and orders the call behind the last
// one; the destructor notes where the call ends. (Inside a stream capture nothing is ordered: a graph's replays and other
// calls on its workspace follow each other by the caller's streams.)
struct WorkScope {
  Work* w = nullptr;
  hipStream_t s = nullptr;
  bool note = false;
  int begin(Work* work, size_t need, hipStream_t stream, const char* what);
  ~WorkScope();
};
// bytes carved from a workspace in turn, 256-aligned; with a null base it only counts
struct Carve {
  char* base;
  size_t at = 0;
  explicit Carve(void* b) : base(static_cast<char*>(b)) {}
  template <class T>
  T* take(size_t count) {
    const size_t a = at;
    at = (a + count * sizeof(T) + 255) / 256 * 256;
    return base ? reinterpret_cast<T*>(base + a) : nullptr;
  }
};

// the device of a call's handles made current for its duration
struct OnDevice {
  int was = -1;
  int set(int device);
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};
// a kernel's dynamic LDS beyond the default, set once on each device (current when it is launched)
struct DeviceOnce {
  std::atomic<uint64_t> done{0};
  bool lds(const void* kernel, size_t bytes) {
    int d = 0;
    if (hipGetDevice(&d) != hipSuccess) return false;
    const uint64_t bit = uint64_t(1) << (d & 63);
    if (done.load(std::memory_order_acquire) & bit) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != hipSuccess) return false;
    done.fetch_or(bit, std::memory_order_release);
    return true;
  }
};
// p: device memory of `device`
int check_device(const void* p, int device, const char* what);

}  // namespace artlite

struct artlite_workspace {
  artlite::Work w;
};

struct artlite_matrix {
  int device = -1;
  const artlite::QType* t = nullptr;
  int64_t N = 0, K = 0;
  int64_t tiles = 0;
  int units = 0;
  int ub = 0;              // bytes a unit of a tile
  bool have = false, has_bias = false;
  bool direct = false;     // no group's scale and offset are many times its values (k_qgemm, hgemm.hip)
  artlite::DevBuf w, bias;
  int max_exp = 0;         // every |value| < 2^max_exp
  int row_exp = 0;         // every row's 2-norm < 2^row_exp
};

namespace artlite {

// ---- the dense products over few rows (linear.hip)

// One launch: out[m][n] = sum_k x[m][k] W[n][k] (+ bias[n]) for M rows of x given as planes of bf16 (x = the sum of its
// planes) or, where few_apart, as fp32, or with `up` set the gated products act(x W^T) (x U^T), written as planes of bf16 for
// the launch after.
struct FewArgs {
  const artlite_matrix *w, *up;
  int act;                  // (gated) artlite_act
  const void* x;            // plane p of row m at x + p x_plane + m x_stride (bf16), at any address
  int64_t x_stride, x_plane;
  int planes;               // 1, 2 or 3
  bool x32;                 // x is fp32 (3 planes as it is used)
  int64_t M;
  void* y;                  // plain: bf16 or fp32 rows, y_stride values apart
  int64_t y_stride;
  int dtype;
  uint16_t* h;              // gated: h_planes planes of M rows of h_stride values
  int64_t h_stride, h_plane;
  int h_planes;
  float* parts;             // scratch for sums in parts: few_parts_bytes of it
  // (gated) the two products' sums as they are: `raw` parts of them in parts (few_raw_parts), rows of 2 pad64(N) values, the
  // second matrix's behind the first's
  int raw;
};
int launch_few(const FewArgs& a, hipStream_t s);
// Whether a workgroup takes 16 rows of x of one tile, and blocks of 16 rows are workgroups of their own: up to 16 rows, and
// where the product is small (below).
bool few_apart(const artlite_matrix* w, int planes, bool gated, int64_t M);
int few_raw_parts(const artlite_matrix* w, int planes, int64_t M);
size_t few_parts_bytes(const artlite_matrix* w, int planes, bool gated, int64_t M);

// The transposed product, for few rows: sum over one or two (W, x) of x W -> parts of M rows of pad64(K) fp32 sums each (of
// the values times 2^-e as they are rounded to fp16: few_t_parts of them, few_t_bytes). x: `planes` (1 or 2) planes of fp16
// rows, ld a multiple of 64 and at least the matrix's rows, zeros behind them. The matrices are alike, with a
// multiple of 32 rows.
struct FewTArgs {
  const artlite_matrix* w[2];
  const uint16_t* x[2];
  int pairs;                // 1 or 2
  int64_t ld, x_plane;
  int planes, e;
  int64_t M;
  float* parts;
};
int few_t_parts(const artlite_matrix* w, int pairs, int planes, int64_t M);
size_t few_t_bytes(const artlite_matrix* w, int pairs, int planes, int64_t M);
int launch_few_t(const FewTArgs& a, hipStream_t s);
// Rows past which the dense products go by way of 16-bit operands and large tiles: one matrix's of bf16 rows (4096 x 4096 Q4_K,
// 256 rows, 27 us against 35, 257 rows 36 against the few rows' 40), of more than FEW_LARGE units where its values can be made
// from its blocks (4096 x 12288 Q4_0, 128 rows 33 against 49, 129 rows 56 against 49; 32768 x 2048 Q4_K, 128 rows 58 against
// 53, 256 rows 100 against 48; 4096 units above: 27 against 35); of fp32 rows (4096 x 4096, 128 rows, 45 against 55, 192 rows 68
// against 62). The gated block's: of bf16 rows where its matrices' values can be made so (2048 x 8192 Q4_K, 64 rows 41 against
// 53, 96 rows 57 against 55, 192 rows 81 against 65; 4096 x 11008 Q4_0, 64 rows 72 against 72, 96 rows 109 against 75), else
// (fp32, 2048 x 8192, 144, 192 and 256 rows, 143, 150 and 217 against 153, 149 and 155). And any number of rows that are
// few_apart.
constexpr int FEW_ROWS_LARGE = 128, FEW_LARGE = 8192, FEW_ROWS_FFN_DIRECT = 64;
constexpr int FEW_ROWS = 256, FEW_ROWS_F32 = 128, FEW_ROWS_FFN = 192;
// x (M rows of K fp32 values, stride apart) as three planes of bf16, M rows of K values each
int launch_planes(const float* x, int64_t M, int64_t K, int64_t stride, uint16_t* out, hipStream_t s);

// ---- 16-bit operands of the large tiles (matrix.hip)

// W (or its transpose) as fp16 rows of ld values, times 2^-e (e: `wexp16`): plane 0, with planes 2 also what its rounding
// left (at out + plane). Values past the matrix's columns (transposed: rows) up to ld are zeros.
// m2: with a second matrix of the same shape and format, into out2.
int launch_unpack(const artlite_matrix* m, const artlite_matrix* m2, bool transposed, int e, int e2, uint16_t* out,
                  uint16_t* out2, int64_t ld, int64_t plane, int planes, hipStream_t s);
// the scale of a `direct` matrix's values where their scales and offsets are fp16 too (offsets up to 8 times the values)
inline int qexp16(const artlite_matrix* m);
// the scale that brings a matrix's largest value into [2^14, 2^15)
inline int wexp16(const artlite_matrix* m) { return m->max_exp - 15; }
inline int qexp16(const artlite_matrix* m) {
  return wexp16(m) + (m->t->id == ARTLITE_Q4_1 || m->t->id == ARTLITE_Q4_K ? 3 : 0);
}

__host__ __device__ inline int64_t pad64(int64_t v) { return (v + 63) / 64 * 64; }

}  // namespace artlite
