// Matrices of 4-bit GGUF blocks in the tile layout (matrix.h): upload, the bounds that scale their 16-bit forms, those forms
// (unpacked into a workspace for the large tiles); workspaces; the C entry points of both and of device arrays.
//
// What bounds the kernels here: memory (k_unpack reads 0.56 bytes a value and writes 2). Uploads happen once a matrix and are
// not tuned.
#include "matrix.h"

#include <type_traits>

#include <cmath>
#include <initializer_list>
#include <new>

namespace artlite {

int tile_unit_bytes(int qtype) {
  switch (qtype) {
    case ARTLITE_Q4_0: return unit_bytes<ARTLITE_Q4_0>();
    case ARTLITE_Q4_1: return unit_bytes<ARTLITE_Q4_1>();
    case ARTLITE_Q4_K: return unit_bytes<ARTLITE_Q4_K>();
    case ARTLITE_IQ4_NL: return unit_bytes<ARTLITE_IQ4_NL>();
    case ARTLITE_IQ4_XS: return unit_bytes<ARTLITE_IQ4_XS>();
    default: return 0;
  }
}

namespace {

// code v (of 32) of group g of the file's block at b (a block of 32 values has one group)
template <int QT>
__device__ __forceinline__ uint32_t file_code(const uint8_t* b, int g, int v) {
  if constexpr (QT == ARTLITE_Q4_K) {
    const uint32_t c = b[16 + 32 * (g >> 1) + v];
    return g & 1 ? c >> 4 : c & 15u;
  } else {
    const uint8_t* q = b + (QT == ARTLITE_Q4_1 ? 4 : QT == ARTLITE_IQ4_XS ? 8 + 16 * g : 2);
    return v < 16 ? q[v] & 15u : uint32_t(q[v - 16]) >> 4;
  }
}

// the file's rows -> the tile layout: a workgroup per unit of a tile, thread 64 h + l the 16 code bytes of half h, lane l;
// then a header's halves-words each
template <int QT, int PER, int BYTES>
__global__ __launch_bounds__(128) void k_tile(const uint8_t* __restrict__ raw, int64_t N, int64_t K, int units,
                                              uint8_t* __restrict__ out) {
  const int64_t tile = int64_t(blockIdx.x) / units;
  const int u = int(int64_t(blockIdx.x) % units);
  uint8_t* o = out + int64_t(blockIdx.x) * unit_bytes<QT>();
  const int h = threadIdx.x >> 6, l = threadIdx.x & 63, lg = l >> 4, lr = l & 15;
  const int64_t n = tile * TROWS + lr, row_bytes = K / PER * BYTES;
  const uint8_t* row = raw + n * row_bytes;
  uint4 v;
  uint32_t* d = reinterpret_cast<uint32_t*>(&v);
  for (int j = 0; j < 4; j++) {
    const int g = 4 * h + j;
    const int64_t k = int64_t(u) * UNIT + 32 * g;
    d[j] = 0;
    if (n < N && k < K) {
      const uint8_t* b = row + k / PER * BYTES;
      for (int p = 0; p < 4; p++) {
        d[j] |= file_code<QT>(b, int(k % PER) / 32, 8 * lg + 2 * p) << (4 * p);
        d[j] |= file_code<QT>(b, int(k % PER) / 32, 8 * lg + 2 * p + 1) << (4 * p + 16);
      }
    }
  }
  *reinterpret_cast<uint4*>(o + 1024 * h + 16 * l) = v;
  constexpr int HW = hdr_bytes<QT>() / 2;  // (16-bit words of a header)
  for (int i = threadIdx.x; i < TROWS * HW; i += 128) {
    const int r = i / HW, w = i % HW;
    const int64_t nr = tile * TROWS + r;
    uint16_t x = 0;
    if (nr < N) {
      const uint8_t* rr = raw + nr * row_bytes;
      if constexpr (PER == UNIT) {
        if (int64_t(u) * UNIT < K) {
          const uint8_t* b = rr + int64_t(u) * BYTES + 2 * w;
          x = uint16_t(b[0] | b[1] << 8);
        }
      } else {
        constexpr int F = HW / 8;  // (the fp16 fields of a block)
        const int64_t k = int64_t(u) * UNIT + 32 * (w / F);
        if (k < K) {
          const uint8_t* b = rr + k / 32 * BYTES + 2 * (w % F);
          x = uint16_t(b[0] | b[1] << 8);
          if constexpr (QT == ARTLITE_Q4_0) {
            // (a block of zeros keeps no scale, which the sums' roundings would carry; one that is no number stays)
            bool zeros = (x & 0x7C00) != 0x7C00;
            for (int j = 0; j < 16; j++) zeros &= b[2 + j] == 0x88;
            if (zeros) x = 0;
          }
        }
      }
    }
    *reinterpret_cast<uint16_t*>(o + 2048 + hdr_bytes<QT>() * r + 2 * w) = x;
  }
}

// a lane's 32 values of half H of a unit: f(g, v) with values 8 lg .. + 8 of each of its groups g, or f(g, v, scale, offset)
template <int QT, int H, class F>
__device__ __forceinline__ void tile_half(const uint8_t* ub, int lane, F&& f) {
  TileHdr<QT> hd;
  hd.load(ub + 2048 + hdr_bytes<QT>() * (lane & 15));
  const uint4 c = *reinterpret_cast<const uint4*>(ub + 1024 * H + 16 * lane);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  float s[4], o[4] = {0, 0, 0, 0};
  hd.template fields<H>(s, o);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float v[8];
    tile_values<QT>(w[j], s[j], o[j], v);
    if constexpr (std::is_invocable_v<F, int, const float(&)[8]>)
      f(4 * H + j, v);
    else
      f(4 * H + j, v, s[j], o[j]);
  }
}
template <int QT, class F>
__device__ __forceinline__ void tile_unit(const uint8_t* ub, int lane, F&& f) {
  tile_half<QT, 0>(ub, lane, f);
  tile_half<QT, 1>(ub, lane, f);
}

// eight values times 2^-e as fp16, and what that rounding left
__device__ __forceinline__ void halves(const float (&v)[8], int e, uint16_t (&a)[8], uint16_t (&b)[8]) {
#pragma unroll
  for (int p = 0; p < 8; p++) {
    const float x = __builtin_amdgcn_ldexpf(v[p], -e);
    const _Float16 hi = _Float16(x);
    a[p] = __builtin_bit_cast(uint16_t, hi);
    b[p] = __builtin_bit_cast(uint16_t, _Float16(x - float(hi)));
  }
}

// out[0] = max |value|, out[1] = the largest 2-norm of a row (out[2]: whether a group's scale and offset are many times its
// values, which are then a small difference of theirs), as bits (finite values; atomic maxima of floats that are not
// negative): a workgroup of 4 waves per tile
template <int QT>
__global__ __launch_bounds__(256) void k_bounds(const uint8_t* __restrict__ w, int units, int64_t K, uint32_t* out) {
  __shared__ float red[4][TROWS];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const uint8_t* t = w + int64_t(blockIdx.x) * units * unit_bytes<QT>();
  float mx = 0.0f, ss = 0.0f;
  bool far = false;
  for (int u = wv; u < units; u += 4)
    tile_unit<QT>(
        t + int64_t(u) * unit_bytes<QT>(), lane,
        [&](int g, const float(&v)[8], float s, float o) {
          if (int64_t(u) * UNIT + 32 * g >= K) return;
          float gx = 0.0f;
#pragma unroll
          for (int p = 0; p < 8; p++) {
            gx = fmaxf(gx, fabsf(v[p]) < __builtin_inff() ? fabsf(v[p]) : 0.0f);
            ss = __builtin_fmaf(v[p], v[p], ss);
          }
          mx = fmaxf(mx, gx);
          if constexpr (has_offset<QT>) {
            gx = fmaxf(gx, __shfl_xor(gx, 16));  // (the row's other lanes)
            gx = fmaxf(gx, __shfl_xor(gx, 32));
            far |= !(15.0f * fabsf(s) + fabsf(o) <= 8.0f * gx);
          }
        });
  if (has_offset<QT> && far) atomicMax(out + 2, 1u);
  for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  ss += __shfl_xor(ss, 16);
  ss += __shfl_xor(ss, 32);
  if (lane < TROWS) red[wv][lane] = ss;
  if (lane == 0) atomicMax(out, __float_as_uint(mx));
  __syncthreads();
  if (threadIdx.x < TROWS) {
    const float s = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
    if (s < __builtin_inff()) atomicMax(out + 1, __float_as_uint(sqrtf(s) * 1.001f));
  }
}

// one or two matrices of a launch: their blocks, where their values go, times 2^-e
struct Unpack {
  const uint8_t* w[2];
  uint16_t* out[2];
  int e[2];
};

// W as fp16 rows of ld values: a wave per unit of a tile, a half at a time turned in its own part of LDS so that a store takes
// 256 bytes of each of 4 rows (as it is held, 64 bytes of 16 rows: 60 us where this takes 38); plane 1 (where there is one)
// what plane 0's rounding left. Bound by its writes: 38 us are 2 x 4096 x 11008 Q4_K, 5.9 TB/s.
template <int QT, int PLANES>
__global__ __launch_bounds__(256) void k_unpack(const Unpack two, int units, uint32_t all, int64_t N, int64_t K, int64_t ld,
                                                int64_t plane) {
  const uint8_t* w = two.w[blockIdx.y];
  uint16_t* out = two.out[blockIdx.y];
  const int e = two.e[blockIdx.y];
  __shared__ __attribute__((aligned(16))) uint8_t turn[4][PLANES][TROWS * 256];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lg = lane >> 4, lr = lane & 15;
  const uint32_t i = blockIdx.x * 4 + wv;
  if (i >= all) return;
  const uint32_t tile = i / units, u = i % units;
  const int r4 = lane >> 4, c = lane & 15;  // (out again: row r4 + 4 q, 16 bytes at 16 c)
  const auto half = [&](auto hv) __attribute__((always_inline)) {
    constexpr int H = decltype(hv)::value;
    tile_half<QT, H>(w + int64_t(i) * unit_bytes<QT>(), lane, [&](int g, const float(&v)[8]) {
      uint16_t a[8], b[8];
      halves(v, e, a, b);
      if (int64_t(u) * UNIT + 32 * g >= K)
        for (int p = 0; p < 8; p++) a[p] = b[p] = 0;
      const int at = lr * 256 + (((4 * (g & 3) + lg) ^ (lr & 7)) << 4);
      __builtin_memcpy(__builtin_assume_aligned(&turn[wv][0][at], 16), a, 16);
      if (PLANES == 2) __builtin_memcpy(__builtin_assume_aligned(&turn[wv][PLANES - 1][at], 16), b, 16);
    });
    __builtin_amdgcn_wave_barrier();  // (the wave's own part: its writes come before its reads)
    const int64_t k = int64_t(u) * UNIT + 128 * H + 8 * c;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int r = r4 + 4 * q;
      const int64_t n = int64_t(tile) * TROWS + r;
      if (n < N && k < ld)
#pragma unroll
        for (int pl = 0; pl < PLANES; pl++)
          *reinterpret_cast<uint4*>(out + pl * plane + n * ld + k) =
              *reinterpret_cast<const uint4*>(&turn[wv][pl][r * 256 + ((c ^ (r & 7)) << 4)]);
    }
    __builtin_amdgcn_wave_barrier();
  };
  half(std::integral_constant<int, 0>{});
  half(std::integral_constant<int, 1>{});
}

// W's transpose as fp16 rows of ld values: a workgroup per unit of 4 tiles (64 rows of W), a half at a time turned in LDS
template <int QT, int PLANES>
__global__ __launch_bounds__(256) void k_unpack_t(const Unpack two, int units, int64_t tiles, int64_t N, int64_t K,
                                                  int64_t ld, int64_t plane) {
  const uint8_t* w = two.w[blockIdx.y];
  uint16_t* out = two.out[blockIdx.y];
  const int e = two.e[blockIdx.y];
  constexpr int LD = 72;  // (a row's 64 values and 8 more: 16-byte rows, their banks spread)
  __shared__ __attribute__((aligned(16))) uint16_t t[PLANES][UNIT / 2][LD];
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, lg = lane >> 4, lr = lane & 15;
  const int64_t g4 = blockIdx.x / uint32_t(units), tile = 4 * g4 + wv;
  const int u = int(blockIdx.x % uint32_t(units));
  const bool live = tile < tiles && tile * TROWS + lr < N;
  const uint8_t* ub = w + ((tile < tiles ? tile : 0) * units + u) * unit_bytes<QT>();
  const auto put = [&](int g, const float(&v)[8]) {
    uint16_t a[8], b[8];
    halves(v, e, a, b);
#pragma unroll
    for (int p = 0; p < 8; p++) {
      t[0][32 * (g & 3) + 8 * lg + p][16 * wv + lr] = live ? a[p] : 0;
      if (PLANES == 2) t[PLANES - 1][32 * (g & 3) + 8 * lg + p][16 * wv + lr] = live ? b[p] : 0;
    }
  };
#pragma unroll
  for (int h = 0; h < 2; h++) {
    if (h == 0)
      tile_half<QT, 0>(ub, lane, put);
    else
      tile_half<QT, 1>(ub, lane, put);
    __syncthreads();
    for (int i = threadIdx.x; i < UNIT / 2 * 8; i += 256) {
      const int row = i >> 3, c = i & 7;
      const int64_t k = int64_t(u) * UNIT + 128 * h + row, n = 64 * g4 + 8 * c;
      if (k >= K || n >= ld) continue;
#pragma unroll
      for (int pl = 0; pl < PLANES; pl++)
        *reinterpret_cast<uint4*>(out + pl * plane + k * ld + n) = *reinterpret_cast<const uint4*>(&t[pl][row][8 * c]);
    }
    __syncthreads();
  }
}

}  // namespace

int launch_unpack(const artlite_matrix* m, const artlite_matrix* m2, bool transposed, int e, int e2, uint16_t* out,
                  uint16_t* out2, int64_t ld, int64_t plane, int planes, hipStream_t s) {
  const Unpack w{{m->w.as<uint8_t>(), m2 ? m2->w.as<uint8_t>() : nullptr}, {out, out2}, {e, e2}};
  const int64_t all = m->tiles * m->units;
  const dim3 grid(unsigned(transposed ? (m->tiles + 3) / 4 * m->units : (all + 3) / 4), m2 ? 2 : 1);
#define ART_U(QT)                                                                                          \
  if (transposed && planes == 1)                                                                           \
    k_unpack_t<QT, 1><<<grid, 256, 0, s>>>(w, m->units, m->tiles, m->N, m->K, ld, plane);          \
  else if (transposed)                                                                                     \
    k_unpack_t<QT, 2><<<grid, 256, 0, s>>>(w, m->units, m->tiles, m->N, m->K, ld, plane);          \
  else if (planes == 1)                                                                                    \
    k_unpack<QT, 1><<<grid, 256, 0, s>>>(w, m->units, uint32_t(all), m->N, m->K, ld, plane);                 \
  else                                                                                                     \
    k_unpack<QT, 2><<<grid, 256, 0, s>>>(w, m->units, uint32_t(all), m->N, m->K, ld, plane);                 \
  break
  ART_TILE_QTYPES(m->t->id, ART_U)
#undef ART_U
  ART_HIP(hipGetLastError());
  return ARTLITE_OK;
}

int OnDevice::set(int device) {
  int cur = -1;
  ART_HIP(hipGetDevice(&cur));
  if (cur == device) return ARTLITE_OK;
  ART_HIP(hipSetDevice(device));
  was = cur;
  return ARTLITE_OK;
}

int check_device(const void* p, int device, const char* what) {
  hipPointerAttribute_t a;
  if (!p) return fail(ARTLITE_EINVAL, "%s: null", what);
  if (hipPointerGetAttributes(&a, p) != hipSuccess) {
    (void)hipGetLastError();
    return fail(ARTLITE_EINVAL, "%s: not device memory", what);
  }
  if (a.type != hipMemoryTypeDevice) return fail(ARTLITE_EINVAL, "%s: not device memory", what);
  if (a.device != device) return fail(ARTLITE_EINVAL, "%s: memory of device %d, not %d", what, a.device, device);
  return ARTLITE_OK;
}

int WorkScope::begin(Work* work, size_t need, hipStream_t stream, const char* what) {
  if (need == 0) return ARTLITE_OK;
  if (!work) return fail(ARTLITE_EINVAL, "%s: needs a workspace of %zu bytes", what, need);
  if (work->n < need) return fail(ARTLITE_EINVAL, "%s: a workspace of %zu bytes, not %zu", what, work->n, need);
  work->mu.lock();
  w = work;
  s = stream;
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  ART_HIP(hipStreamIsCapturing(stream, &st));
  if (st != hipStreamCaptureStatusNone)
    return w->eager ? fail(ARTLITE_EINVAL, "%s: a captured call takes a workspace of its own", what) : ARTLITE_OK;
  // (the per-thread default stream is one handle, and each thread's own stream behind it)
  if (w->used && (w->last != stream || stream == hipStreamPerThread)) ART_HIP(hipStreamWaitEvent(stream, w->done, 0));
  note = true;
  return ARTLITE_OK;
}

WorkScope::~WorkScope() {
  if (!w) return;
  if (note && hipEventRecord(w->done, s) == hipSuccess) {
    w->used = true;
    w->last = s;
  }
  w->mu.unlock();
}

namespace {
int matrix_upload(artlite_matrix* m, const void* data) {
  HostCtx* c;
  ART_TRY(host_ctx(&c));
  const size_t nb = size_t(m->N) * size_t(m->K / m->t->per) * m->t->bytes;
  DevBuf raw;
  ART_TRY(raw.reserve(nb));
  ART_TRY(c->flag.reserve(256));
  ART_TRY(m->w.reserve(size_t(m->tiles) * m->units * m->ub + WEIGHT_TAIL));
  uint32_t b[3] = {0, 0, 0};
  ART_HIP(hipMemcpyAsync(raw.p, data, nb, hipMemcpyHostToDevice, c->stream));
  ART_HIP(hipMemcpyAsync(c->flag.p, b, 12, hipMemcpyHostToDevice, c->stream));
  const unsigned grid = unsigned(m->tiles * m->units);
#define ART_T(QT)                                                                                                   \
  k_tile<QT, QT == ARTLITE_Q4_K || QT == ARTLITE_IQ4_XS ? 256 : 32,                                                 \
         QT == ARTLITE_Q4_K ? 144 : QT == ARTLITE_IQ4_XS ? 136 : QT == ARTLITE_Q4_1 ? 20 : 18>                      \
      <<<grid, 128, 0, c->stream>>>(raw.as<uint8_t>(), m->N, m->K, m->units, m->w.as<uint8_t>());                   \
  k_bounds<QT><<<unsigned(m->tiles), 256, 0, c->stream>>>(m->w.as<uint8_t>(), m->units, m->K, c->flag.as<uint32_t>()); \
  break
  ART_TILE_QTYPES(m->t->id, ART_T)
#undef ART_T
  ART_HIP(hipGetLastError());
  ART_HIP(hipMemcpyAsync(b, c->flag.p, 12, hipMemcpyDeviceToHost, c->stream));
  ART_HIP(hipStreamSynchronize(c->stream));
  float f[2];
  std::memcpy(f, b, 8);
  // (of finite values; a matrix without any, or of zeros: any bound will do)
  m->max_exp = f[0] > 0.0f ? exp_above(f[0]) : 0;
  m->row_exp = f[1] > 0.0f ? exp_above(f[1]) : 0;
  m->direct = b[2] == 0;
  m->have = true;
  return ARTLITE_OK;
}
}  // namespace

}  // namespace artlite

using namespace artlite;

extern "C" int artlite_matrix_supported(int qtype) { return tile_unit_bytes(qtype) != 0; }

extern "C" int artlite_matrix_create(int qtype, int64_t rows, int64_t cols, artlite_matrix** out) {
  if (!out) return fail(ARTLITE_EINVAL, "matrix: null");
  *out = nullptr;
  const QType* t = qtype_by_id(qtype);
  const int ub = tile_unit_bytes(qtype);
  if (!t || !ub)
    return fail(ARTLITE_EINVAL, "matrix: weight type %d (%s) is not one of Q4_0, Q4_1, Q4_K, IQ4_NL, IQ4_XS", qtype,
                t ? t->name : "unknown");
  // (sizes whose tiles and rows every launch's grid reaches)
  if (rows < 1 || cols < 1 || rows > (int64_t(1) << 24) || cols > (int64_t(1) << 20) || cols % t->per)
    return fail(ARTLITE_EINVAL, "matrix: %lld rows of %lld values in blocks of %d", (long long)rows, (long long)cols, t->per);
  const int64_t tiles = (rows + TROWS - 1) / TROWS, units = (cols + UNIT - 1) / UNIT;
  if (tiles * units > (int64_t(1) << 30))
    return fail(ARTLITE_EINVAL, "matrix: %lld rows of %lld values", (long long)rows, (long long)cols);
  HostCtx* c;
  ART_TRY(host_ctx(&c, false));
  artlite_matrix* m = new (std::nothrow) artlite_matrix;
  if (!m) return fail(ARTLITE_ENOMEM, "matrix: no memory");
  m->device = c->device;
  m->t = t;
  m->N = rows, m->K = cols;
  m->tiles = tiles, m->units = int(units), m->ub = ub;
  *out = m;
  return ARTLITE_OK;
}

extern "C" int artlite_matrix_destroy(artlite_matrix* m) {
  if (!m) return ARTLITE_OK;
  OnDevice on;
  const int rc = on.set(m->device);
  delete m;
  return rc;
}

extern "C" int artlite_matrix_upload(artlite_matrix* m, const void* data, size_t nbytes) {
  if (!m || !data) return fail(ARTLITE_EINVAL, "matrix upload: null argument");
  const size_t want = size_t(m->N) * size_t(m->K / m->t->per) * m->t->bytes;
  if (nbytes != want) return fail(ARTLITE_EINVAL, "matrix upload: %zu bytes, not %zu", nbytes, want);
  OnDevice on;
  ART_TRY(on.set(m->device));
  // (calls that read the bytes of an earlier upload come to their end first)
  if (m->have) ART_HIP(hipDeviceSynchronize());
  m->have = false;
  return matrix_upload(m, data);
}

extern "C" int artlite_matrix_upload_bias(artlite_matrix* m, const float* data, size_t n) {
  if (!m) return fail(ARTLITE_EINVAL, "matrix bias: null argument");
  if (n && (!data || int64_t(n) != m->N))
    return fail(ARTLITE_EINVAL, "matrix bias: %zu values for %lld rows", n, (long long)m->N);
  OnDevice on;
  ART_TRY(on.set(m->device));
  if (m->has_bias) ART_HIP(hipDeviceSynchronize());
  m->has_bias = false;
  if (!n) return ARTLITE_OK;
  ART_TRY(m->bias.reserve(n * 4));
  ART_HIP(hipMemcpy(m->bias.p, data, n * 4, hipMemcpyHostToDevice));
  m->has_bias = true;
  return ARTLITE_OK;
}

extern "C" int artlite_matrix_device(const artlite_matrix* m, int* device) {
  if (!m || !device) return fail(ARTLITE_EINVAL, "matrix: null");
  *device = m->device;
  return ARTLITE_OK;
}

extern "C" int artlite_workspace_create(int device, size_t nbytes, int eager_only, artlite_workspace** out) {
  if (!out) return fail(ARTLITE_EINVAL, "workspace: null");
  *out = nullptr;
  HostCtx* c;
  ART_TRY(host_ctx(&c, false));
  OnDevice on;
  ART_TRY(on.set(device < 0 ? c->device : device));
  artlite_workspace* w = new (std::nothrow) artlite_workspace;
  if (!w) return fail(ARTLITE_ENOMEM, "workspace: no memory");
  w->w.device = device < 0 ? c->device : device;
  w->w.n = nbytes;
  w->w.eager = eager_only != 0;
  hipError_t e = hipMalloc(reinterpret_cast<void**>(&w->w.p), nbytes ? nbytes : 256);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&w->w.done, hipEventDisableTiming);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    if (w->w.p) (void)hipFree(w->w.p);
    delete w;
    return fail(ARTLITE_ENOMEM, "workspace of %zu bytes: %s", nbytes, hipGetErrorString(e));
  }
  *out = w;
  return ARTLITE_OK;
}

extern "C" int artlite_stream_capturing(void* stream, int* out) {
  if (!out) return fail(ARTLITE_EINVAL, "stream: null");
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  ART_HIP(hipStreamIsCapturing(static_cast<hipStream_t>(stream), &st));
  *out = st != hipStreamCaptureStatusNone;
  return ARTLITE_OK;
}

extern "C" int artlite_stream_wait(int device, void* stream, void* other) {
  OnDevice on;
  ART_TRY(on.set(device));
  for (void* s : {stream, other}) {
    int capturing = 0;
    ART_TRY(artlite_stream_capturing(s, &capturing));
    if (capturing) return fail(ARTLITE_EINVAL, "stream wait: a stream that is being captured");
  }
  hipEvent_t e;
  ART_HIP(hipEventCreateWithFlags(&e, hipEventDisableTiming));
  hipError_t rc = hipEventRecord(e, static_cast<hipStream_t>(other));
  if (rc == hipSuccess) rc = hipStreamWaitEvent(static_cast<hipStream_t>(stream), e, 0);
  (void)hipEventDestroy(e);  // (once it has come, if it is still to come)
  ART_HIP(rc);
  return ARTLITE_OK;
}

extern "C" int artlite_workspace_destroy(artlite_workspace* w) {
  if (!w) return ARTLITE_OK;
  OnDevice on;
  const int rc = on.set(w->w.device);
  if (w->w.used) (void)hipEventSynchronize(w->w.done);  // (its calls outside captures)
  if (w->w.done) (void)hipEventDestroy(w->w.done);
  if (w->w.p) (void)hipFree(w->w.p);
  delete w;
  return rc;
}

extern "C" int artlite_device_alloc(int* device, size_t nbytes, void** out) {
  if (!out || !device) return fail(ARTLITE_EINVAL, "device memory: null");
  *out = nullptr;
  HostCtx* c;
  ART_TRY(host_ctx(&c, false));
  OnDevice on;
  if (*device < 0) *device = c->device;
  ART_TRY(on.set(*device));
  if (hipMalloc(out, nbytes ? nbytes : 1) != hipSuccess) {
    (void)hipGetLastError();
    return fail(ARTLITE_ENOMEM, "device memory: %zu bytes", nbytes);
  }
  return ARTLITE_OK;
}

extern "C" int artlite_device_free(void* p) {
  if (p) ART_HIP(hipFree(p));
  return ARTLITE_OK;
}

extern "C" int artlite_device_copy(int device, void* dst, const void* src, size_t nbytes, int to_host) {
  if (!nbytes) return ARTLITE_OK;
  if (!dst || !src) return fail(ARTLITE_EINVAL, "device copy: null");
  OnDevice on;
  ART_TRY(on.set(device));
  // (behind everything queued on the device, whichever streams it is on)
  ART_HIP(hipDeviceSynchronize());
  ART_HIP(hipMemcpy(dst, src, nbytes, to_host ? hipMemcpyDeviceToHost : hipMemcpyHostToDevice));
  return ARTLITE_OK;
}
