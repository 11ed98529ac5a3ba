/* artlite_moe: an MI355X (gfx950) HIP library for artlite's mixture-of-experts FFN layer over GGUF-quantized experts.
 *
 * A C ABI of plain pointers and sizes. Every function returns an int status (ARTLITE_OK = 0); on failure the
 * calling thread's message is available from artlite_last_error. Host-pointer entry points copy their inputs to the
 * GPU, compute there, and copy the results back before returning (the caller owns every buffer, as with the
 * reference's _native module). A layer handle owns its device memory and a HIP stream; it is safe for one caller at
 * a time.
 */
#ifndef ARTLITE_MOE_H
#define ARTLITE_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum artlite_status {
  ARTLITE_OK = 0,
  ARTLITE_EINVAL = 1, /* an argument or shape error (the reference's artlite::Error) */
  ARTLITE_EHIP = 2,   /* a HIP runtime error, or no GPU */
  ARTLITE_ENOMEM = 3,
};

/* ggml tensor type ids of the supported weight formats (src/artlite/gguf_model.py:385-390 of the reference) */
enum artlite_qtype { ARTLITE_F32 = 0, ARTLITE_F16 = 1, ARTLITE_Q4_0 = 2, ARTLITE_Q4_1 = 3, ARTLITE_Q8_0 = 8,
                     ARTLITE_Q3_K = 11, ARTLITE_Q4_K = 12, ARTLITE_Q5_K = 13, ARTLITE_Q6_K = 14, ARTLITE_IQ4_NL = 20,
                     ARTLITE_IQ4_XS = 23, ARTLITE_BF16 = 30 };

/* The calling thread's last error message into buf (NUL-terminated, truncated to cap); returns its full length. */
size_t artlite_last_error(char* buf, size_t cap);

/* The library's version string. */
const char* artlite_version(void);

/* Number of visible GPUs into *n (0 without a GPU; the call itself succeeds). */
int artlite_device_count(int* n);

/* ---- routing: replaces _native.moe_route (reference csrc/bindings/moe.cpp:20-35 -> artlite::moe_route,
 * csrc/artlite/moe_host.h:9-15). The top k of n tokens' E fp32 logits (token t's at logits[t row ..], expert e at
 * (e / per_col) pitch + e % per_col), largest first, ties to the lower id, -0 as +0; weights e^(l - l_max) over the k
 * in double, normalized in numpy's summation order, rounded to fp32; sigmoid != 0: sigmoid(l) over their sum (at
 * least 2^-14). logits_len: the floats readable at logits (the reference's "arrays too small" check). ids, weights:
 * n x k. Errors: k < 1, k > E, E % per_col != 0, a short array. */
int artlite_moe_route(const float* logits, size_t logits_len, int64_t n, int64_t row, int per_col, int64_t pitch,
                      int E, int k, int sigmoid, int32_t* ids, float* weights);

/* ---- the decode cores' top k: replaces the reference's numpy model route.top_k (src/artlite/moe/route.py:69-80).
 * Plain (n, E) logits; the same ids as artlite_moe_route; weights in float64: the softmax over the k (numpy's
 * summation order) or, sigmoid != 0, the sigmoids over their sum (at least 2^-14). */
int artlite_moe_top_k(const float* logits, int64_t n, int E, int k, int sigmoid, int32_t* ids, double* weights);

/* ---- the chunk plan: replaces _native.moe_plan (reference csrc/bindings/moe.cpp:37-58 -> artlite::moe_plan,
 * csrc/artlite/moe_host.h:17-22), same argument order. ids: n x k; experts, sizes: cols x cap; counts: cols;
 * rows: cols x cap x chunk; pos: n x k. An expert's (token, slot) pairs in pair order, in chunks of at most chunk,
 * dealt to the columns in turn (expert by expert); rows hold tokens (padding: the chunk's first); pos the row
 * (c cap + j) chunk + i of each pair. Errors: an id outside [0, E), more than cap chunks in a column. */
int artlite_moe_plan(const int32_t* ids, int64_t n, int k, int E, int cols, int cap, int chunk, int32_t* experts,
                     int32_t* counts, int32_t* sizes, int32_t* rows, int64_t* pos);

/* ---- the chunk plan without allocating: no counterpart in the reference. For callers that cannot allocate device
 * memory (tight serving loops, harnesses that forbid hipMalloc): artlite_moe_plan's
 * arguments and results, with every device buffer it needs (the staged ids, the per-block histograms, counters,
 * the results before their copy back) carved from one static 8 MiB array per GPU, held until the process ends, and
 * the null stream. It calls no hipMalloc / hipFree. A call needing more than that array returns ARTLITE_EINVAL
 * (about 250000 pairs at E = 128). Calls share the GPU's array: calls that overlap on one GPU (other threads) race;
 * each call clears the counters it needs. Its host copies and synchronization make it unsuitable under HIP graph
 * capture. */
int artlite_moe_plan_static(const int32_t* ids, int64_t n, int k, int E, int cols, int cap, int chunk,
                            int32_t* experts, int32_t* counts, int32_t* sizes, int32_t* rows, int64_t* pos);

/* ---- dequantization: replaces _native.dequant_supported / dequant_rows (reference csrc/bindings/gguf.cpp:62-76 ->
 * artlite::dequant_rows, csrc/artlite/dequant.h:12-17). n rows of qtype (the reference's native types: "F32", "F16",
 * "BF16", "Q4_0", "Q4_1", "Q8_0", "Q3_K", "Q4_K", "Q5_K", "Q6_K", "IQ4_NL", "IQ4_XS"), row_bytes apart in raw, into
 * out (n x cols fp32): the reference's fp32 values bit for bit. */
int artlite_dequant_supported(const char* qtype);
int artlite_dequant_rows(const char* qtype, const uint8_t* raw, size_t n, size_t row_bytes, size_t cols, float* out);

/* ---- the MoE layer: the device-resident form of the reference's MoE block (src/artlite/moe/prefill.py:33-214, its
 * semantics tests/moe/ref.py:43-60): router logits (x W^T, float64 accumulation, fp32), routing as
 * artlite_moe_route, the stable dispatch of the (token, slot) pairs by expert, the experts' SwiGLU FFNs over the
 * raw GGUF blocks, the weighted combine in slot order, plus an optional shared expert. */
typedef struct artlite_moe_layer artlite_moe_layer;

typedef struct artlite_moe_desc {
  int32_t hidden;       /* H */
  int32_t n_experts;    /* E */
  int32_t top_k;        /* k */
  int32_t expert_ffn;   /* F */
  int32_t gate_type;    /* artlite_qtype of ffn_gate_exps / ffn_up_exps (any quantized type of the enum) */
  int32_t down_type;    /* artlite_qtype of ffn_down_exps */
  int32_t shared_ffn;   /* the shared expert's width, 0: none */
  int32_t shared_type;  /* artlite_qtype of the shared expert's gate / up (and down, see shared_down_type) */
  int32_t shared_gated; /* 1: the shared expert times sigmoid(x . ffn_gate_inp_shexp) */
  int32_t gating;       /* 0: softmax, 1: sigmoid */
  int32_t max_tokens;   /* the most tokens of one call */
  float norm_eps;       /* > 0: x is first RMS-normalised by ffn_norm, x / sqrt(mean(x^2) + eps) * w (the steps
                           before the block's router: llama.cpp's ffn_norm, the reference's tests/np_ops.py:27-32);
                           0: none */
  int32_t residual;     /* 1: y += x (the block's residual add after the combine, x as given, before any norm) */
  int32_t shared_down_type; /* artlite_qtype of ffn_down_shexp when it differs from shared_type (a GGUF file's
                               mixed quantisation, e.g. Q4_K gate / up with a Q6_K down); 0: shared_type */
} artlite_moe_desc;

/* Tensors of artlite_moe_layer_upload, as laid out in a GGUF file. */
enum artlite_tensor {
  ARTLITE_ROUTER = 0,      /* ffn_gate_inp: E x H fp32 */
  ARTLITE_GATE_EXPS = 1,   /* ffn_gate_exps: E F rows of H values, raw blocks */
  ARTLITE_UP_EXPS = 2,     /* ffn_up_exps */
  ARTLITE_DOWN_EXPS = 3,   /* ffn_down_exps: E H rows of F values */
  ARTLITE_GATE_SHEXP = 4,  /* ffn_gate_shexp: Fs rows of H */
  ARTLITE_UP_SHEXP = 5,
  ARTLITE_DOWN_SHEXP = 6,  /* H rows of Fs */
  ARTLITE_GATE_INP_SHEXP = 7, /* H fp32 */
  ARTLITE_FFN_NORM = 8,    /* ffn_norm: H fp32 (with norm_eps > 0) */
};

/* Activation dtypes. */
enum artlite_dtype { ARTLITE_X_F32 = 0, ARTLITE_X_BF16 = 1 };

int artlite_moe_layer_create(const artlite_moe_desc* desc, artlite_moe_layer** out);
int artlite_moe_layer_destroy(artlite_moe_layer* layer);
/* Copy a tensor's bytes (exactly its size) into the layer's device memory. */
int artlite_moe_layer_upload(artlite_moe_layer* layer, int tensor, const void* data, size_t nbytes);
/* y (T x H fp32, host) = the layer of x (T x H, host, x_dtype); synchronous. */
int artlite_moe_layer_forward(artlite_moe_layer* layer, const void* x, int x_dtype, int64_t T, float* y);

/* Device-resident use: stage x into the layer's device input, then run (enqueued on the layer's stream, returns at
 * once), synchronize, and read y. */
int artlite_moe_layer_stage(artlite_moe_layer* layer, const void* x, int x_dtype, int64_t T);
int artlite_moe_layer_run(artlite_moe_layer* layer, int64_t T);
int artlite_moe_layer_sync(artlite_moe_layer* layer);
int artlite_moe_layer_output(artlite_moe_layer* layer, float* y, int64_t T);

/* Intermediate results of the last run, copied to the host (nbytes: the size of out, at least the tap's). */
enum artlite_tap {
  ARTLITE_TAP_LOGITS = 0,  /* T x E fp32 */
  ARTLITE_TAP_IDS = 1,     /* T x k int32 */
  ARTLITE_TAP_WEIGHTS = 2, /* T x k fp32 */
  ARTLITE_TAP_COUNTS = 3,  /* E int32: pairs per expert */
  ARTLITE_TAP_OFFSETS = 4, /* E + 1 int32: exclusive prefix of counts */
  ARTLITE_TAP_ORDER = 5,   /* T k int32: pair indices t k + i sorted by expert, pair order within an expert */
  ARTLITE_TAP_SLOT = 6,    /* T k int32: each pair's position in that order */
  ARTLITE_TAP_H = 7,       /* T k x F fp32: silu(gate) up of each sorted pair (as the run's path holds it) */
  ARTLITE_TAP_Y = 8,       /* T k x H fp32: each sorted pair's expert output (before the weights) */
  ARTLITE_TAP_XN = 9,      /* T x H fp32: the RMS-normalised x (norm_eps > 0) */
  ARTLITE_TAP_YS = 10,     /* T x H fp32: the shared expert's output, before its gate (shared_ffn > 0) */
};
int artlite_moe_layer_tap(artlite_moe_layer* layer, int tap, void* out, size_t nbytes);

/* Timing on the layers' stream with HIP events: warmup then iters runs of T tokens, cycling through the n layers
 * (distinct weight sets, so a working set larger than the GPU's caches is streamed from HBM). ms_per_run: the
 * average over a timed region of back-to-back runs (events only at its ends). run_ms (may be NULL; iters entries):
 * each run's duration, from an event recorded before each run of a second region (those events hold each run back
 * by a few microseconds). kernel_ms (may be NULL): with per-kernel events in a further timed region, each kernel's
 * average duration (artlite_moe_kernel_names order), kernel_cap entries at most; *n_kernels the count. */
int artlite_moe_layer_time(artlite_moe_layer** layers, int n, int64_t T, int warmup, int iters, double* ms_per_run,
                           double* run_ms, double* kernel_ms, int kernel_cap, int* n_kernels);
/* The names of the kernels of a run of T tokens on this layer, ';'-separated, into buf; a product's on the streamed tiles
 * with '@' and their rows after it ("gate_up@stream16"), a shared expert's on the streamed dense rows with "@stream". */
int artlite_moe_kernel_names(artlite_moe_layer* layer, int64_t T, char* buf, size_t cap);

/* Bytes copied per ms by a plain device copy of nbytes (HBM calibration of the profile counters). */
int artlite_hbm_copy(size_t nbytes, int iters, double* ms_per_copy);

/* ---- dense products over 4-bit blocks: no counterpart in the reference's native module (its models run them as NPU
 * programs). A matrix of a GGUF file (rows = output features, cols = K) in HBM, in the format's own bytes re-ordered for the
 * kernels; Q4_0, Q4_1, Q4_K, IQ4_NL or IQ4_XS; cols a multiple of the format's block, at most 2^20; at most 2^24 rows.
 * Created on the calling thread's current device, which its calls then use whichever device is current.
 *
 * x, y and the gradients below are DEVICE memory of that device (anything else is refused), bf16 or fp32 (artlite_dtype;
 * y and gradients in x's type), rows of consecutive values `stride` values apart: x's at least 0 (0: one row for all),
 * those of what is written at least the row's values; what is written overlaps nothing else of the call's. Calls are
 * enqueued on `stream` (a hipStream_t; null: the null stream) and return at once; 0 rows write nothing (a backward call: zeros
 * to the weights' gradients that are asked for). They may be captured into a graph: its replays use the workspace that was
 * given, and whatever else uses that workspace has to be ordered with them by the caller's streams (a workspace for each graph
 * that runs beside others). Outside captures, calls on one workspace order themselves, whichever streams and threads they come
 * from (hipStreamPerThread among them). The same call gives the same bits.
 * A value of x that is infinite or no number reaches its own row alone, one of a matrix its own row's outputs. Few rows' sums
 * are of codes, a group's times its scale: exact to about 2^-15 of the group's scale and offset, also where its values
 * themselves come out far smaller than both; values beyond 2^100 in size may overflow them, and fp32 ones are held to 2^-134.
 * Past few rows (see artlite_linear) a row of x and a matrix's values are fp16, of fp32 calls two of them, each row times a
 * power of two from its largest finite value and the matrix from its own: what is below 2^-29 (fp32: 2^-17) of that loses
 * bits, what is below 2^-40 of it is 0. */
typedef struct artlite_matrix artlite_matrix;
int artlite_matrix_supported(int qtype);
int artlite_matrix_create(int qtype, int64_t rows, int64_t cols, artlite_matrix** out);
int artlite_matrix_destroy(artlite_matrix* m); /* its calls have come to their end */
/* The rows' raw blocks (host, exactly their size); replaces earlier ones once the device is idle. A graph that captured calls on
 * the matrix is captured again after that. */
int artlite_matrix_upload(artlite_matrix* m, const void* data, size_t nbytes);
/* n = rows fp32 values added to every output row of artlite_linear; n = 0: none. */
int artlite_matrix_upload_bias(artlite_matrix* m, const float* data, size_t n);

int artlite_matrix_device(const artlite_matrix* m, int* device);

/* Scratch memory of calls, of a fixed size, on a device (-1: the current one). eager_only: a call under stream capture that
 * would use it is refused (for one that many callers share). A stream's calls have come to their end before it is destroyed.
 * artlite_stream_capturing: whether a stream is being captured (memory is then not to be allocated). artlite_stream_wait: what
 * is queued on `stream` from now on waits for what is on `other` by now (streams of `device`, neither being captured). */
typedef struct artlite_workspace artlite_workspace;
int artlite_workspace_create(int device, size_t nbytes, int eager_only, artlite_workspace** out);
int artlite_stream_capturing(void* stream, int* out);
int artlite_stream_wait(int device, void* stream, void* other);
int artlite_workspace_destroy(artlite_workspace* work); /* its calls have come to their end */

/* y (n x rows) = x (n x cols) W^T (+ bias). x's products with the blocks' values are summed in fp32 and rounded once to y's
 * type (up to 128 rows, 256 bf16 ones of a matrix that is not large, more of a small one, without rounding a weight; past that
 * weights are fp16 of 11 bits for bf16 x, of 22 for fp32 x).
 * artlite_linear_workspace: the bytes of workspace that a call of n rows needs (0 for up to 16 rows); work may be null where
 * that is 0. */
int artlite_linear_workspace(const artlite_matrix* w, int dtype, int64_t n, size_t* nbytes);
int artlite_linear(const artlite_matrix* w, const void* x, int dtype, int64_t n, int64_t x_stride, void* y,
                   int64_t y_stride, artlite_workspace* work, void* stream);

/* ---- the gated feed-forward block (a model's dense blocks: ffn_gate, ffn_up F x H, ffn_down H x F):
 * y = (act(x gate^T) (x up^T)) down^T, and its backward pass from x and dy (n x H):
 * dx = dg gate + du up, dgate = dg^T x, dup = du^T x, ddown = dy^T h, where g = x gate^T, u = x up^T, h = act(g) u,
 * dh = dy down, dg = dh u act'(g), du = dh act(g); dgate, dup (F x H) and ddown (H x F) are the gradients of the blocks'
 * values. The forward keeps nothing; the backward computes g and u again. Outputs that are null are not computed (dx too);
 * dgate, dup, ddown: rows without gaps.
 * Sums, activations and their derivatives are fp32. Between the products a forward's h goes as two planes of bf16 (2^-17; fp32
 * calls three, 2^-24) on the few rows' way, up to 64 bf16 or 192 rows, more of a small block. Past that h, and in
 * every backward the weights, x, dy, h, dh, dg and du, go as fp16 (2^-11; fp32 calls two of them, 2^-22), a row of h, dh, dg
 * and du times a power of two from bounds: |x|^2 |gate| |up|, |dy| max |down| sqrt(H), and the latter times 2 |x| and the
 * larger of |gate| and |up| (2-norms of rows, a matrix's largest one), each factor up to twice as large. What is below 2^-29
 * (fp32: 2^-17) of a bound loses bits, what is below 2^-40 of it is 0.
 * A value of x or dy that is infinite or no number reaches its own row of dx, all of dgate and dup, and, of x, all of ddown,
 * of dy, its own row of ddown. */
enum artlite_act { ARTLITE_ACT_SILU = 0, ARTLITE_ACT_GELU_TANH = 1 };
typedef struct artlite_ffn {
  const artlite_matrix *gate, *up, *down;
  int32_t act; /* artlite_act */
} artlite_ffn;
/* The bytes of workspace that a forward call of n rows needs (backward = 0), or a backward one (1: dx alone, 2: weights'
 * gradients). (Not always less for fewer rows: few rows' sums are taken in parts.) */
int artlite_ffn_workspace(const artlite_ffn* f, int dtype, int64_t n, int backward, size_t* nbytes);
int artlite_ffn_forward(const artlite_ffn* f, const void* x, int dtype, int64_t n, int64_t x_stride, void* y,
                        int64_t y_stride, artlite_workspace* work, void* stream);
int artlite_ffn_backward(const artlite_ffn* f, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride,
                         int dtype, int64_t n, void* dx, int64_t dx_stride, void* dgate, void* dup, void* ddown,
                         artlite_workspace* work, void* stream);

/* Device memory for callers that have no allocator of their own: allocated on *device (-1: the current one, which it becomes),
 * and copied to (to_host 0) or from the host behind everything queued on the device. */
int artlite_device_alloc(int* device, size_t nbytes, void** out);
int artlite_device_free(void* p);
int artlite_device_copy(int device, void* dst, const void* src, size_t nbytes, int to_host);

#ifdef __cplusplus
}
#endif

#endif /* ARTLITE_MOE_H */
