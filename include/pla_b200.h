/*
 * pla_b200.h — C ABI of the B200 (sm_100a) 7x7 depthwise-convolution and
 * 7x7 stencil library.
 *
 * Every entry point takes plain device pointers, element counts/strides and a
 * CUDA stream, launches asynchronously on that stream and returns a status
 * code (PLA_OK == 0).  Nothing here allocates device memory, synchronises the
 * stream or falls back to a CPU path: a non-zero status means no kernel ran.
 *
 * Numerical contract (shared by every kernel and by the CPU oracle that the
 * tests check against): each output point is
 *
 *     acc = 0;  for ky in 0..6: for kx in 0..6:
 *                   acc = fma(x[i+ky-3][j+kx-3], w[ky][kx], acc)
 *     y[i][j] = round_to_output_dtype(acc + bias)      (bias add skipped if null)
 *
 * with x == 0 outside the plane (zero padding 3, cross-correlation, output size
 * == input size), the accumulator in fp32 for fp32/bf16/fp16 data and fp64 for
 * fp64 data.  This is the semantics of torch.nn.Conv2d(C, C, 7, stride=1,
 * padding=3, groups=C) used by the reference modules, evaluated in one fixed
 * tap order so that results are bit-reproducible.
 */
#ifndef PLA_B200_H_
#define PLA_B200_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define PLA_API __attribute__((visibility("default")))
#else
#define PLA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Opaque CUDA stream handle (binary-compatible with cudaStream_t). */
typedef struct CUstream_st* pla_stream_t;

/* Element type codes.  The values are the ones the reference stencil launcher
 * uses for its `type` argument (data/stencil_direct_cuda_v7/stencil_cuda.cpp:30:
 * 0=float16, 1=float32, 2=float64, 3=bfloat16). */
enum pla_dtype {
  PLA_F16 = 0,
  PLA_F32 = 1,
  PLA_F64 = 2,
  PLA_BF16 = 3
};

/* Memory layout of a depthwise activation tensor [N, C, H, W]. */
enum pla_layout {
  PLA_NCHW = 0, /* torch.contiguous_format */
  PLA_NHWC = 1  /* torch.channels_last */
};

/* Status codes. */
enum pla_status {
  PLA_OK = 0,
  PLA_ERR_INVALID_ARGUMENT = 1, /* null pointer, negative size, bad enum   */
  PLA_ERR_UNSUPPORTED = 2,      /* dtype/layout/shape outside this library */
  PLA_ERR_TOO_LARGE = 3,        /* size exceeds grid/indexing limits       */
  PLA_ERR_CUDA = 4,             /* a CUDA runtime/driver call failed       */
  PLA_ERR_NO_DEVICE = 5,        /* no sm_100 device current                */
  PLA_ERR_DEVICE_FAULT = 6      /* a kernel recorded a bounded-wait timeout */
};

/* Human-readable text for a status code (static storage, never NULL). */
PLA_API const char* pla_status_string(int status);

/* Detail text of the last failure seen by this thread inside the library
 * (CUDA error strings, size limits). */
PLA_API const char* pla_last_cuda_error(void);

/* Library ABI version: (major << 16) | minor.  1.1 added pla_depthwise_forward,
 * 1.2 pla_depthwise7x7_layernorm_nhwc, 1.3 pla_depthwise7x7_forward_many, 1.4 the
 * sequence operators. */
PLA_API int pla_version(void);

/*
 * Single-step 7x7 stencil, one filter for all planes:
 *     y[n,0,:,:] = stencil(x[n,0,:,:]; w[0..48]) + b[0]
 *
 * Replaces the reference launchers
 *   launch_direct()  data/stencil_direct_cuda_v7/stencil_cuda_kernel.cu:230-244
 *   launch_stencil() data/stencil_cuda_v2/stencil_cuda_kernel.cu:195-209
 * with the argument meaning of launch_direct: x may be strided
 * (element strides sn, sh, sw; sn ignored when n == 1), y is contiguous
 * [n, h, width], w holds 49 taps row-major, b is NULL or one element, all of
 * dtype `dtype` (enum pla_dtype).  y must not overlap x (as with the
 * reference, whose extension allocates a fresh output): overlapping byte
 * spans return PLA_ERR_INVALID_ARGUMENT.  Unlike the reference it returns a
 * status.
 */
PLA_API int pla_stencil7x7_forward(const void* x, const void* w, const void* b, void* y,
                           int n, int h, int width,
                           int64_t sn, int64_t sh, int64_t sw,
                           int dtype, pla_stream_t stream);

/*
 * pla_stencil7x7_forward with the filter given by value: `taps` points to 49
 * fp32 taps in HOST memory (row-major), `bias` to one host fp32 value or is
 * NULL.  The taps travel in the kernel's parameter block, so the kernel reads
 * them as uniform constant operands instead of holding them in registers
 * (the fast path; same results bit for bit).  16-bit filters widen to fp32
 * exactly.  Only inputs that qualify for the TMA path are accepted (unit
 * column stride, 16-byte aligned rows); others return PLA_ERR_UNSUPPORTED
 * and should use pla_stencil7x7_forward.  Same reference counterpart as
 * pla_stencil7x7_forward.
 */
PLA_API int pla_stencil7x7_forward_taps(const void* x, const float* taps, const float* bias, void* y,
                                        int n, int h, int width,
                                        int64_t sn, int64_t sh, int64_t sw,
                                        int dtype, pla_stream_t stream);

/*
 * Depthwise 7x7 convolution (groups = C, stride 1, padding 3):
 *     y[n,c] = stencil(x[n,c]; w[c, 0..48]) + b[c]
 *
 * Replaces launch_depthwise_7x7_cutlass()
 *   data/depthwise_conv_7x7_cuda/model_cutlass_autotune_v6.py:428-458
 *   (and the v1/v5 launchers, model_cutlass.py:263-279,
 *    model_cutlass_autotune_v5.py:403-420).
 * Differences: w is the module's own [C,1,7,7] weight (no [C,8,80] repack),
 * b may be non-NULL ([C]), dtype may be f32/bf16/f16/f64 and layout NCHW or
 * NHWC.  x and y are dense in `layout` and must not overlap
 * (PLA_ERR_INVALID_ARGUMENT otherwise).
 */
PLA_API int pla_depthwise7x7_forward(const void* x, const void* w, const void* b, void* y,
                             int n, int c, int h, int width,
                             int dtype, int layout, pla_stream_t stream);

/*
 * Depthwise k x k convolution, k in {3, 5, 7} (groups = C, stride 1,
 * padding k / 2), w [C,1,k,k], same arguments otherwise.  k = 7 is
 * pla_depthwise7x7_forward.
 *
 * Replaces the operator of the reference's MetaSchedule benchmark
 *   benchmark/MetaSchedule/depthwise_conv.py:7-13 and :32-33
 *   (topi.nn.depthwise_conv2d_nchw(X, W, 1, k // 2, 1), kernel 3 or 7,
 *    NCHW, no bias, fp32/fp16/bf16),
 * whose numpy check (:41-46) accumulates the k*k products in fp32 in
 * row-major (ry, rx) order.  Here every output is one fp32 FMA chain in that
 * order plus the optional bias, rounded once; NHWC, bias and fp64 are also
 * accepted.  Other k: PLA_ERR_UNSUPPORTED.
 */
PLA_API int pla_depthwise_forward(const void* x, const void* w, const void* b, void* y,
                                  int n, int c, int h, int width, int k,
                                  int dtype, int layout, pla_stream_t stream);

/*
 * Several independent depthwise 7x7 problems in one call, for instance the
 * four stages of the ConvNeXt-T-shaped sweep (data/depthwise_conv_7x7.py's
 * benchmark shapes, one launcher call each in the reference,
 * model_cutlass_autotune_v6.py:428-458).  Problem i is
 * pla_depthwise7x7_forward(p[i].x, p[i].w, p[i].b, p[i].y, p[i].n, p[i].c,
 * p[i].h, p[i].width, dtype, layout): same arguments and results.
 *
 * The problems run concurrently: the call forks from `stream` onto up to 4
 * streams of the library (created once per device, on the first call made
 * with that device current), launches the problems round-robin and joins
 * back, so one problem's first tiles overlap another's last ones instead of
 * each launch paying its own ramp and drain.  Problems are launched smallest
 * first (by element count; ties in the given order): a large problem's
 * persistent grid occupies every SM, so a small one queued behind it would
 * start only in its drain.  Work queued on `stream` before
 * the call is finished before any problem starts; work queued after it
 * starts after every problem is done.  No problem's output may overlap any
 * problem's input or output (PLA_ERR_INVALID_ARGUMENT).  Arguments are
 * checked for every problem before anything is launched.
 *
 * The library streams are shared by every caller on the device: calls made
 * on different streams are ordered after one another on them (correct, but
 * not concurrent with each other), and a stream capture that contains a
 * call holds them in capture mode until the capture ends, so while it is
 * open no other thread may call this function on that device.
 */
typedef struct pla_dw_problem {
  const void* x;
  const void* w;
  const void* b; /* NULL: no bias */
  void* y;
  int n, c, h, width;
} pla_dw_problem;
PLA_API int pla_depthwise7x7_forward_many(const pla_dw_problem* problems, int count, int dtype, int layout,
                                          pla_stream_t stream);

/*
 * Depthwise 7x7 followed by LayerNorm over the channels of every pixel, in
 * one pass over HBM: the "dwconv -> norm" pair of a ConvNeXt block,
 *     v = depthwise7x7(x; w, b) rounded to dtype   (pla_depthwise7x7_forward)
 *     y[n,i,j,:] = (v[n,i,j,:] - mean) / sqrt(var + eps) * gamma + beta
 * with mean / biased variance over the C channels of the pixel.
 *
 * No reference counterpart: the reference's operator is the depthwise half
 * (data/depthwise_conv_7x7.py:15-29, whose CUDA launchers
 * pla_depthwise7x7_forward replaces); the LayerNorm is the next layer of the
 * ConvNeXt stages its benchmark shapes come from.
 *
 * x and y are channels_last (NHWC) [n, h, width, c], dense, of dtype f32 /
 * bf16 / f16, and must not overlap; w [c,1,7,7]; b, gamma, beta [c] of the
 * same dtype or NULL (no bias / scale 1 / shift 0); eps >= 0.  The
 * normalisation runs in fp32 on the rounded depthwise outputs in a fixed
 * order (sums per 32-channel group, then over the groups), one rounding of
 * y.  Supported: c * element size a multiple of 16 bytes and at most 16
 * channel groups per pixel (c <= 512; c <= 2048 for 7 x 7 planes, whose
 * groups hold 128 channels); other shapes return PLA_ERR_UNSUPPORTED.
 */
PLA_API int pla_depthwise7x7_layernorm_nhwc(const void* x, const void* w, const void* b,
                                            const void* gamma, const void* beta, float eps,
                                            void* y, int n, int c, int h, int width, int dtype,
                                            pla_stream_t stream);

/*
 * Iterated stencil on one device (no reference counterpart; the reference
 * path is data/stencil_7x7.py:10-12 applied `steps` times with zero padding
 * each step, i.e. a zero Dirichlet boundary):
 *     u_0 = x;  u_{t+1} = stencil(u_t; w) (+ b if non-NULL);  y = u_steps
 * fp32/bf16/f16 planes [h, width], contiguous.  `scratch` is a caller-owned
 * device buffer of at least h*width elements used as the second ping-pong
 * buffer; x is only read; y may be x itself.  A partial overlap of x and y,
 * or a scratch overlapping either, returns PLA_ERR_INVALID_ARGUMENT.
 */
PLA_API int pla_stencil7x7_iterate(const void* x, const void* w, const void* b, void* y,
                           void* scratch, int h, int width, int steps,
                           int dtype, pla_stream_t stream);

/*
 * pla_stencil7x7_iterate without a caller scratch buffer, for callers that
 * cannot allocate device memory: a plugin running inside a host framework
 * that owns every device allocation, a fixed-budget embedded runtime, or a
 * real-time loop that cannot afford cudaMalloc's implicit synchronisation.
 * This entry point has no counterpart in the reference.
 *
 * The second ping-pong plane is a 16 MiB static device array inside this
 * library (PLA_NOALLOC_SCRATCH_BYTES), held by every GPU that loads the
 * library until the process exits.  Grids larger than that (h * width *
 * element size > 16 MiB, e.g. more than 2048 x 2048 fp32) return
 * PLA_ERR_TOO_LARGE with the sizes in pla_last_cuda_error().  Nothing is
 * allocated: no cudaMalloc/cudaFree or allocating library call.
 *
 * The first call on a device looks up the array's device address
 * (cudaGetSymbolAddress) with that device current; make that first call
 * before any stream capture.  Only a successful lookup is kept: after a
 * failed one the next call tries again.  All calls on a device share the one array and
 * leave the last call's data in it (no call needs it cleared: every step
 * overwrites the whole plane before reading it), so calls that overlap on
 * the GPU (concurrent streams) race on it; serialise them.
 * Arguments and results are those of pla_stencil7x7_iterate.
 */
#define PLA_NOALLOC_SCRATCH_BYTES (16u << 20)
PLA_API int pla_stencil7x7_iterate_noalloc(const void* x, const void* w, const void* b, void* y,
                                           int h, int width, int steps,
                                           int dtype, pla_stream_t stream);

/* pla_stencil7x7_iterate with host taps (see pla_stencil7x7_forward_taps). */
PLA_API int pla_stencil7x7_iterate_taps(const void* x, const float* taps, const float* bias, void* y,
                                        void* scratch, int h, int width, int steps,
                                        int dtype, pla_stream_t stream);

/*
 * One Jacobi step of a row band of a larger grid (building block of the
 * row-band multi-GPU iterated stencil; no reference counterpart).
 * `in` and `out` are band buffers of (rows + 6) x width elements: rows 0..2
 * hold the 3 halo rows above the band, rows 3..rows+2 the band itself and
 * rows rows+3..rows+5 the halo rows below it.  The step writes output band
 * rows [row_begin, row_end) (0 <= row_begin <= row_end <= rows) into
 * out rows 3+row_begin .. 3+row_end-1; halo rows of `out` are not touched.
 * `in` and `out` must not overlap (PLA_ERR_INVALID_ARGUMENT).
 */
PLA_API int pla_stencil7x7_band_step(const void* in, const void* w, const void* b, void* out,
                             int rows, int width, int row_begin, int row_end,
                             int dtype, pla_stream_t stream);

/* pla_stencil7x7_band_step with host taps (see pla_stencil7x7_forward_taps). */
PLA_API int pla_stencil7x7_band_step_taps(const void* in, const float* taps, const float* bias, void* out,
                                          int rows, int width, int row_begin, int row_end,
                                          int dtype, pla_stream_t stream);

/*
 * One band step fused with the halo exchange over peer memory (NVLink), the
 * row-band multi-GPU iterated stencil without a separate collective (no
 * reference counterpart).  Band buffers as in pla_stencil7x7_band_step; the
 * step computes every band row (rows >= 64) with the host taps, and
 *  - before reading its halo, waits (bounded, ~2 s, then fault bit 1) until
 *    flags[0] >= step (neighbour above delivered) / flags[1] >= step (below);
 *  - stores its first 3 band rows into up_out rows up_rows+3..up_rows+5 and
 *    its last 3 into down_out rows 0..2 (the neighbours' `out` buffers, peer
 *    pointers from pla_ipc_import), then raises up_flags[1] / down_flags[0]
 *    (the neighbours' flags) to step+1.
 * up_out/down_out NULL = grid edge (zero halo kept).  flags[2] and counters[2]
 * are this GPU's zero-initialised words; steps must be launched 0, 1, 2, ...
 * on every rank.  Ranks are separate GPUs (never two on one device).
 */
PLA_API int pla_stencil7x7_band_step_halo(const void* in, const float* taps, const float* bias, void* out,
                                          int rows, int width, int dtype,
                                          void* up_out, int up_rows, void* down_out,
                                          unsigned int* flags, unsigned int* up_flags,
                                          unsigned int* down_flags, unsigned int* counters,
                                          unsigned int step, pla_stream_t stream);

/* ------------------------------------------------------------------------
 * Sequence operators: the layers of a sequence block built from the same
 * pieces as above (depthwise convolution, fused norm, a state updated
 * linearly).  No reference counterpart.  dtype is f32 / bf16 / f16; sums,
 * norms and states are fp32.  Strides are in elements; the innermost
 * dimension is dense.  Outputs are dense and must not overlap an input.
 * Tensors need no more than their elements' alignment (whole vectors are moved
 * where addresses and strides allow it); workspaces as stated.
 *
 * A ragged batch is one batch row (batch == 1) of `tokens` tokens cut by
 * cu_seqlens, an int32 device array of sequences + 1 ascending entries that
 * starts at 0: sequence i holds tokens [cu_seqlens[i], cu_seqlens[i + 1]).
 * Entries are clamped to [0, tokens] on the device, so wrong ones give wrong
 * results but touch nothing outside the tensors.  Output rows that belong to
 * no sequence are zero.  cu_seqlens NULL: every batch row is one sequence
 * (sequences == batch).
 * ------------------------------------------------------------------------ */

/*
 * Causal depthwise convolution along time, channels last:
 *     p[t] = b + sum_{j < taps} w[c, j] x[t - taps + 1 + j],  taps in 2..4
 *     y[t] = silu ? p[t] / (1 + e^-p[t]) : p[t].
 * x [batch, tokens, channels]; w [channels, taps]; b [channels] or NULL.
 * state_in [sequences, taps - 1, channels] holds the inputs before each
 * sequence, oldest first (NULL: zeros); state_out, if not NULL, receives the
 * last taps - 1 inputs (it may not be state_in).
 */
typedef struct pla_causal {
  const void* x;
  int64_t x_batch, x_token;
  const void* w;
  const void* b;
  const int* cu_seqlens;
  const void* state_in;
  void* state_out;
  void* y;
  int batch, tokens, channels, taps, sequences, silu, dtype;
} pla_causal;
PLA_API int pla_causal_depthwise_forward(const pla_causal* a, pla_stream_t stream);

/*
 * Gradients of pla_causal_depthwise_forward (a->y and a->state_out unused):
 * dx (dense) from dy and, if not NULL, dstate_out; dw, db and dstate_in each
 * if not NULL.  workspace holds pla_causal_depthwise_workspace(a) bytes,
 * 16-byte aligned, needed when dw or db is wanted.  No atomics: the same
 * inputs give the same bits.
 */
typedef struct pla_causal_gradient {
  const void* dy;
  int64_t dy_batch, dy_token;
  const void* dstate_out;
  void* dx;
  void* dw;
  void* db;
  void* dstate_in;
  void* workspace;
  size_t workspace_bytes;
} pla_causal_gradient;
PLA_API size_t pla_causal_depthwise_workspace(const pla_causal* a);
PLA_API int pla_causal_depthwise_backward(const pla_causal* a, const pla_causal_gradient* g, pla_stream_t stream);

/* One more token for each of n sequences: x [n, channels] (row stride x_row),
 * state [n, taps - 1, channels] (row stride state_row) moved up in place, y
 * dense. */
PLA_API int pla_causal_depthwise_step(const void* x, int64_t x_row, void* state, int64_t state_row, const void* w,
                                      const void* b, void* y, int n, int channels, int taps, int silu, int dtype,
                                      pla_stream_t stream);

/*
 * Norm of queries and keys for each head, then the position rotation, in one
 * pass: n = x w / sqrt(mean(x^2) + eps) (l2 == 0) or x w / sqrt(sum(x^2) +
 * eps) (l2 == 1; w usually NULL); the first `rot` features are rotated in
 * pairs (a, b) -> (a c - b s, b c + a s) with c, s from row m of the fp32
 * tables cos_table / sin_table [table_rows, rot / 2] (NULL: no rotation),
 * pairs (2i, 2i + 1) if interleaved, else (i, i + rot / 2).  m is the token's
 * entry of `positions` ([batch, tokens], 4- or 8-byte integers, row stride
 * position_batch) or, if NULL, its number.  A position outside the tables
 * reads nothing and makes the rotated features NaN.  dim <= 256, rot even.
 */
typedef struct pla_norm_side {
  const void* x; /* [batch, tokens, heads, dim] */
  int64_t x_batch, x_token, x_head;
  const void* w; /* [dim] or NULL */
  void* y;       /* dense; backward: the gradient of x */
  const void* dy; /* backward */
  int64_t dy_batch, dy_token, dy_head;
  void* dw;      /* backward: [dim] or NULL */
  int heads;
} pla_norm_side;
typedef struct pla_qk_norm {
  pla_norm_side q, k;
  const float* cos_table;
  const float* sin_table;
  const void* positions;
  int64_t position_batch;
  int position_bytes, table_rows, batch, tokens, dim, rot, interleaved, l2;
  float eps;
  int dtype;
} pla_qk_norm;
PLA_API int pla_qk_norm_rotate_forward(const pla_qk_norm* a, pla_stream_t stream);
/* workspace: pla_qk_norm_rotate_workspace(a) bytes, needed when a dw is wanted.
 * batch x tokens x heads is at most 2^30 (forward: batch at most 65535). */
PLA_API size_t pla_qk_norm_rotate_workspace(const pla_qk_norm* a);
PLA_API int pla_qk_norm_rotate_backward(const pla_qk_norm* a, void* workspace, size_t workspace_bytes,
                                        pla_stream_t stream);

/*
 * Gated delta rule: per value head h (key head h / (hv / hk)) the state
 * S [dk, dv] starts as state_in[sequence, h] (fp32, NULL: zeros) and follows
 *     S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q.
 * q, k [batch, tokens, hk, dk]; v [batch, tokens, hv, dv]; g, beta [batch,
 * tokens, hv], both of dtype or both fp32 (gates32); o dense like v;
 * state_out [sequences, hv, dk, dv] fp32 or NULL.  dk, dv <= 128, hv a
 * multiple of hk.  It is stable for |k| up to about 1 and beta in [0, 2]; a g
 * below -200 is taken as -200 (its decay is 0 in fp32 either way).  Tokens are
 * worked on in chunks of 64 from a sequence's start: a value that is not finite
 * reaches its head's outputs (one of v: its feature's) from its chunk's start on.
 * workspace: pla_gated_delta_rule_workspace(a, 0) bytes, 256-byte aligned.
 */
typedef struct pla_delta {
  const void *q, *k, *v, *g, *beta;
  int64_t q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
  int64_t g_batch, g_token, g_head, beta_batch, beta_token, beta_head;
  const int* cu_seqlens;
  const float* state_in;
  float* state_out;
  void* o;
  int batch, tokens, sequences, hk, hv, dk, dv, gates32, dtype;
  float scale;
  void* workspace;
  size_t workspace_bytes;
} pla_delta;
PLA_API size_t pla_gated_delta_rule_workspace(const pla_delta* a, int backward);
PLA_API int pla_gated_delta_rule_forward(const pla_delta* a, pla_stream_t stream);

/*
 * Gradients of pla_gated_delta_rule_forward (a->o and a->state_out unused;
 * the chunks' states are computed again): from d_o and, if not NULL,
 * dstate_out, all of dq, dk, dv, dg, dbeta (dense, of their input's type) and,
 * if not NULL, dstate_in.  workspace: pla_gated_delta_rule_workspace(a, 1).
 */
typedef struct pla_delta_gradient {
  const void* d_o;
  int64_t do_batch, do_token, do_head;
  const float* dstate_out;
  float* dstate_in;
  void *dq, *dk, *dv, *dg, *dbeta;
} pla_delta_gradient;
PLA_API int pla_gated_delta_rule_backward(const pla_delta* a, const pla_delta_gradient* g, pla_stream_t stream);

/*
 * One more token for each of n sequences, the state updated in place:
 * q, k [n, hk, dk], v [n, hv, dv], g, beta [n, hv], state [n, hv, dk, dv]
 * fp32 (state_row elements between sequences), o [n, hv, dv] dense.
 * dk <= 256, dv any.
 */
typedef struct pla_delta_step {
  const void *q, *k, *v, *g, *beta;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head, beta_row, beta_head;
  float* state;
  int64_t state_row;
  void* o;
  int n, hk, hv, dk, dv, gates32, dtype;
  float scale;
} pla_delta_step;
PLA_API int pla_gated_delta_rule_step(const pla_delta_step* a, pla_stream_t stream);

/* CUDA IPC: export a device pointer as (64-byte handle of its allocation,
 * byte offset), import it in another process (peer access enabled lazily),
 * close an imported pointer. */
PLA_API int pla_ipc_export(const void* ptr, void* handle, uint64_t* offset);
PLA_API int pla_ipc_import(const void* handle, uint64_t offset, void** ptr);
PLA_API int pla_ipc_close(void* ptr, uint64_t offset);

/*
 * Device-side fault word of the current device: bit 0 = an mbarrier wait in a
 * kernel gave up after its time bound (its output is incomplete; a delta rule
 * step leaves that head's state as it was); bit 1 = a wait for a neighbouring
 * GPU's halo flag gave up.  Reading it synchronises the
 * device.  pla_clear_device_faults() zeroes it.
 */
PLA_API int pla_read_device_faults(unsigned int* faults);
PLA_API int pla_clear_device_faults(void);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* PLA_B200_H_ */
