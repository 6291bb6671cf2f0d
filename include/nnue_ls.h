/*
 * nnue_ls.h -- C ABI of the layer-stack operators for B200 (sm_100a): the dense
 * layers behind the feature transformer (reference
 * src/model/modules/layer_stacks.py, stacked_linear.py, moe_stacks.py).
 *
 * Conventions
 *   - All tensors are caller-owned DEVICE memory on the current CUDA device;
 *     nothing here allocates device memory.  Scratch comes from a caller
 *     workspace (256-byte aligned) sized by the call's *_workspace_size().
 *   - `stream` is a cudaStream_t (NULL = legacy default stream).  Calls only
 *     enqueue work; none synchronises the host, and every call can be captured
 *     in a CUDA graph.
 *   - Element types: NNUE_LS_F32, NNUE_LS_BF16, NNUE_LS_F16.  Sums, statistics
 *     and norms are held in fp32 whatever the type, and fp32 products are
 *     accurate to fp32 rounding (with more than 8 rows, and in every backward,
 *     operands below 2^-110 are held to 2^-134 instead of 24 bits).  Results do
 *     not depend on scheduling: no sum is formed with floating-point atomics.
 *   - Matrices are row-major with unit column stride; ld* is the row stride in
 *     elements.  Row counts may be 0 (then nothing is read).  Pointers are
 *     aligned to their elements, or to more where the field says so.
 *   - Return value: NNUE_LS_OK or a negative NNUE_LS_ERR_* code; no exceptions
 *     cross this boundary.  nnue_ls_last_error() describes the last failure on
 *     the calling thread.
 */
#ifndef NNUE_LS_H
#define NNUE_LS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NNUE_LS_OK 0
#define NNUE_LS_ERR_INVALID_ARGUMENT (-1) /* null pointer, bad shape, misaligned */
#define NNUE_LS_ERR_UNSUPPORTED (-2)      /* sizes beyond the documented limits */
#define NNUE_LS_ERR_WORKSPACE (-3)        /* workspace null, misaligned or too small */
#define NNUE_LS_ERR_CUDA (-4)             /* a CUDA launch or runtime call failed */

#define NNUE_LS_F32 0
#define NNUE_LS_BF16 1
#define NNUE_LS_F16 2

/* Device error flags (nnue_ls_device_errors). */
#define NNUE_LS_DEVERR_WAIT_TIMEOUT 1u /* a matrix kernel's wait ran out: what it had not formed by then is NaN */
#define NNUE_LS_DEVERR_BAD_INDEX 2u    /* route backward: a chosen index outside [-1, experts) was skipped */

int nnue_ls_version(void);
const char *nnue_ls_last_error(void);
/* Kernels this library has launched in this process. */
uint64_t nnue_ls_launch_count(void);
/* Reads (and with clear != 0 resets) the sticky device error flags of the
 * current device.  Synchronises the device. */
int nnue_ls_device_errors(uint32_t *flags, int clear);
/* How long a matrix kernel launched from now on (by any thread) waits for its
 * own copies and products, which take microseconds, before it gives up: raises
 * the flag, stores NaN for what it has not formed and returns.  4 s at first;
 * more where the GPU may be taken away from the process for longer, 0 to see
 * what giving up looks like (no wait is made and no product formed).  Returns
 * the limit so far. */
uint64_t nnue_ls_set_wait_limit(uint64_t ns);

/* ---- fused linear layer --------------------------------------------------
 *   z = x W^T + bias;  out = act(z) + residual
 * x: [rows, inputs]; weight: [outputs, inputs]; bias: [outputs] or null;
 * residual, out: [rows, outputs] (residual may be null).  1 <= inputs,
 * outputs < 2^30, 0 <= rows < 2^30. */
#define NNUE_LS_ACT_NONE 0
#define NNUE_LS_ACT_RELU 1
#define NNUE_LS_ACT_CRELU 2     /* clamp(z, 0, 1); its derivative is 1 on the closed interval */
#define NNUE_LS_ACT_SQR_CRELU 3 /* clamp(z, 0, 1)^2 */
#define NNUE_LS_ACT_SILU 4
#define NNUE_LS_ACT_GELU 5      /* z * Phi(z), the normal distribution's Phi */

typedef struct {
  int64_t rows, inputs, outputs;
  int32_t dtype;      /* of x, weight, residual, out, act_grad, grad_out, grad_x, grad_weight */
  int32_t bias_dtype; /* of bias and grad_bias: dtype or NNUE_LS_F32 */
  int32_t activation;
  int32_t reserved;
  const void *x, *weight, *bias, *residual;
  int64_t ldx, ldw, ldr;
  void *out;      /* forward; row stride outputs */
  /* Kept from the forward for the backward, each null or placed as nnue_ls_linear_saved_layout() says: act'(z) in a
     form of the library's own (the backward needs it for every activation but NNUE_LS_ACT_NONE), and x and weight
     in the form their products read, which the backward then reads instead. */
  void *act_grad, *x_packed, *weight_packed;
  const void *grad_out; /* backward */
  int64_t ldg;
  void *grad_x, *grad_weight, *grad_bias; /* contiguous; null = not wanted */
} nnue_ls_linear;

/* Where act_grad, x_packed and weight_packed lie in one 256-byte aligned buffer
 * of the returned size; parts: 1, 2 and 4 ask for each.  An offset of -1: not
 * asked for, or the operand is read as it lies and its pointer has to be null. */
size_t nnue_ls_linear_saved_layout(const nnue_ls_linear *a, int32_t parts, int64_t offsets[3]);
size_t nnue_ls_linear_forward_workspace_size(const nnue_ls_linear *a);
int nnue_ls_linear_forward(const nnue_ls_linear *a, void *workspace, size_t workspace_bytes, void *stream);

/* dz = grad_out * act'(z);  grad_x = dz W;  grad_weight = dz^T x;  grad_bias =
 * column sums of dz.  (The residual's gradient is grad_out itself.) */
size_t nnue_ls_linear_backward_workspace_size(const nnue_ls_linear *a);
int nnue_ls_linear_backward(const nnue_ls_linear *a, void *workspace, size_t workspace_bytes, void *stream);

/* ---- norms around a residual block ----------------------------------------
 *   n = norm(f) * post_weight + post_bias     (n = f without post_weight)
 *   y = scale * x + gate * n                  (y = x without f; then y may be null)
 *   h = norm(y) * pre_weight + pre_bias       (only with pre_weight)
 * x, f, y, h: [rows, width], contiguous.  norm(v) = (v - m) / sqrt(mean((v -
 * m)^2) + eps) with m = mean(v) for NNUE_LS_NORM_LAYER and 0 for
 * NNUE_LS_NORM_RMS.  Squares are summed in fp32: a row whose sum passes its range
 * (values from 1.8e19 / sqrt(width) up) becomes NaN.
 * 1 <= width <= NNUE_LS_NORM_MAX_WIDTH. */
#define NNUE_LS_NORM_RMS 0
#define NNUE_LS_NORM_LAYER 1
#define NNUE_LS_GATE_NONE 0
#define NNUE_LS_GATE_ROW 1  /* gate: [rows] */
#define NNUE_LS_GATE_FULL 2 /* gate: [rows, width], in dtype */
#define NNUE_LS_NORM_MAX_WIDTH 65536

typedef struct {
  int64_t rows;
  int32_t width;
  int32_t dtype;        /* of x, f, y, h, a full gate, and their gradients */
  int32_t params_dtype; /* of post_weight ... pre_bias, scale and their gradients: dtype or NNUE_LS_F32 */
  int32_t gate_dtype;   /* of a row gate and its gradient: dtype or NNUE_LS_F32 */
  int32_t kind, gate_mode, gate_sigmoid;
  float scale_value; /* the residual scale when scale is null */
  float eps;
  int32_t reserved;
  const void *x, *f, *gate;
  const void *post_weight, *post_bias, *scale, *pre_weight, *pre_bias;
  void *y, *h;  /* forward */
  float *stats; /* [rows, 4], 16-byte aligned: written by the forward when not null, read by the backward */
  const void *grad_y, *grad_h; /* backward; null = zero */
  void *grad_x, *grad_f, *grad_gate; /* null = not wanted */
  void *grad_post_weight, *grad_post_bias, *grad_scale, *grad_pre_weight, *grad_pre_bias;
} nnue_ls_norm;

int nnue_ls_norm_forward(const nnue_ls_norm *a, void *stream);
size_t nnue_ls_norm_backward_workspace_size(const nnue_ls_norm *a);
int nnue_ls_norm_backward(const nnue_ls_norm *a, void *workspace, size_t workspace_bytes, void *stream);

/* ---- router with its balance loss ------------------------------------------
 * p = softmax(logits) per row; the k largest logits of a row, largest first,
 * ties to the lowest index; gates = their p, divided by their sum with
 * renormalize; counts[e] = how often expert e was chosen;
 *   loss = experts / (k n^2) * sum_e counts[e] * sum_b p[b, e]
 * over the n rows that count: valid[b] != 0 (all rows when valid is null) and
 * some logit other than -inf.  A row that does not count, and a choice beyond
 * the row's logits above -inf, has index -1 and gate 0.  A NaN logit is never
 * chosen and makes the gates of its row's choices and the loss NaN.
 * 1 <= k <= experts <= NNUE_LS_MAX_EXPERTS. */
#define NNUE_LS_MAX_EXPERTS 1024

typedef struct {
  int64_t rows;
  int32_t experts, k, dtype, renormalize;
  const void *logits; /* row stride ld */
  int64_t ld;
  const uint8_t *valid;
  int64_t *indices; /* [rows, k] */
  float *gates;     /* [rows, k] */
  int64_t *counts;  /* [experts] */
  float *loss;      /* [2]: the loss; its unit experts / (k n^2), kept for the backward */
  const float *grad_gates, *grad_loss; /* backward; null = zero */
  void *grad_logits;                   /* [rows, experts] */
} nnue_ls_route;

size_t nnue_ls_route_forward_workspace_size(const nnue_ls_route *a);
int nnue_ls_route_forward(const nnue_ls_route *a, void *workspace, size_t workspace_bytes, void *stream);
/* Reads logits, valid, indices, gates, counts and loss as the forward left them. */
int nnue_ls_route_backward(const nnue_ls_route *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NNUE_LS_H */
