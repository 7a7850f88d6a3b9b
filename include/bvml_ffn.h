/*
 * bvml_ffn.h -- C ABI of the MI355X (gfx950) feed-forward operators: the
 * feed-forward half of a pre-norm transformer block, forward and backward.
 *
 *   add_rms_norm   s = x + r;  y = s / sqrt(mean(s^2) + eps) * w
 *   linear         y = act(x W^T + b) + r
 *   gated          h = act(x Wg^T + bg) * (x Wu^T + bu),  W = [Wg; Wu]
 *
 * For transformer blocks that a program runs beside the DSINE path, which uses
 * none of them.  The reference composes such blocks from brotensor ops; these
 * fused forms have no counterpart in it.
 *
 * Every matrix is row-major with its rows `ld` elements apart and the elements
 * of a row adjacent, at most 2^23 - 256 bytes from row to row; no alignment is
 * required (16-byte aligned rows take the fastest kernels).  Plain pointers and scalars only: every pointer is a device
 * pointer, every call is asynchronous on `stream` (NULL = the null stream),
 * allocates nothing, keeps nothing, and nothing throws.  Calls can be captured
 * into a HIP graph.  Equal inputs give equal bits.
 *
 * Sums, statistics and activations are fp32 whatever the types; a result is
 * rounded once, to nearest even, when it is stored.
 *
 * A workspace holds at least what the operator's *_workspace function says,
 * overlaps no other argument and, but for the norm's, begins on 16 bytes.
 *
 * Return value: 0 on success; a negative BVML_FFN_E* code for a rejected
 * argument (nothing is launched); a positive hipError_t value when the HIP
 * runtime reports an error at launch, or hipErrorOutOfMemory when the host has
 * no memory for a message.  bvml_ffn_last_error() returns the
 * calling thread's message for the last non-zero status.
 */
#ifndef BVML_FFN_H
#define BVML_FFN_H

#ifdef __cplusplus
extern "C" {
#endif

#define BVML_FFN_OK 0
#define BVML_FFN_ENULL (-1)   /* a required pointer is NULL */
#define BVML_FFN_ESHAPE (-2)  /* a negative size, a width below 1 or rows closer than their width */
#define BVML_FFN_ETYPE (-3)   /* a type or a mixture of types the operator does not take */
#define BVML_FFN_ESIZE (-4)   /* a size beyond the kernels' index range */
#define BVML_FFN_EALIAS (-5)  /* an output or the workspace overlaps another argument */
#define BVML_FFN_EPARAM (-6)  /* eps negative or not finite in fp32, an unknown activation */
#define BVML_FFN_EWORK (-7)   /* the workspace is missing, too small or not on 16 bytes */

/* Element types. */
#define BVML_FFN_F32 0
#define BVML_FFN_F16 1
#define BVML_FFN_BF16 2
#define BVML_FFN_E4M3 3 /* 8 bits: 4 of exponent, 3 of mantissa, no infinities, largest 448 */

/* Activations. */
#define BVML_FFN_NONE 0
#define BVML_FFN_RELU 1
#define BVML_FFN_GELU 2      /* x Phi(x) */
#define BVML_FFN_GELU_TANH 3 /* 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) */
#define BVML_FFN_SILU 4      /* x / (1 + exp(-x)) */

/*
 * s = x + residual (x alone when residual is NULL);
 * y = s * rstd * weight, rstd = 1 / sqrt(mean(s^2) + eps); weight may be NULL
 * (ones).  rows x cols, cols 1..32768.
 *   x_type      F32, F16 or BF16: x, residual and stream_out
 *   w_type      F32 or x_type
 *   y_type      x_type, or F16 / BF16 (from F32), or E4M3
 *   stream_out  s rounded to x_type, or NULL; may be x or residual (same rows)
 *   scale       (rows) fp32, with E4M3 only: y = q * scale,
 *               scale = max(max|y| / 448, 2^-126), q = y / scale to nearest
 *   rstd        (rows) fp32, or NULL: kept for the backward pass
 * A row with a NaN or an infinity in s has NaN where the formula has; in E4M3
 * its scale is NaN or infinite with it.  y is formed from the unrounded s.  The
 * mean of squares is fp32's: a finite s beyond 1.8e19 makes rstd, and y, 0.
 */
int bvml_ffn_add_rms_norm(const void* x, long long ldx, const void* residual, long long ldr,
                          const void* weight, int rows, int cols, double eps, int x_type,
                          int w_type, int y_type, void* y, long long ldy, void* stream_out,
                          long long lds, float* scale, float* rstd, void* stream);

/*
 * The gradient of add_rms_norm: with n = s * rstd and a = dy * weight,
 *   ds = rstd (a - n mean(a n)) + dstream    the gradient of x and of residual
 *   dweight = sum over rows of dy n          of w_type, or NULL
 * dstream (the stream's own gradient) may be NULL.  s and ds are of s_type,
 * dy of dy_type (F32, F16 or BF16).  ds may be dstream (same rows).
 */
int bvml_ffn_add_rms_norm_backward(const void* dy, long long lddy, const void* s, long long lds,
                                   const void* weight, const float* rstd, const void* dstream,
                                   long long lddst, int rows, int cols, int dy_type, int s_type,
                                   int w_type, void* ds, long long ldds, void* dweight,
                                   void* workspace, long long workspace_bytes, void* stream);
long long bvml_ffn_add_rms_norm_backward_workspace(int rows, int cols);

/*
 * y = act(z) + residual, z = x W^T + bias; x (M, K), W (N, K), y (M, N).
 *   in_type   F16 or BF16: x and W.  E4M3: x and W with x_scale (M) and
 *             w_scale (N), z = x W^T * x_scale * w_scale + bias
 *   out_type  in_type or F32 (from E4M3: F16, BF16 or F32): y and residual
 *   bias_type F32, out_type or in_type (16 bits); bias may be NULL
 *   residual  may be NULL, or y itself (same rows)
 *   z         the pre-activations in in_type for the backward pass, or NULL
 *             (NULL with E4M3)
 */
int bvml_ffn_linear(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                    const float* x_scale, const float* w_scale, const void* residual,
                    long long ldr, int M, int N, int K, int in_type, int out_type, int bias_type,
                    int act, void* y, long long ldy, void* z, long long ldz, void* workspace,
                    long long workspace_bytes, void* stream);
/* Bytes of workspace for these sizes, whatever the pointers (0 for most). */
long long bvml_ffn_linear_workspace(int M, int N, int K, int in_type);

/*
 * h = act(g) * u, [g u] = x [Wg; Wu]^T + bias; x (M, K), W (2N, K), h (M, N).
 * As linear, without a residual; bias and w_scale hold 2N, z (M, 2N).
 */
int bvml_ffn_gated(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                   const float* x_scale, const float* w_scale, int M, int N, int K, int in_type,
                   int out_type, int bias_type, int act, void* h, long long ldh, void* z,
                   long long ldz, void* workspace, long long workspace_bytes, void* stream);
long long bvml_ffn_gated_workspace(int M, int N, int K, int in_type);

/*
 * The gradients of linear, in `type` (F16 or BF16, x's and W's): with
 * dz = dy act'(z) rounded to `type` for the products,
 *   dx = dz W (M, K);  dw = dz^T x (N, K);  db = sum over rows of dz (N).
 * Any of the three may be NULL.  dy is of dy_type (`type` or F32); z may be
 * NULL with act NONE.  The residual's gradient is dy itself.  With F16 dz ends
 * at 65504 and below 2^-25 it is 0, from an F32 dy too: scale the loss for it.
 */
int bvml_ffn_linear_backward(const void* dy, long long lddy, const void* x, long long ldx,
                             const void* w, long long ldw, const void* z, long long ldz, int M,
                             int N, int K, int type, int dy_type, int act, void* dx,
                             long long lddx, void* dw, long long lddw, void* db, void* workspace,
                             long long workspace_bytes, void* stream);
long long bvml_ffn_linear_backward_workspace(int M, int N, int K);

/*
 * The gradients of gated from the saved z = [g u] (M, 2N): with
 * dz = [dh u act'(g), dh act(g)], dx (M, K), dw (2N, K), db (2N).
 */
int bvml_ffn_gated_backward(const void* dh, long long lddh, const void* x, long long ldx,
                            const void* w, long long ldw, const void* z, long long ldz, int M,
                            int N, int K, int type, int dh_type, int act, void* dx,
                            long long lddx, void* dw, long long lddw, void* db, void* workspace,
                            long long workspace_bytes, void* stream);
long long bvml_ffn_gated_backward_workspace(int M, int N, int K);

/*
 * The kernel a product of C (M, R) over K takes, without launching: *tile
 * receives its rows of C a workgroup (256, 128, 64; 0: the few-rows kernel),
 * *deep 1 for the tiles with four LDS slots (128 x 128; 64 x 64, two without
 * aligned), *whole the tiles that one workgroup sums, *splits the workgroups
 * that share each of the others; any of them may be NULL.  layout 0: the
 * forward product (R = N, or 2N when gated), 1: the input's gradient, 2: the
 * weight's; 3: both at once from dz (M, R) for x (M, K), *whole and *splits of
 * the one whose sums are split.  aligned: whether every operand row begins on
 * 16 bytes and is whole pieces of them (3: taken as given).  For tests and
 * tuning.
 */
int bvml_ffn_plan(int M, int R, int K, int in_type, int layout, int gated, int aligned, int* tile,
                  int* deep, int* whole, int* splits);

const char* bvml_ffn_last_error(void);
const char* bvml_ffn_version(void);

#ifdef __cplusplus
}
#endif

#endif /* BVML_FFN_H */
