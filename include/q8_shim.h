/*
 * C-ABI of the 8-bit operators for language models in libsgemm_shim.so (gfx950):
 * a linear layer whose product runs in 8-bit integers, the norm before it, and
 * the gradients of both.
 *
 *   q8_rmsnorm           residual added, root-mean-square norm, result in 8 bits
 *   q8_gemm              8-bit product, scales of tokens and channels, bias
 *   q8_grad_input        gradient of the product's input, from the 8-bit weights
 *   q8_grad_weight       gradient of its weights, from the 8-bit activations that
 *                        the forward pass kept (the checkpoint)
 *   q8_rmsnorm_backward  gradients of the norm's input (and residual) and gain
 *   q8_quantize          rows to 8 bits (weights; activations from elsewhere)
 *   q8_dequantize        and back (a checkpoint restored)
 *
 * Conventions (those of sgemm_shim.h where not said otherwise)
 *   - 0 on success, a positive hipError_t, or a negative SGEMM_E_* code, with
 *     sgemm_last_error()'s message.  Nothing throws across this ABI.  A refused
 *     call has launched nothing.
 *   - A matrix of `rows` x `cols` holds row i's values one after the other from
 *     element i * ld (ld >= cols): the column-major cols x rows matrix of the
 *     SGEMM entry points, a token being a column there.  Pointers are aligned
 *     to their element's size; any ld.  Rows and pointers of whole 16 bytes are
 *     the fast ones.  What lies between cols and ld is neither used nor written.
 *   - Types: Q8_F32, Q8_F16, Q8_BF16.  Every sum, norm and scale is computed in
 *     32 bits, and a result rounded once (to nearest, ties to even).
 *   - 8-bit data: int8 values q in -127 .. 127 with one FP32 scale s a row,
 *     standing for q s.  s = max(largest |x| of the row / 127, 2^-126), so a
 *     row of zeros has q = 0.  A row that holds an infinity or a NaN gets s =
 *     NaN and q = 0: all that is computed from it is NaN.  (-128 is taken as an
 *     operand too.)
 *   - Zero rows, columns or products: a call with nothing to write succeeds and
 *     launches nothing; a sum over nothing is 0.
 *   - Outputs may not overlap inputs or one another (SGEMM_E_INVALID), but for
 *     those that an entry point names.
 *   - All work is enqueued on the handle's stream and not waited for.  One
 *     handle is used by one thread at a time.  The products keep a workspace in
 *     the handle, which grows on the first call that needs more (q8_reserve
 *     beforehand); under graph capture it cannot grow, and a call that needs
 *     more is refused with SGEMM_E_SHAPE.  Work of one handle, replays of its
 *     captured calls among it, must run in order.
 * No counterpart in the reference, which multiplies FP32 matrices only.
 */
#ifndef Q8_SHIM_H
#define Q8_SHIM_H

#include "sgemm_shim.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    Q8_F32 = 0,
    Q8_F16 = 1,
    Q8_BF16 = 2
};

/* Calls that q8_workspace_size tells the workspace of. */
enum {
    Q8_CALL_RMSNORM_BACKWARD = 0,
    Q8_CALL_GEMM = 1,
    Q8_CALL_GRAD_INPUT = 2,
    Q8_CALL_GRAD_WEIGHT = 3
};

/* Longest sum of q8_gemm: 131071 products of -128 * -128 fit 32 bits. */
#define Q8_MAX_K 131071u
/* Longest sums of the gradients (n of q8_grad_input, m of q8_grad_weight), with 16-bit types and with Q8_F32:
 * an operand's row laid out for the matrix cores ends at 2^22 bytes.  A longer one is refused with SGEMM_E_SHAPE;
 * q8_grad_weight can add the parts of one with `accumulate`. */
#define Q8_MAX_SUM 2097152u
#define Q8_MAX_SUM_F32 699048u

typedef struct q8_handle q8_handle;

/* A handle on the current device, with a stream of its own. */
int q8_open(q8_handle** out);

/* Waits for the handle's work and releases its stream and workspace. */
void q8_close(q8_handle* h);

/* As sgemm_set_stream: later calls run on `stream` (of the handle's device; the
 * caller keeps it alive), NULL: on the handle's own.  Waits for the work
 * already enqueued, so the old stream must not be capturing. */
int q8_set_stream(q8_handle* h, void* stream);

/* Waits for all work of the handle's stream. */
int q8_synchronize(q8_handle* h);

/* Grows the handle's workspace to `bytes` if it is smaller. */
int q8_reserve(q8_handle* h, size_t bytes);

/* Most workspace that a call of this kind and size takes, whatever its
 * alignment (Q8_CALL_RMSNORM_BACKWARD: m rows of k; n is not used). */
int q8_workspace_size(int call, int dtype, uint32_t m, uint32_t n, uint32_t k, size_t* bytes);

/* Rows of x to 8 bits: q, and scale[rows]. */
int q8_quantize(q8_handle* h, int dtype, const void* x, uint32_t ldx, int8_t* q, uint32_t ldq, float* scale,
                uint32_t rows, uint32_t cols);

/* y = q scale, rounded to `dtype`. */
int q8_dequantize(q8_handle* h, int dtype, const int8_t* q, uint32_t ldq, const float* scale, void* y, uint32_t ldy,
                  uint32_t rows, uint32_t cols);

/* hidden = x + residual, rounded to `dtype`; the norm of hidden as stored,
 *   n_ij = hidden_ij rstd_i gain_j,  rstd_i = (mean_j hidden_ij^2 + eps)^-1/2,
 * in 8 bits: q and scale[rows].  residual may be NULL (hidden = x); hidden and
 * rstd may be NULL where they are not wanted.  hidden may be x or residual
 * itself (same pointer and ld).  The squares are summed in FP32: a row whose
 * sum passes its largest value (4096 values of 2^58) has rstd = 0, and with eps = 0 one whose squares vanish (zeros,
 * or values below 2^-75) has rstd = infinity and scale = NaN.  hidden_ij gain_j is an FP32 value too. */
int q8_rmsnorm(q8_handle* h, int dtype, const void* x, uint32_t ldx, const void* residual, uint32_t ldr,
               const void* gain, void* hidden, uint32_t ldh, int8_t* q, uint32_t ldq, float* scale, float* rstd,
               uint32_t rows, uint32_t cols, float eps);

/* Gradients of q8_rmsnorm from dn, the gradient of n (the rounding to 8 bits is
 * passed through), with u = dn gain and xhat = hidden rstd:
 *   dx_ij = rstd_i (u_ij - xhat_ij mean_j(u_ij xhat_ij)) + dres_ij
 *   dgain_j = sum_i dn_ij xhat_ij      (FP32; the order of the sum is fixed)
 * dres, the gradient that reaches hidden from elsewhere, may be NULL, and so
 * may dgain.  dx, the gradient of x and of the residual alike, may be dn or
 * dres itself (same pointer and ld). */
int q8_rmsnorm_backward(q8_handle* h, int dtype, const void* dn, uint32_t lddn, const void* hidden, uint32_t ldh,
                        const void* gain, const float* rstd, const void* dres, uint32_t lddr, void* dx, uint32_t lddx,
                        float* dgain, uint32_t rows, uint32_t cols);

/* y_ij = sx_i sw_j sum_k qx_ik qw_jk + bias_j for m tokens (qx, m x k), n
 * channels (qw, n x k): exact 32-bit integer sums.  y and bias in `dtype`;
 * bias may be NULL.  k at most Q8_MAX_K; n below 2^28 where m is at most 64. */
int q8_gemm(q8_handle* h, int dtype, const int8_t* qx, uint32_t ldx, const float* sx, const int8_t* qw, uint32_t ldw,
            const float* sw, const void* bias, void* y, uint32_t ldy, uint32_t m, uint32_t n, uint32_t k);

/* dx_ik = sum_j dy_ij sw_j qw_jk: m tokens, n channels, k features; dy (m x n)
 * and dx (m x k) in `dtype`.  The products run on the 16-bit matrix cores with
 * FP32 sums; sw_j qw_jk is rounded to `dtype` for it, to 2^-8 of it in Q8_BF16, in
 * Q8_F16 to 2^-11 of it or 2^-32 of the largest scale.  In Q8_F32 sw_j dy_ij is rounded to FP32 and split into
 * three BF16 terms, which hold all its bits where it is 2^-110 and more, and its steps of 2^-133 below; past FP32's
 * largest value it is infinite. */
int q8_grad_input(q8_handle* h, int dtype, const void* dy, uint32_t lddy, const int8_t* qw, uint32_t ldw,
                  const float* sw, void* dx, uint32_t lddx, uint32_t m, uint32_t n, uint32_t k);

/* dw_jk = sum_i dy_ij sx_i qx_ik, added to what dw holds where `accumulate` is
 * not 0.  dy in `dtype`; dw (n x k) in `out_dtype`: `dtype` or Q8_F32.  Rounding as
 * in q8_grad_input, of sx_i qx_ik. */
int q8_grad_weight(q8_handle* h, int dtype, const void* dy, uint32_t lddy, const int8_t* qx, uint32_t ldx,
                   const float* sx, int out_dtype, void* dw, uint32_t lddw, uint32_t m, uint32_t n, uint32_t k,
                   int accumulate);

#ifdef __cplusplus
}
#endif

#endif /* Q8_SHIM_H */
