/* sdfnn — C ABI of the gated feed-forward block's operators (libsdfnn.so, gfx950): root-mean-square norm, 8-bit products, gated MLP.
 *
 * The block is the pre-norm residual form  h <- h + W_d (act(W_g n) * (W_u n)),  n = norm(h) w:  a training form in fp32 / bf16 / fp16 with
 * its backward pass, and a serving form whose products run on 8-bit integers.  A separate library, as libsdfmesh.so is: the sources of
 * libsdfhip.so do not change with it.
 *
 * Conventions (as include/sdfhip.h): plain C, device pointers and sizes, the HIP stream to launch on; nothing synchronises and nothing is
 * allocated: the caller owns every buffer, workspaces included (sizes from the *_workspace_size queries).  One workspace serves one call at
 * a time: calls on two streams, or two captured graphs that may replay at once, need one each.  Every entry returns 0 on success and a
 * negative code on error, with sdfnn_last_error() (thread-local) saying why; arguments are checked before anything is launched.  No entry
 * uses atomics: results do not change from run to run.
 *
 * Matrices are row-major; a row stride (ld*, in elements) may exceed the row's width, elements of a row are adjacent.  Tensors need their
 * element's alignment; where a product of more than 32 rows (or a backward pass) reads its operands in place - 16-bit rows of a multiple of
 * 8 elements, codes of a multiple of 16 - every row has to start at a 16-byte boundary, and rows have to be less than 8 MiB apart, else the
 * call is refused.  Outputs are contiguous; what lies behind their last row is left as it was.
 */
#ifndef SDFNN_H_
#define SDFNN_H_
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* sdfnn_stream_t; /* hipStream_t */

enum { SDFNN_F32 = 0, SDFNN_BF16 = 1, SDFNN_F16 = 2 };           /* element type of a call's floating tensors */
enum { SDFNN_SILU = 0, SDFNN_GELU = 1, SDFNN_RELU = 2 };         /* z sigmoid(z); z Phi(z) with the error function; max(z, 0) */

int sdfnn_version(void);
const char* sdfnn_last_error(void);

/* ---- root-mean-square norm
 * h = x + residual (residual NULL: h = x);  inv = 1 / sqrt(mean(h^2) + eps);  y = h inv weight, all in fp32 from the unrounded sum
 * (a row with values beyond 1e19 overflows its sum of squares, as in fp32 anywhere: inv = 0).
 * x, residual [rows, dim] with strides ldx / ldr; weight [dim]; y, h [rows, dim] contiguous (h: only with a residual, may be NULL);
 * inv [rows] fp32, what the backward reads (may be NULL). */
int sdfnn_rms_norm_forward(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int32_t dtype, int64_t rows,
                           int64_t dim, float eps, void* y, void* h, float* inv, sdfnn_stream_t stream);
/* dy (stride lddy) and, for a caller that uses h, dh (stride lddh, or NULL); either may be NULL, not both.  dx [rows, dim] contiguous is the gradient of x AND of
 * residual; dweight [dim].  Either output may be NULL.  workspace: sdfnn_rms_norm_backward_workspace_size(rows, dim) bytes. */
int64_t sdfnn_rms_norm_backward_workspace_size(int64_t rows, int64_t dim);
int sdfnn_rms_norm_backward(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, const float* inv,
                            const void* dy, int64_t lddy, const void* dh, int64_t lddh, int32_t dtype, int64_t rows, int64_t dim, void* dx,
                            void* dweight, void* workspace, int64_t workspace_bytes, sdfnn_stream_t stream);
/* The norm with an output in 8 bits: v = h weight, q = round(127 v / max|v|) (half to even) in [-127, 127] and
 * scales [rows] = inv max|v| / 127, so that q scale = y to half a step.  weight NULL: no norm, v = h and inv = 1 - the rows of x quantised
 * as they are (eps is not read).  A row of zeros has scale 0 and codes 0; a row that holds an infinity or a NaN has a scale that is not
 * finite, and what is computed from it is NaN. */
int sdfnn_rms_norm_quantize(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int32_t dtype, int64_t rows,
                            int64_t dim, float eps, int8_t* q, float* scales, void* h, sdfnn_stream_t stream);

/* ---- products of 8-bit integers
 * y[m, n] = (sum_k q[m, k] w[n, k]) sq[m] sw[n] + bias[n]: the sum exact in 32-bit integers (k <= 131072, so that 127 127 k < 2^31; codes
 * of -128 are allowed up to k = 131071), the rest in fp32.  q [rows, k] (stride ldq), w [n, k] (stride ldw), bias [n] fp32 or NULL,
 * y [rows, n] contiguous in `dtype`.  workspace: sdfnn_int8_linear_workspace_size(rows, n, k, projections) bytes. */
int64_t sdfnn_int8_linear_workspace_size(int64_t rows, int64_t n, int64_t k, int32_t projections);
/* Which kernel the product takes, for tests and traces: 256 or 128, the side of its tiles, or 0, the kernel of few rows (-1: refused); *splits (may be
 * NULL): over how many workgroups k is split.  Nothing is launched. */
int32_t sdfnn_int8_product(int64_t rows, int64_t n, int64_t k, int32_t projections, int32_t* splits);
int sdfnn_int8_linear(const int8_t* q, int64_t ldq, const float* sq, const int8_t* w, int64_t ldw, const float* sw, const float* bias,
                      int32_t dtype, int64_t rows, int64_t n, int64_t k, void* y, void* workspace, int64_t workspace_bytes,
                      sdfnn_stream_t stream);
/* Two of them under a gate in one kernel: y = act(gate) * up (projections = 2 in the workspace query). */
int sdfnn_int8_gated_linear(const int8_t* q, int64_t ldq, const float* sq, const int8_t* w_gate, int64_t ldg, const float* s_gate,
                            const int8_t* w_up, int64_t ldu, const float* s_up, int32_t act, int32_t dtype, int64_t rows, int64_t n,
                            int64_t k, void* y, void* workspace, int64_t workspace_bytes, sdfnn_stream_t stream);

/* ---- gated MLP
 * g = x Wg^T, u = x Wu^T, a = act(g) u, y = a Wd^T.  x [rows, dim] (stride ldx), w_gate / w_up [hidden, dim], w_down [out, hidden], all
 * contiguous, y [rows, out] contiguous.  16-bit types: products of those types with fp32 sums; a is rounded to the type before the second
 * product (up to 16 rows it goes there as two numbers of the type that hold twice its bits), and so are the gradients of g
 * and u before theirs (fp16: a hidden value beyond 65504 becomes infinite - up to 16 rows of a forward pass: beyond 131008 - and gradients below 6e-8
 * vanish, as everywhere in that type: scale the loss).  fp32: fp32 instructions up to 64 rows; beyond, every operand as three bf16 parts that
 * hold its 24 bits, six products, fp32 sums (magnitudes below 2^-110 hold fewer bits).  A row with an input that is not finite has no finite result:
 * infinities or NaN as the arithmetic gives them, in fp32 beyond 64 rows NaN alone.
 * saved: sdfnn_gated_saved_size bytes, what the backward needs (act(g) and u act'(g) in fp32, a in the type; fp32 above 64 rows: a and x as
 * their three parts); NULL when none will follow. */
int64_t sdfnn_gated_saved_size(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden);
int64_t sdfnn_gated_workspace_size(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out, int32_t backward);
/* As sdfnn_int8_product, of product `index` of a pass.  Forward: 0 gate and up, 1 down; backward: 0 the gradients of g and u, 1 dx, 2 dw_down,
 * 3 dw_gate and dw_up. */
int32_t sdfnn_gated_product(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out, int32_t backward, int32_t index, int32_t* splits);
int sdfnn_gated_forward(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* w_down, int32_t dtype, int32_t act,
                        int64_t rows, int64_t dim, int64_t hidden, int64_t out, void* saved, void* y, void* workspace,
                        int64_t workspace_bytes, sdfnn_stream_t stream);
/* dy [rows, out] (stride lddy).  dx [rows, dim], dw_gate, dw_up [hidden, dim], dw_down [out, hidden] are overwritten; each may be NULL
 * (dw_gate and dw_up together). */
int sdfnn_gated_backward(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* w_down, const void* saved,
                         const void* dy, int64_t lddy, int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out, void* dx,
                         void* dw_gate, void* dw_up, void* dw_down, void* workspace, int64_t workspace_bytes, sdfnn_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* SDFNN_H_ */
