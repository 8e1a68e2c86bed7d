/*
 * gsr_linear.h -- C ABI of libgsr's fused matrix products: a linear layer with its bias,
 * activation and residual in the product's epilogue, and a gated pair of products.  They are what
 * a feature head is made of: render() returns a 3-channel feature per pixel
 * (gaussian_renderer/__init__.py:280-326), the head maps it to the wide space it stands for.
 *
 * Shapes: x [M,K], w [N,K] (row n holds output n's weights), bias [N], residual / y / dy [M,N].
 * dtype is one of GSR_F32 / GSR_F16 / GSR_BF16 for every operand of a call; sums and activations
 * are held in 32 bits and each output is rounded once.  GSR_F32 operands below 2^-110 are held to
 * 2^-134, larger ones exactly.  Strides are in elements.
 *   x:  x_row = distance between rows, x_col = distance between columns; one of them is 1
 *       (x_col = 1: rows as they come; x_row = 1: a channel-major image [K,H,W] read in place)
 *   w, residual, y, dy, gradients: rows contiguous, any row stride >= the row's length
 * M = 0 is a no-op (weight gradients are set to zero); K is 1 to 2^22, N 1 to 2^21, M up to 2^36.
 * Every launch goes to `stream` on the current device.  scratch: device memory of the size the
 * matching *_scratch_bytes function gives (NULL for 0), 256-byte aligned, untouched by others until
 * the call's work is done; it holds nothing between calls.  Results do not depend on timing (no atomics).
 * Returns 0, 1 on invalid arguments, 2 on a launch error.
 */
#ifndef GSR_LINEAR_H
#define GSR_LINEAR_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { GSR_F32 = 0, GSR_F16 = 1, GSR_BF16 = 2 };
enum { GSR_ACT_NONE = 0, GSR_ACT_RELU = 1, GSR_ACT_GELU = 2, GSR_ACT_SILU = 3 };

/* y = act(x w^T + bias) + residual.  bias, residual may be NULL.  gelu is the erf form. */
size_t gsr_linear_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N);
int gsr_linear(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
               int64_t x_col, const void* w, int64_t w_row, const void* bias,
               const void* residual, int64_t residual_row, int act, void* y, int64_t y_row,
               void* scratch, void* stream);

/* Gradients of gsr_linear: with z = x w^T + bias (computed again, so a forward keeps nothing)
 * and dz = dy act'(z): dx = dz w [M,K], dw = dz^T x [N,K], dbias = the column sums of dz [N], all
 * contiguous; any of them may be NULL.  The residual's gradient is dy.  16-bit dz of an activation is
 * rounded for the products, not for its sums: in GSR_F16 it is infinite beyond 65504 and 0 up to 2^-25
 * there, and dx and dw are what such factors give.  need_dw: GSR_NEED_DW if dw is going to be asked for (with dbias or
 * not), GSR_NEED_DB if dbias alone, 0 if neither. */
enum { GSR_NEED_DW = 1, GSR_NEED_DB = 2 };
size_t gsr_linear_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N, int act,
                                         int need_dw);
int gsr_linear_backward(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                        int64_t x_col, const void* w, int64_t w_row, const void* bias, int act,
                        const void* dy, int64_t dy_row, void* dx, void* dw, void* dbias,
                        void* scratch, void* stream);

/* h = act(x wg^T + bg) * (x wu^T + bu), both products in one pass over x [M,K] (rows contiguous).
 * bg and bu may be NULL. */
size_t gsr_gated_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N);
int gsr_gated(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
              const void* wg, const void* wu, int64_t w_row, const void* bg, const void* bu,
              int act, void* h, int64_t h_row, void* scratch, void* stream);

/* Gradients of gsr_gated (g, u computed again): dg = dh u act'(g), du = dh act(g);
 * dx = dg wg + du wu [M,K]; dw [2N,K] = the gradients of wg and then wu; db [2N] likewise.  Any of
 * them may be NULL.  need_dw as above. */
size_t gsr_gated_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N, int need_dw);
int gsr_gated_backward(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                       const void* wg, const void* wu, int64_t w_row, const void* bg,
                       const void* bu, int act, const void* dh, int64_t dh_row, void* dx, void* dw,
                       void* db, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GSR_LINEAR_H */
