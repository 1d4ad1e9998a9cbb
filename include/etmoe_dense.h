/*
 * etmoe_dense.h -- C ABI of the operators on the dense matrices beside the routed
 * experts of etmoe.h, in the same library (libetmoe.so): the gated projection of a
 * shared expert, forward and backward; the orthogonalised optimizer step of
 * matrices (Newton-Schulz, batched); and low-rank adapters of many requests
 * beside a shared projection.
 *
 * Conventions are those of etmoe.h: device pointers unless a comment says
 * otherwise, work enqueued on `stream` (NULL: the legacy default stream), no
 * allocation, no synchronisation, 0 or a negative ET_ERR_* code with
 * et_last_error(), argument errors found before anything is enqueued, no
 * state between calls.  Every entry point can be captured in a HIP graph;
 * values passed by value are then fixed in it.
 * No entry point has a counterpart in the reference.
 */
#ifndef ETMOE_DENSE_H
#define ETMOE_DENSE_H

#include "etmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ET_DENSE_ABI_VERSION 1

int et_dense_abi_version(void);

/* ------------------------------------------------------------------------ *
 * The gated projection
 * ------------------------------------------------------------------------ */

#define ET_GATED_SILU 0    /* act(g) = g * sigmoid(g) */
#define ET_GATED_GELU 1    /* act(g) = g * Phi(g), Phi the normal distribution function */

/*
 *   g[t, f] = sum_k x[t, k] * w[f, k],  u[t, f] = sum_k x[t, k] * w[F + f, k]
 *   h[t, f] = act(g[t, f]) * u[t, f]
 * bf16 x [rows, K] with a row stride in elements (a multiple of 8, >= K), bf16 w
 * [2F, K] (the gate rows, then the up rows), bf16 h [rows, F], dense.  Binary32
 * sums in a fixed order, h rounded once: repeated calls give identical bits.  K
 * (below 2^21) and F (below 2^20) are multiples of 8, w is below 2 GiB, every pointer 16-byte aligned.
 */
int et_gated_linear(const void* x, int64_t x_stride, const void* w, int64_t rows, int64_t K, int64_t F, int activation,
                    void* h, void* stream);

/* Bytes of device workspace et_gated_linear_bwd needs (dp, and dW's partial sums
 * where there are few tiles of it; 0 for invalid sizes). */
size_t et_gated_linear_bwd_workspace_bytes(int64_t rows, int64_t K, int64_t F);

/*
 * Backward, from x and w alone (g and u are computed again):
 *   dp[t, f] = dh[t, f] * u[t, f] * act'(g[t, f]),  dp[t, F + f] = dh[t, f] * act(g[t, f])
 *   dx = dp w,  dw = dp^T x
 * dh bf16 [rows, F] and dx bf16 [rows, K], dense; dw [2F, K] of dw_dtype.  dp is
 * rounded to bf16 once, dx and dw (binary32 sums in a fixed order) once.  dx or
 * dw may be NULL.  No rows: dw is 0.
 */
int et_gated_linear_bwd(const void* dh, const void* x, int64_t x_stride, const void* w, int64_t rows, int64_t K, int64_t F,
                        int activation, void* dx, void* dw, int dw_dtype, void* workspace, size_t workspace_bytes,
                        void* stream);

/* ------------------------------------------------------------------------ *
 * Orthogonalised updates of matrices
 * ------------------------------------------------------------------------ */

/* Bytes of device workspace et_orthogonalize and et_muon need for `count` tensors
 * of shapes[3 i] matrices of shapes[3 i + 1] rows and shapes[3 i + 2] columns (HOST
 * array), or for some of them.  0 for invalid shapes, and where no tensor needs any. */
size_t et_orthogonalize_workspace_bytes(const int64_t* shapes, int64_t count);

/*
 * Newton-Schulz steps on every matrix U [m, n] of every tensor:
 *   X = U / (|U| + eps)                              (|U| the Frobenius norm)
 *   `iterations` times:  A = X X^T,  X = (a + b A + c A A) X
 * (with m > n: A = X^T X, X = X (a + b A + c A A), the same), X rounded to bf16.
 * g, out and shapes are HOST arrays: device pointers (element-aligned) to
 * [E, m, n] of `dtype` and bf16.  coefficients (HOST) a, b, c: a > 0, and the
 * polynomial keeps singular values from [0, 1] below 1.9.  The sums are binary32,
 * X, A and the polynomial are held in f16 with 11 bits: the result is 0.1 to 0.2%
 * off in norm.  Fixed order: repeated calls give identical bits.  A matrix
 * that is all zero gives zero; one with a value that is not finite gives NaN,
 * and no other matrix does.  Sides below 65536, a tensor below 2^23 matrices and 2^36
 * elements.  workspace 256-byte aligned.
 */
int et_orthogonalize(const void* const* g, void* const* out, const int64_t* shapes, int64_t count, int dtype,
                     int iterations, const float* coefficients, float eps, void* workspace, size_t workspace_bytes,
                     void* stream);

/* The scalars of one step (passed by value from the host). */
typedef struct {
    float beta, one_minus_beta;
    float decay;                /* 1 - lr * weight_decay */
    float eps;
    float a, b, c;
    int32_t iterations;
    int32_t nesterov;           /* 0 or 1 */
} et_muon_scalars;

/*
 * One optimizer step, in place, on `count` tensors of matrices:
 *   g = grad * grad_scale
 *   m = beta * m + one_minus_beta * g
 *   U = one_minus_beta * g + beta * m  (nesterov), or m
 *   w = decay * w - step_sizes[i] * X   X as above, of U, not rounded to bf16
 * params, grads, momentum (f32), masters and step_sizes are HOST arrays.
 * param_dtype F32: w is the parameter and masters is NULL.  BF16: w is the f32
 * master, and the parameter is w rounded.  grad_scale (f32 [1] on the device) may
 * be NULL (1); where it is not finite every buffer keeps its bits.  Tensors must
 * not overlap.
 */
int et_muon(void* const* params, const void* const* grads, float* const* momentum, float* const* masters,
            const float* step_sizes, const int64_t* shapes, int64_t count, int param_dtype, int grad_dtype,
            et_muon_scalars scalars, const float* grad_scale, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------ *
 * Low-rank adapters of many requests
 * ------------------------------------------------------------------------ */

#define ET_MAX_ADAPTERS 4096
#define ET_MAX_ADAPTER_RANK 128

/* Entries of et_adapter_plan's items (-1 for invalid sizes). */
int64_t et_adapter_plan_items(int64_t num_tokens, int64_t num_adapters);

/*
 * The tokens sorted by adapter, once for all projections of a step.  index
 * [num_tokens]: each token's adapter; a value outside [0, num_adapters) is none.
 * order [num_tokens]; items [et_adapter_plan_items()][4] (16-byte aligned): an
 * adapter (-1: none) and a range of the order; num_items [1].  The order of the
 * tokens of one adapter may change from call to call; it changes no result.
 */
int et_adapter_plan(const int32_t* index, int64_t num_tokens, int64_t num_adapters, int32_t* order, int32_t* items,
                    int32_t* num_items, void* stream);

/* Bytes of device workspace et_adapter_add needs (0 for invalid sizes). */
size_t et_adapter_add_workspace_bytes(int64_t num_tokens, int64_t num_adapters, int64_t K, int64_t rank);

/*
 *   out[t, n] = y[t, n] + sum_r b[i, n, r] * (scale[i] * sum_k a[i, r, k] * x[t, k])
 * with i token t's adapter in the plan (none: out[t] = y[t]).  bf16 x [num_tokens, K],
 * y and out [num_tokens, N] with row strides in elements (multiples of 8), out may
 * be y; bf16 a [num_adapters, rank, K] and b [num_adapters, N, rank], f32 scale
 * [num_adapters].  K, N and rank multiples of 8, rank at most
 * ET_MAX_ADAPTER_RANK.  order, items and num_items are those of et_adapter_plan for the
 * same num_tokens and num_adapters; num_tokens is below 2^27, and the plan's items times
 * N / 1024 (rounded up) below 2^24.  Binary32 sums in a fixed order, the inner one
 * kept to 16 bits, one rounding of out: repeated calls give identical bits.  An
 * inner sum that is not finite gives NaN in its token's row.
 * Pointers 16-byte aligned (scale, order and num_items 4).
 */
int et_adapter_add(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* a, const void* b,
                   const float* scale, const int32_t* order, const int32_t* items, const int32_t* num_items,
                   int64_t num_tokens, int64_t num_adapters, int64_t K, int64_t N, int64_t rank, void* out,
                   int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ETMOE_DENSE_H */
