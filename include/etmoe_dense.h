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

#ifdef __cplusplus
}
#endif

#endif /* ETMOE_DENSE_H */
