/*
 * etmoe_block.h -- C ABI of the operators that an MoE block needs around the
 * dispatch path of etmoe.h, in the same library (libetmoe.so): the layer norm
 * before the block, forward and backward; the optimizer step of its weights
 * (AdamW over many tensors at once, with states in 32 or in 8 bits, and the
 * global gradient norm that clips it); and the experts' and a dense layer's
 * products with 4-bit weights, for serving a few tokens at a time.
 *
 * Conventions are those of etmoe.h: device pointers unless a comment says
 * otherwise, work enqueued on `stream` (NULL: the legacy default stream), no
 * allocation, no synchronisation, 0 or a negative ET_ERR_* code with
 * et_last_error(), argument errors found before anything is enqueued, no
 * state between calls.  Every entry point can be captured in a HIP graph;
 * values passed by value are then fixed in it.
 * No entry point has a counterpart in the reference.
 */
#ifndef ETMOE_BLOCK_H
#define ETMOE_BLOCK_H

#include "etmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ET_BLOCK_ABI_VERSION 2      /* 2: the values of a packed 4-bit weight lie three bits further */

int et_block_abi_version(void);

/* ------------------------------------------------------------------------ *
 * Layer norm
 * ------------------------------------------------------------------------ */

/* Longest row of the layer norm (a row is held in one block's registers). */
#define ET_MAX_NORM_WIDTH 16384

/*
 * Layer norm over rows of d elements, with the residual add before it:
 *   h[t, c]  = x[t, c] + residual[t, c], rounded to `dtype`, written to sum
 *              (without a residual: h = x, nothing written)
 *   mean[t]  = sum_c h[t, c] / d
 *   rstd[t]  = 1 / sqrt(sum_c (h[t, c] - mean[t])^2 / d + eps)
 *   y[t, c]  = (h[t, c] - mean[t]) * rstd[t] * weight[c] + bias[c]
 * in binary32 in a fixed order, y rounded once to `dtype`: repeated calls give
 * identical bits.  x and residual [rows, d] of `dtype` with row strides in
 * elements (>= d); sum and y dense.  weight and bias [d] of weight_dtype: that
 * of the rows, or ET_DTYPE_F32.  residual and sum go together, and mean and
 * rstd (f32 [rows], what the backward needs); each pair may be NULL, and
 * bias.  Every pointer element-aligned; 1 <= d <= ET_MAX_NORM_WIDTH.  A NaN or
 * an infinity in a row makes that row's outputs NaN and no other's.  sum may
 * be x or residual, and y may be x or residual, where those rows are dense.
 */
int et_layer_norm_fwd(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                      const void* weight, const void* bias, int64_t rows, int64_t d, int dtype, int weight_dtype,
                      float eps, void* y, void* sum, float* mean, float* rstd, void* stream);

/* Bytes of device workspace et_layer_norm_bwd needs (partial column sums of
 * its blocks; 0 for invalid sizes). */
size_t et_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t d);

/*
 * Backward of the layer norm, with h its input (x or sum of the forward):
 *   xhat = (h - mean) * rstd,  g = dy * weight
 *   dx[t, c]   = rstd[t] * (g - sum_c(g) / d - xhat * sum_c(g * xhat) / d) + dsum[t, c]
 *   dweight[c] = sum_t dy[t, c] * xhat[t, c],  dbias[c] = sum_t dy[t, c]
 * in binary32, dx rounded once to `dtype` and dense, dweight and dbias f32 [d].
 * dy, h and dsum [rows, d] with row strides in elements.  dsum, the gradient
 * that reaches h past the norm (the residual branch), and dbias may be NULL.
 * The column sums are over blocks of rows, then over the blocks, in a fixed order.
 * No rows: dweight and dbias are 0.  workspace 4-byte aligned.
 */
int et_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* h, int64_t h_stride, const void* dsum,
                      int64_t dsum_stride, const void* weight, const float* mean, const float* rstd, int64_t rows,
                      int64_t d, int dtype, int weight_dtype, void* dx, float* dweight, float* dbias,
                      void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------ *
 * AdamW over many tensors
 * ------------------------------------------------------------------------ */

/* Elements that share one scale of the 8-bit states. */
#define ET_ADAMW8_BLOCK 256

/* Bytes of device workspace et_grad_norm needs for `count` tensors of
 * numel[i] elements (HOST array): one binary64 partial sum for every 16384
 * elements of a tensor.  0 where count or a numel is negative. */
size_t et_grad_norm_workspace_bytes(const int64_t* numel, int64_t count);

/*
 * Global 2-norm of many tensors:
 *   norm[0]  = sqrt(sum over every element of g^2)
 *   scale[0] = min(1, max_norm / (norm + 1e-6)); NaN if the norm is not finite
 * grads, numel and dtypes are HOST arrays of `count` entries: device pointers
 * (element-aligned), element counts, ET_DTYPE_*.  Squares and sums are binary64 in a
 * fixed order, norm is rounded once: repeated calls give identical bits.
 * scale (f32 [1]) may be NULL; max_norm is then not read.  workspace 8-byte
 * aligned.
 */
int et_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int64_t count,
                 float max_norm, float* norm, float* scale, void* workspace, size_t workspace_bytes,
                 void* stream);

/* The scalars of one AdamW step (passed by value from the host). */
typedef struct {
    float beta1, one_minus_beta1;   /* each rounded from the host's binary64 value */
    float beta2, one_minus_beta2;
    float inv_root_bias2;           /* 1 / sqrt(1 - beta2^step) */
    float eps;
    float decay;                    /* 1 - lr * weight_decay */
    float step_size;                /* lr / (1 - beta1^step) */
} et_adamw_scalars;

/*
 * One AdamW step, in place, on `count` tensors:
 *   g = grad * grad_scale
 *   m = beta1 * m + one_minus_beta1 * g
 *   v = beta2 * v + one_minus_beta2 * (g * g)
 *   w = decay * w - step_size * (m / (sqrt(v) * inv_root_bias2 + eps))
 * in binary32, each operation of m and v rounded in the order written.
 * params, grads, m, v and masters are HOST arrays of device pointers, numel a
 * HOST array.  param_dtype F32: w is the parameter and masters is NULL.  BF16:
 * w is the f32 master, and the parameter is w rounded to bf16.  m and v f32.
 * grads f32 or bf16 (grad_dtype).  grad_scale (f32 [1] on the device) may be
 * NULL (1).  Where it is not finite the step is skipped: every buffer keeps
 * its bits.  Pointers are element-aligned; a tensor whose pointers are all
 * 16-byte aligned (bf16: 8) moves in wide accesses.  Tensors must not overlap.
 */
int et_adamw(void* const* params, const void* const* grads, float* const* m, float* const* v,
             float* const* masters, const int64_t* numel, int64_t count, int param_dtype, int grad_dtype,
             et_adamw_scalars scalars, const float* grad_scale, void* stream);

/*
 * The same step with 8-bit states.  m and u = sqrt(v) are held as OCP e4m3
 * values, one byte per element, times an f32 scale for every block of
 * ET_ADAMW8_BLOCK consecutive elements of a tensor (the last may be short;
 * m_scale and u_scale have ceil(numel / 256) entries):
 *   m = m8 * m_scale, u = u8 * u_scale, v = u * u
 *   m, v and w stepped as in et_adamw; u = sqrt(v)
 *   a = the largest |x| of the block (x = m, u; below 1e-35: 0)
 *   scale = a * (1 / 448),  r = min(|x| * (448 / a), 448)  (0 where a is 0)
 *   x8 = r rounded to e4m3, with x's sign
 * so the largest element of a block is kept to f32.  rounding 0: to nearest,
 * ties to even.  rounding 1: stochastic, up with the probability of the
 * fraction left out, from 16 random bits: word(seed, i) of element i (counted
 * over the call's tensors, each beginning at a multiple of 256), m from its
 * high half and u from its low one:
 *   x = i * 0x9E3779B1 + seed;           x = (x ^ x >> 15) * 0x6A09E667
 *   x = (x ^ x >> 13) * 0xBB67AE85;      word = x ^ x >> 16       (mod 2^32)
 * A moving average needs it: with 1 - beta2 = 0.001 and steps of 1/8 rounding
 * to nearest returns every value to where it was.  u > 0 is held as 2^-9 of
 * the scale at least, so no denominator falls to eps.  A block whose largest
 * value is not finite gets a NaN scale.  The step's own w uses m and v before
 * they are rounded.
 */
int et_adamw8(void* const* params, const void* const* grads, uint8_t* const* m8, float* const* m_scale,
              uint8_t* const* u8, float* const* u_scale, float* const* masters, const int64_t* numel,
              int64_t count, int param_dtype, int grad_dtype, et_adamw_scalars scalars, const float* grad_scale,
              int rounding, uint32_t seed, void* stream);

/* ------------------------------------------------------------------------ *
 * Products with 4-bit weights and group scales
 * ------------------------------------------------------------------------ */

/* types of the group scales */
#define ET_W4_SCALE_BF16 0
#define ET_W4_SCALE_F16 1

/*
 * A 4-bit weight of E experts (1: a dense layer), N rows (output features) and
 * K columns each:
 *   w[e, n, k] = (q[e, n, k] - 8) * scale[e, n, k / group],  q in 0..15
 * group 32, 64 or 128; the last group of a row may be short.  K a multiple of 8 below
 * 2^22, N below 2^22, N*K below 2^31.  q is given as bytes [E, N, K / 2], the even k in the
 * low half, scales as 16-bit numbers [E, N, ceil(K / group)].
 *
 * et_w4_pack lays both out once in the order in which the product reads them:
 * `packed` of et_w4_packed_bytes bytes and `packed_scales` of
 * et_w4_packed_scales 16-bit numbers, 16-byte aligned.  parts 2 lays the first and the
 * second half of the rows out each for itself, as SwiGLU's gate and up rows
 * need it (N a multiple of 8 for each part); 1 else.  The layout is that of
 * one ET_BLOCK_ABI_VERSION.  Sizes are 0 for invalid arguments.
 */
size_t et_w4_packed_bytes(int64_t num_experts, int64_t N, int64_t K, int64_t parts);
size_t et_w4_packed_scales(int64_t num_experts, int64_t N, int64_t K, int64_t group, int64_t parts);
int et_w4_pack(const void* q, const void* scales, int64_t num_experts, int64_t N, int64_t K, int64_t group,
               int64_t parts, void* packed, void* packed_scales, void* stream);

/*
 * 4-bit weights of a weight w [E, N, K] (ET_DTYPE_*), group by group:
 *   scale = max(largest / 7, -smallest / 8) (0 counts), rounded to scale_type
 *   q     = 8 + w / scale rounded to nearest, held to 0..15  (8 where scale is 0)
 * A group with a value (or a scale) that is not finite gets a NaN scale.  q 4-byte
 * aligned.
 */
int et_w4_quantize(const void* w, int dtype, int64_t num_experts, int64_t N, int64_t K, int64_t group,
                   int scale_type, void* q, void* scales, void* stream);

/*
 * The weight as bf16 [E, N, K] (16-byte aligned), each value rounded once, of
 * the experts with slots below slot_capacity; of all with expert_offsets NULL.
 * The other experts' rows are left as they were.  With it, batches of many
 * slots per expert run through et_expert_gemm.
 */
int et_w4_unpack(const void* packed, const void* packed_scales, int scale_type, const int32_t* expert_offsets,
                 int64_t num_experts, int64_t N, int64_t K, int64_t group, int64_t parts, int64_t slot_capacity,
                 void* w, void* stream);

/*
 * The expert grouped GEMM of et_expert_gemm on 4-bit weights:
 *   p[s, n] = sum over groups g of scale[e(s), n, g] *
 *             sum over k in g of a[row(s), k] * (q[e(s), n, k] - 8)
 * and c[s, :] = the epilogue of p[s, :], rounded once to bf16.  row(s), the modes (gather with
 * sorted_token, slot-major with NULL), slot_capacity, the epilogues and c are
 * those of et_expert_gemm; ET_GEMM_SWIGLU needs parts 2.  expert_offsets NULL
 * (with one expert and sorted_token NULL) is the dense layer: every slot below
 * slot_capacity.  Binary32 sums in a fixed order: repeated calls give
 * identical bits.  The inner sum is taken as sum a * (16 + q) from
 * -24 * sum a on, so a row of a that holds an infinity (or values whose
 * 24 |a| add up to 2^128 within a group) gives NaN.  a and c 16-byte aligned.
 * slot_capacity may be larger than the slots (T * E where no count is read back): which kernel
 * runs is then decided on the device, by expert_offsets[num_experts].
 * Implements a 4-bit form of the expert GEMM (no reference counterpart).
 */
int et_expert_gemm_w4(const void* a, int64_t a_rows, const int32_t* sorted_token, const void* packed,
                      const void* packed_scales, int scale_type, const int32_t* expert_offsets,
                      int64_t num_experts, int64_t K, int64_t N, int64_t group, int64_t parts,
                      int64_t slot_capacity, int epilogue, const float* row_scale, void* c, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ETMOE_BLOCK_H */
