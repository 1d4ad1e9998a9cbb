// et_ortho.hip -- Newton-Schulz orthogonalisation of batches of matrices, and the
// optimizer step that takes it for its direction (gfx950).
//
//   X = U / (|U| + eps);  steps times:  A = X X^T,  S = a I + b A + c A A,  X = S X
//
// (X X^T over the shorter side: for more rows than columns A = X^T X and X = X S.)
// The matrices of many tensors go through one launch a product, each tile finding
// its matrix in a table.  64 matrices of 1024 x 2048: X X^T 172 us, S 129 (the tiles on and above
// the diagonal alone), S X 268, 1.0, 0.67 and 1.03 PFLOP/s of what is computed.
//
// Number format.  X, A and S are held in f16 times fixed powers of two and
// multiplied on the matrix units with binary32 sums.  The largest singular value
// of X stays below 1.9 and that of S below 1.01 a, for the coefficients that the host
// accepts, so no entry of X, A or S is larger than 1.9, 3.61 or 1.01 a: X and A times 2^14 and S
// times the largest power of two that keeps a below 60000 stay below f16's largest
// number, 65504, and entries down to 2^-28 keep all 11 bits.  A bf16
// number has 8 bits, and rounding errors of X grow by a in each step where a
// singular value is still small: with bf16 operands the result is 1 to 2% off, with
// f16 0.1 to 0.2%, about the rounding of a bf16 result (measured on gradients of
// full and of low rank, 64 to 1024 rows).  Operands split in two would cost three
// products for one.
#include "et_dense_gemm.hpp"
#include "etmoe_dense.h"

namespace et {
namespace {

constexpr int kScaleX = 14;                  // X and A are held times 2^14
constexpr int kChunk = 4096;                 // elements a block of the elementwise kernels takes
constexpr int64_t kSums = 1024;              // partial sums of a matrix's norm, which every block of the next kernel adds
constexpr int kTensors = 20;                 // tensors of one launch

float pow2(int e) { return std::ldexp(1.0f, e); }

// --------------------------------------------------------------------------
// momentum, norm and scaling
// --------------------------------------------------------------------------

// A tensor of E matrices [m, n], its momentum and its place in the workspace
// (X [E, m, ldx], columns n .. ldx - 1 zero).
struct OrthoTensor {
    const void* g;
    float* mom;               // null: U = g
    uint16_t* x;
    double* partial;          // [E, sums]
    void* out;                // bf16 result, or the parameter
    float* master;
    uint32_t m, n, ldx;
    uint32_t sums;            // partial sums a matrix
    uint32_t first, each;     // first block and blocks a matrix
    float step;               // of the update
    uint32_t wide;            // matrices begin and rows end at multiples of 8 elements, 16-byte aligned
};

struct OrthoList {
    OrthoTensor t[kTensors];
    int count;
    const float* grad_scale;
    float beta, one_minus_beta, eps, decay;
    int nesterov;
};
static_assert(sizeof(OrthoList) <= 4096, "kernel arguments");

__device__ __forceinline__ int tensor_of(const OrthoList& list, uint32_t block)
{
    int i = 0;
    while (i + 1 < list.count && list.t[i + 1].first <= block) ++i;
    return i;
}

template <typename T>
__device__ __forceinline__ float read1(const void* p, int64_t i)
{
    if constexpr (sizeof(T) == 4) return ((const float*)p)[i];
    else return u2f((uint32_t)((const uint16_t*)p)[i] << 16);
}

template <typename T>
__device__ __forceinline__ void read8(const void* p, int64_t i, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        const f32x4_t* q = reinterpret_cast<const f32x4_t*>((const float*)p + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = q[e >> 2][e & 3];
    } else {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>((const uint16_t*)p + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e & 1 ? bf16hi(w[e >> 1]) : bf16lo(w[e >> 1]);
    }
}

__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double part[4];
    v = wave_sum_dpp_f64(v);
    if (lane_id() == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

// U of one element, and (WRITE) the momentum's new value.
__device__ __forceinline__ float direction(const OrthoList& l, float g, float& mom)
{
    mom = l.beta * mom + l.one_minus_beta * g;
    return l.nesterov ? l.one_minus_beta * g + l.beta * mom : mom;
}

// Momentum, and a block's sum of squares of U.  A step whose grad_scale is not
// finite leaves the momentum as it is.
template <typename G, bool MOM>
__global__ __launch_bounds__(kDenseThreads) void ortho_norm_kernel(OrthoList l)
{
    const OrthoTensor& t = l.t[tensor_of(l, blockIdx.x)];
    const uint32_t b = blockIdx.x - t.first;
    const uint32_t e = b / t.each, c = b - e * t.each;
    if (c >= t.sums) return;
    const int64_t size = (int64_t)t.m * t.n, base = e * size;
    float scale = 1.0f;
    if (MOM && l.grad_scale) {
        scale = *l.grad_scale;
        if (!(__builtin_fabsf(scale) < __builtin_inff())) return;
    }
    double sum = 0.0;
    for (int64_t at0 = (int64_t)c * kChunk; at0 < size; at0 += (int64_t)t.sums * kChunk) {
        if (t.wide) {
#pragma unroll
            for (int i = 0; i < kChunk / (8 * kDenseThreads); ++i) {
                const int64_t at = at0 + (i * kDenseThreads + (int)threadIdx.x) * 8;
                if (at >= size) break;
                float v[8];
                read8<G>(t.g, base + at, v);
                if constexpr (MOM) {
                    f32x4_t* const q = reinterpret_cast<f32x4_t*>(t.mom + base + at);
                    f32x4_t m[2] = {q[0], q[1]};
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float w = m[j >> 2][j & 3];
                        v[j] = direction(l, v[j] * scale, w);
                        m[j >> 2][j & 3] = w;
                    }
                    q[0] = m[0];
                    q[1] = m[1];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += (double)v[j] * (double)v[j];
            }
        } else {
            // (all loads before the first sum)
            constexpr int N = kChunk / kDenseThreads;
            float v[N], w[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t at = base + min(at0 + i * kDenseThreads + (int)threadIdx.x, size - 1);
                v[i] = read1<G>(t.g, at);
                if constexpr (MOM) w[i] = t.mom[at];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t at = at0 + i * kDenseThreads + (int)threadIdx.x;
                if (at >= size) break;
                if constexpr (MOM) {
                    v[i] = direction(l, v[i] * scale, w[i]);
                    t.mom[base + at] = w[i];
                }
                sum += (double)v[i] * (double)v[i];
            }
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) t.partial[(int64_t)e * t.sums + c] = sum;
}

// X = U / (|U| + eps) in f16 times 2^14, from U's matrix's sums and U again (of the
// momentum as it is now).
template <typename G, bool MOM>
__global__ __launch_bounds__(kDenseThreads) void ortho_scale_kernel(OrthoList l)
{
    const OrthoTensor& t = l.t[tensor_of(l, blockIdx.x)];
    const uint32_t b = blockIdx.x - t.first;
    const uint32_t e = b / t.each, c = b - e * t.each;
    const int64_t base = (int64_t)e * t.m * t.n;
    float gs = 1.0f;
    if (MOM && l.grad_scale) {
        gs = *l.grad_scale;
        if (!(__builtin_fabsf(gs) < __builtin_inff())) return;
    }
    // (With a momentum all of U is loaded first, on its way while the norm is summed: 64 x 512
    // x 2048 f32, this and the last kernel 20 us less of 676 each.  A bf16 gradient alone is
    // better taken piece by piece: 64 x 1024 x 2048 90 us, 112 at once.)
    constexpr int N = kChunk / (8 * kDenseThreads);
    const uint32_t row_segs = t.ldx / 8, segs = t.m * row_segs;
    float v[N][8];
    const auto load = [&](int i) {
        const uint32_t seg = min(c * (kChunk / 8) + i * kDenseThreads + threadIdx.x, segs - 1);
        const uint32_t row = seg / row_segs, col = (seg - row * row_segs) * 8;
        const int64_t at = base + (int64_t)row * t.n + col;
        float m[8];
        if (t.wide) {
            read8<G>(t.g, at, v[i]);
            if constexpr (MOM) read8<float>(t.mom, at, m);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t from = base + (int64_t)row * t.n + min(col + j, t.n - 1);
                v[i][j] = read1<G>(t.g, from);
                if constexpr (MOM) m[j] = t.mom[from];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (MOM) v[i][j] = l.nesterov ? l.one_minus_beta * (v[i][j] * gs) + l.beta * m[j] : m[j];
            if (col + j >= t.n) v[i][j] = 0.0f;
        }
    };
    if constexpr (MOM) {
#pragma unroll
        for (int i = 0; i < N; ++i) load(i);
    }
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < t.sums; i += kDenseThreads) sum += t.partial[(int64_t)e * t.sums + i];
    sum = block_sum(sum);
    // (in binary64: the norm of values near binary32's smallest or largest is in its range)
    // (a matrix of zeros stays one, without eps too)
    const double inv = sum == 0.0 ? 0.0 : (double)(1 << kScaleX) / (sqrt(sum) + (double)l.eps);
    uint16_t* const x = t.x + (int64_t)e * t.m * t.ldx;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t seg = c * (kChunk / 8) + i * kDenseThreads + threadIdx.x;
        if (seg >= segs) break;
        if constexpr (!MOM) load(i);
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_f16x2((float)(v[i][2 * j] * inv), (float)(v[i][2 * j + 1] * inv));
        *reinterpret_cast<u32x4_t*>(x + (int64_t)seg * 8) = w;
    }
}

// The result: bf16 out = X, or the update w = decay w - step X of f32 parameters, or
// of bf16 ones with f32 masters.
enum { kOutBf16 = 0, kOutParam = 1, kOutMaster = 2 };
template <int OUT>
__global__ __launch_bounds__(kDenseThreads) void ortho_finish_kernel(OrthoList l)
{
    const OrthoTensor& t = l.t[tensor_of(l, blockIdx.x)];
    const uint32_t b = blockIdx.x - t.first;
    const uint32_t e = b / t.each, c = b - e * t.each;
    if (OUT != kOutBf16 && l.grad_scale && !(__builtin_fabsf(*l.grad_scale) < __builtin_inff())) return;
    const int64_t base = (int64_t)e * t.m * t.n;
    const uint32_t row_segs = t.ldx / 8, segs = t.m * row_segs;
    const uint16_t* const x = t.x + (int64_t)e * t.m * t.ldx;
    const float unit = 1.0f / (1 << kScaleX), step = t.step * unit;
    float* const w = OUT == kOutMaster ? t.master : (float*)t.out;
    constexpr int N = kChunk / (8 * kDenseThreads);
    f16x8_t v[N];
    float p[N][8];
    int64_t at[N];
    uint32_t cols[N];         // that there are; 0: none of the block's
    const auto load = [&](int i) {
        const uint32_t seg = c * (kChunk / 8) + i * kDenseThreads + threadIdx.x, held = min(seg, segs - 1);
        const uint32_t row = held / row_segs, col = (held - row * row_segs) * 8;
        cols[i] = seg < segs ? min(t.n - col, 8u) : 0u;
        at[i] = base + (int64_t)row * t.n + col;
        v[i] = *reinterpret_cast<const f16x8_t*>(x + (int64_t)held * 8);
        if constexpr (OUT != kOutBf16) {
            if (t.wide) {
                read8<float>(w, at[i], p[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[i][j] = w[at[i] + min((uint32_t)j, t.n - 1 - col)];
            }
        }
    };
    // (the loads of a parameter first, as in ortho_scale_kernel)
    if constexpr (OUT != kOutBf16) {
#pragma unroll
        for (int i = 0; i < N; ++i) load(i);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (OUT == kOutBf16) load(i);
        if (cols[i] == 0) break;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            p[i][j] = OUT == kOutBf16 ? (float)v[i][j] * unit : __builtin_fmaf(-step, (float)v[i][j], l.decay * p[i][j]);
        if (t.wide) {
            if constexpr (OUT != kOutBf16) {
                f32x4_t* const q = reinterpret_cast<f32x4_t*>(w + at[i]);
                q[0] = f32x4_t{p[i][0], p[i][1], p[i][2], p[i][3]};
                q[1] = f32x4_t{p[i][4], p[i][5], p[i][6], p[i][7]};
            }
            if constexpr (OUT != kOutParam) {
                u32x4_t o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(p[i][2 * j], p[i][2 * j + 1]);
                *reinterpret_cast<u32x4_t*>((uint16_t*)t.out + at[i]) = o;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((uint32_t)j < cols[i]) {
                    if constexpr (OUT != kOutBf16) w[at[i] + j] = p[i][j];
                    if constexpr (OUT != kOutParam) ((uint16_t*)t.out)[at[i] + j] = (uint16_t)f32_to_bf16_bits(p[i][j]);
                }
        }
    }
}

// --------------------------------------------------------------------------
// small matrices: everything in one block
// --------------------------------------------------------------------------

// A matrix whose shorter side r is at most 64 and which fits into LDS in f16 is
// taken by one block from its gradient to its result: X [r][c], A and S stay in LDS,
// rows 16 bytes apart from a multiple of 64, so that 16 rows' segments fall on
// all banks.  X = S X goes column by column: a wave replaces 16 columns of X by
// their own product, in place.  The products above launch 17 kernels for the same
// (three layers' routers and 8 experts of 64 x 512 and 512 x 32: 227 us, here 35).
constexpr int kFusedThreads = 512, kFusedWaves = kFusedThreads / kWave;
constexpr int kFusedSide = 64;
constexpr int kFusedSmall = 30 * 1024, kFusedLarge = 150 * 1024;     // bytes of LDS: four blocks a CU, or one

__host__ __device__ inline int64_t round_to(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct FusedLayout {
    int r16, ldx, lds;        // rows; elements from a row to the next of X, and of A and S
    int64_t bytes;
};
__host__ __device__ inline FusedLayout fused_layout(int64_t r, int64_t c)
{
    FusedLayout f;
    f.r16 = (int)round_to(r, 16);
    f.ldx = (int)round_to(c, 32) + 8;
    f.lds = (int)round_to(r, 32) + 8;
    f.bytes = ((int64_t)f.r16 * f.ldx + 2 * (int64_t)f.r16 * f.lds) * 2;
    return f;
}

struct FusedScalars {
    float alpha_a, alpha_s, beta_s, gamma_s, alpha_x;
    int iterations;
};

// How a matrix's elements go by fours: in a row of X, down a column of it, one by one.
enum { kLines = 0, kTall = 1, kOdd = 2 };

template <typename G, bool MOM, int OUT, int LDS_BYTES>
__global__ __launch_bounds__(kFusedThreads) void ortho_fused_kernel(OrthoList l, FusedScalars q)
{
    __shared__ __attribute__((aligned(16))) unsigned char smem[LDS_BYTES];
    __shared__ double part[kFusedWaves];
    __shared__ f32x4_t sums[kFusedWaves][kWave];
    const OrthoTensor& t = l.t[tensor_of(l, blockIdx.x)];
    const int m = (int)t.m, n = (int)t.n, size = m * n;
    const bool tall = m > n;
    const int c = max(m, n);
    const FusedLayout f = fused_layout(min(m, n), c);
    const int64_t base = (int64_t)(blockIdx.x - t.first) * size;
    float gs = 1.0f;
    if (MOM && l.grad_scale) {
        gs = *l.grad_scale;
        if (!(__builtin_fabsf(gs) < __builtin_inff())) return;
    }
    const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
    const int r16 = lane & 15, rho = lane >> 4;
    uint16_t* const X = (uint16_t*)smem;
    uint16_t* const A = X + f.r16 * f.ldx;
    uint16_t* const S = A + f.r16 * f.lds;
    // Elements go by groups of four, group tid + 512 i to a thread.
    const auto load4 = [&](auto mode, const void* p, auto type, int at, float (&v)[4]) {
        using T = decltype(type);
        if constexpr (decltype(mode)::value != kOdd) {
            if constexpr (sizeof(T) == 4) {
                const f32x4_t w = *reinterpret_cast<const f32x4_t*>((const float*)p + base + min(at, size - 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = w[e];
            } else {
                const u32x2_t w = *reinterpret_cast<const u32x2_t*>((const uint16_t*)p + base + min(at, size - 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = e & 1 ? bf16hi(w[e >> 1]) : bf16lo(w[e >> 1]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = read1<T>(p, base + min(at + e, size - 1));
        }
    };
    const auto store4 = [&](auto mode, float* p, int at, const float (&v)[4]) {
        if constexpr (decltype(mode)::value != kOdd) {
            *reinterpret_cast<f32x4_t*>(p + base + at) = f32x4_t{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at + e < size) p[base + at + e] = v[e];
        }
    };
    const auto first_of = [&](int group) { return (group * kFusedThreads + tid) * 4; };
    // row and column of element `at` of the matrix
    const float per_n = 1.0f / (float)n;
    const auto place = [&](int at, int& i, int& j) {
        i = (int)((float)at * per_n);         // (at < 2^17: one off at most)
        j = at - i * n;
        if (j < 0) {
            j += n;
            --i;
        } else if (j >= n) {
            j -= n;
            ++i;
        }
    };
    // f4(e, X's place) for the four elements from `at` on
    const auto walk = [&](int at, auto f4) {
        int i, j;
        place(at, i, j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (at + e < size) f4(e, X + (tall ? j * f.ldx + i : i * f.ldx + j));
            if (++j == n) {
                j = 0;
                ++i;
            }
        }
    };
    constexpr int NG = LDS_BYTES == kFusedSmall ? 8 : 16;
    const auto enter = [&](auto mode) {
        // Momentum and norm; the first NG groups' U stay in registers.  (The places between
        // and behind X's values are 0.)
        for (int64_t i = tid; i < f.bytes / 16; i += kFusedThreads) reinterpret_cast<u32x4_t*>(smem)[i] = u32x4_t{};
        float u[NG][4];
        double sum = 0.0;
        const auto take = [&](int at, float (&v)[4], float (&w)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (MOM) v[e] = direction(l, v[e] * gs, w[e]);
                if (at + e >= size) v[e] = 0.0f;
                sum += (double)v[e] * (double)v[e];
            }
            if constexpr (MOM) {
                if (at < size) store4(mode, t.mom, at, w);
            }
        };
        {
            float w[NG][4];
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                if (i * kFusedThreads * 4 >= size) break;
                load4(mode, t.g, G{}, first_of(i), u[i]);
                if constexpr (MOM) load4(mode, t.mom, float{}, first_of(i), w[i]);
            }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                if (i * kFusedThreads * 4 >= size) break;
                take(first_of(i), u[i], w[i]);
            }
        }
        for (int i = NG; i * kFusedThreads * 4 < size; ++i) {
            float v[4], w[4];
            load4(mode, t.g, G{}, first_of(i), v);
            if constexpr (MOM) load4(mode, t.mom, float{}, first_of(i), w);
            take(first_of(i), v, w);
        }
        sum = wave_sum_dpp_f64(sum);
        if (lane == 0) part[wave] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < kFusedWaves; ++w) sum += part[w];
        // 2^14 / (|U| + eps) as the product of two binary32 factors, each of half its
        // exponent: its own may pass their range (a matrix of zeros is taken times 1, without eps too)
        const double inv = sum == 0.0 ? 1.0 : (double)(1 << kScaleX) / (sqrt(sum) + (double)l.eps);
        const double half_inv = sqrt(inv);
        const float inv0 = (float)half_inv, inv1 = (float)(inv / (double)inv0);
        const auto scale4 = [&](int at, const float (&v)[4]) {
            if constexpr (decltype(mode)::value == kLines) {
                if (at >= size) return;
                int i, j;
                place(at, i, j);
                *reinterpret_cast<u32x2_t*>(X + i * f.ldx + j) =
                    u32x2_t{pack_f16x2(v[0] * inv0 * inv1, v[1] * inv0 * inv1), pack_f16x2(v[2] * inv0 * inv1, v[3] * inv0 * inv1)};
            } else {
                walk(at, [&](int e, uint16_t* x) { *x = __builtin_bit_cast(uint16_t, (_Float16)(v[e] * inv0 * inv1)); });
            }
        };
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (i * kFusedThreads * 4 >= size) break;
            scale4(first_of(i), u[i]);
        }
        for (int i = NG; i * kFusedThreads * 4 < size; ++i) {
            float v[4], w[4];
            load4(mode, t.g, G{}, first_of(i), v);
            if constexpr (MOM) {
                // (as this thread wrote it)
                load4(mode, t.mom, float{}, first_of(i), w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = l.nesterov ? l.one_minus_beta * (v[e] * gs) + l.beta * w[e] : w[e];
            }
            scale4(first_of(i), v);
        }
    };
    // (a kind of matrix's code lies together: it runs once, and is read from memory)
    const int kind = !t.wide ? kOdd : tall ? kTall : kLines;
    if (kind == kLines) enter(std::integral_constant<int, kLines>{});
    else if (kind == kTall) enter(std::integral_constant<int, kTall>{});
    else enter(std::integral_constant<int, kOdd>{});
    __syncthreads();
    const auto frag = [&](const uint16_t* p) {
        return __builtin_bit_cast(f16x8_t, *reinterpret_cast<const u32x4_t*>(p));
    };
    // four values of row i from column j on, rounded to f16
    const auto put = [&](uint16_t* p, const float (&v)[4]) {
        *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
    };
    // One step, for matrices of RT tiles of 16 rows
    const auto iterate = [&](auto rows) {
        constexpr int RT = decltype(rows)::value, tiles = RT * RT, KS = (RT + 1) / 2;
        // A: up to two tiles of a row of tiles to a wave (their sums share fragments); with
        // one or four tiles in all the waves share the sum over c instead
        if constexpr (RT <= 2) {
            const int tile = wave % tiles, share = kFusedWaves / tiles;
            const int ti = tile / RT, tj = tile - ti * RT;
            const uint16_t* const pa = X + (16 * ti + r16) * f.ldx + 8 * rho;
            const uint16_t* const pb = X + (16 * tj + r16) * f.ldx + 8 * rho;
            f32x4_t acc = {};
#pragma unroll 4
            for (int k = wave / tiles * 32; k + 32 < f.ldx; k += 32 * share)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(frag(pb + k), frag(pa + k), acc, 0, 0, 0);
            sums[wave][lane] = acc;
            __syncthreads();
            if (wave < tiles) {
                float v[4];
                for (int w = wave + tiles; w < kFusedWaves; w += tiles) acc += sums[w][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[e] * q.alpha_a;
                put(A + (16 * ti + r16) * f.lds + 16 * tj + 4 * rho, v);
            }
        } else {
            // (3 x 3 or 4 x 4 tiles: 6 or 8 pairs, the third row's second tile left out)
            const int ti = wave >> 1, tj = 2 * (wave & 1);
            if (ti < RT) {
                const bool two = tj + 1 < RT;
                const uint16_t* const pa = X + (16 * ti + r16) * f.ldx + 8 * rho;
                const uint16_t* const pb = X + (16 * tj + r16) * f.ldx + 8 * rho;
                const uint16_t* const pc = two ? pb + 16 * f.ldx : pb;
                f32x4_t acc[2] = {};
#pragma unroll 4
                for (int k = 0; k + 32 < f.ldx; k += 32) {
                    const f16x8_t fa = frag(pa + k);
                    acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(frag(pb + k), fa, acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(frag(pc + k), fa, acc[1], 0, 0, 0);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[h][e] * q.alpha_a;
                    if (h == 0 || two) put(A + (16 * ti + r16) * f.lds + 16 * (tj + h) + 4 * rho, v);
                }
            }
        }
        __syncthreads();
        for (int tile = wave; tile < tiles; tile += kFusedWaves) {
            const int ti = tile / RT, tj = tile - ti * RT;
            f32x4_t acc = {};
            for (int ks = 0; ks < KS; ++ks)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(frag(A + (16 * tj + r16) * f.lds + 32 * ks + 8 * rho),
                                                             frag(A + (16 * ti + r16) * f.lds + 32 * ks + 8 * rho), acc, 0, 0, 0);
            const int i = 16 * ti + r16, j = 16 * tj + 4 * rho;
            const u32x2_t d = *reinterpret_cast<const u32x2_t*>(A + i * f.lds + j);
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t word = d[e >> 1];
                const _Float16 w = __builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? word >> 16 : word & 0xffffu));
                v[e] = __builtin_fmaf(q.beta_s, (float)w, acc[e] * q.alpha_s);
                if (i == j + e) v[e] += q.gamma_s;
            }
            put(S + i * f.lds + j, v);
        }
        __syncthreads();
        // (S's fragments stay in registers; rows past r16 are read as the last one's: S is
        // 0 there)
        f16x8_t fs[KS][RT];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int ti = 0; ti < RT; ++ti) fs[ks][ti] = frag(S + (16 * ti + r16) * f.lds + 32 * ks + 8 * rho);
#pragma unroll 2
        for (int jb = wave; 16 * jb < c; jb += kFusedWaves) {
            f32x4_t acc[RT] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint2 half[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = min(32 * ks + 8 * rho + 4 * h + (r16 >> 2), f.r16 - 1);
                    half[h] = dense_read_tr((const unsigned char*)(X + row * f.ldx + 16 * jb + 4 * (r16 & 3)));
                }
                const u32x4_t w = {half[0].x, half[0].y, half[1].x, half[1].y};
                const f16x8_t fb = __builtin_bit_cast(f16x8_t, w);
#pragma unroll
                for (int ti = 0; ti < RT; ++ti)
                    acc[ti] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb, fs[ks][ti], acc[ti], 0, 0, 0);
            }
#pragma unroll
            for (int ti = 0; ti < RT; ++ti) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[ti][e] * q.alpha_x;
                put(X + (16 * ti + r16) * f.ldx + 16 * jb + 4 * rho, v);
            }
        }
        __syncthreads();
    };
    for (int it = 0; it < q.iterations; ++it) {
        if (f.r16 == 16) iterate(std::integral_constant<int, 1>{});
        else if (f.r16 == 32) iterate(std::integral_constant<int, 2>{});
        else if (f.r16 == 48) iterate(std::integral_constant<int, 3>{});
        else iterate(std::integral_constant<int, 4>{});
    }
    const auto leave = [&](auto mode) {
        const float unit = 1.0f / (1 << kScaleX), step = t.step * unit;
        float* const p = OUT == kOutMaster ? t.master : (float*)t.out;
        const auto give = [&](int at, float (&w)[4]) {
            float x[4] = {};
            if (at >= size) return;
            if constexpr (decltype(mode)::value == kLines) {
                int i, j;
                place(at, i, j);
                const u32x2_t d = *reinterpret_cast<const u32x2_t*>(X + i * f.ldx + j);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu));
            } else {
                walk(at, [&](int e, uint16_t* from) { x[e] = (float)__builtin_bit_cast(_Float16, *from); });
            }
            if constexpr (OUT == kOutBf16) {
                uint16_t* const o = (uint16_t*)t.out + base + at;
                if constexpr (decltype(mode)::value != kOdd) {
                    *reinterpret_cast<u32x2_t*>(o) = u32x2_t{pack_bf16x2(x[0] * unit, x[1] * unit), pack_bf16x2(x[2] * unit, x[3] * unit)};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < size) o[e] = (uint16_t)f32_to_bf16_bits(x[e] * unit);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __builtin_fmaf(-step, x[e], l.decay * w[e]);
                store4(mode, p, at, w);
                if constexpr (OUT == kOutMaster) {
                    uint16_t* const o = (uint16_t*)t.out + base + at;
                    if constexpr (decltype(mode)::value != kOdd) {
                        *reinterpret_cast<u32x2_t*>(o) = u32x2_t{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (at + e < size) o[e] = (uint16_t)f32_to_bf16_bits(w[e]);
                    }
                }
            }
        };
        for (int i0 = 0; i0 * kFusedThreads * 4 < size; i0 += NG) {
            float w[NG][4];
            if constexpr (OUT != kOutBf16) {
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    if ((i0 + i) * kFusedThreads * 4 >= size) break;
                    load4(mode, p, float{}, first_of(i0 + i), w[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                if ((i0 + i) * kFusedThreads * 4 >= size) break;
                give(first_of(i0 + i), w[i]);
            }
        }
    };
    if (kind == kLines) leave(std::integral_constant<int, kLines>{});
    else if (kind == kTall) leave(std::integral_constant<int, kTall>{});
    else leave(std::integral_constant<int, kOdd>{});
}

template <typename G, int LDS_BYTES>
void launch_fused(const OrthoList& l, const FusedScalars& q, int out, bool mom, unsigned blocks, hipStream_t s)
{
    const dim3 grid(blocks), block(kFusedThreads);
    if (!mom) ortho_fused_kernel<G, false, kOutBf16, LDS_BYTES><<<grid, block, 0, s>>>(l, q);
    else if (out == kOutParam) ortho_fused_kernel<G, true, kOutParam, LDS_BYTES><<<grid, block, 0, s>>>(l, q);
    else ortho_fused_kernel<G, true, kOutMaster, LDS_BYTES><<<grid, block, 0, s>>>(l, q);
}

// --------------------------------------------------------------------------
// the products
// --------------------------------------------------------------------------

// E products C = alpha A B^T (+ beta D + gamma I), all f16, of one tensor.
struct OrthoGemm {
    const uint16_t* a;
    const uint16_t* b;
    const uint16_t* d;        // [M, N], ldc (poly only)
    uint16_t* c;
    int64_t sa, sb, sc;       // elements from a matrix to the next
    int M, N, K;              // N: columns of c with a value; ldc the stored ones (the others 0)
    int lda, ldb, ldc;
    int nm, nn, first;        // tiles of a matrix, first tile of the tensor
};

struct OrthoArgs {
    OrthoGemm t[kTensors];
    int count, tiles;
    float alpha, beta, gamma;
};
static_assert(sizeof(OrthoArgs) <= 4096, "kernel arguments");

// SYM: A B^T is symmetric (X X^T, A A): the tiles on and above the diagonal are
// computed and those above it written a second time, across it, by way of LDS.
template <int KIND, bool ACOL, bool BCOL, bool POLY, bool SYM>
struct OrthoPolicy : DenseTile<KIND, 2> {
    using DenseTile<KIND, 2>::MI;
    using DenseTile<KIND, 2>::NJ;
    static constexpr bool kACol = ACOL, kBCol = BCOL, kF16 = true;
    static constexpr int BM = 32 * MI, BN = 32 * NJ;
    static constexpr int kLine = 16 * MI + 16;          // bytes of half of a wave's rows of a column, and 16
    static constexpr bool kMid = false;
    static constexpr int kScratch = SYM ? 32 * kLine : 0;
    using Args = OrthoArgs;
    struct Tile : GemmTile {
        int at, e, m0, n0;
    };
    __device__ static int tiles(const Args& g) { return g.tiles; }
    __device__ static void tile(const Args& g, int q, Tile& t)
    {
        int i = 0;
        while (i + 1 < g.count && g.t[i + 1].first <= q) ++i;
        const OrthoGemm& p = g.t[i];
        const int each = SYM ? p.nm * (p.nm + 1) / 2 : p.nm * p.nn;
        const int e = (q - p.first) / each;
        TileAt at;
        if constexpr (SYM) {
            at = {0, q - p.first - e * each};
            for (; at.n >= p.nm - at.m; ++at.m) at.n -= p.nm - at.m;
            at.n += at.m;
        } else {
            at = tile_at(q - p.first - e * each, p.nm, p.nn, 8);
        }
        t.at = i;
        t.e = e;
        t.m0 = at.m * BM;
        t.n0 = at.n * BN;
        t.a = (const unsigned char*)(p.a + e * p.sa + (ACOL ? (int64_t)t.m0 : (int64_t)t.m0 * p.lda));
        t.b = (const unsigned char*)(p.b + e * p.sb + (BCOL ? (int64_t)t.n0 : (int64_t)t.n0 * p.ldb));
        t.a_rows = min(BM, p.M - t.m0);
        t.b_rows = min(BN, p.N - t.n0);
        t.lda = p.lda;
        t.ldb = p.ldb;
        t.k = p.K;
    }
    __device__ static int b_row(const Args&, const Tile&, int R) { return R; }
    __device__ static void epilogue(const Args& g, const Tile& t, f32x4_t (&acc)[MI][NJ], int wm, int wn, int r16, int rho,
                                    unsigned char* scratch)
    {
        const OrthoGemm& p = g.t[t.at];
        const int ldc = p.ldc;
        const int64_t first = t.e * p.sc + (int64_t)t.m0 * ldc;
        const __amdgpu_buffer_rsrc_t res = dense_rsrc(p.c + first, t.a_rows * ldc * 2);
        const __amdgpu_buffer_rsrc_t dres = dense_rsrc(POLY ? p.d + first : nullptr, t.a_rows * ldc * 2);
        const float alpha = g.alpha;
        // the values of two tiles side by side, rows of tile i
        const auto values = [&](int i, int j, const u32x2_t (&d)[2], float (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int jj = j + (e >> 2);
                v[e] = acc[i][jj][e & 3] * alpha;
                if constexpr (POLY) {
                    // (halves by a shift: as elements of a pair, hipcc 7.2 takes both words of the
                    // load for the first)
                    const uint32_t word = d[e >> 2][(e & 3) >> 1];
                    const _Float16 w = __builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? word >> 16 : word & 0xffffu));
                    v[e] = __builtin_fmaf(g.beta, (float)w, v[e]);
                    if (t.m0 + (wm * MI + i) * 16 + r16 == t.n0 + (wn * NJ + jj) * 16 + 4 * rho + (e & 3)) v[e] += g.gamma;
                }
            }
        };
        const auto load_d = [&](int i, int j, u32x2_t (&d)[2]) {
            const int row = (wm * MI + i) * 16 + r16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = t.n0 + (wn * NJ + j + h) * 16 + 4 * rho;
                d[h] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(
                    dres, row < t.a_rows && col < ldc ? (uint32_t)(row * ldc + col) * 2u : kOOR, 0, 0));
            }
        };
        // SYM, above the diagonal: 32 columns x half of the wave's rows also go through LDS, and
        // from there to c as rows n0 + j, columns m0 .. (which are all there)
        const __amdgpu_buffer_rsrc_t cres = dense_rsrc(SYM ? p.c + t.e * p.sc + (int64_t)t.n0 * ldc : nullptr, t.b_rows * ldc * 2);
        const bool both = SYM && t.m0 != t.n0;
        constexpr int HI = SYM ? MI / 2 : MI;
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
#pragma unroll
            for (int i0 = 0; i0 < MI; i0 += HI) {
                __builtin_amdgcn_sched_barrier(0);
                u32x2_t d[HI][2];
                if constexpr (POLY) {
#pragma unroll
                    for (int i = 0; i < HI; ++i) load_d(i0 + i, j, d[i]);
                }
#pragma unroll
                for (int i = 0; i < HI; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int row = (wm * MI + i0 + i) * 16 + r16;
                    float v[8];
                    values(i0 + i, j, d[i], v);
                    store_pair<true>(v, res, row < t.a_rows, (uint32_t)(row * ldc), t.n0 + (wn * NJ + j) * 16, ldc, rho);
                    if (SYM && both) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            *reinterpret_cast<_Float16*>(scratch + (16 * (e >> 2) + 4 * rho + (e & 3)) * kLine + (16 * i + r16) * 2) = (_Float16)v[e];
                    }
                }
                if (SYM && both) {
                    constexpr int kSegs = 2 * HI, kLines = 64 / kSegs;      // 16-byte pieces of a line, lines a store
                    const int lane = 16 * rho + r16;
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int h = 0; h < 32 / kLines; ++h) {
                        const int line = h * kLines + lane / kSegs, seg = lane % kSegs;
                        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(scratch + line * kLine + seg * 16);
                        const int to = (wn * NJ + j) * 16 + line;
                        __builtin_amdgcn_raw_buffer_store_b128(
                            w, cres, to < t.b_rows ? (uint32_t)(to * ldc + t.m0 + (wm * MI + i0) * 16 + seg * 8) * 2u : kOOR, 0, 0);
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            }
        }
    }
};

// The same products where there are few tiles, so that a call is its way from memory: a
// block owns 32 x 32, its 8 waves take k's chunks of 64 in turn, each through a
// ring of D stages of LDS of its own (no barriers), and their sums meet in LDS.  With k
// up to 512 all of it is on its way at once: 512 x 512 4.2 us a product, 6.7 with 64 x 64 tiles.
constexpr int kShortWaves = 8, kShortThreads = kShortWaves * kWave;

template <bool ACOL, bool BCOL, bool POLY, bool SYM, int D>
__global__ __launch_bounds__(kShortThreads) void ortho_short_kernel(OrthoArgs g)
{
    using P = OrthoPolicy<1, ACOL, BCOL, POLY, SYM>;
    constexpr int kStageBytes = 8192, NI = 8, kLine = 40;      // f16 from a line of the result to the next
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kShortWaves * D * kStageBytes];
    const int per = (g.tiles + 7) / 8;
    const int q = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (q >= g.tiles) return;
    typename P::Tile t = {};
    P::tile(g, q, t);
    const OrthoGemm& p = g.t[t.at];
    const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, rho = lane >> 4;
    // this thread's two values of the result: row, col and col + 1
    const int part_of = tid >> 7, place = (tid >> 1) & 63;
    const int row = 16 * (part_of >> 1) + (place & 15), col = 16 * (part_of & 1) + 4 * (place >> 4) + 2 * (tid & 1);
    const int ldc = p.ldc;
    const int64_t first = t.e * p.sc + (int64_t)t.m0 * ldc;
    uint32_t d = 0;
    if constexpr (POLY) {
        if (row < t.a_rows && t.n0 + col < ldc) d = *reinterpret_cast<const uint32_t*>(p.d + first + (int64_t)row * ldc + t.n0 + col);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t*)smem + wave * (D * kStageBytes);
    const int seg0 = (lane & 7) ^ (lane >> 3);
    // a chunk of an operand in 4 KB: k along rows 32 lines of 128 bytes, swizzled as
    // the large tiles'; k down columns 64 lines of 64 bytes, piece s of line r at slot
    // s ^ 2 (r >> 3 & 1)
    const auto load = [&](auto down, const unsigned char* from, int rows, int ld, int c, uint32_t lds) {
        const int left = t.k - c * 64;
        if constexpr (decltype(down)::value) {
            const __amdgpu_buffer_rsrc_t res =
                dense_rsrc(from + (int64_t)c * 128 * ld, left > 0 ? (min(64, left) - 1) * ld * 2 + ((rows + 7) & ~7) * 2 : 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                dense_dma(res, (uint32_t)((16 * i + (lane >> 2)) * 2 * ld + (((lane & 3) ^ (lane >> 4 & 2)) << 4)), 0u, lds + i * 1024);
        } else {
            const __amdgpu_buffer_rsrc_t res = dense_rsrc(from, (rows - 1) * ld * 2 + ((t.k + 7) & ~7) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int seg = seg0 ^ (i & 1);
                dense_dma(res, seg * 8 < left ? (uint32_t)((8 * i + (lane >> 3)) * 2 * ld + c * 128 + seg * 16) : kOOR, 0u, lds + i * 1024);
            }
        }
    };
    const auto load_both = [&](int j, uint32_t lds) {
        const int c = kShortWaves * j + wave;
        load(std::bool_constant<ACOL>{}, t.a, t.a_rows, t.lda, c, lds);
        load(std::bool_constant<BCOL>{}, t.b, t.b_rows, t.ldb, c, lds + 4096);
    };
    const int fkey = (lane & 7) ^ ((lane >> 3) & 1);
    const int frow = (r16 >> 3) * 1024 + (lane & 7) * 128;
    const int tin = (r16 >> 2) * 64 + ((r16 & 3) >> 1) * 16 + (r16 & 1) * 8;
    const auto read = [&](auto down, const unsigned char* op, int tile, int ks) -> f16x8_t {
        if constexpr (decltype(down)::value) {
            const unsigned char* const at = op + (32 * ks + 8 * rho) * 64 + ((tile ^ (rho & 1)) << 5) + tin;
            const uint2 lo = dense_read_tr(at), hi = dense_read_tr(at + 256);
            return __builtin_bit_cast(f16x8_t, u32x4_t{lo.x, lo.y, hi.x, hi.y});
        } else {
            return __builtin_bit_cast(f16x8_t, *reinterpret_cast<const u32x4_t*>(op + tile * 2048 + frow + (((4 * ks + rho) ^ fkey) << 4)));
        }
    };
    f32x4_t acc[2][2] = {};
    const int turns = (t.k + kShortWaves * 64 - 1) / (kShortWaves * 64);
#pragma unroll
    for (int i = 0; i < D; ++i) load_both(i, lds0 + i * kStageBytes);
    for (int j = 0, stage = 0; j < turns; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * NI) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        const unsigned char* const at = smem + (wave * D + stage) * kStageBytes;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            f16x8_t fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = read(std::bool_constant<ACOL>{}, at, i, ks);
                fb[i] = read(std::bool_constant<BCOL>{}, at + 4096, i, ks);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) acc[i][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[h], fa[i], acc[i][h], 0, 0, 0);
        }
        // (the reads above have ended; chunks past the end load nothing and keep the count)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
        if (j + 1 < turns) load_both(j + D, lds0 + stage * kStageBytes);
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    dense_wait_barrier<0>();
    f32x4_t* const part = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) part[(wave * 4 + 2 * i + h) * kWave + lane] = acc[i][h];
    __syncthreads();
    float v[2] = {};
#pragma unroll
    for (int w = 0; w < kShortWaves; ++w) {
        const float* const from = reinterpret_cast<const float*>(part) + ((w * 4 + part_of) * kWave + place) * 4 + 2 * (tid & 1);
        v[0] += from[0];
        v[1] += from[1];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        v[e] *= g.alpha;
        if constexpr (POLY) {
            v[e] = __builtin_fmaf(g.beta, (float)__builtin_bit_cast(_Float16, (uint16_t)(e ? d >> 16 : d & 0xffffu)), v[e]);
            if (t.m0 + row == t.n0 + col + e) v[e] += g.gamma;
        }
    }
    // The result's lines, and those across the diagonal, by way of LDS (behind the sums).
    const bool both = SYM && t.m0 != t.n0;
    uint16_t* const line = reinterpret_cast<uint16_t*>(smem + kShortWaves * 4096);
    const uint32_t pair = pack_f16x2(v[0], v[1]);
    *reinterpret_cast<uint32_t*>(line + row * kLine + col) = pair;
    if (both) {
        line[(32 + col) * kLine + row] = (uint16_t)pair;
        line[(33 + col) * kLine + row] = (uint16_t)(pair >> 16);
    }
    __syncthreads();
    if (tid < (both ? 256 : 128)) {
        const int to = tid >> 2, seg = (tid & 3) * 8;      // line 0 .. 63
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(line + to * kLine + seg);
        if (to < 32) {
            if (to < t.a_rows && t.n0 + seg < ldc) *reinterpret_cast<u32x4_t*>(p.c + first + (int64_t)to * ldc + t.n0 + seg) = w;
        } else if (to - 32 < t.b_rows) {
            *reinterpret_cast<u32x4_t*>(p.c + t.e * p.sc + (int64_t)(t.n0 + to - 32) * ldc + t.m0 + seg) = w;
        }
    }
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round8(int64_t n) { return up(n, 8) * 8; }

template <bool ACOL, bool BCOL, bool POLY, bool SYM>
struct Products {
    template <int KIND> using Policy = OrthoPolicy<KIND, ACOL, BCOL, POLY, SYM>;
};

// Launches the products in `args` (nm, nn, first and tiles are set here).
template <bool ACOL, bool BCOL, bool POLY, bool SYM>
int launch_products(OrthoArgs& args, const int64_t* batch, hipStream_t s)
{
    const int cus = dense_cus();
    int64_t big = 0, small = 0, thin = 0, few = 0, k = 0;
    const auto tiles = [](const OrthoGemm& p, int64_t side) {
        const int64_t m = up(p.M, side), n = up(p.N, side);
        return SYM ? m * (m + 1) / 2 : m * n;
    };
    for (int i = 0; i < args.count; ++i) {
        const OrthoGemm& p = args.t[i];
        big += batch[i] * tiles(p, 256);
        small += batch[i] * tiles(p, 128);
        thin += batch[i] * tiles(p, 64);
        few += batch[i] * tiles(p, 32);
        k = std::max<int64_t>(k, p.K);
    }
    const auto lay_out = [&](int64_t side) {
        args.tiles = 0;
        for (int i = 0; i < args.count; ++i) {
            OrthoGemm& p = args.t[i];
            p.nm = (int)up(p.M, side);
            p.nn = (int)up(p.N, side);
            p.first = args.tiles;
            args.tiles += (int)(batch[i] * tiles(p, side));
        }
    };
    // One round of the short kernel's blocks.  Five steps, with it and without: 512 x 512 72
    // and 102 us, 300 x 4000 127 and 194, 8 of 80 x 1000 64 and 83; two or four rounds would
    // take 512 x 1024 89 to 84, but 2 of 128 x 2048 77 to 80 and 16 of 256 x 256 79 to 109.
    if (few <= cus) {
        lay_out(32);
        const dim3 grid((unsigned)(up(args.tiles, 8) * 8)), block(kShortThreads);
        if (k <= kShortWaves * 64) ortho_short_kernel<ACOL, BCOL, POLY, SYM, 1><<<grid, block, 0, s>>>(args);
        else ortho_short_kernel<ACOL, BCOL, POLY, SYM, 2><<<grid, block, 0, s>>>(args);
        return check_launch("ortho_short_kernel");
    }
    const int kind = dense_kind(big, 0, small, thin, false, cus), side = kind == kTileBig ? 256 : kind == kTileSmall ? 128 : 64;
    lay_out(side);
    return launch_dense<Products<ACOL, BCOL, POLY, SYM>::template Policy>(args, kind, args.tiles, cus, s, "ortho_products");
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------

struct Shape {
    int64_t E, m, n;
    bool tall() const { return m > n; }
    int64_t r() const { return std::min(m, n); }
    int64_t ldx() const { return round8(n); }
    int64_t ldr() const { return round8(r()); }
    int64_t sums() const { return std::min(up(m * n, kChunk), kSums); }
    int64_t blocks() const { return up(m * ldx(), kChunk); }
    int64_t x_bytes() const { return up(E * m * ldx() * 2, 256) * 256; }
    int64_t a_bytes() const { return up(E * r() * ldr() * 2, 256) * 256; }
    int64_t sum_bytes() const { return up(E * sums() * 8, 256) * 256; }
    // 0: products of wide matrices, 1: of tall ones, 2, 3: one block a matrix
    int way() const
    {
        if (r() <= kFusedSide) {
            const int64_t lds = fused_layout(r(), std::max(m, n)).bytes;
            if (lds <= kFusedLarge) return lds <= kFusedSmall ? 2 : 3;
        }
        return tall() ? 1 : 0;
    }
    // of all its matrices, in blocks of kDenseThreads threads
    int64_t launch_blocks() const { return E * (way() >= 2 ? kFusedThreads / kDenseThreads : blocks()); }
    int64_t bytes() const { return way() >= 2 ? 0 : 2 * x_bytes() + 2 * a_bytes() + sum_bytes(); }
};
constexpr int kWays = 4;

constexpr int64_t kMostSide = 1 << 16;
// A launch has less than 2^32 threads: 2^24 blocks of the elementwise kernels, 2^23 of the one
// that takes a matrix in one block.
constexpr int64_t kMostBlocks = 1 << 24, kMostMatrices = 1 << 23;
static_assert(kMostBlocks * kDenseThreads <= (int64_t)1 << 32 && kMostMatrices * kFusedThreads <= (int64_t)1 << 32, "threads");

bool shape_ok(const Shape& s)
{
    if (s.E < 0 || s.m < 0 || s.n < 0 || s.m >= kMostSide || s.n >= kMostSide || s.E >= kMostMatrices) return false;
    return s.E * s.m * s.n == 0 || s.launch_blocks() < kMostBlocks;
}

struct OrthoCall {
    const char* fn;
    const int64_t* shapes;    // [count, 3]
    int64_t count;
    const void* const* g;
    float* const* mom;
    void* const* out;
    float* const* master;
    const float* step;
    int dtype, out_kind;
    int iterations;
    float a, b, c;
};

Shape shape_at(const int64_t* shapes, int64_t i) { return {shapes[3 * i], shapes[3 * i + 1], shapes[3 * i + 2]}; }

template <bool MOM>
void launch_elementwise(const OrthoList& list, int dtype, unsigned blocks, bool scale, hipStream_t s)
{
    const dim3 grid(blocks), block(kDenseThreads);
    if (dtype == ET_DTYPE_F32) {
        if (scale) ortho_scale_kernel<float, MOM><<<grid, block, 0, s>>>(list);
        else ortho_norm_kernel<float, MOM><<<grid, block, 0, s>>>(list);
    } else {
        if (scale) ortho_scale_kernel<uint16_t, MOM><<<grid, block, 0, s>>>(list);
        else ortho_norm_kernel<uint16_t, MOM><<<grid, block, 0, s>>>(list);
    }
}

// One set of up to kTensors tensors that go one way.
int run_set(const OrthoCall& call, OrthoList list, int way, const int64_t* index, unsigned char* const* place, hipStream_t s)
{
    const int count = list.count;
    uint16_t *x[kTensors], *y[kTensors], *ga[kTensors], *gs[kTensors];
    int64_t batch[kTensors];
    uint32_t blocks = 0;
    bool tall = false;
    for (int i = 0; i < count; ++i) {
        const int64_t k = index[i];
        const Shape sh = shape_at(call.shapes, k);
        tall = sh.tall();
        batch[i] = sh.E;
        unsigned char* p = place[i];
        x[i] = (uint16_t*)p;
        y[i] = (uint16_t*)(p += sh.x_bytes());
        ga[i] = (uint16_t*)(p += sh.x_bytes());
        gs[i] = (uint16_t*)(p += sh.a_bytes());
        OrthoTensor& t = list.t[i];
        t.g = call.g[k];
        t.mom = call.mom ? call.mom[k] : nullptr;
        t.x = x[i];
        t.partial = (double*)(p += sh.a_bytes());
        t.out = call.out[k];
        t.master = call.master ? call.master[k] : nullptr;
        t.m = (uint32_t)sh.m;
        t.n = (uint32_t)sh.n;
        t.ldx = (uint32_t)sh.ldx();
        t.sums = (uint32_t)sh.sums();
        t.first = blocks;
        t.each = way >= 2 ? 1u : (uint32_t)sh.blocks();
        t.step = call.step ? call.step[k] : 0.0f;
        t.wide = sh.n % 8 == 0 && ((uintptr_t)t.g | (uintptr_t)t.mom | (uintptr_t)t.out | (uintptr_t)t.master) % 16 == 0;
        blocks += (uint32_t)(sh.E * t.each);
    }
    // S is held times 2^scale_s, its largest singular value being below a
    int scale_s = 0;
    while (call.a * pow2(scale_s + 1) < 60000.0f) ++scale_s;
    const float alpha_a = pow2(-kScaleX), alpha_s = call.c * pow2(scale_s - 2 * kScaleX);
    const float beta_s = call.b * pow2(scale_s - kScaleX), gamma_s = call.a * pow2(scale_s), alpha_x = pow2(-scale_s);
    if (way >= 2) {
        const FusedScalars q = {alpha_a, alpha_s, beta_s, gamma_s, alpha_x, call.iterations};
        const bool mom = call.mom != nullptr;
        if (call.dtype == ET_DTYPE_F32) {
            if (way == 2) launch_fused<float, kFusedSmall>(list, q, call.out_kind, mom, blocks, s);
            else launch_fused<float, kFusedLarge>(list, q, call.out_kind, mom, blocks, s);
        } else {
            if (way == 2) launch_fused<uint16_t, kFusedSmall>(list, q, call.out_kind, mom, blocks, s);
            else launch_fused<uint16_t, kFusedLarge>(list, q, call.out_kind, mom, blocks, s);
        }
        return check_launch("ortho_fused_kernel");
    }
    for (const bool scale : {false, true}) {
        if (call.mom) launch_elementwise<true>(list, call.dtype, blocks, scale, s);
        else launch_elementwise<false>(list, call.dtype, blocks, scale, s);
        if (const int rc = check_launch("ortho_norm_kernel")) return rc;
    }
    OrthoArgs args = {};
    args.count = count;
    const auto fill = [&](auto f) {
        for (int i = 0; i < count; ++i) {
            const Shape sh = shape_at(call.shapes, index[i]);
            args.t[i] = {};
            f(args.t[i], i, sh, (int)sh.r(), (int)sh.ldr(), (int)sh.ldx());
        }
    };
    for (int it = 0; it < call.iterations; ++it) {
        fill([&](OrthoGemm& p, int i, const Shape& sh, int r, int ldr, int ldx) {
            p.a = p.b = x[i];
            p.sa = p.sb = sh.m * ldx;
            p.c = ga[i];
            p.sc = (int64_t)r * ldr;
            p.M = p.N = r;
            p.K = (int)(tall ? sh.m : ldx);
            p.lda = p.ldb = ldx;
            p.ldc = ldr;
        });
        args.alpha = alpha_a;
        int rc = tall ? launch_products<true, true, false, true>(args, batch, s) : launch_products<false, false, false, true>(args, batch, s);
        if (rc) return rc;
        fill([&](OrthoGemm& p, int i, const Shape&, int r, int ldr, int) {
            p.a = p.b = p.d = ga[i];
            p.c = gs[i];
            p.sa = p.sb = p.sc = (int64_t)r * ldr;
            p.M = p.N = r;
            p.K = p.lda = p.ldb = p.ldc = ldr;
        });
        args.alpha = alpha_s;
        args.beta = beta_s;
        args.gamma = gamma_s;
        rc = launch_products<false, false, true, true>(args, batch, s);
        if (rc) return rc;
        fill([&](OrthoGemm& p, int i, const Shape& sh, int r, int ldr, int ldx) {
            // wide: S X, X read down its columns; tall: X S, S symmetric
            p.a = tall ? x[i] : gs[i];
            p.b = tall ? gs[i] : x[i];
            p.sa = tall ? sh.m * ldx : (int64_t)r * ldr;
            p.sb = tall ? (int64_t)r * ldr : sh.m * ldx;
            p.lda = tall ? ldx : ldr;
            p.ldb = tall ? ldr : ldx;
            p.c = y[i];
            p.sc = sh.m * ldx;
            p.M = (int)sh.m;
            p.N = (int)sh.n;
            p.K = r;
            p.ldc = ldx;
        });
        args.alpha = alpha_x;
        rc = tall ? launch_products<false, false, false, false>(args, batch, s) : launch_products<false, true, false, false>(args, batch, s);
        if (rc) return rc;
        for (int i = 0; i < count; ++i) std::swap(x[i], y[i]);
    }
    for (int i = 0; i < count; ++i) list.t[i].x = x[i];
    const dim3 grid(blocks), block(kDenseThreads);
    if (call.out_kind == kOutBf16) ortho_finish_kernel<kOutBf16><<<grid, block, 0, s>>>(list);
    else if (call.out_kind == kOutParam) ortho_finish_kernel<kOutParam><<<grid, block, 0, s>>>(list);
    else ortho_finish_kernel<kOutMaster><<<grid, block, 0, s>>>(list);
    return check_launch("ortho_finish_kernel");
}

int fail_at(const char* fn, const char* what) { return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + what); }

int check_list(const char* fn, const char* name, const void* const* list, const int64_t* shapes, int64_t count, uintptr_t align)
{
    if (count > 0 && !list) return fail_at(fn, (std::string("null ") + name).c_str());
    for (int64_t i = 0; i < count; ++i) {
        const Shape s = shape_at(shapes, i);
        if (s.E * s.m * s.n == 0) continue;
        if (!list[i]) return fail_at(fn, (std::string("null pointer in ") + name).c_str());
        if ((uintptr_t)list[i] % align) return fail_at(fn, (std::string("a pointer in ") + name + " is not aligned").c_str());
    }
    return ET_OK;
}

int check_call(const char* fn, const int64_t* shapes, int64_t count, int dtype, int iterations, const float* abc, float eps)
{
    if (count < 0) return fail_at(fn, "count must be >= 0");
    if (count > 0 && !shapes) return fail_at(fn, "null shapes");
    for (int64_t i = 0; i < count; ++i)
        if (!shape_ok(shape_at(shapes, i))) return fail_at(fn, "sides must be in [0, 65536), and a tensor below 2^23 matrices and 2^36 elements");
    if (dtype != ET_DTYPE_F32 && dtype != ET_DTYPE_BF16) return fail_at(fn, "dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    if (iterations < 1 || iterations > 64) return fail_at(fn, "iterations must be in [1, 64]");
    if (!abc) return fail_at(fn, "null coefficients");
    if (!(eps >= 0.0f) || !(eps < __builtin_inff())) return fail_at(fn, "eps must be finite and >= 0");
    // the scaled f16 numbers hold X's singular values up to 1.9 (A's up to 3.61, 59146 times
    // 2^-14) and S's up to 1.01 a
    const double a = abc[0], b = abc[1], c = abc[2];
    bool ok = a > 0.0 && a < 16.0 && __builtin_fabs(b) < 64.0 && __builtin_fabs(c) < 64.0;
    double most = 1.0;        // the largest singular value that a step can start from
    for (int it = 0; ok && it < iterations; ++it) {
        double next = 0.0;
        for (int k = 0; k <= 256; ++k) {
            const double s = most * k / 256.0, f = a + b * s * s + c * s * s * s * s;
            ok = ok && __builtin_fabs(f) <= 1.01 * a;
            next = std::max(next, __builtin_fabs(f * s));
        }
        const double before = most;
        most = std::max(most, 1.01 * next);
        ok = ok && most < 1.9;
        if (most == before) break;      // (all further steps are alike)
    }
    if (!ok) return fail_at(fn, "coefficients must keep singular values in [0, 1] below 1.9 and |a + b s^2 + c s^4| at most a (below 16)");
    return ET_OK;
}

// The tensors that go one way, in sets of one launch a kernel: f(index, offset, count), with each
// tensor's place in the workspace.  The sets run one behind the other on a stream, so they share it.
template <typename W, typename F>
int each_set(const int64_t* shapes, int64_t count, int way, const W& way_of, const F& f)
{
    int64_t index[kTensors], offset[kTensors], blocks = 0, bytes = 0;
    int n = 0;
    for (int64_t i = 0; i < count; ++i) {
        const Shape sh = shape_at(shapes, i);
        if (sh.E * sh.m * sh.n == 0 || way_of(sh) != way) continue;
        if (n == kTensors || blocks + sh.launch_blocks() >= kMostBlocks) {
            if (n) {
                if (const int rc = f(index, offset, n)) return rc;
            }
            n = 0;
            blocks = bytes = 0;
        }
        index[n] = i;
        offset[n++] = bytes;
        blocks += sh.launch_blocks();
        bytes += sh.bytes();
    }
    return n ? f(index, offset, n) : ET_OK;
}

int run_call(const OrthoCall& call, const OrthoList& scalars, unsigned char* workspace, hipStream_t s)
{
    // Blocks of both sizes of LDS that find a CU each go in one launch, beside one another
    // (three routers and 3 x 8 matrices of 64 x 512 and of 512 x 32, in one or the other: 57 us
    // in two launches, 41 in one, before other steps).
    int64_t small = 0, large = 0;
    for (int64_t i = 0; i < call.count; ++i) {
        const Shape sh = shape_at(call.shapes, i);
        if (sh.way() == 2) small += sh.E;
        if (sh.way() == 3) large += sh.E;
    }
    const bool together = small > 0 && large > 0 && small + large <= dense_cus();
    const auto way_of = [together](const Shape& sh) {
        const int way = sh.way();
        return together && way == 2 ? 3 : way;
    };
    for (int way = 0; way < kWays; ++way) {
        const int rc = each_set(call.shapes, call.count, way, way_of, [&](const int64_t* index, const int64_t* offset, int count) {
            OrthoList list = scalars;
            list.count = count;
            unsigned char* place[kTensors];
            for (int i = 0; i < count; ++i) place[i] = workspace + offset[i];
            return run_set(call, list, way, index, place, s);
        });
        if (rc) return rc;
    }
    return ET_OK;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" size_t et_orthogonalize_workspace_bytes(const int64_t* shapes, int64_t count)
{
    if (count < 0 || (count > 0 && !shapes)) return 0;
    for (int64_t i = 0; i < count; ++i)
        if (!shape_ok(shape_at(shapes, i))) return 0;
    // The largest kTensors of a way: whatever set they come in, so that the space for a list is
    // enough for any part of it.  (Matrices that one block takes need none.)
    int64_t most = 0;
    for (const int way : {0, 1}) {
        int64_t bytes[kTensors] = {};           // falling
        for (int64_t i = 0; i < count; ++i) {
            const Shape s = shape_at(shapes, i);
            if (s.E * s.m * s.n == 0 || s.way() != way || s.bytes() <= bytes[kTensors - 1]) continue;
            int at = kTensors - 1;
            for (; at > 0 && bytes[at - 1] < s.bytes(); --at) bytes[at] = bytes[at - 1];
            bytes[at] = s.bytes();
        }
        int64_t sum = 0;
        for (const int64_t n : bytes) sum += n;
        most = std::max(most, sum);
    }
    return (size_t)most;
}

namespace {

int check_workspace(const char* fn, const int64_t* shapes, int64_t count, const void* workspace, size_t bytes)
{
    const size_t need = et_orthogonalize_workspace_bytes(shapes, count);
    if (bytes < need || (need && !workspace))
        return fail(ET_ERR_WORKSPACE_TOO_SMALL, std::string(fn) + ": workspace needs " + std::to_string(need) + " bytes");
    if ((uintptr_t)workspace % 256) return fail_at(fn, "workspace must be 256-byte aligned");
    return ET_OK;
}

}  // namespace

extern "C" int et_orthogonalize(const void* const* g, void* const* out, const int64_t* shapes, int64_t count, int dtype,
                                int iterations, const float* coefficients, float eps, void* workspace,
                                size_t workspace_bytes, void* stream)
{
    const char* fn = "et_orthogonalize";
    int rc = check_call(fn, shapes, count, dtype, iterations, coefficients, eps);
    if (!rc) rc = check_list(fn, "g", g, shapes, count, dtype == ET_DTYPE_F32 ? 4 : 2);
    if (!rc) rc = check_list(fn, "out", out, shapes, count, 2);
    if (!rc) rc = check_workspace(fn, shapes, count, workspace, workspace_bytes);
    if (rc) return rc;
    OrthoCall call = {};
    call.fn = fn;
    call.shapes = shapes;
    call.count = count;
    call.g = g;
    call.out = out;
    call.dtype = dtype;
    call.out_kind = kOutBf16;
    call.iterations = iterations;
    call.a = coefficients[0];
    call.b = coefficients[1];
    call.c = coefficients[2];
    OrthoList scalars = {};
    scalars.eps = eps;
    return run_call(call, scalars, (unsigned char*)workspace, (hipStream_t)stream);
}

extern "C" int et_muon(void* const* params, const void* const* grads, float* const* momentum, float* const* masters,
                       const float* step_sizes, const int64_t* shapes, int64_t count, int param_dtype, int grad_dtype,
                       et_muon_scalars scalars, const float* grad_scale, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* fn = "et_muon";
    const float abc[3] = {scalars.a, scalars.b, scalars.c};
    int rc = check_call(fn, shapes, count, grad_dtype, scalars.iterations, abc, scalars.eps);
    if (rc) return rc;
    if (param_dtype != ET_DTYPE_F32 && param_dtype != ET_DTYPE_BF16) return fail_at(fn, "dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    if ((param_dtype == ET_DTYPE_BF16) != (masters != nullptr))
        return fail_at(fn, "bf16 parameters need f32 masters, f32 parameters take none");
    if (count > 0 && !step_sizes) return fail_at(fn, "null step_sizes");
    rc = check_list(fn, "params", (const void* const*)params, shapes, count, param_dtype == ET_DTYPE_F32 ? 4 : 2);
    if (!rc) rc = check_list(fn, "grads", grads, shapes, count, grad_dtype == ET_DTYPE_F32 ? 4 : 2);
    if (!rc) rc = check_list(fn, "momentum", (const void* const*)momentum, shapes, count, 4);
    if (!rc && masters) rc = check_list(fn, "masters", (const void* const*)masters, shapes, count, 4);
    if (!rc && (uintptr_t)grad_scale % 4) rc = fail_at(fn, "grad_scale is not aligned");
    if (!rc) rc = check_workspace(fn, shapes, count, workspace, workspace_bytes);
    if (rc) return rc;
    OrthoCall call = {};
    call.fn = fn;
    call.shapes = shapes;
    call.count = count;
    call.g = grads;
    call.mom = momentum;
    call.out = params;
    call.master = masters;
    call.step = step_sizes;
    call.dtype = grad_dtype;
    call.out_kind = param_dtype == ET_DTYPE_BF16 ? kOutMaster : kOutParam;
    call.iterations = scalars.iterations;
    call.a = scalars.a;
    call.b = scalars.b;
    call.c = scalars.c;
    OrthoList list = {};
    list.eps = scalars.eps;
    list.beta = scalars.beta;
    list.one_minus_beta = scalars.one_minus_beta;
    list.decay = scalars.decay;
    list.nesterov = scalars.nesterov;
    list.grad_scale = grad_scale;
    return run_call(call, list, (unsigned char*)workspace, (hipStream_t)stream);
}
