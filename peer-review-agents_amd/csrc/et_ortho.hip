// et_ortho.hip -- Newton-Schulz orthogonalisation of batches of matrices, and the
// optimizer step that takes it for its direction (gfx950).
//
//   X = U / (|U| + eps);  steps times:  A = X X^T,  S = a I + b A + c A A,  X = S X
//
// (X X^T over the shorter side: for more rows than columns A = X^T X and X = X S.)
// The matrices of many tensors go through one launch a product, each tile finding
// its matrix in a table.
//
// Number format.  X, A and S are held in f16 times fixed powers of two and
// multiplied on the matrix units with binary32 sums.  The largest singular value
// of X stays below 1.21 and that of S below a, for the coefficients that the host
// accepts, so no entry is larger: X and A times 2^14 and S times 2^kScaleS stay
// below f16's largest number, and entries down to 2^-28 keep all 11 bits.  A bf16
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
    int steps_only;
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
    const int64_t at0 = (int64_t)c * kChunk;
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
        for (int i = 0; i < kChunk / kDenseThreads; ++i) {
            const int64_t at = at0 + i * kDenseThreads + (int)threadIdx.x;
            if (at >= size) break;
            float v = read1<G>(t.g, base + at);
            if constexpr (MOM) {
                float w = t.mom[base + at];
                v = direction(l, v * scale, w);
                t.mom[base + at] = w;
            }
            sum += (double)v * (double)v;
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
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < t.sums; i += kDenseThreads) sum += t.partial[(int64_t)e * t.sums + i];
    sum = block_sum(sum);
    // (in binary64: the norm of values near binary32's smallest or largest is in its range)
    const double inv = (double)(1 << kScaleX) / (sqrt(sum) + (double)l.eps);
    const uint32_t row_segs = t.ldx / 8, segs = t.m * row_segs;
    uint16_t* const x = t.x + (int64_t)e * t.m * t.ldx;
#pragma unroll
    for (int i = 0; i < kChunk / (8 * kDenseThreads); ++i) {
        const uint32_t seg = c * (kChunk / 8) + i * kDenseThreads + threadIdx.x;
        if (seg >= segs) break;
        const uint32_t row = seg / row_segs, col = (seg - row * row_segs) * 8;
        const int64_t at = base + (int64_t)row * t.n + col;
        float v[8];
        if (t.wide) {
            read8<G>(t.g, at, v);
            if constexpr (MOM) {
                float m[8];
                read8<float>(t.mom, at, m);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = l.nesterov ? l.one_minus_beta * (v[j] * gs) + l.beta * m[j] : m[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.0f;
                if (col + j < t.n) {
                    v[j] = read1<G>(t.g, at + j);
                    if constexpr (MOM) {
                        const float m = t.mom[at + j];
                        v[j] = l.nesterov ? l.one_minus_beta * (v[j] * gs) + l.beta * m : m;
                    }
                }
            }
        }
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_f16x2((float)(v[2 * j] * inv), (float)(v[2 * j + 1] * inv));
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
#pragma unroll
    for (int i = 0; i < kChunk / (8 * kDenseThreads); ++i) {
        const uint32_t seg = c * (kChunk / 8) + i * kDenseThreads + threadIdx.x;
        if (seg >= segs) break;
        const uint32_t row = seg / row_segs, col = (seg - row * row_segs) * 8;
        const int64_t at = base + (int64_t)row * t.n + col;
        const f16x8_t v = *reinterpret_cast<const f16x8_t*>(x + (int64_t)seg * 8);
        if constexpr (OUT == kOutBf16) {
            if (t.wide) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2((float)v[2 * j] * unit, (float)v[2 * j + 1] * unit);
                *reinterpret_cast<u32x4_t*>((uint16_t*)t.out + at) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < t.n) ((uint16_t*)t.out)[at + j] = (uint16_t)f32_to_bf16_bits((float)v[j] * unit);
            }
        } else {
            float* const w = OUT == kOutMaster ? t.master : (float*)t.out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (t.wide) {
                    f32x4_t* const q = reinterpret_cast<f32x4_t*>(w + at) + h;
                    f32x4_t p = *q;
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = __builtin_fmaf(-step, (float)v[4 * h + j], l.decay * p[j]);
                    *q = p;
                    if constexpr (OUT == kOutMaster)
                        reinterpret_cast<u32x2_t*>((uint16_t*)t.out + at)[h] =
                            u32x2_t{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])};
                } else {
#pragma unroll
                    for (int j = 4 * h; j < 4 * h + 4; ++j)
                        if (col + j < t.n) {
                            const float p = __builtin_fmaf(-step, (float)v[j], l.decay * w[at + j]);
                            w[at + j] = p;
                            if constexpr (OUT == kOutMaster) ((uint16_t*)t.out)[at + j] = (uint16_t)f32_to_bf16_bits(p);
                        }
                }
            }
        }
    }
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

template <int SIDE, bool ACOL, bool BCOL, bool POLY>
struct OrthoPolicy {
    static constexpr int MI = SIDE, NJ = SIDE;
    static constexpr bool kACol = ACOL, kBCol = BCOL, kF16 = true;
    static constexpr int kBlocks = SIDE == 8 ? 1 : 2;
    static constexpr int BM = 32 * MI, BN = 32 * NJ;
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
        const int each = p.nm * p.nn;
        const int e = (q - p.first) / each;
        const TileAt at = tile_at(q - p.first - e * each, p.nm, p.nn, 8);
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
    __device__ static void epilogue(const Args& g, const Tile& t, f32x4_t (&acc)[MI][NJ], int wm, int wn, int r16, int rho)
    {
        const OrthoGemm& p = g.t[t.at];
        const int ldc = p.ldc;
        const int64_t first = t.e * p.sc + (int64_t)t.m0 * ldc;
        const __amdgpu_buffer_rsrc_t res = dense_rsrc(p.c + first, t.a_rows * ldc * 2);
        const __amdgpu_buffer_rsrc_t dres = dense_rsrc(POLY ? p.d + first : nullptr, t.a_rows * ldc * 2);
        const float alpha = g.alpha;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            const int row = (wm * MI + i) * 16 + r16;
            u32x2_t d[NJ];
            if constexpr (POLY) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int col = t.n0 + (wn * NJ + j) * 16 + 4 * rho;
                    d[j] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(
                        dres, row < t.a_rows && col < ldc ? (uint32_t)(row * ldc + col) * 2u : kOOR, 0, 0));
                }
            }
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                __builtin_amdgcn_sched_barrier(0);
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int jj = j + (e >> 2);
                    v[e] = acc[i][jj][e & 3] * alpha;
                    if constexpr (POLY) {
                        // (halves by a shift: as elements of a pair, hipcc 7.2 takes both words of the
                        // load for the first)
                        const uint32_t word = d[jj][(e & 3) >> 1];
                        const _Float16 w = __builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? word >> 16 : word & 0xffffu));
                        v[e] = __builtin_fmaf(g.beta, (float)w, v[e]);
                        if (t.m0 + row == t.n0 + (wn * NJ + jj) * 16 + 4 * rho + (e & 3)) v[e] += g.gamma;
                    }
                }
                store_pair<true>(v, res, row < t.a_rows, (uint32_t)(row * ldc), t.n0 + (wn * NJ + j) * 16, ldc, rho);
            }
        }
    }
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round8(int64_t n) { return up(n, 8) * 8; }

// Launches the products in `args` (nm, nn, first and tiles are set here).
template <bool ACOL, bool BCOL, bool POLY>
int launch_products(OrthoArgs& args, const int64_t* batch, hipStream_t s)
{
    const int cus = dense_cus();
    int64_t big = 0, small = 0;
    for (int i = 0; i < args.count; ++i) {
        const OrthoGemm& p = args.t[i];
        big += batch[i] * up(p.M, 256) * up(p.N, 256);
        small += batch[i] * up(p.M, 128) * up(p.N, 128);
    }
    const int side = 4 * up(big, cus) <= 3 * up(small, 2 * cus) ? 8 : 4;
    args.tiles = 0;
    for (int i = 0; i < args.count; ++i) {
        OrthoGemm& p = args.t[i];
        p.nm = (int)up(p.M, 32 * side);
        p.nn = (int)up(p.N, 32 * side);
        p.first = args.tiles;
        args.tiles += (int)batch[i] * p.nm * p.nn;
    }
    if (side == 8)
        dense_gemm_kernel<OrthoPolicy<8, ACOL, BCOL, POLY>><<<dim3(dense_grid(args.tiles, 1, cus)), dim3(kDenseThreads), 0, s>>>(args);
    else
        dense_gemm_kernel<OrthoPolicy<4, ACOL, BCOL, POLY>><<<dim3(dense_grid(args.tiles, 2, cus)), dim3(kDenseThreads), 0, s>>>(args);
    return check_launch("ortho_products");
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
    int64_t sums() const { return up(m * n, kChunk); }
    int64_t blocks() const { return std::max(sums(), up(m * ldx(), kChunk)); }
    int64_t x_bytes() const { return up(E * m * ldx() * 2, 256) * 256; }
    int64_t a_bytes() const { return up(E * r() * ldr() * 2, 256) * 256; }
    int64_t sum_bytes() const { return up(E * sums() * 8, 256) * 256; }
    int64_t bytes() const { return 2 * x_bytes() + 2 * a_bytes() + sum_bytes(); }
};

constexpr int64_t kMostSide = 1 << 16;

bool shape_ok(const Shape& s)
{
    // (a launch has less than 2^32 threads)
    if (s.E < 0 || s.m < 0 || s.n < 0 || s.m >= kMostSide || s.n >= kMostSide || s.E >= 1 << 24) return false;
    return s.E * s.m * s.n == 0 || s.E * s.blocks() < 1 << 24;
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

// One set of up to kTensors tensors of one orientation.
int run_set(const OrthoCall& call, OrthoList list, const int64_t* index, unsigned char* const* place, hipStream_t s)
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
        t.each = (uint32_t)sh.blocks();
        t.step = call.step ? call.step[k] : 0.0f;
        t.wide = sh.n % 8 == 0 && ((uintptr_t)t.g | (uintptr_t)t.mom | (uintptr_t)t.out | (uintptr_t)t.master) % 16 == 0;
        blocks += (uint32_t)(sh.E * sh.blocks());
    }
    for (const bool scale : {false, true}) {
        if (call.mom) launch_elementwise<true>(list, call.dtype, blocks, scale, s);
        else launch_elementwise<false>(list, call.dtype, blocks, scale, s);
        if (const int rc = check_launch("ortho_norm_kernel")) return rc;
    }
    // S is held times 2^scale_s, its largest singular value being below a
    int scale_s = 0;
    while (call.a * pow2(scale_s + 1) < 60000.0f) ++scale_s;
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
        args.alpha = pow2(-kScaleX);
        int rc = tall ? launch_products<true, true, false>(args, batch, s) : launch_products<false, false, false>(args, batch, s);
        if (rc) return rc;
        fill([&](OrthoGemm& p, int i, const Shape&, int r, int ldr, int) {
            p.a = p.b = p.d = ga[i];
            p.c = gs[i];
            p.sa = p.sb = p.sc = (int64_t)r * ldr;
            p.M = p.N = r;
            p.K = p.lda = p.ldb = p.ldc = ldr;
        });
        args.alpha = call.c * pow2(scale_s - 2 * kScaleX);
        args.beta = call.b * pow2(scale_s - kScaleX);
        args.gamma = call.a * pow2(scale_s);
        rc = launch_products<false, false, true>(args, batch, s);
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
        args.alpha = pow2(-scale_s);
        rc = tall ? launch_products<false, false, false>(args, batch, s) : launch_products<false, true, false>(args, batch, s);
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
        if (!shape_ok(shape_at(shapes, i))) return fail_at(fn, "sides must be in [0, 65536), and a tensor below 2^24 matrices and 2^36 elements");
    if (dtype != ET_DTYPE_F32 && dtype != ET_DTYPE_BF16) return fail_at(fn, "dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    if (iterations < 1 || iterations > 64) return fail_at(fn, "iterations must be in [1, 64]");
    if (!abc) return fail_at(fn, "null coefficients");
    if (!(eps >= 0.0f) || !(eps < __builtin_inff())) return fail_at(fn, "eps must be finite and >= 0");
    // the scaled f16 numbers hold X's singular values up to 3.9 and S's up to a
    const double a = abc[0], b = abc[1], c = abc[2];
    bool ok = a > 0.0 && a < 16.0 && __builtin_fabs(b) < 64.0 && __builtin_fabs(c) < 64.0;
    double most = 1.0;        // the largest singular value that a step can start from
    for (int it = 0; ok && it < iterations && it < 8; ++it) {
        double next = 0.0;
        for (int k = 0; k <= 4096; ++k) {
            const double s = most * k / 4096.0, f = a + b * s * s + c * s * s * s * s;
            ok = ok && __builtin_fabs(f) <= 1.01 * a;
            next = std::max(next, __builtin_fabs(f * s));
        }
        most = std::max(most, 1.01 * next);
        ok = ok && most < 1.9;
    }
    if (!ok) return fail_at(fn, "coefficients must keep singular values in [0, 1] below 1.9 and |a + b s^2 + c s^4| at most a (below 16)");
    return ET_OK;
}

int run_call(const OrthoCall& call, const OrthoList& scalars, unsigned char* workspace, hipStream_t s)
{
    for (const bool tall : {false, true}) {
        OrthoList list = scalars;
        list.count = 0;
        int64_t index[kTensors];
        unsigned char* place[kTensors];
        unsigned char* at = workspace;
        int64_t blocks = 0;
        const auto flush = [&]() -> int {
            if (!list.count) return ET_OK;
            const int rc = run_set(call, list, index, place, s);
            list.count = 0;
            blocks = 0;
            return rc;
        };
        for (int64_t i = 0; i < call.count; ++i) {
            const Shape sh = shape_at(call.shapes, i);
            unsigned char* const here = at;
            if (sh.E * sh.m * sh.n == 0) continue;
            at += sh.bytes();
            if (sh.tall() != tall) continue;
            if (list.count == kTensors || blocks + sh.E * sh.blocks() >= 1 << 24) {
                if (const int rc = flush()) return rc;
            }
            index[list.count] = i;
            place[list.count++] = here;
            blocks += sh.E * sh.blocks();
        }
        if (const int rc = flush()) return rc;
    }
    return ET_OK;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" size_t et_orthogonalize_workspace_bytes(const int64_t* shapes, int64_t count)
{
    if (count < 0 || (count > 0 && !shapes)) return 0;
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) {
        const Shape s = shape_at(shapes, i);
        if (!shape_ok(s)) return 0;
        if (s.E * s.m * s.n) n += s.bytes();
    }
    return (size_t)n;
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
