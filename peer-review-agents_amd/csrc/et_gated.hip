// et_gated.hip -- the gated projection of a dense (shared) expert, forward and
// backward (gfx950):
//
//   g = x Wg^T,  u = x Wu^T       W [2F, K]: the F gate rows, then the F up rows
//   h = act(g) * u                act: SiLU g sigmoid(g), or GELU g Phi(g)
//
//   dp = [dh u act'(g) | dh act(g)],  dx = dp W,  dW = dp^T x
//
// Forward: one kernel; a tile's weight rows are gate rows and the up rows of the
// same hidden units, so a lane holds both of a unit in its accumulators and writes
// h alone.  Backward: nothing but x and W is kept from the forward.  The same
// product runs again with dh in its epilogue, which writes dp (bf16, the one
// rounding between the two products: dp is an operand of the matrix units), and
// two products follow, dx with W read down its columns and dW with dp and x both
// read down their columns, its sum over the tokens split where there are too few
// tiles to fill the GPU.
// 65536 x 4096 x 2048: 1.71 ms forward, 1.84 + 1.65 (dx) + 1.60 (dW) backward, 1.28, 1.19, 1.33 and
// 1.37 PFLOP/s; the library's product of these sizes, without an epilogue, is at 1.56, 1.29 and
// 1.18 for the three orders of operands.  The MFMAs' rate at the clock that the card
// holds under them bounds all four.
#include "et_dense_gemm.hpp"
#include "etmoe_dense.h"

namespace et {
namespace {

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr float kRootHalf = 0.70710678118654752f, kInvRoot2Pi = 0.39894228040143268f;

// Phi(g), the normal distribution function, and e = exp(-g^2 / 2).  With x = |g| / sqrt 2 and
// u = 1 / (1 + x / 2), erfc(x) = u 2^q(u) exp(-x^2): q is the degree-9 Chebyshev fit of
// log2(erfc(x) exp(x^2) / u) for x in [0, 10], 5e-8 of erfc off (3e-7 in binary32), and
// exp(-87) and below are 0.  The exponent's rounding error is taken out by an fma, so
// the relative error is the same far out on the left, where 1 + erf would cancel.
// (Instead of erfcf and expf with their branches for each range: the backward's kernel of
// projections 27.6 to 25.6 us at 3001 x 1000 x 712, the forward 24.2 to 24.0.)
__device__ __forceinline__ float normal_distribution(float g, float& e)
{
    const float a = __builtin_fminf(__builtin_fabsf(g), 16.0f);
    const float hi = 0.5f * a * a;
    e = exp_neg_abs(hi);
    e = __builtin_fmaf(-e, __builtin_fmaf(0.5f * a, a, -hi), e);
    const float u = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f * kRootHalf, __builtin_fabsf(g), 1.0f));
    float q = 0.209090101f;
    q = __builtin_fmaf(q, u, -0.982225993f);
    q = __builtin_fmaf(q, u, 1.66881405f);
    q = __builtin_fmaf(q, u, -1.00447916f);
    q = __builtin_fmaf(q, u, -0.115820182f);
    q = __builtin_fmaf(q, u, 0.0018287411f);
    q = __builtin_fmaf(q, u, 0.0499212878f);
    q = __builtin_fmaf(q, u, 0.557804205f);
    q = __builtin_fmaf(q, u, 1.44072256f);
    q = __builtin_fmaf(q, u, -1.82565555f);
    const float tail = 0.5f * u * __builtin_amdgcn_exp2f(q) * e;
    return g < 0.0f ? tail : 1.0f - tail;
}

// act(g) and, for the backward, act'(g).
// SiLU: s = sigmoid(g), g s, s (1 + g (1 - s)).  GELU: g Phi, Phi + g phi.
template <int ACT>
__device__ __forceinline__ float gate_value(float g)
{
    float e;
    if constexpr (ACT == ET_GATED_SILU) return g * sigmoid(g);
    else return g * normal_distribution(g, e);
}

template <int ACT>
__device__ __forceinline__ void gate_slope(float g, float& value, float& slope)
{
    if constexpr (ACT == ET_GATED_SILU) {
        const float s = sigmoid(g);
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else {
        float e;
        const float p = normal_distribution(g, e);
        value = g * p;
        slope = p + g * (kInvRoot2Pi * e);
    }
}

struct GatedArgs {
    const unsigned char* x;    // [T, K], row stride ldx
    const unsigned char* w;    // [2F, K]
    uint16_t* out;             // h [T, F], or dp [T, 2F]
    const uint16_t* dh;        // [T, F]
    int64_t T;
    int ldx, K, F;
    int nm, nn;
};

// x (rows) times gate and up rows: a wave's first NJ / 2 tiles are gate rows, the
// others the up rows of the same hidden units.
template <int KIND, int ACT, bool BACKWARD>
struct GatedPolicy : DenseTile<KIND, 4> {
    using DenseTile<KIND, 4>::MI;
    using DenseTile<KIND, 4>::NJ;
    static constexpr bool kACol = false, kBCol = false, kF16 = false, kMid = true;
    static constexpr int kScratch = 0;
    static constexpr int BM = 32 * MI, BH = 16 * NJ;      // rows and hidden units of a tile
    using Args = GatedArgs;
    struct Tile : GemmTile {
        int64_t m0;
        int n0;
    };
    __device__ static int tiles(const Args& g) { return g.nm * g.nn; }
    __device__ static void tile(const Args& g, int q, Tile& t)
    {
        const TileAt at = tile_at(q, g.nm, g.nn, 8);
        t.m0 = (int64_t)at.m * BM;
        t.n0 = at.n * BH;
        t.a = g.x + t.m0 * g.ldx * 2;
        t.b = g.w;
        t.a_rows = (int)min<int64_t>(BM, g.T - t.m0);
        t.b_rows = 2 * g.F;
        t.lda = g.ldx;
        t.ldb = g.K;
        t.k = g.K;
    }
    // the weight row of the tile's rows R ..  R + 7 (F is a multiple of 8)
    __device__ static int b_row(const Args& g, const Tile& t, int R)
    {
        const int tt = (R % (16 * NJ)) / 16;
        const int hid = t.n0 + R / (16 * NJ) * (8 * NJ) + tt % (NJ / 2) * 16 + (R & 15);
        return hid < g.F ? (tt >= NJ / 2 ? g.F + hid : hid) : -1;
    }
    __device__ static void epilogue(const Args& g, const Tile& t, f32x4_t (&acc)[MI][NJ], int wm, int wn, int r16, int rho, unsigned char*)
    {
        const int F = g.F;
        const int width = BACKWARD ? 2 * F : F;
        const __amdgpu_buffer_rsrc_t res = dense_rsrc(g.out + t.m0 * width, t.a_rows * width * 2);
        const __amdgpu_buffer_rsrc_t dres = dense_rsrc(BACKWARD ? g.dh + t.m0 * F : nullptr, t.a_rows * F * 2);
        const int c0 = t.n0 + wn * (8 * NJ);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            __builtin_amdgcn_sched_barrier(0);       // one row tile at a time: few temporaries
            const int row = (wm * MI + i) * 16 + r16;
            const bool ok = row < t.a_rows;
            u32x2_t d[NJ / 2];
            if constexpr (BACKWARD) {
#pragma unroll
                for (int j = 0; j < NJ / 2; ++j) {
                    const int col = c0 + j * 16 + 4 * rho;
                    d[j] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(
                        dres, ok && col < F ? (uint32_t)(row * F + col) * 2u : kOOR, 0, 0));
                }
            }
#pragma unroll
            for (int j = 0; j < NJ / 2; j += 2) {
                float v[8], w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int jj = j + (e >> 2);
                    const float gate = acc[i][jj][e & 3], up = acc[i][jj + NJ / 2][e & 3];
                    if constexpr (BACKWARD) {
                        const uint32_t word = d[jj][(e & 3) >> 1];
                        const float dh = (e & 1) ? bf16hi(word) : bf16lo(word);
                        float value, slope;
                        gate_slope<ACT>(gate, value, slope);
                        v[e] = dh * up * slope;
                        w[e] = dh * value;
                    } else {
                        v[e] = gate_value<ACT>(gate) * up;
                    }
                }
                store_pair<false>(v, res, ok, (uint32_t)(row * width), c0 + j * 16, F, rho);
                if constexpr (BACKWARD)
                    store_pair<false>(w, res, ok, (uint32_t)(row * width + F), c0 + j * 16, F, rho);
            }
        }
    }
};

// The forward of few tokens, where reading the weight is the work.  A block
// owns 8 hidden units, whose gate and up rows fill one MFMA tile of 16 rows, and
// TT tiles of 16 tokens; its 8 waves take K's chunks of 64 in turn, each through a
// ring of D stages of LDS of its own (no barriers), and their sums meet in LDS.
// F = 2048 then makes a block for each CU.  A direct load fills 8 rows x 128
// bytes: whole cache lines.  (Loads straight into the operands' registers take 16
// rows x 64 bytes, which move 14 bytes a cycle and CU: 64 tokens took 23 us at
// K = 4096, F = 2048.)  What lies past K and the tokens reads 0, without traffic.
constexpr int kSkinnyWaves = 8;

template <int TT, int D, int ACT>
__global__ __launch_bounds__(kSkinnyWaves * kWave) void gated_skinny_kernel(GatedArgs g)
{
    constexpr int kStageBytes = (1 + TT) * 2048, NI = 2 * (1 + TT);
    constexpr int kRing = kSkinnyWaves * D * kStageBytes, kPart = kSkinnyWaves * TT * kWave * 16;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kRing > kPart ? kRing : kPart];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int r16 = lane & 15, rho = lane >> 4;
    const int hid0 = (int)blockIdx.x * 8;
    const int m0 = (int)blockIdx.y * (16 * TT);
    const int T = min(16 * TT, (int)g.T - m0), K = g.K, F = g.F;
    const __amdgpu_buffer_rsrc_t wres = dense_rsrc(g.w, 2 * F * K * 2);
    const __amdgpu_buffer_rsrc_t xres = dense_rsrc(g.x + (int64_t)m0 * g.ldx * 2, ((T - 1) * g.ldx + K) * 2);
    unsigned char* const mine = smem + wave * (D * kStageBytes);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t*)mine;
    const int seg0 = (lane & 7) ^ (lane >> 3);
    // chunk j of the wave: k from (8 j + wave) 64 on
    const auto load = [&](int j, uint32_t lds) {
        const int k0 = (kSkinnyWaves * j + wave) * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = k0 + (seg0 ^ i) * 8;
            const uint32_t row = (uint32_t)((i ? F : 0) + hid0 + (lane >> 3));
            dense_dma(wres, k < K ? (row * (uint32_t)K + (uint32_t)k) * 2u : kOOR, 0u, lds + i * 1024);
        }
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = k0 + (seg0 ^ i) * 8;
                const uint32_t row = (uint32_t)(16 * t + 8 * i + (lane >> 3));
                dense_dma(xres, k < K && (int)row < T ? (row * (uint32_t)g.ldx + (uint32_t)k) * 2u : kOOR, 0u,
                          lds + (1 + t) * 2048 + i * 1024);
            }
    };
    f32x4_t acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = f32x4_t{};
    const int turns = (K + kSkinnyWaves * 64 - 1) / (kSkinnyWaves * 64);
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, lds0 + d * kStageBytes);
    const int fkey = (lane & 7) ^ ((lane >> 3) & 1);
    const int frow = (r16 >> 3) * 1024 + (lane & 7) * 128;
    for (int j = 0, stage = 0; j < turns; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * NI) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        const unsigned char* const at = mine + stage * kStageBytes;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const auto read = [&](int tile) {
                return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(at + tile * 2048 + frow + (((4 * ks + rho) ^ fkey) << 4)));
            };
            const bf16x8_t fw = read(0);
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, read(1 + t), acc[t], 0, 0, 0);
        }
        // (the reads above have ended: their results were used.  Chunks past K load
        // nothing, so that the count of loads in flight is the same)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
        load(j + D, lds0 + stage * kStageBytes);
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    dense_wait_barrier<0>();
    f32x4_t* const part = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
    for (int t = 0; t < TT; ++t) part[(wave * TT + t) * kWave + lane] = acc[t];
    __syncthreads();
    // (row r of the tile, token c: lane 16 (r / 4) + c, element r % 4)
    for (int q = (int)threadIdx.x; q < TT * 128; q += kSkinnyWaves * kWave) {
        const int token = q >> 3, h = q & 7;
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int w = 0; w < kSkinnyWaves; ++w) {
            const f32x4_t* const p = part + (w * TT + (token >> 4)) * kWave + 16 * (h >> 2) + (token & 15);
            gate += p[0][h & 3];
            up += p[32][h & 3];
        }
        if (token < T) g.out[(int64_t)(m0 + token) * F + hid0 + h] = (uint16_t)f32_to_bf16_bits(gate_value<ACT>(gate) * up);
    }
}

template <int ACT>
void launch_skinny(const GatedArgs& g, hipStream_t s)
{
    const dim3 grid((unsigned)(g.F / 8), (unsigned)up(g.T, 64)), block(kSkinnyWaves * kWave);
    if (g.T <= 16) gated_skinny_kernel<1, 4, ACT><<<grid, block, 0, s>>>(g);
    else if (g.T <= 32) gated_skinny_kernel<2, 3, ACT><<<grid, block, 0, s>>>(g);
    else gated_skinny_kernel<4, 2, ACT><<<grid, block, 0, s>>>(g);
}

// dx [T, K] = dp [T, 2F] W, W read down its columns.
struct InputGradArgs {
    const unsigned char* dp;
    const unsigned char* w;
    uint16_t* dx;
    int64_t T;
    int K, F;
    int nm, nn;
};

template <int KIND>
struct InputGradPolicy : DenseTile<KIND, 4> {
    using DenseTile<KIND, 4>::MI;
    using DenseTile<KIND, 4>::NJ;
    static constexpr bool kACol = false, kBCol = true, kF16 = false, kMid = true;
    static constexpr int kScratch = 0;
    static constexpr int BM = 32 * MI, BN = 32 * NJ;
    using Args = InputGradArgs;
    struct Tile : GemmTile {
        int64_t m0;
        int n0;
    };
    __device__ static int tiles(const Args& g) { return g.nm * g.nn; }
    __device__ static void tile(const Args& g, int q, Tile& t)
    {
        const TileAt at = tile_at(q, g.nm, g.nn, 8);
        t.m0 = (int64_t)at.m * BM;
        t.n0 = at.n * BN;
        t.a = g.dp + t.m0 * (2 * g.F) * 2;
        t.b = g.w + (int64_t)t.n0 * 2;
        t.a_rows = (int)min<int64_t>(BM, g.T - t.m0);
        t.b_rows = min(BN, g.K - t.n0);
        t.lda = 2 * g.F;
        t.ldb = g.K;
        t.k = 2 * g.F;
    }
    __device__ static int b_row(const Args&, const Tile&, int) { return -1; }
    __device__ static void epilogue(const Args& g, const Tile& t, f32x4_t (&acc)[MI][NJ], int wm, int wn, int r16, int rho, unsigned char*)
    {
        const __amdgpu_buffer_rsrc_t res = dense_rsrc(g.dx + t.m0 * g.K, t.a_rows * g.K * 2);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = (wm * MI + i) * 16 + r16;
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                __builtin_amdgcn_sched_barrier(0);
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][j + (e >> 2)][e & 3];
                store_pair<false>(v, res, row < t.a_rows, (uint32_t)(row * g.K), t.n0 + (wn * NJ + j) * 16, g.K, rho);
            }
        }
    }
};

// dW [2F, K] = dp^T x over tokens [split * step, + step): bf16, or f32 (dW itself,
// or a split's partial sums).
struct WeightGradArgs {
    const unsigned char* dp;   // [T, 2F]
    const unsigned char* x;    // [T, K], row stride ldx
    void* dw;                  // [splits, 2F, K]
    int64_t T, step;
    int ldx, K, F;
    int nm, nn, splits;
    bool f32;
};

template <int KIND>
struct WeightGradPolicy : DenseTile<KIND, 4> {
    using DenseTile<KIND, 4>::MI;
    using DenseTile<KIND, 4>::NJ;
    static constexpr bool kACol = true, kBCol = true, kF16 = false, kMid = false;
    static constexpr int kScratch = 0;
    static constexpr int BM = 32 * MI, BN = 32 * NJ;
    using Args = WeightGradArgs;
    struct Tile : GemmTile {
        int split, m0, n0;
    };
    __device__ static int tiles(const Args& g) { return g.nm * g.nn * g.splits; }
    __device__ static void tile(const Args& g, int q, Tile& t)
    {
        t.split = q / (g.nm * g.nn);
        const TileAt at = tile_at(q - t.split * (g.nm * g.nn), g.nm, g.nn, 8);
        t.m0 = at.m * BM;
        t.n0 = at.n * BN;
        const int64_t k0 = t.split * g.step;
        t.a = g.dp + (k0 * (2 * g.F) + t.m0) * 2;
        t.b = g.x + (k0 * g.ldx + t.n0) * 2;
        t.a_rows = min(BM, 2 * g.F - t.m0);
        t.b_rows = min(BN, g.K - t.n0);
        t.lda = 2 * g.F;
        t.ldb = g.ldx;
        t.k = (int)min<int64_t>(g.step, g.T - k0);
    }
    __device__ static int b_row(const Args&, const Tile&, int) { return -1; }
    __device__ static void epilogue(const Args& g, const Tile& t, f32x4_t (&acc)[MI][NJ], int wm, int wn, int r16, int rho, unsigned char*)
    {
        const int es = g.f32 ? 4 : 2;
        const int64_t first = ((int64_t)t.split * 2 * g.F + t.m0) * g.K;
        const __amdgpu_buffer_rsrc_t res = dense_rsrc((unsigned char*)g.dw + first * es, t.a_rows * g.K * es);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = (wm * MI + i) * 16 + r16;
            if (g.f32) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int col = t.n0 + (wn * NJ + j) * 16 + 4 * rho;
                    const uint32_t off = row < t.a_rows && col < g.K ? (uint32_t)(row * g.K + col) * 4u : kOOR;
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[i][j]), res, off, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NJ; j += 2) {
                    __builtin_amdgcn_sched_barrier(0);
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[i][j + (e >> 2)][e & 3];
                    store_pair<false>(v, res, row < t.a_rows, (uint32_t)(row * g.K), t.n0 + (wn * NJ + j) * 16, g.K, rho);
                }
            }
        }
    }
};

// The splits' partial sums added in order (n a multiple of 8).
__global__ __launch_bounds__(kDenseThreads) void gated_fold_kernel(const float* partial, int64_t n, int splits, void* dw, bool f32)
{
    for (int64_t at = ((int64_t)blockIdx.x * kDenseThreads + threadIdx.x) * 4; at < n;
         at += (int64_t)gridDim.x * kDenseThreads * 4) {
        f32x4_t v = *reinterpret_cast<const f32x4_t*>(partial + at);
        for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4_t*>(partial + s * n + at);
        if (f32) *reinterpret_cast<f32x4_t*>((float*)dw + at) = v;
        else *reinterpret_cast<u32x2_t*>((uint16_t*)dw + at) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
}

__global__ __launch_bounds__(kDenseThreads) void gated_zero_kernel(uint32_t* p, int64_t words)
{
    for (int64_t at = (int64_t)blockIdx.x * kDenseThreads + threadIdx.x; at < words; at += (int64_t)gridDim.x * kDenseThreads)
        p[at] = 0u;
}

template <int KIND> using SiluFwd = GatedPolicy<KIND, ET_GATED_SILU, false>;
template <int KIND> using GeluFwd = GatedPolicy<KIND, ET_GATED_GELU, false>;
template <int KIND> using SiluBwd = GatedPolicy<KIND, ET_GATED_SILU, true>;
template <int KIND> using GeluBwd = GatedPolicy<KIND, ET_GATED_GELU, true>;

// Rows and columns of a kind's tiles.
int rows_of(int kind) { return kind == kTileBig ? 256 : kind == kTileMid ? 192 : kind == kTileSmall ? 128 : 64; }
int cols_of(int kind) { return kind == kTileBig ? 256 : 128; }

// The tiles of a product of m x n outputs.
DenseChoice choice_of(int64_t m, int64_t n)
{
    return dense_choice(up(m, 256) * up(n, 256), up(m, 192) * up(n, 128), up(m, 128) * up(n, 128), up(m, 64) * up(n, 128), true,
                        dense_cus());
}
int kind_of(int64_t m, int64_t n) { return choice_of(m, n).kind; }

// Few tokens or tiles: what their rounds take.  A round of few tokens' blocks (one a CU) is 2 us
// and, for each 512 of K, 0.7, 0.9 or 1.0 us with 16, 32 or 64 tokens a block; tiles take
// dense_choice's cost for each chunk of 64, 10% more beside the epilogue, and 7 chunks besides.
// Measured in us, few tokens' blocks / tiles, another weight each call: K = 512, F = 2048, 64
// tokens 5.0 / 7.6, 128 8.0 / 7.6, 192 11.0 / 7.7; F = 8192, 8 tokens 11.7 / 8.8; K = 2048, F =
// 256, 1024 tokens 13.0 / 16.9, 1536 18.4 / 17.0; K = 4096, F = 2048, 8 tokens 9.4 / 35.9, 64
// 14.5 / 38.3, 192 32.6 / 38.4, 256 41.5 / 38.1; K = 7168, F = 8192, 17 tokens 53 / 69.  Over 900
// sizes (K 512 to 7168, F 64 to 8192, up to 6000 tokens) the choice is 8% from the faster one at
// most.  Above 2048 tokens the XCDs' readings of x, each of all of it, take longer than the tiles
// do (K = 7168, F = 64: 2048 tokens 34 / 48, 4096 65 / 48).
bool is_skinny(int64_t T, int64_t K, int64_t F)
{
    if (T > 2048) return false;
    const int64_t rounds = up(F / 8 * up(T, 64), dense_cus());
    const int64_t skinny = rounds * (200 + (T <= 16 ? 70 : T <= 32 ? 90 : 100) * up(K, 512));
    return skinny * 10 <= choice_of(T, 2 * F).cost * (11 * up(K, 64) + 70);
}

// What is wrong with the sizes, or null.
const char* size_error(int64_t T, int64_t K, int64_t F)
{
    if (T < 0 || T >= (int64_t)1 << 31) return "rows must be in [0, 2^31)";
    if (K < 8 || K % 8 || K >= 1 << 21) return "K must be a positive multiple of 8 below 2^21";
    if (F < 8 || F % 8 || F >= 1 << 20) return "F must be a positive multiple of 8 below 2^20";
    if (2 * F * K * 2 >= (int64_t)1 << 31) return "the weight must be below 2 GiB";
    return nullptr;
}

int check_sizes(const char* fn, int64_t T, int64_t K, int64_t F, int64_t ldx, int act)
{
    const std::string at = std::string(fn) + ": ";
    if (const char* const error = size_error(T, K, F)) return fail(ET_ERR_INVALID_ARGUMENT, at + error);
    if (ldx < K || ldx % 8 || ldx >= 1 << 22)
        return fail(ET_ERR_INVALID_ARGUMENT, at + "the row stride of x must be a multiple of 8, at least K and below 2^22");
    if (act != ET_GATED_SILU && act != ET_GATED_GELU) return fail(ET_ERR_INVALID_ARGUMENT, at + "unknown activation");
    return ET_OK;
}

int check_pointer(const char* fn, const char* name, const void* p)
{
    if (!p) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null " + name);
    if ((uintptr_t)p % 16) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + name + " must be 16-byte aligned");
    return ET_OK;
}

// kind: the tiles (0: by size)
int launch_gated(GatedArgs g, int act, bool backward, int kind, hipStream_t s)
{
    if (kind == 0 && !backward && is_skinny(g.T, g.K, g.F)) {
        if (act == ET_GATED_SILU) launch_skinny<ET_GATED_SILU>(g, s);
        else launch_skinny<ET_GATED_GELU>(g, s);
        return check_launch("gated_skinny_kernel");
    }
    if (kind == 0) kind = kind_of(g.T, 2 * g.F);
    g.nm = (int)up(g.T, rows_of(kind));
    g.nn = (int)up(g.F, cols_of(kind) / 2);
    const int64_t tiles = (int64_t)g.nm * g.nn;
    const int cus = dense_cus();
    if (act == ET_GATED_SILU)
        return backward ? launch_dense<SiluBwd>(g, kind, tiles, cus, s, "gated_backward")
                        : launch_dense<SiluFwd>(g, kind, tiles, cus, s, "gated_linear");
    return backward ? launch_dense<GeluBwd>(g, kind, tiles, cus, s, "gated_backward")
                    : launch_dense<GeluFwd>(g, kind, tiles, cus, s, "gated_linear");
}

// Splits of dW's sum over the tokens: a block takes its share of the chunks of 64 that
// the launch has, of dW and of `others`, 8 chunks at least.
struct Split {
    int kind, splits;
    int64_t step;
};
Split split_tokens(int64_t T, int64_t K, int64_t F, int64_t others = 0)
{
    const int cus = dense_cus();
    if (up(2 * F, 256) * up(K, 256) * 4 >= 3 * cus) return {kTileBig, 1, T};
    const int64_t tiles = up(2 * F, 128) * up(K, 128), chunks = std::max<int64_t>(1, up(T, 64));
    const int64_t share = std::max<int64_t>(8, up(tiles * chunks + others, 2 * cus));
    const int64_t step = up(chunks, std::max<int64_t>(1, up(chunks, share))) * 64;
    return {kTileSmall, (int)std::max<int64_t>(1, up(T, step)), step};
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" int et_gated_linear_impl(const void* x, int64_t x_stride, const void* w, int64_t rows, int64_t K, int64_t F,
                                    int activation, void* h, int kind, void* stream)
{
    const char* fn = "et_gated_linear";
    int rc = check_sizes(fn, rows, K, F, x_stride, activation);
    if (rc || rows == 0) return rc;
    for (const auto& [p, name] : {std::pair<const void*, const char*>{x, "x"}, {w, "w"}, {h, "h"}}) {
        rc = check_pointer(fn, name, p);
        if (rc) return rc;
    }
    GatedArgs g = {};
    g.x = (const unsigned char*)x;
    g.w = (const unsigned char*)w;
    g.out = (uint16_t*)h;
    g.T = rows;
    g.ldx = (int)x_stride;
    g.K = (int)K;
    g.F = (int)F;
    return launch_gated(g, activation, false, kind, (hipStream_t)stream);
}

extern "C" int et_gated_linear(const void* x, int64_t x_stride, const void* w, int64_t rows, int64_t K, int64_t F,
                               int activation, void* h, void* stream)
{
    return et_gated_linear_impl(x, x_stride, w, rows, K, F, activation, h, 0, stream);
}

extern "C" size_t et_gated_linear_bwd_workspace_bytes(int64_t rows, int64_t K, int64_t F)
{
    if (size_error(rows, K, F)) return 0;
    const Split sp = split_tokens(rows, K, F);
    const size_t dp = (size_t)up(rows * 2 * F * 2, 256) * 256;
    return dp + (sp.splits > 1 ? (size_t)sp.splits * 2 * F * K * 4 : 0);
}

extern "C" int et_gated_linear_bwd(const void* dh, const void* x, int64_t x_stride, const void* w, int64_t rows, int64_t K,
                                   int64_t F, int activation, void* dx, void* dw, int dw_dtype, void* workspace,
                                   size_t workspace_bytes, void* stream)
{
    const char* fn = "et_gated_linear_bwd";
    int rc = check_sizes(fn, rows, K, F, x_stride, activation);
    if (rc) return rc;
    if (dw_dtype != ET_DTYPE_F32 && dw_dtype != ET_DTYPE_BF16)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_gated_linear_bwd: dw_dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    hipStream_t s = (hipStream_t)stream;
    const bool f32 = dw_dtype == ET_DTYPE_F32;
    if (dw && (rc = check_pointer(fn, "dw", dw))) return rc;
    if (rows == 0) {
        if (!dw) return ET_OK;
        const int64_t words = 2 * F * K * (f32 ? 4 : 2) / 4;
        gated_zero_kernel<<<dim3((unsigned)std::min<int64_t>(1024, up(words, kDenseThreads))), dim3(kDenseThreads), 0, s>>>(
            (uint32_t*)dw, words);
        return check_launch("gated_zero_kernel");
    }
    for (const auto& [p, name] : {std::pair<const void*, const char*>{dh, "dh"}, {x, "x"}, {w, "w"}}) {
        rc = check_pointer(fn, name, p);
        if (rc) return rc;
    }
    if (dx && (rc = check_pointer(fn, "dx", dx))) return rc;
    const size_t need = et_gated_linear_bwd_workspace_bytes(rows, K, F);
    if (workspace_bytes < need) return fail(ET_ERR_WORKSPACE_TOO_SMALL, "et_gated_linear_bwd: workspace needs " + std::to_string(need) + " bytes");
    if ((rc = check_pointer(fn, "workspace", workspace))) return rc;
    unsigned char* const dp = (unsigned char*)workspace;
    GatedArgs g = {};
    g.x = (const unsigned char*)x;
    g.w = (const unsigned char*)w;
    g.out = (uint16_t*)dp;
    g.dh = (const uint16_t*)dh;
    g.T = rows;
    g.ldx = (int)x_stride;
    g.K = (int)K;
    g.F = (int)F;
    rc = launch_gated(g, activation, true, 0, s);
    if (rc) return rc;
    const int cus = dense_cus();
    const int kind = kind_of(rows, K);
    const Split sp = split_tokens(rows, K, F, dx && kind != kTileBig ? up(rows, 128) * up(K, 128) * up(2 * F, 64) : 0);
    InputGradArgs a = {};
    a.dp = dp;
    a.w = (const unsigned char*)w;
    a.dx = (uint16_t*)dx;
    a.T = rows;
    a.K = (int)K;
    a.F = (int)F;
    WeightGradArgs b = {};
    b.dp = dp;
    b.x = (const unsigned char*)x;
    float* const partial = (float*)(dp + up(rows * 2 * F * 2, 256) * 256);
    b.dw = sp.splits > 1 ? (void*)partial : dw;
    b.f32 = f32 || sp.splits > 1;
    b.T = rows;
    b.step = sp.step;
    b.splits = sp.splits;
    b.ldx = (int)x_stride;
    b.K = (int)K;
    b.F = (int)F;
    const auto lay_out = [](auto& g, int64_t m, int64_t n, int kind) {
        g.nm = (int)up(m, rows_of(kind));
        g.nn = (int)up(n, cols_of(kind));
        return (int64_t)g.nm * g.nn;
    };
    if (dx && dw && kind != kTileBig && sp.kind == kTileSmall) {
        // In one launch, where neither has tiles for the whole GPU: its tail is the other's
        // work (3001 x 1000 x 712: 28 us for 18 and 19).  dW's blocks, which may be the
        // longer ones, come first.
        const int64_t ta = lay_out(a, rows, K, kTileSmall), tb = lay_out(b, 2 * F, K, kTileSmall) * sp.splits;
        const unsigned first = dense_grid(tb, 2, cus), second = dense_grid(ta, 2, cus);
        dense_pair_kernel<WeightGradPolicy<kTileSmall>, InputGradPolicy<kTileSmall>>
            <<<dim3(first + second), dim3(kDenseThreads), 0, s>>>(b, a, (int)first);
        rc = check_launch("gated_gradients");
        if (rc) return rc;
    } else {
        if (dx) rc = launch_dense<InputGradPolicy>(a, kind, lay_out(a, rows, K, kind), cus, s, "gated_input_grad");
        if (!rc && dw) {
            const int64_t tiles = lay_out(b, 2 * F, K, sp.kind) * sp.splits;
            const dim3 block(kDenseThreads), grid(dense_grid(tiles, sp.kind == kTileBig ? 1 : 2, cus));
            if (sp.kind == kTileBig) dense_gemm_kernel<WeightGradPolicy<kTileBig>><<<grid, block, 0, s>>>(b);
            else dense_gemm_kernel<WeightGradPolicy<kTileSmall>><<<grid, block, 0, s>>>(b);
            rc = check_launch("gated_weight_grad");
        }
        if (rc) return rc;
    }
    if (dw) {
        if (sp.splits > 1) {
            const int64_t n = 2 * F * K;
            gated_fold_kernel<<<dim3((unsigned)std::min<int64_t>(4096, up(n, 4 * kDenseThreads))), dim3(kDenseThreads), 0, s>>>(
                partial, n, sp.splits, dw, f32);
            rc = check_launch("gated_fold_kernel");
        }
    }
    return rc;
}
