// et_layer_norm.hip -- layer norm over rows, with the residual add before it,
// and its backward with the reductions of the weight's and bias's gradients
// (gfx950).
#include <algorithm>
#include <cmath>

#include "et_common.hpp"
#include "etmoe_block.h"

namespace et {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// 16 bytes at an address aligned to the element only: rows may start anywhere
// (one global_load_dwordx4 all the same; a row that starts at a 16-byte
// address costs no more than with an aligned type).
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// An element type: V of them in 16 bytes.
template <typename X>
struct Elem {
    static constexpr int V = 16 / sizeof(X);
    static __device__ __forceinline__ float get(u32x4_t w, int j)
    {
        if constexpr (sizeof(X) == 2) return j & 1 ? bf16hi(w[j >> 1]) : bf16lo(w[j >> 1]);
        else return u2f(w[j]);
    }
    static __device__ __forceinline__ u32x4_t pack(const float (&v)[V])
    {
        if constexpr (sizeof(X) == 2)
            return u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                           pack_bf16x2(v[6], v[7])};
        else
            return u32x4_t{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
    }
    static __device__ __forceinline__ float to_float(X x)
    {
        if constexpr (sizeof(X) == 2) return u2f((uint32_t)x << 16);
        else return x;
    }
    static __device__ __forceinline__ X from_float(float v)
    {
        if constexpr (sizeof(X) == 2) return (X)f32_to_bf16_bits(v);
        else return v;
    }
};

// A row dealt to TPR threads: NV whole vectors of V elements each (vector t +
// TPR i to thread t), and the d % V elements behind them one to a thread.
template <typename X, int TPR, int NV>
struct Row {
    static constexpr int V = Elem<X>::V;
    u32x4_t v[NV];
    float tail;
    X raw;

    __device__ __forceinline__ void load(const X* row, int d, int t)
    {
        const int nvec = d / V;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = u32x4_t{};
            const int k = t + TPR * i;
            if (k < nvec) v[i] = *reinterpret_cast<const u32x4_any_t*>(row + (int64_t)k * V);
        }
        tail = 0.0f;
        if (t < d % V) tail = Elem<X>::to_float(row[nvec * V + t]);
    }
    // The same without a branch, so that rows can be loaded ahead of the one
    // that is worked on (behind branches every wait is for all loads): what a
    // thread does not have is read from the row's last vector or element and
    // replaced by 0.  d >= V; TAIL: d is no multiple of V.
    template <bool TAIL>
    __device__ __forceinline__ void load_ahead(const X* row, int d, int t)
    {
        const int nvec = d / V;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = t + TPR * i;
            v[i] = *reinterpret_cast<const u32x4_any_t*>(row + (int64_t)min(k, nvec - 1) * V);
        }
        if constexpr (TAIL) raw = row[min(nvec * V + t, d - 1)];
    }
    template <bool TAIL>
    __device__ __forceinline__ void settle(int d, int t)
    {
        const int nvec = d / V;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = t + TPR * i < nvec ? v[i] : u32x4_t{};
        tail = TAIL && t < d % V ? Elem<X>::to_float(raw) : 0.0f;
    }
    // f(vector, its first column, whether the row holds it) and g(tail, its column), in a fixed order
    template <typename F, typename G>
    __device__ __forceinline__ void each(int d, int t, F f, G g)
    {
        const int nvec = d / V;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = t + TPR * i;
            if (k < nvec) f(v[i], k * V, i);
        }
        if (t < d % V) g(tail, nvec * V + t);
    }
};

template <typename W, int V>
__device__ __forceinline__ void load_weights(const W* w, int col, float (&out)[V])
{
    if constexpr (sizeof(W) == 2) {
        static_assert(V == 8, "bf16 weights go with bf16 rows");
        const u32x4_t u = *reinterpret_cast<const u32x4_any_t*>(w + col);
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = Elem<W>::get(u, j);
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const f32x4_any_t u = *reinterpret_cast<const f32x4_any_t*>(w + col + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[j + i] = u[i];
        }
    }
}

// Sums over the threads of a row: a wave's lanes, then its waves through LDS
// (the caller's slots; one barrier).  Every thread gets the same bits.
template <int WPR, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float (*slots)[N], int wave)
{
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = wave_sum_dpp(s[j]);
    if constexpr (WPR > 1) {
        if (lane_id() == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) slots[wave][j] = s[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            s[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) s[j] += slots[w][j];
        }
    }
}

struct FwdArgs {
    const void* x;
    const void* residual;     // or null
    const void* weight;
    const void* bias;         // or null
    void* y;
    void* sum;                // with a residual
    float* mean;              // or null
    float* rstd;
    int64_t ldx, ldr, T;
    int d;
    float eps;
};

// mean = sum x / d, v = sum (x - mean)^2 / d, y = (x - mean) / sqrt(v + eps) w + b, of
// x + residual where there is one.  WPR waves per row; blocks of one row, or of four waves.
// The row stays in registers, so it is read once and v is of centred values; HBM bounds
// it (65536 x 4096 bf16 with a residual and the sum, 2.15 GB, 370 us, 5.8 TB/s; 8 rows
// of 4096 4.1 us, of which 1.7 are an empty launch).
constexpr int norm_threads(int wpr) { return wpr > 4 ? wpr * kWave : 256; }

template <typename X, typename W, int WPR, int NV>
__global__ __launch_bounds__(norm_threads(WPR)) void layer_norm_fwd_kernel(FwdArgs a)
{
    constexpr int TPR = WPR * kWave, V = Elem<X>::V, kRows = norm_threads(WPR) / TPR;
    __shared__ float slots[2][WPR][1];
    const int t = (int)threadIdx.x % TPR, wave = t / kWave;
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    if (row >= a.T) return;               // (whole waves; whole blocks where there are barriers)
    const int d = a.d;
    Row<X, TPR, NV> r;
    r.load((const X*)a.x + row * a.ldx, d, t);
    if (a.residual) {
        Row<X, TPR, NV> q;
        q.load((const X*)a.residual + row * a.ldr, d, t);
        X* const sum = (X*)a.sum + row * d;
        r.each(
            d, t,
            [&](u32x4_t& v, int col, int i) {
                float s[V];
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] = Elem<X>::get(v, j) + Elem<X>::get(q.v[i], j);
                v = Elem<X>::pack(s);
                *reinterpret_cast<u32x4_any_t*>(sum + col) = v;
            },
            [&](float& v, int col) {
                const X s = Elem<X>::from_float(v + q.tail);
                sum[col] = s;
                v = Elem<X>::to_float(s);
            });
    }
    float s[1] = {0.0f};
    r.each(
        d, t,
        [&](u32x4_t& v, int, int) {
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += Elem<X>::get(v, j);
        },
        [&](float v, int) { s[0] += v; });
    row_sums<WPR, 1>(s, slots[0], wave);
    const float mean = s[0] / (float)d;
    s[0] = 0.0f;
    r.each(
        d, t,
        [&](u32x4_t& v, int, int) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float c = Elem<X>::get(v, j) - mean;
                s[0] = __builtin_fmaf(c, c, s[0]);
            }
        },
        [&](float v, int) { s[0] = __builtin_fmaf(v - mean, v - mean, s[0]); });
    row_sums<WPR, 1>(s, slots[1], wave);
    const float rstd = 1.0f / __builtin_sqrtf(s[0] / (float)d + a.eps);
    const W* const w = (const W*)a.weight;
    const W* const b = (const W*)a.bias;
    X* const y = (X*)a.y + row * d;
    r.each(
        d, t,
        [&](u32x4_t& v, int col, int) {
            float wv[V], bv[V] = {}, out[V];
            load_weights(w, col, wv);
            if (b) load_weights(b, col, bv);
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = __builtin_fmaf((Elem<X>::get(v, j) - mean) * rstd, wv[j], bv[j]);
            *reinterpret_cast<u32x4_any_t*>(y + col) = Elem<X>::pack(out);
        },
        [&](float v, int col) {
            y[col] = Elem<X>::from_float(__builtin_fmaf((v - mean) * rstd, Elem<W>::to_float(w[col]),
                                                        b ? Elem<W>::to_float(b[col]) : 0.0f));
        });
    if (a.mean && t == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

struct BwdArgs {
    const void* dy;
    const void* x;
    const void* dsum;         // or null
    const void* weight;
    const float* mean;
    const float* rstd;
    void* dx;
    float* partial;           // [blocks][2][d]: the blocks' sums of dy * xhat and of dy
    int64_t lddy, ldx, ldds, T;
    int d;
    int fold;                 // turns (of D rows of a thread) between two foldings of its columns' sums
};

// With g = dy w and xhat = (x - mean) rstd: dx = rstd (g - mean(g) - xhat mean(g xhat)),
// dweight = sum over rows of dy xhat, dbias of dy.
//
// HBM bounds it (65536 x 4096 bf16 with DSUM, 2.15 GB, 383 to 395 us, 5.4 to 5.6 TB/s).
// One block to a CU keeps the partial sums few; to keep HBM busy with so few, the next
// rows of a ring of D are in flight while one is worked on (with 1024 blocks and rows
// loaded when needed: 433 us; 16384 x 4096 107 against 77, 32768 x 7168 398 against 262,
// 3001 x 2889 f32 40.6 against 25.7).
//
// A block walks rows blockIdx, blockIdx + gridDim, ... (4 / WPR at a time), its
// threads keeping their columns' sums for the weight and the bias.  After as many rows as
// the root of their number (32 at least) the sums are added to second ones and begin
// anew, so that none is a chain of more (262144 rows of 520 in f32: 1.8e-7 of the sum's size
// off, 6.0e-7 in one chain of 1024).  The second ones are in LDS, the thread's own places (a
// wave a row: in registers they cost as much).  With 16 waves a row (rows of more than 8192)
// the first are in LDS, which spares registers that would spill (6 to 20 still do in f32 with
// DSUM), and the second in memory, every 64 rows (4096 x 16384 bf16 with DSUM 162 to 124 us,
// 2048 x 9000 f32 126 to 72; 32768 x 16384, where memory's part counts, 702 to 734).  DSUM: a
// gradient past the norm is added.
template <typename X, typename W, int WPR, int NV, int D, bool TAIL, bool DSUM>
__global__ __launch_bounds__(norm_threads(WPR)) void layer_norm_bwd_kernel(BwdArgs a)
{
    constexpr int TPR = WPR * kWave, V = Elem<X>::V, kRows = norm_threads(WPR) / TPR;
    constexpr bool kLean = WPR == 16 || NV * V > 16;   // (registers are better spent on rows)
    __shared__ float slots[2][WPR][2];
    const int t = (int)threadIdx.x % TPR, wave = t / kWave;
    const int sub = __builtin_amdgcn_readfirstlane((int)threadIdx.x / TPR);
    const int d = a.d;
    const W* const w = (const W*)a.weight;
    float dw[NV][V], db[NV][V], dwt = 0.0f, dbt = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
    // the sums' second place; with 16 waves a row their first, the second being in memory
    constexpr bool kInLds = WPR == 16;
    float* const out = a.partial + (int64_t)blockIdx.x * 2 * d;
    const int nvec = d / V;
    __shared__ f32x4_t kept[NV][V / 4][2][norm_threads(WPR)];
    const auto place = [&](int i, int q, int of) -> f32x4_t& { return kept[i][q][of][threadIdx.x]; };
    float dwt_kept = 0.0f, dbt_kept = 0.0f;
    bool folded = false;
    // f(number, the place of four of the thread's sums, the sums, their address in the
    // block's, whether the row has them)
    const auto each_sum = [&](auto f) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                const int n = 2 * (i * (V / 4) + q), k = t + TPR * i;
                float* const at = out + k * V + 4 * q;
                f(n, place(i, q, 0), &dw[i][4 * q], at, k < nvec);
                f(n + 1, place(i, q, 1), &db[i][4 * q], at + d, k < nvec);
            }
    };
    const auto add_to_memory = [&]() {
        // (all loads before the first store: the compiler keeps their order)
        f32x4_t there[2 * NV * V / 4];
        each_sum([&](int n, f32x4_t&, float*, float* at, bool in) {
            there[n] = f32x4_t{};
            if (in && folded) there[n] = *reinterpret_cast<f32x4_any_t*>(at);
        });
        each_sum([&](int n, f32x4_t& sums, float*, float* at, bool in) {
            if (in) *reinterpret_cast<f32x4_any_t*>(at) = there[n] + sums;
        });
    };
    const auto fold = [&]() {
        if constexpr (kInLds) add_to_memory();
        each_sum([](int, f32x4_t& there, float* sum, float*, bool) {
            if constexpr (kInLds) there = f32x4_t{};
            else there += f32x4_t{sum[0], sum[1], sum[2], sum[3]};
            sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
        });
        dwt_kept += dwt;
        dbt_kept += dbt;
        dwt = dbt = 0.0f;
        folded = true;
    };
    each_sum([](int, f32x4_t& there, float*, float*, bool) { there = f32x4_t{}; });
    // the weight stays in registers: read twice a row it would be as much L1
    // traffic as the rows are
    float wr[NV][V], wt = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const bool in = t + TPR * i < nvec;
        if (!kLean) load_weights(w, in ? (t + TPR * i) * V : 0, wr[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) wr[i][j] = in ? wr[i][j] : 0.0f;
    }
    if (TAIL && t < d % V) wt = Elem<W>::to_float(w[nvec * V + t]);
    struct Rows {
        Row<X, TPR, NV> x, dy, ds;
        float mean, rstd;
    } ring[D];
    const auto load = [&](Rows& r, int64_t row) {
        row = min(row, a.T - 1);
        r.x.template load_ahead<TAIL>((const X*)a.x + row * a.ldx, d, t);
        r.dy.template load_ahead<TAIL>((const X*)a.dy + row * a.lddy, d, t);
        if constexpr (DSUM) r.ds.template load_ahead<TAIL>((const X*)a.dsum + row * a.ldds, d, t);
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
    };
    const auto weights_of = [&](int i) {
        if constexpr (kLean) load_weights(w, min(t + TPR * i, nvec - 1) * V, wr[i]);
    };
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + sub;
    int turn = 0;
    const auto process = [&](Rows& cur) {
        cur.x.template settle<TAIL>(d, t);
        cur.dy.template settle<TAIL>(d, t);
        if constexpr (DSUM) cur.ds.template settle<TAIL>(d, t);
        const float mean = cur.mean, rstd = cur.rstd;
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            weights_of(i);
            // (columns past the row have to add 0: 0 - mean, times a large rstd, may be an infinity)
            const float mu = t + TPR * i < nvec ? mean : 0.0f;
            f32x4_t sw[V / 4], sb[V / 4];
            if constexpr (kInLds) {
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    sw[q] = place(i, q, 0);
                    sb[q] = place(i, q, 1);
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (Elem<X>::get(cur.x.v[i], j) - mu) * rstd, dyv = Elem<X>::get(cur.dy.v[i], j);
                const float g = dyv * wr[i][j];
                s[0] += g;
                s[1] = __builtin_fmaf(g, xh, s[1]);
                if constexpr (kInLds) {
                    sw[j / 4][j % 4] = __builtin_fmaf(dyv, xh, sw[j / 4][j % 4]);
                    sb[j / 4][j % 4] += dyv;
                } else {
                    dw[i][j] = __builtin_fmaf(dyv, xh, dw[i][j]);
                    db[i][j] += dyv;
                }
            }
            if constexpr (kInLds) {
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    place(i, q, 0) = sw[q];
                    place(i, q, 1) = sb[q];
                }
            }
        }
        if constexpr (TAIL) {
            const float xh = (cur.x.tail - (t < d % V ? mean : 0.0f)) * rstd, g = cur.dy.tail * wt;
            s[0] += g;
            s[1] = __builtin_fmaf(g, xh, s[1]);
            dwt = __builtin_fmaf(cur.dy.tail, xh, dwt);
            dbt += cur.dy.tail;
        }
        row_sums<WPR, 2>(s, slots[turn], wave);
        const float c1 = s[0] / (float)d, c2 = s[1] / (float)d;
        X* const dx = (X*)a.dx + row * d;
        const auto gradient = [&](float x, float dy, float wv, float ds) {
            const float xh = (x - mean) * rstd;
            const float g = rstd * __builtin_fmaf(-xh, c2, __builtin_fmaf(dy, wv, -c1));
            return DSUM ? g + ds : g;
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float out[V];
            weights_of(i);
#pragma unroll
            for (int j = 0; j < V; ++j)
                out[j] = gradient(Elem<X>::get(cur.x.v[i], j), Elem<X>::get(cur.dy.v[i], j), wr[i][j],
                                  DSUM ? Elem<X>::get(cur.ds.v[i], j) : 0.0f);
            if (t + TPR * i < nvec)
                *reinterpret_cast<u32x4_any_t*>(dx + (t + TPR * i) * V) = Elem<X>::pack(out);
        }
        if (TAIL && t < d % V)
            dx[nvec * V + t] = Elem<X>::from_float(gradient(cur.x.tail, cur.dy.tail, wt, DSUM ? cur.ds.tail : 0.0f));
        turn ^= 1;
    };
    // rows in flight: the one that is worked on and D - 1 behind it
#pragma unroll
    for (int u = 0; u < D - 1; ++u) load(ring[u], row + u * step);
    int turns = a.fold;
    for (bool more = true; more;) {
#pragma unroll
        for (int u = 0; u < D; ++u) {
            more = row < a.T;
            if (!more) break;
            load(ring[(u + D - 1) % D], row + (D - 1) * step);
            process(ring[u]);
            row += step;
        }
        if (--turns == 0 && more) {
            fold();
            turns = a.fold;
        }
    }
    dwt += dwt_kept;
    dbt += dbt_kept;
    // the block's sums; with several rows at a time their threads' are added first
    if constexpr (!kInLds) {
        each_sum([](int, f32x4_t& there, float* sum, float*, bool) {
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] += there[k];
        });
    }
    if constexpr (kRows > 1) {
        constexpr int kCols = TPR * NV * V;
        __shared__ float cols[2][kCols + kWave];
        for (int q = 0; q < kRows; ++q) {
            if (sub == q) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int c = (t + TPR * i) * V + j;
                        cols[0][c] = q ? cols[0][c] + dw[i][j] : dw[i][j];
                        cols[1][c] = q ? cols[1][c] + db[i][j] : db[i][j];
                    }
                if (t < V) {
                    cols[0][kCols + t] = q ? cols[0][kCols + t] + dwt : dwt;
                    cols[1][kCols + t] = q ? cols[1][kCols + t] + dbt : dbt;
                }
            }
            __syncthreads();
        }
        for (int c = (int)threadIdx.x; c < d; c += 256) {
            const int at = c < nvec * V ? c : kCols + c - nvec * V;
            out[c] = cols[0][at];
            out[d + c] = cols[1][at];
        }
    } else {
        if constexpr (kInLds) add_to_memory();
        else each_sum([](int, f32x4_t&, float* sum, float* at, bool in) {
            if (in) *reinterpret_cast<f32x4_any_t*>(at) = f32x4_t{sum[0], sum[1], sum[2], sum[3]};
        });
        if (t < d % V) {
            out[nvec * V + t] = dwt;
            out[d + nvec * V + t] = dbt;
        }
    }
}

// Column sums of the blocks' partials, in a fixed order: 64 columns to a
// block, wave w of 16 the partials w, w + 16, ..., eight loads at a time (256 partials
// of 4096 columns, 8 MB: 5 us).
constexpr int kColWaves = 16;

__global__ __launch_bounds__(kColWaves * kWave) void layer_norm_cols_kernel(const float* partial, int blocks, int d,
                                                                            float* dweight, float* dbias)
{
    __shared__ float part[kColWaves][kWave];
    const int lane = lane_id(), wave = (int)threadIdx.x / kWave;
    const int col = (int)blockIdx.x * kWave + lane;
    const int at = min(col, 2 * d - 1);
    float s = 0.0f;
    int b = wave;
    for (; b + 7 * kColWaves < blocks; b += 8 * kColWaves) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = partial[(int64_t)(b + j * kColWaves) * 2 * d + at];
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; b < blocks; b += kColWaves) s += partial[(int64_t)b * 2 * d + at];
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < 2 * d) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < kColWaves; ++w) s += part[w][lane];
        if (col < d) dweight[col] = s;
        else if (dbias) dbias[col - d] = s;
    }
}

constexpr int kMaxWidth = ET_MAX_NORM_WIDTH;
constexpr int64_t kMaxBlocks = 256;

int64_t bwd_blocks(int64_t T) { return std::max<int64_t>(1, std::min(T, kMaxBlocks)); }

// Rows whose sums a thread adds up before it folds them, of those that it has of T: as
// many as it then has results, `least` at least.
int rows_between_folds(int64_t T, int64_t walkers, int least)
{
    const int64_t rows = (T + walkers - 1) / walkers;
    return std::max(least, (int)std::ceil(std::sqrt((double)rows)));
}

// Vectors of a row of d elements for each of `threads`.
int vectors(int64_t d, int V, int threads) { return (int)((d / V + threads - 1) / threads); }

template <typename X, typename W>
int launch_fwd(const FwdArgs& a, hipStream_t s)
{
    constexpr int V = Elem<X>::V;
    const auto go = [&](auto kernel, int wpr) -> int {
        // (a launch has less than 2^32 threads)
        const int64_t rows = norm_threads(wpr) / (wpr * kWave), most = (((int64_t)1 << 32) / norm_threads(wpr) - 1) * rows;
        for (int64_t from = 0; from < a.T; from += most) {
            FwdArgs part = a;
            const int64_t es = sizeof(X);
            const auto skip = [&](const void* p, int64_t bytes) { return p ? (const char*)p + from * bytes : nullptr; };
            part.T = std::min(most, a.T - from);
            part.x = skip(a.x, a.ldx * es);
            part.residual = skip(a.residual, a.ldr * es);
            part.y = (void*)skip(a.y, a.d * es);
            part.sum = (void*)skip(a.sum, a.d * es);
            part.mean = (float*)skip(a.mean, 4);
            part.rstd = (float*)skip(a.rstd, 4);
            kernel<<<dim3((unsigned)((part.T + rows - 1) / rows)), dim3(norm_threads(wpr)), 0, s>>>(part);
            const int rc = check_launch("layer_norm_fwd_kernel");
            if (rc) return rc;
        }
        return ET_OK;
    };
    const auto fits = [&](int wpr, int nv) { return vectors(a.d, V, wpr * kWave) <= nv; };
    if (fits(1, 1)) return go(layer_norm_fwd_kernel<X, W, 1, 1>, 1);
    if (fits(1, 2)) return go(layer_norm_fwd_kernel<X, W, 1, 2>, 1);
    if (fits(1, 4)) return go(layer_norm_fwd_kernel<X, W, 1, 4>, 1);
    if (fits(4, 2)) return go(layer_norm_fwd_kernel<X, W, 4, 2>, 4);
    if (fits(4, 4)) return go(layer_norm_fwd_kernel<X, W, 4, 4>, 4);
    return go(layer_norm_fwd_kernel<X, W, 16, 16 / V>, 16);
}

template <typename X, typename W, bool TAIL, bool DSUM>
int launch_bwd(const BwdArgs& a, int64_t blocks, hipStream_t s)
{
    constexpr int V = Elem<X>::V;
    const auto go = [&](auto kernel, int wpr, int depth) {
        BwdArgs b = a;
        const int64_t walkers = blocks * (norm_threads(wpr) / (wpr * kWave));
        b.fold = (rows_between_folds(a.T, walkers, wpr == 16 ? 64 : 32) + depth - 1) / depth;
        kernel<<<dim3((unsigned)blocks), dim3(norm_threads(wpr)), 0, s>>>(b);
        return check_launch("layer_norm_bwd_kernel");
    };
    const auto fits = [&](int wpr, int nv) { return vectors(a.d, V, wpr * kWave) <= nv; };
    if (fits(1, 1)) return go(layer_norm_bwd_kernel<X, W, 1, 1, 4, TAIL, DSUM>, 1, 4);
    if (fits(1, 2)) return go(layer_norm_bwd_kernel<X, W, 1, 2, 2, TAIL, DSUM>, 1, 2);
    if (fits(4, 1)) return go(layer_norm_bwd_kernel<X, W, 4, 1, 3, TAIL, DSUM>, 4, 3);
    if (fits(4, 2)) return go(layer_norm_bwd_kernel<X, W, 4, 2, 2, TAIL, DSUM>, 4, 2);
    if (fits(8, 2)) return go(layer_norm_bwd_kernel<X, W, 8, 2, 2, TAIL, DSUM>, 8, 2);
    if constexpr (sizeof(X) == 2) {
        return go(layer_norm_bwd_kernel<X, W, 16, 2, 1, TAIL, DSUM>, 16, 1);
    } else {
        if (fits(8, 4)) return go(layer_norm_bwd_kernel<X, W, 8, 4, 2, TAIL, DSUM>, 8, 2);
        return go(layer_norm_bwd_kernel<X, W, 16, 4, 1, TAIL, DSUM>, 16, 1);
    }
}

// Rows of fewer than V elements: nothing to do in vectors, and no more than 7
// columns; a thread for each of them and 256 rows a block.
template <typename X, typename W>
__global__ __launch_bounds__(256) void layer_norm_bwd_narrow_kernel(BwdArgs a)
{
    __shared__ float part[4][2][8];
    const int d = a.d;
    float dw[8], db[8], dw_kept[8], db_kept[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) dw[c] = db[c] = dw_kept[c] = db_kept[c] = 0.0f;
    int turns = a.fold;
    for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.T; row += (int64_t)gridDim.x * 256) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        float xh[8], dy[8], g[8], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (c >= d) break;
            xh[c] = (Elem<X>::to_float(((const X*)a.x)[row * a.ldx + c]) - mean) * rstd;
            dy[c] = Elem<X>::to_float(((const X*)a.dy)[row * a.lddy + c]);
            g[c] = dy[c] * Elem<W>::to_float(((const W*)a.weight)[c]);
            s0 += g[c];
            s1 = __builtin_fmaf(g[c], xh[c], s1);
            dw[c] = __builtin_fmaf(dy[c], xh[c], dw[c]);
            db[c] += dy[c];
        }
        const float c1 = s0 / (float)d, c2 = s1 / (float)d;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (c >= d) break;
            const float v = rstd * __builtin_fmaf(-xh[c], c2, g[c] - c1);
            ((X*)a.dx)[row * d + c] =
                Elem<X>::from_float(a.dsum ? v + Elem<X>::to_float(((const X*)a.dsum)[row * a.ldds + c]) : v);
        }
        if (--turns == 0) {
            turns = a.fold;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                dw_kept[c] += dw[c];
                db_kept[c] += db[c];
                dw[c] = db[c] = 0.0f;
            }
        }
    }
    for (int c = 0; c < d; ++c) {
        const float sw = wave_sum_dpp(dw[c] + dw_kept[c]), sb = wave_sum_dpp(db[c] + db_kept[c]);
        if (lane_id() == 0) {
            part[threadIdx.x / kWave][0][c] = sw;
            part[threadIdx.x / kWave][1][c] = sb;
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < 2 * d) {
        const int k = (int)threadIdx.x / d, c = (int)threadIdx.x % d;
        a.partial[(int64_t)blockIdx.x * 2 * d + threadIdx.x] =
            (part[0][k][c] + part[1][k][c]) + (part[2][k][c] + part[3][k][c]);
    }
}

template <typename X, typename W>
int launch_bwd(const BwdArgs& a, int64_t blocks, hipStream_t s)
{
    if (a.d < Elem<X>::V) {
        BwdArgs b = a;
        b.fold = rows_between_folds(a.T, blocks * 256, 32);
        layer_norm_bwd_narrow_kernel<X, W><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(b);
        return check_launch("layer_norm_bwd_narrow_kernel");
    }
    if (a.d % Elem<X>::V)
        return a.dsum ? launch_bwd<X, W, true, true>(a, blocks, s) : launch_bwd<X, W, true, false>(a, blocks, s);
    return a.dsum ? launch_bwd<X, W, false, true>(a, blocks, s) : launch_bwd<X, W, false, false>(a, blocks, s);
}

// Checks that both directions share.
int check_common(const char* fn, int64_t T, int64_t d, int dtype, int wdtype, int& esize)
{
    const std::string f(fn);
    if (dtype != ET_DTYPE_F32 && dtype != ET_DTYPE_BF16)
        return fail(ET_ERR_INVALID_ARGUMENT, f + ": dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    if (wdtype != ET_DTYPE_F32 && wdtype != dtype)
        return fail(ET_ERR_INVALID_ARGUMENT, f + ": weight_dtype must be ET_DTYPE_F32 or that of the rows");
    if (T < 0 || T >= (int64_t)1 << 31) return fail(ET_ERR_INVALID_ARGUMENT, f + ": rows must be in [0, 2^31)");
    if (d < 1 || d > kMaxWidth)
        return fail(ET_ERR_INVALID_ARGUMENT, f + ": d must be in [1, " + std::to_string(kMaxWidth) + "]");
    esize = dtype == ET_DTYPE_F32 ? 4 : 2;
    return ET_OK;
}

int check_rows(const char* fn, const char* name, const void* p, int64_t ld, int64_t d, int esize)
{
    if (!p) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null " + name);
    if (ld < d) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": the row stride of " + name + " is below d");
    if ((uintptr_t)p % esize) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + name + " is not aligned");
    return ET_OK;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" int et_layer_norm_fwd(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                 const void* weight, const void* bias, int64_t rows, int64_t d, int dtype,
                                 int weight_dtype, float eps, void* y, void* sum, float* mean, float* rstd,
                                 void* stream)
{
    const char* fn = "et_layer_norm_fwd";
    int es = 0;
    int rc = check_common(fn, rows, d, dtype, weight_dtype, es);
    if (rc) return rc;
    if (!(eps >= 0.0f && eps < __builtin_inff())) return fail(ET_ERR_INVALID_ARGUMENT, "et_layer_norm_fwd: eps must be >= 0");
    if ((mean == nullptr) != (rstd == nullptr))
        return fail(ET_ERR_INVALID_ARGUMENT, "et_layer_norm_fwd: mean and rstd go together");
    if ((residual == nullptr) != (sum == nullptr))
        return fail(ET_ERR_INVALID_ARGUMENT, "et_layer_norm_fwd: residual and sum go together");
    if (rows == 0) return ET_OK;
    const int ws = weight_dtype == ET_DTYPE_F32 ? 4 : 2;
    rc = check_rows(fn, "x", x, x_stride, d, es);
    if (!rc && residual) rc = check_rows(fn, "residual", residual, residual_stride, d, es);
    if (!rc && sum) rc = check_rows(fn, "sum", sum, d, d, es);
    if (!rc) rc = check_rows(fn, "y", y, d, d, es);
    if (!rc) rc = check_rows(fn, "weight", weight, d, d, ws);
    if (!rc && bias) rc = check_rows(fn, "bias", bias, d, d, ws);
    if (!rc && mean) rc = check_rows(fn, "mean", mean, d, d, 4);
    if (!rc && rstd) rc = check_rows(fn, "rstd", rstd, d, d, 4);
    if (rc) return rc;
    const FwdArgs a{x, residual, weight, bias, y, sum, mean, rstd, x_stride, residual_stride, rows, (int)d, eps};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == ET_DTYPE_F32) return launch_fwd<float, float>(a, s);
    return weight_dtype == ET_DTYPE_F32 ? launch_fwd<uint16_t, float>(a, s) : launch_fwd<uint16_t, uint16_t>(a, s);
}

extern "C" size_t et_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t d)
{
    if (rows < 0 || d < 1 || d > kMaxWidth) return 0;
    return (size_t)bwd_blocks(rows) * 2 * (size_t)d * sizeof(float);
}

extern "C" int et_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* dsum,
                                 int64_t dsum_stride, const void* weight, const float* mean, const float* rstd,
                                 int64_t rows, int64_t d, int dtype, int weight_dtype, void* dx, float* dweight,
                                 float* dbias, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* fn = "et_layer_norm_bwd";
    int es = 0;
    int rc = check_common(fn, rows, d, dtype, weight_dtype, es);
    if (rc) return rc;
    const int ws = weight_dtype == ET_DTYPE_F32 ? 4 : 2;
    if (rows) {
        rc = check_rows(fn, "dy", dy, dy_stride, d, es);
        if (!rc) rc = check_rows(fn, "x", x, x_stride, d, es);
        if (!rc && dsum) rc = check_rows(fn, "dsum", dsum, dsum_stride, d, es);
        if (!rc) rc = check_rows(fn, "dx", dx, d, d, es);
        if (!rc) rc = check_rows(fn, "mean", mean, d, d, 4);
        if (!rc) rc = check_rows(fn, "rstd", rstd, d, d, 4);
    }
    if (!rc) rc = check_rows(fn, "weight", weight, d, d, ws);
    if (!rc) rc = check_rows(fn, "dweight", dweight, d, d, 4);
    if (!rc && dbias) rc = check_rows(fn, "dbias", dbias, d, d, 4);
    if (rc) return rc;
    const size_t need = et_layer_norm_bwd_workspace_bytes(rows, d);
    if (!workspace || workspace_bytes < need)
        return fail(ET_ERR_WORKSPACE_TOO_SMALL, "et_layer_norm_bwd: workspace needs " + std::to_string(need) + " bytes");
    if ((uintptr_t)workspace % 4) return fail(ET_ERR_INVALID_ARGUMENT, "et_layer_norm_bwd: workspace is not aligned");
    const int64_t blocks = bwd_blocks(rows);
    const BwdArgs a{dy, x, dsum, weight, mean, rstd, dx, (float*)workspace, dy_stride, x_stride, dsum_stride, rows, (int)d, 0};
    hipStream_t s = (hipStream_t)stream;
    // (the kernels read rows ahead, the last one at least: they are for rows > 0)
    if (rows == 0) rc = ET_OK;
    else if (dtype == ET_DTYPE_F32) rc = launch_bwd<float, float>(a, blocks, s);
    else rc = weight_dtype == ET_DTYPE_F32 ? launch_bwd<uint16_t, float>(a, blocks, s)
                                           : launch_bwd<uint16_t, uint16_t>(a, blocks, s);
    if (rc) return rc;
    layer_norm_cols_kernel<<<dim3((unsigned)((2 * d + kWave - 1) / kWave)), dim3(kColWaves * kWave), 0, s>>>(
        (const float*)workspace, rows ? (int)blocks : 0, (int)d, dweight, dbias);
    return check_launch("layer_norm_cols_kernel");
}
