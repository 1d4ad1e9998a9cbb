// et_adapters.hip -- low-rank adapters of many requests beside a shared projection
// (gfx950):
//
//   out[t] = y[t] + scale[i] B_i (A_i x[t]),   i = index[t]   (no adapter: out = y)
//
// A plan sorts the tokens by adapter once for all projections of a step: items of up
// to 16 or 64 tokens of one adapter, so that every item is a pair of small matrix
// products.  Two launches a projection:
//   shrink  v = scale_i A_i x of an item's tokens: the sum over K split over the
//           waves of a block, and over blocks where there are few items;
//   expand  out = y + B_i v: 64 columns of a wave at a time.  v is taken as a sum of two bf16
//           numbers (16 bits of it; with rank 16 both fill one MFMA's k of 32), so
//           the one rounding that counts is that of the result.
// The bytes of x, y, out and the adapters in use bound both.  Which tokens share an item
// changes no result: every sum runs within a token.  Measured: 48 tokens, K = N = 4096, rank
// 16, 64 adapters 4.3 + 4.2 us (two launches' latency; 8.7 MB); 8192 tokens, K = 4096, N =
// 7168, rank 32, 24 adapters 14.9 + 48.4 us (4.6 and 4.9 TB/s of x, y and out).
#include <algorithm>

#include "et_dense_gemm.hpp"
#include "etmoe_dense.h"

namespace et {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct Item {
    int adapter, first, rows, unused;
};

// --------------------------------------------------------------------------
// plan
// --------------------------------------------------------------------------

// One block.  order: the tokens by adapter (those without one last); items and
// their number.  Within an adapter the order is that in which the lanes' atomics
// come.
__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(const int32_t* index, int64_t T, int n, int tile,
                                                                    int32_t* order, Item* items, int32_t* num_items)
{
    __shared__ int32_t at[ET_MAX_ADAPTERS + 1];      // counts, then each adapter's next place
    __shared__ int32_t wave_tokens[kPlanThreads / kWave], wave_items[kPlanThreads / kWave];
    const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
    for (int a = tid; a <= n; a += kPlanThreads) at[a] = 0;
    __syncthreads();
    // (n: no adapter)
    const auto adapter_of = [&](int64_t t) -> int {
        const int i = index[t];
        return (uint32_t)i < (uint32_t)n ? i : n;
    };
    for (int pass = 0; pass < 2; ++pass) {
        for (int64_t t = tid; t < T; t += kPlanThreads) {
            // (tokens of one request follow each other: the lanes with the first one's
            // adapter take their places at once)
            const int a = adapter_of(t), first = __builtin_amdgcn_readfirstlane(a);
            const uint64_t same = __ballot(a == first);
            int place = 0;
            if (a != first || rank_below(same) == 0) place = atomicAdd(&at[a], a == first ? (int)__popcll(same) : 1);
            if (a == first) place = __builtin_amdgcn_readfirstlane(place) + rank_below(same);
            if (pass == 1) order[place] = (int32_t)t;
        }
        __syncthreads();
        if (pass == 1) break;
        // counts to places; the items of each adapter
        int tokens = 0, made = 0;
        for (int a0 = 0; a0 <= n; a0 += kPlanThreads) {
            const int a = a0 + tid;
            const int c = a <= n ? at[a] : 0, k = (c + tile - 1) / tile;
            const int ci = wave_incl_scan(c), ki = wave_incl_scan(k);
            __syncthreads();
            if (lane == kWave - 1) {
                wave_tokens[wave] = ci;
                wave_items[wave] = ki;
            }
            __syncthreads();
            int ct = tokens, kt = made;
            for (int w = 0; w < kPlanThreads / kWave; ++w) {
                if (w < wave) {
                    ct += wave_tokens[w];
                    kt += wave_items[w];
                }
                tokens += wave_tokens[w];
                made += wave_items[w];
            }
            if (a <= n) {
                const int first = ct + ci - c;
                at[a] = first;
                for (int j = 0; j < k; ++j)
                    items[kt + ki - k + j] = Item{a < n ? a : -1, first + j * tile, min(tile, c - j * tile), 0};
            }
        }
        if (tid == 0) *num_items = made;
        __syncthreads();
    }
}

// --------------------------------------------------------------------------
// shrink
// --------------------------------------------------------------------------

struct AdapterArgs {
    const unsigned char* x;
    const unsigned char* y;
    const unsigned char* a;      // [n, r, K]
    const unsigned char* b;      // [n, N, r]
    const float* scale;
    const int32_t* order;
    const Item* items;
    const int32_t* num_items;
    float* v;                    // by place in the order: [splits, T, r], or (large items) bf16 hi and lo [2, T, r]
    unsigned char* out;
    int64_t ldx, ldy, ldo, T;
    int K, N, r, splits, step;   // step: the k of a split
    int col_blocks, chunks;      // of an item, and of a wave, in the expand kernel
};

// RT: tiles of 16 rows of A; TT: tiles of 16 tokens.  A wave brings its chunks of 64
// k through a ring of D stages of LDS of its own: a direct load fills 8 rows x 128
// bytes, whole cache lines.  (Loads of an operand's 16 rows x 64 bytes into
// registers move 14 bytes a cycle and CU: 8192 tokens, K = 4096, rank 32 22 us.)
// (items has room for every block: it is read beside their number)
template <int RT, int TT>
struct ShrinkShape {
    static constexpr int kStageBytes = (RT + TT) * 2048;
    static constexpr int kWaves = RT + TT <= 3 ? 8 : 4;
    // (tiles of 32 tokens: two blocks a CU)
    static constexpr int kFit = (TT == 2 && RT <= 4 ? 72 : 144) * 1024 / (kWaves * kStageBytes), D = kFit > 4 ? 4 : kFit;
    static_assert(D >= 1, "LDS");
};

// The same direct load from an address of each lane's own.
__device__ __forceinline__ void dma_global(const unsigned char* p, uint32_t lds)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(lds) : "memory");
}

// SUBS: blocks of 16 TT tokens an item.  SPLIT: partial sums of v in f32 (of splits of
// K); otherwise v as two bf16 numbers, as the other kernel takes it.
template <int RT, int TT, int SUBS, bool SPLIT>
__global__ __launch_bounds__((ShrinkShape<RT, TT>::kWaves * kWave)) void adapter_shrink_kernel(AdapterArgs g)
{
    using Shape = ShrinkShape<RT, TT>;
    constexpr int W = Shape::kWaves, D = Shape::D, kStageBytes = Shape::kStageBytes, NI = 2 * (RT + TT);
    constexpr int kRing = W * D * kStageBytes, kPart = W * RT * TT * kWave * 16;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kRing > kPart ? kRing : kPart];
    const int item = (int)blockIdx.x / SUBS;
    Item it = g.items[item];
    it.first += (int)blockIdx.x % SUBS * (16 * TT);
    it.rows -= (int)blockIdx.x % SUBS * (16 * TT);
    if (item >= *g.num_items || it.adapter < 0 || it.rows <= 0) return;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int r16 = lane & 15, rho = lane >> 4;
    const int split = (int)blockIdx.y;
    const int k0 = split * g.step, k1 = min(g.K, k0 + g.step);
    const __amdgpu_buffer_rsrc_t ares = dense_rsrc(g.a + (int64_t)it.adapter * g.r * g.K * 2, g.r * g.K * 2);
    // (tokens past the item's repeat its last one: their columns are not used)
    const unsigned char* xr[TT][2];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t token = g.order[it.first + min(16 * t + 8 * i + (lane >> 3), it.rows - 1)];
            xr[t][i] = g.x + token * g.ldx * 2;
        }
    unsigned char* const mine = smem + wave * (D * kStageBytes);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t*)mine;
    const int seg0 = (lane & 7) ^ (lane >> 3);
    // Chunk j of the wave.  Past the end A is 0 (and x any of the row's own values: one
    // that is not finite makes the token's sum so anyway).
    const auto load = [&](int j, uint32_t lds) {
        const int c = k0 + (W * j + wave) * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = c + (seg0 ^ i) * 8;
#pragma unroll
            for (int a = 0; a < RT; ++a) {
                const int row = 16 * a + 8 * i + (lane >> 3);
                dense_dma(ares, k < k1 && row < g.r ? (uint32_t)(row * g.K + k) * 2u : kOOR, 0u, lds + a * 2048 + i * 1024);
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) dma_global(xr[t][i] + 2 * (int64_t)min(k, g.K - 8), lds + (RT + t) * 2048 + i * 1024);
        }
    };
    f32x4_t acc[RT][TT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[i][t] = f32x4_t{};
    const int turns = (k1 - k0 + W * 64 - 1) / (W * 64);
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
            bf16x8_t fa[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) fa[i] = read(i);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const bf16x8_t fx = read(RT + t);
#pragma unroll
                for (int i = 0; i < RT; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fx, acc[i][t], 0, 0, 0);
            }
        }
        // (the reads above have ended; chunks past the end keep the count of loads)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
        load(j + D, lds0 + stage * kStageBytes);
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    dense_wait_barrier<0>();
    f32x4_t* const part = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) part[(wave * RT * TT + i * TT + t) * kWave + lane] = acc[i][t];
    __syncthreads();
    const float scale = g.scale[it.adapter];
    for (int q = (int)threadIdx.x; q < RT * TT * kWave; q += W * kWave) {
        const int tile = q >> 6, l = q & 63;
        f32x4_t sum = part[q];
#pragma unroll
        for (int w = 1; w < W; ++w) sum += part[w * RT * TT * kWave + q];
        const int row = 16 * (tile / TT) + 4 * (l >> 4), token = 16 * (tile % TT) + (l & 15);
        if (row >= g.r || token >= it.rows) continue;
        sum *= scale;
        const int64_t to = (int64_t)(it.first + token) * g.r + row;
        if constexpr (SPLIT) {
            *reinterpret_cast<f32x4_t*>(g.v + (int64_t)split * g.T * g.r + to) = sum;
        } else {
            const u32x2_t hi = {pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
            uint16_t* const v = (uint16_t*)g.v;
            *reinterpret_cast<u32x2_t*>(v + to) = hi;
            *reinterpret_cast<u32x2_t*>(v + g.T * g.r + to) =
                u32x2_t{pack_bf16x2(sum[0] - bf16lo(hi[0]), sum[1] - bf16hi(hi[0])), pack_bf16x2(sum[2] - bf16lo(hi[1]), sum[3] - bf16hi(hi[1]))};
        }
    }
}

// --------------------------------------------------------------------------
// expand
// --------------------------------------------------------------------------

// KS: k-steps of 32 over v's two parts (2 r / 32, rounded up).  A wave goes through
// g.chunks chunks of 64 columns with its tokens' v in registers.  The products go
// through LDS so that y and out move in whole cache lines, 8 rows x 128 bytes a load;
// a chunk's y is on its way while its products are made.  Blocks take an item's
// columns in turn, so that those that run together cover whole rows of y.
template <int KS, int TT, bool EVEN, bool SPLIT>
__global__ __launch_bounds__(kThreads) void adapter_expand_kernel(AdapterArgs g)
{
    constexpr int kRow = 64 + 4;      // floats from a token's products to the next's
    __shared__ __attribute__((aligned(16))) float smem[kWaves * 16 * kRow];
    const int item = (int)(blockIdx.x / (uint32_t)g.col_blocks);
    const Item it = g.items[item];
    if (item >= *g.num_items) return;
    const int lane = lane_id(), wave = (int)threadIdx.x >> 6;
    const int r16 = lane & 15, rho = lane >> 4;
    int n0 = (int)(blockIdx.x - (uint32_t)item * g.col_blocks) * g.chunks * (64 * kWaves) + wave * 64;
    if (n0 >= g.N || (it.adapter < 0 && g.out == g.y && g.ldo == g.ldy)) return;
    const int segs = g.r / 8;
    // this lane's rows of y (8 q + lane / 8), and its 8 columns
    const int line = 8 * (lane & 7);
    int64_t token[2 * TT];
#pragma unroll
    for (int q = 0; q < 2 * TT; ++q) token[q] = g.order[it.first + min(8 * q + (lane >> 3), it.rows - 1)];
    u32x4_t fv[KS][TT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int s = 4 * ks + rho;
        const int at = s >= 2 * segs ? 0 : (s >= segs ? s - segs : s) * 8;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            // (a token past the item's repeats its last one, unwritten)
            const int64_t from = (it.first + min(16 * t + r16, it.rows - 1)) * (int64_t)g.r + at;
            const bool low = s >= segs;
            u32x4_t w = {};
            if constexpr (SPLIT) {
                f32x4_t v[2] = {};
                if (it.adapter >= 0) {
                    const float* p = g.v + from;
                    v[0] = *reinterpret_cast<const f32x4_t*>(p);
                    v[1] = *reinterpret_cast<const f32x4_t*>(p + 4);
                    for (int sp = 1; sp < g.splits; ++sp) {
                        p += g.T * g.r;
                        v[0] += *reinterpret_cast<const f32x4_t*>(p);
                        v[1] += *reinterpret_cast<const f32x4_t*>(p + 4);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = v[i >> 1][2 * (i & 1)], b = v[i >> 1][2 * (i & 1) + 1];
                    const uint32_t hi = pack_bf16x2(a, b);
                    w[i] = low ? pack_bf16x2(a - bf16lo(hi), b - bf16hi(hi)) : hi;
                }
            } else if (it.adapter >= 0) {
                w = *reinterpret_cast<const u32x4_t*>((const uint16_t*)g.v + (low ? g.T * g.r : 0) + from);
            }
            fv[ks][t] = s >= 2 * segs ? u32x4_t{} : w;
        }
    }
    const int64_t first_row = max(it.adapter, 0) * (int64_t)g.N;
    float* const mine = smem + wave * (16 * kRow);
    for (int c = 0; c < g.chunks && n0 < g.N; ++c, n0 += 64 * kWaves) {
        const int col = n0 + line;
        u32x4_t y[2 * TT];
#pragma unroll
        for (int q = 0; q < 2 * TT; ++q)
            y[q] = *reinterpret_cast<const u32x4_t*>(g.y + (token[q] * g.ldy + min(col, g.N - 8)) * 2);
        if (it.adapter >= 0) {
            const __amdgpu_buffer_rsrc_t bres = dense_rsrc(g.b + (first_row + n0) * g.r * 2, min(64, g.N - n0) * g.r * 2);
            f32x4_t acc[TT][4];
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][j] = f32x4_t{};
            // (EVEN: rank a multiple of 32, the second half of the k-steps has the first
            // half's columns of b)
            constexpr int STEPS = EVEN ? KS / 2 : KS;
#pragma unroll
            for (int ks = 0; ks < STEPS; ++ks) {
                const int s = 4 * ks + rho;
                const int at = (!EVEN && s >= segs ? s - segs : s) * 8;
                u32x4_t fb[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    fb[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                        bres, s < 2 * segs ? (uint32_t)((16 * j + r16) * g.r + at) * 2u : kOOR, 0, 0));
#pragma unroll
                for (int half = 0; half < (EVEN ? 2 : 1); ++half)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(bf16x8_t, fb[j]), __builtin_bit_cast(bf16x8_t, fv[ks + half * STEPS][t]), acc[t][j], 0, 0, 0);
            }
            // (one wave's own part of LDS: its operations stay in order)
#pragma unroll
            for (int t = 0; t < TT; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4_t*>(mine + r16 * kRow + 16 * j + 4 * rho) = acc[t][j];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int q = 2 * t; q < 2 * t + 2; ++q) {
                    const float* const p = mine + (8 * (q & 1) + (lane >> 3)) * kRow + line;
                    const f32x4_t d[2] = {*reinterpret_cast<const f32x4_t*>(p), *reinterpret_cast<const f32x4_t*>(p + 4)};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        y[q][w] = pack_bf16x2(bf16lo(y[q][w]) + d[w >> 1][2 * (w & 1)], bf16hi(y[q][w]) + d[w >> 1][2 * (w & 1) + 1]);
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * TT; ++q)
            if (8 * q + (lane >> 3) < it.rows && col < g.N)
                *reinterpret_cast<u32x4_t*>(g.out + (token[q] * g.ldo + col) * 2) = y[q];
    }
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

int refuse(const char* fn, const char* what) { return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + what); }

// Tokens of an item: 16 up to 2048 tokens, 64 above, where an adapter's matrices
// are read from the caches once for four times as many tokens.
int tile_of(int64_t T) { return T <= 2048 ? 16 : 64; }

int64_t most_items(int64_t T, int64_t n) { return up(T, tile_of(T)) + std::min(T, n + 1); }

// What is wrong with the sizes of adapter_add (N apart), or null; its plan has `items`.
const char* size_error(int64_t items, int64_t K, int64_t rank)
{
    if (items < 0) return "num_tokens must be in [0, 2^30) and num_adapters in [1, ET_MAX_ADAPTERS]";
    // (a launch has less than 2^32 threads: the first kernel's has two blocks of up to 512 an item)
    if (items >= 1 << 22) return "num_tokens is too large";
    if (K < 8 || K % 8 || K >= 1 << 22) return "K must be a positive multiple of 8 below 2^22";
    if (rank < 8 || rank % 8 || rank > ET_MAX_ADAPTER_RANK) return "rank must be a positive multiple of 8, at most ET_MAX_ADAPTER_RANK";
    return nullptr;
}

// Splits of the sum over K, where the items leave CUs idle: the fewest rounds of
// blocks for the work of each, a chunk for each of 8 waves at least.
int splits_of(int64_t T, int64_t items, int64_t K)
{
    const int64_t cus = dense_cus(), most = tile_of(T) == 16 ? std::min<int64_t>(4, K / 512) : 1;
    int best = 1;
    for (int s = 2; s <= most; ++s)
        if (up(items * s, cus) * best < up(items * best, cus) * s) best = s;
    return best;
}

template <int RT>
void launch_shrink(const AdapterArgs& g, int tile, dim3 grid, hipStream_t s)
{
    if (tile == 16) {
        adapter_shrink_kernel<RT, 1, 1, true><<<grid, dim3(ShrinkShape<RT, 1>::kWaves * kWave), 0, s>>>(g);
    } else {
        grid.x *= 2;
        adapter_shrink_kernel<RT, 2, 2, false><<<grid, dim3(ShrinkShape<RT, 2>::kWaves * kWave), 0, s>>>(g);
    }
}

template <int KS>
void launch_expand(const AdapterArgs& g, int tile, dim3 grid, hipStream_t s)
{
    const dim3 block(kThreads);
    if (KS > 1 && g.r == 16 * KS) {
        if (tile == 16) adapter_expand_kernel<KS, 1, true, true><<<grid, block, 0, s>>>(g);
        else adapter_expand_kernel<KS, 4, true, false><<<grid, block, 0, s>>>(g);
    } else {
        if (tile == 16) adapter_expand_kernel<KS, 1, false, true><<<grid, block, 0, s>>>(g);
        else adapter_expand_kernel<KS, 4, false, false><<<grid, block, 0, s>>>(g);
    }
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" int64_t et_adapter_plan_items(int64_t num_tokens, int64_t num_adapters)
{
    if (num_tokens < 0 || num_tokens >= (int64_t)1 << 30 || num_adapters < 1 || num_adapters > ET_MAX_ADAPTERS) return -1;
    return most_items(num_tokens, num_adapters);
}

extern "C" int et_adapter_plan(const int32_t* index, int64_t num_tokens, int64_t num_adapters, int32_t* order, int32_t* items,
                               int32_t* num_items, void* stream)
{
    const char* fn = "et_adapter_plan";
    if (et_adapter_plan_items(num_tokens, num_adapters) < 0)
        return refuse(fn, "num_tokens must be in [0, 2^30) and num_adapters in [1, ET_MAX_ADAPTERS]");
    if (!num_items || (uintptr_t)num_items % 4) return refuse(fn, "num_items must be a 4-byte aligned pointer");
    if (num_tokens && (!index || !order || !items)) return refuse(fn, "null index, order or items");
    if ((uintptr_t)index % 4 || (uintptr_t)order % 4 || (uintptr_t)items % 16)
        return refuse(fn, "index and order must be 4-byte, items 16-byte aligned");
    adapter_plan_kernel<<<dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream>>>(
        index, num_tokens, (int)num_adapters, tile_of(num_tokens), order, (Item*)items, num_items);
    return check_launch("adapter_plan_kernel");
}

extern "C" size_t et_adapter_add_workspace_bytes(int64_t num_tokens, int64_t num_adapters, int64_t K, int64_t rank)
{
    const int64_t items = et_adapter_plan_items(num_tokens, num_adapters);
    if (size_error(items, K, rank)) return 0;
    return (size_t)splits_of(num_tokens, items, K) * num_tokens * rank * 4;
}

extern "C" int et_adapter_add(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* a, const void* b,
                              const float* scale, const int32_t* order, const int32_t* items, const int32_t* num_items,
                              int64_t num_tokens, int64_t num_adapters, int64_t K, int64_t N, int64_t rank, void* out,
                              int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* fn = "et_adapter_add";
    const int64_t most = et_adapter_plan_items(num_tokens, num_adapters);
    if (const char* const error = size_error(most, K, rank)) return refuse(fn, error);
    if (N < 8 || N % 8 || N >= 1 << 22) return refuse(fn, "N must be a positive multiple of 8 below 2^22");
    for (const auto& [ld, least] : {std::pair<int64_t, int64_t>{x_stride, K}, {y_stride, N}, {out_stride, N}})
        if (ld < least || ld % 8 || ld >= (int64_t)1 << 40) return refuse(fn, "row strides must be multiples of 8 and at least a row");
    if (num_tokens == 0) return ET_OK;
    for (const auto& [p, name] : {std::pair<const void*, const char*>{y, "y"}, {x, "x"}, {a, "a"}, {b, "b"}, {items, "items"}, {out, "out"}}) {
        if (!p) return refuse(fn, (std::string("null ") + name).c_str());
        if ((uintptr_t)p % 16) return refuse(fn, (std::string(name) + " must be 16-byte aligned").c_str());
    }
    if (!scale || !order || !num_items || ((uintptr_t)scale | (uintptr_t)order | (uintptr_t)num_items) % 4)
        return refuse(fn, "scale, order and num_items must be 4-byte aligned pointers");
    const size_t need = et_adapter_add_workspace_bytes(num_tokens, num_adapters, K, rank);
    if (workspace_bytes < need || !workspace)
        return fail(ET_ERR_WORKSPACE_TOO_SMALL, std::string(fn) + ": workspace needs " + std::to_string(need) + " bytes");
    if ((uintptr_t)workspace % 16) return refuse(fn, "workspace must be 16-byte aligned");
    AdapterArgs g = {};
    g.x = (const unsigned char*)x;
    g.y = (const unsigned char*)y;
    g.a = (const unsigned char*)a;
    g.b = (const unsigned char*)b;
    g.scale = scale;
    g.order = order;
    g.items = (const Item*)items;
    g.num_items = num_items;
    g.v = (float*)workspace;
    g.out = (unsigned char*)out;
    g.ldx = x_stride;
    g.ldy = y_stride;
    g.ldo = out_stride;
    g.T = num_tokens;
    g.K = (int)K;
    g.N = (int)N;
    g.r = (int)rank;
    g.splits = splits_of(num_tokens, most, K);
    g.step = (int)(up(up(K, g.splits), 64) * 64);
    g.splits = (int)up(K, g.step);
    // (several chunks a wave where there are many blocks all the same)
    g.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(4, most * up(N, 64 * kWaves) / 2048));
    g.col_blocks = (int)up(N, 64 * kWaves * g.chunks);
    // (a launch has less than 2^32 threads)
    if (most * g.col_blocks >= (int64_t)1 << 24)
        return refuse(fn, "num_tokens * N is too large");
    const int tile = tile_of(num_tokens);
    hipStream_t s = (hipStream_t)stream;
    const dim3 shrink((unsigned)most, (unsigned)g.splits), expand((unsigned)(most * g.col_blocks));
    if (rank <= 16) launch_shrink<1>(g, tile, shrink, s);
    else if (rank <= 32) launch_shrink<2>(g, tile, shrink, s);
    else if (rank <= 64) launch_shrink<4>(g, tile, shrink, s);
    else launch_shrink<8>(g, tile, shrink, s);
    if (const int rc = check_launch("adapter_shrink_kernel")) return rc;
    if (rank <= 16) launch_expand<1>(g, tile, expand, s);
    else if (rank <= 32) launch_expand<2>(g, tile, expand, s);
    else if (rank <= 64) launch_expand<4>(g, tile, expand, s);
    else launch_expand<8>(g, tile, expand, s);
    return check_launch("adapter_expand_kernel");
}
