// et_adapters.hip -- low-rank adapters of many requests beside a shared projection
// (gfx950):
//
//   out[t] = y[t] + scale[i] B_i (A_i x[t]),   i = index[t]   (no adapter: out = y)
//
// A plan sorts the tokens by adapter once for all projections of a step: items of up
// to 16 or 32 tokens of one adapter, so that every item is a pair of small matrix
// products.  Two launches a projection:
//   shrink  v = scale_i A_i x of an item's tokens: the sum over K split over the
//           waves of a block, and over blocks where there are few items; A and x go
//           from memory straight into the matrix units' operands (both have k along
//           their rows, and each is read once a block);
//   expand  out = y + B_i v: 64 columns a wave.  v is taken as a sum of two bf16
//           numbers (16 bits of it; with rank 16 both fill one MFMA's k of 32), so
//           the one rounding that counts is that of the result.
// The bytes of x, y, out and the adapters in use bound both.  Which tokens share an item
// changes no result: every sum runs within a token.
#include <algorithm>

#include "et_gemm_common.hpp"
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
// their number.  Within an adapter the order is that in which the waves come.
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
        for (int64_t t0 = 0; t0 < T; t0 += kPlanThreads) {
            const int64_t t = t0 + tid;
            const int a = t < T ? adapter_of(t) : -1;
            uint64_t left = __ballot(a >= 0);
            while (left) {
                // the lanes with the first one's adapter
                const int leader = (int)__builtin_ctzll(left);
                const int which = __shfl(a, leader, kWave);
                const uint64_t same = __ballot(a == which);
                int base = 0;
                if (lane == leader) base = atomicAdd(&at[which], (int)__popcll(same));
                base = __shfl(base, leader, kWave);
                if (pass == 1 && a == which) order[base + rank_below(same)] = (int32_t)t;
                left &= ~same;
            }
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
    float* v;                    // [splits, T, r], by place in the order
    unsigned char* out;
    int64_t ldx, ldy, ldo, T;
    int K, N, r, splits, step;   // step: the k of a split
};

// RT: tiles of 16 rows of A; TT: tiles of 16 tokens.
template <int RT, int TT>
__global__ __launch_bounds__(kThreads) void adapter_shrink_kernel(AdapterArgs g)
{
    __shared__ f32x4_t part[kWaves][TT * RT][kWave];
    if ((int)blockIdx.x >= *g.num_items) return;
    const Item it = g.items[blockIdx.x];
    if (it.adapter < 0) return;
    const int lane = lane_id(), wave = (int)threadIdx.x >> 6;
    const int r16 = lane & 15, rho = lane >> 4;
    const int split = (int)blockIdx.y;
    const int k0 = split * g.step, k1 = min(g.K, k0 + g.step);
    const unsigned char* xr[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        // (tokens past the item's repeat its last one: their columns are not used)
        const int64_t token = g.order[it.first + min(16 * t + r16, it.rows - 1)];
        xr[t] = g.x + token * g.ldx * 2;
    }
    const unsigned char* ar[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) ar[i] = g.a + ((int64_t)it.adapter * g.r + min(16 * i + r16, g.r - 1)) * g.K * 2;
    f32x4_t acc[RT][TT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[i][t] = f32x4_t{};
    // chunks of 64 k, dealt to the waves in turn: a row's 128 bytes in two loads of
    // one wave
    const auto one = [&](int c) {
        u32x4_t fa[2][RT], fx[2][TT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = k0 + 64 * c + 32 * h + 8 * rho;
            const bool in = k < k1;
#pragma unroll
            for (int i = 0; i < RT; ++i) fa[h][i] = in ? *reinterpret_cast<const u32x4_t*>(ar[i] + 2 * (int64_t)k) : u32x4_t{};
#pragma unroll
            for (int t = 0; t < TT; ++t) fx[h][t] = in ? *reinterpret_cast<const u32x4_t*>(xr[t] + 2 * (int64_t)k) : u32x4_t{};
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fa[h][i]),
                                                                        __builtin_bit_cast(bf16x8_t, fx[h][t]), acc[i][t], 0, 0, 0);
    };
    const int chunks = (k1 - k0 + 63) / 64;
    for (int c = wave; c < chunks; c += kWaves) one(c);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) part[wave][i * TT + t][lane] = acc[i][t];
    __syncthreads();
    const float scale = g.scale[it.adapter];
    for (int q = (int)threadIdx.x; q < RT * TT * kWave; q += kThreads) {
        const int tile = q >> 6, l = q & 63;
        f32x4_t sum = part[0][tile][l];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w][tile][l];
        const int row = 16 * (tile / TT) + 4 * (l >> 4), token = 16 * (tile % TT) + (l & 15);
        if (row < g.r && token < it.rows)
            *reinterpret_cast<f32x4_t*>(g.v + ((int64_t)split * g.T + it.first + token) * g.r + row) = sum * scale;
    }
}

// --------------------------------------------------------------------------
// expand
// --------------------------------------------------------------------------

// KS: k-steps of 32 over v's two parts (2 r / 32, rounded up).  A wave's 64 columns
// are dealt to four MFMA tiles so that a lane holds 16 consecutive ones of a token:
// row i of tile j is column 16 (i / 4) + 4 j + i % 4.
template <int KS, int TT>
__global__ __launch_bounds__(kThreads) void adapter_expand_kernel(AdapterArgs g)
{
    if ((int)blockIdx.x >= *g.num_items) return;
    const Item it = g.items[blockIdx.x];
    const int lane = lane_id(), wave = (int)threadIdx.x >> 6;
    const int r16 = lane & 15, rho = lane >> 4;
    const int n0 = ((int)blockIdx.y * kWaves + wave) * 64;
    if (n0 >= g.N) return;
    const int col = n0 + 16 * rho;
    u32x4_t y[TT][2];
    int64_t token[TT];
    bool ok[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        ok[t] = 16 * t + r16 < it.rows;
        token[t] = g.order[it.first + min(16 * t + r16, it.rows - 1)];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            y[t][h] = ok[t] && col + 8 * h < g.N
                          ? *reinterpret_cast<const u32x4_t*>(g.y + (token[t] * g.ldy + col + 8 * h) * 2) : u32x4_t{};
    }
    if (it.adapter >= 0) {
        const int segs = g.r / 8;
        f32x4_t acc[TT][4];
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][j] = f32x4_t{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int s = 4 * ks + rho;
            const bool in = s < 2 * segs, low = s >= segs;
            const int at = (low ? s - segs : s) * 8;
            u32x4_t fb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + 16 * (r16 >> 2) + 4 * j + (r16 & 3);
                fb[j] = in && n < g.N ? *reinterpret_cast<const u32x4_t*>(g.b + (((int64_t)it.adapter * g.N + n) * g.r + at) * 2)
                                      : u32x4_t{};
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                if (in && ok[t]) {
                    const float* p = g.v + (it.first + 16 * t + r16) * (int64_t)g.r + at;
                    for (int sp = 0; sp < g.splits; ++sp, p += g.T * g.r) {
                        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(p), hi = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] += lo[e];
                            v[4 + e] += hi[e];
                        }
                    }
                }
                u32x4_t fv;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t hi = pack_bf16x2(v[2 * w], v[2 * w + 1]);
                    fv[w] = low ? pack_bf16x2(v[2 * w] - bf16lo(hi), v[2 * w + 1] - bf16hi(hi)) : hi;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fb[j]),
                                                                        __builtin_bit_cast(bf16x8_t, fv), acc[t][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4_t& q = y[t][j >> 1];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint32_t w = q[2 * (j & 1) + p];
                    q[2 * (j & 1) + p] = pack_bf16x2(bf16lo(w) + acc[t][j][2 * p], bf16hi(w) + acc[t][j][2 * p + 1]);
                }
            }
    } else if (g.out == g.y) {
        return;
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (ok[t] && col + 8 * h < g.N)
                *reinterpret_cast<u32x4_t*>(g.out + (token[t] * g.ldo + col + 8 * h) * 2) = y[t][h];
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

int refuse(const char* fn, const char* what) { return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + what); }

// Tokens of an item: 16 up to 2048 tokens, 32 above, where an adapter's matrices
// are read from the caches once for twice as many tokens.
int tile_of(int64_t T) { return T <= 2048 ? 16 : 32; }

int64_t most_items(int64_t T, int64_t n) { return up(T, tile_of(T)) + std::min(T, n + 1); }

// Splits of the sum over K: blocks for all CUs, 256 k a split at least.
int splits_of(int64_t items, int64_t K)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>({8, 512 / std::max<int64_t>(1, items), K / 256}));
}

template <int RT>
void launch_shrink(const AdapterArgs& g, int tile, dim3 grid, hipStream_t s)
{
    if (tile == 16) adapter_shrink_kernel<RT, 1><<<grid, dim3(kThreads), 0, s>>>(g);
    else adapter_shrink_kernel<RT, 2><<<grid, dim3(kThreads), 0, s>>>(g);
}

template <int KS>
void launch_expand(const AdapterArgs& g, int tile, dim3 grid, hipStream_t s)
{
    if (tile == 16) adapter_expand_kernel<KS, 1><<<grid, dim3(kThreads), 0, s>>>(g);
    else adapter_expand_kernel<KS, 2><<<grid, dim3(kThreads), 0, s>>>(g);
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
    if (items < 0 || K < 8 || rank < 8 || rank > ET_MAX_ADAPTER_RANK) return 0;
    return (size_t)splits_of(items, K) * num_tokens * rank * 4;
}

extern "C" int et_adapter_add(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* a, const void* b,
                              const float* scale, const int32_t* order, const int32_t* items, const int32_t* num_items,
                              int64_t num_tokens, int64_t num_adapters, int64_t K, int64_t N, int64_t rank, void* out,
                              int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* fn = "et_adapter_add";
    const int64_t most = et_adapter_plan_items(num_tokens, num_adapters);
    if (most < 0) return refuse(fn, "num_tokens must be in [0, 2^30) and num_adapters in [1, ET_MAX_ADAPTERS]");
    if (K < 8 || K % 8 || K >= 1 << 22) return refuse(fn, "K must be a positive multiple of 8 below 2^22");
    if (N < 8 || N % 8 || N >= 1 << 22) return refuse(fn, "N must be a positive multiple of 8 below 2^22");
    if (rank < 8 || rank % 8 || rank > ET_MAX_ADAPTER_RANK)
        return refuse(fn, "rank must be a positive multiple of 8, at most ET_MAX_ADAPTER_RANK");
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
    g.splits = splits_of(most, K);
    g.step = (int)(up(up(K, g.splits), 64) * 64);
    g.splits = (int)up(K, g.step);
    const int tile = tile_of(num_tokens);
    hipStream_t s = (hipStream_t)stream;
    const dim3 shrink((unsigned)most, (unsigned)g.splits), expand((unsigned)most, (unsigned)up(N, 64 * kWaves));
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
