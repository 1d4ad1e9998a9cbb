// et_w4.hip -- products with 4-bit weights and group scales (gfx950): the
// experts' projections over the routing CSR and a dense layer's, for batches of
// a few tokens, where the time is that of reading the weights.
//
//   p[s, n] = sum_k a[row(s), k] * (q[e(s), n, k] - 8) * scale[e(s), n, k / G]
//
// Weights are laid out once, in the order in which waves read them.  A tile is
// 16 weight rows x 128 k, 1 KiB: lane l of the wave that reads it takes 16
// bytes, its dword s the 8 values of row l % 16 at k = 32 s + 8 (l / 16) + 0..7,
// the operand fragment of v_mfma_f32_16x16x32_bf16 as it is.  Value 2 i of a
// dword is at bit 4 i + 3, value 2 i + 1 at bit 16 + 4 i + 3 (modulo 32), so turning
// it by 4 i and masking gives two of them, each on the upper four fraction bits
// of a bf16 number, and the bits 0x4180 around them make that 16 + q: 7
// instructions for 8 weights, where a conversion through f32 takes 12.  The 16
// too much (and the 8) go out again through the accumulator: a group's MFMAs
// begin at -24 * sum(a), which is an MFMA chain of the same activations with a
// constant operand, shared by the tiles of a wave.  (q - 8) * a is summed as it
// would be in binary32 but for the size of the partial sums, up to 4 times
// larger: 2 bits of 24.  (16 is the least power of two that all of 0..15 lie
// behind without a step of the exponent.  128 + q, whose bits need no turning, makes them up
// to 17 times larger: where sums of 512 products cancel, 2.2e-5 to 1.1e-4 was
// left of them, and 1.5e-6 to 6.9e-6 is now, at the same speed.)
// A group's sum is then scaled and added in binary32.
//
// Two tiles (32 rows) of one k range are neighbours, their k ranges follow each
// other, and their scales lie in the lanes' order: a wave's loads are whole
// KiBs of consecutive addresses.
#include <algorithm>
#include <utility>

#include "et_gemm_common.hpp"
#include "etmoe_block.h"

namespace et {
namespace {

constexpr int kSb = 32;                 // weight rows of a superblock: two tiles
constexpr int kKt = 128;                // k of a tile
constexpr int kTileBytes = 1024;
constexpr uint32_t kMask = 0x00780078u;     // the bits of two values
constexpr uint32_t kMagic = 0x41804180u;    // bf16 16, twice
constexpr uint32_t kOffset = 0xC1C0C1C0u;   // bf16 -24, twice

// Sizes of a weight; the derived ones are the host's (a division takes a wave
// some 40 instructions).
struct W4Shape {
    int E, N, K, parts, group;
    int part_rows, part_sbs;   // rows of a part, and its superblocks
    int sbs, kts;              // superblocks of an expert, tiles along K
    __host__ __device__ int gpt() const { return kKt / group; }               // groups of a tile
    __host__ __device__ int64_t expert_bytes() const { return (int64_t)sbs * kts * 2 * kTileBytes; }
    __host__ __device__ int64_t expert_scales() const { return (int64_t)sbs * kts * gpt() * kSb; }
    // the first weight row of superblock b, and how many of its rows there are
    __host__ __device__ int row0(int b) const { return b < part_sbs ? b * kSb : part_rows + (b - part_sbs) * kSb; }
    __host__ __device__ int rows(int b) const
    {
        const int left = part_rows - (b < part_sbs ? b : b - part_sbs) * kSb;
        return left < kSb ? left : kSb;
    }
};

// Values 2 i and 2 i + 1 of a dword as bf16 16 + q, `turn` = 4 i: one instruction
// behind the turning (v_and_or_b32 takes one scalar register and no two literals).
__device__ __forceinline__ uint32_t turned(uint32_t v, int turn) { return v >> turn | v << (-turn & 31); }

__device__ __forceinline__ uint32_t unpack2(uint32_t v, int turn, uint32_t mask_s, uint32_t magic_v)
{
    // (only the last two wrap; a shift's encoding is half as long)
    return ((turn < 12 ? v >> turn : turned(v, turn)) & mask_s) | magic_v;
}

__device__ __forceinline__ float scale16(uint32_t bits16, bool half)
{
    return half ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits16) : u2f(bits16 << 16);
}

// ---------------------------------------------------------------------------
// laying the weights out, and back
// ---------------------------------------------------------------------------

// Row of a superblock at place i of its scales: lane row rho's 4 rows of the
// first tile, then its 4 rows of the second.
__device__ __forceinline__ int scale_row(int i) { return 16 * (i >> 2 & 1) + 4 * (i >> 3) + (i & 3); }

__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* q, const uint16_t* scales, W4Shape w, int64_t blocks,
                                                      uint32_t* packed, uint16_t* packed_scales)
{
    const int kts = w.kts, gpt = w.gpt(), groups = (w.K + w.group - 1) / w.group;
    // a block at a time: the tiles of one superblock at one k range
    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int kt = (int)(blk % kts);
        const int b = (int)(blk / kts % w.sbs);
        const int e = (int)(blk / kts / w.sbs);
        const int row0 = w.row0(b), rows = w.rows(b);
        for (int i = (int)threadIdx.x; i < 2 * kTileBytes / 4; i += 256) {
            const int tile = i >> 8, lane = i >> 2 & 63, s = i & 3;
            const int r = 16 * tile + (lane & 15), k = kt * kKt + 32 * s + 8 * (lane >> 4);
            uint32_t out = 0x88888888u;    // value 2 j at bit 4 j, value 2 j + 1 at bit 16 + 4 j
            if (r < rows && k < w.K) {     // (K a multiple of 8: all of the 8 or none)
                const uint8_t* src = q + (((int64_t)e * w.N + row0 + r) * w.K + k) / 2;
                out = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    out |= (uint32_t)(src[j] & 15) << (4 * j);
                    out |= (uint32_t)(src[j] >> 4) << (16 + 4 * j);
                }
            }
            packed[blk * (2 * kTileBytes / 4) + i] = turned(out, 29);
        }
        for (int i = (int)threadIdx.x; i < gpt * kSb; i += 256) {
            const int r = scale_row(i % kSb), g = kt * gpt + i / kSb;
            packed_scales[blk * gpt * kSb + i] =
                r < rows && g < groups ? scales[((int64_t)e * w.N + row0 + r) * groups + g] : (uint16_t)0;
        }
    }
}

// bf16 [E, N, K] of the experts with slots (all without offsets).
__global__ __launch_bounds__(256) void w4_unpack_kernel(const uint32_t* packed, const uint16_t* packed_scales, bool half,
                                                        W4Shape w, int64_t blocks, const int32_t* expert_offsets,
                                                        int64_t cap, uint16_t* out)
{
    const int kts = w.kts, gpt = w.gpt();
    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int kt = (int)(blk % kts);
        const int b = (int)(blk / kts % w.sbs);
        const int e = (int)(blk / kts / w.sbs);
        if (expert_offsets && min<int64_t>(expert_offsets[e], cap) >= min<int64_t>(expert_offsets[e + 1], cap)) continue;
        const int row0 = w.row0(b), rows = w.rows(b);
        for (int i = (int)threadIdx.x; i < 2 * kTileBytes / 4; i += 256) {
            // (16 threads write 256 bytes of one row)
            const int tile = i >> 8, r16 = i >> 4 & 15, s = i >> 2 & 3, rho = i & 3;
            const int r = 16 * tile + r16, in = 32 * s + 8 * rho, k = kt * kKt + in;
            if (r >= rows || k >= w.K) continue;
            const uint32_t v = turned(packed[blk * (2 * kTileBytes / 4) + 256 * tile + 4 * (16 * rho + r16) + s], 3);
            const int at = 8 * ((r & 15) >> 2) + 4 * (r >> 4) + (r & 3);
            const float sc = scale16(packed_scales[(blk * gpt + in / w.group) * kSb + at], half);
            u32x4_t o;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] = pack_bf16x2((float)((int)(v >> (4 * j) & 15) - 8) * sc, (float)((int)(v >> (16 + 4 * j) & 15) - 8) * sc);
            *reinterpret_cast<u32x4_t*>(out + ((int64_t)e * w.N + row0 + r) * w.K + k) = o;
        }
    }
}

// Groups of G weights to 4 bits: scale = max(largest / 7, -smallest / 8), so that
// both ends are reached, rounded to 16 bits; q = 8 + the nearest whole number
// of scales, held to 0..15.  8 weights to a thread, G / 8 threads to a group.
template <typename X, int G>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const X* w, int64_t rows, int K, bool half, uint32_t* q,
                                                          uint16_t* scales)
{
    const int cols = (K + G - 1) / G * (G / 8);     // threads of a row, whole groups
    // (whole waves take part in every turn)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i - lane_id() < rows * cols; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / cols;
        const int k = (int)(i % cols) * 8;
        const bool in = row < rows && k < K;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.0f;
            if (in) {
                if constexpr (sizeof(X) == 2) v[j] = u2f((uint32_t)w[row * K + k + j] << 16);
                else v[j] = w[row * K + k + j];
            }
        }
        float hi = 0.0f, lo = 0.0f;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi = __builtin_fmaxf(hi, v[j]);
            lo = __builtin_fminf(lo, v[j]);
            nan |= !(__builtin_fabsf(v[j]) < __builtin_inff());
        }
        float s = nan ? __builtin_inff() : __builtin_fmaxf(hi / 7.0f, lo / -8.0f);
#pragma unroll
        for (int off = G / 16; off >= 1; off >>= 1) s = __builtin_fmaxf(s, __shfl_xor(s, off, kWave));
        const uint16_t bits = half ? __builtin_bit_cast(uint16_t, (_Float16)s) : (uint16_t)f32_to_bf16_bits(s);
        const float sc = scale16(bits, half);
        uint32_t out = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (a group whose scale is not finite, or 0, is all 8: its products are NaN, or 0)
            const float t = sc > 0.0f && sc < __builtin_inff() ? __builtin_rintf(v[j] / sc) : 0.0f;
            const int n = (int)__builtin_fminf(__builtin_fmaxf(t, -8.0f), 7.0f) + 8;
            out |= (uint32_t)n << (4 * j);
        }
        if (in) {
            q[(row * K + k) / 8] = out;
            if (k % G == 0) scales[row * ((K + G - 1) / G) + k / G] = sc < __builtin_inff() ? bits : (uint16_t)(half ? 0x7E00 : 0x7FC0);
        }
    }
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------

struct W4Args {
    const uint16_t* a;              // gather: X [a_rows, K]; else [cap, K]
    const int32_t* sorted_token;    // gather only
    const unsigned char* packed;
    const uint16_t* scales;
    const int32_t* expert_offsets;  // null: one expert, all rows
    uint16_t* c;                    // [cap, N], or [cap, N / 2] for SwiGLU
    const float* row_scale;
    int64_t a_rows, cap;
    W4Shape w;
    bool half;                      // scales f16, else bf16
};

struct W4Tile {
    int64_t s0;     // first slot
    int rows;       // slots
    int e;
    int b;          // first superblock (SwiGLU: of the gate part)
};

// Lane i of each row of 16 lanes, to the whole row.
template <int I>
__device__ __forceinline__ float row_bcast(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + I, 0xf, 0xf, true));
}

// f(0), f(1), ... with the numbers as constants.
template <int... I, typename F>
__device__ __forceinline__ void constants(std::integer_sequence<int, I...>, F f)
{
    (f(std::integral_constant<int, I>{}), ...);
}

// The two constants of unpacking, kept in registers.
struct Unpack {
    uint32_t mask = kMask, magic = kMagic;
    __device__ __forceinline__ Unpack()
    {
        asm("" : "+s"(mask));
        asm("" : "+v"(magic));
    }
};

// Scales of R = 4 turns (4 GPT groups) of the superblocks of a wave: lane
// (rho, i) loads those of group i for the rows that lanes (rho, *) add up, 16
// bytes; a broadcast of lane i along its row hands them out.  (Loaded group by
// group, the same 64 bytes in all of a row's lanes, they cost 8 to 13% of a
// call of 4 to 16 tokens.)
constexpr int kTurns = 4;
template <int NSB>
struct Scales {
    u32x4_t raw[NSB];
    float f[NSB][8];
    __device__ __forceinline__ void convert(bool half)
    {
        // (a branch of the whole grid: each way 8 instructions for 4 turns)
        if (half) {
#pragma unroll
            for (int j = 0; j < NSB; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) f[j][k] = scale16(raw[j][k / 2] >> (16 * (k & 1)) & 0xFFFFu, true);
        } else {
#pragma unroll
            for (int j = 0; j < NSB; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) f[j][k] = k & 1 ? bf16hi(raw[j][k / 2]) : bf16lo(raw[j][k / 2]);
        }
    }
};

// acc += one k range of 128 of NT tiles (two to a superblock) by MT tiles of 16
// slots; a(i, s) is the fragment of slots 16 i.. at k-step s, TURN the place of
// the range among those that the scales at hand are for.
template <int MT, int NT, int GPT, int TURN, typename A>
__device__ __forceinline__ void w4_mul(const u32x4_t (&w)[NT], const Scales<NT / 2>& scales, const Unpack& un, A a,
                                       f32x4_t (&acc)[NT][MT])
{
    constexpr int SPG = 4 / GPT;
    const bf16x8_t offset = __builtin_bit_cast(bf16x8_t, u32x4_t{kOffset, kOffset, kOffset, kOffset});
    constants(std::make_integer_sequence<int, GPT>{}, [&](auto group) {
        constexpr int q = decltype(group)::value;
        bf16x8_t x[MT][SPG];
        f32x4_t base[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            base[i] = f32x4_t{};
#pragma unroll
            for (int s = 0; s < SPG; ++s) {
                x[i][s] = __builtin_bit_cast(bf16x8_t, a(i, q * SPG + s));
                base[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(offset, x[i][s], base[i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            // (a tile at a time: the scheduler would else unpack them all first)
            __builtin_amdgcn_sched_barrier(0);
            f32x4_t p[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) p[i] = base[i];
#pragma unroll
            for (int s = 0; s < SPG; ++s) {
                u32x4_t f;
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = unpack2(w[j][q * SPG + s], 4 * k, un.mask, un.magic);
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f), x[i][s], p[i], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float scale = row_bcast<TURN * GPT + q>(scales.f[j / 2][4 * (j & 1) + r]);
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[j][i][r] = __builtin_fmaf(scale, p[i][r], acc[j][i][r]);
            }
        }
    });
}

// Where a wave reads the weights and scales of superblock b (clamped to the last).
struct W4Rows {
    const unsigned char* w;
    const uint16_t* s;
    __device__ __forceinline__ W4Rows() {}
    __device__ __forceinline__ W4Rows(const W4Args& g, int e, int b, int gpt)
    {
        b = min(b, g.w.sbs - 1);
        w = g.packed + e * g.w.expert_bytes() + (int64_t)b * g.w.kts * 2 * kTileBytes;
        s = g.scales + e * g.w.expert_scales() + (int64_t)b * g.w.kts * gpt * kSb;
    }
};

// Rows of A of a tile as a buffer, and the offset of row r in it (out of range
// past the tile and for invalid tokens, which read 0).
struct W4Acts {
    __amdgpu_buffer_rsrc_t res;
    __device__ __forceinline__ W4Acts(const W4Args& g, const W4Tile& t)
    {
        const int K = g.w.K;
        res = g.sorted_token
                  ? __builtin_amdgcn_make_buffer_rsrc((void*)g.a, (short)0, (int)(g.a_rows * K * 2), kBufDword3)
                  : __builtin_amdgcn_make_buffer_rsrc((void*)(g.a + t.s0 * K), (short)0, t.rows * K * 2, kBufDword3);
    }
    __device__ __forceinline__ uint32_t row(const W4Args& g, const W4Tile& t, int r) const
    {
        if (r >= t.rows) return kOOR;
        uint32_t at = (uint32_t)r;
        if (g.sorted_token) {
            at = (uint32_t)g.sorted_token[t.s0 + r];
            if (at >= (uint32_t)g.a_rows) return kOOR;
        }
        return at * (uint32_t)g.w.K * 2u;
    }
    // 16 bytes from column k (uniform) + in of the row at byte offset `at`; 0 past K
    __device__ __forceinline__ u32x4_t load(uint32_t at, int k, int in, int K) const
    {
        return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                               res, (int)(k + in < K ? at + 2u * (uint32_t)in : kOOR), 2 * k, 0));
    }
};

// Tiles of few slots: 16 slots x NSB superblocks (SwiGLU: one of the gate part,
// its twin of the up part) to a block, the k range dealt to the block's waves
// one 128 at a time, their sums joined through LDS in the waves' order.
template <bool SWIGLU, int NSB, int GPT, int WAVES>
__device__ __forceinline__ void w4_split_tile(const W4Args& g, const W4Tile& t, float* lds)
{
    constexpr int NT = 2 * NSB, U = 2, MT = 1;
    const bool half = g.half;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int r16 = lane & 15, rho = lane >> 4;
    const int K = g.w.K, kts = g.w.kts, twin = g.w.part_sbs;
    W4Rows rows[NSB];
#pragma unroll
    for (int j = 0; j < NSB; ++j) rows[j] = W4Rows(g, t.e, t.b + (SWIGLU ? j * twin : j), GPT);
    const W4Acts acts(g, t);
    const uint32_t ao = acts.row(g, t, r16);
    // (kts of this wave: wave, wave + WAVES, ...; loads past the last repeat it)
    const int n = (kts - wave + WAVES - 1) / WAVES;
    const auto kt_of = [&](int i) { return wave + WAVES * min(i, n - 1); };
    struct Step {
        u32x4_t w[NT], a[4];
    } ring[U];
    const auto load = [&](Step& x, int i) {
        const int kt = kt_of(i);
        const uint32_t at = (uint32_t)kt * (2 * kTileBytes);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            x.w[j] = *reinterpret_cast<const u32x4_t*>(rows[j / 2].w + at + (j & 1) * kTileBytes + 16 * lane);
#pragma unroll
        for (int s = 0; s < 4; ++s) x.a[s] = acts.load(ao, kt * kKt, 32 * s + 8 * rho, K);
    };
    Scales<NSB> scales;
    const auto load_scales = [&](int i) {
        const int at = (kt_of(i + min(r16 / GPT, kTurns - 1)) * GPT + r16 % GPT) * kSb + 8 * rho;
#pragma unroll
        for (int j = 0; j < NSB; ++j) scales.raw[j] = *reinterpret_cast<const u32x4_t*>(rows[j].s + at);
    };
    f32x4_t acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = f32x4_t{};
    const Unpack un;
    if (n > 0) {
        load_scales(0);
#pragma unroll
        for (int u = 0; u < U; ++u) load(ring[u], u);
        for (int i = 0; i < n; i += kTurns) {
            scales.convert(half);
            load_scales(i + kTurns);
            constants(std::make_integer_sequence<int, kTurns>{}, [&](auto turn) {
                constexpr int v = decltype(turn)::value;
                const Step& x = ring[v % U];
                if (i + v < n) w4_mul<MT, NT, GPT, v>(x.w, scales, un, [&](int, int s) { return x.a[s]; }, acc);
                __builtin_amdgcn_sched_barrier(0);
                load(ring[v % U], i + v + U);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }
    // the waves' sums, in order: wave w takes tiles w, w + WAVES, ...
#pragma unroll
    for (int j = 0; j < NT; ++j)
        *reinterpret_cast<f32x4_t*>(lds + (wave * NT + j) * 4 * kWave + 4 * lane) = acc[j][0];
    __syncthreads();
    const auto total = [&](int j) {
        f32x4_t s = {};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) s += *reinterpret_cast<const f32x4_t*>(lds + (v * NT + j) * 4 * kWave + 4 * lane);
        return s;
    };
    const int cols = SWIGLU ? g.w.part_rows : g.w.N;
    for (int j = wave; j < (SWIGLU ? 2 : NT); j += WAVES) {
        const int b = t.b + j / 2, in = 16 * (j & 1) + 4 * rho;
        f32x4_t v = total(j);
        if constexpr (SWIGLU) {
            const f32x4_t up = total(j + 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (v[k] * sigmoid(v[k])) * up[k];
        }
        if (b >= (SWIGLU ? twin : g.w.sbs) || r16 >= t.rows || in >= g.w.rows(b)) continue;
        if (g.row_scale) v *= g.row_scale[t.s0 + r16];
        *reinterpret_cast<u32x2_t*>(g.c + (t.s0 + r16) * cols + g.w.row0(b) + in) =
            u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
    __syncthreads();
}

// Tiles of more slots: the waves lie side by side in the weight rows, 64 each
// (SwiGLU: 32 gate rows and their 32 up rows), every one over the whole of K, and
// share the rows of A, 128 k at a time, through two LDS buffers (one barrier
// each): read from L2 by every wave, as above, they are 2 to 4 times the weight's
// bytes at 32 and 64 slots.
//
// What bounds them at 64 slots is the issue of instructions: 80 MFMAs and 204
// others for a wave's 4 KiB of weights.  (On one SIMD 32 MFMAs of one wave take
// 584 cycles, 256 v_and_or and shifts of another 1218, both at once 1471: an MFMA costs the
// other wave 8 cycles.)  With 32 slots a weight is unpacked twice as often.  64 experts of
// a mean of 64 slots, K = 2048, N = 2816, 32 slots to a tile, 90 us: CUs busy 82% of the
// time; of that the matrix pipes 39%, while 27 M vector instructions are issued (66% at 4
// cycles each).  The order in which a wave issues them, its priority, a ring of four k
// ranges and (at 64 slots) a third block to a CU change nothing.
// Against the bf16 GEMM on unpacked weights (us): mean of 62 slots 110 / 216, 256
// 318 / 353, 1026 1098 / 987, 2061 2250 / 1872 (32 experts, K = 2048, N = 7168).
constexpr int kWideWaves = 4;
constexpr int kWidePitch = 2 * kKt + 16;               // bytes of a row of A in LDS
// MAXMT tiles of 16 slots at most: 32 or 64 slots
constexpr int wide_buf(int maxmt) { return 16 * maxmt * kWidePitch; }

template <bool SWIGLU, int MT, int MAXMT, int GPT>
__device__ __forceinline__ void w4_wide_tile(const W4Args& g, const W4Tile& t, unsigned char* lds)
{
    constexpr int NSB = 2, NT = 4, U = 2, kBuf = wide_buf(MAXMT);
    const bool half = g.half;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int r16 = lane & 15, rho = lane >> 4;
    const int K = g.w.K, kts = g.w.kts, twin = g.w.part_sbs;
    const int b0 = t.b + wave * (SWIGLU ? 1 : NSB);      // the wave's first superblock
    W4Rows rows[NSB];
#pragma unroll
    for (int j = 0; j < NSB; ++j) rows[j] = W4Rows(g, t.e, b0 + (SWIGLU ? j * twin : j), GPT);
    u32x4_t ring[U][NT];
    const auto load_w = [&](int kt, int u) {
        const uint32_t at = (uint32_t)min(kt, kts - 1) * (2 * kTileBytes);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            ring[u][j] = *reinterpret_cast<const u32x4_t*>(rows[j / 2].w + at + (j & 1) * kTileBytes + 16 * lane);
    };
    Scales<NSB> scales;
    const auto load_scales = [&](int kt) {
        const int at = (min(kt + min(r16 / GPT, kTurns - 1), kts - 1) * GPT + r16 % GPT) * kSb + 8 * rho;
#pragma unroll
        for (int j = 0; j < NSB; ++j) scales.raw[j] = *reinterpret_cast<const u32x4_t*>(rows[j].s + at);
    };
    load_scales(0);
#pragma unroll
    for (int u = 0; u < U; ++u) load_w(u, u);
    // thread i: 16 bytes from column 8 (i % 16) of rows i / 16 + 16 m
    const W4Acts acts(g, t);
    const int seg = (int)threadIdx.x & 15, sr = (int)threadIdx.x >> 4;
    uint32_t ao[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) ao[m] = acts.row(g, t, 16 * m + sr);
    u32x4_t stage[MT];
    const auto load_a = [&](int kt) {
        kt = min(kt, kts - 1);
#pragma unroll
        for (int m = 0; m < MT; ++m) stage[m] = acts.load(ao[m], kt * kKt, 8 * seg, K);
    };
    const auto store_a = [&](int b) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
            *reinterpret_cast<u32x4_t*>(lds + b * kBuf + (16 * m + sr) * kWidePitch + 16 * seg) = stage[m];
    };
    f32x4_t acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4_t{};
    const Unpack un;
    load_a(0);
    store_a(0);
    load_a(1);
    __syncthreads();
    for (int kt = 0; kt < kts; kt += kTurns) {
        scales.convert(half);
        load_scales(kt + kTurns);
        constants(std::make_integer_sequence<int, kTurns>{}, [&](auto turn) {
            constexpr int v = decltype(turn)::value;
            if (kt + v < kts) {      // (the same for the whole block)
                // range kt + v is in buffer v % 2; the next one goes to the
                // other, which every wave has read before the last barrier
                store_a((v & 1) ^ 1);
                load_a(kt + v + 2);
                __builtin_amdgcn_sched_barrier(0);
                const unsigned char* const x = lds + (v & 1) * kBuf + r16 * kWidePitch + 16 * rho;
                w4_mul<MT, NT, GPT, v>(ring[v % U], scales, un, [&](int m, int s) {
                    return *reinterpret_cast<const u32x4_t*>(x + 16 * m * kWidePitch + 64 * s);
                }, acc);
                __builtin_amdgcn_sched_barrier(0);
                load_w(kt + v + U, v % U);
                __builtin_amdgcn_sched_barrier(0);
                __syncthreads();
            }
        });
    }
    const int cols = SWIGLU ? g.w.part_rows : g.w.N;
    const __amdgpu_buffer_rsrc_t cres =
        __builtin_amdgcn_make_buffer_rsrc((void*)(g.c + t.s0 * cols), (short)0, t.rows * cols * 2, kBufDword3);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = 16 * i + r16;
        float scale = 1.0f;
        if (g.row_scale) scale = g.row_scale[t.s0 + min(row, t.rows - 1)];
#pragma unroll
        for (int j = 0; j < (SWIGLU ? 1 : NSB); ++j) {
            const int b = b0 + j;
            if (b >= (SWIGLU ? twin : g.w.sbs)) break;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = acc[2 * j + k / 4][i][k % 4];
                if constexpr (SWIGLU) v[k] = (v[k] * sigmoid(v[k])) * acc[2 + k / 4][i][k % 4];
                else if (g.row_scale) v[k] *= scale;
            }
            store_pair16(v, cres, row < t.rows, (uint32_t)row * (uint32_t)cols, g.w.row0(b), g.w.row0(b) + g.w.rows(b), rho);
        }
    }
}

// Inclusive sums along the wave, with DPP moves only.
__device__ __forceinline__ int wave_scan_dpp(int v)
{
    v += (int)dpp_mov_u32<0x111>((uint32_t)v);        // row_shr:1
    v += (int)dpp_mov_u32<0x112>((uint32_t)v);
    v += (int)dpp_mov_u32<0x114>((uint32_t)v);
    v += (int)dpp_mov_u32<0x118>((uint32_t)v);
    v += (int)dpp_mov_u32<0x142, 0xA>((uint32_t)v);   // row_bcast:15 into rows 1 and 3
    v += (int)dpp_mov_u32<0x143, 0xC>((uint32_t)v);   // row_bcast:31 into rows 2 and 3
    return v;
}

// Slot tile `at` of 1 << LOG slots, counted over the experts' slots: its
// expert, first slot and slots.  False past the last.  Every wave for itself
// (E loads, 64 at a time): no barrier before the first weight is asked for.
template <int LOG>
__device__ __forceinline__ bool find_slots(const W4Args& g, int at, W4Tile& t)
{
    if (!g.expert_offsets) {
        t.e = 0;
        t.s0 = (int64_t)at << LOG;
        t.rows = (int)min<int64_t>(g.cap - t.s0, 1 << LOG);
        return t.rows > 0;
    }
    const int lane = lane_id(), E = g.w.E, cap = (int)g.cap;
    int before = 0;
    for (int e0 = 0; e0 < E; e0 += kWave) {
        const int e = e0 + lane;
        const int lo = min(g.expert_offsets[min(e, E)], cap), hi = min(g.expert_offsets[min(e + 1, E)], cap);
        const int n = max(hi - lo, 0);
        const int tiles = (n + (1 << LOG) - 1) >> LOG;
        const int upto = wave_scan_dpp(tiles) + before;
        const uint64_t past = __ballot(upto > at);
        if (past) {
            const int who = __builtin_ctzll(past);
            const int in = at - __builtin_amdgcn_readlane(upto - tiles, who);
            t.e = e0 + who;
            t.s0 = __builtin_amdgcn_readlane(lo, who) + (in << LOG);
            t.rows = min(__builtin_amdgcn_readlane(n, who) - (in << LOG), 1 << LOG);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

// Tile q of the wide kernel: an expert's slot tiles (1 << LOG slots at most, the
// expert's slots dealt evenly in sixteens) times nb blocks of weight rows, the
// slot tile the faster.  q below the count.
template <int LOG>
__device__ __forceinline__ void find_tile(const W4Args& g, uint32_t q, uint32_t nb, W4Tile& t)
{
    const int lane = lane_id(), E = g.w.E, cap = (int)g.cap;
    int first = 0, n = cap, before = 0;
    t.e = 0;
    if (g.expert_offsets) {
        for (int e0 = 0; e0 < E; e0 += kWave) {
            const int e = e0 + lane;
            const int lo = min(g.expert_offsets[min(e, E)], cap), hi = min(g.expert_offsets[min(e + 1, E)], cap);
            const int rows = max(hi - lo, 0), tiles = (rows + (1 << LOG) - 1) >> LOG;
            const int upto = wave_scan_dpp(tiles) + before;
            const uint64_t past = __ballot((uint32_t)upto * nb > q);
            if (past) {
                const int who = __builtin_ctzll(past);
                t.e = e0 + who;
                first = __builtin_amdgcn_readlane(lo, who);
                n = __builtin_amdgcn_readlane(rows, who);
                before = __builtin_amdgcn_readlane(upto - tiles, who);
                break;
            }
            before = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
    }
    const uint32_t in = q - (uint32_t)before * nb, mine = (uint32_t)(n + (1 << LOG) - 1) >> LOG;
    const int share = (int)(((uint32_t)(n + 15) / 16 + mine - 1) / mine) * 16;
    const int at = (int)(in % mine) * share;
    t.b = (int)(in / mine);
    t.s0 = first + at;
    t.rows = min(n - at, share);
}

constexpr int split_lds(int nsb, int waves) { return waves * 2 * nsb * 4 * kWave; }    // floats

template <bool SWIGLU, int NSB, int GPT, int WAVES>
__device__ __forceinline__ void w4_split(const W4Args& g, float* lds)
{
    constexpr int LOG = 4;
    // units of superblocks: pairs of twins for SwiGLU, NSB side by side else
    const uint32_t nb = (uint32_t)(SWIGLU ? g.w.part_sbs : (g.w.sbs + NSB - 1) / NSB);
    for (uint32_t q = blockIdx.x;; q += gridDim.x) {
        W4Tile t;
        if (!find_slots<LOG>(g, (int)(q / nb), t)) break;
        // (uniform as they are, but the compiler has to know)
        t.e = __builtin_amdgcn_readfirstlane(t.e);
        t.s0 = __builtin_amdgcn_readfirstlane((int)t.s0);
        t.rows = __builtin_amdgcn_readfirstlane(t.rows);
        t.b = (int)(q % nb) * (SWIGLU ? 1 : NSB);
        w4_split_tile<SWIGLU, NSB, GPT, WAVES>(g, t, lds);
    }
}

template <bool SWIGLU, int NSB, int GPT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void w4_split_kernel(W4Args g)
{
    __shared__ __attribute__((aligned(16))) float lds[split_lds(NSB, WAVES)];
    w4_split<SWIGLU, NSB, GPT, WAVES>(g, lds);
}

// Slot tiles of 1 << LOG slots of all experts.
template <int LOG>
__device__ __forceinline__ int count_slots(const W4Args& g)
{
    const int E = g.w.E, cap = (int)g.cap;
    if (!g.expert_offsets) return (cap + (1 << LOG) - 1) >> LOG;
    int tiles = 0;
    for (int e = lane_id(); e < E; e += kWave)
        tiles += (max(min(g.expert_offsets[e + 1], cap) - min(g.expert_offsets[e], cap), 0) + (1 << LOG) - 1) >> LOG;
    return __builtin_amdgcn_readlane(wave_scan_dpp(tiles), kWave - 1);
}

// Blocks of the wide kernel to a CU: 168 registers allow three of those with
// 32 slots, whose time is the weight's stream (61 tokens, 32 experts, K = 2048,
// N = 7168, groups of 32: 60.5 us against 65.6 with two).  With groups of 128 the
// bounds make them spill 13 to 19 registers, of 64 2 or 3, outside the loop over k.
constexpr int wide_blocks(int maxmt) { return maxmt == 2 ? 3 : 2; }

// `tiles`: the experts' slot tiles.
template <bool SWIGLU, int MAXMT, int GPT>
__device__ __forceinline__ void w4_wide(const W4Args& g, unsigned char* lds, int tiles)
{
    constexpr int LOG = MAXMT == 2 ? 5 : 6;
    constexpr int kSbs = kWideWaves * (SWIGLU ? 1 : 2);      // superblocks of a tile (SwiGLU: of the gate part)
    const uint32_t nb = (uint32_t)(((SWIGLU ? g.w.part_sbs : g.w.sbs) + kSbs - 1) / kSbs);
    // XCD x (blocks b % 8 = x) takes a contiguous range of tiles, an expert's
    // slot tiles innermost, so that they read its weight through the same L2
    const uint32_t Q = (uint32_t)__builtin_amdgcn_readfirstlane(tiles) * nb;
    const uint32_t per = (Q + 7) / 8;
    for (uint32_t l = blockIdx.x >> 3; l < per; l += gridDim.x >> 3) {
        const uint32_t q = (blockIdx.x & 7) * per + l;
        if (q >= Q) break;
        W4Tile t;
        find_tile<LOG>(g, q, nb, t);
        t.e = __builtin_amdgcn_readfirstlane(t.e);
        t.s0 = __builtin_amdgcn_readfirstlane((int)t.s0);
        t.rows = __builtin_amdgcn_readfirstlane(t.rows);
        t.b = __builtin_amdgcn_readfirstlane(t.b) * kSbs;
        __syncthreads();        // (the last tile's reads of LDS)
        if (t.rows <= 16) {
            w4_wide_tile<SWIGLU, 1, MAXMT, GPT>(g, t, lds);
        } else if (MAXMT == 2 || t.rows <= 32) {
            w4_wide_tile<SWIGLU, 2, MAXMT, GPT>(g, t, lds);
        } else if constexpr (MAXMT == 4) {
            if (t.rows <= 48) w4_wide_tile<SWIGLU, 3, MAXMT, GPT>(g, t, lds);
            else w4_wide_tile<SWIGLU, 4, MAXMT, GPT>(g, t, lds);
        }
    }
}

// All slots, where the host doesn't know them.
__device__ __forceinline__ int slots_of(const W4Args& g) { return min(g.expert_offsets[g.w.E], (int)g.cap); }

// from: the slots below which another kernel does the work (0: none does).
template <bool SWIGLU, int MAXMT, int GPT>
__global__ __launch_bounds__(kWideWaves * kWave, wide_blocks(MAXMT)) void w4_wide_kernel(W4Args g, int from)
{
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * wide_buf(MAXMT)];
    if (from && slots_of(g) < from) return;
    w4_wide<SWIGLU, MAXMT, GPT>(g, lds, count_slots<MAXMT == 2 ? 5 : 6>(g));
}

// The same choice as the host's (w4_route) with the slots that there are: split
// below `wide` of them, wide below `wide64`, where w4_wide_kernel's 64-slot tiles take over.
// A program that doesn't read the count back gives a capacity with room to spare, T * E for certain;
// chosen by that, 100 tokens of two experts of 8 (K = 4096, N = 2048) took 39.2 us, and
// 18.2 so (18.1 with the count known), 70 of two of 64 (2048, 2816) 43.6 and 40.1 (38.5: the launch
// that finds no work takes the rest).  At an exact capacity that the host doesn't know to be exact
// it costs nothing measurable.
template <bool SWIGLU, int GPT>
__global__ __launch_bounds__(kWideWaves * kWave, wide_blocks(2)) void w4_choose_kernel(W4Args g, int wide, int wide64)
{
    __shared__ __attribute__((aligned(16))) unsigned char lds[std::max<int>(2 * wide_buf(2), 4 * split_lds(2, 4))];
    // (both loads at once: one wait in front of the work)
    const int tiles = count_slots<5>(g), slots = slots_of(g);
    if (slots >= wide64) return;
    if (slots >= wide) w4_wide<SWIGLU, 2, GPT>(g, lds, tiles);
    else w4_split<SWIGLU, 2, GPT, 4>(g, (float*)lds);
}

// What the host knows of a call, and what follows from it.
struct W4Load {
    int64_t busy, mean;    // experts with slots, and slots of one, as far as the capacity tells
    int64_t cus;
};

// Units of the split kernel: 64 weight rows (SwiGLU: 32 hidden units) by 16
// slots; tiles of the wide one: 256 weight rows by 32 slots.  A mean of n slots
// makes about n / 16 + 1/2 slot tiles of 16.
int64_t split_units(const W4Args& g, bool swiglu, const W4Load& l)
{
    return l.busy * std::max<int64_t>(16, l.mean + 8) * (swiglu ? g.w.part_sbs : (g.w.sbs + 1) / 2) / 16;
}

int64_t wide_tiles(const W4Args& g, bool swiglu, const W4Load& l)
{
    const int sbs = kWideWaves * (swiglu ? 1 : 2);
    return l.busy * std::max<int64_t>(32, l.mean + 16) * (((swiglu ? g.w.part_sbs : g.w.sbs) + sbs - 1) / sbs) / 32;
}

// Slots from which the wide kernels are taken.
struct W4From {
    int64_t wide, wide64;
};

enum W4Route { kSplit4 = 0, kSplit8 = 1, kWide32 = 2, kWide64 = 3 };

// Which kernel a call takes.
//
// Split K or lay the waves side by side.  Where the weights' stream is what
// counts the split kernel is 9% faster up to a mean of 2 slots, they are equal at 4
// and the wide one is 2 to 27% faster from 6 on (us, split / wide; K = 4096,
// N = 4096, 128 experts, 17 to 128 tokens: 141 / 155, 177 / 194, 201 / 204, 226 / 208;
// 32 experts, K = 2048, N = 7168, 24 and 61 tokens: 54 / 53, 79 / 58).  In calls of few
// tiles a wide one takes 33 us at K = 4096 however few they are, and 768 of them
// (three to a CU) little more, while 45 units of the split kernel pass in a us:
// 8 experts, 40 tokens 20 / 34, dense, 48 and 200 tokens: 8.6 / 32, 42 / 33.
//
// Eight waves on one superblock where there are then no more blocks than CUs
// (dense, one token, K = N = 4096: 5.4 us against 7.7 with four waves on two; 48
// tokens, 384 blocks: 14.4 against 8.6).
//
// Slot tiles of 64 where there are many slots and tiles (32 experts of 75 slots,
// K = 2048, N = 7168: 111 us against 123; up to a mean of 64 equal, in calls of few
// tiles 35% slower: dense, 64 tokens, K = N = 4096 45 against 33).
int w4_route(const W4Args& g, bool swiglu, const W4Load& l, int64_t most)
{
    const int64_t units = split_units(g, swiglu, l), tiles = wide_tiles(g, swiglu, l);
    if (most > 16 && l.mean > 4 && units * 3 * l.cus > 1500 * std::max<int64_t>(3 * l.cus, tiles))
        return l.mean > 64 && tiles >= 4 * l.cus ? kWide64 : kWide32;
    return 2 * units <= l.cus ? kSplit8 : kSplit4;
}

template <bool SWIGLU, int NSB, int WAVES>
int launch_split(const W4Args& g, int cus, hipStream_t s)
{
    const int64_t nb = SWIGLU ? g.w.part_sbs : (g.w.sbs + NSB - 1) / NSB;
    const int64_t tiles = std::min<int64_t>(g.cap, g.cap / 16 + g.w.E);
    // (12 waves to a CU are what the registers allow)
    const dim3 grid((unsigned)std::min<int64_t>(tiles * nb, (int64_t)cus * (12 / WAVES))), block(WAVES * kWave);
    switch (g.w.gpt()) {
        case 1: w4_split_kernel<SWIGLU, NSB, 1, WAVES><<<grid, block, 0, s>>>(g); break;
        case 2: w4_split_kernel<SWIGLU, NSB, 2, WAVES><<<grid, block, 0, s>>>(g); break;
        default: w4_split_kernel<SWIGLU, NSB, 4, WAVES><<<grid, block, 0, s>>>(g); break;
    }
    return check_launch("w4_split_kernel");
}

template <bool SWIGLU, int MAXMT>
int launch_wide(const W4Args& g, int cus, hipStream_t s, int from = 0)
{
    constexpr int kSbs = kWideWaves * (SWIGLU ? 1 : 2);
    const int64_t nb = ((SWIGLU ? g.w.part_sbs : g.w.sbs) + kSbs - 1) / kSbs;
    const int64_t tiles = std::min<int64_t>(g.cap, g.cap / (16 * MAXMT) + g.w.E);
    const int64_t blocks = std::min<int64_t>(tiles * nb, (int64_t)cus * wide_blocks(MAXMT));
    const dim3 grid((unsigned)(8 * ((blocks + 7) / 8))), block(kWideWaves * kWave);
    switch (g.w.gpt()) {
        case 1: w4_wide_kernel<SWIGLU, MAXMT, 1><<<grid, block, 0, s>>>(g, from); break;
        case 2: w4_wide_kernel<SWIGLU, MAXMT, 2><<<grid, block, 0, s>>>(g, from); break;
        default: w4_wide_kernel<SWIGLU, MAXMT, 4><<<grid, block, 0, s>>>(g, from); break;
    }
    return check_launch("w4_wide_kernel");
}

template <bool SWIGLU>
int launch_choose(const W4Args& g, const W4From& from, int cus, hipStream_t s)
{
    const int64_t nb = SWIGLU ? g.w.part_sbs : (g.w.sbs + 1) / 2;
    const int64_t tiles = std::min<int64_t>(g.cap, g.cap / 16 + g.w.E);
    const int64_t blocks = std::min<int64_t>(tiles * nb, (int64_t)cus * wide_blocks(2));
    const dim3 grid((unsigned)(8 * ((blocks + 7) / 8))), block(kWideWaves * kWave);
    const int wide = (int)from.wide, wide64 = (int)from.wide64;
    switch (g.w.gpt()) {
        case 1: w4_choose_kernel<SWIGLU, 1><<<grid, block, 0, s>>>(g, wide, wide64); break;
        case 2: w4_choose_kernel<SWIGLU, 2><<<grid, block, 0, s>>>(g, wide, wide64); break;
        default: w4_choose_kernel<SWIGLU, 4><<<grid, block, 0, s>>>(g, wide, wide64); break;
    }
    const int rc = check_launch("w4_choose_kernel");
    return rc || from.wide64 > g.cap ? rc : launch_wide<SWIGLU, 4>(g, cus, s, wide64);
}

template <bool SWIGLU>
int launch_w4(const W4Args& g, int route, int cus, hipStream_t s)
{
    switch (route) {
        case kSplit4: return launch_split<SWIGLU, 2, 4>(g, cus, s);
        case kSplit8: return launch_split<SWIGLU, SWIGLU ? 2 : 1, 8>(g, cus, s);
        case kWide32: return launch_wide<SWIGLU, 2>(g, cus, s);
        default: return launch_wide<SWIGLU, 4>(g, cus, s);
    }
}

W4Load load_of(int64_t num_experts, int64_t slots, int64_t most, int64_t cus)
{
    const int64_t busy = std::max<int64_t>(1, std::min(num_experts, slots));
    return W4Load{busy, std::min(most, (slots + busy - 1) / busy), cus};
}

// The kernel for a number of slots.
int route_of(const W4Args& g, bool swiglu, int64_t slots, int64_t max_slots, int64_t cus)
{
    const int64_t most = std::min(max_slots, slots);
    return w4_route(g, swiglu, load_of(g.w.E, slots, most, cus), most);
}

// The fewest slots, of 1 to the capacity, that take a wide kernel, and the one of 64-slot tiles: more than the
// capacity where none do.  (A route never comes before another's with more slots.)
W4From from_of(const W4Args& g, bool swiglu, int64_t max_slots, int64_t cus)
{
    const auto first = [&](int route) {
        int64_t lo = 1, hi = g.cap + 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (route_of(g, swiglu, mid, max_slots, cus) >= route) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };
    return W4From{first(kWide32), route_of(g, swiglu, g.cap, max_slots, cus) < kWide64 ? g.cap + 1 : first(kWide64)};
}

int check_shape(const char* fn, int64_t E, int64_t N, int64_t K, int64_t group, int64_t parts)
{
    const std::string f(fn);
    if (E < 1 || E > ET_MAX_EXPERTS) return fail(ET_ERR_INVALID_ARGUMENT, f + ": num_experts must be in [1, 1024]");
    if (parts != 1 && parts != 2) return fail(ET_ERR_INVALID_ARGUMENT, f + ": parts must be 1 or 2");
    if (N < 8 * parts || N % (8 * parts)) return fail(ET_ERR_INVALID_ARGUMENT, f + ": N must be a positive multiple of 8 for each part");
    if (K < 8 || K % 8 || K >= (int64_t)1 << 22) return fail(ET_ERR_INVALID_ARGUMENT, f + ": K must be a positive multiple of 8 below 2^22");
    if (group != 32 && group != 64 && group != 128) return fail(ET_ERR_INVALID_ARGUMENT, f + ": group must be 32, 64 or 128");
    if (N >= (int64_t)1 << 22 || N * K >= (int64_t)1 << 31) return fail(ET_ERR_INVALID_ARGUMENT, f + ": N * K must be below 2^31, N below 2^22");
    return ET_OK;
}

W4Shape shape_of(int64_t E, int64_t N, int64_t K, int64_t group, int64_t parts)
{
    const int rows = (int)(N / parts), part_sbs = (rows + kSb - 1) / kSb;
    return W4Shape{(int)E, (int)N, (int)K, (int)parts, (int)group, rows, part_sbs, (int)parts * part_sbs,
                   (int)((K + kKt - 1) / kKt)};
}

// Blocks of the layout kernels, and of a launch of them (less than 2^32 threads).
int64_t blocks_of(const W4Shape& w) { return (int64_t)w.E * w.sbs * w.kts; }
dim3 layout_grid(int64_t blocks) { return dim3((unsigned)std::min<int64_t>(blocks, (int64_t)1 << 22)); }

int check_ptr(const char* fn, const char* name, const void* p, uintptr_t align)
{
    if (!p) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null " + name);
    if ((uintptr_t)p % align) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + name + " is not aligned");
    return ET_OK;
}

int check_scale_type(const char* fn, int t)
{
    if (t != ET_W4_SCALE_BF16 && t != ET_W4_SCALE_F16)
        return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": scale_type must be ET_W4_SCALE_BF16 or ET_W4_SCALE_F16");
    return ET_OK;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" size_t et_w4_packed_bytes(int64_t num_experts, int64_t N, int64_t K, int64_t parts)
{
    if (check_shape("et_w4_packed_bytes", num_experts, N, K, 128, parts)) return 0;
    return (size_t)num_experts * shape_of(num_experts, N, K, 128, parts).expert_bytes();
}

extern "C" size_t et_w4_packed_scales(int64_t num_experts, int64_t N, int64_t K, int64_t group, int64_t parts)
{
    if (check_shape("et_w4_packed_scales", num_experts, N, K, group, parts)) return 0;
    return (size_t)num_experts * shape_of(num_experts, N, K, group, parts).expert_scales();
}

extern "C" int et_w4_pack(const void* q, const void* scales, int64_t num_experts, int64_t N, int64_t K, int64_t group,
                          int64_t parts, void* packed, void* packed_scales, void* stream)
{
    const char* fn = "et_w4_pack";
    int rc = check_shape(fn, num_experts, N, K, group, parts);
    if (rc) return rc;
    const W4Shape w = shape_of(num_experts, N, K, group, parts);
    rc = check_ptr(fn, "q", q, 1);
    if (!rc) rc = check_ptr(fn, "scales", scales, 2);
    if (!rc) rc = check_ptr(fn, "packed", packed, 16);
    if (!rc) rc = check_ptr(fn, "packed_scales", packed_scales, 16);
    if (rc) return rc;
    const int64_t blocks = blocks_of(w);
    w4_pack_kernel<<<layout_grid(blocks), dim3(256), 0, (hipStream_t)stream>>>(
        (const uint8_t*)q, (const uint16_t*)scales, w, blocks, (uint32_t*)packed, (uint16_t*)packed_scales);
    return check_launch("w4_pack_kernel");
}

extern "C" int et_w4_unpack(const void* packed, const void* packed_scales, int scale_type, const int32_t* expert_offsets,
                            int64_t num_experts, int64_t N, int64_t K, int64_t group, int64_t parts,
                            int64_t slot_capacity, void* w, void* stream)
{
    const char* fn = "et_w4_unpack";
    int rc = check_shape(fn, num_experts, N, K, group, parts);
    if (!rc) rc = check_scale_type(fn, scale_type);
    if (rc) return rc;
    const W4Shape sh = shape_of(num_experts, N, K, group, parts);
    rc = check_ptr(fn, "packed", packed, 16);
    if (!rc) rc = check_ptr(fn, "packed_scales", packed_scales, 16);
    if (!rc) rc = check_ptr(fn, "w", w, 16);
    if (rc) return rc;
    if (slot_capacity < 0) return fail(ET_ERR_INVALID_ARGUMENT, "et_w4_unpack: slot_capacity must be >= 0");
    const int64_t blocks = blocks_of(sh);
    w4_unpack_kernel<<<layout_grid(blocks), dim3(256), 0, (hipStream_t)stream>>>(
        (const uint32_t*)packed, (const uint16_t*)packed_scales, scale_type == ET_W4_SCALE_F16, sh, blocks, expert_offsets,
        slot_capacity, (uint16_t*)w);
    return check_launch("w4_unpack_kernel");
}

namespace et {
namespace {

template <typename X>
void launch_quantize(const void* w, int64_t rows, int64_t K, int64_t group, bool half, void* q, void* scales, hipStream_t s)
{
    const int64_t threads = rows * ((K + group - 1) / group * (group / 8));
    const dim3 grid = layout_grid((threads + 255) / 256), block(256);
    switch (group) {
        case 32: w4_quantize_kernel<X, 32><<<grid, block, 0, s>>>((const X*)w, rows, (int)K, half, (uint32_t*)q, (uint16_t*)scales); break;
        case 64: w4_quantize_kernel<X, 64><<<grid, block, 0, s>>>((const X*)w, rows, (int)K, half, (uint32_t*)q, (uint16_t*)scales); break;
        default: w4_quantize_kernel<X, 128><<<grid, block, 0, s>>>((const X*)w, rows, (int)K, half, (uint32_t*)q, (uint16_t*)scales); break;
    }
}

int cus_of_device()
{
    static thread_local int cus[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (!cus[dev] && (hipDeviceGetAttribute(&cus[dev], hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus[dev] < 1))
        cus[dev] = 256;
    return cus[dev];
}

}  // namespace
}  // namespace et

extern "C" int et_w4_quantize(const void* w, int dtype, int64_t num_experts, int64_t N, int64_t K, int64_t group,
                              int scale_type, void* q, void* scales, void* stream)
{
    const char* fn = "et_w4_quantize";
    int rc = check_shape(fn, num_experts, N, K, group, 1);
    if (!rc) rc = check_scale_type(fn, scale_type);
    if (rc) return rc;
    if (dtype != ET_DTYPE_F32 && dtype != ET_DTYPE_BF16)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_w4_quantize: dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    rc = check_ptr(fn, "w", w, dtype == ET_DTYPE_F32 ? 4 : 2);
    if (!rc) rc = check_ptr(fn, "q", q, 4);
    if (!rc) rc = check_ptr(fn, "scales", scales, 2);
    if (rc) return rc;
    const bool half = scale_type == ET_W4_SCALE_F16;
    if (dtype == ET_DTYPE_F32) launch_quantize<float>(w, num_experts * N, K, group, half, q, scales, (hipStream_t)stream);
    else launch_quantize<uint16_t>(w, num_experts * N, K, group, half, q, scales, (hipStream_t)stream);
    return check_launch("w4_quantize_kernel");
}

// The kernel that et_expert_gemm_w4_impl takes of itself (W4Route).
extern "C" int et_w4_route_impl(int64_t num_experts, int64_t K, int64_t N, int64_t group, int64_t parts,
                                int64_t slot_capacity, int epilogue, int64_t max_slots, int64_t cus)
{
    W4Args g = {};
    g.w = shape_of(num_experts, N, K, group, parts);
    return route_of(g, epilogue == EPI_SWIGLU, slot_capacity, max_slots, cus);
}

// The slots from which it takes a wide one (which 0) or that of 64-slot tiles (1), where
// the slots are known on the device alone.
extern "C" int64_t et_w4_from_impl(int64_t num_experts, int64_t K, int64_t N, int64_t group, int64_t parts,
                                   int64_t slot_capacity, int epilogue, int64_t max_slots, int64_t cus, int which)
{
    W4Args g = {};
    g.w = shape_of(num_experts, N, K, group, parts);
    g.cap = slot_capacity;
    const W4From from = from_of(g, epilogue == EPI_SWIGLU, max_slots, cus);
    return which ? from.wide64 : from.wide;
}

// max_slots: slots of one expert at most, as far as the host knows.  route: a
// W4Route, or -1 for the one that w4_route says.  known: the slots are as many as the
// capacity; else they may be fewer, and where that decides, the device chooses.
extern "C" int et_expert_gemm_w4_impl(const void* a, int64_t a_rows, const int32_t* sorted_token, const void* packed,
                                      const void* packed_scales, int scale_type, const int32_t* expert_offsets,
                                      int64_t num_experts, int64_t K, int64_t N, int64_t group, int64_t parts,
                                      int64_t slot_capacity, int epilogue, const float* row_scale, void* c,
                                      int64_t max_slots, int route, int known, void* stream)
{
    const char* fn = "et_expert_gemm_w4";
    int rc = check_shape(fn, num_experts, N, K, group, parts);
    if (!rc) rc = check_scale_type(fn, scale_type);
    if (rc) return rc;
    if (epilogue != EPI_PLAIN && epilogue != EPI_ROW_SCALE && epilogue != EPI_SWIGLU)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: unknown epilogue");
    if (epilogue == EPI_SWIGLU && parts != 2)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: SwiGLU needs a weight laid out in two parts");
    if (slot_capacity < 0 || slot_capacity >= (int64_t)1 << 31 || a_rows < 0)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: slot_capacity must be in [0, 2^31), a_rows >= 0");
    if (sorted_token && a_rows * K * 2 >= (int64_t)1 << 31)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: in gather mode the token matrix must be below 2 GiB");
    if (!expert_offsets && num_experts != 1)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: more than one expert needs expert_offsets");
    if (!expert_offsets && sorted_token)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: gather mode needs expert_offsets");
    if (slot_capacity == 0) return ET_OK;
    rc = check_ptr(fn, "a", a, 16);
    if (!rc) rc = check_ptr(fn, "packed", packed, 16);
    if (!rc) rc = check_ptr(fn, "packed_scales", packed_scales, 16);
    if (!rc) rc = check_ptr(fn, "c", c, 16);
    if (!rc && epilogue == EPI_ROW_SCALE) rc = check_ptr(fn, "row_scale", row_scale, 4);
    if (rc) return rc;
    W4Args g{(const uint16_t*)a, sorted_token, (const unsigned char*)packed, (const uint16_t*)packed_scales, expert_offsets,
             (uint16_t*)c, epilogue == EPI_ROW_SCALE ? row_scale : nullptr, a_rows, slot_capacity,
             shape_of(num_experts, N, K, group, parts), scale_type == ET_W4_SCALE_F16};
    // (tiles are counted in 32 bits: 16 slots by 32 rows at the least)
    if ((slot_capacity / 16 + num_experts + 1) * (int64_t)g.w.sbs >= (int64_t)1 << 31)
        return fail(ET_ERR_INVALID_ARGUMENT, "et_expert_gemm_w4: slot_capacity times N is too large");
    const bool swiglu = epilogue == EPI_SWIGLU;
    const int cus = cus_of_device();
    if (route < kSplit4 || route > kWide64) {
        route = route_of(g, swiglu, slot_capacity, max_slots, cus);
        if (!known && expert_offsets && route >= kWide32) {
            const W4From from = from_of(g, swiglu, max_slots, cus);
            return swiglu ? launch_choose<true>(g, from, cus, (hipStream_t)stream)
                          : launch_choose<false>(g, from, cus, (hipStream_t)stream);
        }
    }
    return swiglu ? launch_w4<true>(g, route, cus, (hipStream_t)stream) : launch_w4<false>(g, route, cus, (hipStream_t)stream);
}

extern "C" int et_expert_gemm_w4(const void* a, int64_t a_rows, const int32_t* sorted_token, const void* packed,
                                 const void* packed_scales, int scale_type, const int32_t* expert_offsets,
                                 int64_t num_experts, int64_t K, int64_t N, int64_t group, int64_t parts,
                                 int64_t slot_capacity, int epilogue, const float* row_scale, void* c, void* stream)
{
    return et_expert_gemm_w4_impl(a, a_rows, sorted_token, packed, packed_scales, scale_type, expert_offsets, num_experts, K,
                                  N, group, parts, slot_capacity, epilogue, row_scale, c, slot_capacity, -1, 0, stream);
}
