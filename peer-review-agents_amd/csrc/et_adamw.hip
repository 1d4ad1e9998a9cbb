// et_adamw.hip -- AdamW over many tensors, with states in 32 or in 8 bits, and
// the global gradient norm (gfx950).
#include <algorithm>

#include "et_common.hpp"
#include "etmoe_block.h"

namespace et {
namespace {

constexpr int kThreads = 256;
// Elements of one block of the AdamW kernels: one vector of four for a thread,
// one block of the 8-bit states for a wave.  HBM bounds the kernels, and blocks
// that come and go keep the range in flight narrow.  One tensor of 201.5M elements, f32
// gradients, back to back on one card (us; 1024, 4096 and 8192 elements to a block):
//   f32 parameters, f32 states, 28 bytes an element, 5.64 GB      919   923   938   6.14 TB/s
//   bf16 parameters and masters, f32 states, 30 bytes, 6.04 GB    980   987   996   6.16
//   f32 parameters, 8-bit states, 16.06 bytes, 3.24 GB            537   579   573   6.03
//   bf16 and masters, 8-bit states, stochastic, 18.06, 3.64 GB    611   620   617   5.95
constexpr int kChunk = 1024;
constexpr int kNormChunk = 16384;     // elements of one block of the norm
// Tensors of one launch: their table is a kernel argument of 4 KiB at most.
constexpr int kTensors = 64, kTensors8 = 48, kNormTensors = 64;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// The tensors of one launch.  Blocks first[i] to first[i + 1] - 1 are tensor
// i's chunks; unused entries hold the launch's block count.
template <int N>
struct Spans {
    uint32_t first[N];
    int64_t numel[N];
};

// Chunk of a block: the last first.  Behind a gradient norm the gradients that
// are still in the last-level cache are those at the end (201.5M elements with
// masters and the norm 1133 to 1122 us).
__device__ __forceinline__ uint32_t chunk_of_block() { return gridDim.x - 1 - blockIdx.x; }

// The tensor of a chunk, found by the wave at once: lane i looks at entry i.
template <int N>
__device__ __forceinline__ int find_tensor(const Spans<N>& s, uint32_t block)
{
    static_assert(N <= kWave, "one lane per tensor");
    const int lane = lane_id();
    const bool at = lane < N && s.first[lane < N ? lane : 0] <= block;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at)) - 1);
}

template <typename G>
__device__ __forceinline__ float load_grad(const G* g)
{
    if constexpr (sizeof(G) == 2) return u2f((uint32_t)*g << 16);
    else return *g;
}

template <typename G>
__device__ __forceinline__ f32x4_t load_grad4(const G* g)
{
    if constexpr (sizeof(G) == 2) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(g);
        return f32x4_t{bf16lo(w[0]), bf16hi(w[0]), bf16lo(w[1]), bf16hi(w[1])};
    } else {
        return *reinterpret_cast<const f32x4_t*>(g);
    }
}

template <typename P>
__device__ __forceinline__ void store_param(P* p, float v)
{
    if constexpr (sizeof(P) == 2) *p = (P)f32_to_bf16_bits(v);
    else *p = v;
}

template <typename P>
__device__ __forceinline__ void store_param4(P* p, const float (&v)[4])
{
    if constexpr (sizeof(P) == 2)
        *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else
        *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
}

// g scaled; m and v stepped; the weight from them and from root = sqrt(v).
__device__ __forceinline__ void step_moments(const et_adamw_scalars& a, float g, float& m, float& v)
{
    m = m * a.beta1 + g * a.one_minus_beta1;
    v = v * a.beta2 + (g * g) * a.one_minus_beta2;
}

__device__ __forceinline__ float step_weight(const et_adamw_scalars& a, float w, float m, float root)
{
    return w * a.decay - (m / (root * a.inv_root_bias2 + a.eps)) * a.step_size;
}

// 1 without a scale; a scale that is not finite skips the step.
__device__ __forceinline__ bool read_scale(const float* scale, float& s)
{
    s = scale ? *scale : 1.0f;
    return __builtin_fabsf(s) < __builtin_inff();
}

// ---------------------------------------------------------------------------
// f32 states
// ---------------------------------------------------------------------------

struct AdamWArgs {
    Spans<kTensors> spans;
    void* param[kTensors];
    const void* grad[kTensors];
    float* m[kTensors];
    float* v[kTensors];
    float* master[kTensors];
    et_adamw_scalars a;
    const float* grad_scale;
};

// 28 bytes an element, 30 with a bf16 parameter and its f32 master, for some 20
// operations: HBM bounds it (times at kChunk, from the second call on the same tensors;
// 201.5M elements with masters, other ones every call: 996 and 1078 us on two cards).
template <typename P, typename G>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamWArgs t)
{
    constexpr bool kMaster = sizeof(P) == 2;
    float scale;
    if (!read_scale(t.grad_scale, scale)) return;
    const uint32_t chunk = chunk_of_block();
    const int i = find_tensor(t.spans, chunk);
    const int64_t base = (int64_t)(chunk - t.spans.first[i]) * kChunk;
    const int n = (int)min<int64_t>(t.spans.numel[i] - base, kChunk);
    P* const p = (P*)t.param[i] + base;
    const G* const g = (const G*)t.grad[i] + base;
    float* const m = t.m[i] + base;
    float* const v = t.v[i] + base;
    float* const w = kMaster ? t.master[i] + base : (float*)p;
    const bool wide = (((uintptr_t)m | (uintptr_t)v | (uintptr_t)w) & 15) == 0 &&
                      ((uintptr_t)g & (4 * sizeof(G) - 1)) == 0 && ((uintptr_t)p & (4 * sizeof(P) - 1)) == 0;
    int at = 0;
    if (wide) {
        for (; at + 4 * kThreads <= n; at += 4 * kThreads) {
            const int k = at + 4 * (int)threadIdx.x;
            const f32x4_t gv = load_grad4(g + k);
            f32x4_t mv = *reinterpret_cast<const f32x4_t*>(m + k), vv = *reinterpret_cast<const f32x4_t*>(v + k);
            const f32x4_t wv = *reinterpret_cast<const f32x4_t*>(w + k);
            float out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float mj = mv[j], vj = vv[j];
                step_moments(t.a, gv[j] * scale, mj, vj);
                out[j] = step_weight(t.a, wv[j], mj, __builtin_sqrtf(vj));
                mv[j] = mj;
                vv[j] = vj;
            }
            *reinterpret_cast<f32x4_t*>(m + k) = mv;
            *reinterpret_cast<f32x4_t*>(v + k) = vv;
            if constexpr (kMaster) *reinterpret_cast<f32x4_t*>(w + k) = f32x4_t{out[0], out[1], out[2], out[3]};
            store_param4(p + k, out);
        }
    }
    for (int k = at + (int)threadIdx.x; k < n; k += kThreads) {
        float mj = m[k], vj = v[k];
        step_moments(t.a, load_grad(g + k) * scale, mj, vj);
        const float out = step_weight(t.a, w[k], mj, __builtin_sqrtf(vj));
        m[k] = mj;
        v[k] = vj;
        if constexpr (kMaster) w[k] = out;
        store_param(p + k, out);
    }
}

// ---------------------------------------------------------------------------
// 8-bit states
// ---------------------------------------------------------------------------

struct AdamW8Args {
    Spans<kTensors8> spans;
    void* param[kTensors8];
    const void* grad[kTensors8];
    uint8_t* m8[kTensors8];
    float* m_scale[kTensors8];
    uint8_t* u8[kTensors8];
    float* u_scale[kTensors8];
    float* master[kTensors8];
    et_adamw_scalars a;
    const float* grad_scale;
    uint32_t seed;
    uint32_t origin[kTensors8];   // index of each tensor's first element in the call
};

__device__ __forceinline__ uint32_t random_word(uint32_t seed, uint32_t i)
{
    uint32_t x = i * 0x9E3779B1u + seed;
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    x = (x ^ (x >> 13)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

// r in [0, 448] up or down to a multiple of its e4m3 step, by 16 random bits:
// the 20 fraction bits that are left out and the random ones carry.  Below 2^-6
// the steps stay 2^-9, as they are in [2^-6, 2^-5), so r moves there and back.
__device__ __forceinline__ float dither(float r, uint32_t bits16)
{
    const float small = r < 0.015625f ? 0.015625f : 0.0f;
    const uint32_t b = (f2u(r + small) + (bits16 << 4)) & 0xFFF00000u;
    return __builtin_fminf(u2f(b) - small, 448.0f);
}

// The scale of a block whose largest |x| has the bits `most` (an unsigned
// maximum of the bits, which puts NaN above infinity above the finite), and
// the factor that makes it 448.
__device__ __forceinline__ void block_scale(uint32_t most, float& scale, float& inv)
{
    const float a = u2f(most);
    const bool zero = a < 1e-35f;
    scale = zero ? 0.0f : most < 0x7F800000u ? a * (1.0f / 448.0f) : u2f(0x7FC00000u);
    inv = zero ? 0.0f : 448.0f / a;
}

// Four elements' values of a block to e4m3 bytes.
template <bool STOCHASTIC, bool ROOT>
__device__ __forceinline__ uint32_t to_e4m3x4(const float (&x)[4], float inv, const uint32_t (&words)[4])
{
    float r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float q = __builtin_fminf(__builtin_fabsf(x[j]) * inv, 448.0f);
        if constexpr (STOCHASTIC) q = dither(q, ROOT ? words[j] & 0xFFFFu : words[j] >> 16);
        if constexpr (ROOT) q = x[j] > 0.0f && inv > 0.0f ? __builtin_fmaxf(q, 0.001953125f) : q;
        r[j] = ROOT ? q : __builtin_copysignf(q, x[j]);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], w, true);
}

__device__ __forceinline__ void from_e4m3x4(uint32_t w, float scale, float (&x)[4])
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0] * scale;
    x[1] = lo[1] * scale;
    x[2] = hi[0] * scale;
    x[3] = hi[1] * scale;
}

// A block of 256 elements is a wave's, four to a lane, so its largest |m| and sqrt(v)
// are found within the wave and nothing is read twice.  16 to 18 bytes an element: HBM
// bounds it (times at kChunk; 201.5M elements with masters, other ones every call: 652 and
// 664 us on two cards).
template <typename P, typename G, bool STOCHASTIC>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(AdamW8Args t)
{
    constexpr bool kMaster = sizeof(P) == 2;
    constexpr int kB = ET_ADAMW8_BLOCK;
    float scale;
    if (!read_scale(t.grad_scale, scale)) return;
    const uint32_t chunk = chunk_of_block();
    const int i = find_tensor(t.spans, chunk);
    const int64_t base = (int64_t)(chunk - t.spans.first[i]) * kChunk;
    const int64_t left = t.spans.numel[i] - base;
    const int n = (int)min<int64_t>(left, kChunk);
    P* const p = (P*)t.param[i] + base;
    const G* const g = (const G*)t.grad[i] + base;
    uint8_t* const m8 = t.m8[i] + base;
    uint8_t* const u8 = t.u8[i] + base;
    float* const ms = t.m_scale[i] + base / kB;
    float* const us = t.u_scale[i] + base / kB;
    float* const w = kMaster ? t.master[i] + base : (float*)p;
    const bool aligned = ((uintptr_t)w & 15) == 0 && (((uintptr_t)m8 | (uintptr_t)u8) & 3) == 0 &&
                         ((uintptr_t)g & (4 * sizeof(G) - 1)) == 0 && ((uintptr_t)p & (4 * sizeof(P) - 1)) == 0;
    const int lane = lane_id(), wave = (int)threadIdx.x / kWave;
    const uint32_t index = t.origin[i] + (uint32_t)base;
    for (int b = wave; b * kB < n; b += kThreads / kWave) {
        const int k = b * kB + 4 * lane;
        const int live = min(max(n - k, 0), 4);      // this lane's elements
        const bool wide = aligned && (b + 1) * kB <= n;
        float gv[4], wv[4], mv[4], uv[4];
        uint32_t mw = 0, uw = 0;
        if (wide) {
            const f32x4_t g4 = load_grad4(g + k), w4 = *reinterpret_cast<const f32x4_t*>(w + k);
            mw = *reinterpret_cast<const uint32_t*>(m8 + k);
            uw = *reinterpret_cast<const uint32_t*>(u8 + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                gv[j] = g4[j];
                wv[j] = w4[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = j < live;
                gv[j] = in ? load_grad(g + k + j) : 0.0f;
                wv[j] = in ? w[k + j] : 0.0f;
                mw |= in ? (uint32_t)m8[k + j] << (8 * j) : 0u;
                uw |= in ? (uint32_t)u8[k + j] << (8 * j) : 0u;
            }
        }
        from_e4m3x4(mw, ms[b], mv);
        from_e4m3x4(uw, us[b], uv);
        uint32_t mmax = 0, umax = 0;
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v = uv[j] * uv[j];
            step_moments(t.a, gv[j] * scale, mv[j], v);
            uv[j] = __builtin_sqrtf(v);
            wv[j] = step_weight(t.a, wv[j], mv[j], uv[j]);
            mmax = max(mmax, f2u(mv[j]) & 0x7FFFFFFFu);
            umax = max(umax, f2u(uv[j]) & 0x7FFFFFFFu);
            if constexpr (STOCHASTIC) words[j] = random_word(t.seed, index + (uint32_t)(k + j));
        }
        float mscale, minv, uscale, uinv;
        block_scale(wave_max_u32_dpp(mmax), mscale, minv);
        block_scale(wave_max_u32_dpp(umax), uscale, uinv);
        mw = to_e4m3x4<STOCHASTIC, false>(mv, minv, words);
        uw = to_e4m3x4<STOCHASTIC, true>(uv, uinv, words);
        if (wide) {
            *reinterpret_cast<uint32_t*>(m8 + k) = mw;
            *reinterpret_cast<uint32_t*>(u8 + k) = uw;
            if constexpr (kMaster) *reinterpret_cast<f32x4_t*>(w + k) = f32x4_t{wv[0], wv[1], wv[2], wv[3]};
            store_param4(p + k, wv);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= live) continue;
                m8[k + j] = (uint8_t)(mw >> (8 * j));
                u8[k + j] = (uint8_t)(uw >> (8 * j));
                if constexpr (kMaster) w[k + j] = wv[j];
                store_param(p + k + j, wv[j]);
            }
        }
        if (lane == 0) {
            ms[b] = mscale;
            us[b] = uscale;
        }
    }
}

// ---------------------------------------------------------------------------
// gradient norm
// ---------------------------------------------------------------------------

struct NormArgs {
    Spans<kNormTensors> spans;
    const void* grad[kNormTensors];
    uint8_t bf16[kNormTensors];
    double* partial;             // of this launch's blocks
};

// Squares of binary32 are exact in binary64; four loads of a thread at a time.
template <typename G>
__device__ __forceinline__ double sum_squares(const G* g, int n)
{
    constexpr int kStep = 4 * kThreads, kUnroll = 4;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    int at = 0;
    if (((uintptr_t)g & (4 * sizeof(G) - 1)) == 0) {
        const G* const mine = g + 4 * (int)threadIdx.x;
        for (; at + kUnroll * kStep <= n; at += kUnroll * kStep) {
            f32x4_t v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) v[u] = load_grad4(mine + at + u * kStep);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = __builtin_fma((double)v[u][j], (double)v[u][j], s[j]);
        }
        for (; at + kStep <= n; at += kStep) {
            const f32x4_t v = load_grad4(mine + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = __builtin_fma((double)v[j], (double)v[j], s[j]);
        }
    }
    for (int k = at + (int)threadIdx.x; k < n; k += kThreads) {
        const double v = load_grad(g + k);
        s[0] = __builtin_fma(v, v, s[0]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double s)
{
    __shared__ double part[THREADS / kWave];
    s = wave_sum_dpp_f64(s);
    if (lane_id() == 0) part[threadIdx.x / kWave] = s;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) all += part[i];
    return all;
}

// Each block's sum of squares in binary64, of squares in binary64.  Reading bounds it:
// 806 MB 136 us, 5.94 TB/s (140 with one load at a time instead of four).
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(NormArgs t)
{
    const int i = find_tensor(t.spans, blockIdx.x);
    const int64_t base = (int64_t)(blockIdx.x - t.spans.first[i]) * kNormChunk;
    const int n = (int)min<int64_t>(t.spans.numel[i] - base, kNormChunk);
    const double s = t.bf16[i] ? sum_squares((const uint16_t*)t.grad[i] + base, n)
                               : sum_squares((const float*)t.grad[i] + base, n);
    const double all = block_sum<kThreads>(s);
    if (threadIdx.x == 0) t.partial[blockIdx.x] = all;
}

// One block, eight loads of a thread at a time (12297 partials, of 201.5M elements: 5 us;
// 15 one by one in 256 threads).
constexpr int kFinishThreads = 1024;

__global__ __launch_bounds__(kFinishThreads) void grad_norm_finish_kernel(const double* partial, int64_t n, float max_norm,
                                                                          float* norm, float* scale)
{
    double s = 0.0;
    int64_t k = threadIdx.x;
    for (; k + 7 * kFinishThreads < n; k += 8 * kFinishThreads) {
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = partial[k + j * kFinishThreads];
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; k < n; k += kFinishThreads) s += partial[k];
    const double all = block_sum<kFinishThreads>(s);
    if (threadIdx.x == 0) {
        const float v = (float)__builtin_sqrt(all);
        *norm = v;
        if (scale) *scale = v < __builtin_inff() ? __builtin_fminf(1.0f, max_norm / (v + 1e-6f)) : u2f(0x7FC00000u);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int64_t chunks(int64_t numel, int chunk) { return (numel + chunk - 1) / chunk; }

int check_list(const char* fn, const int64_t* numel, int64_t count)
{
    if (count < 0) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": count must be >= 0");
    if (count > 0 && !numel) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null numel");
    for (int64_t i = 0; i < count; ++i) {
        if (numel[i] < 0 || numel[i] >= (int64_t)1 << 40)
            return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": numel must be in [0, 2^40)");
    }
    return ET_OK;
}

int check_pointers(const char* fn, const char* name, const void* const* list, const int64_t* numel, int64_t count,
                   uintptr_t align)
{
    if (count > 0 && !list) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null " + name);
    for (int64_t i = 0; i < count; ++i) {
        if (numel[i] == 0) continue;
        if (!list[i]) return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": null pointer in " + name);
        if ((uintptr_t)list[i] % align)
            return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": a pointer in " + name + " is not aligned");
    }
    return ET_OK;
}

int check_step(const char* fn, int param_dtype, int grad_dtype, const void* masters)
{
    for (const int dt : {param_dtype, grad_dtype})
        if (dt != ET_DTYPE_F32 && dt != ET_DTYPE_BF16)
            return fail(ET_ERR_INVALID_ARGUMENT, std::string(fn) + ": dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    if ((param_dtype == ET_DTYPE_BF16) != (masters != nullptr))
        return fail(ET_ERR_INVALID_ARGUMENT,
                    std::string(fn) + ": bf16 parameters need f32 masters, f32 parameters take none");
    return ET_OK;
}

// Walks the tensors with elements in launches of up to N of them: put(slot, i,
// element of tensor i that the slot begins at, that element's index in the
// call) fills a slot, go(blocks) enqueues.  A launch has less than 2^32 threads: a
// tensor of more is dealt to several slots.
template <int N, typename Put, typename Go>
int each_launch(const int64_t* numel, int64_t count, int chunk, Spans<N>& spans, Put put, Go go)
{
    constexpr int64_t kMostBlocks = ((int64_t)1 << 32) / kThreads - 1;
    uint64_t element = 0;
    int slot = 0;
    int64_t blocks = 0;
    const auto flush = [&]() -> int {
        for (int j = slot; j < N; ++j) {
            spans.first[j] = (uint32_t)blocks;
            spans.numel[j] = 0;
        }
        const int rc = slot ? go((unsigned)blocks) : ET_OK;
        slot = 0;
        blocks = 0;
        return rc;
    };
    for (int64_t i = 0; i < count; ++i) {
        int64_t from = 0;
        while (from < numel[i]) {
            if (slot == N || blocks == kMostBlocks) {
                const int rc = flush();
                if (rc) return rc;
            }
            const int64_t n = std::min(chunks(numel[i] - from, chunk), kMostBlocks - blocks);
            const int64_t size = std::min(numel[i] - from, n * chunk);
            spans.first[slot] = (uint32_t)blocks;
            spans.numel[slot] = size;
            put(slot++, i, from, (uint32_t)(element + (uint64_t)from));
            blocks += n;
            from += size;
        }
        element += (uint64_t)chunks(numel[i], ET_ADAMW8_BLOCK) * ET_ADAMW8_BLOCK;
    }
    return flush();
}

// Entry i of a list, `from` elements of `size` bytes on.
template <typename T>
T* at(T* p, int64_t from, int64_t size)
{
    return p ? (T*)((uintptr_t)p + (uintptr_t)(from * size)) : p;
}

}  // namespace
}  // namespace et

using namespace et;

extern "C" size_t et_grad_norm_workspace_bytes(const int64_t* numel, int64_t count)
{
    if (count < 0 || (count > 0 && !numel)) return 0;
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (numel[i] < 0) return 0;
        n += chunks(numel[i], kNormChunk);
    }
    return (size_t)n * sizeof(double);
}

extern "C" int et_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int64_t count,
                            float max_norm, float* norm, float* scale, void* workspace, size_t workspace_bytes,
                            void* stream)
{
    const char* fn = "et_grad_norm";
    int rc = check_list(fn, numel, count);
    if (rc) return rc;
    if (count > 0 && !dtypes) return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: null dtypes");
    for (int64_t i = 0; i < count; ++i)
        if (dtypes[i] != ET_DTYPE_F32 && dtypes[i] != ET_DTYPE_BF16)
            return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: dtype must be ET_DTYPE_F32 or ET_DTYPE_BF16");
    rc = check_pointers(fn, "grads", grads, numel, count, 2);
    if (rc) return rc;
    for (int64_t i = 0; i < count; ++i)
        if (numel[i] && dtypes[i] == ET_DTYPE_F32 && (uintptr_t)grads[i] % 4)
            return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: a pointer in grads is not aligned");
    if (!norm) return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: null norm");
    if (scale && !(max_norm > 0.0f)) return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: max_norm must be > 0");
    const size_t need = et_grad_norm_workspace_bytes(numel, count);
    if (workspace_bytes < need || (need && !workspace))
        return fail(ET_ERR_WORKSPACE_TOO_SMALL, "et_grad_norm: workspace needs " + std::to_string(need) + " bytes");
    if ((uintptr_t)workspace % 8) return fail(ET_ERR_INVALID_ARGUMENT, "et_grad_norm: workspace must be 8-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    NormArgs args = {};
    double* const partial = (double*)workspace;
    args.partial = partial;
    rc = each_launch<kNormTensors>(
        numel, count, kNormChunk, args.spans,
        [&](int slot, int64_t i, int64_t from, uint32_t) {
            args.grad[slot] = at(grads[i], from, dtypes[i] == ET_DTYPE_BF16 ? 2 : 4);
            args.bf16[slot] = dtypes[i] == ET_DTYPE_BF16;
        },
        [&](unsigned blocks) {
            grad_norm_kernel<<<dim3(blocks), dim3(kThreads), 0, s>>>(args);
            args.partial += blocks;
            return check_launch("grad_norm_kernel");
        });
    if (rc) return rc;
    grad_norm_finish_kernel<<<dim3(1), dim3(kFinishThreads), 0, s>>>(partial, (int64_t)(need / sizeof(double)), max_norm, norm,
                                                               scale);
    return check_launch("grad_norm_finish_kernel");
}

extern "C" int et_adamw(void* const* params, const void* const* grads, float* const* m, float* const* v,
                        float* const* masters, const int64_t* numel, int64_t count, int param_dtype, int grad_dtype,
                        et_adamw_scalars scalars, const float* grad_scale, void* stream)
{
    const char* fn = "et_adamw";
    const auto list = [](auto* p) { return (const void* const*)p; };
    const int pa = param_dtype == ET_DTYPE_BF16 ? 2 : 4, ga = grad_dtype == ET_DTYPE_BF16 ? 2 : 4;   // bytes
    int rc = check_list(fn, numel, count);
    if (!rc) rc = check_step(fn, param_dtype, grad_dtype, masters);
    if (!rc) rc = check_pointers(fn, "params", list(params), numel, count, pa);
    if (!rc) rc = check_pointers(fn, "grads", list(grads), numel, count, ga);
    if (!rc) rc = check_pointers(fn, "m", list(m), numel, count, 4);
    if (!rc) rc = check_pointers(fn, "v", list(v), numel, count, 4);
    if (!rc && masters) rc = check_pointers(fn, "masters", list(masters), numel, count, 4);
    if (rc) return rc;
    if ((uintptr_t)grad_scale % 4) return fail(ET_ERR_INVALID_ARGUMENT, "et_adamw: grad_scale is not aligned");
    hipStream_t s = (hipStream_t)stream;
    AdamWArgs args = {};
    args.a = scalars;
    args.grad_scale = grad_scale;
    return each_launch<kTensors>(
        numel, count, kChunk, args.spans,
        [&](int slot, int64_t i, int64_t from, uint32_t) {
            args.param[slot] = at(params[i], from, pa);
            args.grad[slot] = at(grads[i], from, ga);
            args.m[slot] = m[i] + from;
            args.v[slot] = v[i] + from;
            args.master[slot] = masters ? masters[i] + from : nullptr;
        },
        [&](unsigned blocks) {
            const dim3 grid(blocks), block(kThreads);
            if (param_dtype == ET_DTYPE_F32) {
                if (grad_dtype == ET_DTYPE_F32) adamw_kernel<float, float><<<grid, block, 0, s>>>(args);
                else adamw_kernel<float, uint16_t><<<grid, block, 0, s>>>(args);
            } else {
                if (grad_dtype == ET_DTYPE_F32) adamw_kernel<uint16_t, float><<<grid, block, 0, s>>>(args);
                else adamw_kernel<uint16_t, uint16_t><<<grid, block, 0, s>>>(args);
            }
            return check_launch("adamw_kernel");
        });
}

namespace et {
namespace {

template <bool STOCHASTIC>
void launch_adamw8(int param_dtype, int grad_dtype, dim3 grid, const AdamW8Args& args, hipStream_t s)
{
    const dim3 block(kThreads);
    if (param_dtype == ET_DTYPE_F32) {
        if (grad_dtype == ET_DTYPE_F32) adamw8_kernel<float, float, STOCHASTIC><<<grid, block, 0, s>>>(args);
        else adamw8_kernel<float, uint16_t, STOCHASTIC><<<grid, block, 0, s>>>(args);
    } else {
        if (grad_dtype == ET_DTYPE_F32) adamw8_kernel<uint16_t, float, STOCHASTIC><<<grid, block, 0, s>>>(args);
        else adamw8_kernel<uint16_t, uint16_t, STOCHASTIC><<<grid, block, 0, s>>>(args);
    }
}

}  // namespace
}  // namespace et

extern "C" int et_adamw8(void* const* params, const void* const* grads, uint8_t* const* m8, float* const* m_scale,
                         uint8_t* const* u8, float* const* u_scale, float* const* masters, const int64_t* numel,
                         int64_t count, int param_dtype, int grad_dtype, et_adamw_scalars scalars,
                         const float* grad_scale, int rounding, uint32_t seed, void* stream)
{
    const char* fn = "et_adamw8";
    const auto list = [](auto* p) { return (const void* const*)p; };
    const int pa = param_dtype == ET_DTYPE_BF16 ? 2 : 4, ga = grad_dtype == ET_DTYPE_BF16 ? 2 : 4;   // bytes
    int rc = check_list(fn, numel, count);
    if (!rc) rc = check_step(fn, param_dtype, grad_dtype, masters);
    if (!rc) rc = check_pointers(fn, "params", list(params), numel, count, pa);
    if (!rc) rc = check_pointers(fn, "grads", list(grads), numel, count, ga);
    if (!rc) rc = check_pointers(fn, "m8", list(m8), numel, count, 1);
    if (!rc) rc = check_pointers(fn, "m_scale", list(m_scale), numel, count, 4);
    if (!rc) rc = check_pointers(fn, "u8", list(u8), numel, count, 1);
    if (!rc) rc = check_pointers(fn, "u_scale", list(u_scale), numel, count, 4);
    if (!rc && masters) rc = check_pointers(fn, "masters", list(masters), numel, count, 4);
    if (rc) return rc;
    if ((uintptr_t)grad_scale % 4) return fail(ET_ERR_INVALID_ARGUMENT, "et_adamw8: grad_scale is not aligned");
    if (rounding != 0 && rounding != 1) return fail(ET_ERR_INVALID_ARGUMENT, "et_adamw8: rounding must be 0 or 1");
    hipStream_t s = (hipStream_t)stream;
    AdamW8Args args = {};
    static_assert(sizeof(AdamW8Args) <= 4096 && sizeof(AdamWArgs) <= 4096 && sizeof(NormArgs) <= 4096,
                  "kernel arguments");
    args.a = scalars;
    args.grad_scale = grad_scale;
    args.seed = seed;
    return each_launch<kTensors8>(
        numel, count, kChunk, args.spans,
        [&](int slot, int64_t i, int64_t from, uint32_t element) {
            args.param[slot] = at(params[i], from, pa);
            args.grad[slot] = at(grads[i], from, ga);
            args.m8[slot] = m8[i] + from;
            args.m_scale[slot] = m_scale[i] + from / ET_ADAMW8_BLOCK;
            args.u8[slot] = u8[i] + from;
            args.u_scale[slot] = u_scale[i] + from / ET_ADAMW8_BLOCK;
            args.master[slot] = masters ? masters[i] + from : nullptr;
            args.origin[slot] = element;
        },
        [&](unsigned blocks) {
            if (rounding) launch_adamw8<true>(param_dtype, grad_dtype, dim3(blocks), args, s);
            else launch_adamw8<false>(param_dtype, grad_dtype, dim3(blocks), args, s);
            return check_launch("adamw8_kernel");
        });
}
