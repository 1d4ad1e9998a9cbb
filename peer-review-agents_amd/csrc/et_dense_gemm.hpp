// et_dense_gemm.hpp -- the tile loop of the dense products (the gated projection
// and its gradients, Newton-Schulz):
//
//   C[i, j] = sum_k A(i, k) * B(j, k)      bf16 or f16 operands, binary32 sums
//
// over the tiles of one or many matrices, with an epilogue on the accumulators.
// Either operand lies with k along its rows (element (i, k) at i * ld + k) or
// down its columns (at k * ld + i); the second is read through gfx950's
// transposing LDS reads, so no operand is ever transposed in memory.
//
// Tiling.  A block of 2 x 2 waves owns a tile of 32 MI x 32 NJ; a wave owns
// MI x NJ tiles of v_mfma_f32_16x16x32.  k advances in chunks of 64 through two
// LDS stages filled by direct-to-LDS buffer loads.  The shapes (TileKind): big,
// 256 x 256, one block per CU, 16 fragment reads for 64 MFMAs, so LDS is read for
// half of the MFMAs' time; small, 128 x 128, two blocks per CU, LDS reads as long as
// the MFMAs, but four times as many tiles; mid, 192 x 128, between them (for A along its
// rows); thin, 64 x 128 or 64 x 64, for calls that have few tiles all the same (dense_kind).
// A wave holds a whole chunk's fragments in registers, so a stage is free again
// as soon as every wave has read it and two chunks stream in while one is
// multiplied; loads and fragment reads are placed between MFMAs in a pinned
// order.  The grid is persistent and a block's tiles form one stream of chunks:
// a tile's last two chunks load the next tile's first two.  (Four stages, one block
// per CU, change little: 128 x 128 at K = 4096 45 to 42 us, at K = 1024 13.3 to 14.5: a
// chunk of a small tile is its two barriers and LDS reads, not its way from memory.)
//
// LDS layout.  k along rows: 128 bytes (64 k) per row, the 16-byte segment s of
// row R at slot s ^ (R & 7) ^ (R >> 3 & 1).  k down columns: 64 rows (k) of 64 MI
// bytes, segment s of row r at slot s ^ 4 (r & 3) ^ 2 (r >> 3 & 1) (MI = 2, two rows to 256
// bytes: s ^ 4 (r >> 1 & 1) ^ 2 (r >> 3 & 1)).  Either way the fragment reads spread over
// all banks.
//
// A policy P has: a DenseTile's MI, NJ and kBlocks (per CU); kACol, kBCol, kF16; kMid, whether it has mid tiles; kScratch, the
// bytes of LDS that its epilogue has for a wave; Args, Tile (with a GemmTile first), tiles(), tile(), b_row() and epilogue().
#pragma once

#include <type_traits>

#include "et_gemm_common.hpp"

namespace et {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int kDenseThreads = 256;

enum TileKind { kTileThin = 2, kTileSmall = 4, kTileMid = 6, kTileBig = 8 };

// THIN: thin tiles are 64 x 32 THIN.
template <int KIND, int THIN>
struct DenseTile {
    static constexpr int MI = KIND, NJ = KIND == kTileThin ? THIN : KIND == kTileMid ? 4 : KIND;
    static constexpr int kBlocks = KIND == kTileBig ? 1 : 2;
};

// Operands of a tile, all wave-uniform.  a and b point at the tile's first row
// and first k (k along rows) or first k and first column (k down columns).
struct GemmTile {
    const unsigned char* a;
    const unsigned char* b;
    int a_rows, b_rows;       // rows (columns) of the tile that there are
    int lda, ldb;             // in elements
    int k;                    // length of the sum
};

// One direct-to-LDS load: this lane's 16 bytes at voff + soff of the buffer land
// at LDS address lds + 16 * lane.  In inline assembly, since the compiler would
// otherwise wait for every load in flight before each LDS read; the s_nop covers
// the wait state after M0 is written.  Masked lanes carry kOOR.
__device__ __forceinline__ void dense_dma(__amdgpu_buffer_rsrc_t res, uint32_t voff, uint32_t soff, uint32_t lds)
{
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(res), "s"(soff), "{m0}"(lds)
                 : "memory");
}

// ds_read_b64_tr_b16: within each 16-lane group, if lane j points at 4
// consecutive 16-bit elements M[j][0..3], lane i receives M[4 m + i / 4][i % 4].
typedef short dense_s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) dense_s16x4_t dense_lds_s16x4_t;

__device__ __forceinline__ uint2 dense_read_tr(const unsigned char* p)
{
    const dense_s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (dense_lds_s16x4_t*)(__attribute__((address_space(3))) unsigned char*)p);
    return __builtin_bit_cast(uint2, v);
}

// At most N of this wave's vector-memory operations in flight, then all waves meet.
template <int N>
__device__ __forceinline__ void dense_wait_barrier()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi)
{
    return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// Two 16 x 16 accumulator tiles side by side (output columns col0 .. col0 + 31 of
// one row): after the swap of 16-lane rows lane l holds columns 16 (rho & 1) +
// 8 (rho >> 1) + 0..7 and stores them at once (ncols is a multiple of 8).
template <bool F16>
__device__ __forceinline__ void store_pair(const float (&v)[8], __amdgpu_buffer_rsrc_t res, bool row_ok,
                                           uint32_t row_base, int col0, int ncols, int rho)
{
    const auto lo = __builtin_amdgcn_permlane16_swap(pack16x2<F16>(v[0], v[1]), pack16x2<F16>(v[4], v[5]), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(pack16x2<F16>(v[2], v[3]), pack16x2<F16>(v[6], v[7]), false, false);
    const u32x4_t out = {lo[0], hi[0], lo[1], hi[1]};
    const int col = col0 + 16 * (rho & 1) + 8 * (rho >> 1);
    const uint32_t off = (row_ok && col < ncols) ? (row_base + (uint32_t)col) * 2u : kOOR;
    __builtin_amdgcn_raw_buffer_store_b128(out, res, off, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t dense_rsrc(const void* p, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, kBufDword3);
}

// Tile q of a grid of nm x nn: groups of gm rows of tiles, so that the blocks that
// run together share operand tiles through an XCD's L2.
struct TileAt {
    int m, n;
};
__device__ __forceinline__ TileAt tile_at(int q, int nm, int nn, int gm)
{
    const int grp = q / (gm * nn);
    const int g = min(gm, nm - grp * gm);
    const int idx = q - grp * gm * nn;
    return {grp * gm + idx % g, idx / g};
}

template <class P>
constexpr int kDenseLds = 2 * (P::MI + P::NJ) * 4096 + 4 * P::kScratch;

// Block `block` of `blocks` (a multiple of 8) goes through its tiles.
template <class P>
__device__ __forceinline__ void dense_tiles(const typename P::Args& g, unsigned char* smem, int block, int blocks)
{
    constexpr int MI = P::MI, NJ = P::NJ;
    constexpr int kA = MI * 4096, kB = NJ * 4096, kStage = kA + kB;    // a chunk's bytes
    constexpr int NM = MI * NJ, NL = MI + NJ;                          // MFMAs a k-step, loads a wave and chunk
    constexpr int RPK = MI + NJ;                                       // fragments a k-step
    constexpr int Q1 = NM / 2;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int r16 = lane & 15, rho = lane >> 4;
    const int wm = wave >> 1, wn = wave & 1;
    const int Q = P::tiles(g), per = (Q + 7) / 8;
    const int nloc = blocks / 8, xcd = block & 7;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t*)smem;
    const int seg0 = (lane & 7) ^ (lane >> 3);

    typename P::Tile cur = {}, nxt = {};
    const auto setup = [&](int l, typename P::Tile& t) -> bool {
        const int q = xcd * per + l;
        if (l >= per || q >= Q) return false;
        P::tile(g, q, t);
        return true;
    };
    // A chunk of an operand, as its loads need it.  A load fills 8 rows (k along
    // rows) or 16 / MI of them (k down columns); which ones is uniform and added to
    // the lane's own offset.  What lies past the operand is read as 0 by the
    // descriptor's size: rows past the tile's (k along rows: rows are no longer
    // than ld) and k past the sum (k down columns; columns past the tile's may
    // hold anything, no output takes them).  k past the sum along rows is masked.
    struct RowChunk {
        __amdgpu_buffer_rsrc_t res;
        uint32_t at[2], soff;
    };
    struct ColChunk {
        __amdgpu_buffer_rsrc_t res;
        uint32_t at[4];
    };
    const auto row_chunk = [&](const unsigned char* p, int rows, int ld, int k, int c) -> RowChunk {
        RowChunk r;
        r.res = dense_rsrc(p, (rows - 1) * ld * 2 + ((k + 7) & ~7) * 2);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r.at[i] = c * 64 + (seg0 ^ i) * 8 < k ? (uint32_t)((lane >> 3) * 2 * ld + (seg0 ^ i) * 16) : kOOR;
        r.soff = (uint32_t)c * 128u;
        return r;
    };
    const auto col_chunk = [&](auto n, const unsigned char* p, int cols, int ld, int k, int c) -> ColChunk {
        constexpr int N = decltype(n)::value, LPR = 4 * N;                        // lanes a row
        static_assert(N == 8 || N == 4 || N == 2, "tile side");
        ColChunk r;
        r.res = dense_rsrc(p + (int64_t)c * 128 * ld, (min(64, k - c * 64) - 1) * ld * 2 + ((cols + 7) & ~7) * 2);
        const int in = lane / LPR;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            r.at[v] = (uint32_t)(in * 2 * ld + ((lane % LPR) ^ (N == 2 ? 4 * (in >> 1 & 1) ^ 2 * (v & 1)
                                                                : 4 * in ^ (N == 8 ? 8 * (v & 1) ^ 2 * (v >> 1) : 2 * (v & 1)))) * 16);
        return r;
    };
    const auto a_chunk = [&](const typename P::Tile& t, int c) {
        if constexpr (P::kACol) return col_chunk(std::integral_constant<int, MI>{}, t.a, t.a_rows, t.lda, t.k, c);
        else return row_chunk(t.a, t.a_rows, t.lda, t.k, c);
    };
    const auto b_chunk = [&](const typename P::Tile& t, int c) {
        if constexpr (P::kBCol) return col_chunk(std::integral_constant<int, NJ>{}, t.b, t.b_rows, t.ldb, t.k, c);
        else return row_chunk(t.b, t.b_rows, t.ldb, t.k, c);
    };
    // (row: the load's first row, uniform; past every operand where it is negative)
    const auto load_rows = [&](const RowChunk& r, int row, int ld, int i, uint32_t lds) {
        dense_dma(r.res, r.at[i & 1] + (row >= 0 ? (uint32_t)row * (uint32_t)(2 * ld) : kOOR - (r.at[i & 1] & kOOR)), r.soff, lds);
    };
    const auto load_cols = [&](auto n, const ColChunk& r, int ld, int i, uint32_t lds) {
        constexpr int N = decltype(n)::value, RPI = 16 / N;                       // rows a load
        const int v = N == 8 ? (i & 1) + 2 * (i >> 2 & 1) : N == 4 ? i >> 1 & 1 : i & 1;
        dense_dma(r.res, r.at[v] + (uint32_t)((wave * N + i) * RPI) * (uint32_t)(2 * ld), 0u, lds);
    };
    const auto dma_one = [&](const typename P::Tile& t, const auto& ra, const auto& rb, int c, int par, int q) {
        const uint32_t st = lds0 + (uint32_t)((c + par) & 1) * kStage;
        constexpr int kBoth = 2 * (MI < NJ ? MI : NJ);
        const bool of_b = q < kBoth ? (q & 1) : MI < NJ;
        const int i = q < kBoth ? q >> 1 : q - kBoth / 2;
        if (!of_b) {
            const uint32_t lds = st + (uint32_t)(wave * MI + i) * 1024u;
            if constexpr (P::kACol) load_cols(std::integral_constant<int, MI>{}, ra, t.lda, i, lds);
            else load_rows(ra, 8 * (wave * MI + i), t.lda, i, lds);
        } else {
            const uint32_t lds = st + kA + (uint32_t)(wave * NJ + i) * 1024u;
            if constexpr (P::kBCol) load_cols(std::integral_constant<int, NJ>{}, rb, t.ldb, i, lds);
            else load_rows(rb, P::b_row(g, t, 8 * (wave * NJ + i)), t.ldb, i, lds);
        }
    };

    f32x4_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{};

    // Fragments of a chunk: [k-step][tile], lane l the 8 k from 8 (l / 16) on of row
    // l % 16.
    u32x4_t fa[2][MI], fb[2][NJ];
    const int fkey = (lane & 7) ^ ((lane >> 3) & 1);
    const int frow = (r16 >> 3) * 1024 + (lane & 7) * 128;
    const int tkey = (2 * (r16 >> 2) ^ (rho & 1)) << 5, tkey2 = (2 * (r16 >> 3) ^ (rho & 1)) << 5;
    const int tin = ((r16 & 3) >> 1) * 16 + (r16 & 1) * 8;
    const auto read_rows = [&](const unsigned char* op, int tile, int ks) -> u32x4_t {
        return *reinterpret_cast<const u32x4_t*>(op + tile * 2048 + frow + (((4 * ks + rho) ^ fkey) << 4));
    };
    const auto read_cols = [&](auto n, const unsigned char* op, int tile, int ks) -> u32x4_t {
        constexpr int RBytes = 64 * decltype(n)::value;
        const unsigned char* const p = op + (32 * ks + 8 * rho + (r16 >> 2)) * RBytes + ((tile << 5) ^ (decltype(n)::value == 2 ? tkey2 : tkey)) + tin;
        const uint2 lo = dense_read_tr(p), hi = dense_read_tr(p + 4 * RBytes);
        return u32x4_t{lo.x, lo.y, hi.x, hi.y};
    };
    const auto read_r = [&](int st, int ks, int r) {
        const unsigned char* const op = smem + st * kStage;
        if (r < MI) {
            if constexpr (P::kACol) fa[ks][r] = read_cols(std::integral_constant<int, MI>{}, op, wm * MI + r, ks);
            else fa[ks][r] = read_rows(op, wm * MI + r, ks);
        } else {
            if constexpr (P::kBCol) fb[ks][r - MI] = read_cols(std::integral_constant<int, NJ>{}, op + kA, wn * NJ + r - MI, ks);
            else fb[ks][r - MI] = read_rows(op + kA, wn * NJ + r - MI, ks);
        }
    };
    // (B's fragment first: C's columns are then A's rows, and a lane holds 4
    // consecutive j of one row i)
    const auto mfma_one = [&](int ks, int m) {
        const int i = m / NJ, j = m % NJ;
        if constexpr (P::kF16) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, fb[ks][j]),
                                                               __builtin_bit_cast(f16x8_t, fa[ks][i]), acc[i][j], 0, 0, 0);
        } else {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fb[ks][j]),
                                                                __builtin_bit_cast(bf16x8_t, fa[ks][i]), acc[i][j], 0, 0, 0);
        }
    };
    const auto pin = [&]() { __builtin_amdgcn_sched_barrier(0); };

    int l = block >> 3;
    bool more = setup(l, cur);
    if (!more) return;
    int par = 0;              // stage of chunk c: (c + par) & 1
    int nk = (cur.k + 63) / 64;
    // A tile's first two chunks: waits for the first.
    const auto begin = [&](const typename P::Tile& t, int n, int par2) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (c < n) {
                const auto a0 = a_chunk(t, c);
                const auto b0 = b_chunk(t, c);
#pragma unroll
                for (int q = 0; q < NL; ++q) dma_one(t, a0, b0, c, par2, q);
            }
        }
        if (n > 1) dense_wait_barrier<NL>();
        else dense_wait_barrier<0>();
    };
    begin(cur, nk, par);
#pragma unroll
    for (int r = 0; r < RPK; ++r) read_r(0, 0, r);
    // Chunk c, its first k-step's fragments in registers: the second one's are read
    // under the first quarter of the MFMAs; then no wave reads this stage any more
    // and the stream's chunk two ahead is loaded into it under the next half; the
    // stream's next chunk is waited for and its first k-step read under the last
    // quarter (within the tile; the next tile's after the epilogue).
    // (t, c2, par2: the tile, chunk and parity that are loaded)
    const auto step = [&](int c, const typename P::Tile& t, int c2, int par2, bool more2, bool more1) {
        const int st = (c + par) & 1;
        const bool rd1 = c + 1 < nk;
#pragma unroll
        for (int m = 0; m < Q1; ++m) {
            mfma_one(0, m);
            pin();
#pragma unroll
            for (int r = m * RPK / Q1; r < (m + 1) * RPK / Q1; ++r) read_r(st, 1, r);
            pin();
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0): the builtin, so that the compiler knows
        pin();
        asm volatile("s_barrier" ::: "memory");
        const auto ra = a_chunk(t, c2);
        const auto rb = b_chunk(t, c2);
        pin();
#pragma unroll
        for (int m = Q1; m < Q1 + NM; ++m) {
            mfma_one(m / NM, m % NM);
            pin();
            if (more2) {
#pragma unroll
                for (int q = (m - Q1) * NL / NM; q < (m - Q1 + 1) * NL / NM; ++q) dma_one(t, ra, rb, c2, par2, q);
            }
            pin();
        }
        if (more1) {
            if (more2) dense_wait_barrier<NL>();
            else dense_wait_barrier<0>();
        }
#pragma unroll
        for (int m = Q1 + NM; m < 2 * NM; ++m) {
            mfma_one(1, m % NM);
            pin();
            if (rd1) {
#pragma unroll
                for (int r = (m - Q1 - NM) * RPK / (NM - Q1); r < (m - Q1 - NM + 1) * RPK / (NM - Q1); ++r)
                    read_r(st ^ 1, 0, r);
            }
            pin();
        }
    };

    for (;;) {
        l += nloc;
        more = setup(l, nxt);
        const int nk1 = more ? (nxt.k + 63) / 64 : 0;
        // (a tile of one chunk, or one before it, is not prefetched)
        const bool stream = more && nk >= 2 && nk1 >= 2;
        const int nmain = nk - 2;
        for (int c = 0; c < nmain; ++c) step(c, cur, c + 2, par, true, true);
        for (int c = max(nmain, 0); c < nk; ++c) step(c, nxt, c + 2 - nk, par + nk, stream, c + 1 < nk || stream);
        // (the accumulators stay in the accumulation registers up to here)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) asm volatile("" : "+a"(acc[i][j]));
        P::epilogue(g, cur, acc, wm, wn, r16, rho, smem + 2 * kStage + wave * P::kScratch);
        if (!more) break;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                acc[i][j] = f32x4_t{};
                // (opaque: with constants here the allocator renames the accumulators
                // in the loop, some 600 moves a chunk)
                asm volatile("" : "+a"(acc[i][j]));
            }
        if (!stream) {
            // (every wave has read its last fragments: they were consumed above)
            dense_wait_barrier<0>();
            begin(nxt, nk1, par + nk);
        }
#pragma unroll
        for (int r = 0; r < RPK; ++r) read_r((par + nk) & 1, 0, r);
        par = (par + nk) & 1;
        cur = nxt;
        nk = nk1;
    }
}

template <class P>
__global__ __launch_bounds__(kDenseThreads, P::kBlocks) void dense_gemm_kernel(typename P::Args g)
{
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kDenseLds<P>];
    dense_tiles<P>(g, smem, (int)blockIdx.x, (int)gridDim.x);
}

// Two calls' tiles in one launch: the first `blocks` blocks have the first's.
template <class P, class Q>
__global__ __launch_bounds__(kDenseThreads, P::kBlocks) void dense_pair_kernel(typename P::Args p, typename Q::Args q, int blocks)
{
    static_assert(P::kBlocks == Q::kBlocks, "one shape");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kDenseLds<P> > kDenseLds<Q> ? kDenseLds<P> : kDenseLds<Q>];
    if ((int)blockIdx.x < blocks) dense_tiles<P>(p, smem, (int)blockIdx.x, blocks);
    else dense_tiles<Q>(q, smem, (int)blockIdx.x - blocks, (int)gridDim.x - blocks);
}

// Blocks of a launch: a multiple of 8 (the XCDs take them in turn), no more than
// the device holds at once, no more than there are tiles.
inline unsigned dense_grid(int64_t tiles, int blocks_per_cu, int cus)
{
    const int64_t held = (int64_t)cus * blocks_per_cu / 8 * 8;
    return (unsigned)std::max<int64_t>(8, std::min<int64_t>(held, (tiles + 7) / 8 * 8));
}

// The tile's shape for a call of so many tiles of each kind (mid 0: a product without
// them), by what their rounds take.  In 1/100 of a chunk of two small tiles a CU (1.0 us):
// a big one 134, two mid ones 122 and one 74, a small one 60, thin ones 71 and 48 (64 x
// 128) or 60 and 40 (64 x 64).  Measured at K = 2048 and 4096, SwiGLU forward: 192 small tiles
// 40 us, as 128 mid ones 49, as 352 thin ones 41; 96 small 38, 160 thin 30; 512 small 68, 352
// mid 79, 128 big 88, 1024 thin 91; 1056 small 79, 704 mid 69, 264 big 104.  Newton-Schulz,
// five steps: 512 x 512 138 us small, 100 thin; 8 of them 153 and 126; 24 of 512 x 1024
// 305 and 403.  The chunks' costs are the SwiGLU forward's, for the other products too; what lies
// beside the chunks is left out, which is much where a tile has few of them: the polynomial
// of 64 matrices of 1024 x 1024 takes 129 us, its chunks 64 of them.
struct DenseChoice {
    int kind;
    int64_t cost;
};
inline DenseChoice dense_choice(int64_t big, int64_t mid, int64_t small, int64_t thin, bool wide, int cus)
{
    const auto rounds = [cus](int64_t tiles, int alone, int pair) {
        const int64_t full = tiles / (2 * cus), rest = tiles - full * 2 * cus;
        return full * pair + (rest == 0 ? 0 : rest <= cus ? alone : pair);
    };
    DenseChoice best = {kTileBig, (big + cus - 1) / cus * 134};
    const auto other = [&best](int kind, int64_t cost) {
        if (cost < best.cost) best = {kind, cost};
    };
    if (mid) other(kTileMid, rounds(mid, 74, 122));
    other(kTileSmall, rounds(small, 60, 100));
    other(kTileThin, wide ? rounds(thin, 48, 71) : rounds(thin, 40, 60));
    return best;
}

inline int dense_kind(int64_t big, int64_t mid, int64_t small, int64_t thin, bool wide, int cus)
{
    return dense_choice(big, mid, small, thin, wide, cus).kind;
}

// Launches POLICY<kind> on `tiles` tiles.
template <template <int> class POLICY, class ARGS>
int launch_dense(const ARGS& g, int kind, int64_t tiles, int cus, hipStream_t s, const char* what)
{
    const dim3 block(kDenseThreads), grid(dense_grid(tiles, kind == kTileBig ? 1 : 2, cus));
    if (kind == kTileBig) dense_gemm_kernel<POLICY<kTileBig>><<<grid, block, 0, s>>>(g);
    else if (kind == kTileMid) {
        if constexpr (POLICY<kTileMid>::kMid) dense_gemm_kernel<POLICY<kTileMid>><<<grid, block, 0, s>>>(g);
    } else if (kind == kTileSmall) dense_gemm_kernel<POLICY<kTileSmall>><<<grid, block, 0, s>>>(g);
    else dense_gemm_kernel<POLICY<kTileThin>><<<grid, block, 0, s>>>(g);
    return check_launch(what);
}

// Compute units of the current device, looked up once per device.
inline int dense_cus()
{
    static int cache[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0) dev = 0;
    int* slot = dev < 64 ? &cache[dev] : nullptr;
    if (slot && *slot > 0) return *slot;
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    if (slot) *slot = n;
    return n;
}

}  // namespace
}  // namespace et
