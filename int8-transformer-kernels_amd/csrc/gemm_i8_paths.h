// gemm_i8_paths.h — the int8 GEMM's smaller tilings and their plans: 128 x 128 tiles, the
// weight-streaming kernel for few rows, the operand loads of the skinny one.
//
// Internal header of libint8k, shared by the MLP (mlp.hip) and the linear layer (linear.hip);
// both put their own epilogues behind these loops.
#pragma once

#include <algorithm>

#include "gemm_i8.h"

namespace int8k {
namespace {

using namespace gemm;

// ------------------------------------------------------------ mid-size grids
// gemm_i8_mid_kernel<EPI>: 128 x 128 output tiles for GEMMs whose 256 x 256
// grid leaves CUs idle (T = 4096 at d_model 1024: GEMM2 has 16 x 4 big tiles
// for 256 CUs).  Four waves in a 2 x 2 grid each own 64 x 64 (2 x 2 MFMA
// tiles of 32 x 32 x 32); A and Bt go global -> VGPR -> LDS in the big
// kernel's padded layout, double-buffered, the next K-step's loads in flight
// during the current one.  75 KiB of LDS: two blocks per CU, whose waves hide
// each other's waits.  Half the MFMA work per fragment read of the big tile,
// so it runs only where the big grid is too small.  Same epilogue code and
// bytes as gemm_i8_kernel, with one absmax partial per row and 128 columns.
constexpr int kMidB = 128, kMidW = 64, kMidT = kMidW / 32;
constexpr int kMidAStage = kMidB * LDS_STRIDE;
constexpr int kMidChunks = kMidB * kChunksPerRow / kThreads;
// BKN: B stored [K][N], staged as 128 rows of k and read with transposing LDS reads
// (rows 160 bytes apart: the 8 rows of a read start 32 bytes apart in the banks)
template <bool BKN>
struct MidLds {
    static constexpr int kBStride = BKN ? kMidB + 32 : LDS_STRIDE;
    static constexpr int kStage = kMidAStage + 128 * kBStride;
    static constexpr int kScales = 2 * kStage;  // the epilogue's scales lie past the stages
    static constexpr int kBytes = kScales + 3 * kMidB * 4;
};
static_assert(kMidChunks == 4 && 2 * MidLds<true>::kBytes <= 160 * 1024, "two blocks per CU");

// The K range [kb, ke) of a tile (kb a multiple of 16).  SWAP: tiles transposed, as mfma_ab's.
template <bool EDGE, bool BKN, bool SWAP = false>
__device__ __forceinline__ void mid_mainloop(v16i (&acc)[kMidT][kMidT],
                                             const int8_t* __restrict__ A,
                                             const int8_t* __restrict__ Bt, int M, int N, int K,
                                             int kb, int ke, int m0, int n0, char* lds) {
    constexpr int kMidStage = MidLds<BKN>::kStage, kBStride = MidLds<BKN>::kBStride;
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int i = 0; i < kMidT; ++i)
#pragma unroll
        for (int j = 0; j < kMidT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int nk = (ke - kb + BK - 1) / BK;
    const int a_off = (wm * kMidW + (lane & 31)) * LDS_STRIDE + (lane >> 5) * 16;
    const int g16 = lane >> 4, s16 = lane & 15;
    const int b_off =
        kMidAStage + (BKN ? (16 * (g16 >> 1) + (s16 >> 1)) * kBStride + wn * kMidW + 16 * (g16 & 1) +
                                8 * (s16 & 1)
                          : (wn * kMidW + (lane & 31)) * kBStride + (lane >> 5) * 16);
    int4 fa[kMidChunks], fb[kMidChunks];
    // chunk c = t + 256 i of a 128 x 128-byte operand tile: row c / 8, bytes (c % 8) * 16;
    // rows past the matrix and K past the end load clamped addresses, zeroed on EDGE
    auto load = [&](int ks) {
        const int k0 = kb + ks;
#pragma unroll
        for (int i = 0; i < kMidChunks; ++i) {
            const int c = threadIdx.x + i * kThreads;
            const int row = c / kChunksPerRow, kc = (c % kChunksPerRow) * 16;
            const int gk = min(k0 + kc, K - 16);
            fa[i] = *reinterpret_cast<const int4*>(A + (size_t)min(m0 + row, M - 1) * K + gk);
            if constexpr (BKN)
                fb[i] = *reinterpret_cast<const int4*>(Bt + (size_t)min(k0 + row, K - 1) * N +
                                                       min(n0 + kc, N - 16));
            else
                fb[i] = *reinterpret_cast<const int4*>(Bt + (size_t)min(n0 + row, N - 1) * K + gk);
        }
    };
    auto store = [&](char* stage, int ks) {
        const int k0 = kb + ks;
#pragma unroll
        for (int i = 0; i < kMidChunks; ++i) {
            const int c = threadIdx.x + i * kThreads;
            const int row = c / kChunksPerRow, kc = (c % kChunksPerRow) * 16;
            int4 va = fa[i], vb = fb[i];
            if constexpr (EDGE) {
                const bool kok = k0 + kc < ke;
                const bool bok = BKN ? k0 + row < ke && n0 + kc < N : kok && n0 + row < N;
                if (!(kok && m0 + row < M)) va = make_int4(0, 0, 0, 0);
                if (!bok) vb = make_int4(0, 0, 0, 0);
            }
            *reinterpret_cast<int4*>(stage + row * LDS_STRIDE + kc) = va;
            *reinterpret_cast<int4*>(stage + kMidAStage + row * kBStride + kc) = vb;
        }
    };
    // fragments of k-slice s of a stage: rows (l % 32) of the wave's two 32-row
    // blocks of A and of Bt, 16-byte half (l / 32)
    auto read = [&](v4i (&a)[kMidT], v4i (&b)[kMidT], const char* stage, int s) {
#pragma unroll
        for (int i = 0; i < kMidT; ++i)
            a[i] = *reinterpret_cast<const v4i*>(stage + a_off + i * 32 * LDS_STRIDE + s * 32);
#pragma unroll
        for (int j = 0; j < kMidT; ++j) {
            if constexpr (BKN) {
                typedef int v2i __attribute__((ext_vector_type(2)));
                typedef __attribute__((address_space(3))) v2i lds_v2i;
                const char* p = stage + b_off + s * 32 * kBStride + j * 32;
                const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(p));
                const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(p + 8 * kBStride));
                b[j] = v4i{lo.x, lo.y, hi.x, hi.y};
            } else {
                b[j] = *reinterpret_cast<const v4i*>(stage + b_off + j * 32 * kBStride + s * 32);
            }
        }
    };
    auto mma = [&](const v4i (&a)[kMidT], const v4i (&b)[kMidT]) {
#pragma unroll
        for (int i = 0; i < kMidT; ++i)
#pragma unroll
            for (int j = 0; j < kMidT; ++j)
                acc[i][j] = mfma_ab<SWAP>(a[i], b[j], acc[i][j]);
    };
    load(0);
    store(lds, 0);
    if (nk > 1) load(BK);
    __syncthreads();
    v4i a[2][kMidT], b[2][kMidT];
    read(a[0], b[0], lds, 0);
    // Step kt reads buffer kt & 1 and writes buffer (kt + 1) & 1, whose last
    // reads (step kt - 1) finished before that step's barrier.  The fragments
    // of slice 3 are in registers before the barrier, so its MFMAs run after
    // it, while the reads of the next stage's slice 0 are in flight.
    for (int kt = 0; kt < nk; ++kt) {
        const char* cur = lds + (kt & 1) * kMidStage;
        char* nxt = lds + ((kt + 1) & 1) * kMidStage;
        read(a[1], b[1], cur, 1);
        mma(a[0], b[0]);
        read(a[0], b[0], cur, 2);
        mma(a[1], b[1]);
        read(a[1], b[1], cur, 3);
        mma(a[0], b[0]);
        if (kt + 1 < nk) store(nxt, (kt + 1) * BK);
        if (kt + 2 < nk) load((kt + 2) * BK);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        if (kt + 1 < nk) read(a[0], b[0], nxt, 0);
        mma(a[1], b[1]);
    }
}

// ---------------------------------------------------------------- few tokens
// gemm_i8_stream_kernel<MT, BKN>: a GEMM of up to 32 MT rows per row block, whose time
// is the read of the weights (4096 -> 16384 as stored, 32 rows: 17.5 us per GEMM of 64
// MiB, 3.8 TB/s, of which ~5 us are the first loads, the merge and the stores).  A wave
// owns 128 columns over its own range of K and streams 128 x 128-byte weight tiles
// through its own piece of LDS: 16 loads of 16 bytes per lane in flight, each
// covering whole 128-byte runs (8 weight rows per instruction) for both layouts, the
// next tile's loads issued before the current one's MFMAs, no block barrier in the
// loop.  Fragments come from LDS as in the tiled kernels: 16-byte reads of [N][K] rows, or transposing reads of
// [K][N] rows (BKN), so weights as stored need no transpose.  A's fragments are
// read from global memory (L2) into registers one step ahead.  The waves of a
// block meet in LDS, and the block writes exact int32 partials P[split][M][N],
// which rows_epilogue_kernel sums.
// MFMA operands are swapped, so a lane holds one row and 4 adjacent columns.
// K past the end: A is zero there.  N past the end: those columns are not stored.
constexpr int kStN = 128, kStK = 128;
constexpr int kStMaxWaves = 8;
template <bool BKN>
struct StreamTile {
    // bytes per LDS row: 16-byte fragment reads of consecutive [N][K] rows spread
    // over the banks at 144; the 8 rows of a transposing read start 32 bytes apart
    // (modulo the 256 of all banks) at 160
    static constexpr int kStride = BKN ? kStN + 32 : kStK + 16;
    static constexpr int kBytes = 128 * kStride;
};
constexpr int kStRedStride = kStN + 4;  // words per row of a wave's partial tile
static_assert(32 * kStRedStride * 4 <= StreamTile<false>::kBytes, "a partial tile fits the stage");

template <int MT, bool BKN>
__global__ __launch_bounds__(64 * kStMaxWaves, 1) void gemm_i8_stream_kernel(
    const int8_t* __restrict__ A, const int8_t* __restrict__ B, int32_t* __restrict__ P, int M,
    int N, int K, int steps_per_wave) {
    extern __shared__ __align__(16) char lds[];
    using ST = StreamTile<BKN>;
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nw = blockDim.x >> 6;
    const int n0 = blockIdx.x * kStN, m0 = blockIdx.z * 32 * MT;
    const int kw = steps_per_wave * kStK;
    const long long kb = ((long long)blockIdx.y * nw + wave) * kw;
    const int k_begin = (int)min(kb, (long long)K);
    const int k_end = min(K - k_begin, kw) + k_begin;
    const int nsteps = (k_end - k_begin + kStK - 1) / kStK;
    char* stage = lds + wave * ST::kBytes;

    v16i acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    // weight tile: load i covers tile rows 8 i + lane / 8 (columns n of [N][K], or k of
    // [K][N]), 16 bytes at 16 (lane % 8)
    const uint32_t ldw = BKN ? (uint32_t)N : (uint32_t)K;
    const uint32_t w_voff = (uint32_t)(lane >> 3) * ldw + (lane & 7) * 16;
    v4u w[16];
    auto load_w = [&](int k0) {
        // the resource starts at the tile and ends with the matrix: rows past it read zero
        const size_t off = BKN ? (size_t)k0 * N + n0 : (size_t)n0 * K + k0;
        const size_t left = (size_t)N * K - off;
        const __amdgpu_buffer_rsrc_t r = make_buffer(B + off, (uint32_t)min(left, (size_t)0xffffffffu));
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w[i] = __builtin_amdgcn_raw_buffer_load_b128(r, w_voff, (uint32_t)(8 * i) * ldw, 0);
    };
    // A fragments of the step: rows 32 i + lane % 32, 16 bytes at k + 32 s + 16 (lane / 32)
    const __amdgpu_buffer_rsrc_t ra =
        make_buffer(A + (size_t)m0 * K, (uint32_t)min((size_t)(M - m0) * K, (size_t)0xffffffffu));
    v4i a[MT][4];
    auto load_a = [&](int k0, int s) {
        const int k = k0 + 32 * s + 16 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t voff = (uint32_t)(32 * i + (lane & 31)) * (uint32_t)K + (uint32_t)k;
            const v4u x = __builtin_amdgcn_raw_buffer_load_b128(ra, k < K ? voff : 0xffffffffu, 0, 0);
            a[i][s] = __builtin_bit_cast(v4i, x);
        }
    };
    const int wr_off = (lane >> 3) * ST::kStride + (lane & 7) * 16;
    const int g16 = lane >> 4, s16 = lane & 15;
    const int rd_off = BKN ? (16 * (g16 >> 1) + (s16 >> 1)) * ST::kStride + 16 * (g16 & 1) + 8 * (s16 & 1)
                           : (lane & 31) * ST::kStride + (lane >> 5) * 16;
    auto read_b = [&](int j, int s) -> v4i {
        if constexpr (BKN) {
            typedef int v2i __attribute__((ext_vector_type(2)));
            typedef __attribute__((address_space(3))) v2i lds_v2i;
            const char* p = stage + rd_off + s * 32 * ST::kStride + j * 32;
            const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(p));
            const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(p + 8 * ST::kStride));
            return v4i{lo.x, lo.y, hi.x, hi.y};
        } else {
            return *reinterpret_cast<const v4i*>(stage + rd_off + j * 32 * ST::kStride + s * 32);
        }
    };
    if (nsteps > 0) {
        load_w(k_begin);
#pragma unroll
        for (int s = 0; s < 4; ++s) load_a(k_begin, s);
    }
    for (int st = 0; st < nsteps; ++st) {
        const int k_next = k_begin + (st + 1) * kStK;
        const bool more = st + 1 < nsteps;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            *reinterpret_cast<v4u*>(stage + wr_off + 8 * i * ST::kStride) = w[i];
        // lanes read what other lanes of the wave wrote: keep the compiler from moving LDS
        // accesses across (the wave's LDS operations complete in order)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (more) load_w(k_next);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            v4i b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = read_b(j, s);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[j], a[i][s], acc[i][j], 0, 0, 0);
            if (more) load_a(k_next, s);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // 32 rows at a time: each wave leaves its 32 x 128 partial tile in its own stage, the
    // block sums the waves' tiles and stores them
    int32_t* Pp = P + (size_t)blockIdx.y * M * N;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (m0 + 32 * i >= M) break;
        int* mine = reinterpret_cast<int*>(stage) + (lane & 31) * kStRedStride + 4 * (lane >> 5);
        if (i > 0) __syncthreads();  // the previous rows have been read
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<v4i*>(mine + 32 * j + 8 * q) =
                    v4i{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __syncthreads();
        for (int e = threadIdx.x; e < 32 * (kStN / 4); e += blockDim.x) {
            const int row = e / (kStN / 4), c4 = e % (kStN / 4);
            v4i sum = {0, 0, 0, 0};
            for (int v = 0; v < nw; ++v)
                sum += *reinterpret_cast<const v4i*>(lds + v * ST::kBytes +
                                                     (row * kStRedStride + 4 * c4) * 4);
            const int m = m0 + 32 * i + row, n = n0 + 4 * c4;
            if (m < M && n < N) *reinterpret_cast<v4i*>(Pp + (size_t)m * N + n) = sum;
        }
    }
}

// Split of a few-token GEMM over waves and blocks: `waves` waves of `steps` 128-deep
// K steps per block, `splits` blocks per column tile.
struct StreamPlan {
    int mt, waves, steps, splits, tiles_n, tiles_m;
};
constexpr int kRowsEpiMaxN = 32768;  // 1024 threads x 8 groups of 4 columns
constexpr int kStWaves = 2048;       // 8 waves on each of 256 CUs

inline StreamPlan stream_plan(int M, int N, int K) {
    StreamPlan pl{};
    pl.mt = M > 32 ? 2 : 1;
    pl.tiles_n = (N + kStN - 1) / kStN;
    pl.tiles_m = (M + 32 * pl.mt - 1) / (32 * pl.mt);
    const int ksteps = (K + kStK - 1) / kStK;
    const long long units = (long long)pl.tiles_n * pl.tiles_m * ksteps;
    pl.steps = (int)std::max<long long>(1, units / kStWaves);
    const int chain = (ksteps + pl.steps - 1) / pl.steps;  // waves per column tile
    pl.waves = std::min(kStMaxWaves, chain);
    pl.splits = (chain + pl.waves - 1) / pl.waves;
    return pl;
}

// Split of a 128 x 128-tile GEMM over K (splits == 1: whole K, fp16 epilogue).
struct MidPlan {
    int tiles_m, tiles_n, splits, k_per_split;
};

// The split with the smallest time in units of 0.01 us: a K step of a block takes
// about 0.6 us alone on its CU and 0.9 us beside a second block; the rows reach the
// requantization as fp16 (written and read once) or as `splits` int32 partials, at
// about 4.5 TB/s.  Measured, us per MLP with at most 512 / 256 blocks: T = 1024, 1024
// -> 4096 48 / 34 (33 MB of partials for 4 K steps saved), T = 512, 2048 -> 8192
// 53 / 45, T = 333, 4096 -> 16384 99 / 112 (GEMM2: 26 or 64 K steps per block).
inline MidPlan mid_plan(int M, int N, int K) {
    MidPlan pl{};
    pl.tiles_m = (M + kMidB - 1) / kMidB;
    pl.tiles_n = (N + kMidB - 1) / kMidB;
    const long long tiles = (long long)pl.tiles_m * pl.tiles_n;
    const long long ksteps = (K + BK - 1) / BK;
    long long best = -1, steps = ksteps;
    for (long long sp = 1; sp <= std::min(16LL, ksteps); ++sp) {
        const long long st = ceil_div(ksteps, sp), n = ceil_div(ksteps, st);
        const long long blocks = tiles * n;
        const long long gemm = blocks <= 256 ? 60 * st : 90 * st * ceil_div(blocks, 512);
        const long long rows = (n > 1 ? 8 * n : 4) * (long long)M * N / 45000;
        if (best < 0 || gemm + rows < best) best = gemm + rows, steps = st;
    }
    pl.k_per_split = (int)(steps * BK);
    pl.splits = (int)ceil_div(ksteps, steps);
    return pl;
}

__device__ __forceinline__ void skinny_load(v4i (&b)[4], v4i (&a)[4], const int8_t* arow,
                                            const int8_t* brow, int k) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        b[u] = *reinterpret_cast<const v4i*>(brow + k + 32 * u);
        a[u] = *reinterpret_cast<const v4i*>(arow + k + 32 * u);
    }
}

__device__ __forceinline__ void skinny_mfma(v16i& acc, const v4i (&b)[4], const v4i (&a)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[u], b[u], acc, 0, 0, 0);
}

template <bool BKN>
int launch_gemm_stream(const int8_t* A, const int8_t* B, int M, int N, int K,
                       const StreamPlan& pl, int32_t* partial, hipStream_t stream) {
    const dim3 grid(pl.tiles_n, pl.splits, pl.tiles_m);
    const int lds = pl.waves * StreamTile<BKN>::kBytes;
    if (pl.mt == 1)
        gemm_i8_stream_kernel<1, BKN><<<grid, 64 * pl.waves, lds, stream>>>(A, B, partial, M, N, K,
                                                                          pl.steps);
    else
        gemm_i8_stream_kernel<2, BKN><<<grid, 64 * pl.waves, lds, stream>>>(A, B, partial, M, N, K,
                                                                          pl.steps);
    return check_launch("gemm_i8_stream_kernel");
}

}  // namespace
}  // namespace int8k
