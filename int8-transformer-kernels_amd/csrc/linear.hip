// linear.hip — INT8 matrix product with a scale per token and per output channel, gfx950.
//
//   y[t, n] = T( (f32(acc) * sx[t]) * sw[n] (+ b[n]) ),  acc = sum_k x[t, k] w[k, n], exact int32
//
// x int8 [T, K]; w int8 [K, N] as stored, or [N, K] packed; y fp16, bf16 or fp32, rounded once
// from the fp32 value.  The products run on the loops of the MLP's GEMMs (gemm_i8.h,
// gemm_i8_paths.h); the routes differ in how the result leaves:
//   skinny   32 x 32 tiles, K over the waves of a block (few tokens, packed weights)
//   stream   the weights streamed once over all CUs, exact int32 partials, then rows
//   small    64 x 64 tiles, four blocks per CU, or one of two wave groups that halve K
//   mid      128 x 128 tiles, two blocks per CU; K split into partials where CUs would idle
//   wide     256 x 192 tiles, packed weights
//   tiled    256 x 256 tiles
// The tiles are computed transposed (SWAP), so a lane holds 4 adjacent columns of one row: 32
// rows at a time go through the wave's own piece of LDS and leave as whole lines.
#include "gemm_i8_paths.h"
#include "rows.h"

namespace int8k {
namespace {

struct LinearArgs {
    const int8_t *x, *w;
    void* y;
    int32_t* part;  // [splits][M][N]
    const float *sx, *sw, *bias;
    int sx_stride, sw_stride;  // 0: one scale for all
    int M, N, K;
};

template <int DT>
constexpr int kOutBytes = DT == INT8K_DTYPE_F32 ? 4 : 2;

// The value of a sum; the same expression on every route.
__device__ __forceinline__ float linear_value(int acc, float sx, float sw, float b) {
    return static_cast<float>(acc) * sx * sw + b;
}

// 4 consecutive values to dst (8 or 16 bytes).
template <int DT>
__device__ __forceinline__ void store_four(void* dst, const float (&v)[4]) {
    if constexpr (DT == INT8K_DTYPE_F32)
        *static_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *static_cast<uint2*>(dst) = make_uint2(pack_pair<DT>(v[0], v[1]), pack_pair<DT>(v[2], v[3]));
}

// The row and column scales and the bias of a tile of B x B outputs, loaded before the main
// loop (clamped, unconditional) by threads t < B and parked in LDS behind it.
struct TileScales {
    float sx, sw, b;
};
template <int B>
__device__ __forceinline__ TileScales load_scales(const LinearArgs& p, int m0, int n0) {
    const int t = threadIdx.x & (B - 1);
    TileScales s;
    s.sx = p.sx[(size_t)min(m0 + t, p.M - 1) * p.sx_stride];
    s.sw = p.sw[(size_t)min(n0 + t, p.N - 1) * p.sw_stride];
    s.b = p.bias != nullptr ? p.bias[min(n0 + t, p.N - 1)] : 0.f;
    return s;
}

// The outputs of a wave's (32 TM_) x (32 TN_) sub-tile at (row0, col0) of the matrix, (rl, cl)
// of the tile.  stage: this wave's LDS, 32 rows of kEpiRow bytes; scales: [sx B][sw B][bias B].
template <int DT, int TN_>
constexpr int kEpiRow = TN_ * 32 * kOutBytes<DT> + 16;
template <int DT, int TM_, int TN_, int B>
__device__ __forceinline__ void epilogue_rows(const v16i (&acc)[TM_][TN_], const LinearArgs& p,
                                              int m0, int n0, int rl, int cl, char* stage,
                                              const float* scales) {
    constexpr int E = kOutBytes<DT>, kRow = kEpiRow<DT, TN_>;
    constexpr int kLanes = TN_ * 32 * E / 16;  // 16-byte pieces of a row
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const float* ssw = scales + B + cl + 4 * half;
    const float* sb = ssw + B;
#pragma unroll
    for (int i = 0; i < TM_; ++i) {
        const float sx = scales[rl + 32 * i + (lane & 31)];
        char* mine = stage + (lane & 31) * kRow + 4 * half * E;
#pragma unroll
        for (int j = 0; j < TN_; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 w4 = *reinterpret_cast<const float4*>(ssw + 32 * j + 8 * q);
                const float4 b4 = *reinterpret_cast<const float4*>(sb + 32 * j + 8 * q);
                const float v[4] = {linear_value(acc[i][j][4 * q], sx, w4.x, b4.x),
                                    linear_value(acc[i][j][4 * q + 1], sx, w4.y, b4.y),
                                    linear_value(acc[i][j][4 * q + 2], sx, w4.z, b4.z),
                                    linear_value(acc[i][j][4 * q + 3], sx, w4.w, b4.w)};
                store_four<DT>(mine + (32 * j + 8 * q) * E, v);
            }
        // lanes read what other lanes of the wave wrote (its LDS operations complete in order)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = lane; e < 32 * kLanes; e += 64) {
            const int r = e / kLanes, piece = e % kLanes;
            const int row = m0 + rl + 32 * i + r, col = n0 + cl + piece * (16 / E);
            const uint4 w = *reinterpret_cast<const uint4*>(stage + r * kRow + piece * 16);
            // N is a multiple of 16: a piece is wholly in or out
            if (row < p.M && col < p.N)
                *reinterpret_cast<uint4*>(static_cast<char*>(p.y) + ((size_t)row * p.N + col) * E) = w;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int B>
__device__ __forceinline__ void park_scales(const TileScales& s, float* scales) {
    if (B == kThreads || (int)threadIdx.x < B) {
        scales[threadIdx.x] = s.sx;
        scales[B + threadIdx.x] = s.sw;
        scales[2 * B + threadIdx.x] = s.b;
    }
    __syncthreads();  // every wave is done with the operand stages, too
}

// ------------------------------------------------------------------ 256 x 256 tiles
constexpr int kTiledLds = LDS_BYTES + 3 * BM * 4;

template <int DT, bool BKN>
__global__ __launch_bounds__(kThreads, 1) void linear_tiled_kernel(LinearArgs p, int tiles_m,
                                                                   int tiles_n) {
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const TileScales s = load_scales<BM>(p, m0, n0);
    v16i acc[TM][TN];
    const int ldb = BKN ? p.N : p.K;
    if (m0 + BM <= p.M && n0 + BN <= p.N && p.K % BK == 0)
        mainloop<false, true, BKN>(acc, p.x, p.w, p.M, p.N, p.K, p.K, ldb, m0, n0, lds);
    else
        mainloop<true, true, BKN>(acc, p.x, p.w, p.M, p.N, p.K, p.K, ldb, m0, n0, lds);
    float* scales = reinterpret_cast<float*>(lds + LDS_BYTES);
    park_scales<BM>(s, scales);
    const int wave = threadIdx.x >> 6;
    static_assert(4 * 32 * kEpiRow<INT8K_DTYPE_F32, TN> <= LDS_BYTES, "the waves' pieces fit");
    epilogue_rows<DT, TM, TN, BM>(acc, p, m0, n0, (wave >> 1) * WM, (wave & 1) * WN,
                                  lds + wave * 32 * kEpiRow<DT, TN>, scales);
}

// ------------------------------------------------------------------ 256 x 192 tiles
// For packed weights whose 256 x 256 tiles leave the last round of CUs part empty: waves of
// 128 x 96, on the schedule of the 256 x 256 loop (mainloop) with 12 MFMAs a slice.
constexpr int kWideN = 192, kWideWN = kWideN / 2, kWideTN = kWideWN / 32;
constexpr int kWideStage = A_STAGE + kWideN * LDS_STRIDE;
constexpr int kWideLds = 2 * kWideStage + 3 * BM * 4;

template <bool EDGE>
__device__ __forceinline__ void wide_mainloop(v16i (&acc)[TM][kWideTN], const LinearArgs& p, int m0,
                                              int n0, char* lds) {
    constexpr int TN_ = kWideTN, kA = kChunks, kB = kWideN * kChunksPerRow / kThreads;
    constexpr int kMfmas = TM * TN_, kReads = TM + TN_;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int a_off = ((wave >> 1) * WM + (lane & 31)) * LDS_STRIDE + (lane >> 5) * 16;
    const int b_off = A_STAGE + ((wave & 1) * kWideWN + (lane & 31)) * LDS_STRIDE + (lane >> 5) * 16;
    const OperandSrc srcA = operand_rowmajor(p.x, p.M, p.K, p.K, m0);
    const OperandSrc srcB = operand_rowmajor(p.w, p.N, p.K, p.K, n0);
    const int nk = (p.K + BK - 1) / BK;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN_; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    int4 f[kA + kB];  // chunks of A, then of B, of the stage after next
    auto load = [&](int k0, int c) { f[c] = c < kA ? load_operand(srcA, k0, c) : load_operand(srcB, k0, c - kA); };
    auto store = [&](char* stage, int k0, int c) {
        if (c < kA) store_chunk<EDGE>(f[c], stage, p.M, p.K, m0, k0, c);
        else store_chunk<EDGE>(f[c], stage + A_STAGE, p.N, p.K, n0, k0, c - kA);
    };
    v4i a[2][TM], b[2][TN_];
    // fragment r of a slice: the A ones, then the B ones
    auto read = [&](int to, const char* stage, int slice, int r) {
        if (r < TM) a[to][r] = read_frag(stage, a_off, r, slice);
        else b[to][r - TM] = read_frag(stage, b_off, r - TM, slice);
    };
    auto mfma = [&](int from, int g) {
        const int i = g / TN_, j = g % TN_;
        acc[i][j] = mfma_ab<true>(a[from][i], b[from][j], acc[i][j]);
    };
#pragma unroll
    for (int c = 0; c < kA + kB; ++c) load(0, c);
#pragma unroll
    for (int c = 0; c < kA + kB; ++c) store(lds, 0, c);
#pragma unroll
    for (int c = 0; c < kA + kB; ++c) load(BK, c);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kReads; ++r) read(0, lds, 0, r);
    for (int kt = 0; kt < nk; ++kt) {
        const char* cur = lds + (kt & 1) * kWideStage;
        char* nxt = lds + ((kt + 1) & 1) * kWideStage;
        // slices 0 and 1: the next slice's fragments between their MFMAs
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < kMfmas; ++g) {
                if (g < kReads) read((s + 1) & 1, cur, s + 1, g);
                mfma(s & 1, g);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // slice 2: slice 3's fragments, the next stage's chunks to LDS and their replacements
#pragma unroll
        for (int g = 0; g < kMfmas; ++g) {
            if (g < kReads) read(1, cur, 3, g);
#pragma unroll
            for (int c = g * (kA + kB) / kMfmas; c < (g + 1) * (kA + kB) / kMfmas; ++c) {
                store(nxt, (kt + 1) * BK, c);
                load((kt + 2) * BK, c);
            }
            mfma(0, g);
            __builtin_amdgcn_sched_barrier(0);
        }
        // slice 3: half of its MFMAs cover the writes, the others the next slice 0
#pragma unroll
        for (int g = 0; g < kMfmas / 2; ++g) {
            mfma(1, g);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
#pragma unroll
        for (int g = kMfmas / 2; g < kMfmas; ++g) {
            const int u = g - kMfmas / 2;
#pragma unroll
            for (int r = u * kReads / (kMfmas / 2); r < (u + 1) * kReads / (kMfmas / 2); ++r) read(0, nxt, 0, r);
            mfma(1, g);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads, 1) void linear_wide_kernel(LinearArgs p, int tiles_m, int tiles_n) {
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * kWideN;
    const TileScales s = load_scales<BM>(p, m0, n0);
    v16i acc[TM][kWideTN];
    if (m0 + BM <= p.M && n0 + kWideN <= p.N && p.K % BK == 0) wide_mainloop<false>(acc, p, m0, n0, lds);
    else wide_mainloop<true>(acc, p, m0, n0, lds);
    float* scales = reinterpret_cast<float*>(lds + 2 * kWideStage);
    park_scales<BM>(s, scales);
    const int wave = threadIdx.x >> 6;
    static_assert(4 * 32 * kEpiRow<INT8K_DTYPE_F32, kWideTN> <= 2 * kWideStage, "the waves' pieces fit");
    epilogue_rows<DT, TM, kWideTN, BM>(acc, p, m0, n0, (wave >> 1) * WM, (wave & 1) * kWideWN,
                                       lds + wave * 32 * kEpiRow<DT, kWideTN>, scales);
}

// ------------------------------------------------------------------ 128 x 128 tiles
template <bool BKN>
constexpr int kMidScales = 2 * MidLds<BKN>::kStage;
static_assert(4 * 32 * kEpiRow<INT8K_DTYPE_F32, kMidT> <= 2 * MidLds<false>::kStage, "fits");

template <int DT, bool BKN>
__global__ __launch_bounds__(kThreads, 2) void linear_mid_kernel(LinearArgs p, int tiles_m,
                                                                 int tiles_n) {
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * kMidB, n0 = tn * kMidB;
    const TileScales s = load_scales<kMidB>(p, m0, n0);
    v16i acc[kMidT][kMidT];
    if (m0 + kMidB <= p.M && n0 + kMidB <= p.N && p.K % BK == 0)
        mid_mainloop<false, BKN, true>(acc, p.x, p.w, p.M, p.N, p.K, 0, p.K, m0, n0, lds);
    else
        mid_mainloop<true, BKN, true>(acc, p.x, p.w, p.M, p.N, p.K, 0, p.K, m0, n0, lds);
    float* scales = reinterpret_cast<float*>(lds + kMidScales<BKN>);
    park_scales<kMidB>(s, scales);
    const int wave = threadIdx.x >> 6;
    epilogue_rows<DT, kMidT, kMidT, kMidB>(acc, p, m0, n0, (wave >> 1) * kMidW,
                                           (wave & 1) * kMidW, lds + wave * 32 * kEpiRow<DT, kMidT>,
                                           scales);
}

// A K range per blockIdx.y, exact int32 partials.
template <bool BKN>
__global__ __launch_bounds__(kThreads, 2) void linear_mid_split_kernel(LinearArgs p, int tiles_m,
                                                                       int tiles_n,
                                                                       int k_per_split) {
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * kMidB, n0 = tn * kMidB;
    const int kb = (int)blockIdx.y * k_per_split, ke = min(p.K - kb, k_per_split) + kb;
    v16i acc[kMidT][kMidT];
    if (m0 + kMidB <= p.M && n0 + kMidB <= p.N && (ke - kb) % BK == 0)
        mid_mainloop<false, BKN, true>(acc, p.x, p.w, p.M, p.N, p.K, kb, ke, m0, n0, lds);
    else
        mid_mainloop<true, BKN, true>(acc, p.x, p.w, p.M, p.N, p.K, kb, ke, m0, n0, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row0 = m0 + (wave >> 1) * kMidW + (lane & 31);
    const int col0 = n0 + (wave & 1) * kMidW + 4 * (lane >> 5);
    int32_t* c = p.part + (size_t)blockIdx.y * p.M * p.N;
#pragma unroll
    for (int i = 0; i < kMidT; ++i) {
        const int row = row0 + 32 * i;
        if (row >= p.M) continue;
#pragma unroll
        for (int j = 0; j < kMidT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = col0 + 32 * j + 8 * q;
                if (col < p.N)
                    *reinterpret_cast<v4i*>(c + (size_t)row * p.N + col) =
                        v4i{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                            acc[i][j][4 * q + 3]};
            }
    }
}

// ------------------------------------------------------------------ 64 x 64 tiles
// 64 x 64 tiles for the sizes between: a wave owns 32 x 32 and a block 37 KiB of LDS, so four
// blocks share a CU and hide each other's barriers and LDS round trips.  A 128 x 128 tile alone
// on its CU takes 0.70-0.86 us a step, bound by those (loading its operands a step earlier
// changed nothing).  Operands are loaded two steps ahead into registers.
constexpr int kSmB = 64;
template <bool BKN>
struct SmallLds {
    // rows of a [K][N] stage lie 96 bytes apart: the 8 rows of a transposing read start 32
    // bytes apart in the banks
    static constexpr int kBStride = BKN ? kSmB + 32 : LDS_STRIDE;
    static constexpr int kA = kSmB * LDS_STRIDE;
    static constexpr int kStage = kA + (BKN ? BK : kSmB) * kBStride;
    static constexpr int scales(int groups) { return groups * 2 * kStage; }
    static constexpr int bytes(int groups) { return scales(groups) + 3 * kSmB * 4; }
};

// nk steps of K from kb, the part of them below ke; t: thread within its group of 4 waves.
template <bool EDGE, bool BKN>
__device__ __forceinline__ void small_mainloop(v16i& acc, const LinearArgs& p, int kb, int ke, int nk,
                                               int m0, int n0, int t, char* lds) {
    using L = SmallLds<BKN>;
    const int lane = t & 63, wave = t >> 6;
    const int wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0;
    const int a_off = (wm * 32 + (lane & 31)) * LDS_STRIDE + (lane >> 5) * 16;
    const int g16 = lane >> 4, s16 = lane & 15;
    const int b_off = L::kA + (BKN ? (16 * (g16 >> 1) + (s16 >> 1)) * L::kBStride + wn * 32 +
                                         16 * (g16 & 1) + 8 * (s16 & 1)
                                   : (wn * 32 + (lane & 31)) * L::kBStride + (lane >> 5) * 16);
    struct Step {
        int4 a[2], b[2];
    };
    Step f0, f1;  // even and odd steps on their way
    // A (and a packed B): chunk c = t + 256 i, row c / 8, bytes (c % 8) * 16 of the step; B as
    // stored: k row c / 4, bytes (c % 4) * 16 of the tile's 64 columns.  Chunks past the matrix
    // load clamped addresses and are zeroed on EDGE.
    auto load = [&](Step& f, int kt) {
        const int k0 = kb + kt * BK;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = t + i * kThreads;
            const int row = c / kChunksPerRow, gk = min(k0 + (c % kChunksPerRow) * 16, p.K - 16);
            f.a[i] = *reinterpret_cast<const int4*>(p.x + (size_t)min(m0 + row, p.M - 1) * p.K + gk);
            if constexpr (BKN)
                f.b[i] = *reinterpret_cast<const int4*>(
                    p.w + (size_t)min(k0 + (c >> 2), p.K - 1) * p.N + min(n0 + (c & 3) * 16, p.N - 16));
            else
                f.b[i] = *reinterpret_cast<const int4*>(p.w + (size_t)min(n0 + row, p.N - 1) * p.K + gk);
        }
    };
    auto store = [&](const Step& f, char* stage, int kt) {
        const int k0 = kb + kt * BK;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = t + i * kThreads;
            const int row = c / kChunksPerRow, kc = (c % kChunksPerRow) * 16;
            const int br = BKN ? c >> 2 : row, bc = BKN ? (c & 3) * 16 : kc;
            int4 va = f.a[i], vb = f.b[i];
            if constexpr (EDGE) {
                if (!(k0 + kc < ke && m0 + row < p.M)) va = make_int4(0, 0, 0, 0);
                const bool bok = BKN ? k0 + br < ke && n0 + bc < p.N : k0 + bc < ke && n0 + br < p.N;
                if (!bok) vb = make_int4(0, 0, 0, 0);
            }
            *reinterpret_cast<int4*>(stage + row * LDS_STRIDE + kc) = va;
            *reinterpret_cast<int4*>(stage + L::kA + br * L::kBStride + bc) = vb;
        }
    };
    auto read = [&](v4i& a, v4i& b, const char* stage, int s) {
        a = *reinterpret_cast<const v4i*>(stage + a_off + s * 32);
        if constexpr (BKN) {
            typedef int v2i __attribute__((ext_vector_type(2)));
            typedef __attribute__((address_space(3))) v2i lds_v2i;
            const char* q = stage + b_off + s * 32 * L::kBStride;
            const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(q));
            const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(q + 8 * L::kBStride));
            b = v4i{lo.x, lo.y, hi.x, hi.y};
        } else {
            b = *reinterpret_cast<const v4i*>(stage + b_off + s * 32);
        }
    };
    // Step kt reads buffer kt & 1; f holds step kt + 1, which goes to the other buffer (its last
    // reads, step kt - 1's, finished before that step's barrier) and is refilled with step
    // kt + 3.  Loads past the end of K repeat its last bytes and are not used.
    auto step = [&](Step& f, int kt) {
        const char* cur = lds + (kt & 1) * L::kStage;
        v4i a[4], b[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) read(a[s], b[s], cur, s);
        store(f, lds + ((kt + 1) & 1) * L::kStage, kt + 1);
        load(f, kt + 3);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = mfma_ab<true>(a[s], b[s], acc);
        __syncthreads();
    };
    load(f0, 0);
    load(f1, 1);
    store(f0, lds, 0);
    load(f0, 2);
    __syncthreads();
    for (int kt = 0; kt < nk; kt += 2) {
        step(f1, kt);
        if (kt + 1 >= nk) break;
        step(f0, kt + 1);
    }
}

static_assert(4 * 32 * kEpiRow<INT8K_DTYPE_F32, 1> <= 2 * SmallLds<false>::kStage, "fits");

// KG groups of 4 waves take a KG-th of K each, with stages of their own; their sums meet in LDS.
template <int DT, bool BKN, int KG>
__global__ __launch_bounds__(kThreads * KG, 4 / KG) void linear_small_kernel(LinearArgs p, int tiles_m,
                                                                             int tiles_n) {
    using L = SmallLds<BKN>;
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * kSmB, n0 = tn * kSmB;
    const TileScales s = load_scales<kSmB>(p, m0, n0);
    const int t = threadIdx.x % kThreads, group = KG == 1 ? 0 : threadIdx.x / kThreads;
    const int nk = (p.K + KG * BK - 1) / (KG * BK);
    const int kb = group * nk * BK, ke = min(p.K, kb + nk * BK);
    char* stages = lds + group * 2 * L::kStage;
    v16i acc[1][1];
    if (m0 + kSmB <= p.M && n0 + kSmB <= p.N && p.K % (KG * BK) == 0)
        small_mainloop<false, BKN>(acc[0][0], p, kb, ke, nk, m0, n0, t, stages);
    else
        small_mainloop<true, BKN>(acc[0][0], p, kb, ke, nk, m0, n0, t, stages);
    if constexpr (KG > 1) {
        static_assert(KG == 2 && kThreads * 64 <= 2 * L::kStage, "the second group's sums fit its stages");
        if (group > 0)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                reinterpret_cast<v4i*>(stages)[q * kThreads + t] =
                    v4i{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
    }
    float* scales = reinterpret_cast<float*>(lds + L::scales(KG));
    park_scales<kSmB>(s, scales);
    if constexpr (KG > 1) {
        if (group > 0) return;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const v4i x = reinterpret_cast<const v4i*>(lds + 2 * L::kStage)[q * kThreads + t];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[0][0][4 * q + k] += x[k];
        }
    }
    const int wave = t >> 6;
    epilogue_rows<DT, 1, 1, kSmB>(acc, p, m0, n0, (wave >> 1) * 32, (wave & 1) * 32,
                                  lds + wave * 32 * kEpiRow<DT, 1>, scales);
}

// ------------------------------------------------------------------ partials to rows
// 4 columns per thread: the splits' sums, eight loads in flight, then the value.
template <int DT>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinearArgs p, int splits) {
    const int groups = p.N / 4;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= (long long)p.M * groups) return;
    const int row = (int)(e / groups), n = 4 * (int)(e - (long long)row * groups);
    const float sx = p.sx[(size_t)row * p.sx_stride];
    float sw[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        sw[k] = p.sw[(size_t)(n + k) * p.sw_stride];
        b[k] = p.bias != nullptr ? p.bias[n + k] : 0.f;
    }
    const int32_t* src = p.part + (size_t)row * p.N + n;
    const size_t plane = (size_t)p.M * p.N;
    v4i sum = {0, 0, 0, 0};
    for (int s0 = 0; s0 < splits; s0 += 8) {
        v4i x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            x[k] = *reinterpret_cast<const v4i*>(src + min(s0 + k, splits - 1) * plane);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < splits) sum += x[k];
    }
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = linear_value(sum[k], sx, sw[k], b[k]);
    store_four<DT>(static_cast<char*>(p.y) + ((size_t)row * p.N + n) * kOutBytes<DT>, v);
}

// ------------------------------------------------------------------ few tokens, small weights
// A block owns a 32 x 32 output tile; its 8 waves take every 8th 128-deep step of K
// straight from global memory (packed weights), two steps in flight, and meet in LDS.
constexpr int kSkinnyWaves = 8;  // (4 and 16: 2-10% slower from T = 1 to 512)

template <int DT>
__global__ __launch_bounds__(64 * kSkinnyWaves) void linear_skinny_kernel(LinearArgs p) {
    constexpr int kCol = 36, nw = kSkinnyWaves;
    __shared__ __align__(16) int part[nw * 32 * kCol];  // [wave][32 columns][32 rows + 4]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32;
    const size_t koff = (size_t)(lane >> 5) * 16;
    const int8_t* arow = p.x + (size_t)min(m0 + (lane & 31), p.M - 1) * p.K + koff;
    const int8_t* brow = p.w + (size_t)min(n0 + (lane & 31), p.N - 1) * p.K + koff;
    v16i acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0;
    const int step = 128 * nw;
    v4i b0[4], a0[4], b1[4], a1[4];
    int k = 128 * wave;
    if (k < p.K) skinny_load(b0, a0, arow, brow, k);
    for (; k < p.K; k += 2 * step) {
        if (k + step < p.K) skinny_load(b1, a1, arow, brow, k + step);
        skinny_mfma(acc, b0, a0);
        if (k + step >= p.K) break;
        if (k + 2 * step < p.K) skinny_load(b0, a0, arow, brow, k + 2 * step);
        skinny_mfma(acc, b1, a1);
    }
    // lane: column lane % 32, rows 8 q + 4 (lane / 32) ..
    int* mine = part + (wave * 32 + (lane & 31)) * kCol + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4i*>(mine + 8 * q) =
            v4i{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    __syncthreads();
    // 4 columns of a row per thread
    for (int e = threadIdx.x; e < 256; e += blockDim.x) {
        const int row = e >> 3, c = (e & 7) * 4;
        const int m = m0 + row, n = n0 + c;
        if (m >= p.M || n >= p.N) continue;
        const float sx = p.sx[(size_t)m * p.sx_stride];
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < nw; ++w) sum += part[(w * 32 + c + i) * kCol + row];
            v[i] = linear_value(sum, sx, p.sw[(size_t)(n + i) * p.sw_stride],
                                p.bias != nullptr ? p.bias[n + i] : 0.f);
        }
        store_four<DT>(static_cast<char*>(p.y) + ((size_t)m * p.N + n) * kOutBytes<DT>, v);
    }
}

// ------------------------------------------------------------------ plan, launch

enum class LinearRoute { kSkinny, kStream, kSmall, kSmallTwo, kMid, kWide, kTiled };

struct LinearPlan {
    LinearRoute route;
    StreamPlan st;
    MidPlan mid;
    int splits;      // int32 partials, 0: none
    size_t bytes(int M, int N) const { return (size_t)splits * M * N * 4; }
};

// The route with the least estimated time (us).  Fitted to every route timed at 318 sizes: T = 1 to
// 4096, K = 16 to 131056, N = 16 to 128256, weights that come from memory wherever they do not fit
// its cache.  No estimate is below the time to read the weights: 5.9 TB/s is the most that any
// route reached (525 MB in 89 us; a stream that only reads 7.0), and the routes that reach less
// have their own rate.  `steps` are 128 deep; `cold` is 1 for weights of 16 MiB and more, whose
// loads take longer than those of small ones.
//  - small: a step of a block takes a load's latency, or from 256 blocks on its share of the
//    CU (T = 512, 4096 -> 4096: 21 packed, 26 as stored).  As stored it reads 64 bytes a row:
//    5.0 TB/s, 3.7 where rows lie a multiple of 4096 bytes apart (28672 columns 35.5 us, 28736 28.8);
//  - two: up to 256 tiles, a step for each group (T = 64, 4096 -> 6144: 14.5 and 22.7);
//  - mid: a block alone on its CU, or two; split over K, the partials' traffic and a second kernel
//    (T = 16, 14336 -> 4096 in 16 splits 16.9, streamed 19.6; T = 128, 4096 -> 28672 whole 35.6);
//  - wide (packed weights), tiled: the share of rounds and the clock that falls as the GPU fills
//    (T = 4096, 4096 -> 6144: 100 and 115);
//  - stream: a read of the weights per 32 or 64 rows behind a start and a second kernel (T = 1,
//    4096 -> 128256 96 us; as stored in rows of whole 128 bytes, or half as much again);
//  - skinny (packed weights): per 1024 of K and round of 256 blocks, less for few rows, whose lanes
//    load the same lines (T = 1, 4096 -> 6144 8.6, 4096 -> 128256 92).
// Chosen / fastest over those sizes: 1.01 in the mean, 1.23 at worst.
constexpr double kReadRate = 5.9;    // TB/s
constexpr int kMidSplitTiles = 512;  // 128 x 128 tiles split over K, at most
constexpr int kStreamRows = 512;     // rows streamed, at most

LinearPlan linear_plan(int M, int K, int N, bool packed) {
    LinearPlan pl{};
    const double steps = (double)ceil_div(K, BK);
    const double mb = (double)N * K * 1e-6, out = (double)M * N * 1e-6;  // MB of weights, M outputs
    const double cold = std::min((double)N * K, 16777216.0) / 16777216.0;
    const bool ragged = !packed && N % 128 != 0;  // rows as stored are no whole lines
    double best = -1;
    auto better = [&](double time, LinearRoute route) {
        if (best >= 0 && time >= best) return false;
        best = time, pl.route = route, pl.splits = 0;
        return true;
    };
    {
        const long long tiles = ceil_div(M, BM) * ceil_div(N, BN);
        const double rounds = (double)ceil_div(tiles, 256), share = tiles / 256.0;
        better(packed ? 6.4 + std::max(steps * (0.89 * rounds + 0.93 * share), mb / kReadRate) + 0.35 * out
                      : 4.9 + std::max(steps * (1.02 * rounds + 0.80 * share), mb / kReadRate) + 0.42 * out,
               LinearRoute::kTiled);
    }
    if (packed) {
        const long long tiles = ceil_div(M, BM) * ceil_div(N, kWideN);
        const double rounds = (double)ceil_div(tiles, 256), share = tiles / 256.0;
        better(5.0 + std::max(steps * (0.83 * rounds + 0.52 * share), mb / kReadRate) + 0.52 * out,
               LinearRoute::kWide);
    }
    const long long mid_tiles = ceil_div(M, kMidB) * ceil_div(N, kMidB);
    // split where the blocks of whole K leave CUs without their two
    const long long most = mid_tiles <= kMidSplitTiles ? std::min(16LL, (long long)steps) : 1;
    for (long long sp = 1; sp <= most; ++sp) {
        const long long st = ceil_div((long long)steps, sp), n = ceil_div((long long)steps, st);
        if (n != sp) continue;  // the same plan as fewer splits
        const long long blocks = mid_tiles * n, rest = blocks % 512;
        const double alone = packed ? 0.59 + 0.22 * cold : 0.66 + 0.28 * cold;
        const double both = packed ? 1.01 : 1.19, more = packed ? 0.16 : 0.09;
        const double last = rest > 256 ? both + more * (rest - 256) / 256.0 : rest > 0 ? alone : 0.0;
        const double gemm = st * ((both + more) * (double)(blocks / 512) + last);
        const double rate = ragged ? 4.0 : n > 1 ? kReadRate : packed ? 4.4 : 5.4;
        const double rows = n > 1 ? (packed ? 3.65 : 3.23) + 1.56 * n * out : 0.5 * out;
        if (better(3.3 + std::max(gemm, mb / rate) + rows, LinearRoute::kMid)) {
            pl.mid = MidPlan{(int)ceil_div(M, kMidB), (int)ceil_div(N, kMidB), (int)n, (int)(st * BK)};
            pl.splits = n > 1 ? (int)n : 0;
        }
    }
    {
        const long long tiles = ceil_div(M, kSmB) * ceil_div(N, kSmB);
        const double share = tiles / 256.0;
        const double step = packed ? std::max(0.24 + 0.256 * cold, 0.08 + 0.224 * share)
                                   : std::max(0.225 + 0.37 * cold, 0.284 * share);
        const double rate = packed || N % 4096 != 0 ? 5.0 : 3.7;
        better((packed ? 3.05 : 3.35) + std::max(steps * step, mb / rate) + 0.5 * out, LinearRoute::kSmall);
        if (tiles <= 256) {
            const double two = (double)ceil_div((long long)steps, 2) * (packed ? 0.31 + 0.32 * cold : 0.33 + 0.65 * cold);
            better((packed ? 3.8 : 4.05) + std::max(two, mb / kReadRate) + 0.5 * out, LinearRoute::kSmallTwo);
        }
    }
    if (M <= kStreamRows) {
        const StreamPlan sp = stream_plan(M, N, K);
        const double rate = packed || (!ragged && N % 4096 != 0) ? kReadRate : ragged ? 3.6 : 4.9;
        const double start = sp.mt == 1 ? (packed ? 5.7 : 6.4) : (packed ? 8.1 : 8.9);
        const double rows = sp.mt == 1 ? 0.0 : (0.22 + 0.115 * (sp.tiles_m - 1)) * (ragged ? 1.5 : 1.0);
        const double join = (packed ? 0.88 : 0.51) * (double)ceil_div(sp.splits, 8) + (packed ? 1.43 : 1.0) * sp.splits * out;
        if (better(start + std::max(mb * rows, mb / rate) + join, LinearRoute::kStream)) {
            pl.st = sp;
            pl.splits = sp.splits;
        }
    }
    if (packed && K % 128 == 0) {
        const double rounds = (double)ceil_div(ceil_div(N, 32) * ceil_div(M, 32), 256);
        better(2.7 + std::max((1.3 + 0.021 * std::min(M, 32)) * rounds * K / 1024.0, mb / kReadRate),
               LinearRoute::kSkinny);
    }
    return pl;
}

int set_lds(PerDeviceOnce& once, const void* kernel, int bytes) {
    return once.run([=] {
        const hipError_t e =
            hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess) return (int)INT8K_OK;
        set_last_error("hipFuncSetAttribute", e);
        return (int)INT8K_ERR_HIP;
    });
}

template <int DT>
int launch_rows(const LinearArgs& p, int splits, hipStream_t stream) {
    const long long threads = (long long)p.M * (p.N / 4);
    linear_rows_kernel<DT><<<(unsigned)ceil_div(threads, 256), 256, 0, stream>>>(p, splits);
    return check_launch("linear_rows_kernel");
}

template <int DT, bool BKN, int KG>
int launch_small(const LinearArgs& p, hipStream_t stream) {
    static PerDeviceOnce once;
    constexpr int kBytes = SmallLds<BKN>::bytes(KG);
    const int tiles_m = (int)ceil_div(p.M, kSmB), tiles_n = (int)ceil_div(p.N, kSmB);
    if (const int st = set_lds(once, (const void*)linear_small_kernel<DT, BKN, KG>, kBytes)) return st;
    linear_small_kernel<DT, BKN, KG><<<tiles_m * tiles_n, kThreads * KG, kBytes, stream>>>(p, tiles_m, tiles_n);
    return check_launch("linear_small_kernel");
}

template <int DT, bool BKN>
int launch_linear(const LinearArgs& p, const LinearPlan& pl, hipStream_t stream) {
    switch (pl.route) {
        case LinearRoute::kSkinny: {
            const dim3 grid((unsigned)ceil_div(p.N, 32), (unsigned)ceil_div(p.M, 32));
            linear_skinny_kernel<DT><<<grid, 64 * kSkinnyWaves, 0, stream>>>(p);
            return check_launch("linear_skinny_kernel");
        }
        case LinearRoute::kStream: {
            static PerDeviceOnce once1, once2;
            constexpr int kMax = kStMaxWaves * StreamTile<BKN>::kBytes;
            if (const int st = pl.st.mt == 1
                                   ? set_lds(once1, (const void*)gemm_i8_stream_kernel<1, BKN>, kMax)
                                   : set_lds(once2, (const void*)gemm_i8_stream_kernel<2, BKN>, kMax))
                return st;
            if (const int st = launch_gemm_stream<BKN>(p.x, p.w, p.M, p.N, p.K, pl.st, p.part, stream))
                return st;
            return launch_rows<DT>(p, pl.splits, stream);
        }
        case LinearRoute::kSmall:
            return launch_small<DT, BKN, 1>(p, stream);
        case LinearRoute::kSmallTwo:
            return launch_small<DT, BKN, 2>(p, stream);
        case LinearRoute::kMid: {
            static PerDeviceOnce once, once_split;
            const int tiles = pl.mid.tiles_m * pl.mid.tiles_n;
            if (pl.splits > 0) {
                if (const int st = set_lds(once_split, (const void*)linear_mid_split_kernel<BKN>,
                                           MidLds<BKN>::kBytes))
                    return st;
                linear_mid_split_kernel<BKN>
                    <<<dim3(tiles, pl.splits), kThreads, MidLds<BKN>::kBytes, stream>>>(
                        p, pl.mid.tiles_m, pl.mid.tiles_n, pl.mid.k_per_split);
                if (const int st = check_launch("linear_mid_split_kernel")) return st;
                return launch_rows<DT>(p, pl.splits, stream);
            }
            if (const int st = set_lds(once, (const void*)linear_mid_kernel<DT, BKN>,
                                       MidLds<BKN>::kBytes))
                return st;
            linear_mid_kernel<DT, BKN><<<tiles, kThreads, MidLds<BKN>::kBytes, stream>>>(
                p, pl.mid.tiles_m, pl.mid.tiles_n);
            return check_launch("linear_mid_kernel");
        }
        case LinearRoute::kWide: {
            static PerDeviceOnce once;
            if (const int st = set_lds(once, (const void*)linear_wide_kernel<DT>, kWideLds)) return st;
            const int tiles_m = (int)ceil_div(p.M, BM), tiles_n = (int)ceil_div(p.N, kWideN);
            linear_wide_kernel<DT><<<tiles_m * tiles_n, kThreads, kWideLds, stream>>>(p, tiles_m, tiles_n);
            return check_launch("linear_wide_kernel");
        }
        default: {
            static PerDeviceOnce once;
            if (const int st = set_lds(once, (const void*)linear_tiled_kernel<DT, BKN>, kTiledLds))
                return st;
            const int tiles_m = (int)ceil_div(p.M, BM), tiles_n = (int)ceil_div(p.N, BN);
            linear_tiled_kernel<DT, BKN>
                <<<tiles_m * tiles_n, kThreads, kTiledLds, stream>>>(p, tiles_m, tiles_n);
            return check_launch("linear_tiled_kernel");
        }
    }
}

// |x w| <= 2^14 and K products: below 2^17 of them the int32 sum cannot overflow.
constexpr int kMaxK = (1 << 17) - 16;

}  // namespace
}  // namespace int8k

using namespace int8k;

static bool linear_shape_ok(int T, int K, int N) {
    return T > 0 && K > 0 && N > 0 && K % 16 == 0 && N % 16 == 0 && K <= kMaxK &&
           // operands are read through 32-bit buffer offsets
           (long long)T * K < (1LL << 32) && (long long)N * K < (1LL << 32) &&
           ceil_div(T, kMidB) * ceil_div(N, kMidB) < (1LL << 22) &&
           (long long)T * N < (1LL << 36);
}

extern "C" size_t int8k_linear_call_workspace_bytes(int T, int K, int N, int flags) {
    if (!linear_shape_ok(T, K, N)) return 0;
    return linear_plan(T, K, N, (flags & INT8K_LINEAR_WEIGHT_PREPACKED) != 0).bytes(T, N);
}

extern "C" size_t int8k_linear_workspace_bytes(int T, int K, int N, int flags) {
    if (!linear_shape_ok(T, K, N)) return 0;
    const bool packed = (flags & INT8K_LINEAR_WEIGHT_PREPACKED) != 0;
    size_t need = 0;
    auto cover = [&](int first, int last) {
        need = std::max(need, linear_plan(first, K, N, packed).bytes(last, N));
    };
    const int few = std::min(T, kStreamRows);
    for (int t = 1; t <= few; ++t) cover(t, t);
    // Past the streamed rows the estimates of 32 rows differ in their terms per row alone, and the
    // steepest are those of the K splits, steeper the more there are: none has more than the first.
    for (int t = few + 1; t <= T && ceil_div(t, kMidB) * ceil_div(N, kMidB) <= kMidSplitTiles; t += 32)
        cover(t, std::min(t + 31, T));
    return need;
}

extern "C" int int8k_linear(const int8_t* x, const int8_t* W, void* out, int dtype,
                            const float* scale_x, int n_scale_x, const float* scale_W,
                            int n_scale_W, const float* bias, int T, int K, int N, int flags,
                            void* workspace, size_t workspace_bytes, void* stream) {
    clear_last_error();
    if (!x || !W || !out || !scale_x || !scale_W) return INT8K_ERR_INVALID_ARGUMENT;
    if (T <= 0 || K <= 0 || N <= 0 || dtype < INT8K_DTYPE_F16 || dtype > INT8K_DTYPE_F32 ||
        (flags & ~INT8K_LINEAR_WEIGHT_PREPACKED))
        return INT8K_ERR_INVALID_ARGUMENT;
    if ((n_scale_x != 1 && n_scale_x != T) || (n_scale_W != 1 && n_scale_W != N))
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!linear_shape_ok(T, K, N)) return INT8K_ERR_UNSUPPORTED;
    if (!aligned_to(x, 16) || !aligned_to(W, 16) || !aligned_to(out, 16) ||
        !aligned_to(scale_x, 4) || !aligned_to(scale_W, 4) || !aligned_to(bias, 4))
        return INT8K_ERR_MISALIGNED;
    const bool packed = (flags & INT8K_LINEAR_WEIGHT_PREPACKED) != 0;
    const LinearPlan pl = linear_plan(T, K, N, packed);
    if (const size_t need = pl.bytes(T, N)) {
        if (!workspace || workspace_bytes < need) return INT8K_ERR_WORKSPACE;
        if (!aligned_to(workspace, 16)) return INT8K_ERR_MISALIGNED;
    }
    const LinearArgs p{x, W, out, static_cast<int32_t*>(workspace), scale_x, scale_W, bias,
                       n_scale_x == 1 ? 0 : 1, n_scale_W == 1 ? 0 : 1, T, N, K};
    int st = INT8K_OK;
    with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        st = packed ? launch_linear<DT, false>(p, pl, as_stream(stream))
                    : launch_linear<DT, true>(p, pl, as_stream(stream));
    });
    return st;
}
