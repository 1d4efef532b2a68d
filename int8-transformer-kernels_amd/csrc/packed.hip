// packed.hip — INT8 flash attention over packed prompts of different lengths, with grouped
// heads, gfx950.
//
//   Q int8 [heads, T, D], K, V int8 [kv_heads, T, D], per-token scales [heads or kv_heads, T];
//   sequence i holds the tokens cu_seqlens[i] .. cu_seqlens[i+1]-1 of every head, and query
//   head h reads key head h / (heads / kv_heads).  Inside a sequence the math is
//   int8_attention_forward's (prefill.hip):
//     s_ij = (q_i . k_j) sQ_i sK_j / sqrt(D),  out_i = sum_j softmax_j(s_ij) v_j sV_j
//
// A block of 4 waves owns one tile of 128 queries of one head of one sequence, 32 per wave, and
// walks the keys in tiles of 64 transposed, so that each lane owns one query:
// S^T = K . Q^T on v_mfma_i32_32x32x32_i8, O^T += V^T . P^T on v_mfma_f32_32x32x16_f16.  Unlike
// prefill.hip's blocks:
//  - V enters as exact fp16 and its scale goes into the weights p sV, each carried in two fp16, its
//    rounding and what that leaves (22 bits); l sums p in fp32.  The error against 64 bits is that
//    of the formula in fp32 with the output rounded once (1.1-1.3 times it with one fp16 a
//    weight, 1.8 with V sV rounded beside it).  The second product with V costs 22-30% more
//    time at D = 128, 13% at 64 and 17% at 256: 304 us against 238 for the prompts below.
//  - Only a wave's first tile takes the exact step that finds a maximum; diagonal and ragged
//    tiles run the ordinary step with a mask.  Prompts of 300 to 2000 tokens gain 6-20%.
//
// What bounds it: each wave's own chain of scores, softmax and product.  At D = 128 a tile is 40
// large MFMAs (1340 cycles with the small ones) and 330 vector instructions, 32 of them
// exponentials of two slots (1450 cycles).  Two waves share a SIMD, but the matrix and the vector
// units overlap by half at best (32 MFMAs and 256 vector instructions, interleaved or from two
// waves: 710-740 ns, 530 and 320 by themselves); by the counters a wave waits 22% of its time on
// LDS and the barrier, and the clock falls to 1.84 GHz under the load (2.4 at most).  Measured:
// 304-322 us for prompts of 333, 4096, 17, 1000, 2500, 1, 200 and 45 tokens, 32 heads on 8 key heads
// of 128 (49.6 G multiply-adds under the mask in each product); 780 us for one prompt of 8192; 9
// us for five requests of at most 70.  Tried:
//  - the product of one half of a tile among the softmax of the other: 3% slower;
//  - wave priorities around the products or the softmax: no gain;
//  - the sum of p times the tile's largest |sV| as the bound on its weights, one instruction a
//    tile in place of 16: it overestimates so much that tiles leave the ordinary step often (325
//    us); that step's maximum spares the exact one two passes (307 without);
//  and with one fp16 a weight (231 us, 590-600 and 9):
//  - the softmax of a tile next to the MFMAs of its neighbours in one block of instructions (the
//    next scores and the last product with V): no gain, with three K buffers and all 256 registers;
//  - 8 waves and 256 queries per block, half the staging per query: no gain, and 51 against 43 us
//    for eight prompts of 512;
//  - steps of 32 keys, half the code and three quarters of the registers: 5% more for long prompts,
//    8.5 against 9.1 us for the five short requests;
//  - log2 sV in the exponent and l by an MFMA over 4 x 4 blocks, 2 vector instructions less per
//    score: no gain, each small MFMA waiting for the large ones.
//
// The lengths are on the device, so the grid is sized for the most tiles that T tokens of n
// sequences can have (T / kQ + n) and each wave finds its tile from the lengths itself: a
// plan kernel would cost a launch of its own.  Up to 64 sequences, one per lane, tiles are taken
// in the order of their index inside their sequence, the highest first: under the causal mask
// that is heaviest first over all sequences, so short ones fill the end of the grid.  More are
// walked 256 at a time, at most twice: the tiles of sequences of at least kLongTiles tiles come
// first, sequence by sequence, then the others' (200 short prompts in 8192 tokens, 32 heads of
// 128: 117 us, 188 with the order of fewer, whose search reads all lengths a dozen times; 1000
// prompts 0.54 ms, 1.75).
#include "prefill_tiles.h"

namespace int8k {
namespace {

// Sum over the wave on the VALU; every lane gets it.
__device__ __forceinline__ int wave_sum(int v) {
    v = group8_sum(v);
    v += dpp_row_mirror(v);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = (int)(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane((int)(b[0] + b[1]));
}

constexpr int kLongTiles = 8;
// Every block reads the bounds of all sequences, so the time grows with their square.
constexpr int kMaxSeqs = 1 << 16;

// The query tile that rank `i` of the packed order is: sequence tokens [start, start + len),
// tile qt of them.  False past the last tile; `i` is then the rank behind it.
struct PackedTile {
    int start, len, qt;
};
template <int kQ>
__device__ __forceinline__ bool packed_tile(const int32_t* __restrict__ cu, int n, int T, int& i,
                                            PackedTile& t) {
    const int lane = threadIdx.x & 63;
    // bounds that would leave the T tokens are cut, so none leads outside the tensors
    auto bound = [&](int s) { return min(max(cu[min(s, n)], 0), T); };
    auto tiles_in = [](int from, int to) { return (max(to - from, 0) + kQ - 1) / kQ; };
    auto take = [&](int start, int end, int qt) {
        t.start = start, t.len = end - start, t.qt = qt;
        return true;
    };
    if (n <= 64) {
        const int start = bound(lane), end = bound(lane + 1), tiles = tiles_in(start, end);
        auto count = [&](int k) { return wave_sum(max(tiles - k, 0)); };  // tiles with index >= k
        const int total = count(0);
        if (i >= total) {
            i -= total;
            return false;
        }
        // the tile's index is the largest k with count(k) > i
        int lo = 0, hi = (T + kQ - 1) / kQ;  // count(hi) == 0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (count(mid) > i) lo = mid;
            else hi = mid;
        }
        // the j-th sequence that has a tile of that index
        const int j = i - count(lo + 1);
        const bool has = tiles > lo;
        const uint64_t mask = __ballot(has);
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        const int src = __builtin_ctzll(__ballot(has && rank == j));
        return take(__builtin_amdgcn_readlane(start, src), __builtin_amdgcn_readlane(end, src), lo);
    }
    int at[5];  // bounds of this lane's 4 sequences
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < 5; ++k) at[k] = bound(s0 + 4 * lane + k);
    };
    load(0);
    for (int pass = 0; pass < 2; ++pass) {
        auto counted = [&](int from, int to) {  // the sequence's tiles if this pass takes them
            const int tiles = tiles_in(from, to);
            return (tiles >= kLongTiles) == (pass == 0) ? tiles : 0;
        };
        for (int s0 = 0; s0 < n; s0 += 256) {
            if (n > 256 && (pass > 0 || s0 > 0)) load(s0);
            int mine = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) mine += counted(at[k], at[k + 1]);
            const int here = wave_sum(mine);
            if (i >= here) {
                i -= here;
                continue;
            }
            int upto = mine;  // inclusive sum over the lanes
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int below = __shfl_up(upto, d);
                upto += lane >= d ? below : 0;
            }
            const int src = __builtin_ctzll(__ballot(upto > i));
            int left = i - __builtin_amdgcn_readlane(upto - mine, src);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int start = __builtin_amdgcn_readlane(at[k], src);
                const int end = __builtin_amdgcn_readlane(at[k + 1], src);
                const int tiles = counted(start, end);
                if (left < tiles) return take(start, end, tiles - 1 - left);
                left -= tiles;
            }
        }
    }
    return false;
}

// ------------------------------------------------------------------ the block

// LDS of a block, all twice: a K tile (int8 rows, 16-byte padded), a V tile (fp16 [key][dim]),
// the scales of its keys.
template <int D>
struct PackedLds {
    static constexpr int kKStride = D + 16;
    static constexpr int kKBytes = kKV * kKStride;
    static constexpr int kVRow = D + 32;  // halfs: see VLayout
    static constexpr int kVBytes = kKV * kVRow * 2;
    static constexpr int kV = 2 * kKBytes;
    static constexpr int kS = kV + 2 * kVBytes;
    static constexpr int kSFloats = 2 * kKV;  // sK, sV
    static constexpr int kBytes = kS + 2 * kSFloats * 4;
};

constexpr int kPackedWaves = 4;              // per block, 32 queries each
constexpr float kPackedMaxWeight = 60000.f;  // fp16 weights stay below it
constexpr float kPackedMaxShift = 60.f;      // |m - running maximum| where m is set
constexpr float kPackedTopExp = 8.f;         // the largest weight there is 2^kPackedTopExp

struct ExactStep : std::true_type {};  // the step that sets m; masked, as some of the others are

template <int D, bool CAUSAL, bool PAD, typename OutRow>
__device__ __forceinline__ void packed_block(char* smem, const int8_t* __restrict__ Qh,
                                             const int8_t* __restrict__ Kh,
                                             const int8_t* __restrict__ Vh,
                                             const float* __restrict__ sQh,
                                             const float* __restrict__ sKh,
                                             const float* __restrict__ sVh,
                                             uint16_t* __restrict__ out, int S, int qt,
                                             float qk_scale_log2, int d_mem, OutRow out_row) {
    constexpr int QW = kPackedWaves;
    constexpr int NS = D / 32;  // 32-wide d slices (QK k-steps) and O^T row tiles
    constexpr int kQ = 32 * QW, kT = 64 * QW;
    using L = PackedLds<D>;
    using St = Stage<D, QW>;
    using VL = VLayout<D, QW>;
    const int dm = PAD ? d_mem : D;
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int h = lane >> 5;
    const int qw0 = qt * kQ + wave * 32;  // first query of this wave
    const int q = qw0 + (lane & 31);      // this lane's query
    const bool qok = q < S;

    // Q^T fragments (B operand of the QK MFMA): column q, 16 bytes of d-slice s.
    v4i qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
        qf[s] = (!PAD || 32 * s + 16 * h < dm)
                    ? *reinterpret_cast<const v4i*>(Qh + (size_t)min(q, S - 1) * dm + 32 * s + 16 * h)
                    : v4i{0, 0, 0, 0};
    const float qscale = qok ? sQh[q] * qk_scale_log2 : 0.f;

    // Step i of the walk is tile tile_of(i): first the nd tiles that some query of the block
    // does not see whole (the diagonal, the last tile of a ragged sequence), which are masked,
    // the last of them first, so a wave that skips some of them skips the first ones; then the
    // whole ones.
    const int kv_end = CAUSAL ? min(S, (qt + 1) * kQ) : S;
    const int n = (kv_end + kKV - 1) / kKV;
    const int kd = CAUSAL ? qt * kQ / kKV : S / kKV;  // whole tiles
    const int nd = n - kd;
    auto tile_of = [&](int i) {
        i = min(i, n - 1);  // steps past the end repeat the last tile's loads
        return i < nd ? n - 1 - i : i - nd;
    };
    const int q_wave_last = min(qw0 + 31, S - 1);
    auto computes = [&](int i) { return qw0 < S && !(CAUSAL && tile_of(i) * kKV > q_wave_last); };

    // ---- loads
    const TileSrc src = make_tile_src<D, QW>(Kh, Vh, sKh, sVh, S, dm, t);
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    struct KeyLoads {
        int4 k[St::kKChunks];
    };
    struct ScaleLoads {
        float k, v;
    };
    uint2 pvr[St::kVItems][4];
    auto fetch_k = [&](int i) {
        KeyLoads l;
        const uint32_t k0 = tile_of(i) * kKV;  // (offsets below 2^32 by the entry's check)
#pragma unroll
        for (int c = 0; c < St::kKChunks; ++c) {
            v4u w = {0, 0, 0, 0};
            if (!PAD || src.kvalid)
                w = __builtin_amdgcn_raw_buffer_load_b128(
                    src.k, src.voff_k, k0 * dm + c * (PAD ? src.kstep : (uint32_t)(kT * 16)), 0);
            l.k[c] = make_int4((int)w.x, (int)w.y, (int)w.z, (int)w.w);
        }
        return l;
    };
    auto fetch_v = [&](int i) {
        const uint32_t k0 = tile_of(i) * kKV;
#pragma unroll
        for (int c = 0; c < St::kVItems; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pvr[c][r] = make_uint2(0, 0);
                if (!PAD || (src.vvalid >> c) & 1u)
                    pvr[c][r] = load_v_f16x4(src.v, src.voff_v, (k0 + r) * dm + c * 4 * VL::kW);
            }
    };
    // (every wave holds the scales, the first one stores them)
    auto fetch_s = [&](int i) {
        const uint32_t k0 = tile_of(i) * kKV;
        return ScaleLoads{
            __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(src.s, src.voff_s, k0 * 4, 0)),
            __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(src.sv, src.voff_s, k0 * 4, 0))};
    };
    auto put_k = [&](char* buf, const KeyLoads& l) {
#pragma unroll
        for (int c = 0; c < St::kKChunks; ++c) {
            const int e = t + c * kT;
            *reinterpret_cast<int4*>(buf + e / (D / 16) * L::kKStride + e % (D / 16) * 16) = l.k[c];
        }
    };
    auto put_v = [&](char* buf) {
        _Float16* vs = reinterpret_cast<_Float16*>(buf) + (t / VL::kW) * 4 * L::kVRow + (t % VL::kW) * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < St::kVItems; ++c)
                *reinterpret_cast<uint2*>(vs + r * L::kVRow + c * 4 * VL::kW) = pvr[c][r];
    };
    auto put_s = [&](int i, const ScaleLoads& l) {
        if (wave != 0) return;
        float* s = reinterpret_cast<float*>(smem + L::kS) + (i & 1) * L::kSFloats;
        s[lane] = l.k;
        s[kKV + lane] = l.v;
    };

    // ---- compute
    v16f o[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, l = 0.f;

    // S^T = K . Q^T of a tile's 32 keys from 32 T
    const int k_lane = (lane & 31) * L::kKStride + 16 * h;
    auto scores = [&](const char* kbuf, int T) {
        v4i kf[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s)
            kf[s] = *reinterpret_cast<const v4i*>(kbuf + k_lane + T * 32 * L::kKStride + s * 32);
        v16i a;
#pragma unroll
        for (int z = 0; z < 16; ++z) a[z] = 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) a = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[s], qf[s], a, 0, 0, 0);
        return a;
    };
    // O^T += V^T . P^T, the V^T fragments by transposing reads (see VLayout)
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    const int v_lane = (4 * h + ((lane & 15) >> 2)) * 2 * L::kVRow +
                       2 * (16 * ((lane >> 4) & 1) + 4 * (lane & 3));
    auto product = [&](const char* vbuf, const v8h (&p)[4], const v8h (&r)[4]) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const char* a = vbuf + v_lane + ks * 32 * L::kVRow + j * 64;
                const v4h lo = __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)a));
                const v4h hi = __builtin_bit_cast(
                    v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(a + 16 * L::kVRow)));
                const v8h v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[ks], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, r[ks], o[j], 0, 0, 0);
            }
        // the fragments (two reads each) kAhead pairs of MFMAs ahead of their use
        constexpr int kAhead = 2;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int i = 0; i < 4 * NS - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * kAhead, 0);
    };
    // The weights of a lane's four keys of chunk ch, 32 (ch / 4) + 8 (ch % 4) + 4 h + 0..3, their
    // scores being registers 4 (ch % 4) .. + 3 of s: e = 2^(x - m), p = fp16(e sV), r = fp16(e sV - p).
    // Returns the sum of e; wide takes in the largest |e sV|.  sQ sK comes from an MFMA over 4 x 4
    // blocks (lanes 4b .. 4b + 3, the outer product of a lane's own key scale with the lanes'
    // query scales), which leaves one multiplication less per score than sK read as it is (2% at
    // 8192 tokens, 32 heads of 128).
    typedef float v4f __attribute__((ext_vector_type(4)));
    auto scale_qk = [&](int ch, const float* sc) {
        return __builtin_amdgcn_mfma_f32_4x4x1f32(sc[32 * (ch >> 2) + 8 * (ch & 3) + 4 * h + (lane & 3)], qscale,
                                                  v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    };
    auto scale_v = [&](int ch, const float* sc) {
        return *reinterpret_cast<const v4f*>(sc + kKV + 32 * (ch >> 2) + 8 * (ch & 3) + 4 * h);
    };
    auto weights = [&](int ch, const v16i& s, const float* sc, v8h (&p)[4], v8h (&r)[4], float& wide, auto mask, auto seen) {
        const int T = ch >> 2, g = ch & 3;
        const v4f sqk = scale_qk(ch, sc), sv = scale_v(ch, sc);
        float e[4], w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            e[c] = fast_exp2(fmaf(static_cast<float>(s[4 * g + c]), sqk[c], -m));
            w[c] = e[c] * sv[c];
            asm("" : "+v"(w[c]));  // rounded to fp32 first in every copy of this code
            if constexpr (decltype(mask)::value) {
                const bool ok = seen(32 * T + 8 * g + 4 * h + c);
                e[c] = ok ? e[c] : 0.f;
                w[c] = ok ? w[c] : 0.f;
            }
        }
        wide = fmaxf(fmaxf(wide, fabsf(w[0])), fabsf(w[1]));
        wide = fmaxf(fmaxf(wide, fabsf(w[2])), fabsf(w[3]));
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            typedef float f2 __attribute__((ext_vector_type(2)));
            const h2 top = __builtin_convertvector((f2){w[c], w[c + 1]}, h2);
            float rest0 = minus_half<0>(w[c], top), rest1 = minus_half<1>(w[c + 1], top);
            if constexpr (std::is_same_v<decltype(mask), ExactStep>) {
                // (a weight past fp16's range, by an infinite value scale, leaves no rest)
                rest0 = fabsf(w[c]) < 65520.f ? rest0 : 0.f;
                rest1 = fabsf(w[c + 1]) < 65520.f ? rest1 : 0.f;
            }
            const h2 rest = __builtin_convertvector((f2){rest0, rest1}, h2);
            const int at = 4 * (g & 1) + c;
            p[2 * T + (g >> 1)][at] = top.x, p[2 * T + (g >> 1)][at + 1] = top.y;
            r[2 * T + (g >> 1)][at] = rest.x, r[2 * T + (g >> 1)][at + 1] = rest.y;
        }
        return (e[0] + e[1]) + (e[2] + e[3]);
    };
    auto k_buf = [&](int i) { return smem + (i & 1) * L::kKBytes; };
    // 0 where the query's weights fit m; else the largest of them, or infinity
    float over = INFINITY;
    // The exact path: sets m by the tile's largest weight and rescales O and l.
    auto slow = [&](int i, const float* sc, v8h (&p)[4], v8h (&r)[4]) {
        const int last = (CAUSAL ? min(q, S - 1) : S - 1) - tile_of(i) * kKV;  // last key seen
        auto seen = [&](int key) { return key <= last; };
        const v16i sacc[2] = {scores(k_buf(i), 0), scores(k_buf(i), 1)};
        // The largest weight becomes 2^kPackedTopExp, which fp16 holds exactly.  Below 2^-14 fp16
        // steps by 2^-24, so a weight is off by at most 2^-33 of the largest, and long flat
        // tails add up; the factor of 234 up to kPackedMaxWeight is the room before a tile
        // takes this path again.  The step that was left has found the largest under m, unless
        // it left fp32's range or there is no m yet.
        const float left = max_xor32(over);
        float raised = m + __builtin_amdgcn_logf(left) - kPackedTopExp;
        if (__ballot(left == INFINITY) != 0) {
            float top = -INFINITY;
#pragma unroll
            for (int ch = 0; ch < 8; ++ch) {
                const v4f sqk = scale_qk(ch, sc);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float x = static_cast<float>(sacc[ch >> 2][4 * (ch & 3) + c]) * sqk[c];
                    top = fmaxf(top, seen(32 * (ch >> 2) + 8 * (ch & 3) + 4 * h + c) ? x : -INFINITY);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            top = max_xor32(top);
            const float base = top == -INFINITY ? 0.f : top;
            float pm = 0.f;
#pragma unroll
            for (int ch = 0; ch < 8; ++ch) {
                const v4f sqk = scale_qk(ch, sc), sv = scale_v(ch, sc);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float x = sv[c] * fast_exp2(fmaf(static_cast<float>(sacc[ch >> 2][4 * (ch & 3) + c]),
                                                           sqk[c], -base));
                    pm = fmaxf(pm, seen(32 * (ch >> 2) + 8 * (ch & 3) + 4 * h + c) ? fabsf(x) : 0.f);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            pm = max_xor32(pm);
            const float shift = pm > 0.f && pm < INFINITY ? __builtin_amdgcn_logf(pm) : 0.f;
            const float set =
                fmaxf(m, top + fminf(fmaxf(shift - kPackedTopExp, -kPackedMaxShift), kPackedMaxShift));
            raised = left == INFINITY ? set : raised;
        }
        // (a query whose weights fit keeps its m, whatever its neighbours in the wave hold)
        const float m_new = left != 0.f ? raised : m;
        const float alpha = fast_exp2(m - (m_new == -INFINITY ? 0.f : m_new));
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[j][r] *= alpha;
        float psum = 0.f, wide = 0.f;  // (summed as in a step that keeps m)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            psum += weights(c, sacc[c >> 2], sc, p, r, wide, ExactStep{}, seen);
            __builtin_amdgcn_sched_barrier(0);
        }
        l += psum;
    };
    auto scales_of = [&](int i) {
        return reinterpret_cast<const float*>(smem + L::kS) + (i & 1) * L::kSFloats;
    };

    // Step i reads buffer i & 1 while the registers hold tile i + 1, loaded during step i - 1;
    // at its end that goes to the other buffer, the loads of tile i + 2 go out, and the step's
    // one barrier follows.
    auto v_buf = [&](int i) { return smem + L::kV + (i & 1) * L::kVBytes; };
    KeyLoads pk;
    ScaleLoads ps;
    auto fetch = [&](int i) {
        pk = fetch_k(i);
        fetch_v(i);
        ps = fetch_s(i);
    };
    auto put = [&](int i) {
        put_k(k_buf(i), pk);
        put_v(v_buf(i));
        put_s(i, ps);
    };
    fetch(0);
    put(0);
    fetch(1);
    __syncthreads();
    auto advance = [&](int i) {
        put(i + 1);
        fetch(i + 2);
        __syncthreads();
    };
    // The steps up to `end` that keep m; false where step i has weights that leave the range m
    // gives them, before anything of it is in O.
    int i = 0;
    auto steps = [&](int end, auto mask) {
        for (; i < end; ++i) {
            const float* sc = scales_of(i);
            const int last = (CAUSAL ? min(q, S - 1) : S - 1) - tile_of(i) * kKV;  // last key seen
            v8h p[4], r[4];
            float psum = 0.f, wide = 0.f;
            const v16i sacc[2] = {scores(k_buf(i), 0), scores(k_buf(i), 1)};
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                psum += weights(c, sacc[c >> 2], sc, p, r, wide, mask, [&](int key) { return key <= last; });
                // (keeps the scales of all chunks from being read first: 2-9% at D = 256)
                if (c & 1) __builtin_amdgcn_sched_barrier(0);
            }
            over = psum <= 0x1p60f ? (wide <= kPackedMaxWeight ? 0.f : wide) : INFINITY;
            if (__ballot(over != 0.f) != 0) return false;
            l += psum;
            product(v_buf(i), p, r);
            advance(i);
        }
        return true;
    };
    bool running = false;  // wave-uniform: an exact step has set m
    while (i < n) {
        if (running) {
            if (steps(nd, std::true_type{}) && steps(n, std::false_type{})) break;
        }
        if (computes(i)) {
            running = true;
            v8h p[4], r[4];
            slow(i, scales_of(i), p, r);
            product(v_buf(i), p, r);
        }
        advance(i);
        ++i;
    }

    const float Lsum = sum_xor32(l);
    if (!qok) return;  // lanes l and l^32 share q, so both leave or both stay
    const float inv = 1.f / Lsum;
    uint16_t* orow = out + out_row(q) * dm;
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * j + 8 * g + 4 * h;
            if (PAD && d >= dm) continue;
            uint32_t w[2];
#pragma unroll
            for (int c = 0; c < 2; ++c)
                w[c] = __half_as_ushort(f16_of_f32(o[j][4 * g + 2 * c] * inv)) |
                       ((uint32_t)__half_as_ushort(f16_of_f32(o[j][4 * g + 2 * c + 1] * inv)) << 16);
            *reinterpret_cast<uint2*>(orow + d) = make_uint2(w[0], w[1]);
        }
}

// zero_rest: the rows of out that no sequence holds are written as zeros by the blocks that
// have no tile (the grid has one rank more than there can be tiles).
// Heads: every XCD takes workgroups in turn, so where 8 divides the heads XCD x gets heads
// x heads / 8 .. and its L2 the K and V of their key heads alone (231 against 252 us for the
// prompts above).
template <int D, bool CAUSAL, bool PAD>
__global__ __launch_bounds__(64 * kPackedWaves, D == 256 ? 1 : 2) void packed_kernel(
    const int8_t* __restrict__ Q, const int8_t* __restrict__ K, const int8_t* __restrict__ V,
    const float* __restrict__ sQ, const float* __restrict__ sK, const float* __restrict__ sV,
    uint16_t* __restrict__ out, const int32_t* __restrict__ cu, int n, int T, int heads,
    int group, float qk_scale_log2, int thd, int zero_rest, int d_mem) {
    extern __shared__ __align__(16) char smem_all[];
    const int dm = PAD ? d_mem : D;
    int rank = (int)blockIdx.x / heads;
    const int ranks = (int)gridDim.x / heads;
    int h = (int)blockIdx.x % heads;
    if (heads % 8 == 0) h = h % 8 * (heads / 8) + h / 8;
    PackedTile t;
    const int wanted = rank;
    if (!packed_tile<32 * kPackedWaves>(cu, n, T, rank, t)) {
        if (!zero_rest) return;
        // rank is now this block's index among the idle ones of its head
        const int idle = ranks - (wanted - rank);
        const int begin = min(max(cu[0], 0), T), end = min(max(cu[n], begin), T);
        const int words = dm / 4;  // 8-byte pieces of a row
        const int rows = begin + (T - end);
        for (int r = rank; r < rows; r += idle) {
            const int row = r < begin ? r : end + (r - begin);
            const size_t o = thd ? (size_t)row * heads + h : (size_t)h * T + row;
            if ((int)threadIdx.x < words)
                reinterpret_cast<uint2*>(out + o * dm)[threadIdx.x] = make_uint2(0, 0);
        }
        return;
    }
    const size_t qrow = (size_t)h * T + t.start, krow = (size_t)(h / group) * T + t.start;
    packed_block<D, CAUSAL, PAD>(
        smem_all, Q + qrow * dm, K + krow * dm, V + krow * dm, sQ + qrow, sK + krow, sV + krow,
        out, t.len, t.qt, qk_scale_log2, d_mem, [&](int q) {
            return thd ? (size_t)(t.start + q) * heads + h : qrow + q;
        });
}

struct PackedArgs {
    const int8_t *Q, *K, *V;
    const float *sQ, *sK, *sV;
    uint16_t* out;
    const int32_t* cu;
    int n, T, heads, kv_heads, dm;
    bool causal, thd, zero_rest;
};

template <int D>
int launch_packed(const PackedArgs& a, hipStream_t stream) {
    constexpr int kQ = 32 * kPackedWaves, kThreads = 64 * kPackedWaves;
    // (a tile that is not whole is the last of a sequence that holds a token)
    const long long ranks = (long long)a.T / kQ + std::min(a.n, a.T) + 1;
    const float qk = (1.0f / std::sqrt((float)a.dm)) * kLog2e;
    constexpr int kLds = PackedLds<D>::kBytes;
    if (ranks * a.heads * kThreads >= (1LL << 32)) return INT8K_ERR_UNSUPPORTED;
    static PerDeviceOnce lds_once;
    const int st = set_lds_limit(
        lds_once, kLds, packed_kernel<D, true, false>, packed_kernel<D, false, false>,
        packed_kernel<D, true, true>, packed_kernel<D, false, true>);
    if (st != INT8K_OK) return st;
    const unsigned blocks = (unsigned)(ranks * a.heads);
#define INT8K_PACKED_LAUNCH(C, P)                                                               \
    packed_kernel<D, C, P><<<blocks, kThreads, kLds, stream>>>(                             \
        a.Q, a.K, a.V, a.sQ, a.sK, a.sV, a.out, a.cu, a.n, a.T, a.heads, a.heads / a.kv_heads,  \
        qk, a.thd ? 1 : 0, a.zero_rest ? 1 : 0, a.dm)
    if (a.dm == D) {
        if (a.causal) INT8K_PACKED_LAUNCH(true, false);
        else INT8K_PACKED_LAUNCH(false, false);
    } else {
        if (a.causal) INT8K_PACKED_LAUNCH(true, true);
        else INT8K_PACKED_LAUNCH(false, true);
    }
#undef INT8K_PACKED_LAUNCH
    return check_launch("packed_kernel");
}

}  // namespace
}  // namespace int8k

using namespace int8k;

extern "C" int int8k_attention_forward_packed(
    const int8_t* Q, const int8_t* K, const int8_t* V, uint16_t* out, const float* scale_Q,
    const float* scale_K, const float* scale_V, const int32_t* cu_seqlens, int num_seqs,
    int total_tokens, int heads, int kv_heads, int head_dim, int flags, void* stream) {
    clear_last_error();
    if (!Q || !K || !V || !out || !scale_Q || !scale_K || !scale_V || !cu_seqlens)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (flags & ~(INT8K_ATTN_CAUSAL | INT8K_ATTN_OUT_THD | INT8K_ATTN_ZERO_REST))
        return INT8K_ERR_INVALID_ARGUMENT;
    if (num_seqs <= 0 || total_tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
        heads % kv_heads != 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!on_mfma(head_dim) || num_seqs > kMaxSeqs) return INT8K_ERR_UNSUPPORTED;
    if ((long long)total_tokens * head_dim >= (1LL << 32)) return INT8K_ERR_UNSUPPORTED;  // buffer range
    if (!aligned_to(Q, 16) || !aligned_to(K, 16) || !aligned_to(V, 16) || !aligned_to(out, 8) ||
        !aligned_to(scale_Q, 4) || !aligned_to(scale_K, 4) || !aligned_to(scale_V, 4) ||
        !aligned_to(cu_seqlens, 4))
        return INT8K_ERR_MISALIGNED;
    const PackedArgs a{Q,
                       K,
                       V,
                       scale_Q,
                       scale_K,
                       scale_V,
                       out,
                       cu_seqlens,
                       num_seqs,
                       total_tokens,
                       heads,
                       kv_heads,
                       head_dim,
                       (flags & INT8K_ATTN_CAUSAL) != 0,
                       (flags & INT8K_ATTN_OUT_THD) != 0,
                       (flags & INT8K_ATTN_ZERO_REST) != 0};
    hipStream_t s = as_stream(stream);
    if (head_dim <= 64) return launch_packed<64>(a, s);
    if (head_dim <= 128) return launch_packed<128>(a, s);
    return launch_packed<256>(a, s);
}
