// kv4.hip — a paged KV cache held in 4 bits: append, read back, and grouped decode attention,
// gfx950.
//
// A cache row is one token of one key head: D codes of 4 bits, two a byte (element 2i in the
// low half of byte i, 2i + 1 in the high half), each stored as code + 8, and one fp32 scale:
//   s = max(|row|, 1e-8) * fl(1/7),  code = rn(clamp(x / s, -8, 7)),  x ~= code * s
// (the product with the rounded reciprocal is what `amax / 7` is on the device in PyTorch, whose
// division by a host number multiplies)
// K_pages and V_pages uint8 [num_pages, kv_heads, page, D/2], scales fp32 [num_pages,
// kv_heads, page].  A NaN in a row makes its scale NaN (as amax does in PyTorch).
#include <algorithm>
#include <cmath>

#include "rows.h"

namespace int8k {
namespace {

__device__ unsigned int g_kv4_bad_ids;

// ------------------------------------------------------------------ append, read

// |x| as ordered bits: NaN above infinity, so a maximum keeps it.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float kv4_scale(uint32_t amax_bits) {
    const float m = __uint_as_float(amax_bits);
    return (m < 1e-8f ? 1e-8f : m) * (1.f / 7.f);  // NaN stays NaN
}

// rn(clamp(x / s, -8, 7)) + 8 from inv = 1 / s (the correctly rounded quotient of rows.h; NaN
// clamps to -8).  Adding 1.5 * 2^23 + 8 rounds half to even onto the integers and leaves the
// sum in the low bits.
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float inv) {
    const float q = fminf(fmaxf(quotient(x, s, inv), -8.f), 7.f);
    return __float_as_uint(q + 12582920.0f) & 15u;
}

template <int DT>
__device__ __forceinline__ void load_row8(const void* x, size_t i, float (&v)[8]) {
    if constexpr (DT == INT8K_DTYPE_F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + i);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        unpack_chunk<DT>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i), v);
    }
}

struct Kv4Side {
    const void* x;        // [T, H, D] with strides st, sh (elements), D contiguous
    long long st, sh;
    uint8_t* pages;
    float* scales;
};

// 8 lanes (D = 64) or 16 (D = 128) per row, 8 elements each; blockIdx.y: 0 = K, 1 = V.  A block
// holds consecutive tokens of one head, whose rows and scales are neighbours in the cache
// where the slots are (8191 tokens of 8 heads of 128: heads side by side 11.5 us).
// A row is read as 16-byte pieces and written as one run of D/2 bytes.  Bound by its
// instructions with a true division per element (8191 tokens of 8 heads of 128 15.2 us).
// R rows per lane group, whose loads go out together: with one, the waves of a long prompt come
// and go at the pace of their latencies (8191 tokens 11.6 us, with 4 the time below).
template <int DT, int D, int R>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Side k, Kv4Side v,
                                                         const int32_t* __restrict__ slots,
                                                         int T, int H, int num_pages,
                                                         int log2_page) {
    constexpr int L = D / 8, kLg = D == 64 ? 3 : 4, kRows = 256 / L;
    const int h = (int)(blockIdx.x % (unsigned)H), c = threadIdx.x & (L - 1);
    const int t0 = (int)(blockIdx.x / (unsigned)H) * (kRows * R) + (int)threadIdx.x / L;
    if (t0 >= T) return;  // whole lane groups leave together
    const Kv4Side sd = blockIdx.y == 0 ? k : v;
    int slot[R];
    float e[R][8];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int t = min(t0 + i * kRows, T - 1);  // rows past the last token repeat it, unstored
        slot[i] = slots[t];
        load_row8<DT>(sd.x, (size_t)(t * sd.st + h * sd.sh) + 8 * c, e[i]);
    }
    const long long cap = (long long)num_pages << log2_page;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, abs_bits(e[i][j]));
        m = __float_as_uint(row_reduce(__uint_as_float(m), kLg, [](float a, float b) {
            return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
        }));
        const float s = kv4_scale(m), inv = 1.f / s;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= kv4_code(e[i][j], s, inv) << (4 * j);
        if (t0 + i * kRows >= T || slot[i] < 0) continue;
        if (slot[i] >= cap) {
            if (h == 0 && c == 0 && blockIdx.y == 0) atomicAdd(&g_kv4_bad_ids, 1u);
            continue;
        }
        const int page = slot[i] >> log2_page, off = slot[i] & ((1 << log2_page) - 1);
        const size_t r = (((size_t)page * H + h) << log2_page) + off;
        reinterpret_cast<uint32_t*>(sd.pages + r * (D / 2))[c] = w;
        if (c == 0) sd.scales[r] = s;
    }
}

// Rows at `slots` as numbers of the dtype; slots outside the cache read as zeros.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ pages,
                                                       const float* __restrict__ scales,
                                                       const int32_t* __restrict__ slots,
                                                       void* __restrict__ out, int T, int H,
                                                       int num_pages, int log2_page) {
    constexpr int L = D / 8;
    const int h = (int)(blockIdx.x % (unsigned)H), c = threadIdx.x & (L - 1);
    const int t = (int)(blockIdx.x / (unsigned)H) * (256 / L) + (int)threadIdx.x / L;
    if (t >= T) return;
    const int slot = slots[t];
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0 && slot < ((long long)num_pages << log2_page)) {
        const int page = slot >> log2_page, off = slot & ((1 << log2_page) - 1);
        const size_t r = (((size_t)page * H + h) << log2_page) + off;
        const uint32_t w = reinterpret_cast<const uint32_t*>(pages + r * (D / 2))[c];
        const float s = scales[r];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
    }
    const size_t o = ((size_t)t * H + h) * D + 8 * c;
    if constexpr (DT == INT8K_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + o);
        p[0] = make_float4(y[0], y[1], y[2], y[3]);
        p[1] = make_float4(y[4], y[5], y[6], y[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo = y[2 * i], hi = y[2 * i + 1];
            asm("" : "+v"(lo), "+v"(hi));
            w[i] = pack_pair<DT>(lo, hi);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + o) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ------------------------------------------------------------------ decode
// The scores and the weighted values of up to 16 query heads that share a key head are one
// MFMA tile, so a wave reads every cache row once for all of them: tiles of 32 positions,
//   S^T[32 keys x 16 q] = K . Q^T    v_mfma_i32_16x16x64_i8, exact int32: the codes enter as
//                                    0..15 (one AND, one shift), -8 sum(q) as the initial sum
//   O^T[D x 16 q]      += V^T . P^T  v_mfma_f32_16x16x32_f16, the codes as exact fp16
// In the accumulator layout lane l holds query l % 16 and rows 4 (l / 16) + r.  Rows are keys
// in the order 4 (m % 4) + m / 4, so lane group g = l / 16 ends up with the scores of keys
// 4 j + g, j = 0..7, as the B operand of the second product wants them: P never changes lanes.
// The A operand of that product is 8 keys of one dim per lane: lane l reads word l % 16 (8
// dims) of those 8 rows and picks a byte of two keys at a time (v_perm), each half of which
// becomes two fp16 codes with an AND, an OR and one packed operation.  No LDS in the loop.
//
// Positions are uniform over the wave, so pages and addresses are scalar.  A wave holds the
// next tile's loads in registers while it computes one (4.3 KiB at D = 128).  Every load
// instruction covers whole lines and is non-temporal (B32, 8 key heads of 128, up to 16K
// positions: 80 -> 71 us; the loads alone 75 -> 66).
//
// p_j = 2^(s_j - m) with a reference m per query that is not the running maximum: it is set so
// that the largest weight p sV of the tile that set it lies in [2^9, 2^10), whatever the size of
// the value scales, and a tile whose weights stay in fp16's range under the current m takes
// the short path, with no exchange between lanes and no rescaling.  l sums p and O the
// weighted codes, both in fp32 and both relative to m.  Below 2^-14 fp16 steps by 2^-24, so a
// weight is off by at most 2^-25 beside a largest one of 2^9 or more: 65536 equal keys behind
// one that outweighs them together by 2^8 still add up (with a largest weight below 1 they
// vanish).  The factor of 60 up to kMaxWeight is the room before a tile takes the long path.
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;       // keys per tile
constexpr int kMaxRows = 16;    // query heads per block
constexpr float kMaxWeight = 60000.f;  // fp16 weights stay below it
constexpr float kMaxSum = 0x1p60f;      // and the sum of a lane's 8 p below this
constexpr int kMaxShift = 60;           // |m - running maximum| where m is set
constexpr int kTopExp = 10;             // the largest weight there: below 2^kTopExp

struct Kv4Decode {
    const int8_t* Q;
    const uint8_t *K, *V;
    const float *sQ, *sK, *sV;
    const int32_t *tables, *lens;
    uint16_t* out;
    float *part_ml, *part_acc;  // [B * Hq][nsplit][2] and [..][D] (nsplit > 1)
    int B, Hq, Hkv, num_pages, log2_page, max_pages, max_context;
    int groups, rows, nsplit;   // blocks of query heads per key head, heads in each
    float qk;
};

// Value of lane N of each row of 16 lanes (DPP row_newbcast).
template <int N>
__device__ __forceinline__ float bcast16(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + N, 0xF, 0xF, true));
}

// max or sum over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    return max_xor32(fmaxf(__int_as_float(a[0]), __int_as_float(a[1])));
}
__device__ __forceinline__ float sum_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    return sum_xor32(__int_as_float(a[0]) + __int_as_float(a[1]));
}

template <int D>
struct Kv4Tile {
    static constexpr int kW = D / 32;  // 4-byte words of a K row per lane
    uint32_t k[2][kW];                 // rows 4 (m % 4) + m / 4 (+ 16): bytes 4 kW g ..
    uint32_t v[8];                     // word of key 4 j + g
    float sk, sv;                      // lane n of a row of lanes: key 4 (n % 8) + g
};

template <int D>
__global__ __launch_bounds__(512) void kv4_decode_kernel(Kv4Decode p) {
    constexpr int kRow = D / 2;         // bytes per cache row
    constexpr int NF = D / 16;          // fragments of O^T
    constexpr int kW = Kv4Tile<D>::kW;
    constexpr int kORow = D + 4;        // floats per row of O in LDS
    extern __shared__ __align__(16) float s_merge[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nw = blockDim.x >> 6;
    const int g = lane >> 4, m16 = lane & 15;

    // Block -> (sequence, split), key head and heads of it.  Blocks go to the 8 XCDs in turn;
    // the key heads of one piece of a sequence, whose pages lie side by side in memory, run one
    // after the other on one XCD (B = 1, 8 heads, 1000 positions: 9.0 us in 4 splits dealt out
    // head by head, 7.3 in 8, where that falls so by itself).
    const int heads_here = p.Hkv * p.groups;
    const int local = (int)blockIdx.x / 8;
    const int piece = local / heads_here * 8 + (int)blockIdx.x % 8;
    if (piece >= p.B * p.nsplit) return;
    const int b = piece / p.nsplit, split = piece % p.nsplit;
    const int kvh = local % heads_here / p.groups, grp = local % p.groups;
    const int per_kv = p.Hq / p.Hkv;
    const int rows = min(p.rows, per_kv - grp * p.rows);
    const int head0 = kvh * per_kv + grp * p.rows;  // first query head
    const int len = min(max(__builtin_amdgcn_readfirstlane(p.lens[b]), 0), p.max_context);
    const int tiles = (len + kTile - 1) / kTile;
    const int per_split = (tiles + p.nsplit - 1) / p.nsplit;
    const int t_begin = min(split * per_split, tiles), t_end = min(t_begin + per_split, tiles);
    const int32_t* __restrict__ table = p.tables + (size_t)b * p.max_pages;
    const int pmask = (1 << p.log2_page) - 1;

    // this lane's query row (lanes past the rows hold zeros) and -8 sum(q)
    const bool qok = m16 < rows;
    const size_t qrow = (size_t)b * p.Hq + head0 + min(m16, rows - 1);
    uint32_t qlo[kW], qhi[kW];  // even and odd elements of 8 kW consecutive ones
    int qsum = 0;
    {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p.Q + qrow * D) + 2 * kW * g;
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const uint32_t a = qok ? q[2 * w] : 0u, c = qok ? q[2 * w + 1] : 0u;
            qlo[w] = __builtin_amdgcn_perm(c, a, 0x06040200u);
            qhi[w] = __builtin_amdgcn_perm(c, a, 0x07050301u);
            qsum = __builtin_amdgcn_sdot4((int)a, 0x01010101, qsum, false);
            qsum = __builtin_amdgcn_sdot4((int)c, 0x01010101, qsum, false);
        }
        const auto s16 = __builtin_amdgcn_permlane16_swap(qsum, qsum, false, false);
        qsum = (int)(s16[0] + s16[1]);
        const auto s32 = __builtin_amdgcn_permlane32_swap(qsum, qsum, false, false);
        qsum = -8 * (int)(s32[0] + s32[1]);
    }
    const float qs = qok ? p.sQ[qrow] * p.qk : 0.f;

    // lane offsets inside 16 rows
    const uint32_t k_off = (uint32_t)(4 * (m16 & 3) + (m16 >> 2)) * kRow + 4 * kW * g;
    const uint32_t v_off = (uint32_t)g * kRow + 4 * (D == 128 ? m16 : m16 & 7);
    const int s_off = 4 * (m16 & 3) + g;        // row of this lane's scales inside its 16
    const bool s_upper = (m16 & 4) != 0;        // they lie in the second 16 keys
    bool bad = false;

    // The two runs of 16 rows of tile t: their page ids (a page holds whole runs; entries past
    // the length are not read), and from those the first row of each.  The ids are read a tile
    // before the rows are needed, which is a tile before the data is: nothing waits on them.
    const bool two_pages = p.log2_page == 4;
    int id0 = 0, id1 = 0;
    auto fetch_ids = [&](int t) {
        if (t >= t_end) return;
        id0 = table[(t * kTile) >> p.log2_page];
        if (two_pages) id1 = table[min(t * kTile + 16, len - 1) >> p.log2_page];
    };
    size_t row0 = 0, row1 = 0;
    auto rows_of_ids = [&](int t) {
        if (t >= t_end) return;
        auto first = [&](int raw, int key) {
            const int page = (int)min((unsigned)raw, (unsigned)(p.num_pages - 1));
            bad = bad || page != raw;
            return (((size_t)page * p.Hkv + kvh) << p.log2_page) + (size_t)(key & pmask);
        };
        const int raw0 = __builtin_amdgcn_readfirstlane(id0);
        row0 = first(raw0, t * kTile);
        row1 = row0 + 16;
        if (two_pages) row1 = first(__builtin_amdgcn_readfirstlane(id1), t * kTile + 16);
    };
    auto load = [&](Kv4Tile<D>& r) {
        const size_t first = row0, second = row1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const size_t row = h == 0 ? first : second;
            const uint8_t* kb = p.K + row * kRow + k_off;
            if constexpr (kW == 4) {
                const v4u w = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(kb));
                r.k[h][0] = w.x, r.k[h][1] = w.y, r.k[h][2] = w.z, r.k[h][3] = w.w;
            } else {
                const v2u w = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(kb));
                r.k[h][0] = w.x, r.k[h][1] = w.y;
            }
            const uint8_t* vb = p.V + row * kRow + v_off;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r.v[4 * h + j] =
                    __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vb + 4 * j * kRow));
        }
        const size_t srow = (s_upper ? second : first) + s_off;
        r.sk = __builtin_nontemporal_load(p.sK + srow);
        r.sv = __builtin_nontemporal_load(p.sV + srow);
    };

    v4f o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = v4f{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // bytes of two keys' words: b0/b1 are this lane's byte pair at D = 64 (dims 4..7 of the
    // word for the upper 8 rows of the fragment)
    uint32_t sel[D == 128 ? 4 : 2];
#pragma unroll
    for (int i = 0; i < (D == 128 ? 4 : 2); ++i) {
        const uint32_t byte = D == 128 ? i : i + (m16 & 8 ? 2 : 0);
        sel[i] = byte | 0x0c000c00u | ((4u + byte) << 16);
    }

    auto compute = [&](const Kv4Tile<D>& r, int t) {
        v4i sa[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sa[h] = v4i{qsum, qsum, qsum, qsum};
            if constexpr (D == 128) {
                v4i lo, hi, ql, qh;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    lo[w] = (int)(r.k[h][w] & 0x0f0f0f0fu);
                    hi[w] = (int)((r.k[h][w] >> 4) & 0x0f0f0f0fu);
                    ql[w] = (int)qlo[w];
                    qh[w] = (int)qhi[w];
                }
                sa[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, ql, sa[h], 0, 0, 0);
                sa[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, qh, sa[h], 0, 0, 0);
            } else {
                const v4i a = {(int)(r.k[h][0] & 0x0f0f0f0fu), (int)(r.k[h][1] & 0x0f0f0f0fu),
                               (int)((r.k[h][0] >> 4) & 0x0f0f0f0fu),
                               (int)((r.k[h][1] >> 4) & 0x0f0f0f0fu)};
                const v4i q = {(int)qlo[0], (int)qlo[1], (int)qhi[0], (int)qhi[1]};
                sa[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, q, sa[h], 0, 0, 0);
            }
        }
        // u_j = q . k_j sK_j of key 4 j + g
        const float skj[8] = {bcast16<0>(r.sk), bcast16<1>(r.sk), bcast16<2>(r.sk), bcast16<3>(r.sk),
                              bcast16<4>(r.sk), bcast16<5>(r.sk), bcast16<6>(r.sk), bcast16<7>(r.sk)};
        const float svj[8] = {bcast16<0>(r.sv), bcast16<1>(r.sv), bcast16<2>(r.sv), bcast16<3>(r.sv),
                              bcast16<4>(r.sv), bcast16<5>(r.sv), bcast16<6>(r.sv), bcast16<7>(r.sv)};
        float u[8], w[8], pj[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = static_cast<float>(sa[j >> 2][j & 3]) * skj[j];
        auto weights = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                pj[j] = fast_exp2(fmaf(u[j], qs, -m));
                w[j] = pj[j] * svj[j];
            }
        };
        auto sum8 = [&]() {
            return ((pj[0] + pj[1]) + (pj[2] + pj[3])) + ((pj[4] + pj[5]) + (pj[6] + pj[7]));
        };
        const bool partial = t * kTile + kTile > len;  // wave-uniform
        float psum = 0.f;
        bool slow = partial;
        if (!partial) {
            weights();
            psum = sum8();
            float wide = fmaxf(fabsf(w[0]), fabsf(w[1]));
#pragma unroll
            for (int j = 2; j < 8; j += 2) wide = fmaxf(wide, fmaxf(fabsf(w[j]), fabsf(w[j + 1])));
            // (the first tile, whose m is -inf, has an infinite sum)
            slow = __ballot(fmaxf(wide, psum * (kMaxWeight / kMaxSum)) > kMaxWeight) != 0;
        }
        if (slow) {
            // the exact maximum, then the largest weight under it
            float top = -INFINITY, pm = 0.f;
            bool seen[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                seen[j] = t * kTile + 4 * j + g < len;
                if (seen[j]) top = fmaxf(top, u[j] * qs);
            }
            top = max_groups(top);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (seen[j]) pm = fmaxf(pm, fabsf(fast_exp2(fmaf(u[j], qs, -base)) * svj[j]));
            pm = max_groups(pm);
            int e = 0;
            if (pm > 0.f && pm < INFINITY) frexpf(pm, &e);
            const float m_new = fmaxf(m, top + (float)min(max(e - kTopExp, -kMaxShift), kMaxShift));
            const float alpha = fast_exp2(m - (m_new == -INFINITY ? 0.f : m_new));
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[f][i] *= alpha;
            weights();
#pragma unroll
            for (int j = 0; j < 8; ++j)  // rows behind the length may hold anything
                if (!seen[j]) pj[j] = w[j] = 0.f;
            psum = sum8();
        }
        l += psum;
        // p sV as two fp16, 22 bits of it down to 2^-3 (2^-12 of the largest): in one, the
        // rounding of a row's largest weights outweighs that of the output (error against 64
        // bits 1.3 to 1.6 times the plain form's, 1.0 so; the matrix units have the time)
        v8h pw, pr;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            pw[j] = (_Float16)w[j];
            pr[j] = (_Float16)(w[j] - (float)pw[j]);
        }
        if (slow) {  // (a weight past fp16's range, by an infinite value scale, leaves no rest)
#pragma unroll
            for (int j = 0; j < 8; ++j) pr[j] = fabsf(w[j]) < 65520.f ? pr[j] : (_Float16)0.f;
        }
        // codes of a byte of two keys: 0x6400 | n is 1024 + n in fp16 and 0x6400 | 16 n is
        // 1024 + 16 n, both exact, as are the sums below
        uint32_t magic = 0x64006400u;
        asm("" : "+v"(magic));  // in a register: with a literal mask, v_and_or_b32 takes no second literal
        const h2 low_bias = {(_Float16)-1032.f, (_Float16)-1032.f};
        const h2 high_scale = {(_Float16)0.0625f, (_Float16)0.0625f};
        const h2 high_bias = {(_Float16)-72.f, (_Float16)-72.f};
#pragma unroll
        for (int i = 0; i < NF / 2; ++i) {
            v8h lo, hi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t c = __builtin_amdgcn_perm(r.v[2 * j + 1], r.v[2 * j], sel[i]);
                const h2 a = __builtin_bit_cast(h2, (c & 0x000f000fu) | magic) + low_bias;
                const h2 d = __builtin_elementwise_fma(
                    __builtin_bit_cast(h2, (c & 0x00f000f0u) | magic), high_scale, high_bias);
                lo[2 * j] = a.x, lo[2 * j + 1] = a.y;
                hi[2 * j] = d.x, hi[2 * j + 1] = d.y;
            }
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pw, o[2 * i], 0, 0, 0);
            o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pw, o[2 * i + 1], 0, 0, 0);
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pr, o[2 * i], 0, 0, 0);
            o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pr, o[2 * i + 1], 0, 0, 0);
        }
    };

    {
        int t = t_begin + wave;
        Kv4Tile<D> ra, rb;
        // Data of tile t in ra, rows of tile t + nw, ids of tile t + 2 nw.  The loads are not
        // conditional: past the last tile they repeat its rows (in a branch, the wait for
        // this tile's data would have to cover the next one's as well).
        fetch_ids(t);
        rows_of_ids(t);
        fetch_ids(t + nw);
        if (t < t_end) load(ra);
        rows_of_ids(t + nw);
        fetch_ids(t + 2 * nw);
        while (t < t_end) {
            load(rb);
            rows_of_ids(t + 2 * nw);
            fetch_ids(t + 3 * nw);
            __builtin_amdgcn_sched_barrier(0);
            compute(ra, t);
            t += nw;
            if (t >= t_end) break;
            load(ra);
            rows_of_ids(t + 2 * nw);
            fetch_ids(t + 3 * nw);
            __builtin_amdgcn_sched_barrier(0);
            compute(rb, t);
            t += nw;
        }
    }
    if (bad && lane == 0) atomicAdd(&g_kv4_bad_ids, 1u);

    // Join the waves: m, l and O of each row go to LDS, then element by element.
    // Layout: [wave][m, l of 16 rows][rows][kORow].
    l = sum_groups(l);
    const int wave_words = 2 * kMaxRows + p.rows * kORow;
    float* mine = s_merge + wave * wave_words;
    if (qok) {
        if (g == 0) mine[m16] = m, mine[kMaxRows + m16] = l;
        float* orow = mine + 2 * kMaxRows + m16 * kORow;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int mr = 4 * g + i;  // row of the fragment: dims d0 ..
            const int d0 = D == 128 ? 8 * mr : 8 * (mr & 7) + 4 * (mr >> 3);
#pragma unroll
            for (int f = 0; f < NF; f += 4)
                *reinterpret_cast<float4*>(orow + d0 + f) =
                    make_float4(o[f][i], o[f + 1][i], o[f + 2][i], o[f + 3][i]);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * D; e += blockDim.x) {
        const int row = e / D, d = e % D;
        float top = -INFINITY, sum = 0.f, acc = 0.f;
        for (int w = 0; w < nw; ++w) top = fmaxf(top, s_merge[w * wave_words + row]);
        const float use = top == -INFINITY ? 0.f : top;
        for (int w = 0; w < nw; ++w) {
            const float* q = s_merge + w * wave_words;
            const float a = fast_exp2(q[row] - use);
            sum += q[kMaxRows + row] * a;
            acc += q[2 * kMaxRows + row * kORow + d] * a;
        }
        const size_t orow = (size_t)b * p.Hq + head0 + row;
        if (p.nsplit == 1) {
            p.out[orow * D + d] = len > 0 ? __half_as_ushort(f16_of_f32(acc / sum)) : (uint16_t)0;
        } else {
            const size_t part = orow * p.nsplit + split;
            if (d == 0) p.part_ml[2 * part] = top, p.part_ml[2 * part + 1] = sum;
            p.part_acc[part * D + d] = acc;
        }
    }
}

// Joins the splits of each row, one thread per dim: eight partials in flight at a time (slots
// past the last repeat it with weight zero; one at a time, six splits took 2 us more than
// eight).
template <int D>
__global__ __launch_bounds__(D) void kv4_combine_kernel(const float* __restrict__ ml,
                                                        const float* __restrict__ acc,
                                                        const int32_t* __restrict__ lens,
                                                        uint16_t* __restrict__ out, int Hq,
                                                        int nsplit) {
    const size_t row = blockIdx.x;
    const int d = threadIdx.x;
    const float2* r = reinterpret_cast<const float2*>(ml) + row * nsplit;
    const float* x = acc + row * nsplit * D + d;
    const int len = lens[blockIdx.x / Hq];
    float m = -INFINITY, sum = 0.f, a = 0.f;
    for (int i0 = 0; i0 < nsplit; i0 += 8) {
        float2 s[8];
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(i0 + k, nsplit - 1);
            s[k] = r[i];
            v[k] = x[(size_t)i * D];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, s[k].x);
        const float use = top == -INFINITY ? 0.f : top;
        const float keep = fast_exp2(m - use);
        sum *= keep;
        a *= keep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = i0 + k < nsplit ? fast_exp2(s[k].x - use) : 0.f;
            // (a repeated slot must not turn an infinite partial into NaN)
            sum += i0 + k < nsplit ? s[k].y * f : 0.f;
            a += i0 + k < nsplit ? v[k] * f : 0.f;
        }
        m = top;
    }
    out[row * D + d] = len > 0 ? __half_as_ushort(f16_of_f32(a / sum)) : (uint16_t)0;
}

struct Kv4Plan {
    int groups, rows, waves, nsplit;
    size_t lds(int D) const { return (size_t)waves * (2 * kMaxRows + rows * (D + 4)) * 4; }
};

// Waves per block and splits of a sequence with the least estimated time (0.01 us) for
// sequences of max_context.  A wave takes 0.63 us per tile alone on its SIMD and 0.12 us per
// wave resident on the CU where they share it (16: the rate of memory); a round of blocks
// costs 2 us of first loads and merging, a second kernel 1 us, 0.05 per split and the partials' traffic.
// Few blocks per CU end unevenly when the sequences differ in length (12% / blocks).
// Estimated / measured, us: B32, 8 key heads of 128, 16K positions, 4 splits of 4 waves
// 70 / 68, 8 of 4 72 / 72; B1 32K, 32 of 8 12 / 14, 16 of 8 16 / 16, one of 8 128 / 123; B8 8K,
// 4 of 8 16 / 16; B64 2K, one of 4 22 / 22, 2 of 4 24 / 25; B64 300, one of 4 9.4 / 9.2, of 8
// 10.3 / 10.3.
Kv4Plan kv4_plan(int B, int Hq, int Hkv, int max_context) {
    Kv4Plan pl{};
    const int per_kv = Hq / Hkv;
    pl.groups = (per_kv + kMaxRows - 1) / kMaxRows;
    pl.rows = (per_kv + pl.groups - 1) / pl.groups;
    pl.groups = (per_kv + pl.rows - 1) / pl.rows;
    const long long units = (long long)B * Hkv * pl.groups;
    const long long tiles = ceil_div(max_context, kTile);
    constexpr int kCus = 256, kResident = 16;  // waves per CU
    const int max_split = (int)std::min<long long>(64, std::max<long long>(1, 1024 / units));
    pl.nsplit = 1, pl.waves = 4;
    long long best = -1;
    for (int s : {1, 2, 3, 4, 5, 6, 8, 11, 16, 24, 32, 48, 64}) {
        if (s > max_split || s > tiles) break;
        for (int w : {4, 8}) {
            const long long blocks = units * s;
            const long long waves = ceil_div(blocks, kCus) * w;  // per CU
            const long long resident = std::min<long long>(waves, kResident);
            const long long rounds = ceil_div(waves, kResident);
            const long long tile = std::max<long long>(63, 12 * resident);
            long long time = rounds * (200 + ceil_div(ceil_div(tiles, s), w) * tile);
            if (blocks >= kCus) time += time * 12 * kCus / (100 * blocks);
            if (s > 1) time += 100 + 5 * s + blocks / 10;
            if (best < 0 || time < best) best = time, pl.nsplit = s, pl.waves = w;
        }
    }
    return pl;
}

int log2_of(int page) {
    int l = 0;
    while ((1 << l) < page) ++l;
    return l;
}

bool page_ok(int page) { return page >= 16 && page <= 1024 && (page & (page - 1)) == 0; }

template <typename F>
void with_head_dim(int D, F&& f) {
    if (D == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

struct Kv4Partials {
    size_t ml_bytes, bytes;
};
Kv4Partials kv4_partials(size_t parts, int D) {
    if (parts == 0) return {0, 0};
    const size_t ml = round_up(parts * 2 * sizeof(float), kWorkspaceAlign);
    return {ml, ml + round_up(parts * D * sizeof(float), kWorkspaceAlign)};
}

// Shared checks of the cache's shape: INT8K_OK or the status to return.
int check_cache(int num_pages, int page_size, int kv_heads, int head_dim) {
    if (num_pages <= 0 || kv_heads <= 0) return INT8K_ERR_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return INT8K_ERR_UNSUPPORTED;
    if (!page_ok(page_size)) return INT8K_ERR_UNSUPPORTED;
    // slots are int32
    if ((long long)num_pages * page_size > 0x7fffffffLL) return INT8K_ERR_UNSUPPORTED;
    if ((long long)num_pages * page_size >= (1LL << 40) / ((long long)kv_heads * head_dim))
        return INT8K_ERR_UNSUPPORTED;
    return INT8K_OK;
}

}  // namespace
}  // namespace int8k

using namespace int8k;

extern "C" int int8k_kv4_cache_append(const void* k_new, const void* v_new, int dtype,
                                      long long k_token_stride, long long k_head_stride,
                                      long long v_token_stride, long long v_head_stride,
                                      uint8_t* K_pages, uint8_t* V_pages, float* sK_pages,
                                      float* sV_pages, const int32_t* slots, int T, int kv_heads,
                                      int head_dim, int num_pages, int page_size, void* stream) {
    clear_last_error();
    if (!k_new || !v_new || !K_pages || !V_pages || !sK_pages || !sV_pages || !slots)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (T <= 0 || dtype < INT8K_DTYPE_F16 || dtype > INT8K_DTYPE_F32)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_cache(num_pages, page_size, kv_heads, head_dim)) return st;
    const int w = dtype == INT8K_DTYPE_F32 ? 4 : 8;  // elements per 16 bytes
    for (long long s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
        if (s % w) return INT8K_ERR_MISALIGNED;
    if (!aligned_to(k_new, 16) || !aligned_to(v_new, 16) || !aligned_to(K_pages, 16) ||
        !aligned_to(V_pages, 16) || !aligned_to(sK_pages, 4) || !aligned_to(sV_pages, 4) ||
        !aligned_to(slots, 4))
        return INT8K_ERR_MISALIGNED;
    // several rows per lane group once the waves of one row each no longer fit the GPU at once
    const int rows = 256 / (head_dim / 8);
    const bool four = ceil_div(T, rows) * kv_heads >= 2048;
    const long long blocks = ceil_div(T, four ? 4 * rows : rows) * kv_heads;
    if (blocks >= (1LL << 23)) return INT8K_ERR_UNSUPPORTED;
    const Kv4Side k{k_new, k_token_stride, k_head_stride, K_pages, sK_pages};
    const Kv4Side v{v_new, v_token_stride, v_head_stride, V_pages, sV_pages};
    const dim3 grid((unsigned)blocks, 2);
    with_dtype(dtype, [&](auto dt) {
        with_head_dim(head_dim, [&](auto d) {
            constexpr int DT = decltype(dt)::value, D = decltype(d)::value;
            if (four)
                kv4_append_kernel<DT, D, 4><<<grid, 256, 0, as_stream(stream)>>>(
                    k, v, slots, T, kv_heads, num_pages, log2_of(page_size));
            else
                kv4_append_kernel<DT, D, 1><<<grid, 256, 0, as_stream(stream)>>>(
                    k, v, slots, T, kv_heads, num_pages, log2_of(page_size));
        });
    });
    return check_launch("kv4_append_kernel");
}

extern "C" int int8k_kv4_cache_read(const uint8_t* pages, const float* scales,
                                    const int32_t* slots, void* out, int dtype, int T,
                                    int kv_heads, int head_dim, int num_pages, int page_size,
                                    void* stream) {
    clear_last_error();
    if (!pages || !scales || !slots || !out) return INT8K_ERR_INVALID_ARGUMENT;
    if (T <= 0 || dtype < INT8K_DTYPE_F16 || dtype > INT8K_DTYPE_F32)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_cache(num_pages, page_size, kv_heads, head_dim)) return st;
    if (!aligned_to(pages, 16) || !aligned_to(scales, 4) || !aligned_to(slots, 4) ||
        !aligned_to(out, 16))
        return INT8K_ERR_MISALIGNED;
    const long long blocks = ceil_div(T, 256 / (head_dim / 8)) * kv_heads;
    if (blocks >= (1LL << 23)) return INT8K_ERR_UNSUPPORTED;
    with_dtype(dtype, [&](auto dt) {
        with_head_dim(head_dim, [&](auto d) {
            kv4_read_kernel<decltype(dt)::value, decltype(d)::value>
                <<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(
                    pages, scales, slots, out, T, kv_heads, num_pages, log2_of(page_size));
        });
    });
    return check_launch("kv4_read_kernel");
}

extern "C" size_t int8k_decode_attention_kv4_paged_workspace_bytes(int B, int heads, int kv_heads,
                                                                   int max_context, int head_dim) {
    if (B <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_context <= 0 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    // b sequences are split into at most min(64, 1024 / (b units)) each, and b of them into no
    // more than min(64 b, 1024 / units) together: that grows with b, where the plan's own need does not
    const Kv4Plan pl = kv4_plan(1, heads, kv_heads, max_context);
    const long long splits = 1024 / ((long long)kv_heads * pl.groups);
    if (splits < 2) return 0;
    return kv4_partials((size_t)heads * std::min(64LL * B, splits), head_dim).bytes;
}

extern "C" int int8k_decode_attention_forward_kv4_paged(
    const int8_t* Q, const uint8_t* K_pages, const uint8_t* V_pages, uint16_t* out,
    const float* scale_Q, const float* sK_pages, const float* sV_pages,
    const int32_t* block_tables, const int32_t* context_lens, int B, int heads, int kv_heads,
    int head_dim, int num_pages, int page_size, int max_pages_per_seq, int max_context,
    void* workspace, size_t workspace_bytes, void* stream) {
    clear_last_error();
    if (!Q || !K_pages || !V_pages || !out || !scale_Q || !sK_pages || !sV_pages ||
        !block_tables || !context_lens)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (B <= 0 || heads <= 0 || max_pages_per_seq <= 0 || max_context <= 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_cache(num_pages, page_size, kv_heads, head_dim)) return st;
    if (heads % kv_heads || (long long)max_context > (long long)max_pages_per_seq * page_size)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!aligned_to(Q, 16) || !aligned_to(K_pages, 16) || !aligned_to(V_pages, 16) ||
        !aligned_to(scale_Q, 4) || !aligned_to(sK_pages, 4) || !aligned_to(sV_pages, 4) ||
        !aligned_to(block_tables, 4) || !aligned_to(context_lens, 4) || !aligned_to(out, 8))
        return INT8K_ERR_MISALIGNED;
    // (positions, a few tiles past the last among them, are int)
    if ((long long)B * heads >= (1LL << 22) || max_context > (1 << 30)) return INT8K_ERR_UNSUPPORTED;
    const Kv4Plan pl = kv4_plan(B, heads, kv_heads, max_context);
    const Kv4Partials part =
        kv4_partials(pl.nsplit > 1 ? (size_t)B * heads * pl.nsplit : 0, head_dim);
    if (part.bytes > 0) {
        if (!workspace || workspace_bytes < part.bytes) return INT8K_ERR_WORKSPACE;
        if (!aligned_to(workspace, 16)) return INT8K_ERR_MISALIGNED;
    }
    const long long blocks = ceil_div((long long)B * pl.nsplit, 8) * 8 * kv_heads * pl.groups;
    if (blocks * pl.waves >= (1LL << 26)) return INT8K_ERR_UNSUPPORTED;  // work-items below 2^32
    Kv4Decode p{};
    p.Q = Q, p.K = K_pages, p.V = V_pages, p.sQ = scale_Q, p.sK = sK_pages, p.sV = sV_pages;
    p.tables = block_tables, p.lens = context_lens, p.out = out;
    p.part_ml = static_cast<float*>(workspace);
    p.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + part.ml_bytes);
    p.B = B, p.Hq = heads, p.Hkv = kv_heads, p.num_pages = num_pages, p.log2_page = log2_of(page_size);
    p.max_pages = max_pages_per_seq, p.max_context = max_context;
    p.groups = pl.groups, p.rows = pl.rows, p.nsplit = pl.nsplit;
    p.qk = (1.0f / std::sqrt((float)head_dim)) * kLog2e;
    int st = INT8K_OK;
    with_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        static PerDeviceOnce once;
        st = once.run([] {
            const hipError_t e = hipFuncSetAttribute(
                reinterpret_cast<const void*>(&kv4_decode_kernel<D>),
                hipFuncAttributeMaxDynamicSharedMemorySize, 8 * (2 * kMaxRows + kMaxRows * (D + 4)) * 4);
            if (e == hipSuccess) return (int)INT8K_OK;
            set_last_error("hipFuncSetAttribute", e);
            return (int)INT8K_ERR_HIP;
        });
        if (st != INT8K_OK) return;
        kv4_decode_kernel<D><<<(unsigned)blocks, 64 * pl.waves, pl.lds(D), as_stream(stream)>>>(p);
        st = check_launch("kv4_decode_kernel");
        if (st != INT8K_OK || pl.nsplit == 1) return;
        kv4_combine_kernel<D><<<(unsigned)(B * heads), D, 0, as_stream(stream)>>>(
            p.part_ml, p.part_acc, context_lens, out, heads, pl.nsplit);
        st = check_launch("kv4_combine_kernel");
    });
    return st;
}

extern "C" int int8k_kv4_bad_ids(unsigned int* count) {
    clear_last_error();
    if (!count) return INT8K_ERR_INVALID_ARGUMENT;
    const hipError_t e = hipMemcpyFromSymbol(count, HIP_SYMBOL(g_kv4_bad_ids),
                                             sizeof(unsigned int), 0, hipMemcpyDeviceToHost);
    if (e != hipSuccess) {
        set_last_error("hipMemcpyFromSymbol(g_kv4_bad_ids)", e);
        return INT8K_ERR_HIP;
    }
    return INT8K_OK;
}
