// paged.hip — attention over the paged INT8 cache with grouped heads: a tree of drafted tokens per
// sequence, and one token per sequence over selected blocks; gfx950.
//
//   Q int8 [B, Hq, N, D], scales [B * Hq * N]; the N tokens of sequence b lie in the cache at
//   positions len_b .. len_b + count_b - 1 (count_b <= N).  Token i sees every position below
//   len_b and those len_b + j whose bit j is set in its mask (without masks: j <= i).
//   out = sum_j softmax_j(q . k_j sQ sK_j / sqrt(D)) v_j sV_j, q . k exact int32
//
// The query rows of a key head (its Hq / Hkv heads times N tokens, which lie side by side in Q)
// share its keys: F fragments of 16 of them are the columns of MFMA tiles over 32 positions,
//   S^T[32 keys x 16 q] = K . Q^T    v_mfma_i32_16x16x64_i8
//   O^T[D x 16 q]      += V^T . P^T  v_mfma_f32_16x16x32_f16, V as exact fp16
// In the accumulator layout lane l holds query l % 16 and rows 4 (l / 16) + r.  Rows are keys in
// the order 4 (m % 4) + m / 4, so lane group g = l / 16 ends up with the scores of keys 4 j + g,
// j = 0..7, as the B operand of the second product wants them: P never changes lanes.  The A
// operand of that product is 8 keys of one dim per lane: lane l reads D / 16 bytes of those 8
// rows and picks a byte of two keys at a time (v_perm), which an XOR and a packed addition turn
// into two fp16.  K passes through LDS, where a wave's loads of whole lines become that layout.
// A wave takes one or two fragments of every 8th tile of a piece of a sequence, and the 8 waves of
// a block are joined in LDS; or, where a key head has many rows, R = 4 or 8 waves take two
// fragments each of the same tiles, which they load and convert in turn and share through LDS: two
// such slices of a block, joined, or one, whose waves write what they hold.
// Pieces are joined by a second kernel.
//
// With one fragment it reads 5.2 TB/s (8 sequences of 16384, one token of 4 heads on 8), as fast as a
// copy moves data here and three quarters of what a kernel that only reads reaches.  With two, a CU
// that has work is bound by the issue of instructions: 32 rows x 32 keys take 300 vector instructions
// (190 with R = 8: V's conversion is shared) beside 44 MFMAs, each of which keeps the SIMD from
// vector ones for about 10 of its 16 cycles.  Unequal lengths come on top: 16 sequences of up to
// 8192 with trees of 16, 32 heads on 8 of 128, take 65 to 67 us (2.7 TB/s, 0.32 PFLOP/s), one whole
// sequence of a key head and 32 rows per block, and a CU is busy for 66% of that; 16 that are all of
// 8192 take 71.  4 of up to 16320 with trees of 64: 89 to 99 us on different cards (0.43 to 0.48
// PFLOP/s; 115 with R = 1), 9 of them the join.
//
// p_j = 2^(s_j - m) with a reference m per query that is not the running maximum: it is set so
// that the largest weight p sV of the tile that set it lies in [2^9, 2^10), and a tile whose
// weights stay in fp16's range under the current m needs no exchange between lanes and no
// rescaling.  l sums p and O the weighted codes, both in fp32.  A weight is carried as two fp16,
// its rounding and what that leaves (22 bits): in one, the rounding of a row's largest weights
// outweighs that of the output.  Below 2^-14 fp16 steps by 2^-24, so a weight is off by at most
// 2^-25 beside a largest one of 2^9 or more, and long flat tails add up.
#include <algorithm>
#include <cmath>

#include "pages.h"
#include "rows.h"

namespace int8k {
namespace {

__device__ unsigned int g_attend_bad_ids;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;               // positions per tile
constexpr int kWaves = 8;               // per block
constexpr float kMaxWeight = 60000.f;   // fp16 weights stay below it
constexpr float kMaxSum = 0x1p60f;      // and the sum of a lane's 8 p below this
constexpr int kMaxShift = 60;           // |m - running maximum| where m is set
constexpr int kTopExp = 10;             // the largest weight there: below 2^kTopExp

struct Attend {
    const int8_t *Q, *K, *V;
    const float *sQ, *sK, *sV;
    const int32_t* tables;               // page ids of sequence b and key head h:
    long long table_batch, table_head;   //   from b table_batch + h table_head
    const int32_t* lens;                 // [B]: positions before the tree
    bool tree;                           // the N tokens are in the cache behind those positions
    const int32_t* counts;               // tokens of each sequence, or null (N)
    const int64_t* mask;                 // [B or 1][N][words], or null
    long long mask_batch;
    int words;
    uint16_t* out;                       // [B, Hq, N, D], or [B, N, Hq, D] with bshd
    bool bshd;
    float *part_ml, *part_acc;           // [piece][Hq * N][2] and [..][D]
    int B, Hq, Hkv, N, num_pages, log2_page, max_context;
    int groups;                          // blocks per piece and key head
    int pieces, min_tiles;               // see Piece; 0: a sequence is one piece
    int slots;                           // pieces that the grid has room for
    float qk;
};

// What a sequence holds: `prefix` positions that every token sees, `total` with the tokens'.
struct Extent {
    int prefix, total, count;
};
__device__ __forceinline__ Extent extent_of(const Attend& p, int b) {
    Extent e;
    e.prefix = min(max(p.lens[b], 0), p.max_context);
    e.count = !p.tree ? 0 : p.counts == nullptr ? p.N : min(max(p.counts[b], 0), p.N);
    e.total = min(e.prefix + e.count, p.max_context);
    return e;
}

// The lowest n bits (none below 0, all from 32).
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

// Which of the nodes first .. first + 31 token `node` sees, bit by bit (`first` may be negative).
__device__ __forceinline__ uint32_t seen_nodes(const uint32_t* masks, int words, int node, int first) {
    if (masks == nullptr) return low_bits(node + 1 - first);
    const int w = first >> 5, shift = first & 31;
    const uint32_t* row = masks + (size_t)node * (2 * words);
    const uint32_t lo = w >= 0 && w < 2 * words ? row[w] : 0u;
    const uint32_t hi = w + 1 >= 0 && w + 1 < 2 * words ? row[w + 1] : 0u;
    return shift == 0 ? lo : lo >> shift | hi << (32 - shift);
}

// The mask words of sequence b, in halves, or null.
__device__ __forceinline__ const uint32_t* masks_of(const Attend& p, int b) {
    return p.mask == nullptr ? nullptr
                             : reinterpret_cast<const uint32_t*>(p.mask + b * p.mask_batch);
}

// Whether row `node` attends to any position (tokens past the sequence's do not).
__device__ __forceinline__ bool attends(const Attend& p, int b, int node, const Extent& e) {
    if (!p.tree) return e.prefix > 0;
    if (node >= e.count) return false;
    if (e.prefix > 0) return true;
    const uint32_t* masks = masks_of(p, b);
    uint32_t any = 0;
    for (int j = 0; j < e.total; j += 32)
        any |= seen_nodes(masks, p.words, node, j) & low_bits(e.total - j);
    return any != 0;
}

// How the sequences are cut, where the plan cuts them.  Their lengths are on the device, so every wave
// works the cut out from them: into p.pieces pieces over all sequences, at least one each, whose
// largest is about as small as can be, but p.min_tiles.  The host takes as many pieces as the GPU
// holds at a time, so all blocks run at once and end about together.  A plan that does not cut (it
// knows max_context only) takes as long as its longest sequence: one of 8192 beside 15 of 256, with
// trees of 16, 58 us where 16 of up to 8192 take 65.
struct Piece {
    int b, index, count, first;  // sequence, which of its pieces, how many, number of its first
    int tiles;                   // of a piece
};

__device__ __forceinline__ int wave_sum(int v) {
    v = group8_sum(v);
    v += dpp_row_mirror(v);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = (int)(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane((int)(b[0] + b[1]));
}

// The piece that `found(first, count, b)` picks among the sequences (for one of them at most).
template <typename Found>
__device__ __forceinline__ bool find_piece(const Attend& p, Piece& piece, Found&& found) {
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int b) {
        return b < p.B ? (extent_of(p, b).total + kTile - 1) / kTile : 0;
    };
    int mine = tiles_of(lane), all = mine;
    for (int b = lane + 64; b < p.B; b += 64) all += tiles_of(b);
    const unsigned total = (unsigned)wave_sum(all), P = (unsigned)p.pieces;
    auto count_of = [&](unsigned tiles, unsigned each) { return max((tiles + each - 1) / each, 1u); };
    // pieces of total / (P - B) are few enough, of less than total / P too many
    unsigned lo = max((total + P - 1) / P, 1u), hi = max((total + P - p.B - 1) / (P - p.B), 1u);
    for (int step = 0; step < 6 && lo < hi; ++step) {
        const unsigned mid = (lo + hi) / 2;
        int count = lane < p.B ? (int)count_of(mine, mid) : 0;
        for (int b = lane + 64; b < p.B; b += 64) count += (int)count_of(tiles_of(b), mid);
        if ((unsigned)wave_sum(count) <= P) hi = mid;
        else lo = mid + 1;
    }
    const unsigned each = max(hi, (unsigned)p.min_tiles);
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        if (b0 > 0) mine = tiles_of(b0 + lane);
        const int count = b0 + lane < p.B ? (int)count_of(mine, each) : 0;
        int upto = count;  // inclusive sum over the lanes
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int below = __shfl_up(upto, d);
            upto += lane >= d ? below : 0;
        }
        const int first = before + upto - count;
        const uint64_t at = __ballot(count > 0 && found(first, count, b0 + lane));
        if (at != 0) {
            const int src = __builtin_ctzll(at);
            piece.b = b0 + src;
            piece.count = __builtin_amdgcn_readlane(count, src);
            piece.tiles = __builtin_amdgcn_readlane((mine + count - 1) / max(count, 1), src);
            piece.first = __builtin_amdgcn_readlane(first, src);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

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

// Four dims of an output row, acc / sum; a row that attends to nothing is zero.
__device__ __forceinline__ void store_row(const Attend& p, size_t at, const float4& acc, float sum,
                                          bool any) {
    float v[4] = {acc.x / sum, acc.y / sum, acc.z / sum, acc.w / sum};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("" : "+v"(v[i]));  // (see f16_of_f32)
    *reinterpret_cast<uint2*>(p.out + at) =
        any ? make_uint2(pack_pair<INT8K_DTYPE_F16>(v[0], v[1]), pack_pair<INT8K_DTYPE_F16>(v[2], v[3]))
            : make_uint2(0, 0);
}

// A partial row is stored in the order in which lanes hold it, four dims at a time: four lanes (g) of
// a row write 64 bytes.  The first dim of its float4 `at`.
template <int D>
__device__ __forceinline__ int part_dim(int at) {
    constexpr int NF = D / 16;
    const int g = at & 3, i = at / 4 % (NF / 4), c = at / NF;
    return NF * (4 * g + c) + 4 * i;
}

template <int D>
struct AttendTile {
    static constexpr int kV = D / 64;   // 4-byte words of a V row per lane
    uint32_t v[8][kV];                  // key 4 j + g: bytes D / 16 m ..
    float sk[2], sv[2];                 // lane n of a row of lanes: key 4 (n % 4) + g (+ 16)
};

// Where piece c (16 bytes) of K row r of 16 lies in LDS: pieces are exchanged inside runs of 256
// bytes, so that both the 16 lanes that write a run and those that read one piece of all 16 rows
// meet every bank once.
template <int D>
__device__ __forceinline__ uint32_t k_slot(int r, int c) {
    constexpr int C = D / 16, RP = 256 / D;
    return (r / RP) * 256 + ((r % RP) * C + (c ^ (r / RP % C))) * 16;
}

// F fragments of query rows per wave, W waves per block, of which R share their tiles.
template <int D, int F, int R, int W>
__global__ __launch_bounds__(64 * W, 2) void paged_attend_kernel(Attend p) {
    using Tile = AttendTile<D>;
    constexpr int NF = D / 16;          // fragments of O^T
    constexpr int KI = D / 64;          // loads of 1 KiB per 16 rows
    constexpr int MR = 16 * F;          // query rows per wave
    constexpr int BR = MR * R;          // and per block
    constexpr int kORow = D + 4;        // floats per row of O in LDS
    extern __shared__ __align__(16) float s_merge[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int nw = W;
    const int mine = wave & (R - 1), slice = wave / R;  // of the block's rows, and of its waves on them
    const int g = lane >> 4, m16 = lane & 15;

    // Block -> piece of a sequence, key head and rows of it.  Blocks go to the 8 XCDs in turn; each
    // XCD takes a run of the (piece, key head) pairs, and the blocks of one pair, which read the same
    // rows, one after the other.  (Whole sequences that lie in the batch by length load the XCDs
    // unequally: 64 of up to 4096 with trees of 16, 117 us shuffled, 137 with the longest first.)
    const int units = p.slots * p.Hkv, each_xcd = (units + 7) / 8;
    const int local = (int)blockIdx.x / 8 / p.groups;
    const int unit = (int)blockIdx.x % 8 * each_xcd + local;
    if (local >= each_xcd || unit >= units) return;
    const int number = unit / p.Hkv, kvh = unit % p.Hkv, grp = (int)blockIdx.x / 8 % p.groups;
    Piece piece{number, 0, 1, number, 0};
    if (p.pieces > 0) {
        if (!find_piece(p, piece, [&](int first, int count, int) {
                return number >= first && number < first + count;
            }))
            return;
        piece.index = number - piece.first;
    }
    const int b = piece.b;
    const int all_rows = p.Hq / p.Hkv * p.N;
    const int row0_q = grp * BR, rows = min(BR, all_rows - row0_q);
    const size_t first_row = ((size_t)b * p.Hq + (size_t)kvh * (p.Hq / p.Hkv)) * p.N + row0_q;
    Extent e = extent_of(p, b);
    e.prefix = __builtin_amdgcn_readfirstlane(e.prefix);
    e.total = __builtin_amdgcn_readfirstlane(e.total);
    const int tiles = (e.total + kTile - 1) / kTile;
    const int t_begin = piece.index * piece.tiles;
    const int t_end = piece.count == 1 ? tiles : min(t_begin + piece.tiles, tiles);
    const int32_t* __restrict__ table = p.tables + b * p.table_batch + kvh * p.table_head;
    const int pmask = (1 << p.log2_page) - 1;
    const uint32_t* masks = masks_of(p, b);

    // this lane's query row of each fragment (rows past the last hold zeros)
    v4i qf[F][KI];
    float qs[F];
    int node[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int r = min(MR * mine + 16 * f + m16, rows - 1);
        const bool ok = MR * mine + 16 * f + m16 < rows;
        node[f] = (row0_q + r) % p.N;
        qs[f] = ok ? p.sQ[first_row + r] * p.qk : 0.f;
#pragma unroll
        for (int i = 0; i < KI; ++i)
            qf[f][i] = ok ? *reinterpret_cast<const v4i*>(p.Q + (first_row + r) * D + 64 * i + 16 * g)
                          : v4i{0, 0, 0, 0};
    }

    // K goes through LDS, a tile of this wave's own: the MFMA wants piece g of 16 rows from 16 lanes
    // side by side, and loads in that order take four times as long as whole lines (46 against 11
    // cycles of a CU per KiB: the loads of a wave's tile 365 cycles, 225 so).
    char* s_k = reinterpret_cast<char*>(s_merge) + wave * (kTile * D);
    uint32_t k_write[KI], k_read[KI];
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        const int at = 64 * i + lane;  // piece of the 16 rows
        k_write[i] = k_slot<D>(at / NF, at % NF);
        k_read[i] = k_slot<D>(4 * (m16 & 3) + (m16 >> 2), 4 * i + g);
    }
    // lane offsets inside 16 rows
    const uint32_t v_off = (uint32_t)g * D + D / 16 * m16;
    const uint32_t s_off = 4 * (4 * (m16 & 3) + g);  // bytes of this lane's scales
    bool bad = false;

    // The two runs of 16 rows of tile t: their page ids (a page holds whole runs; entries past
    // the last position are not read), and from those their numbers in the cache (below 2^32 by
    // check_pages).  Past the last tile both stay as they are.
    const bool two_pages = p.log2_page == 4;
    int id[2] = {0, 0};
    auto fetch_ids = [&](int t) {
        if (t >= t_end) return;
        id[0] = table[(t * kTile) >> p.log2_page];
        if (two_pages) id[1] = table[min(t * kTile + 16, e.total - 1) >> p.log2_page];
    };
    struct Rows {
        uint32_t run[2];
    };
    auto rows_of_ids = [&](int t, Rows& rows) {
        if (t >= t_end) return;
        auto run = [&](int raw, int key) {
            const uint32_t page = min((uint32_t)raw, (uint32_t)(p.num_pages - 1));
            bad = bad || page != (uint32_t)raw;
            return ((page * (uint32_t)p.Hkv + (uint32_t)kvh) << (p.log2_page - 4)) + ((uint32_t)(key & pmask) >> 4);
        };
        rows.run[0] = run(__builtin_amdgcn_readfirstlane(id[0]), t * kTile);
        rows.run[1] = rows.run[0] + 1;
        if (two_pages) rows.run[1] = run(__builtin_amdgcn_readfirstlane(id[1]), t * kTile + 16);
    };
    v4i k_raw[2][KI], k[2][KI];  // a tile's rows as loaded, and as the MFMA takes them
    auto load_k = [&](const Rows& rows) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const __amdgpu_buffer_rsrc_t kb = make_buffer(p.K + (size_t)rows.run[h] * (16 * D), 16 * D);
#pragma unroll
            for (int i = 0; i < KI; ++i)
                k_raw[h][i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(kb, lane * 16, 1024 * i, 0));
        }
    };
    auto write_k = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < KI; ++i)
                *reinterpret_cast<v4i*>(s_k + h * 16 * D + k_write[i]) = k_raw[h][i];
    };
    auto read_k = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's LDS accesses are in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < KI; ++i)
                k[h][i] = *reinterpret_cast<const v4i*>(s_k + h * 16 * D + k_read[i]);
    };
    auto load_v = [&](Tile& r, const Rows& rows) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const size_t run = rows.run[h];
            const __amdgpu_buffer_rsrc_t vb = make_buffer(p.V + run * (16 * D), 16 * D);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (D == 128) {
                    const v2u w = __builtin_amdgcn_raw_buffer_load_b64(vb, v_off, 4 * j * D, 0);
                    r.v[4 * h + j][0] = w.x, r.v[4 * h + j][1] = w.y;
                } else {
                    r.v[4 * h + j][0] = __builtin_amdgcn_raw_buffer_load_b32(vb, v_off, 4 * j * D, 0);
                }
            }
            r.sk[h] = __builtin_bit_cast(
                float, __builtin_amdgcn_raw_buffer_load_b32(make_buffer(p.sK + run * 16, 64), s_off, 0, 0));
            r.sv[h] = __builtin_bit_cast(
                float, __builtin_amdgcn_raw_buffer_load_b32(make_buffer(p.sV + run * 16, 64), s_off, 0, 0));
        }
    };

    v4f o[F][NF];
    float m[F], l[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        m[f] = -INFINITY, l[f] = 0.f;
#pragma unroll
        for (int i = 0; i < NF; ++i) o[f][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    // byte c of two keys, c + 128 as an unsigned number u: 0x6400 | u is 1024 + u in fp16, and the
    // sum below exact
    auto v_of = [&](const Tile& r, int i) {
        const h2 bias = {(_Float16)-1152.f, (_Float16)-1152.f};
        const uint32_t byte = i & 3;
        v8h v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = __builtin_amdgcn_perm(r.v[2 * j + 1][i >> 2], r.v[2 * j][i >> 2],
                                                     byte | 0x0c000c00u | ((4u + byte) << 16));
            const h2 a = __builtin_bit_cast(h2, c ^ 0x64806480u) + bias;
            v[2 * j] = a.x, v[2 * j + 1] = a.y;
        }
        return v;
    };
    // a tile with scales sk[h] of this lane and svj[j] of key 4 j + g, and fragment i of V by v_at
    auto compute = [&](const float (&sk)[2], const float (&svj)[8], int t, auto next_k, auto v_at) {
        const bool partial = t * kTile + kTile > e.prefix;  // wave-uniform
        // the dot products of key 4 j + g, and sK sQ / sqrt(D) of it and this lane's query: an MFMA
        // over 4 x 4 blocks, the outer product of the lanes' key scales with their query scales
        float dot[F][8], scale[F][8];
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v4i a = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KI; ++i)
                    a = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[h][i], qf[f][i], a, 0, 0, 0);
                const v4f c = __builtin_amdgcn_mfma_f32_4x4x1f32(sk[h], qs[f], v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    dot[f][4 * h + j] = static_cast<float>(a[j]), scale[f][4 * h + j] = c[j];
            }
        v8h pw[F], pr[F];
        float w[F][8], psum[F];
        auto weights = [&](int f) {
            float pj[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                pj[j] = fast_exp2(fmaf(dot[f][j], scale[f][j], -m[f]));
                w[f][j] = pj[j] * svj[j];
            }
            psum[f] = ((pj[0] + pj[1]) + (pj[2] + pj[3])) + ((pj[4] + pj[5]) + (pj[6] + pj[7]));
        };
        // the weights as two fp16; one past fp16's range (checked where it may be: an infinite
        // value scale) leaves no rest
        auto split = [&](int f, auto checked) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const h2 top = __builtin_convertvector((f2){w[f][j], w[f][j + 1]}, h2);
                float rest0 = minus_half<0>(w[f][j], top), rest1 = minus_half<1>(w[f][j + 1], top);
                if constexpr (decltype(checked)::value) {
                    rest0 = fabsf(w[f][j]) < 65520.f ? rest0 : 0.f;
                    rest1 = fabsf(w[f][j + 1]) < 65520.f ? rest1 : 0.f;
                }
                const h2 rest = __builtin_convertvector((f2){rest0, rest1}, h2);
                pw[f][j] = top.x, pw[f][j + 1] = top.y;
                pr[f][j] = rest.x, pr[f][j + 1] = rest.y;
            }
        };
        bool slow = partial;
        if (!partial) {
            float wide = 0.f;
            bool past = false;
#pragma unroll
            for (int f = 0; f < F; ++f) {
                weights(f);
#pragma unroll
                for (int j = 0; j < 8; j += 2) wide = fmaxf(wide, fmaxf(fabsf(w[f][j]), fabsf(w[f][j + 1])));
                // (while m is -inf the sum is infinite, or NaN where a score is -inf too)
                past = past || !(psum[f] <= kMaxSum);
            }
            slow = __ballot(past || wide > kMaxWeight) != 0;
        }
        if (slow) {
            // the exact maximum, then the largest weight under it
#pragma unroll
            for (int f = 0; f < F; ++f) {
                uint32_t visible = ~0u;  // keys of the tile
                if (partial) {
                    const int first = t * kTile - e.prefix;  // node of the tile's first key
                    visible = low_bits(-first);
                    if (p.tree) visible |= seen_nodes(masks, p.words, node[f], first);
                    visible &= low_bits(e.total - t * kTile);
                }
                visible >>= g;
                float top = -INFINITY, pm = 0.f, pj[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {  // unseen rows may hold anything
                    dot[f][j] = (visible >> (4 * j)) & 1 ? dot[f][j] * scale[f][j] : -INFINITY;
                    top = fmaxf(top, dot[f][j]);
                }
                top = max_groups(top);
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    pj[j] = fast_exp2(dot[f][j] - base);
                    w[f][j] = (visible >> (4 * j)) & 1 ? pj[j] * svj[j] : 0.f;
                    pm = fmaxf(pm, fabsf(w[f][j]));
                }
                pm = max_groups(pm);
                int ex = 0;
                if (pm > 0.f && pm < INFINITY) frexpf(pm, &ex);
                const float m_new =
                    fmaxf(m[f], top + (float)min(max(ex - kTopExp, -kMaxShift), kMaxShift));
                const float use = m_new == -INFINITY ? 0.f : m_new;
                if (__ballot(m[f] != -INFINITY) != 0) {  // (not the wave's first tile)
                    const float alpha = fast_exp2(m[f] - use);
                    l[f] *= alpha;
#pragma unroll
                    for (int i = 0; i < NF; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[f][i][c] *= alpha;
                }
                m[f] = m_new;
                const float shift = fast_exp2(base - use);  // 2^(s - base) to 2^(s - m)
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) w[f][j] *= shift, sum += pj[j];
                l[f] = fmaf(sum, shift, l[f]);
                split(f, std::true_type{});
            }
        } else {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                l[f] += psum[f];
                split(f, std::false_type{});
            }
        }
        next_k();
#pragma unroll
        for (int i = 0; i < NF; i += 2) {
            const v8h v[2] = {v_at(i), v_at(i + 1)};
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int f = 0; f < F; ++f)
                    o[f][i + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[x], pw[f], o[f][i + x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int f = 0; f < F; ++f)
                    o[f][i + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[x], pr[f], o[f][i + x], 0, 0, 0);
        }
    };

    if constexpr (R > 1) {
        // W tiles at a time: every wave loads and converts one of them, and the R waves of a slice
        // read the slice's R from LDS, V as the A operands of the MFMA.  The next W are on their
        // way meanwhile.
        char* s_v = reinterpret_cast<char*>(s_merge) + W * kTile * D;
        float* s_s = reinterpret_cast<float*>(s_v + W * kTile * D * 2);  // [tile][sK, sV][g][j]
        const bool any_rows = MR * mine < rows;
        // the queries have arrived: a wait for them inside the loop would be one for the next tiles'
        // loads too
#pragma unroll
        for (int f = 0; f < F; ++f) {
            asm volatile("" : "+v"(qs[f]));
#pragma unroll
            for (int i = 0; i < KI; ++i) asm volatile("" : "+v"(qf[f][i]));
        }
        Tile raw;
        Rows at{};
        int t = t_begin + wave;
        fetch_ids(t);
        rows_of_ids(t, at);
        fetch_ids(t + nw);
        if (t < t_end) {
            load_k(at);
            load_v(raw, at);
        }
        for (int t0 = t_begin; t0 < t_end; t0 += nw, t += nw) {
            if (t < t_end) {
                write_k();
#pragma unroll
                for (int i = 0; i < NF; ++i)
                    *reinterpret_cast<v8h*>(s_v + (wave * NF + i) * 1024 + lane * 16) = v_of(raw, i);
                if (m16 < 4)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        s_s[wave * 64 + 8 * g + 4 * h + m16] = raw.sk[h];
                        s_s[wave * 64 + 32 + 8 * g + 4 * h + m16] = raw.sv[h];
                    }
            }
            __syncthreads();
            rows_of_ids(t + nw, at);
            if (t + nw < t_end) {
                load_k(at);
                load_v(raw, at);
            }
            fetch_ids(t + 2 * nw);
            if (any_rows && t0 + slice * R < t_end) {
                float sk[2], svj[8];
                auto take_k = [&](int slot) {
                    const char* tk = reinterpret_cast<const char*>(s_merge) + slot * (kTile * D);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < KI; ++i)
                            k[h][i] = *reinterpret_cast<const v4i*>(tk + h * 16 * D + k_read[i]);
                    const float* ts = s_s + slot * 64 + 8 * g;
                    sk[0] = ts[m16 & 3], sk[1] = ts[4 + (m16 & 3)];
                };
                take_k(slice * R);
                for (int u = 0; u < R; ++u) {
                    const int slot = slice * R + u;
                    if (t0 + slot >= t_end) break;
                    const char* tv = s_v + slot * (kTile * D * 2) + lane * 16;
                    auto v_at = [&](int i) { return *reinterpret_cast<const v8h*>(tv + i * 1024); };
                    v8h v[NF];
#pragma unroll
                    for (int i = 0; i < NF / 2; ++i) v[i] = v_at(i);
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(s_s + slot * 64 + 32 + 8 * g + j);
                        svj[j] = x.x, svj[j + 1] = x.y, svj[j + 2] = x.z, svj[j + 3] = x.w;
                    }
                    compute(sk, svj, t0 + slot, [&]() { take_k(min(slot + 1, W - 1)); }, [&](int i) {
                        if (i < NF / 2) v[i + NF / 2] = v_at(i + NF / 2);
                        return v[i];
                    });
                }
            }
            __syncthreads();
        }
    } else {
        // While tile t is computed: V of tile t + nw is on its way from the start, K of it is taken
        // through LDS between the softmax and the product with V, and K of tile t + 2 nw is asked
        // for then.  Loads past the last tile repeat its rows: in a branch, the wait for this
        // tile's data would have to cover the next one's as well.
        int t = t_begin + wave;
        Tile ra, rb;
        Rows r1{}, r2{};
        fetch_ids(t);
        rows_of_ids(t, r1);
        fetch_ids(t + nw);
        if (t < t_end) {
            load_k(r1);
            load_v(ra, r1);
        }
        rows_of_ids(t + nw, r1);
        r2 = r1;
        fetch_ids(t + 2 * nw);
        if (t < t_end) {
            write_k();
            load_k(r1);
            read_k();
        }
        rows_of_ids(t + 2 * nw, r2);
        fetch_ids(t + 3 * nw);
        auto step = [&](Tile& now, Tile& next) {
            load_v(next, r1);
            __builtin_amdgcn_sched_barrier(0);
            const float svj[8] = {bcast16<0>(now.sv[0]), bcast16<1>(now.sv[0]), bcast16<2>(now.sv[0]),
                                  bcast16<3>(now.sv[0]), bcast16<0>(now.sv[1]), bcast16<1>(now.sv[1]),
                                  bcast16<2>(now.sv[1]), bcast16<3>(now.sv[1])};
            compute(now.sk, svj, t,
                    [&]() {
                        write_k();
                        load_k(r2);
                        read_k();
                    },
                    [&](int i) { return v_of(now, i); });
            r1 = r2;
            rows_of_ids(t + 3 * nw, r2);
            fetch_ids(t + 4 * nw);
            t += nw;
        };
        while (t < t_end) {
            step(ra, rb);
            if (t >= t_end) break;
            step(rb, ra);
        }
    }
    __syncthreads();  // the tiles of K give way to the join
    if (bad && lane == 0) atomicAdd(&g_attend_bad_ids, 1u);

    if constexpr (R == W) {  // nothing to join: lane l holds NF dims from NF (4 g + c) on of its rows
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const float sum = sum_groups(l[f]);
            const int row = MR * mine + 16 * f + m16;
            if (row >= rows) continue;
            const int r = row0_q + row, n = r % p.N, h = kvh * (p.Hq / p.Hkv) + r / p.N;
            const size_t at = (p.bshd ? ((size_t)b * p.N + n) * p.Hq + h : first_row + row) * D;
            const size_t part = ((size_t)number * p.Hkv + kvh) * all_rows + r;
            const bool any = piece.count > 1 || attends(p, b, n, e);
            if (piece.count > 1 && g == 0)
                reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(m[f], sum);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < NF; i += 4) {
                    const int d = NF * (4 * g + c) + i;
                    const float4 acc = make_float4(o[f][i][c], o[f][i + 1][c], o[f][i + 2][c], o[f][i + 3][c]);
                    if (piece.count == 1) store_row(p, at + d, acc, sum, any);
                    else reinterpret_cast<float4*>(p.part_acc + part * D)[c * NF + i + g] = acc;
                }
        }
        return;
    }

    // Join the waves: m and l of each row go to LDS, and O scaled to the rows' common maximum, which
    // are then added four dims at a time (element by element, with the factors worked out by each
    // thread, the join took 11 us of the 78 of 16 sequences with trees of 16).
    // Layout: [wave][m, l of MR rows], then [wave][MR rows][kORow].
    float* s_ml = s_merge;
    float* s_o = s_merge + nw * 2 * MR;
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const float lf = sum_groups(l[f]);
        if (g == 0)
            s_ml[wave * 2 * MR + 16 * f + m16] = m[f], s_ml[wave * 2 * MR + MR + 16 * f + m16] = lf;
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int r = 16 * f + m16;
        float top = -INFINITY;
        for (int w = mine; w < nw; w += R) top = fmaxf(top, s_ml[w * 2 * MR + r]);
        const float scale = top == -INFINITY ? 0.f : fast_exp2(m[f] - top);
        float* orow = s_o + (wave * MR + r) * kORow;
#pragma unroll
        for (int c = 0; c < 4; ++c)  // rows 4 g + c of the fragments: dims NF (4 g + c) ..
#pragma unroll
            for (int i = 0; i < NF; i += 4)
                *reinterpret_cast<float4*>(orow + NF * (4 * g + c) + i) =
                    make_float4(o[f][i][c] * scale, o[f][i + 1][c] * scale, o[f][i + 2][c] * scale,
                                o[f][i + 3][c] * scale);
    }
    __syncthreads();
    constexpr int L = D / 4;  // threads per row
    for (int x = threadIdx.x; x < rows * L; x += blockDim.x) {
        const int row = x / L, d = part_dim<D>(x % L);
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const int at = row % MR;
        for (int w = row / MR; w < nw; w += R) top = fmaxf(top, s_ml[w * 2 * MR + at]);
        const float use = top == -INFINITY ? 0.f : top;
        for (int w = row / MR; w < nw; w += R) {
            sum = fmaf(s_ml[w * 2 * MR + MR + at], fast_exp2(s_ml[w * 2 * MR + at] - use), sum);
            const float4 v = *reinterpret_cast<const float4*>(s_o + (w * MR + at) * kORow + d);
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
        if (piece.count == 1) {
            const int r = row0_q + row, n = r % p.N, h = kvh * (p.Hq / p.Hkv) + r / p.N;
            const size_t at = p.bshd ? ((size_t)b * p.N + n) * p.Hq + h : first_row + row;
            store_row(p, at * D + d, acc, sum, attends(p, b, n, e));
        } else {
            const size_t part = ((size_t)number * p.Hkv + kvh) * all_rows + row0_q + row;
            if (x % L == 0) reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(top, sum);
            reinterpret_cast<float4*>(p.part_acc + part * D)[x % L] = acc;
        }
    }
}

// Joins the pieces of each row of a sequence that has several, four dims per thread: four partials
// in flight at a time (slots past the last repeat it with weight zero).
template <int D>
constexpr int kCombineRows = 256 / (D / 4);  // rows per block, all of one sequence

template <int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(Attend p, int blocks_each) {
    constexpr int L = D / 4;
    const int b = (int)blockIdx.x / blocks_each, all_rows = p.Hq * p.N;
    const int row = (int)blockIdx.x % blocks_each * kCombineRows<D> + (int)threadIdx.x / L;
    const int c = threadIdx.x % L;
    Piece piece;
    find_piece(p, piece, [&](int, int, int seq) { return seq == b; });
    if (piece.count == 1 || row >= all_rows) return;  // one piece: written already
    const size_t part = (size_t)piece.first * all_rows + row;
    const float2* r = reinterpret_cast<const float2*>(p.part_ml) + part;
    const float4* x = reinterpret_cast<const float4*>(p.part_acc) + part * L + c;
    float m = -INFINITY, sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < piece.count; i0 += 4) {
        float2 s[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const size_t i = (size_t)min(i0 + k, piece.count - 1) * all_rows;
            s[k] = r[i];
            v[k] = x[i * L];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, s[k].x);
        const float use = top == -INFINITY ? 0.f : top;
        const float keep = fast_exp2(m - use);
        sum *= keep;
        a.x *= keep, a.y *= keep, a.z *= keep, a.w *= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i0 + k >= piece.count) continue;  // (it must not turn an infinite partial into NaN)
            const float f = fast_exp2(s[k].x - use);
            sum = fmaf(s[k].y, f, sum);
            a.x = fmaf(v[k].x, f, a.x), a.y = fmaf(v[k].y, f, a.y);
            a.z = fmaf(v[k].z, f, a.z), a.w = fmaf(v[k].w, f, a.w);
        }
        m = top;
    }
    const int h = row / p.N, n = row - h * p.N;
    const size_t at = p.bshd ? ((size_t)b * p.N + n) * p.Hq + h : (size_t)b * all_rows + row;
    store_row(p, at * D + part_dim<D>(c), a, sum, attends(p, b, n, extent_of(p, b)));
}

// ------------------------------------------------------------------ host side

struct AttendPlan {
    int frags, share, waves, groups;
    int pieces, min_tiles;  // 0: one piece per sequence
    int slots(int B) const { return pieces > 0 ? pieces : B; }
};

constexpr int kMaxSplit = 64;            // pieces per sequence, on average
constexpr int kMaxPartRows = 1 << 16;    // rows of all pieces of a cut

// The kernels that a plan picks from, with what they cost in us at head dims 128 and 64: a round of
// blocks, and a tile of a wave while few blocks run and while the GPU is full of them.
struct AttendCost {
    int frags, share, waves;
    double round[2], idle[2], full[2];
};
constexpr AttendCost kAttendCosts[] = {
    {1, 1, 8, {5.5, 6}, {1.3, 0.75}, {1.25, 1.4}},
    {2, 1, 8, {8.5, 6.5}, {1.5, 0.75}, {1.65, 1.3}},
    {2, 4, 8, {11.5, 12.5}, {1.6, 1.0}, {1.4, 1.15}},
    {2, 4, 4, {9, 11.5}, {1.4, 1.05}, {1.25, 0.95}},
    {2, 8, 8, {11, 12}, {1.3, 0.95}, {1.2, 0.95}}};

// rows: query rows per key head.
// The plan is the kernel and the number of pieces of least estimated time, for sequences of unequal
// lengths: one of max_context, 3/4 of that in the mean.  So a max_context far above the lengths, as a
// captured graph's may be, costs what the plan for such lengths costs: 16 sequences of up to 8192 with
// trees of 16, 66 us at 8208, 63 at 16384, 74 at 32768, 75 at 131072 (64 pieces).  A CU runs one block of 8 waves at a time, two
// of 4 waves or where a wave takes at most 128 registers (one fragment at head dim 64), and the
// (piece, key head) pairs go to the 8 XCDs of 32 CUs in equal runs.  The join of pieces costs 6 us and
// 0.25 for a MB of partial rows.
// The costs are fitted to every kernel at one piece per sequence and up to eight cuts, timed at 3993
// sizes (1 to 64 sequences of 16 to 45000, 1 to 256 tokens, 1 to 16 heads on each of 1 to 12, lengths
// drawn evenly from a quarter of max_context up), by the smallest mean loss against the fastest: the
// plan is 0.8% off it in the mean, 20% at the 20 worst and 43% at the worst size of a run (2% at 958
// other sizes, with the plan timed again).  Measured, us, one fragment / two / four of eight waves
// sharing / four / eight, the best cut of each, 8 key heads but where stated:
//   16 sequences of 8192, 32 rows          59 / 53
//   4 of 4096, 32 rows                     18.5 / 21
//   32 of 732, 128 rows                    - / 50 / 34 / 40
//   8 of 732, 128 rows                     - / 16 / 28 / 30
//   16 of 2064, 256 rows                   - / 83 / 66 / 72 / 75
//   4 of 16384, 256 rows                   - / 124 / 107 / 97 / 95
//   19 of 692, 380 rows                    - / 95 / 59 / 46 / 82
//   8 of 12048, 384 rows, 4 key heads      - / 126 / 111 / 94 / 107
//   2 of 20100, 400 rows                   - / 118 / 115 / 106 / 102
//   4 of 3100, 800 rows, 2 key heads       - / 29 / 39 / 37 / 36
// (two of eight waves sharing lost to one or the other everywhere: 43, 24, 80, 136 and 81 at rows 3 to 7).
AttendPlan attend_plan(int B, int rows, int Hkv, int context, int D) {
    AttendPlan pl{};
    pl.min_tiles = kWaves;
    const int d = D == 64;
    const long long tiles = ceil_div(context, kTile), pairs = (long long)B * Hkv;
    double best = INFINITY;
    for (const AttendCost& c : kAttendCosts) {
        if (c.frags == 2 && rows <= 16 * c.share) continue;
        const long long groups = ceil_div(rows, 16 * c.frags * c.share);
        const long long slots = c.waves == 4 || (c.frags == 1 && D == 64) ? 64 : 32;  // blocks of an XCD at a time
        auto wave_tiles = [&](long long t) {  // of a block's t
            return c.share == 1 ? ceil_div(t, c.waves)
                                : t / c.waves * c.share + std::min<long long>(t % c.waves, c.share);
        };
        auto consider = [&](long long pieces) {  // 0: the sequences whole
            const long long blocks = ceil_div(pieces > 0 ? pieces * Hkv : pairs, 8) * groups;  // of an XCD
            const long long rounds = ceil_div(blocks, slots);
            const double tile = c.idle[d] + (c.full[d] - c.idle[d]) * std::min(1.0, (double)blocks / slots);
            double time;
            if (pieces > 0) {  // (0.4 of a piece of each sequence but one is lost)
                const double t = std::ceil(tiles * (1 + 0.75 * (B - 1)) / (pieces - 0.4 * (B - 1)));
                time = (0.15 + 0.85 * rounds) * (c.round[d] + wave_tiles(std::min((long long)t, tiles)) * tile) +
                       6 + 0.25e-6 * 8 * pieces * Hkv * rows * D;
            } else {
                time = rounds * c.round[d] + ((rounds - 1) * wave_tiles(ceil_div(4 * tiles, 5)) + wave_tiles(tiles)) * tile;
            }
            if (time >= best) return;
            best = time;
            pl.frags = c.frags, pl.share = c.share, pl.waves = c.waves, pl.groups = (int)groups;
            pl.pieces = (int)pieces;
        };
        consider(0);
        if (B * tiles >= (1LL << 31)) continue;  // (the sum of all tiles is an int)
        const long long most = std::min(std::min<long long>(kMaxSplit, ceil_div(tiles, pl.min_tiles)) * B,
                                        kMaxPartRows / ((long long)Hkv * rows));
        for (int r = 1; r <= 4; ++r) {
            const long long pieces = std::min(r * slots * 8 / (Hkv * groups), most);
            if (pieces <= B) continue;
            consider(pieces);
            if (pieces % B != 0 && pieces > 2 * B) consider(pieces / B * B);
            if (pieces == most) break;
        }
    }
    return pl;
}

struct Partials {
    size_t ml_bytes, bytes;
};
Partials partials_of(size_t parts, int D) {
    if (parts == 0) return {0, 0};
    const size_t ml = round_up(parts * 2 * sizeof(float), kWorkspaceAlign);
    return {ml, ml + round_up(parts * D * sizeof(float), kWorkspaceAlign)};
}
// rows: of one sequence, all heads
Partials plan_partials(const AttendPlan& pl, int B, size_t rows, int D) {
    return partials_of(pl.pieces > 0 ? pl.slots(B) * rows : 0, D);
}
// Room for every plan of at most `rows` query rows in all: a cut has at most kMaxSplit pieces per
// sequence, and at most kMaxPartRows rows of them.
Partials most_partials(size_t rows, int D) {
    return partials_of(std::min<size_t>(kMaxSplit * rows, kMaxPartRows), D);
}

template <int D, int F, int R, int W>
int launch_instance(const Attend& p, unsigned blocks, hipStream_t stream) {
    constexpr int kTiles = R > 1 ? 3 * kTile * D + 256 : kTile * D;  // bytes of LDS per wave
    constexpr int kWave = R == W ? kTiles : std::max(kTiles, (2 * 16 * F + 16 * F * (D + 4)) * 4);
    static PerDeviceOnce once;
    const int st = once.run([] {
        const hipError_t e = hipFuncSetAttribute(
            reinterpret_cast<const void*>(&paged_attend_kernel<D, F, R, W>),
            hipFuncAttributeMaxDynamicSharedMemorySize, W * kWave);
        if (e == hipSuccess) return (int)INT8K_OK;
        set_last_error("hipFuncSetAttribute", e);
        return (int)INT8K_ERR_HIP;
    });
    if (st != INT8K_OK) return st;
    paged_attend_kernel<D, F, R, W><<<blocks, 64 * W, W * kWave, stream>>>(p);
    return check_launch("paged_attend_kernel");
}

template <int D>
int launch_attend(Attend p, const AttendPlan& pl, void* workspace, hipStream_t stream) {
    p.groups = pl.groups, p.pieces = pl.pieces, p.min_tiles = pl.min_tiles, p.slots = pl.slots(p.B);
    p.part_ml = static_cast<float*>(workspace);
    p.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                          plan_partials(pl, p.B, (size_t)p.Hq * p.N, D).ml_bytes);
    const unsigned blocks = (unsigned)(ceil_div((long long)p.slots * p.Hkv, 8) * 8 * pl.groups);
    const int st = pl.frags == 1 ? launch_instance<D, 1, 1, kWaves>(p, blocks, stream)
                   : pl.share == 1 ? launch_instance<D, 2, 1, kWaves>(p, blocks, stream)
                   : pl.share == 8 ? launch_instance<D, 2, 8, kWaves>(p, blocks, stream)
                   : pl.waves == 4 ? launch_instance<D, 2, 4, 4>(p, blocks, stream)
                                   : launch_instance<D, 2, 4, kWaves>(p, blocks, stream);
    if (st != INT8K_OK || pl.pieces == 0) return st;
    const int blocks_each = (int)ceil_div((long long)p.Hq * p.N, kCombineRows<D>);
    paged_combine_kernel<D><<<(unsigned)(p.B * blocks_each), 256, 0, stream>>>(p, blocks_each);
    return check_launch("paged_combine_kernel");
}

int run_attend(const Attend& p, const AttendPlan& pl, int D, void* workspace, hipStream_t stream) {
    return D == 64 ? launch_attend<64>(p, pl, workspace, stream)
                   : launch_attend<128>(p, pl, workspace, stream);
}

// Sizes that the row indexes and the grid hold: at most B * kv_heads * (rows / 16 + 1) blocks, or a
// cut's, of 512 threads each.
bool attend_fits(long long B, long long heads, long long kv_heads, long long nodes, int max_context) {
    return B * heads * nodes < (1LL << 24) && B * kv_heads < (1LL << 21) && max_context <= (1 << 30);
}

constexpr int kMaxNodes = 256;

}  // namespace

int attend_bad_ids(unsigned int* count) {
    return read_counter(&g_attend_bad_ids, "hipMemcpyFromSymbol(g_attend_bad_ids)", count);
}
}  // namespace int8k

using namespace int8k;

namespace {
bool tree_query_ok(int B, int heads, int kv_heads, int nodes, int max_context, int head_dim) {
    return B > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && nodes > 0 &&
           nodes <= kMaxNodes && max_context > 0 && (head_dim == 64 || head_dim == 128) &&
           (long long)B * heads * nodes < (1LL << 24);
}
bool sparse_query_ok(int B, int heads, int kv_heads, int max_context, int page_size, int top_pages,
                     int head_dim) {
    return B > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && max_context > 0 &&
           max_context <= (1 << 30) && page_size >= 16 && page_size <= 1024 &&
           (page_size & (page_size - 1)) == 0 && top_pages > 0 &&
           (head_dim == 64 || head_dim == 128) && (long long)B * heads < (1LL << 24);
}
}  // namespace

extern "C" size_t int8k_tree_attention_paged_workspace_bytes(int B, int heads, int kv_heads,
                                                             int nodes, int max_context,
                                                             int head_dim) {
    if (!tree_query_ok(B, heads, kv_heads, nodes, max_context, head_dim)) return 0;
    return most_partials((size_t)B * heads * nodes, head_dim).bytes;
}

extern "C" size_t int8k_tree_attention_paged_call_workspace_bytes(int B, int heads, int kv_heads,
                                                                  int nodes, int max_context,
                                                                  int head_dim) {
    if (!tree_query_ok(B, heads, kv_heads, nodes, max_context, head_dim)) return 0;
    const AttendPlan pl = attend_plan(B, heads / kv_heads * nodes, kv_heads, max_context, head_dim);
    return plan_partials(pl, B, (size_t)heads * nodes, head_dim).bytes;
}

extern "C" int int8k_tree_attention_paged_plan(int B, int heads, int kv_heads, int nodes,
                                               int max_context, int head_dim, int* plan) {
    clear_last_error();
    if (!plan || !tree_query_ok(B, heads, kv_heads, nodes, max_context, head_dim))
        return INT8K_ERR_INVALID_ARGUMENT;
    const AttendPlan pl = attend_plan(B, heads / kv_heads * nodes, kv_heads, max_context, head_dim);
    plan[0] = 16 * pl.frags, plan[1] = pl.share, plan[2] = pl.waves, plan[3] = pl.pieces;
    return INT8K_OK;
}

extern "C" int int8k_tree_attention_forward_paged(
    const int8_t* Q, const int8_t* K_pages, const int8_t* V_pages, uint16_t* out,
    const float* scale_Q, const float* sK_pages, const float* sV_pages,
    const int32_t* block_tables, const int32_t* context_lens, const int64_t* tree_mask,
    int mask_words, long long mask_batch_stride, const int32_t* node_counts, int B, int heads,
    int kv_heads, int nodes, int head_dim, int num_pages, int page_size, int max_pages_per_seq,
    int max_context, int flags, void* workspace, size_t workspace_bytes, void* stream) {
    clear_last_error();
    if (!Q || !K_pages || !V_pages || !out || !scale_Q || !sK_pages || !sV_pages ||
        !block_tables || !context_lens)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (B <= 0 || heads <= 0 || nodes <= 0 || max_pages_per_seq <= 0 || max_context <= 0 ||
        (flags & ~INT8K_ATTN_OUT_BSHD))
        return INT8K_ERR_INVALID_ARGUMENT;
    if (tree_mask && (mask_words != (nodes + 63) / 64 ||
                      (mask_batch_stride != 0 && mask_batch_stride < (long long)nodes * mask_words)))
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_pages(num_pages, page_size, kv_heads, head_dim)) return st;
    if (heads % kv_heads || (long long)max_context > (long long)max_pages_per_seq * page_size)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!aligned_to(Q, 16) || !aligned_to(K_pages, 16) || !aligned_to(V_pages, 16) ||
        !aligned_to(scale_Q, 4) || !aligned_to(sK_pages, 4) || !aligned_to(sV_pages, 4) ||
        !aligned_to(block_tables, 4) || !aligned_to(context_lens, 4) || !aligned_to(out, 8) ||
        !aligned_to(tree_mask, 8) || !aligned_to(node_counts, 4))
        return INT8K_ERR_MISALIGNED;
    if (nodes > kMaxNodes || !attend_fits(B, heads, kv_heads, nodes, max_context))
        return INT8K_ERR_UNSUPPORTED;
    const AttendPlan pl = attend_plan(B, heads / kv_heads * nodes, kv_heads, max_context, head_dim);
    const size_t need = plan_partials(pl, B, (size_t)heads * nodes, head_dim).bytes;
    if (need > 0) {
        if (!workspace || workspace_bytes < need) return INT8K_ERR_WORKSPACE;
        if (!aligned_to(workspace, 16)) return INT8K_ERR_MISALIGNED;
    }
    Attend p{};
    p.Q = Q, p.K = K_pages, p.V = V_pages, p.sQ = scale_Q, p.sK = sK_pages, p.sV = sV_pages;
    p.tables = block_tables, p.table_batch = max_pages_per_seq, p.table_head = 0;
    p.lens = context_lens;
    p.tree = true, p.counts = node_counts, p.mask = tree_mask, p.mask_batch = mask_batch_stride;
    p.words = mask_words, p.out = out, p.bshd = (flags & INT8K_ATTN_OUT_BSHD) != 0;
    p.B = B, p.Hq = heads, p.Hkv = kv_heads, p.N = nodes, p.num_pages = num_pages;
    p.log2_page = log2_of(page_size), p.max_context = max_context;
    p.qk = (1.0f / std::sqrt((float)head_dim)) * kLog2e;
    return run_attend(p, pl, head_dim, workspace, as_stream(stream));
}

extern "C" size_t int8k_decode_attention_paged_sparse_workspace_bytes(
    int B, int heads, int kv_heads, int max_context, int page_size, int top_pages, int head_dim) {
    if (!sparse_query_ok(B, heads, kv_heads, max_context, page_size, top_pages, head_dim)) return 0;
    return select_space(B, kv_heads, max_context, page_size, top_pages).bytes +
           most_partials((size_t)B * heads, head_dim).bytes;
}

extern "C" size_t int8k_decode_attention_paged_sparse_call_workspace_bytes(
    int B, int heads, int kv_heads, int max_context, int page_size, int top_pages, int head_dim) {
    if (!sparse_query_ok(B, heads, kv_heads, max_context, page_size, top_pages, head_dim)) return 0;
    const int context = (int)std::min<long long>(max_context, (long long)top_pages * page_size);
    const AttendPlan pl = attend_plan(B, heads / kv_heads, kv_heads, context, head_dim);
    return select_space(B, kv_heads, max_context, page_size, top_pages).bytes +
           plan_partials(pl, B, (size_t)heads, head_dim).bytes;
}

extern "C" int int8k_decode_attention_forward_paged_sparse(
    const int8_t* Q, const int8_t* K_pages, const int8_t* V_pages, uint16_t* out,
    int32_t* selected, const float* scale_Q, const float* sK_pages, const float* sV_pages,
    const int8_t* K_means, const float* sK_means, const int32_t* block_tables,
    const int32_t* context_lens, int B, int heads, int kv_heads, int head_dim, int num_pages,
    int page_size, int max_pages_per_seq, int max_context, int top_pages, void* workspace,
    size_t workspace_bytes, void* stream) {
    clear_last_error();
    if (!Q || !K_pages || !V_pages || !out || !selected || !scale_Q || !sK_pages || !sV_pages ||
        !K_means || !sK_means || !block_tables || !context_lens)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (B <= 0 || heads <= 0 || max_pages_per_seq <= 0 || max_context <= 0 || top_pages <= 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_pages(num_pages, page_size, kv_heads, head_dim)) return st;
    if (heads % kv_heads || (long long)max_context > (long long)max_pages_per_seq * page_size)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!aligned_to(Q, 16) || !aligned_to(K_pages, 16) || !aligned_to(V_pages, 16) ||
        !aligned_to(K_means, 16) || !aligned_to(scale_Q, 4) || !aligned_to(sK_pages, 4) ||
        !aligned_to(sV_pages, 4) || !aligned_to(sK_means, 4) || !aligned_to(block_tables, 4) ||
        !aligned_to(context_lens, 4) || !aligned_to(out, 8) || !aligned_to(selected, 4))
        return INT8K_ERR_MISALIGNED;
    const int context = (int)std::min<long long>(max_context, (long long)top_pages * page_size);
    if (!attend_fits(B, heads, kv_heads, 1, max_context) || (long long)B * kv_heads > 65535 ||
        (long long)B * kv_heads * top_pages >= (1LL << 31))
        return INT8K_ERR_UNSUPPORTED;
    const AttendPlan pl = attend_plan(B, heads / kv_heads, kv_heads, context, head_dim);
    const SelectSpace sel = select_space(B, kv_heads, max_context, page_size, top_pages);
    if (!workspace ||
        workspace_bytes < sel.bytes + plan_partials(pl, B, (size_t)heads, head_dim).bytes)
        return INT8K_ERR_WORKSPACE;
    if (!aligned_to(workspace, 16)) return INT8K_ERR_MISALIGNED;

    char* ws = static_cast<char*>(workspace);
    Select s{};
    s.Q = Q, s.sQ = scale_Q, s.means = K_means, s.s_means = sK_means, s.tables = block_tables;
    s.lens = context_lens, s.keys = reinterpret_cast<uint64_t*>(ws + sel.keys);
    s.pages = reinterpret_cast<int32_t*>(ws + sel.pages);
    s.positions = reinterpret_cast<int32_t*>(ws + sel.positions), s.selected = selected;
    s.B = B, s.Hq = heads, s.Hkv = kv_heads, s.D = head_dim, s.num_pages = num_pages;
    s.log2_page = log2_of(page_size), s.max_pages = max_pages_per_seq, s.max_context = max_context;
    s.max_blocks = (int)ceil_div(max_context, page_size), s.top = top_pages;
    if (const int st = launch_select(s, as_stream(stream))) return st;

    Attend p{};
    p.Q = Q, p.K = K_pages, p.V = V_pages, p.sQ = scale_Q, p.sK = sK_pages, p.sV = sV_pages;
    p.tables = s.pages, p.table_batch = (long long)kv_heads * top_pages, p.table_head = top_pages;
    p.lens = s.positions;
    p.tree = false, p.out = out;
    p.B = B, p.Hq = heads, p.Hkv = kv_heads, p.N = 1, p.num_pages = num_pages;
    p.log2_page = s.log2_page, p.max_context = context;
    p.qk = (1.0f / std::sqrt((float)head_dim)) * kLog2e;
    return run_attend(p, pl, head_dim, ws + sel.bytes, as_stream(stream));
}

extern "C" int int8k_paged_bad_ids(unsigned int* count) {
    clear_last_error();
    if (!count) return INT8K_ERR_INVALID_ARGUMENT;
    unsigned int n[3] = {0, 0, 0};
    for (int i = 0; i < 3; ++i) {
        const int st = i == 0 ? append_bad_slots(n) : i == 1 ? attend_bad_ids(n + 1) : pages_bad_ids(n + 2);
        if (st != INT8K_OK) return st;
    }
    *count = n[0] + n[1] + n[2];
    return INT8K_OK;
}
