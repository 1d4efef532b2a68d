// pages.hip — upkeep of the paged INT8 cache: moving rows, the mean key of each page, and the
// selection of blocks by those means; gfx950.
#include <algorithm>
#include <cmath>

#include "pages.h"
#include "rows.h"

namespace int8k {
namespace {

__device__ unsigned int g_pages_bad_ids;

typedef int v4i __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ move
// Rows src -> dst of every key head, list by list: a block takes one list of one head of one side,
// reads all its rows into registers and writes them after a barrier, so a destination may be
// another pair's source.  Latency-bound: one dependent load after the slots.

struct Move {
    int8_t* pages[2];
    float* scales[2];
    const int32_t *src, *dst;
    int pairs, Hkv, num_pages, log2_page;
};

constexpr int kMaxPairs = 256;

template <int D, int ITEMS>
__global__ __launch_bounds__(256) void move_rows_kernel(Move p) {
    constexpr int C = D / 16;  // 16-byte pieces of a row
    const int h = (int)(blockIdx.x % (unsigned)p.Hkv), list = (int)(blockIdx.x / (unsigned)p.Hkv);
    const int side = blockIdx.y, T = blockDim.x;
    const int32_t *src = p.src + (size_t)list * p.pairs, *dst = p.dst + (size_t)list * p.pairs;
    const long long cap = (long long)p.num_pages << p.log2_page;
    auto row_of = [&](int slot) {
        const int page = slot >> p.log2_page;
        return (((size_t)page * p.Hkv + h) << p.log2_page) + (slot - (page << p.log2_page));
    };
    // the pair's rows, or false where it is left out
    auto rows = [&](int i, size_t& from, size_t& to) {
        const int s = src[i], d = dst[i];
        if (s < 0 || d < 0 || s >= cap || d >= cap) return false;
        from = row_of(s), to = row_of(d);
        return true;
    };
    uint4 v[ITEMS];
    size_t at[ITEMS];
    bool have[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int x = threadIdx.x + k * T;
        size_t from = 0;
        have[k] = x < p.pairs * C && rows(x / C, from, at[k]);
        v[k] = make_uint4(0, 0, 0, 0);
        if (have[k]) v[k] = *reinterpret_cast<const uint4*>(p.pages[side] + from * D + 16 * (x % C));
    }
    // the scales, one or more per thread
    constexpr int kScales = (ITEMS + C - 1) / C;
    float sc[kScales];
    size_t sat[kScales];
    bool shave[kScales];
#pragma unroll
    for (int k = 0; k < kScales; ++k) {
        const int x = threadIdx.x + k * T;
        size_t from = 0;
        shave[k] = x < p.pairs && rows(x, from, sat[k]);
        sc[k] = shave[k] ? p.scales[side][from] : 0.f;
        if (h == 0 && side == 0 && x < p.pairs && (src[x] >= cap || dst[x] >= cap))
            atomicAdd(&g_pages_bad_ids, 1u);
    }
    // the data has arrived, not only been asked for, before any thread writes
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) reload_barrier(v[k]);
#pragma unroll
    for (int k = 0; k < kScales; ++k) asm volatile("" : "+v"(sc[k]));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int x = threadIdx.x + k * T;
        if (have[k]) *reinterpret_cast<uint4*>(p.pages[side] + at[k] * D + 16 * (x % C)) = v[k];
    }
#pragma unroll
    for (int k = 0; k < kScales; ++k)
        if (shave[k]) p.scales[side][sat[k]] = sc[k];
}

// ------------------------------------------------------------------ means
// m_d = sum over a page's rows of code * scale / page, summed in 64 bits (so that a code beside a
// rounding border does not depend on the order of the sum), rounded to fp32 and quantized as
// int8k_quantize_per_token does; a NaN in a mean makes the scale NaN.

// One wave per page and key head up to 64 rows (four waves of a few rows each spend more on joining
// their sums than on the rows: 2048 pages of 64 rows, 8 heads of 128, 84 us, 33 so), two or four
// for longer pages.  A lane owns 16 dims of every 64 / L-th row and loads four rows ahead.

// a of this lane plus a of the lane 32 (16) away where the lane is in the lower half of 64 (32), the
// same of b where it is in the upper: two values of two lanes become one of each.
template <int HALF>
__device__ __forceinline__ double fold(double a, double b) {
    auto swapped = [](uint32_t x, uint32_t y) {
        if constexpr (HALF == 32) return __builtin_amdgcn_permlane32_swap(x, y, false, false);
        else return __builtin_amdgcn_permlane16_swap(x, y, false, false);
    };
    const uint64_t u = (uint64_t)__double_as_longlong(a), v = (uint64_t)__double_as_longlong(b);
    const auto lo = swapped((uint32_t)u, (uint32_t)v), hi = swapped((uint32_t)(u >> 32), (uint32_t)(v >> 32));
    return __longlong_as_double((long long)((uint64_t)hi[0] << 32 | lo[0])) +
           __longlong_as_double((long long)((uint64_t)hi[1] << 32 | lo[1]));
}

template <int D>
__global__ __launch_bounds__(256) void page_means_kernel(const int8_t* __restrict__ pages,
                                                         const float* __restrict__ scales,
                                                         const int32_t* __restrict__ ids,
                                                         int8_t* __restrict__ means,
                                                         float* __restrict__ s_means, int units,
                                                         int Hkv, int num_pages, int log2_page,
                                                         int waves) {
    constexpr int L = D / 16, R = 64 / L;  // lanes per row, rows per wave load
    constexpr int kAhead = 4;
    __shared__ double s_sum[4][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave & (waves - 1);  // of the unit's rows
    const int u = (int)blockIdx.x * (4 / waves) + wave / waves;
    const int h = u % Hkv, id = u < units ? __builtin_amdgcn_readfirstlane(ids[u / Hkv]) : -1;
    const bool ok = id >= 0 && id < num_pages;
    if (id >= num_pages && h == 0 && part == 0 && lane == 0) atomicAdd(&g_pages_bad_ids, 1u);
    const size_t unit = ok ? (size_t)id * Hkv + h : 0, row0 = unit << log2_page;
    const int page = 1 << log2_page;
    double acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0;
    if (ok) {
        const uint4* rows = reinterpret_cast<const uint4*>(pages + row0 * D) + lane % L;
        uint4 w[kAhead];
        float s[kAhead];
        auto load = [&](int k, int r) {  // past the last row: a zero scale
            const int at = min(r, page - 1);
            w[k] = rows[at * L];
            s[k] = r < page ? scales[row0 + at] : 0.f;
        };
        const int step = waves * R;
        int r = part * R + lane / L;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load(k, r + k * step);
        for (int r0 = part * R; r0 < page; r0 += kAhead * step, r += kAhead * step) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (r0 + k * step >= page) break;
                const uint32_t d[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                const double sd = (double)s[k];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    acc[i] = fma((double)(int)(int8_t)((d[i >> 2] >> (8 * (i & 3))) & 0xff), sd, acc[i]);
                load(k, r + (kAhead + k) * step);
            }
        }
    }
    // Over the wave's rows: lanes 32 and 16 apart exchange halves of the dims, so that each ends
    // with 4, 4 (lane / 16) .. of its 16; the rest of the lanes are L .. 8 apart.
    double half[8], sum[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) half[i] = fold<32>(acc[i], acc[i + 8]);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = fold<16>(half[i], half[i + 4]);
#pragma unroll
    for (int x = L; x < 16; x <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += __shfl_xor(sum[i], x);
    const int dim = 16 * (lane % L) + 8 * (lane / 32) + 4 * (lane / 16 % 2);
    if (waves > 1) {
        if (lane % 16 < L)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[wave][dim + i] = sum[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i] = 0.0;
            for (int k = 0; k < waves; ++k) sum[i] += s_sum[(wave & ~(waves - 1)) + k][dim + i];
        }
    }
    if (!ok || part != 0) return;
    float m[4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = (float)(sum[i] / page);
        top = max(top, __float_as_uint(m[i]) & 0x7fffffffu);
    }
    top = __float_as_uint(row_reduce(__uint_as_float(top), 6, [](float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }));
    const float amax = __uint_as_float(top);
    const float s = (amax < 1e-8f ? 1e-8f : amax) / 127.f;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c |= ((uint32_t)quant_code(m[i], s) & 0xffu) << (8 * i);
    if (lane % 16 < L) *reinterpret_cast<uint32_t*>(means + unit * D + dim) = c;
    if (lane == 0) s_means[unit] = s;
}

// ------------------------------------------------------------------ selection
// score of a block = max over the heads of the group of (q . mean) sMean sQ, q . mean exact, the
// products in 64 bits in that order, so the order of two scores is that of the formula.  The
// last block is taken always and has no score.

__device__ __forceinline__ int blocks_of(const Select& p, int b, int& len) {
    len = min(max(p.lens[b], 0), p.max_context);
    return (len + (1 << p.log2_page) - 1) >> p.log2_page;
}

// Larger scores have larger keys; NaN, which no score is above, has 0.
__device__ __forceinline__ uint64_t score_key(double s) {
    if (s != s) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);  // (one zero)
    return u >> 63 ? ~u : u | (1ull << 63);
}

// A group of D / 16 lanes, which hold 16 dims each, scores kEach blocks.  (In the selection's block,
// which spares a launch: 40.2 against 41.4 us for 32 sequences of 512 blocks, 27.5 against 23.9 for one
// of 1024, 42 against 22 for one of 4096; fewer blocks were not timed so.)
template <int D>
__global__ __launch_bounds__(256) void block_scores_kernel(Select p) {
    constexpr int L = D / 16, kRows = 256 / L, kEach = 2;
    constexpr int kHeads = 4;  // whose queries are loaded at a time, the first with the means
    const int row = blockIdx.y, b = row / p.Hkv, h = row % p.Hkv, G = p.Hq / p.Hkv;
    const int base = blockIdx.x * (kRows * kEach), first = base + threadIdx.x / L, c = threadIdx.x % L;
    v4i q[kHeads];
    double sq[kHeads];
    auto load_heads = [&](int g0) {
#pragma unroll
        for (int g = 0; g < kHeads; ++g) {
            const size_t at = (size_t)b * p.Hq + h * G + min(g0 + g, G - 1);
            q[g] = *reinterpret_cast<const v4i*>(p.Q + at * D + 16 * c);
            sq[g] = (double)p.sQ[at];
        }
    };
    load_heads(0);
    int len;
    const int n = blocks_of(p, b, len);
    if (n <= p.top || base >= n - 1) return;  // all are taken, or none is here
    v4i mean[kEach];
    double sm[kEach], best[kEach];
    bool any[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int i = min(first + k * kRows, n - 2);  // blocks past the last repeat it
        const int raw = p.tables[(size_t)b * p.max_pages + i];
        const int id = (int)min((unsigned)raw, (unsigned)(p.num_pages - 1));
        if (id != raw && h == 0 && c == 0 && first + k * kRows < n - 1) atomicAdd(&g_pages_bad_ids, 1u);
        const size_t unit = (size_t)id * p.Hkv + h;
        mean[k] = *reinterpret_cast<const v4i*>(p.means + unit * D + 16 * c);
        sm[k] = (double)p.s_means[unit];
        best[k] = -INFINITY;
        any[k] = false;
    }
    for (int g0 = 0; g0 < G; g0 += kHeads) {
        if (g0 > 0) load_heads(g0);
#pragma unroll
        for (int g = 0; g < kHeads; ++g) {  // (heads past the last repeat it)
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                int dot = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) dot = __builtin_amdgcn_sdot4(q[g][i], mean[k][i], dot, false);
                dot = L == 8 ? group8_sum(dot) : group4_sum(dot);
                const double s = ((double)dot * sm[k]) * sq[g];
                any[k] = any[k] || s == s;
                best[k] = s > best[k] ? s : best[k];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int i = first + k * kRows;
        if (c == 0 && i < n - 1) p.keys[(size_t)row * p.max_blocks + i] = any[k] ? score_key(best[k]) : 0;
    }
}

constexpr int kSelectThreads = 1024;

__device__ __forceinline__ double score_of(uint64_t key) {
    return __longlong_as_double((long long)(key >> 63 ? key & ~(1ull << 63) : ~key));
}

// How many threads before this one hold true, and how many of all.
__device__ __forceinline__ int count_before(bool v, int* s_wave, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t set = __ballot(v);
    __syncthreads();
    if (lane == 0) s_wave[wave] = __popcll(set);
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const int count = s_wave[w];
        before += w < wave ? count : 0;
        all += count;
    }
    return before + __builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
}

// The bin of s_count[256] that holds the need-th largest, and how many lie in the bins above it.
__device__ __forceinline__ void find_bin(const int* s_count, int need, int& s_bin, int& s_above) {
    const int t = threadIdx.x;
    if (t >= 64) return;
    int c[4], mine = 0;  // lane t: bins 255 - 4 t down to 252 - 4 t
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s_count[255 - 4 * t - i], mine += c[i];
    int x = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int below = __shfl_up(x, d);
        x += t >= d ? below : 0;
    }
    int above = x - mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (above < need && need <= above + c[i]) s_bin = 255 - 4 * t - i, s_above = above;
        above += c[i];
    }
}

// The top - 1 largest keys (ties: the lowest blocks) and the last block.  The scores are counted in
// 256 equal bins between their smallest and largest; the few in the bin that the last taken one
// lies in are ranked among each other.  Where that does not do (an infinite or NaN score, all equal,
// a bin of more than kList), by digits of 8 bits of the keys from the highest, until all keys that
// share the digits of the last taken one so far are taken.
constexpr int kList = 256;

__global__ __launch_bounds__(kSelectThreads) void select_blocks_kernel(Select p) {
    __shared__ int s_count[256], s_wave[kSelectThreads / 64], s_bin, s_above, s_listed;
    __shared__ float s_low[kSelectThreads / 64], s_high[kSelectThreads / 64];
    __shared__ uint64_t s_key[kList];
    __shared__ int s_at[kList];
    const int row = blockIdx.x, b = row / p.Hkv, t = threadIdx.x;
    int len;
    const int n = blocks_of(p, b, len), page = 1 << p.log2_page;
    const int32_t* table = p.tables + (size_t)b * p.max_pages;
    int32_t* selected = p.selected + (size_t)row * p.top;
    int32_t* pages = p.pages + (size_t)row * p.top;
    const int taken = min(n, p.top);
    if (t == 0 && row % p.Hkv == 0)
        p.positions[b] = taken == 0 ? 0 : (taken - 1) * page + len - (n - 1) * page;
    // (unsigned: top may be within a step of 2^31)
    for (unsigned i = taken + t; i < (unsigned)p.top; i += blockDim.x) selected[i] = -1;
    if (n <= p.top) {
        for (int i = t; i < n; i += blockDim.x) selected[i] = i, pages[i] = table[i];
        return;
    }
    const uint64_t* keys = p.keys + (size_t)row * p.max_blocks;
    int need = p.top - 1;
    auto emit = [&](auto takes) {  // the taken blocks in order
        int base = 0;
        for (int i0 = 0; i0 < n; i0 += blockDim.x) {
            const int i = i0 + t;
            const bool take = i == n - 1 || (i < n - 1 && takes(i));
            int total;
            const int at = count_before(take, s_wave, total) + base;
            base += total;
            if (take && at < p.top) selected[at] = i, pages[at] = table[i];
        }
    };
    if (need == 0) return emit([](int) { return false; });

    float low = INFINITY, high = -INFINITY;
    bool odd = false;
    for (int i = t; i < n - 1; i += blockDim.x) {
        const uint64_t k = keys[i];
        const float s = (float)score_of(k);
        odd = odd || k == 0 || !(fabsf(s) < INFINITY);
        low = fminf(low, s), high = fmaxf(high, s);
    }
    low = row_reduce(low, 6, [](float x, float y) { return fminf(x, y); });
    high = row_reduce(high, 6, [](float x, float y) { return fmaxf(x, y); });
    if (t % 64 == 0) s_low[t / 64] = low, s_high[t / 64] = high;
    if (t < 256) s_count[t] = 0;
    if (t == 0) s_listed = 0;
    odd = __syncthreads_or(odd);
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) low = fminf(low, s_low[w]), high = fmaxf(high, s_high[w]);
    const double scale = 256.0 / ((double)high - (double)low);
    if (!odd && high > low && scale < 1e300) {
        // (rounded bounds: the cut to 0 .. 255 keeps the order)
        auto bin_of = [&](uint64_t k) { return (int)fmin(fmax((score_of(k) - (double)low) * scale, 0.0), 255.0); };
        for (int i = t; i < n - 1; i += blockDim.x) atomicAdd(&s_count[bin_of(keys[i])], 1);
        __syncthreads();
        find_bin(s_count, need, s_bin, s_above);
        __syncthreads();
        const int bin = s_bin, listed = s_count[bin];
        need -= s_above;
        if (listed <= kList) {
            for (int i = t; i < n - 1; i += blockDim.x) {
                const uint64_t k = keys[i];
                if (bin_of(k) != bin) continue;
                const int at = atomicAdd(&s_listed, 1);
                s_key[at] = k, s_at[at] = i;
            }
            __syncthreads();
            return emit([&](int i) {
                const uint64_t k = keys[i];
                const int mine = bin_of(k);
                if (mine != bin) return mine > bin;
                int before = 0;
                for (int j = 0; j < listed; ++j)
                    before += s_key[j] > k || (s_key[j] == k && s_at[j] < i) ? 1 : 0;
                return before < need;
            });
        }
        need += s_above;
    }

    uint64_t prefix = 0;  // the digits so far; need: of the keys that share them
    int shift = 64;       // keys >> shift == prefix share them (64: all)
    bool exact = false;   // all that share them are taken
    while (!exact && shift > 0) {
        __syncthreads();
        if (t < 256) s_count[t] = 0;
        __syncthreads();
        for (int i = t; i < n - 1; i += blockDim.x) {
            const uint64_t k = keys[i];
            if (shift == 64 || (k >> shift) == prefix) atomicAdd(&s_count[(k >> (shift - 8)) & 255], 1);
        }
        __syncthreads();
        find_bin(s_count, need, s_bin, s_above);
        __syncthreads();
        shift -= 8;
        prefix = prefix << 8 | (uint64_t)s_bin;
        need -= s_above;
        exact = need == s_count[s_bin];
    }
    int base = 0, ties = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + t;
        const uint64_t high_digits = i < n - 1 ? keys[i] >> shift : 0;
        const bool same = i < n - 1 && high_digits == prefix;
        int total;
        const int rank = count_before(same, s_wave, total) + ties;
        ties += total;
        const bool take = i == n - 1 || (i < n - 1 && (high_digits > prefix || (same && rank < need)));
        const int at = count_before(take, s_wave, total) + base;
        base += total;
        if (take && at < p.top) selected[at] = i, pages[at] = table[i];
    }
}

}  // namespace

int launch_select(const Select& s, hipStream_t stream) {
    const int rows = s.B * s.Hkv;
    if (s.max_blocks > s.top) {
        const int per = 256 / (s.D / 16) * 2;
        const dim3 grid((unsigned)ceil_div(s.max_blocks, per), (unsigned)rows);
        if (s.D == 64) block_scores_kernel<64><<<grid, 256, 0, stream>>>(s);
        else block_scores_kernel<128><<<grid, 256, 0, stream>>>(s);
        if (const int st = check_launch("block_scores_kernel")) return st;
    }
    select_blocks_kernel<<<(unsigned)rows, kSelectThreads, 0, stream>>>(s);
    return check_launch("select_blocks_kernel");
}

int pages_bad_ids(unsigned int* count) {
    return read_counter(&g_pages_bad_ids, "hipMemcpyFromSymbol(g_pages_bad_ids)", count);
}
}  // namespace int8k

using namespace int8k;

extern "C" int int8k_kv_cache_move_paged(int8_t* K_pages, int8_t* V_pages, float* sK_pages,
                                         float* sV_pages, const int32_t* src_slots,
                                         const int32_t* dst_slots, int lists, int pairs,
                                         int kv_heads, int head_dim, int num_pages, int page_size,
                                         void* stream) {
    clear_last_error();
    if (!K_pages || !V_pages || !sK_pages || !sV_pages || !src_slots || !dst_slots)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (lists <= 0 || pairs <= 0) return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_pages(num_pages, page_size, kv_heads, head_dim)) return st;
    if (!aligned_to(K_pages, 16) || !aligned_to(V_pages, 16) || !aligned_to(sK_pages, 4) ||
        !aligned_to(sV_pages, 4) || !aligned_to(src_slots, 4) || !aligned_to(dst_slots, 4))
        return INT8K_ERR_MISALIGNED;
    if (pairs > kMaxPairs || (long long)lists * kv_heads >= (1LL << 23)) return INT8K_ERR_UNSUPPORTED;
    Move p{{K_pages, V_pages}, {sK_pages, sV_pages}, src_slots, dst_slots, pairs, kv_heads,
           num_pages, log2_of(page_size)};
    const int items = pairs * (head_dim / 16);
    const dim3 grid((unsigned)(lists * kv_heads), 2);
    const unsigned threads = (unsigned)std::min<long long>(256, ceil_div(items, 64) * 64);
    const hipStream_t s = as_stream(stream);
    if (head_dim == 64) {
        if (items <= 256) move_rows_kernel<64, 1><<<grid, threads, 0, s>>>(p);
        else move_rows_kernel<64, 4><<<grid, threads, 0, s>>>(p);
    } else {
        if (items <= 256) move_rows_kernel<128, 1><<<grid, threads, 0, s>>>(p);
        else move_rows_kernel<128, 8><<<grid, threads, 0, s>>>(p);
    }
    return check_launch("move_rows_kernel");
}

extern "C" int int8k_kv_page_means(const int8_t* K_pages, const float* sK_pages,
                                   const int32_t* page_ids, int8_t* K_means, float* sK_means,
                                   int count, int kv_heads, int head_dim, int num_pages,
                                   int page_size, void* stream) {
    clear_last_error();
    if (!K_pages || !sK_pages || !page_ids || !K_means || !sK_means || count <= 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (const int st = check_pages(num_pages, page_size, kv_heads, head_dim)) return st;
    if (!aligned_to(K_pages, 16) || !aligned_to(sK_pages, 4) || !aligned_to(page_ids, 4) ||
        !aligned_to(K_means, 16) || !aligned_to(sK_means, 4))
        return INT8K_ERR_MISALIGNED;
    if ((long long)count * kv_heads >= (1LL << 23)) return INT8K_ERR_UNSUPPORTED;
    const int units = count * kv_heads, waves = page_size <= 64 ? 1 : page_size <= 256 ? 2 : 4;
    const unsigned blocks = (unsigned)ceil_div(units, 4 / waves);
    const hipStream_t s = as_stream(stream);
    if (head_dim == 64)
        page_means_kernel<64><<<blocks, 256, 0, s>>>(K_pages, sK_pages, page_ids, K_means, sK_means, units,
                                                     kv_heads, num_pages, log2_of(page_size), waves);
    else
        page_means_kernel<128><<<blocks, 256, 0, s>>>(K_pages, sK_pages, page_ids, K_means, sK_means, units,
                                                      kv_heads, num_pages, log2_of(page_size), waves);
    return check_launch("page_means_kernel");
}
