// heads.hip — norms of queries and keys per head and the position rotation in one pass, gfx950.
//
// x [B, S, (heads + 2 kv_heads) * D] is a fused QKV projection's output.  For each token and
// each query or key head, with fp32 arithmetic throughout:
//   y_d = x_d / sqrt(mean_d x_d^2 + eps) * w_d              (where the part has weights)
//   (a, b) -> (a cos - b sin, b cos + a sin)                for the rot_dim / 2 pairs (a, b),
//   (y_t, y_{t + rot_dim/2}), or (y_2t, y_2t+1) interleaved, by cos[pos][t], sin[pos][t];
// dims from rot_dim on and the value heads pass through.  The result is rounded to x's dtype
// once and stored as heads [B, H, S, D], or quantized per row as int8k_quantize_per_token
// quantizes those rounded rows.  Quantized keys and values can go straight to the rows `slots`
// of a paged cache [num_pages, kv_heads, page, D] instead: only where a row is stored differs.
//
// Memory-bound: x is read once and the heads are written once.  A lane holds both elements of
// its 8 pairs, 16 elements of a row (D / 16 lanes per row), so the rotation needs no exchange
// between lanes, and a wave holds 64 / (D / 16) consecutive tokens and walks a range of
// heads: the angles of a token, twice the bytes of one of its rows, are read once for all of
// them and the rows that a wave writes for a head are consecutive in memory.  8192 tokens of 48
// heads of 128 in bf16, normed, rotated and quantized: 32 us, 4.7 TB/s of x and codes (47 us
// with the angles and weights loaded float by float, 32 of a lane's 36 loads).
#include <algorithm>
#include <cmath>

#include "pages.h"
#include "rows.h"

namespace int8k {
namespace {

__device__ unsigned int g_rope_bad_positions;
__device__ unsigned int g_append_bad_slots;

struct HeadsArgs {
    const void* x;
    const float *cos, *sin;
    const int32_t* pos;
    const float* w[2];  // norm weights of queries and keys, or null
    float eps;
    void* y[3];       // [B, H_p, S, D] in x's dtype, or
    int8_t* q[3];     // the codes and
    float* s[3];      // their row scales
    long long tokens;
    int S, heads, kv_heads, D, max_pos, half;  // half = rot_dim / 2
    int lg;           // 1 << lg lanes per row
    int heads_per_wave;
    float inv_dim;    // 1 / D
    const int32_t* slots;  // PAGED: row page * page_size + offset of each token's key and value
    int num_pages, log2_page;
};

// How the 8 pairs of lane item c lie in a row.
enum PairLayout {
    kSplit = 0,        // a, b = 8 elements at 8 c and half + 8 c (half a multiple of 8)
    kInterleaved = 1,  // the 16 elements from 16 c
    kSplitAny = 2      // as kSplit for any half: element by element
};

// Element indices of pair t of a row: the rotated pairs first, then neighbours.
__device__ __forceinline__ void pair_at(int t, int half, int& a, int& b) {
    a = t < half ? t : 2 * t;  // 2 half + 2 (t - half)
    b = t < half ? t + half : 2 * t + 1;
}

template <int DT>
__device__ __forceinline__ float load_one(const void* x, size_t i) {
    if constexpr (DT == INT8K_DTYPE_F32) return static_cast<const float*>(x)[i];
    const uint16_t u = static_cast<const uint16_t*>(x)[i];
    if constexpr (DT == INT8K_DTYPE_F16) return __half2float(__ushort_as_half(u));
    return __uint_as_float((uint32_t)u << 16);
}

// Values as numbers of the dtype.
template <int DT>
__device__ __forceinline__ void round_all(float (&v)[8]) {
    if constexpr (DT == INT8K_DTYPE_F32) return;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t w = pack_pair<DT>(v[i], v[i + 1]);
        if constexpr (DT == INT8K_DTYPE_F16) {
            v[i] = __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
            v[i + 1] = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
        } else {
            v[i] = __uint_as_float(w << 16);
            v[i + 1] = __uint_as_float(w & 0xffff0000u);
        }
    }
}

template <int DT>
__device__ __forceinline__ void store_one(void* y, size_t i, float v) {
    if constexpr (DT == INT8K_DTYPE_F32) static_cast<float*>(y)[i] = v;
    else if constexpr (DT == INT8K_DTYPE_F16)
        static_cast<uint16_t*>(y)[i] = f32_to_f16_bits(v);
    else static_cast<uint16_t*>(y)[i] = (uint16_t)(__float_as_uint(v) >> 16);
}

// 8 consecutive elements as loaded.
template <int DT>
struct Raw8 {
    uint4 w[DT == INT8K_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* x, size_t i) {
    Raw8<DT> r;
    if constexpr (DT == INT8K_DTYPE_F32) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(x) + i);
        r.w[0] = p[0], r.w[1] = p[1];
    } else {
        r.w[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, float (&v)[8]) {
    if constexpr (DT == INT8K_DTYPE_F32) {
        const uint32_t d[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w,
                               r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(d[k]);
    } else {
        unpack_chunk<DT>(r.w[0], v);
    }
}
// 8 values that are numbers of the dtype.
template <int DT>
__device__ __forceinline__ void store8(void* y, size_t i, const float (&v)[8]) {
    if constexpr (DT == INT8K_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + i);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + i) =
            make_uint4(pack_pair<DT>(v[0], v[1]), pack_pair<DT>(v[2], v[3]),
                       pack_pair<DT>(v[4], v[5]), pack_pair<DT>(v[6], v[7]));
    }
}

// The codes that store_codes (rows.h) stores, with the rounding and the packing in one step:
// adding 1.5 * 2^23 rounds half to even and leaves the code in the low byte.
__device__ __forceinline__ void store_codes8(const float (&v)[8], float s, float inv, int8_t* dst) {
    uint32_t b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c[i] = __float_as_uint(fminf(fmaxf(quotient(v[4 * j + i], s, inv), -128.f), 127.f) +
                                   12582912.0f);
        b[j] = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u) |
               __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(b[0], b[1]);
}

// 8 floats with a float's alignment.
__device__ __forceinline__ void load_floats(const float* p, float (&v)[8]) {
    typedef float v4f __attribute__((ext_vector_type(4), aligned(4)));
    const v4f a = reinterpret_cast<const v4f*>(p)[0], b = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}

// The pairs (a, b) of an item from its two chunks in memory order.
template <int LAYOUT>
__device__ __forceinline__ void split_pairs(const float (&lo)[8], const float (&hi)[8],
                                            float (&a)[8], float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (LAYOUT == kSplit) a[i] = lo[i], b[i] = hi[i];
        else {
            a[i] = i < 4 ? lo[2 * (i & 3)] : hi[2 * (i & 3)];
            b[i] = i < 4 ? lo[2 * (i & 3) + 1] : hi[2 * (i & 3) + 1];
        }
    }
}

// The heads [h0, h1) of one part (0 queries, 1 keys, 2 values) for this lane's token.
template <int DT, bool QUANT, int LAYOUT>
__device__ __forceinline__ void part_heads(const HeadsArgs& p, int part, int h0, int h1, size_t in,
                                           size_t row, size_t row_step, int cc, bool has, bool ok,
                                           int ia, int ib, const float* cs, const float* sn) {
    // element indices of the pairs of this item
    auto pair = [&](int i, int& ka, int& kb) {
        if constexpr (LAYOUT == kSplitAny) pair_at(8 * cc + i, p.half, ka, kb);
        else if constexpr (LAYOUT == kSplit) ka = ia + i, kb = ib + i;
        else ka = ia + 2 * i, kb = ka + 1;
    };
    // the first head's elements are on their way while the angles are read
    Raw8<DT> lo{}, hi{};
    if constexpr (LAYOUT != kSplitAny) lo = load8<DT>(p.x, in + ia), hi = load8<DT>(p.x, in + ib);
    const float* wp = part < 2 ? p.w[part] : nullptr;
    // (a, b) -> (a ca - b sb, b cb + a sa) / rms: the norm's weights go into the angles.  Pairs
    // past the rotation have cos 1 and take nothing of the other element, not even its product
    // with a sine of zero: an infinity or a NaN there is that element's own.
    float ca[8], cb[8], sa[8], sb[8];
    if (part < 2) {
        float wa[8], wb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.f, ca[i] = 1.f, sa[i] = 0.f;
        if (wp != nullptr) {
            if constexpr (LAYOUT == kSplitAny) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    int ka, kb;
                    pair(i, ka, kb);
                    wa[i] = wp[ka], wb[i] = wp[kb];
                }
            } else {
                float l[8], h[8];
                load_floats(wp + ia, l);
                load_floats(wp + ib, h);
                split_pairs<LAYOUT>(l, h, wa, wb);
            }
        }
        if (8 * cc + 8 <= p.half) {
            load_floats(cs + 8 * cc, ca);
            load_floats(sn + 8 * cc, sa);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (8 * cc + i < p.half) ca[i] = cs[8 * cc + i], sa[i] = sn[8 * cc + i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = ca[i], s = sa[i];
            ca[i] = wa[i] * c, sb[i] = wb[i] * s;
            cb[i] = wb[i] * c, sa[i] = wa[i] * s;
        }
    }
    auto heads = [&](Raw8<DT> lo, Raw8<DT> hi, float (&ga)[8], float (&gv)[8], size_t r) {
        float a[8], v[8];
        if constexpr (LAYOUT == kSplitAny) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = ga[i], v[i] = gv[i];
        } else {
            float l[8], h[8];
            unpack8<DT>(lo, l);
            unpack8<DT>(hi, h);
            split_pairs<LAYOUT>(l, h, a, v);
        }
        if (part < 2) {
            float inv = 1.f;
            if (wp != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(v[i], v[i], ss));
                ss = row_reduce(has ? ss : 0.f, p.lg, [](float m, float n) { return m + n; });
                inv = __builtin_amdgcn_rsqf(fmaf(ss, p.inv_dim, p.eps));  // off by one ulp at most
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // normed first: squares in range do not promise products in range
                const float na = a[i] * inv, nv = v[i] * inv;
                const bool turned = LAYOUT == kSplit ? 8 * cc < p.half : 8 * cc + i < p.half;
                const float ua = na * ca[i], uv = nv * cb[i];
                a[i] = turned ? ua - nv * sb[i] : ua;
                v[i] = turned ? uv + na * sa[i] : uv;
            }
            round_all<DT>(a);
            round_all<DT>(v);
        }
        // back to memory order
        float l[8], h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (LAYOUT == kInterleaved) {
                l[i] = (i & 1) ? v[i / 2] : a[i / 2];
                h[i] = (i & 1) ? v[4 + i / 2] : a[4 + i / 2];
            } else {
                l[i] = a[i], h[i] = v[i];
            }
        }
        const size_t out = r * p.D;
        if constexpr (QUANT) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(v[i])));
            m = row_reduce(has ? m : 0.f, p.lg, [](float x, float y) { return fmaxf(x, y); });
            // exactly the division (whose correction step has no answer for an infinity)
            const float sc = m < INFINITY ? quotient(fmaxf(m, 1e-8f), 127.f, 1.f / 127.f) : m;
            const float rinv = 1.f / sc;
            if (ok) {
                if constexpr (LAYOUT == kSplitAny) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        int ka, kb;
                        pair(i, ka, kb);
                        p.q[part][out + ka] = (int8_t)quant_code(a[i], sc);
                        p.q[part][out + kb] = (int8_t)quant_code(v[i], sc);
                    }
                } else {
                    store_codes8(l, sc, rinv, p.q[part] + out + ia);
                    store_codes8(h, sc, rinv, p.q[part] + out + ib);
                }
                if (cc == 0) p.s[part][r] = sc;
            }
        } else if (ok) {
            if constexpr (LAYOUT == kSplitAny) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    int ka, kb;
                    pair(i, ka, kb);
                    store_one<DT>(p.y[part], out + ka, a[i]);
                    store_one<DT>(p.y[part], out + kb, v[i]);
                }
            } else {
                store8<DT>(p.y[part], out + ia, l);
                store8<DT>(p.y[part], out + ib, h);
            }
        }
    };
    if constexpr (LAYOUT == kSplitAny) {
        for (int h = h0; h < h1; ++h, in += p.D, row += row_step) {
            float a[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                int ka, kb;
                pair(i, ka, kb);
                a[i] = load_one<DT>(p.x, in + ka);
                v[i] = load_one<DT>(p.x, in + kb);
            }
            heads({}, {}, a, v, row);
        }
    } else {
        // the next head's elements are on their way while one is computed (past the last
        // head they repeat it)
        float none[8];
        for (int h = h0; h < h1; ++h, row += row_step) {
            in += h + 1 < h1 ? p.D : 0;
            const Raw8<DT> nl = load8<DT>(p.x, in + ia), nh = load8<DT>(p.x, in + ib);
            heads(lo, hi, none, none, row);
            lo = nl, hi = nh;
        }
    }
}

template <int DT, bool QUANT, int LAYOUT, bool PAGED>
__global__ __launch_bounds__(256, LAYOUT == kSplitAny ? 3 : 4) void qk_norm_rope_kernel(HeadsArgs p) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & ((1 << p.lg) - 1);
    const bool has = 16 * c < p.D;
    const int per_wave = 64 >> p.lg;
    const long long t_raw = ((long long)blockIdx.x * 4 + wave) * per_wave + (lane >> p.lg);
    const bool ok = t_raw < p.tokens && has;
    const long long t = min(t_raw, p.tokens - 1);
    const int cc = has ? c : 0;  // idle lanes of a row read its first item and store nothing

    const int raw_pos = p.pos[t];
    const int pos = min(max(raw_pos, 0), p.max_pos - 1);
    if (blockIdx.y == 0) {
        const uint64_t bad = __ballot(raw_pos != pos && c == 0 && t_raw < p.tokens);
        if (bad != 0 && lane == 0) atomicAdd(&g_rope_bad_positions, (unsigned)__popcll(bad));
    }
    const float* cs = p.cos + (size_t)pos * p.half;
    const float* sn = p.sin + (size_t)pos * p.half;
    // where this item's chunks lie in a row (kSplit, kInterleaved)
    int ia = 16 * cc, ib = 16 * cc + 8;
    if (LAYOUT == kSplit && 8 * cc < p.half) ia = 8 * cc, ib = p.half + 8 * cc;

    const int total = p.heads + 2 * p.kv_heads;
    const int h0 = blockIdx.y * p.heads_per_wave, h1 = min(h0 + p.heads_per_wave, total);
    const long long b = t / p.S;
    const long long s = t - b * p.S;
    const size_t in = (size_t)t * total * p.D;
    bool stored = ok;  // a negative slot stores no key and no value; one past the cache is counted
    size_t cache_row = 0;
    if constexpr (PAGED) {
        const int slot = p.slots[t];
        const bool past = slot >= ((long long)p.num_pages << p.log2_page);
        if (blockIdx.y == 0) {
            const uint64_t bad = __ballot(past && c == 0 && t_raw < p.tokens);
            if (bad != 0 && lane == 0) atomicAdd(&g_append_bad_slots, (unsigned)__popcll(bad));
        }
        stored = ok && slot >= 0 && !past;
        const int at = stored ? slot : 0, page = at >> p.log2_page;
        cache_row = (((size_t)page * p.kv_heads) << p.log2_page) + (at - (page << p.log2_page));
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        const int first = part == 0 ? 0 : part == 1 ? p.heads : p.heads + p.kv_heads;
        const int count = part == 0 ? p.heads : p.kv_heads;
        const int a = max(h0, first), e = min(h1, first + count);
        if (a >= e) continue;
        const bool paged = PAGED && part > 0;
        const size_t row = paged ? cache_row + ((size_t)(a - first) << p.log2_page)
                                 : ((size_t)b * count + (a - first)) * p.S + s;
        const size_t step = paged ? (size_t)1 << p.log2_page : (size_t)p.S;
        part_heads<DT, QUANT, LAYOUT>(p, part, a, e, in + (size_t)a * p.D, row, step, cc, has,
                                      paged ? stored : ok, ia, ib, cs, sn);
    }
}

template <bool QUANT, bool PAGED>
int launch_heads(HeadsArgs p, int dtype, bool interleaved, hipStream_t stream) {
    const int items = p.D / 16;
    while ((1 << p.lg) < items) ++p.lg;
    const int total = p.heads + 2 * p.kv_heads;
    const long long blocks = ceil_div(p.tokens, 4LL * (64 >> p.lg));
    // one head per wave until the grid holds 4 waves per SIMD, then more: a wave reads a token's
    // angles and the weights once (8192 tokens of 48 heads of 128 in bf16 to int8: 32.0 us here,
    // 37 with twice the waves, 39 with half)
    p.heads_per_wave = (int)std::max<long long>(1, std::min<long long>(total, blocks * total / 1024));
    const long long gy = ceil_div(total, p.heads_per_wave);
    if (blocks >= (1LL << 24) || gy > 65535) return INT8K_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, (unsigned)gy);
    const int layout = interleaved ? kInterleaved : p.half % 8 == 0 ? kSplit : kSplitAny;
    with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (layout == kSplit)
            qk_norm_rope_kernel<DT, QUANT, kSplit, PAGED><<<grid, 256, 0, stream>>>(p);
        else if (layout == kInterleaved)
            qk_norm_rope_kernel<DT, QUANT, kInterleaved, PAGED><<<grid, 256, 0, stream>>>(p);
        else qk_norm_rope_kernel<DT, QUANT, kSplitAny, PAGED><<<grid, 256, 0, stream>>>(p);
    });
    return check_launch("qk_norm_rope_kernel");
}

// Where keys and values go to a paged cache (slots not null).
struct HeadsCache {
    const int32_t* slots = nullptr;
    int num_pages = 0, page_size = 0;
};

template <bool QUANT, bool PAGED = false>
int heads_entry(const void* x, int dtype, const float* cos, const float* sin, int max_positions,
                int rot_dim, const int32_t* positions, const float* q_weight,
                const float* k_weight, float eps, void* const (&y)[3], int8_t* const (&q)[3],
                float* const (&s)[3], int B, int S, int heads, int kv_heads, int head_dim,
                int flags, void* stream, const HeadsCache& cache = {}) {
    clear_last_error();
    if (!x || !cos || !sin || !positions) return INT8K_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 3; ++i)
        if (QUANT ? !q[i] || !s[i] : !y[i]) return INT8K_ERR_INVALID_ARGUMENT;
    if (flags & ~INT8K_ROPE_INTERLEAVED) return INT8K_ERR_INVALID_ARGUMENT;
    if (dtype < INT8K_DTYPE_F16 || dtype > INT8K_DTYPE_F32) return INT8K_ERR_INVALID_ARGUMENT;
    if (B <= 0 || S <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_positions <= 0 ||
        rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim || heads > 65535 || kv_heads > 65535)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (head_dim % 16 || head_dim > 256) return INT8K_ERR_UNSUPPORTED;
    if constexpr (PAGED) {
        if (!cache.slots) return INT8K_ERR_INVALID_ARGUMENT;
        if (const int st = check_pages(cache.num_pages, cache.page_size, kv_heads, head_dim)) return st;
        if (!aligned_to(cache.slots, 4) || !aligned_to(q[1], 16) || !aligned_to(q[2], 16))
            return INT8K_ERR_MISALIGNED;
    }
    if (!aligned_to(x, 16) || !aligned_to(cos, 4) || !aligned_to(sin, 4) ||
        !aligned_to(positions, 4) || !aligned_to(q_weight, 4) || !aligned_to(k_weight, 4))
        return INT8K_ERR_MISALIGNED;
    for (int i = 0; i < 3; ++i)
        if (QUANT ? !aligned_to(q[i], 8) || !aligned_to(s[i], 4) : !aligned_to(y[i], 16))
            return INT8K_ERR_MISALIGNED;
    HeadsArgs p{};
    p.x = x, p.cos = cos, p.sin = sin, p.pos = positions;
    p.w[0] = q_weight, p.w[1] = k_weight, p.eps = eps;
    for (int i = 0; i < 3; ++i) p.y[i] = y[i], p.q[i] = q[i], p.s[i] = s[i];
    p.tokens = (long long)B * S;
    p.S = S, p.heads = heads, p.kv_heads = kv_heads, p.D = head_dim;
    p.max_pos = max_positions, p.half = rot_dim / 2, p.inv_dim = 1.f / (float)head_dim;
    if constexpr (PAGED)
        p.slots = cache.slots, p.num_pages = cache.num_pages, p.log2_page = log2_of(cache.page_size);
    return launch_heads<QUANT, PAGED>(p, dtype, (flags & INT8K_ROPE_INTERLEAVED) != 0,
                                      as_stream(stream));
}

}  // namespace
}  // namespace int8k

using namespace int8k;

extern "C" int int8k_qk_norm_rope(const void* x, int dtype, const float* cos, const float* sin,
                                  int max_positions, int rot_dim, const int32_t* positions,
                                  const float* q_weight, const float* k_weight, float eps,
                                  void* q, void* k, void* v, int B, int S, int heads,
                                  int kv_heads, int head_dim, int flags, void* stream) {
    return heads_entry<false>(x, dtype, cos, sin, max_positions, rot_dim, positions, q_weight,
                              k_weight, eps, {q, k, v}, {nullptr, nullptr, nullptr},
                              {nullptr, nullptr, nullptr}, B, S, heads, kv_heads, head_dim, flags,
                              stream);
}

extern "C" int int8k_qk_norm_rope_quantize(
    const void* x, int dtype, const float* cos, const float* sin, int max_positions, int rot_dim,
    const int32_t* positions, const float* q_weight, const float* k_weight, float eps, int8_t* q,
    float* scale_q, int8_t* k, float* scale_k, int8_t* v, float* scale_v, int B, int S, int heads,
    int kv_heads, int head_dim, int flags, void* stream) {
    return heads_entry<true>(x, dtype, cos, sin, max_positions, rot_dim, positions, q_weight,
                             k_weight, eps, {nullptr, nullptr, nullptr}, {q, k, v},
                             {scale_q, scale_k, scale_v}, B, S, heads, kv_heads, head_dim, flags,
                             stream);
}

extern "C" int int8k_qk_norm_rope_append(
    const void* x, int dtype, const float* cos, const float* sin, int max_positions, int rot_dim,
    const int32_t* positions, const float* q_weight, const float* k_weight, float eps, int8_t* q,
    float* scale_q, int8_t* K_pages, int8_t* V_pages, float* sK_pages, float* sV_pages,
    const int32_t* slots, int B, int S, int heads, int kv_heads, int head_dim, int num_pages,
    int page_size, int flags, void* stream) {
    return heads_entry<true, true>(x, dtype, cos, sin, max_positions, rot_dim, positions, q_weight,
                                   k_weight, eps, {nullptr, nullptr, nullptr},
                                   {q, K_pages, V_pages}, {scale_q, sK_pages, sV_pages}, B, S,
                                   heads, kv_heads, head_dim, flags, stream,
                                   {slots, num_pages, page_size});
}

namespace int8k {
int append_bad_slots(unsigned int* count) {
    return read_counter(&g_append_bad_slots, "hipMemcpyFromSymbol(g_append_bad_slots)", count);
}
}  // namespace int8k

extern "C" int int8k_rope_bad_positions(unsigned int* count) {
    clear_last_error();
    if (!count) return INT8K_ERR_INVALID_ARGUMENT;
    return read_counter(&g_rope_bad_positions, "hipMemcpyFromSymbol(g_rope_bad_positions)", count);
}
