// kv4.hip — a paged KV cache held in 4 bits: append, read back, and grouped decode attention,
// gfx950.
//
// A cache row is one token of one key head: D codes of 4 bits, two a byte (element 2i in the
// low half of byte i, 2i + 1 in the high half), each stored as code + 8, and one fp32 scale:
//   s = max(|row|, 1e-8) / 7,  code = rn(clamp(x / s, -8, 7)),  x ~= code * s
// K_pages and V_pages uint8 [num_pages, kv_heads, page, D/2], scales fp32 [num_pages,
// kv_heads, page].  A NaN in a row makes its scale NaN (as amax does in PyTorch).
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
    return (m < 1e-8f ? 1e-8f : m) / 7.f;  // NaN stays NaN
}

__device__ __forceinline__ uint32_t kv4_code(float x, float s) {
    return (uint32_t)((int)__builtin_rintf(fminf(fmaxf(x / s, -8.f), 7.f)) + 8);
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

// 8 lanes (D = 64) or 16 (D = 128) per row, 8 elements each; blockIdx.y: 0 = K, 1 = V.
// Memory-bound and small: a row is read as 16-byte pieces and written as one run of D/2 bytes.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Side k, Kv4Side v,
                                                         const int32_t* __restrict__ slots,
                                                         int T, int H, int num_pages,
                                                         int log2_page) {
    constexpr int L = D / 8, kLg = D == 64 ? 3 : 4;
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int c = threadIdx.x & (L - 1);
    if (row >= (long long)T * H) return;  // whole lane groups leave together
    const int t = (int)(row / H), h = (int)(row - (long long)t * H);
    const int slot = slots[t];
    const long long cap = (long long)num_pages << log2_page;
    if (slot < 0 || slot >= cap) {
        if (slot >= cap && h == 0 && c == 0 && blockIdx.y == 0) atomicAdd(&g_kv4_bad_ids, 1u);
        return;
    }
    const Kv4Side sd = blockIdx.y == 0 ? k : v;
    float e[8];
    load_row8<DT>(sd.x, (size_t)(t * sd.st + h * sd.sh) + 8 * c, e);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(e[i]));
    m = __float_as_uint(row_reduce(__uint_as_float(m), kLg, [](float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }));
    const float s = kv4_scale(m);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= kv4_code(e[i], s) << (4 * i);
    const int page = slot >> log2_page, off = slot & ((1 << log2_page) - 1);
    const size_t r = (((size_t)page * H + h) << log2_page) + off;
    reinterpret_cast<uint32_t*>(sd.pages + r * (D / 2))[c] = w;
    if (c == 0) sd.scales[r] = s;
}

// Rows at `slots` as numbers of the dtype; slots outside the cache read as zeros.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ pages,
                                                       const float* __restrict__ scales,
                                                       const int32_t* __restrict__ slots,
                                                       void* __restrict__ out, int T, int H,
                                                       int num_pages, int log2_page) {
    constexpr int L = D / 8;
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int c = threadIdx.x & (L - 1);
    if (row >= (long long)T * H) return;
    const int t = (int)(row / H), h = (int)(row - (long long)t * H);
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
    const size_t o = (size_t)row * D + 8 * c;
    if constexpr (DT == INT8K_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + o);
        p[0] = make_float4(y[0], y[1], y[2], y[3]);
        p[1] = make_float4(y[4], y[5], y[6], y[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == INT8K_DTYPE_F16) {
                w[i] = __half_as_ushort(f16_of_f32(y[2 * i])) |
                       ((uint32_t)__half_as_ushort(f16_of_f32(y[2 * i + 1])) << 16);
            } else {
                auto rn = [](float v) {
                    const uint32_t u = __float_as_uint(v);
                    return v != v ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
                };
                w[i] = rn(y[2 * i]) | (rn(y[2 * i + 1]) << 16);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + o) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ------------------------------------------------------------------ decode
// One block per (sequence, query head): each group of D/8 lanes takes a position at a time,
// keeps a running maximum and sum of its own, and the groups' states are joined in LDS.
template <int D>
__global__ __launch_bounds__(256) void kv4_decode_kernel(
    const int8_t* __restrict__ Q, const uint8_t* __restrict__ Kp, const uint8_t* __restrict__ Vp,
    const float* __restrict__ sQ, const float* __restrict__ sKp, const float* __restrict__ sVp,
    const int32_t* __restrict__ tables, const int32_t* __restrict__ lens,
    uint16_t* __restrict__ out, int Hq, int Hkv, int num_pages, int log2_page, int max_pages,
    int max_context, float qk) {
    constexpr int L = D / 8, kGroups = 256 / L;
    __shared__ float s_m[kGroups], s_l[kGroups], s_acc[kGroups][D];
    const int b = blockIdx.x / Hq, h = blockIdx.x % Hq, kvh = h / (Hq / Hkv);
    const int c = threadIdx.x & (L - 1), g = threadIdx.x / L;
    const int len = min(max(lens[b], 0), max_context);
    const int32_t* table = tables + (size_t)b * max_pages;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (float)Q[(size_t)blockIdx.x * D + 8 * c + i];
    const float qs = sQ[blockIdx.x] * qk;
    float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    unsigned bad = 0;
    for (int j = g; j < len; j += kGroups) {
        int page = table[j >> log2_page];
        if ((unsigned)page >= (unsigned)num_pages) page = num_pages - 1, bad = 1;
        const size_t r = (((size_t)page * Hkv + kvh) << log2_page) + (j & ((1 << log2_page) - 1));
        const uint32_t kw = reinterpret_cast<const uint32_t*>(Kp + r * (D / 2))[c];
        const uint32_t vw = reinterpret_cast<const uint32_t*>(Vp + r * (D / 2))[c];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf((float)((int)((kw >> (4 * i)) & 15u) - 8), q[i], dot);
        dot = row_reduce(dot, D == 64 ? 3 : 4, [](float x, float y) { return x + y; });
        const float s = dot * qs * sKp[r];
        const float m_new = fmaxf(m, s);
        const float corr = fast_exp2(m - m_new), p = fast_exp2(s - m_new);
        l = l * corr + p;
        const float w = p * sVp[r];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            acc[i] = fmaf(w, (float)((int)((vw >> (4 * i)) & 15u) - 8), acc[i] * corr);
        m = m_new;
    }
    if (__ballot(bad != 0) != 0 && (threadIdx.x & 63) == 0) atomicAdd(&g_kv4_bad_ids, 1u);
    if (c == 0) s_m[g] = m, s_l[g] = l;
#pragma unroll
    for (int i = 0; i < 8; ++i) s_acc[g][8 * c + i] = acc[i];
    __syncthreads();
    if (threadIdx.x < D) {
        float mm = -INFINITY, ll = 0.f, a = 0.f;
        for (int i = 0; i < kGroups; ++i) mm = fmaxf(mm, s_m[i]);
        if (len > 0) {
            for (int i = 0; i < kGroups; ++i) {
                if (i >= len) break;  // groups without a position
                const float f = fast_exp2(s_m[i] - mm);
                ll += s_l[i] * f;
                a += s_acc[i][threadIdx.x] * f;
            }
        }
        out[(size_t)blockIdx.x * D + threadIdx.x] =
            len > 0 ? __half_as_ushort(f16_of_f32(a / ll)) : (uint16_t)0;
    }
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
    const long long blocks = ceil_div((long long)T * kv_heads * (head_dim / 8), 256);
    if (blocks >= (1LL << 24)) return INT8K_ERR_UNSUPPORTED;
    const Kv4Side k{k_new, k_token_stride, k_head_stride, K_pages, sK_pages};
    const Kv4Side v{v_new, v_token_stride, v_head_stride, V_pages, sV_pages};
    with_dtype(dtype, [&](auto dt) {
        with_head_dim(head_dim, [&](auto d) {
            kv4_append_kernel<decltype(dt)::value, decltype(d)::value>
                <<<dim3((unsigned)blocks, 2), 256, 0, as_stream(stream)>>>(
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
    const long long blocks = ceil_div((long long)T * kv_heads * (head_dim / 8), 256);
    if (blocks >= (1LL << 24)) return INT8K_ERR_UNSUPPORTED;
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
    (void)B, (void)heads, (void)kv_heads, (void)max_context, (void)head_dim;
    return 0;
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
    if ((long long)B * heads >= (1LL << 24)) return INT8K_ERR_UNSUPPORTED;
    (void)workspace, (void)workspace_bytes;
    const float qk = (1.0f / std::sqrt((float)head_dim)) * kLog2e;
    with_head_dim(head_dim, [&](auto d) {
        kv4_decode_kernel<decltype(d)::value><<<(unsigned)(B * heads), 256, 0, as_stream(stream)>>>(
            Q, K_pages, V_pages, scale_Q, sK_pages, sV_pages, block_tables, context_lens, out,
            heads, kv_heads, num_pages, log2_of(page_size), max_pages_per_seq, max_context, qk);
    });
    return check_launch("kv4_decode_kernel");
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
