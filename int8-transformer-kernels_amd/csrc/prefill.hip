// prefill.hip — INT8 flash attention for prefill (seq_q == seq_kv), gfx950.
//
// Contract of the reference int8_attention_forward (kernels/int8_attention.cu:
// 926-1028; math at kernels/int8_attention.cu:292-298, 467-643):
//   s_ij  = (q_i . k_j) [exact int32] * sQ_i * sK_j / sqrt(D)
//   p_ij  = softmax_j(s_ij)                          (fp32, online)
//   out_i = sum_j (p_ij * sV_j)[fp16] * v_j[fp16] / sum_j p_ij   -> fp16
// Non-causal by default (the reference has no mask); `causal` adds the
// standard lower-triangular mask (key j visible to query i iff j <= i).
//
// Design (CDNA4): a block owns the queries of one (b,h), 32 per wave (256
// queries on 8 waves at head_dim 128, 128 queries on 4 waves at 64 and 256; fewer
// queries with the keys split over groups of waves where that grid would leave
// CUs idle), and walks the KV sequence in tiles of 64 keys.  K (int8 rows), V (fp16,
// row-major) and both key-scale vectors of a tile are staged in double-buffered LDS
// by buffer loads: the next tile's loads are in flight in registers while the
// current tile is computed, and there is one barrier per tile.  The LDS reads
// of the MFMA fragments and key scales are scheduled ahead of their uses.  The
// wave index is read into a scalar register, so every per-wave condition of the
// tile loop (causal skip, masked tile, fast or slow path) is a scalar branch.
// Everything is computed transposed so that each lane owns one query:
//   S^T[64 keys x 32 q] = K . Q^T   on v_mfma_i32_32x32x32_i8 (A = K rows
//                                   from LDS, B = Q kept in VGPRs)
//   O^T[D x 32 q]      += V^T . P^T on v_mfma_f32_32x32x16_f16
// In the 32x32 accumulator layout lane l holds column l%32 — its query — and
// 16 of the 32 keys, so the row max, the exponentials, the running sum and the
// rescale of O are lane-local except for one exchange with lane l^32, which
// holds the other 16 keys of the same query.  P^T feeds the PV MFMA from the
// registers it was computed in; V is staged once per tile into LDS as fp16
// [key][dim] rows, as it arrives, and each V^T fragment is two transposing LDS
// reads (ds_read_b64_tr_b16) whose key order matches those P^T registers.
//
// Head dims: 64, 128 and 256 run the kernel at their own size; any other
// multiple of 16 up to 256 runs the next of those sizes with the missing dims
// read as zero (Q, V) and never stored.  Any other head_dim up to 512 (the
// reference's scalar fallback, kernels/int8_attention.cu:65-157) runs
// prefill_generic_kernel.
//
// With an int8 destination the epilogue emits the per-token quantization of
// the fp16 output row instead (the attention output as the next INT8 stage's
// input): the fp16 values the fp16 path would store, their row absmax, and
// the per-token quantizer's codes and scale — the same bytes as
// int8k_quantize_per_token over the fp16 output, without its round trip.
#include "prefill_core.h"

namespace int8k {
namespace {

// D: the kernel's head_dim.  PAD: the rows in memory have head_dim d_mem < D
// (a multiple of 16); the dims past it read as zero and are not stored.
template <int D, int QW, int KG, bool CAUSAL, bool PAD>
__global__ __launch_bounds__((Shape<D, QW, KG>::kThreads), (Shape<D, QW, KG>::kMinBlocks)) void prefill_kernel(
    const int8_t* __restrict__ Q, const int8_t* __restrict__ K, const int8_t* __restrict__ V,
    const float* __restrict__ sQ, const float* __restrict__ sK, const float* __restrict__ sV,
    uint16_t* __restrict__ out, int8_t* __restrict__ qout, float* __restrict__ qout_scale, int S,
    int n_qtiles, float qk_scale_log2, int heads, int bshd, int d_mem) {
    extern __shared__ __align__(16) char smem_all[];
    const int dm = PAD ? d_mem : D;  // head_dim of the rows in memory
    // Under the causal mask a query tile's work grows with its index, so the
    // grid is query-tile-major, heaviest tiles of every (b,h) first.  Without
    // it, the query tiles of one (b,h) share its K/V, so they run on one XCD
    // (one L2): blocks are dispatched to the 8 XCDs in turn, and XCD x takes a
    // contiguous range of (b,h, query tile) pairs in (b,h)-major order.
    const int BH = gridDim.x / n_qtiles;
    int bh, qt;
    if constexpr (CAUSAL) {
        bh = (int)(blockIdx.x % BH);
        qt = n_qtiles - 1 - (int)(blockIdx.x / BH);
    } else {
        constexpr int kXcds = 8;
        const int xcd = (int)(blockIdx.x % kXcds), local = (int)(blockIdx.x / kXcds);
        const int per = (int)(gridDim.x / kXcds), rem = (int)(gridDim.x % kXcds);
        const int tile = xcd * per + min(xcd, rem) + local;
        bh = tile / n_qtiles;
        qt = tile - bh * n_qtiles;
    }
    const size_t base = (size_t)bh * S;
    // output row: [B, H, S, D] order, or [B, S, H, D] (the row order of the
    // output projection's input) with bshd
    prefill_block<D, QW, KG, CAUSAL, PAD>(
        smem_all, Q + base * dm, K + base * dm, V + base * dm, sQ + base, sK + base, sV + base,
        out, qout, qout_scale, S, qt, qk_scale_log2, d_mem, [&](int q) {
            return bshd ? ((size_t)(bh / heads) * S + q) * heads + (size_t)(bh % heads) : base + q;
        });
}

// ---------------------------------------------------------------- any head_dim
// Head dims the MFMA kernel does not take (not a multiple of 16, or above 256)
// up to kGenMaxD, the reference's scalar fallback (kernels/int8_attention.cu:
// 65-157, 1019-1027) with the same math.  A block holds kGenQ queries of one
// (b,h), kGenQW per wave, and stages each 64-key tile in LDS: K as zero-padded
// 4-byte words, V as bytes, the key scales as fp32.  Lane j scores key j of
// the tile for the wave's queries (v_dot4 over the words: exact int32), the
// online softmax is a wave reduction, and each lane then accumulates dims
// d = lane + 64 e over the tile's keys with the weights p_j * sV_j broadcast by
// v_readlane.  Outputs as prefill_kernel: fp16 rounded from the fp32 quotient,
// or its per-token int8 codes and scale; [B,H,S,D] or [B,S,H,D] rows.
constexpr int kGenMaxD = 512;
constexpr int kGenQW = 4;                // queries per wave
constexpr int kGenQ = 4 * kGenQW;        // queries per block (4 waves)
constexpr int kGenKV = 64;               // keys per tile
constexpr int kGenDims = kGenMaxD / 64;  // dims per lane, at most

// LDS layout of prefill_generic_kernel for head_dim D (bytes).
struct GenLayout {
    int dw, ks;  // 4-byte words per row (zero-padded), K row stride in words (odd)
    int v_off, s_off, q_off, bytes;
};
__host__ __device__ inline GenLayout gen_layout(int D) {
    GenLayout g;
    g.dw = (D + 3) / 4;
    g.ks = g.dw | 1;  // odd: the 64 lanes' rows start in 64 different banks
    g.v_off = kGenKV * g.ks * 4;
    g.s_off = g.v_off + (kGenKV * D + 15) / 16 * 16;
    g.q_off = g.s_off + 2 * kGenKV * 4;
    g.bytes = g.q_off + kGenQ * g.dw * 4;
    return g;
}

template <bool CAUSAL>
__global__ __launch_bounds__(256) void prefill_generic_kernel(
    const int8_t* __restrict__ Q, const int8_t* __restrict__ K, const int8_t* __restrict__ V,
    const float* __restrict__ sQ, const float* __restrict__ sK, const float* __restrict__ sV,
    uint16_t* __restrict__ out, int8_t* __restrict__ qout, float* __restrict__ qout_scale, int S,
    int D, int n_qtiles, float qk_scale_log2, int heads, int bshd) {
    extern __shared__ __align__(16) char smem[];
    const GenLayout L = gen_layout(D);
    int* kw = reinterpret_cast<int*>(smem);
    int8_t* vb = reinterpret_cast<int8_t*>(smem + L.v_off);
    float* ssk = reinterpret_cast<float*>(smem + L.s_off);
    float* ssv = ssk + kGenKV;
    int* qw = reinterpret_cast<int*>(smem + L.q_off);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // causal grids: heaviest query tiles of every (b,h) first
    const int BH = gridDim.x / n_qtiles;
    int bh, qt;
    if constexpr (CAUSAL) {
        bh = (int)(blockIdx.x % BH);
        qt = n_qtiles - 1 - (int)(blockIdx.x / BH);
    } else {
        bh = (int)(blockIdx.x / n_qtiles);
        qt = (int)(blockIdx.x % n_qtiles);
    }
    const int q0 = qt * kGenQ;
    const size_t base = (size_t)bh * S;
    const int rowb = L.dw * 4;  // bytes per zero-padded row

    int8_t* qb = reinterpret_cast<int8_t*>(qw);
    for (int i = t; i < kGenQ * rowb; i += 256) {
        const int r = i / rowb, c = i - r * rowb;
        qb[i] = (q0 + r < S && c < D) ? Q[(base + q0 + r) * D + c] : (int8_t)0;
    }
    float qs[kGenQW], m[kGenQW], l[kGenQW], acc[kGenQW][kGenDims];
#pragma unroll
    for (int i = 0; i < kGenQW; ++i) {
        const int q = q0 + wave * kGenQW + i;
        qs[i] = q < S ? sQ[base + q] * qk_scale_log2 : 0.f;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < kGenDims; ++e) acc[i][e] = 0.f;
    }
    const int nd = (D + 63) >> 6;
    const int kv_end = CAUSAL ? min(S, q0 + kGenQ) : S;
    for (int k0 = 0; k0 < kv_end; k0 += kGenKV) {
        __syncthreads();  // the previous tile's reads are done
        int8_t* kb = reinterpret_cast<int8_t*>(kw);
        const int krow = L.ks * 4;
        for (int i = t; i < kGenKV * krow; i += 256) {
            const int r = i / krow, c = i - r * krow;
            kb[i] = (k0 + r < S && c < D) ? K[(base + k0 + r) * D + c] : (int8_t)0;
        }
        const int vn = min(kGenKV, S - k0) * D;
        for (int i = t; i < kGenKV * D; i += 256) vb[i] = i < vn ? V[(base + k0) * D + i] : (int8_t)0;
        if (t < kGenKV) ssk[t] = k0 + t < S ? sK[base + k0 + t] : 0.f;
        else if (t < 2 * kGenKV) ssv[t - kGenKV] = k0 + t - kGenKV < S ? sV[base + k0 + t - kGenKV] : 0.f;
        __syncthreads();

        const int key = k0 + lane;
        const float skl = ssk[lane], svl = ssv[lane];
        const int* kr = kw + lane * L.ks;
        float w[kGenQW];
#pragma unroll
        for (int i = 0; i < kGenQW; ++i) {
            const int qi = wave * kGenQW + i, q = q0 + qi;
            const int* qr = qw + qi * L.dw;
            int dot = 0;
            for (int c = 0; c < L.dw; ++c) dot = __builtin_amdgcn_sdot4(qr[c], kr[c], dot, false);
            float s = static_cast<float>(dot) * qs[i] * skl;
            if (key >= S || (CAUSAL && key > q)) s = -INFINITY;
            float mx = s;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
            const float m_new = fmaxf(m[i], mx);
            const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
            const float corr = fast_exp2(m[i] - m_use);
            const float p = fast_exp2(s - m_use);
            float ps = p;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) ps += __shfl_xor(ps, off);
            l[i] = l[i] * corr + ps;
#pragma unroll
            for (int e = 0; e < kGenDims; ++e) acc[i][e] *= corr;
            m[i] = m_new;
            w[i] = p * svl;
        }
        const int nk = min(kGenKV, kv_end - k0);
        for (int j = 0; j < nk; ++j) {
            float v[kGenDims];
#pragma unroll
            for (int e = 0; e < kGenDims; ++e) {
                const int d = lane + 64 * e;
                v[e] = (e < nd && d < D) ? static_cast<float>(vb[j * D + d]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kGenQW; ++i) {
                const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w[i]), j));
#pragma unroll
                for (int e = 0; e < kGenDims; ++e) acc[i][e] = fmaf(wj, v[e], acc[i][e]);
            }
        }
    }

#pragma unroll
    for (int i = 0; i < kGenQW; ++i) {
        const int q = q0 + wave * kGenQW + i;
        if (q >= S) break;  // wave-uniform
        const float inv = 1.f / l[i];
        const size_t orow =
            bshd ? ((size_t)(bh / heads) * S + q) * heads + (size_t)(bh % heads) : base + q;
        float y[kGenDims];
#pragma unroll
        for (int e = 0; e < kGenDims; ++e) y[e] = __half2float(f16_of_f32(acc[i][e] * inv));
        if (qout != nullptr) {
            float am = 0.f;
#pragma unroll
            for (int e = 0; e < kGenDims; ++e)
                if (e < nd && lane + 64 * e < D) am = fmaxf(am, fabsf(y[e]));
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) am = fmaxf(am, __shfl_xor(am, off));
            const float sc = fmaxf(am, 1e-8f) / 127.f;
#pragma unroll
            for (int e = 0; e < kGenDims; ++e) {
                const int d = lane + 64 * e;
                if (e < nd && d < D) qout[orow * D + d] = (int8_t)quant_code(y[e], sc);
            }
            if (lane == 0) qout_scale[orow] = sc;
        } else {
#pragma unroll
            for (int e = 0; e < kGenDims; ++e) {
                const int d = lane + 64 * e;
                if (e < nd && d < D) out[orow * D + d] = f32_to_f16_bits(y[e]);
            }
        }
    }
}

// D: the kernel's head_dim; dm: the head_dim of the rows in memory (dm <= D,
// a multiple of 16; dm < D runs the padded instance).
template <int D, int QW, int KG>
int launch_prefill_shape(const int8_t* Q, const int8_t* K, const int8_t* V, uint16_t* out,
                         int8_t* qout, float* qscale, const float* sQ, const float* sK,
                         const float* sV, int BH, int heads, int S, int dm, bool causal, bool bshd,
                         hipStream_t stream) {
    constexpr int kQ = Shape<D, QW, KG>::kQ, kThreads = Shape<D, QW, KG>::kThreads;
    const int n_qtiles = (S + kQ - 1) / kQ;
    const long long blocks = (long long)BH * n_qtiles;
    const float qk = (1.0f / std::sqrt((float)dm)) * kLog2e;
    const int lds = KG * 2 * Stage<D, QW>::kBytes;
    static PerDeviceOnce lds_once;
    const int st = set_lds_limit(
        lds_once, lds, prefill_kernel<D, QW, KG, true, false>, prefill_kernel<D, QW, KG, false, false>,
        prefill_kernel<D, QW, KG, true, true>, prefill_kernel<D, QW, KG, false, true>);
    if (st != INT8K_OK) return st;
    const int b = bshd ? 1 : 0;
#define INT8K_PREFILL_LAUNCH(C, P)                                                         \
    prefill_kernel<D, QW, KG, C, P><<<(unsigned)blocks, kThreads, lds, stream>>>(          \
        Q, K, V, sQ, sK, sV, out, qout, qscale, S, n_qtiles, qk, heads, b, dm)
    if (dm == D) {
        if (causal) INT8K_PREFILL_LAUNCH(true, false);
        else INT8K_PREFILL_LAUNCH(false, false);
    } else {
        if (causal) INT8K_PREFILL_LAUNCH(true, true);
        else INT8K_PREFILL_LAUNCH(false, true);
    }
#undef INT8K_PREFILL_LAUNCH
    return check_launch("prefill_kernel");
}

template <int D>
int launch_prefill(const int8_t* Q, const int8_t* K, const int8_t* V, uint16_t* out,
                   int8_t* qout, float* qscale, const float* sQ, const float* sK, const float* sV,
                   int BH, int heads, int S, int dm, bool causal, bool bshd, hipStream_t stream) {
#define INT8K_PREFILL_SHAPE(I)                                                                   \
    return launch_prefill_shape<D, kShapes<D>[I].qw, kShapes<D>[I].kg>(                          \
        Q, K, V, out, qout, qscale, sQ, sK, sV, BH, heads, S, dm, causal, bshd, stream)
    if constexpr (D <= 128) {
        const int pick = pick_shape<D>(BH, S, causal);
        if (pick == 1) INT8K_PREFILL_SHAPE(1);
        if (pick == 2) INT8K_PREFILL_SHAPE(2);
    }
    INT8K_PREFILL_SHAPE(0);
#undef INT8K_PREFILL_SHAPE
}

int launch_prefill_generic(const int8_t* Q, const int8_t* K, const int8_t* V, uint16_t* out,
                           int8_t* qout, float* qscale, const float* sQ, const float* sK,
                           const float* sV, int BH, int heads, int S, int D, bool causal,
                           bool bshd, hipStream_t stream) {
    const int n_qtiles = (S + kGenQ - 1) / kGenQ;
    const long long blocks = (long long)BH * n_qtiles;
    const float qk = (1.0f / std::sqrt((float)D)) * kLog2e;
    static PerDeviceOnce lds_once;
    const int st = set_lds_limit(lds_once, gen_layout(kGenMaxD).bytes,
                                 prefill_generic_kernel<true>, prefill_generic_kernel<false>);
    if (st != INT8K_OK) return st;
    const int lds = gen_layout(D).bytes;
    if (causal)
        prefill_generic_kernel<true><<<(unsigned)blocks, 256, lds, stream>>>(
            Q, K, V, sQ, sK, sV, out, qout, qscale, S, D, n_qtiles, qk, heads, bshd ? 1 : 0);
    else
        prefill_generic_kernel<false><<<(unsigned)blocks, 256, lds, stream>>>(
            Q, K, V, sQ, sK, sV, out, qout, qscale, S, D, n_qtiles, qk, heads, bshd ? 1 : 0);
    return check_launch("prefill_generic_kernel");
}

// Shared checks and dispatch of both entry points: exactly one of out
// (fp16) and qout/qscale (int8 + per-token scale) is set.
int prefill_entry(const int8_t* Q, const int8_t* K, const int8_t* V, uint16_t* out, int8_t* qout,
                  float* qscale, const float* scale_Q, const float* scale_K, const float* scale_V,
                  int batch, int heads, int seq_len, int head_dim, int flags, void* stream) {
    if (!Q || !K || !V || !scale_Q || !scale_K || !scale_V) return INT8K_ERR_INVALID_ARGUMENT;
    if (flags & ~(INT8K_ATTN_CAUSAL | INT8K_ATTN_OUT_BSHD)) return INT8K_ERR_INVALID_ARGUMENT;
    if (batch <= 0 || heads <= 0 || seq_len <= 0 || head_dim <= 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (head_dim > kGenMaxD) return INT8K_ERR_UNSUPPORTED;
    const long long BH = (long long)batch * heads;
    const bool mfma = on_mfma(head_dim);
    // work-items of the launch: 2 threads per query (MFMA kernel), 16 (generic)
    if (BH * (((long long)seq_len + 127) / 128) * 256 >= (1LL << 32)) return INT8K_ERR_UNSUPPORTED;
    if (!mfma && BH * (((long long)seq_len + kGenQ - 1) / kGenQ) * 256 >= (1LL << 32))
        return INT8K_ERR_UNSUPPORTED;
    if ((long long)seq_len * head_dim >= (1LL << 32)) return INT8K_ERR_UNSUPPORTED;  // buffer range
    if (!aligned_to(scale_Q, 4) || !aligned_to(scale_K, 4) || !aligned_to(scale_V, 4))
        return INT8K_ERR_MISALIGNED;
    if (mfma) {
        if (!aligned_to(Q, 16) || !aligned_to(K, 16) || !aligned_to(V, 16))
            return INT8K_ERR_MISALIGNED;
        if (out ? !aligned_to(out, 8) : !(aligned_to(qout, 4) && aligned_to(qscale, 4)))
            return INT8K_ERR_MISALIGNED;
    } else if (out ? !aligned_to(out, 2) : !aligned_to(qscale, 4)) {
        return INT8K_ERR_MISALIGNED;
    }
    hipStream_t s = as_stream(stream);
    const bool c = (flags & INT8K_ATTN_CAUSAL) != 0, bshd = (flags & INT8K_ATTN_OUT_BSHD) != 0;
    if (!mfma)
        return launch_prefill_generic(Q, K, V, out, qout, qscale, scale_Q, scale_K, scale_V,
                                      (int)BH, heads, seq_len, head_dim, c, bshd, s);
    if (head_dim <= 64)
        return launch_prefill<64>(Q, K, V, out, qout, qscale, scale_Q, scale_K, scale_V, (int)BH,
                                  heads, seq_len, head_dim, c, bshd, s);
    if (head_dim <= 128)
        return launch_prefill<128>(Q, K, V, out, qout, qscale, scale_Q, scale_K, scale_V,
                                   (int)BH, heads, seq_len, head_dim, c, bshd, s);
    return launch_prefill<256>(Q, K, V, out, qout, qscale, scale_Q, scale_K, scale_V, (int)BH,
                               heads, seq_len, head_dim, c, bshd, s);
}

}  // namespace
}  // namespace int8k

using namespace int8k;

extern "C" int int8k_attention_block_shape(int BH, int seq_len, int head_dim, int flags,
                                           int* query_waves, int* key_groups) {
    clear_last_error();
    if (BH <= 0 || seq_len <= 0 || head_dim <= 0 || !query_waves || !key_groups ||
        (flags & ~(INT8K_ATTN_CAUSAL | INT8K_ATTN_OUT_BSHD)) != 0)
        return INT8K_ERR_INVALID_ARGUMENT;
    if (!on_mfma(head_dim)) return INT8K_ERR_UNSUPPORTED;
    const bool c = (flags & INT8K_ATTN_CAUSAL) != 0;
    const ShapeCost& sh = head_dim <= 64    ? kShapes<64>[pick_shape<64>(BH, seq_len, c)]
                          : head_dim <= 128 ? kShapes<128>[pick_shape<128>(BH, seq_len, c)]
                                            : kShapes<256>[0];
    *query_waves = sh.qw;
    *key_groups = sh.kg;
    return INT8K_OK;
}

extern "C" int int8k_attention_forward(const int8_t* Q, const int8_t* K, const int8_t* V,
                                       uint16_t* out, const float* scale_Q, const float* scale_K,
                                       const float* scale_V, int batch, int heads, int seq_len,
                                       int head_dim, int flags, void* stream) {
    clear_last_error();
    if (!out) return INT8K_ERR_INVALID_ARGUMENT;
    return prefill_entry(Q, K, V, out, nullptr, nullptr, scale_Q, scale_K, scale_V, batch, heads,
                         seq_len, head_dim, flags, stream);
}

extern "C" int int8k_attention_forward_quant(const int8_t* Q, const int8_t* K, const int8_t* V,
                                             int8_t* out_q, float* out_scale,
                                             const float* scale_Q, const float* scale_K,
                                             const float* scale_V, int batch, int heads,
                                             int seq_len, int head_dim, int flags,
                                             void* stream) {
    clear_last_error();
    if (!out_q || !out_scale) return INT8K_ERR_INVALID_ARGUMENT;
    return prefill_entry(Q, K, V, nullptr, out_q, out_scale, scale_Q, scale_K, scale_V, batch,
                         heads, seq_len, head_dim, flags, stream);
}
