// packed.hip — INT8 flash attention over packed prompts of different lengths, with grouped
// heads, gfx950.
//
//   Q int8 [heads, T, D], K, V int8 [kv_heads, T, D], per-token scales [heads or kv_heads, T];
//   sequence i holds the tokens cu_seqlens[i] .. cu_seqlens[i+1]-1 of every head, and query
//   head h reads key head h / (heads / kv_heads).  Inside a sequence the math is
//   int8_attention_forward's (prefill.hip):
//     s_ij = (q_i . k_j) sQ_i sK_j / sqrt(D),  out_i = sum_j softmax_j(s_ij) v_j sV_j
//
// The block is prefill_block (prefill_core.h) on one query tile of one head of one sequence.
// The lengths are on the device, so the grid is sized for the most tiles that T tokens of n
// sequences can have (T / kQ + n) and each wave finds its tile from the lengths itself: a
// plan kernel would cost a launch of its own.  Tiles are taken in the order of their index
// inside their sequence, the highest first: under the causal mask that is heaviest first
// over all sequences, so short ones fill the end of the grid.
#include "prefill_core.h"

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

// The query tile that rank `i` of the packed order is: sequence tokens [start, start + len),
// tile qt of them.  False past the last tile; `i` is then the rank behind it.
struct PackedTile {
    int start, len, qt;
};
template <int kQ>
__device__ __forceinline__ bool packed_tile(const int32_t* __restrict__ cu, int n, int T, int& i,
                                            PackedTile& t) {
    const int lane = threadIdx.x & 63;
    // start and length of this lane's sequence s0 + lane; lengths that would leave the T
    // tokens are cut, so no offsets lead outside the tensors
    auto bounds = [&](int s0, int& c0, int& len) {
        const int s = min(s0 + lane, n - 1);
        c0 = min(max(cu[s], 0), T);
        len = s0 + lane < n ? min(max(cu[s + 1], c0), T) - c0 : 0;
    };
    int c0, len;
    bounds(0, c0, len);
    const int first = (len + kQ - 1) / kQ;  // tiles of the first 64 sequences, kept
    auto tiles_of = [&](int s0) {
        if (s0 == 0) return first;
        int c, l;
        bounds(s0, c, l);
        return (l + kQ - 1) / kQ;
    };
    // tiles with index >= k
    auto count = [&](int k) {
        int c = 0;
        for (int s0 = 0; s0 < n; s0 += 64) c += wave_sum(max(tiles_of(s0) - k, 0));
        return c;
    };
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
    int j = i - count(lo + 1);  // the j-th sequence that has a tile of that index
    for (int s0 = 0; s0 < n; s0 += 64) {
        const bool has = tiles_of(s0) > lo;
        const uint64_t mask = __ballot(has);
        const int here = __popcll(mask);
        if (j >= here) {
            j -= here;
            continue;
        }
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        const int src = __builtin_ctzll(__ballot(has && rank == j));
        if (s0 > 0) bounds(s0, c0, len);
        t.start = __builtin_amdgcn_readlane(c0, src);
        t.len = __builtin_amdgcn_readlane(len, src);
        t.qt = lo;
        return true;
    }
    return false;  // not reached: the ranks below `total` all have a sequence
}

// zero_rest: the rows of out that no sequence holds are written as zeros by the blocks that
// have no tile (the grid has one rank more than there can be tiles).
template <int D, int QW, int KG, bool CAUSAL, bool PAD>
__global__ __launch_bounds__((Shape<D, QW, KG>::kThreads), (Shape<D, QW, KG>::kMinBlocks)) void packed_kernel(
    const int8_t* __restrict__ Q, const int8_t* __restrict__ K, const int8_t* __restrict__ V,
    const float* __restrict__ sQ, const float* __restrict__ sK, const float* __restrict__ sV,
    uint16_t* __restrict__ out, const int32_t* __restrict__ cu, int n, int T, int heads,
    int group, float qk_scale_log2, int thd, int zero_rest, int d_mem) {
    extern __shared__ __align__(16) char smem_all[];
    const int dm = PAD ? d_mem : D;
    int rank = (int)blockIdx.x / heads;
    const int ranks = (int)gridDim.x / heads;
    const int h = (int)blockIdx.x % heads;
    PackedTile t;
    const int wanted = rank;
    if (!packed_tile<Shape<D, QW, KG>::kQ>(cu, n, T, rank, t)) {
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
    prefill_block<D, QW, KG, CAUSAL, PAD>(
        smem_all, Q + qrow * dm, K + krow * dm, V + krow * dm, sQ + qrow, sK + krow, sV + krow,
        out, nullptr, nullptr, t.len, t.qt, qk_scale_log2, d_mem, [&](int q) {
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

template <int D, int QW, int KG>
int launch_packed_shape(const PackedArgs& a, hipStream_t stream) {
    constexpr int kQ = Shape<D, QW, KG>::kQ, kThreads = Shape<D, QW, KG>::kThreads;
    const long long ranks = (long long)a.T / kQ + a.n + 1;
    const float qk = (1.0f / std::sqrt((float)a.dm)) * kLog2e;
    const int lds = KG * 2 * Stage<D, QW>::kBytes;
    if (ranks * a.heads * kThreads >= (1LL << 32)) return INT8K_ERR_UNSUPPORTED;
    static PerDeviceOnce lds_once;
    const int st = set_lds_limit(
        lds_once, lds, packed_kernel<D, QW, KG, true, false>, packed_kernel<D, QW, KG, false, false>,
        packed_kernel<D, QW, KG, true, true>, packed_kernel<D, QW, KG, false, true>);
    if (st != INT8K_OK) return st;
    const unsigned blocks = (unsigned)(ranks * a.heads);
#define INT8K_PACKED_LAUNCH(C, P)                                                               \
    packed_kernel<D, QW, KG, C, P><<<blocks, kThreads, lds, stream>>>(                          \
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

template <int D>
int launch_packed(const PackedArgs& a, hipStream_t stream) {
#define INT8K_PACKED_SHAPE(I) \
    return launch_packed_shape<D, kShapes<D>[I].qw, kShapes<D>[I].kg>(a, stream)
    INT8K_PACKED_SHAPE(0);
#undef INT8K_PACKED_SHAPE
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
    if (!on_mfma(head_dim)) return INT8K_ERR_UNSUPPORTED;
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
