// linear.hip — INT8 matrix product with a scale per token and per output channel, gfx950.
//
//   y[t, n] = T( (f32(acc) * sx[t]) * sw[n] (+ b[n]) ),  acc = sum_k x[t, k] w[k, n], exact int32
//
// x int8 [T, K]; w int8 [K, N] as stored, or [N, K] packed; y fp16, bf16 or fp32, rounded once
// from the fp32 value.  The products run on the GEMM core of gemm_i8.h.
#include "gemm_i8.h"
#include "rows.h"

namespace int8k {
namespace {

using namespace gemm;

struct LinearArgs {
    const int8_t *x, *w;
    void* y;
    const float *sx, *sw, *bias;
    int sx_stride, sw_stride;  // 0: one scale for all
    int M, N, K;
};

template <int DT>
__device__ __forceinline__ void store_value(void* y, size_t i, float v) {
    if constexpr (DT == INT8K_DTYPE_F32) {
        static_cast<float*>(y)[i] = v;
    } else if constexpr (DT == INT8K_DTYPE_F16) {
        static_cast<uint16_t*>(y)[i] = __half_as_ushort(f16_of_f32(v));
    } else {
        const uint32_t u = __float_as_uint(v);
        static_cast<uint16_t*>(y)[i] =
            (uint16_t)(v != v ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
}

// 256 x 256 tiles.
template <int DT, bool BKN>
__global__ __launch_bounds__(kThreads, 1) void linear_tiled_kernel(LinearArgs p, int tiles_m,
                                                                   int tiles_n) {
    extern __shared__ __align__(16) char lds[];
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    v16i acc[TM][TN];
    const int ldb = BKN ? p.N : p.K;
    if (m0 + BM <= p.M && n0 + BN <= p.N && p.K % BK == 0)
        mainloop<false, false, BKN>(acc, p.x, p.w, p.M, p.N, p.K, p.K, ldb, m0, n0, lds);
    else
        mainloop<true, false, BKN>(acc, p.x, p.w, p.M, p.N, p.K, p.K, ldb, m0, n0, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rbase = m0 + (wave >> 1) * WM, cbase = n0 + (wave & 1) * WN + (lane & 31);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int col = cbase + j * 32;
        if (col >= p.N) continue;
        const float sb = p.sw[(size_t)col * p.sw_stride];
        const float bi = p.bias != nullptr ? p.bias[col] : 0.f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = rbase + i * 32 + acc_row(r, lane);
                if (row >= p.M) continue;
                const float v = static_cast<float>(acc[i][j][r]) * p.sx[(size_t)row * p.sx_stride] * sb + bi;
                store_value<DT>(p.y, (size_t)row * p.N + col, v);
            }
    }
}

template <int DT, bool BKN>
int launch_linear_tiled(const LinearArgs& p, hipStream_t stream) {
    static PerDeviceOnce lds_once;
    const int st = lds_once.run([] {
        const hipError_t e = hipFuncSetAttribute(
            reinterpret_cast<const void*>(&linear_tiled_kernel<DT, BKN>),
            hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
        if (e != hipSuccess) {
            set_last_error("hipFuncSetAttribute", e);
            return (int)INT8K_ERR_HIP;
        }
        return (int)INT8K_OK;
    });
    if (st != INT8K_OK) return st;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    linear_tiled_kernel<DT, BKN><<<tiles_m * tiles_n, kThreads, LDS_BYTES, stream>>>(p, tiles_m, tiles_n);
    return check_launch("linear_tiled_kernel");
}

// |x w| <= 2^14 and K products: below 2^17 of them the int32 sum cannot overflow.
constexpr int kMaxK = (1 << 17) - 16;

}  // namespace
}  // namespace int8k

using namespace int8k;

extern "C" size_t int8k_linear_workspace_bytes(int T, int K, int N, int flags) {
    (void)T, (void)K, (void)N, (void)flags;
    return 0;
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
    if (K % 16 || N % 16 || K > kMaxK) return INT8K_ERR_UNSUPPORTED;
    // operands are read through 32-bit buffer offsets
    if ((long long)T * K >= (1LL << 32) || (long long)N * K >= (1LL << 32))
        return INT8K_ERR_UNSUPPORTED;
    if (ceil_div(T, BM) * ceil_div(N, BN) >= (1LL << 24)) return INT8K_ERR_UNSUPPORTED;
    if (!aligned_to(x, 16) || !aligned_to(W, 16) || !aligned_to(out, 16) ||
        !aligned_to(scale_x, 4) || !aligned_to(scale_W, 4) || !aligned_to(bias, 4))
        return INT8K_ERR_MISALIGNED;
    (void)workspace, (void)workspace_bytes;
    const LinearArgs p{x, W, out, scale_x, scale_W, bias, n_scale_x == 1 ? 0 : 1,
                       n_scale_W == 1 ? 0 : 1, T, N, K};
    const bool packed = (flags & INT8K_LINEAR_WEIGHT_PREPACKED) != 0;
    int st = INT8K_OK;
    with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        st = packed ? launch_linear_tiled<DT, false>(p, as_stream(stream))
                    : launch_linear_tiled<DT, true>(p, as_stream(stream));
    });
    return st;
}
