// prefill_tiles.h — how the MFMA attention kernels over whole prompts (prefill.hip, packed.hip)
// load K and V tiles and lay them out in LDS (internal header).
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "int8k_common.h"
#include "rows.h"

namespace int8k {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kKV = 64;  // keys per tile
// Block shapes: QW waves of 32 queries each, times KG groups of waves that share
// the queries and walk every KG-th tile, each group with its own stages; the
// groups' (l, O) are added in LDS at the end.  Large grids run KG = 1: D = 128 with
// 8 waves (256 queries) at 2 waves per SIMD, so each staged K/V tile serves 256
// queries; D = 64 with 4 waves (a 64-key tile has only 256 K chunks of 16 B); D = 256
// with 4 waves at one wave per SIMD for its register budget.  Grids that leave CUs
// idle split the keys of fewer queries over the groups (pick_shape).
template <int D>
constexpr int kOneGroupWaves = D == 128 ? 8 : 4;
template <int D, int QW, int KG = 1>
struct Shape {
    static constexpr int kGroupThreads = 64 * QW;
    static constexpr int kThreads = 64 * QW * KG;
    static constexpr int kQ = 32 * QW;  // queries per block
    static constexpr int kMinBlocks = D == 64 && QW * KG == 4 ? 2 : 1;  // 2 waves per SIMD at D <= 128
};

// V' is staged as it arrives, row-major fp16 [key][dim], and the PV MFMA's
// V^T fragments are formed by transposing LDS reads (ds_read_b64_tr_b16).
// Measured: in each group of 16 lanes, the instruction gives lane
// 4h + e half e of the 8-byte rows that lanes h, h+4, h+8, h+12 address.  So
// lane 16G + 4k + h of a wave addresses key row 4 (G/2) + k and dims
// 16 (G%2) + 4h of a 16-key slice, and lane l then holds dim l % 32 of keys
// 4 (l/32) + 0..3: the first half of its fragment; a read 8 rows further
// gives the second (see tile_pv).  Rows hold D + 32 halfs (2D + 64 bytes, 64
// or 192 mod 256), so the 4 rows a half-wave reads fall in 4 different 64-byte
// bank groups.
//
// Work item n of thread t is the 4x4 block of keys 4 kg .. 4 kg + 3 and dims
// 4 dg .. 4 dg + 3 with kg = t / W, dg = t % W + n W, where W = D / 4 / items
// per thread (32 at D = 128, 16 at D = 64 and 256): dim groups run fastest, so
// a wave's loads of one key cover whole 64- or 128-byte runs of rows in memory
// and its LDS writes whole runs of staged rows, and a thread's items share
// their keys (one sV vector).
template <int D, int QW>
struct VLayout {
    static constexpr int kRow = D + 32;  // halfs per staged row
    static constexpr int kItems = 64 * D / 16 / Shape<D, QW>::kGroupThreads;
    static constexpr int kW = D / 4 / kItems;  // dim groups per item row
};

// One LDS stage: K tile (int8 rows, 16-byte padded), V' tile (fp16 [key][dim],
// the V scales applied), the key scales sK.
template <int D, int QW>
struct Stage {
    static constexpr int kKStride = D + 16;  // bytes per K row
    static constexpr int kKBytes = kKV * kKStride;
    static constexpr int kVtBytes = kKV * VLayout<D, QW>::kRow * 2;
    static constexpr int kBytes = kKBytes + kVtBytes + kKV * 4;
    static constexpr int kKChunks = kKV * D / 16 / Shape<D, QW>::kGroupThreads;  // 16-B K chunks per thread
    static constexpr int kVItems = kKV * D / 16 / Shape<D, QW>::kGroupThreads;   // 4x4 V blocks per thread
    static_assert(kKChunks >= 1 && kKChunks * 16 * Shape<D, QW>::kGroupThreads == kKV * D, "K tile split");
    static_assert(kVItems >= 1 && kVItems * 16 * Shape<D, QW>::kGroupThreads == kKV * D, "V tile split");
};

// Buffer resources over one (b,h)'s K, V and scales.  Rows at or past S read
// as zero, so the tile loads need no clamping; masked keys never reach the
// output.  `dm` is the head_dim of the rows in memory; a padded kernel
// (dm < D) loads only the K chunks and V dim groups below dm and zeroes the
// rest (kvalid, vvalid).
struct TileSrc {
    __amdgpu_buffer_rsrc_t k, s, sv;
    v4i v;  // V descriptor with a typed format: 8_8_8_8 SSCALED (see load_v_f16x4)
    uint32_t voff_k, voff_v, voff_s, voff_sv;
    uint32_t kstep, dm;  // bytes between K chunks n and n+1; row stride in memory
    bool kvalid;
    uint32_t vvalid;  // bit n: item n has dims below dm
};

// A buffer descriptor whose loads convert: data format 8_8_8_8 with numeric
// format SSCALED turns each byte into the float of its signed value, and the
// d16 variant of the format load packs the four as fp16.  So V arrives as exact
// fp16 with no VALU work.  Offsets at or past `bytes` read as zero.
__device__ __forceinline__ v4i make_v_descriptor(const void* base, uint32_t bytes) {
    constexpr uint32_t kDstSelXYZW = 4 | (5 << 3) | (6 << 6) | (7 << 9);
    constexpr uint32_t kNumFormatSscaled = 3, kDataFormat8888 = 10;
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    v4i d;
    d.x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b));
    d.y = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b >> 32) & 0xffffu);  // stride 0
    d.z = __builtin_amdgcn_readfirstlane(bytes);
    d.w = kDstSelXYZW | (kNumFormatSscaled << 12) | (kDataFormat8888 << 15);
    return d;
}

// The LLVM intrinsic behind the typed ("format") raw buffer load, which clang
// exposes no builtin for; declared by name so the compiler schedules it and
// tracks its wait counts like any other load.
typedef _Float16 v4h_t __attribute__((ext_vector_type(4)));
extern "C" __device__ v4h_t int8k_raw_buffer_load_format_v4f16(v4i rsrc, int voffset, int soffset,
                                                              int aux)
    __asm("llvm.amdgcn.raw.buffer.load.format.v4f16");

// Four int8 at voff + soff as four fp16, packed {b0, b1} {b2, b3}.
__device__ __forceinline__ uint2 load_v_f16x4(const v4i& desc, uint32_t voff, uint32_t soff) {
    const v4h_t h = int8k_raw_buffer_load_format_v4f16(desc, (int)voff, (int)soff, 0);
    typedef uint32_t v2u __attribute__((ext_vector_type(2)));
    const v2u r = __builtin_bit_cast(v2u, h);
    return make_uint2(r.x, r.y);
}

// t: thread within its group.
template <int D, int QW>
__device__ __forceinline__ TileSrc make_tile_src(const int8_t* Kbh, const int8_t* Vbh,
                                                 const float* sKbh, const float* sVbh, int S,
                                                 int dm, int t) {
    constexpr int kT = Shape<D, QW>::kGroupThreads;
    TileSrc src;
    src.dm = (uint32_t)dm;
    src.k = make_buffer(Kbh, (uint32_t)S * dm);
    src.v = make_v_descriptor(Vbh, (uint32_t)S * dm);
    src.s = make_buffer(sKbh, (uint32_t)S * 4);    // the group's first wave loads the tile's sK
    src.sv = make_buffer(sVbh, (uint32_t)S * 4);   // every thread: sV of its 4 V keys
    const int kcol = (t % (D / 16)) * 16;
    src.voff_k = (t / (D / 16)) * dm + kcol;
    src.kstep = (uint32_t)(kT * 16 / D) * dm;  // chunk t + n kT is kT*16/D rows further
    src.kvalid = kcol < dm;
    using VL = VLayout<D, QW>;
    const int dg = t % VL::kW, kg = t / VL::kW;
    src.voff_v = 4 * kg * dm + 4 * dg;
    src.vvalid = 0;
#pragma unroll
    for (int n = 0; n < VL::kItems; ++n)
        if (4 * (dg + n * VL::kW) < dm) src.vvalid |= 1u << n;
    src.voff_s = (t & (kKV - 1)) * 4;
    src.voff_sv = 16 * kg;
    return src;
}

// Dynamic LDS above 64 KiB needs the attribute, once per device and kernel.
template <typename... Kernels>
int set_lds_limit(PerDeviceOnce& once, int bytes, Kernels... kernels) {
    return once.run([=] {
        hipError_t e = hipSuccess;
        for (const void* k : {reinterpret_cast<const void*>(kernels)...}) {
            if (e == hipSuccess)
                e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        }
        if (e != hipSuccess) {
            set_last_error("hipFuncSetAttribute", e);
            return (int)INT8K_ERR_HIP;
        }
        return (int)INT8K_OK;
    });
}

// Head dims of the MFMA kernel; the generic one takes the others.
inline bool on_mfma(int head_dim) { return head_dim % 16 == 0 && head_dim <= 256; }

}  // namespace
}  // namespace int8k
