// What the decode-step kernels (norm, rotary append, attention, sampling) share: element types, vector loads, warp and
// block reductions, and the launch with programmatic dependence. Every kernel launched through launch_pdl() executes
// griddepcontrol.wait in every thread block on every path, so that a later grid's wait covers all earlier grids.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/vkb.h"
#include "ptx.cuh"
#include "vkb_internal.h"

namespace vkb {

enum : unsigned { DEV_ERR_BAD_INDEX = 16u };   // a length, offset or page index outside its array: that part skipped

// Positions and row counts stay 4096 below 2^31, so that the end of a tile, a page or a batch of tiles is still an int.
constexpr long long MAX_POSITIONS = 0x7ffff000ll;
inline int max_length(int table_ld, int page) {   // the longest sequence that a table row holds
    const long long n = (long long)table_ld * page;
    return (int)(n < MAX_POSITIONS ? n : MAX_POSITIONS);
}

template <int DT> struct Elem;
template <> struct Elem<VKB_DT_F16> {
    using T = __half;
    static __device__ __forceinline__ float to(T v) { return __half2float(v); }
    static __device__ __forceinline__ T from(float v) { return __float2half_rn(v); }
};
template <> struct Elem<VKB_DT_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float to(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<VKB_DT_F32> {
    using T = float;
    static __device__ __forceinline__ float to(T v) { return v; }
    static __device__ __forceinline__ T from(float v) { return v; }
};

__host__ __device__ constexpr int dt_size(int dt) { return dt == VKB_DT_F32 ? 4 : 2; }
inline bool dt_ok(int dt) { return dt == VKB_DT_F16 || dt == VKB_DT_BF16 || dt == VKB_DT_F32; }
__host__ __device__ inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Eight consecutive elements at a 16-byte aligned address, raw (one 16-byte load, two for fp32) and as floats.
template <int DT> struct Raw8 { uint4 a, b; };
template <int DT> __device__ __forceinline__ void raw8_load(Raw8<DT>& r, const typename Elem<DT>::T* p) {
    r.a = *reinterpret_cast<const uint4*>(p);
    if constexpr (DT == VKB_DT_F32) r.b = *reinterpret_cast<const uint4*>(p + 4);
}
template <int DT> __device__ __forceinline__ void raw8_to(const Raw8<DT>& r, float (&f)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    if constexpr (DT == VKB_DT_F32) {
        const uint32_t v[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = __uint_as_float(w[i]);
            f[4 + i] = __uint_as_float(v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == VKB_DT_F16) {
                f[2 * i] = half_lo_f32(w[i]);
                f[2 * i + 1] = half_hi_f32(w[i]);
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int DT> __device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&f)[8]) {
    if constexpr (DT == VKB_DT_F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = DT == VKB_DT_F16 ? pack_f16(f[2 * i], f[2 * i + 1]) : pack_bf16(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Launch with programmatic dependence where the thread and the stream allow it (see pdl_stream_ok). cluster > 1: a
// cluster of that many blocks along x.
template <typename... P, typename... A>
inline int launch_pdl(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (pdl_enabled() && pdl_stream_ok(st)) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)cluster;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)na;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P(args)...);
    return e == cudaSuccess ? 0 : -(int)e;
}

}  // namespace vkb
