// vkb_rms_norm: r = x + residual, y = r / sqrt(mean(r^2) + eps) * w, and optionally y's Q8 form (one fp16 scale per 32
// values, vkb.h). The sum of squares, the norm and the product with w are fp32 on the unrounded r; each output is
// rounded once.
//
// HBM-bound: every input element is read once and every output written once. A row belongs to one group of threads:
// thread t holds the vectors of eight t, t + threads, ... in registers between the reduction and the output, so the
// row is not read again; rows of up to 512 elements, and wider ones where there are thousands, take one warp each (no
// block-wide barrier), four rows to a block. Measured on a B200, bf16 with residual in and out: 8191 x 2560 in 34 us, 4.9
// TB/s, with the Q8 copy 42 us.
// Rows that are not made of aligned vectors of eight (odd widths, odd strides) or are wider than 16384 go element by element
// and read their inputs a second time (from L1 / L2) instead of holding them: 8191 x 2561 in 119 us, 1.4 TB/s, bound by the
// issue of 2-byte loads and stores; 1024 x 20480 in 55 us. They are the exception that has to be right; rows that a user lays
// out for speed are aligned.
#include "step.cuh"

namespace vkb {

struct NormArgs {
    const void* x;
    const void* res;
    void* res_out;
    const void* w;
    void* y;
    int8_t* q;
    __half* s;
    long long ldx;
    float eps, inv_d;
    int T, d;
};

constexpr int NORM_NV = 2;    // vectors of eight a thread holds (1024 threads x 2 x 8 = 16384 elements)
constexpr int NORM_WNV = 10;  // and where a warp takes a row of its own (rows of up to 2560 elements)

// Sum over the threads of one row: a warp, or the whole block (blockDim.y == 1).
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = warp_sum(v);
    if (blockDim.x == 32) return v;
    const int nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = (threadIdx.x & 31) < nw ? red[threadIdx.x & 31] : 0.f;
    return warp_sum(t);
}

// One fp16 scale and int8 codes of a group whose largest magnitude is amax, by vkb_quantize's rule: d = fp16(amax / 127),
// code = round(v * (1 / d)) with halves away from zero, clamped to +-127.
__device__ __forceinline__ __half q8_scale(float amax) { return __float2half_rn(__fdiv_rn(amax, 127.f)); }
__device__ __forceinline__ float q8_inv(__half d) {
    const float f = __half2float(d);
    return f != 0.f ? __fdiv_rn(1.f, f) : 0.f;
}
__device__ __forceinline__ int q8_code(float v, float inv) {
    return (int)fminf(127.f, fmaxf(-127.f, roundf(v * inv)));
}

// X, R: element types of x / w / y and of the residual (R = -1: none). NV: vectors a thread holds; WARP: a row per warp,
// whose weights are read when they are needed (the row itself fills the registers).
template <int X, int R, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) norm_vec_kernel(const NormArgs a) {
    using TX = typename Elem<X>::T;
    constexpr int RD = R < 0 ? 0 : R;
    using TR = typename Elem<RD>::T;
    __shared__ float red[32];
    const int row = blockIdx.x * blockDim.y + threadIdx.y;
    const int nvec = a.d >> 3, tpr = WARP ? 32 : blockDim.x;
    pdl_trigger();
    Raw8<X> w[WARP ? 1 : NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * tpr;
        if (!WARP && i < nvec) prefetch_l2(reinterpret_cast<const TX*>(a.w) + 8 * i);
    }
    pdl_wait();
    if (row >= a.T) return;   // whole warps: a row's threads leave together
    const TX* x = reinterpret_cast<const TX*>(a.x) + row * a.ldx;
    const long long base = (long long)row * a.d;
    Raw8<X> rx[NV];
    Raw8<RD> rr[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * tpr;
        if (i < nvec) {
            raw8_load<X>(rx[j], x + 8 * i);
            if constexpr (R >= 0) raw8_load<RD>(rr[j], reinterpret_cast<const TR*>(a.res) + base + 8 * i);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * tpr;
        if (!WARP && i < nvec) raw8_load<X>(w[WARP ? 0 : j], reinterpret_cast<const TX*>(a.w) + 8 * i);
    }
    float f[NV][8], ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * tpr;
        if (i >= nvec) continue;
        raw8_to<X>(rx[j], f[j]);
        if constexpr (R >= 0) {
            float r[8];
            raw8_to<RD>(rr[j], r);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[j][e] += r[e];
            if (a.res_out) store8<RD>(reinterpret_cast<TR*>(a.res_out) + base + 8 * i, f[j]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[j][e], f[j][e], ss);
    }
    ss = row_sum(ss, red);
    const float rs = __fdiv_rn(1.f, __fsqrt_rn(fmaf(ss, a.inv_d, a.eps)));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * tpr;
        const bool on = i < nvec;
        float amax = 0.f;
        if (on) {
            float g[8];
            if (WARP) raw8_load<X>(w[0], reinterpret_cast<const TX*>(a.w) + 8 * i);
            raw8_to<X>(w[WARP ? 0 : j], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[j][e] = f[j][e] * rs * g[e];
                amax = fmaxf(amax, fabsf(f[j][e]));
            }
            if (a.y) store8<X>(reinterpret_cast<TX*>(a.y) + base + 8 * i, f[j]);
        }
        if (a.q) {   // a group of 32 is four neighbouring lanes (d % 32 == 0: they are in or out together)
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            if (on) {
                const __half d = q8_scale(amax);
                const float inv = q8_inv(d);
                uint32_t c[2] = {0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e >> 2] |= (uint32_t)(q8_code(f[j][e], inv) & 255) << (8 * (e & 3));
                *reinterpret_cast<uint2*>(a.q + base + 8 * i) = make_uint2(c[0], c[1]);
                if ((i & 3) == 0) a.s[(base + 8 * i) >> 5] = d;
            }
        }
    }
}

// Any width, stride and alignment: element i of a row belongs to thread i % threads; two passes over the inputs.
template <int X, int R>
__global__ void __launch_bounds__(1024) norm_any_kernel(const NormArgs a) {
    using TX = typename Elem<X>::T;
    constexpr int RD = R < 0 ? 0 : R;
    using TR = typename Elem<RD>::T;
    __shared__ float red[32];
    const int row = blockIdx.x * blockDim.y + threadIdx.y, tpr = blockDim.x;
    pdl_trigger();
    pdl_wait();
    if (row >= a.T) return;
    const TX* x = reinterpret_cast<const TX*>(a.x) + row * a.ldx;
    const TX* w = reinterpret_cast<const TX*>(a.w);
    const long long base = (long long)row * a.d;
    const TR* res = reinterpret_cast<const TR*>(a.res) + base;
    auto value = [&](int i) {
        float v = Elem<X>::to(x[i]);
        if constexpr (R >= 0) v += Elem<RD>::to(res[i]);
        return v;
    };
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.d; i += tpr) {
        const float v = value(i);
        ss = fmaf(v, v, ss);
    }
    ss = row_sum(ss, red);
    const float rs = __fdiv_rn(1.f, __fsqrt_rn(fmaf(ss, a.inv_d, a.eps)));
    for (int i = threadIdx.x; i < a.d; i += tpr) {
        const float r = value(i), v = r * rs * Elem<X>::to(w[i]);
        if constexpr (R >= 0)
            if (a.res_out) reinterpret_cast<TR*>(a.res_out)[base + i] = Elem<RD>::from(r);
        if (a.y) reinterpret_cast<TX*>(a.y)[base + i] = Elem<X>::from(v);
        if (a.q) {   // a warp's 32 consecutive elements are one group (d % 32 == 0: whole warps)
            const __half d = q8_scale(warp_max(fabsf(v)));
            a.q[base + i] = (int8_t)q8_code(v, q8_inv(d));
            if ((i & 31) == 0) a.s[(base + i) >> 5] = d;
        }
    }
}

template <int X, int R> static int norm_launch(const NormArgs& a, bool vec, cudaStream_t st) {
    // threads per row: one vector (or element) each where that is at most 1024, a warp for short rows
    const int n = vec ? a.d / 8 : a.d;
    // A warp per row where there are rows for every SM's warps: no block-wide barrier, and a row's loads all in flight at
    // once (B200, bf16 in, residual and out: 8191 rows of 2560 take 34 us, 37 with a block per row; 2047 and 2048 rows 11 us
    // either way).
    if (vec && n > 64 && n <= 32 * NORM_WNV && a.T >= 2048) {
        const dim3 grid((unsigned)((a.T - 1) / 4 + 1)), block(32, 4);
        return launch_pdl(norm_vec_kernel<X, R, NORM_WNV, true>, grid, block, 0, st, 1, a);
    }
    const int tpr = n <= 64 ? 32 : min(1024, (n + 31) / 32 * 32);
    const int rows = tpr == 32 ? 4 : 1;
    const dim3 grid((unsigned)((a.T - 1) / rows + 1)), block((unsigned)tpr, (unsigned)rows);
    return launch_pdl(vec ? norm_vec_kernel<X, R, NORM_NV, false> : norm_any_kernel<X, R>, grid, block, 0, st, 1, a);
}

template <int X> static int norm_res(const NormArgs& a, int res_dt, bool vec, cudaStream_t st) {
    if (!a.res) return norm_launch<X, -1>(a, vec, st);
    switch (res_dt) {
        case VKB_DT_F16: return norm_launch<X, VKB_DT_F16>(a, vec, st);
        case VKB_DT_BF16: return norm_launch<X, VKB_DT_BF16>(a, vec, st);
        default: return norm_launch<X, VKB_DT_F32>(a, vec, st);
    }
}

}  // namespace vkb

using namespace vkb;

extern "C" int vkb_rms_norm(int dt, const void* x, long long ldx, const void* res, void* res_out, int res_dt,
                            const void* w, float eps, void* y, void* q, void* s, int T, int d, vkb_stream_t stream) {
    if (!dt_ok(dt) || (res && !dt_ok(res_dt)) || (res_out && !res)) return VKB_EINVAL;
    if (T < 0 || d < 1 || ldx < d || !(eps >= 0.f)) return VKB_EINVAL;
    if ((q == nullptr) != (s == nullptr)) return VKB_EINVAL;
    if (T == 0) return 0;
    if (!x || !w || (!y && !q)) return VKB_EINVAL;
    const int e = dt_size(dt), er = dt_size(res_dt);
    if (!aligned_to(x, e) || !aligned_to(w, e) || !aligned_to(y, e) || !aligned_to(s, 2) || !aligned_to(res, er) ||
        !aligned_to(res_out, er))
        return VKB_EINVAL;
    if (q && d % 32) return VKB_EUNSUPPORTED;
    const bool vec = d % 8 == 0 && d <= 8 * 1024 * NORM_NV && (ldx * e) % 16 == 0 && aligned_to(x, 16) &&
                     aligned_to(w, 16) && aligned_to(y, 16) && aligned_to(res, 16) && aligned_to(res_out, 16) &&
                     aligned_to(q, 8);
    const NormArgs a{x, res, res_out, w, y, (int8_t*)q, (__half*)s, ldx, eps, 1.f / (float)d, T, d};
    cudaStream_t st = (cudaStream_t)stream;
    switch (dt) {
        case VKB_DT_F16: return norm_res<VKB_DT_F16>(a, res_dt, vec, st);
        case VKB_DT_BF16: return norm_res<VKB_DT_BF16>(a, res_dt, vec, st);
        default: return norm_res<VKB_DT_F32>(a, res_dt, vec, st);
    }
}
