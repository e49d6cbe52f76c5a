// The paged 8-bit cache (vkb_kv_cache_t): vkb_rope_append rotates the new tokens' q and k, and writes k and v as codes;
// vkb_kv_read returns cached tokens as values.
//
// Rotation of the pair (a, b) at position p: (a c - b s, b c + a s) with c, s = cos, sin of 2 pi (p f mod 1). f, the
// turns per position, is a 64-bit fraction of a turn, so p f mod 1 is one integer product, exact at every position; its
// top 32 bits go through cospi / sinpi in fp32 (the angle is within 2^-25 turns of exact, however long the context).
//
// A page of one head has one scale per tensor: scale = max(scale of the tokens it already holds, absmax(new) / 127),
// code = rint(x / scale). Where the scale grows, the codes held before are brought to the new one,
// rint(code * old / new): at most half a code step of the new scale is lost each time the page's maximum grows. Every
// (page, head, tensor) belongs to one block of threads, so nothing is atomic and the result does not depend on order.
// Infinities are held as +-127 and do not enter the scale; NaN is held as 0.
//
// For prompts q is read and written once, and k and v are read once where a page's values fit 40 KB of shared memory as fp32
// (page x (dim + 4) up to 10240): a token's cosines are made once per block, and the turned k stays there between the search for
// its maximum and its codes. Larger pages go in turns and read k and v twice. Single tokens: latency; one launch for q, k and
// v, blocks of 128 threads.
// Measured on a B200: 10492 tokens of ragged prompts, 16 q heads on 4 of 256 (36 us of bytes): pages of 16 in 92 us, bound by
// the start of each block (its sequence, page and scale, one load after another), pages of 32 in 122 (20 KB per block: fewer
// at a time), 64 and 128 in 159 (two and four turns). Read back in 21.5 us (10 us of bytes): a warp waits for a token's
// sequence, position, page and scale one after another.
#include <mutex>

#include "step.cuh"

namespace vkb {

VKB_STATUS_ACCESSOR(status_take_kv)

struct AppendArgs {
    uint8_t* codes[2];      // k, v
    float* scale[2];
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    const int32_t* pos;
    const unsigned long long* turns;
    const void* q;
    void* qo;
    const void* kv[2];
    long long ldq, ldqo, ldkv[2];
    int pages, heads, page, dim, table_ld, B, T, hq, half_rot, layout, items;
    int max_len;                         // of a sequence
    int cs_max, cs_tokens, val_tokens;   // shared memory: cosines in all, of how many tokens; values of how many tokens
    float mscale;
};

constexpr int AP_THREADS = 128;

// cos and sin (times mscale) of pair i at position p.
__device__ __forceinline__ float2 rope_cs(const AppendArgs& a, long long p, int i) {
    const unsigned long long ph = (unsigned long long)p * a.turns[i];
    const float x = (float)(int)(ph >> 32) * 4.656612873077393e-10f;   // 2^-31: half turns in [-1, 1]
    float s, c;
    sincospif(x, &s, &c);
    return make_float2(c * a.mscale, s * a.mscale);
}

// The rotated element e of a head whose elements start at p (turn: this tensor is rotated). cs: the token's cosines and
// sines.
template <int DT>
__device__ __forceinline__ float rope_elem(const AppendArgs& a, const typename Elem<DT>::T* p, int e, const float2* csp,
                                           bool turn) {
    const float v = Elem<DT>::to(p[e]);
    if (!turn || e >= 2 * a.half_rot) return v;
    const bool half = a.layout == VKB_ROPE_HALF;
    const int i = half ? (e < a.half_rot ? e : e - a.half_rot) : e >> 1;
    const bool second = half ? e >= a.half_rot : (e & 1) != 0;
    const int o = half ? (second ? e - a.half_rot : e + a.half_rot) : e ^ 1;
    const float w = Elem<DT>::to(p[o]);
    const float2 cs = csp[i];
    return second ? fmaf(v, cs.x, w * cs.y) : fmaf(v, cs.x, -w * cs.y);
}

// Eight consecutive elements e0.. of a head, rotated. vec: p is 16-byte aligned and the rotated part is made of whole
// vectors (half layout: half_rot % 8 == 0; interleaved: half_rot % 4 == 0), so a vector lies in one part.
template <int DT>
__device__ __forceinline__ void rope_vec(const AppendArgs& a, const typename Elem<DT>::T* p, int e0, const float2* csp,
                                         bool turn, bool vec, float (&f)[8]) {
    if (!vec) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rope_elem<DT>(a, p, e0 + e, csp, turn);
        return;
    }
    Raw8<DT> r, o;
    raw8_load<DT>(r, p + e0);
    if (!turn || e0 >= 2 * a.half_rot) {
        raw8_to<DT>(r, f);
        return;
    }
    if (a.layout == VKB_ROPE_HALF) {
        const bool second = e0 >= a.half_rot;
        const int i0 = second ? e0 - a.half_rot : e0;
        float g[8];
        raw8_load<DT>(o, p + (second ? e0 - a.half_rot : e0 + a.half_rot));
        raw8_to<DT>(r, f);
        raw8_to<DT>(o, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 cs = csp[i0 + e];
            f[e] = fmaf(f[e], cs.x, second ? g[e] * cs.y : -g[e] * cs.y);
        }
    } else {
        raw8_to<DT>(r, f);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float2 cs = csp[(e0 + e) >> 1];
            const float x = f[e], y = f[e + 1];
            f[e] = fmaf(x, cs.x, -y * cs.y);
            f[e + 1] = fmaf(y, cs.x, x * cs.y);
        }
    }
}

// The sequence's new tokens: rows [q0, q0 + n) of the call, positions [len - n, len). Indices that do not fit the call
// or the table raise a status bit and leave the sequence out.
struct SeqSpan { int q0, n, len; };
__device__ __forceinline__ SeqSpan seq_span(const AppendArgs& a, int b) {
    SeqSpan s;
    s.len = a.lens[b];
    s.q0 = a.cu ? a.cu[b] : b;
    s.n = a.cu ? a.cu[b + 1] - s.q0 : 1;
    if (s.len < 0 || s.n < 0 || s.q0 < 0 || s.q0 > a.T - s.n || s.len > a.max_len) {
        raise_status(DEV_ERR_BAD_INDEX);
        s.n = 0;
    }
    return s;
}
// Pages that the new tokens at positions >= 0 touch: [first, first + count).
__device__ __forceinline__ int span_pages(const AppendArgs& a, const SeqSpan& s, int* first) {
    const int lo = max(0, s.len - s.n);
    *first = lo / a.page;
    return s.n > 0 && s.len > lo ? (s.len - 1) / a.page - *first + 1 : 0;
}

__device__ __forceinline__ float finite_abs(float v) {
    const float f = fabsf(v);
    return f <= 3.402823466e38f ? f : 0.f;   // infinities and NaN: no part in the scale
}
__device__ __forceinline__ uint32_t kv_code(float v, float s) {   // code + 128
    if (!(s > 0.f) || v != v) return 128u;
    return (uint32_t)((int)rintf(fminf(127.f, fmaxf(-127.f, __fdiv_rn(v, s)))) + 128);
}

template <int DT> __global__ void __launch_bounds__(AP_THREADS) rope_append_kernel(const AppendArgs a) {
    using T = typename Elem<DT>::T;
    __shared__ int sh[AP_THREADS / 32 + 4];
    __shared__ float red[AP_THREADS / 32];
    extern __shared__ __align__(16) uint8_t ap_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    const int nkv = a.items * a.heads * 2;
    const int rot8 = a.layout == VKB_ROPE_HALF ? 8 : 4;
    const bool rot_ok = a.half_rot % rot8 == 0;
    const int dv = a.dim >> 3;
    if ((int)blockIdx.x >= nkv) {   // ---- one token's q heads ----
        const int t = blockIdx.x - nkv;
        int b = t;   // the sequence of token t: the number of sequences that end at or before it
        if (a.cu) {
            int n = 0;
            for (int i = tid; i < a.B; i += AP_THREADS) n += a.cu[i + 1] <= t;
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) sh[warp] = n;
            __syncthreads();
            b = 0;
#pragma unroll
            for (int w = 0; w < AP_THREADS / 32; ++w) b += sh[w];
        }
        if (b >= a.B) return;   // rows past the last sequence
        const SeqSpan s = seq_span(a, b);
        if (t < s.q0 || t >= s.q0 + s.n) return;   // rows of no sequence, or of one that is left out
        const long long pos = a.pos ? a.pos[t] : (long long)s.len - s.n + (t - s.q0);
        float2* cs = reinterpret_cast<float2*>(ap_smem);
        for (int i = tid; i < a.half_rot; i += AP_THREADS) cs[i] = rope_cs(a, pos, i);
        __syncthreads();
        const T* q = reinterpret_cast<const T*>(a.q) + t * a.ldq;
        T* qo = reinterpret_cast<T*>(a.qo) + t * a.ldqo;
        const bool vin = rot_ok && aligned_to(a.q, 16) && (a.ldq * sizeof(T)) % 16 == 0;
        const bool vout = aligned_to(a.qo, 16) && (a.ldqo * sizeof(T)) % 16 == 0;
        const bool half = a.layout == VKB_ROPE_HALF && a.half_rot > 0;
        // Half layout: a thread takes the two vectors of the same pairs, so that q may be rotated in place. The vectors
        // past the rotated part follow.
        const int hv = half && vin ? a.half_rot >> 3 : 0, rest = dv - 2 * hv;
        if (half && !vin) {   // pair by pair (in place is safe: both elements are one thread's)
            const int per = a.dim - a.half_rot;   // half_rot pairs, then the elements past them
            for (int i = tid; i < a.hq * per; i += AP_THREADS) {
                const int h = i / per, e = i - h * per;
                const T* p = q + h * a.dim;
                T* o = qo + h * a.dim;
                if (e < a.half_rot) {
                    const float x = rope_elem<DT>(a, p, e, cs, true), y = rope_elem<DT>(a, p, e + a.half_rot, cs, true);
                    o[e] = Elem<DT>::from(x);
                    o[e + a.half_rot] = Elem<DT>::from(y);
                } else {
                    o[e + a.half_rot] = p[e + a.half_rot];
                }
            }
            return;
        }
        const int per = hv + rest;
        for (int i = tid; i < a.hq * per; i += AP_THREADS) {
            const int h = i / per, j = i - h * per;
            const T* p = q + h * a.dim;
            T* o = qo + h * a.dim;
            const int e0 = 8 * (j < hv ? j : j + hv);
            float f[8], g[8];
            if (j < hv) rope_vec<DT>(a, p, e0 + a.half_rot, cs, true, true, g);
            rope_vec<DT>(a, p, e0, cs, a.half_rot > 0, vin, f);
            if (vout) {
                store8<DT>(o + e0, f);
                if (j < hv) store8<DT>(o + e0 + a.half_rot, g);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e0 + e] = Elem<DT>::from(f[e]);
                    if (j < hv) o[e0 + a.half_rot + e] = Elem<DT>::from(g[e]);
                }
            }
        }
        return;
    }
    // ---- one touched page of one head, k or v ----
    const int which = blockIdx.x & 1, h = (blockIdx.x >> 1) % a.heads;
    int item = (blockIdx.x >> 1) / a.heads, b = item, blk = -1;
    SeqSpan s{0, 0, 0};
    if (!a.cu) {
        s = seq_span(a, b);
        int first;
        if (span_pages(a, s, &first) > 0) blk = first;
    } else {   // the sequence whose touched pages hold this item: a scan of the page counts, 128 sequences at a time
        if (tid == 0) sh[AP_THREADS / 32 + 1] = -1;
        __syncthreads();
        for (int base = 0; base < a.B; base += AP_THREADS) {
            int first = 0, cnt = 0;
            SeqSpan mine{0, 0, 0};
            if (base + tid < a.B) {
                mine = seq_span(a, base + tid);
                cnt = span_pages(a, mine, &first);
            }
            int inc = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            if (lane == 31) sh[warp] = inc;
            __syncthreads();
            int before = 0, total = 0;
#pragma unroll
            for (int w = 0; w < AP_THREADS / 32; ++w) {
                before += w < warp ? sh[w] : 0;
                total += sh[w];
            }
            const int at = item - (before + inc - cnt);
            if (at >= 0 && at < cnt) {
                sh[AP_THREADS / 32 + 1] = first + at;
                sh[AP_THREADS / 32 + 2] = base + tid;
            }
            __syncthreads();
            if (item < total) break;
            item -= total;
        }
        blk = sh[AP_THREADS / 32 + 1];
        if (blk >= 0) {
            b = sh[AP_THREADS / 32 + 2];
            s = seq_span(a, b);
        }
    }
    if (blk < 0) return;   // the grid is an upper bound of the touched pages
    const int id = a.table[(long long)b * a.table_ld + blk];
    if (id < 0 || id >= a.pages) {
        if (tid == 0) raise_status(DEV_ERR_BAD_INDEX);
        return;
    }
    const int p0 = s.len - s.n;                                      // position of the sequence's first new token
    const int lo = max(max(p0, 0), blk * a.page), hi = min(s.len, (blk + 1) * a.page);
    const int held = lo - blk * a.page;                               // tokens that the page held before
    const T* src = reinterpret_cast<const T*>(a.kv[which]) + h * a.dim;
    const long long ld = a.ldkv[which];
    const bool turn = which == 0 && a.half_rot > 0;
    const bool vec = rot_ok && aligned_to(a.kv[which], 16) && (ld * sizeof(T)) % 16 == 0;
    const bool vsrc = vec || (which == 1 && aligned_to(a.kv[which], 16) && (ld * sizeof(T)) % 16 == 0);
    const long long ph = (long long)id * a.heads + h;
    uint8_t* codes = a.codes[which] + ph * a.page * a.dim;
    const float before = held > 0 ? a.scale[which][ph] : 0.f;
    // The tokens in turns of as many as shared memory holds, as fp32 (turned, for k): one turn where page x (dim + 4) x 4 bytes
    // are at most 40 KB (of 256-wide heads 39 tokens, of 128-wide ones 77); where there is more than one, the second pass
    // makes its values again.
    const int count = hi - lo, dv4 = a.dim + 4;   // 4 floats apart from a multiple of the banks
    float2* cs = reinterpret_cast<float2*>(ap_smem);
    float* vals = reinterpret_cast<float*>(ap_smem + 8 * a.cs_max);
    auto fill = [&](int t0, int n, float amax) {   // tokens t0 .. t0 + n - 1 into vals; their largest magnitude
        for (int c0 = 0; c0 < n; c0 += a.cs_tokens) {
            const int cn = min(a.cs_tokens, n - c0);
            if (turn) {
                __syncthreads();
                for (int i = tid; i < cn * a.half_rot; i += AP_THREADS) {
                    const int t = i / a.half_rot, row = s.q0 + (lo + t0 + c0 + t - p0);
                    cs[i] = rope_cs(a, a.pos ? a.pos[row] : lo + t0 + c0 + t, i - t * a.half_rot);
                }
                __syncthreads();
            }
            for (int i = tid; i < cn * dv; i += AP_THREADS) {
                const int t = i / dv, e0 = 8 * (i - t * dv), row = s.q0 + (lo + t0 + c0 + t - p0);
                float f[8];
                rope_vec<DT>(a, src + row * ld, e0, cs + t * a.half_rot, turn, vsrc, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[e]));
                float4* v = reinterpret_cast<float4*>(vals + (c0 + t) * dv4 + e0);
                v[0] = make_float4(f[0], f[1], f[2], f[3]);
                v[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
        }
        return amax;
    };
    float amax = 0.f;
    for (int t0 = 0; t0 < count; t0 += a.val_tokens) amax = fill(t0, min(a.val_tokens, count - t0), amax);
    amax = warp_max(amax);
    if (lane == 0) red[warp] = amax;
    __syncthreads();   // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < AP_THREADS / 32; ++w) amax = fmaxf(amax, red[w]);
    const float after = fmaxf(before, __fdiv_rn(amax, 127.f));
    if (tid == 0) a.scale[which][ph] = after;
    if (held > 0 && after > before) {   // bring the codes held before to the new scale
        const float k = __fdiv_rn(before, after);
        uint2* c = reinterpret_cast<uint2*>(codes);
        for (int i = tid; i < held * dv; i += AP_THREADS) {
            const uint2 v = c[i];
            uint32_t w[2] = {v.x, v.y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t o = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = (float)((int)((w[j] >> (8 * e)) & 255u) - 128);
                    o |= (uint32_t)((int)rintf(x * k) + 128) << (8 * e);
                }
                w[j] = o;
            }
            c[i] = make_uint2(w[0], w[1]);
        }
    }
    for (int t0 = 0; t0 < count; t0 += a.val_tokens) {
        const int n = min(a.val_tokens, count - t0);
        if (count > a.val_tokens) {
            __syncthreads();
            fill(t0, n, 0.f);
        }
        __syncthreads();
        for (int i = tid; i < n * dv; i += AP_THREADS) {
            const int t = i / dv, e0 = 8 * (i - t * dv);
            const float4* v = reinterpret_cast<const float4*>(vals + t * dv4 + e0);
            const float4 x = v[0], y = v[1];
            const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            uint32_t c[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e >> 2] |= kv_code(f[e], after) << (8 * (e & 3));
            *reinterpret_cast<uint2*>(codes + (held + t0 + t) * a.dim + e0) = make_uint2(c[0], c[1]);
        }
    }
}

struct ReadArgs {
    const uint8_t* codes[2];
    const float* scale[2];
    void* out[2];
    const int32_t *table, *seq, *pos;
    int pages, heads, page, dim, table_ld, B, n;
};

// A warp takes a token's heads and dimensions by 256 codes, eight per lane (an 8-byte load, a 16-byte store of 16-bit
// values: both contiguous over the warp).
template <int DT> __global__ void __launch_bounds__(256) kv_read_kernel(const ReadArgs a) {
    using T = typename Elem<DT>::T;
    pdl_trigger();
    pdl_wait();
    const int which = blockIdx.y, lane = threadIdx.x & 31, warps = gridDim.x * 8, per = a.dim >> 3, all = a.heads * per;
    for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < a.n; t += warps) {
        const int b = a.seq[t], p = a.pos[t];
        bool ok = b >= 0 && b < a.B && p >= 0 && p < (long long)a.table_ld * a.page;
        const int id = ok ? a.table[(long long)b * a.table_ld + p / a.page] : -1;
        ok = ok && id >= 0 && id < a.pages;
        if (!ok && lane == 0) raise_status(DEV_ERR_BAD_INDEX);   // a token that is not in the table reads as zeros
        T* out = reinterpret_cast<T*>(a.out[which]) + (long long)t * a.heads * a.dim;
        for (int i = lane; i < all; i += 32) {
            const int h = i / per, e0 = 8 * (i - h * per);
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (ok) {
                const long long ph = (long long)id * a.heads + h;
                const uint2 v = *reinterpret_cast<const uint2*>(a.codes[which] + (ph * a.page + p % a.page) * a.dim + e0);
                const float s = a.scale[which][ph];
                const uint32_t w[2] = {v.x, v.y};
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (float)((int)((w[e >> 2] >> (8 * (e & 3))) & 255u) - 128) * s;
            }
            store8<DT>(out + 8 * i, f);
        }
    }
}

int kv_cache_check(const vkb_kv_cache_t* c, const int32_t* table, int table_ld) {
    if (!c || !table || table_ld < 1) return VKB_EINVAL;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || c->pages < 1 || c->heads < 1) return VKB_EINVAL;
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4))
        return VKB_EINVAL;
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return VKB_EUNSUPPORTED;
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return VKB_EUNSUPPORTED;
    if ((long long)c->pages * c->heads * c->page > 0x7fffffffll) return VKB_EUNSUPPORTED;
    return 0;
}

}  // namespace vkb

using namespace vkb;

extern "C" int vkb_rope_append(const vkb_kv_cache_t* c, const int32_t* table, int table_ld, const int32_t* lens,
                               const int32_t* cu, int B, int T, int dt, const void* q, long long ldq, void* q_out,
                               long long ldqo, int q_heads, const void* k, long long ldk, const void* v, long long ldv,
                               const int32_t* pos, const uint64_t* turns, int rot, int layout, float mscale,
                               vkb_stream_t stream) {
    if (int r = kv_cache_check(c, table, table_ld)) return r;
    if (!dt_ok(dt) || !lens || B < 1 || T < 0 || (!cu && T != B)) return VKB_EINVAL;
    if (rot < 0 || rot > c->dim || (rot > 0 && !turns)) return VKB_EINVAL;
    if (layout != VKB_ROPE_HALF && layout != VKB_ROPE_INTERLEAVED) return VKB_EINVAL;
    if (rot & 1) return VKB_EUNSUPPORTED;
    if (T == 0) return 0;
    if (!k || !v || q_heads < 0 || (q_heads > 0 && (!q || !q_out))) return VKB_EINVAL;
    const long long kv_row = (long long)c->heads * c->dim, q_row = (long long)q_heads * c->dim;
    if (ldk < kv_row || ldv < kv_row || (q_heads > 0 && (ldq < q_row || ldqo < q_row))) return VKB_EINVAL;
    const int e = dt_size(dt);
    if (!aligned_to(q, e) || !aligned_to(q_out, e) || !aligned_to(k, e) || !aligned_to(v, e)) return VKB_EINVAL;
    if (q == q_out && ldq != ldqo) return VKB_EINVAL;   // in place: the same rows
    // touched pages: at most one per token, and at most n / page + 2 per sequence
    const long long bound = (long long)T / c->page + 2ll * B;
    const long long items = cu ? (bound < T ? bound : T) : B;
    const long long grid = items * c->heads * 2 + (q_heads > 0 ? T : 0);
    if (grid > 0x7fffffffll) return VKB_EUNSUPPORTED;
    AppendArgs a{};
    a.codes[0] = (uint8_t*)c->k; a.codes[1] = (uint8_t*)c->v;
    a.scale[0] = c->k_scale; a.scale[1] = c->v_scale;
    a.table = table; a.lens = lens; a.cu = cu; a.pos = pos; a.turns = (const unsigned long long*)turns;
    a.q = q; a.qo = q_out; a.kv[0] = k; a.kv[1] = v;
    a.ldq = ldq; a.ldqo = ldqo; a.ldkv[0] = ldk; a.ldkv[1] = ldv;
    a.pages = c->pages; a.heads = c->heads; a.page = c->page; a.dim = c->dim; a.table_ld = table_ld;
    a.B = B; a.T = T; a.hq = q_heads; a.half_rot = rot / 2; a.layout = layout; a.items = (int)items;
    a.mscale = mscale;
    a.max_len = max_length(table_ld, c->page);
    // Shared memory of a block: cosines and sines of 1024 pairs (or one token's), values of a page's tokens up to 40 KB (five
    // blocks per SM); single tokens take what one needs.
    const int pairs = rot / 2 > 0 ? rot / 2 : 1, value = 4 * (c->dim + 4);
    a.cs_tokens = !cu ? 1 : 1024 / pairs > 1 ? 1024 / pairs : 1;
    if (a.cs_tokens > c->page) a.cs_tokens = c->page;
    a.cs_max = (a.cs_tokens * pairs + 1) / 2 * 2;
    a.val_tokens = !cu ? 1 : 40960 / value < c->page ? 40960 / value : c->page;
    const size_t smem = 8 * (size_t)a.cs_max + (size_t)a.val_tokens * value;
    auto kern = dt == VKB_DT_F16 ? rope_append_kernel<VKB_DT_F16>
                : dt == VKB_DT_BF16 ? rope_append_kernel<VKB_DT_BF16> : rope_append_kernel<VKB_DT_F32>;
    static std::once_flag once[kMaxDevices][3];
    static cudaError_t err[kMaxDevices][3];
    int dev = 0;
    if (int r = current_device(&dev)) return r;
    std::call_once(once[dev][dt], [&] {
        err[dev][dt] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * 1024 + 40960);
    });
    if (err[dev][dt] != cudaSuccess) return -(int)err[dev][dt];
    return launch_pdl(kern, dim3((unsigned)grid), dim3(AP_THREADS), smem, (cudaStream_t)stream, 1, a);
}

extern "C" int vkb_kv_read(const vkb_kv_cache_t* c, const int32_t* table, int table_ld, int B, const int32_t* seq,
                           const int32_t* pos, int n, int dt, void* k, void* v, vkb_stream_t stream) {
    if (int r = kv_cache_check(c, table, table_ld)) return r;
    if (!dt_ok(dt) || B < 1 || n < 0) return VKB_EINVAL;
    if (n == 0) return 0;
    if (!seq || !pos || !k || !v || !aligned_to(k, 16) || !aligned_to(v, 16)) return VKB_EINVAL;
    const ReadArgs a{{(const uint8_t*)c->k, (const uint8_t*)c->v}, {c->k_scale, c->v_scale}, {k, v}, table, seq, pos,
                     c->pages, c->heads, c->page, c->dim, table_ld, B, n};
    int dev = 0;
    if (int r = current_device(&dev)) return r;
    const long long want = ((long long)n + 7) / 8, most = 16ll * device_info(dev).sm_count;
    const dim3 grid((unsigned)(want < most ? want : most), 2);
    auto kern = dt == VKB_DT_F16 ? kv_read_kernel<VKB_DT_F16>
                : dt == VKB_DT_BF16 ? kv_read_kernel<VKB_DT_BF16> : kv_read_kernel<VKB_DT_F32>;
    return launch_pdl(kern, grid, dim3(256), 0, (cudaStream_t)stream, 1, a);
}
