// vkb_sample: one token per row of logits, from given uniform random numbers.
//
// Order the tokens by (logit descending, index ascending). Top-k keeps the first k; top-p the shortest prefix of those
// whose weight reaches p of theirs, weight w = exp((logit - max) / temperature); min-p those with w >= min_p. The token
// is the first one, in index order, at which the running weight of the kept ones exceeds u times their sum.
//
// Both prefixes are cut at a boundary token, found without a sort: the row is read once into the shared memory of a
// cluster of 1-8 blocks (a slice each); a histogram of (max - logit) / temperature (count and weight per bin) gives the
// bin of each boundary, and the few tokens of that bin are ranked against one another. A bin that holds more than
// SM_CAP tokens is split again by the bits of its logits (a bin of one repeated logit is cut by index). Everything
// after the one read of the logits happens in shared memory.
//
// Deterministic: block-wide sums that atomics make are integers (counts; a bin's weight is its count times the weight at
// the bin's edge, less the sum of the tokens' distances to it in units of 2^-13 of the bin's width), the others have a
// fixed order.
// Weights below e^-32 of the largest do not enter the top-p sums.
#include "step.cuh"

#include <mutex>

namespace vkb {

constexpr int SM_THREADS = 512;
constexpr int SM_NB = 1024;      // bins
constexpr int SM_CAP = 1024;     // tokens of a boundary bin that are ranked directly
constexpr float SM_SPAN = 32.f;  // bins cover distances up to this (the last bin: everything beyond)
constexpr int SM_MAX_SLICE = 49152;   // floats of a row that one block holds

struct SampleArgs {
    const void* logits;
    long long ld;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* token;
    float* prob;
    int V, slice;
};

struct SmEntry { float l; int i; };

// What the blocks of a row share (read by the others through distributed shared memory).
struct SmShared {
    unsigned cnt[SM_NB], eps[SM_NB];
    SmEntry list[SM_CAP];
    SmEntry all[SM_CAP];        // the row's boundary bin
    float2 range;               // this block's max and smallest finite logit
    int arg;                    // index of the max
    int nlist;
    double sum;                 // kept weight of the slice
    unsigned kmin, kmax, ties;
    double wsum[SM_THREADS / 32];
    double scan[SM_THREADS / 32];
    unsigned scan_n[SM_THREADS / 32];
    int out_i;
    unsigned out_n;
    double out_d;
    SmEntry cut;
    double cut_mass;
};

__device__ __forceinline__ unsigned float_key(float f) {   // order of the floats as unsigned integers
    const unsigned b = __float_as_uint(f + 0.f);            // -0 and 0 alike
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <int CL> __device__ __forceinline__ void row_sync() {
    if constexpr (CL > 1) cluster_sync();
    else __syncthreads();
}
// Word of the same shared variable in block r of the cluster.
template <int CL, typename V> __device__ __forceinline__ V peer(const V* p, int r) {
    if constexpr (CL == 1) return *p;
    else {
        static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one or two words");
        const uint32_t ad = mapa_shared(smem_u32(p), (uint32_t)r);
        V v;
        if constexpr (sizeof(V) == 4) {
            uint32_t x;
            asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(x) : "r"(ad) : "memory");
            memcpy(&v, &x, 4);
        } else {
            unsigned long long x;
            asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(x) : "r"(ad) : "memory");
            memcpy(&v, &x, 8);
        }
        return v;
    }
}

struct SmRow {
    float lmax, inv_bin, t;     // inv_bin: bins per unit of distance
    float step;                 // distance per bin
};

__device__ __forceinline__ float sm_dist(const SmRow& r, float l) {   // (max - logit) / temperature, >= 0
    return l == r.lmax ? 0.f : __fdiv_rn(r.lmax - l, r.t);
}
__device__ __forceinline__ int sm_bin(const SmRow& r, float d) {
    return (int)fminf(d * r.inv_bin, (float)(SM_NB - 1));
}
__device__ __forceinline__ float sm_weight(float d) { return expf(-d); }
// Weight at the near edge of a bin, and a token's relative distance to it in units of 2^-13 of a bin's width (0 for the
// last bin, whose weight does not count). SM_MAX_SLICE x 8 blocks x 2^13 < 2^32: a row's sum does not overflow.
__device__ __forceinline__ float sm_edge(const SmRow& r, int bin) { return expf(-(float)bin * r.step); }
__device__ __forceinline__ unsigned sm_eps(const SmRow& r, int bin, float d) {
    if (bin == SM_NB - 1) return 0u;
    const float e = -expm1f(fminf((float)bin * r.step - d, 0.f));   // 1 - w / edge, in [0, step]
    return (unsigned)__float2int_rn(fminf(e * r.inv_bin, 1.f) * 8192.f);
}

// All threads: the first bin at which the running total of the bins' counts (by_count) or weights reaches the target, and
// the totals before it. cnt / eps: the row's summed histogram. edge(bin): a bin's edge weight; unit: of eps.
template <typename Edge>
__device__ __forceinline__ int sm_find(SmShared* s, bool by_count, unsigned tcount, double tmass, Edge edge, double unit,
                                       unsigned* before_n, double* before_m) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int PER = SM_NB / SM_THREADS;
    unsigned c[PER], csum = 0;
    double m[PER], msum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = tid * PER + j;
        c[j] = s->cnt[b];
        m[j] = c[j] ? (double)edge(b) * ((double)c[j] - (double)s->eps[b] * unit) : 0.0;
        csum += c[j];
        msum += m[j];
    }
    unsigned ci = csum;
    double mi = msum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned a = __shfl_up_sync(0xffffffffu, ci, o);
        const double b = __shfl_up_sync(0xffffffffu, mi, o);
        if (lane >= o) { ci += a; mi += b; }
    }
    if (lane == 31) { s->scan_n[warp] = ci; s->scan[warp] = mi; }
    if (tid == 0) s->out_i = SM_NB;
    __syncthreads();
    unsigned cb = 0;
    double mb = 0.0;
    for (int w = 0; w < warp; ++w) { cb += s->scan_n[w]; mb += s->scan[w]; }
    cb += ci - csum;
    mb += mi - msum;
    int found = SM_NB;
    unsigned fc = 0;
    double fm = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (found == SM_NB && c[j] && (by_count ? cb + c[j] >= tcount : mb + m[j] >= tmass)) {
            found = tid * PER + j;
            fc = cb;
            fm = mb;
        }
        cb += c[j];
        mb += m[j];
    }
    if (found < SM_NB) atomicMin(&s->out_i, found);
    __syncthreads();
    const int bin = s->out_i;
    if (found == bin && bin < SM_NB) { s->out_n = fc; s->out_d = fm; }
    __syncthreads();
    *before_n = s->out_n;
    *before_m = s->out_d;
    return bin;
}

// All blocks: the row's histogram from the blocks' (each ends with the sum in its own cnt / eps).
template <int CL> __device__ __forceinline__ void sm_combine(SmShared* s) {
    if constexpr (CL > 1) {
        row_sync<CL>();
        unsigned c[SM_NB / SM_THREADS], e[SM_NB / SM_THREADS];
#pragma unroll
        for (int j = 0; j < SM_NB / SM_THREADS; ++j) {
            const int b = threadIdx.x + j * SM_THREADS;
            c[j] = e[j] = 0;
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                c[j] += peer<CL>(&s->cnt[b], r);
                e[j] += peer<CL>(&s->eps[b], r);
            }
        }
        row_sync<CL>();
#pragma unroll
        for (int j = 0; j < SM_NB / SM_THREADS; ++j) {
            s->cnt[threadIdx.x + j * SM_THREADS] = c[j];
            s->eps[threadIdx.x + j * SM_THREADS] = e[j];
        }
    }
    __syncthreads();
}

// All blocks: the boundary token within level-0 bin `bin` (before_n tokens of weight before_m come earlier in the
// order): the one that is number tcount of the row (by_count), or at which the running weight reaches tmass. Returns
// the weight up to and including it. n: tokens in the bin.
template <int CL>
__device__ __noinline__ double sm_boundary(SmShared* s, const float* x, const SampleArgs& a, const SmRow& row, int n0,
                                           int bin, unsigned n, bool by_count, unsigned tcount, double tmass,
                                           unsigned before_n, double before_m, SmEntry* cut) {
    const int tid = threadIdx.x;
    const int rank = CL > 1 ? (int)cluster_ctarank() : 0;
    unsigned klo = 0u, khi = 0xffffffffu;
    auto in = [&](float l) {
        if (!(l > -INFINITY)) return false;
        const unsigned k = float_key(l);
        return k >= klo && k <= khi && sm_bin(row, sm_dist(row, l)) == bin;
    };
    while (n > SM_CAP) {
        // the span of the bin's keys
        if (tid == 0) { s->kmin = 0xffffffffu; s->kmax = 0u; }
        __syncthreads();
        unsigned lo = 0xffffffffu, hi = 0u;
        for (int i = tid; i < n0; i += SM_THREADS)
            if (in(x[i])) { lo = min(lo, float_key(x[i])); hi = max(hi, float_key(x[i])); }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if ((tid & 31) == 0) { atomicMin(&s->kmin, lo); atomicMax(&s->kmax, hi); }
        row_sync<CL>();
        lo = 0xffffffffu;
        hi = 0u;
#pragma unroll
        for (int r = 0; r < CL; ++r) { lo = min(lo, peer<CL>(&s->kmin, r)); hi = max(hi, peer<CL>(&s->kmax, r)); }
        klo = lo;
        khi = hi;
        if (lo == hi) break;
        const int shift = max(0, 32 - __clz(hi - lo) - 10);   // (hi - key) >> shift < 1024
        for (int b = tid; b < SM_NB; b += SM_THREADS) s->cnt[b] = s->eps[b] = 0u;
        __syncthreads();
        for (int i = tid; i < n0; i += SM_THREADS)
            if (in(x[i])) {
                const int b = (int)((hi - float_key(x[i])) >> shift);
                atomicAdd(&s->cnt[b], 1u);
                atomicAdd(&s->eps[b], sm_eps(row, bin, sm_dist(row, x[i])));
            }
        sm_combine<CL>(s);
        const float edge = bin == SM_NB - 1 ? 0.f : sm_edge(row, bin);
        unsigned bn;
        double bm;
        int b = sm_find(s, by_count, tcount - before_n, tmass - before_m, [&](int) { return edge; }, (double)row.step / 8192.0, &bn, &bm);
        if (b == SM_NB) {   // rounding: the target lies just past the bin's weight; its last token
            b = (int)((hi - lo) >> shift);
            bn = n - s->cnt[b];
            bm = (double)edge * (double)bn;
        }
        n = s->cnt[b];
        before_n += bn;
        before_m += bm;
        khi = hi - ((unsigned)b << shift);
        klo = max(lo, khi - ((1u << shift) - 1u) > khi ? 0u : khi - ((1u << shift) - 1u));
        row_sync<CL>();
    }
    if (n > SM_CAP) {
        // one logit, repeated: cut by index. Its r-th occurrence.
        const float l = __uint_as_float(khi ^ ((khi >> 31) ? 0x80000000u : 0xffffffffu));
        const double w = bin == SM_NB - 1 ? 0.0 : (double)sm_weight(sm_dist(row, l));
        unsigned r;
        if (by_count) r = tcount - before_n;
        else {
            const double q = w > 0.0 ? ceil((tmass - before_m) / w) : (double)n;
            r = q < 1.0 ? 1u : q > (double)n ? n : (unsigned)q;
        }
        // occurrences in the blocks before this one, then per warp (contiguous pieces of the slice)
        const int lane = tid & 31, warp = tid >> 5, nw = SM_THREADS / 32;
        const int piece = (n0 + nw - 1) / nw, i0 = min(n0, warp * piece), i1 = min(n0, i0 + piece);
        unsigned mine = 0;
        for (int i = i0 + lane; i < i1; i += 32) mine += float_key(x[i]) == khi ? 1u : 0u;
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s->scan_n[warp] = mine;
        __syncthreads();
        if (tid == 0) {
            unsigned t = 0;
            for (int w2 = 0; w2 < nw; ++w2) t += s->scan_n[w2];
            s->ties = t;
            s->cut.i = 0x7fffffff;
        }
        row_sync<CL>();
        unsigned ahead = 0;
#pragma unroll
        for (int q = 0; q < CL; ++q) ahead += q < rank ? peer<CL>(&s->ties, q) : 0u;
        for (int w2 = 0; w2 < warp; ++w2) ahead += s->scan_n[w2];
        for (int i = i0; i < i1 && ahead < r; i += 32) {   // whole warp
            const bool hit = i + lane < i1 && float_key(x[i + lane]) == khi;
            const unsigned m = __ballot_sync(0xffffffffu, hit);
            const unsigned at = ahead + __popc(m & ((2u << lane) - 1u));
            if (hit && at == r) s->cut.i = rank * a.slice + i + lane;
            ahead += __popc(m);
        }
        row_sync<CL>();
        int ci = 0x7fffffff;
#pragma unroll
        for (int q = 0; q < CL; ++q) ci = min(ci, peer<CL>(&s->cut.i, q));
        cut->l = l;
        cut->i = ci;
        row_sync<CL>();
        return before_m + (double)r * w;
    }
    // ---- the bin's tokens, in one list ----
    if (tid == 0) s->nlist = 0;
    __syncthreads();
    for (int i = tid; i < n0; i += SM_THREADS)
        if (in(x[i])) {
            const int at = atomicAdd(&s->nlist, 1);
            if (at < SM_CAP) s->list[at] = SmEntry{x[i], rank * a.slice + i};
        }
    row_sync<CL>();
    int base = 0;
#pragma unroll
    for (int r = 0; r < CL; ++r) {
        const int m = min(peer<CL>(&s->nlist, r), SM_CAP - base);
        for (int i = tid; i < m; i += SM_THREADS) s->all[base + i] = peer<CL>(&s->list[i], r);
        base += m;
    }
    row_sync<CL>();
    n = (unsigned)base;
    // every token's number in the order, and the weight before it (integers of 2^-50: any order of adding)
    const unsigned want = by_count ? tcount - before_n : 0u;
    const double tgt = tmass - before_m;
    for (int i = tid; i < (int)n; i += SM_THREADS) {
        const SmEntry e = s->all[i];
        unsigned ahead = 0;
        unsigned long long mass = 0;
        for (int j = 0; j < (int)n; ++j) {
            const SmEntry f = s->all[j];
            const bool first = f.l > e.l || (f.l == e.l && f.i < e.i);
            ahead += first;
            if (first) mass += (unsigned long long)((double)sm_weight(sm_dist(row, f.l)) * 1125899906842624.0);
        }
        const double before = (double)mass * (1.0 / 1125899906842624.0), w = (double)sm_weight(sm_dist(row, e.l));
        const bool hit = by_count ? ahead + 1 == want
                                  : (ahead == 0 || before < tgt) && (ahead + 1 == n || before + w >= tgt);
        if (hit) {
            s->cut = e;
            s->cut_mass = before_m + before + w;
        }
    }
    __syncthreads();
    *cut = s->cut;
    const double m = s->cut_mass;
    __syncthreads();
    return m;
}

template <int DT, int CL>
__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleArgs a) {
    using T = typename Elem<DT>::T;
    extern __shared__ __align__(16) uint8_t smem[];
    SmShared* s = reinterpret_cast<SmShared*>(smem);
    float* x = reinterpret_cast<float*>(smem + (sizeof(SmShared) + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = CL > 1 ? (int)cluster_ctarank() : 0, rw = blockIdx.x / CL;
    const int first = rank * a.slice, n0 = max(0, min(a.slice, a.V - first));
    pdl_trigger();
    pdl_wait();
    const float t = a.temperature ? a.temperature[rw] : 1.f, u = fminf(fmaxf(a.u[rw], 0.f), 1.f);   // NaN: 0
    const int k = a.top_k ? a.top_k[rw] : 0;
    const float tp = a.top_p ? a.top_p[rw] : 1.f, mp = a.min_p ? a.min_p[rw] : 0.f;
    // ---- read the slice; maximum (lowest index among equals), smallest finite logit ----
    const T* g = reinterpret_cast<const T*>(a.logits) + rw * a.ld + first;
    float hi = -INFINITY, lo = INFINITY;
    int arg = 0x7fffffff;
    auto see = [&](float v, int i) {
        if (v > hi) { hi = v; arg = first + i; }
        if (v > -INFINITY) lo = fminf(lo, v);
    };
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
        constexpr int UN = 4;
        const int nv = n0 / 8;
        for (int i = tid; i < nv; i += SM_THREADS * UN) {
            Raw8<DT> r[UN];
#pragma unroll
            for (int j = 0; j < UN; ++j)
                if (i + j * SM_THREADS < nv) raw8_load<DT>(r[j], g + 8 * (i + j * SM_THREADS));
#pragma unroll
            for (int j = 0; j < UN; ++j)
                if (i + j * SM_THREADS < nv) {
                    float f[8];
                    raw8_to<DT>(r[j], f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (f[e] != f[e]) f[e] = -INFINITY;   // NaN: never taken
                        see(f[e], 8 * (i + j * SM_THREADS) + e);
                    }
                    store8<VKB_DT_F32>(x + 8 * (i + j * SM_THREADS), f);
                }
        }
        done = 8 * nv;
    }
    for (int i = done + tid; i < n0; i += SM_THREADS) {
        float f = Elem<DT>::to(g[i]);
        if (f != f) f = -INFINITY;
        see(f, i);
        x[i] = f;
    }
    for (int b = tid; b < SM_NB; b += SM_THREADS) s->cnt[b] = s->eps[b] = 0u;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float h2 = __shfl_xor_sync(0xffffffffu, hi, o);
        const int a2 = __shfl_xor_sync(0xffffffffu, arg, o);
        if (h2 > hi || (h2 == hi && a2 < arg)) { hi = h2; arg = a2; }
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (lane == 0) {   // through the list, which is not in use yet
        s->list[warp] = SmEntry{hi, arg};
        s->list[32 + warp] = SmEntry{lo, 0};
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SM_THREADS / 32; ++w) {
            const SmEntry e = s->list[w];
            if (e.l > hi || (e.l == hi && e.i < arg)) { hi = e.l; arg = e.i; }
            lo = fminf(lo, s->list[32 + w].l);
        }
        s->range = make_float2(hi, lo);
        s->arg = arg;
    }
    row_sync<CL>();
    hi = -INFINITY;
    lo = INFINITY;
    arg = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < CL; ++r) {
        const float2 v = peer<CL>(&s->range, r);
        const int i = peer<CL>(&s->arg, r);
        if (v.x > hi || (v.x == hi && i < arg)) { hi = v.x; arg = i; }
        lo = fminf(lo, v.y);
    }
    const bool none = !(hi > -INFINITY);   // nothing may be taken
    if (none || !(t > 0.f) || k == 1 || tp <= 0.f) {   // greedy
        if (rank == 0 && tid == 0) {
            a.token[rw] = none ? -1 : arg;
            if (a.prob) a.prob[rw] = none ? 0.f : 1.f;
        }
        row_sync<CL>();   // no block leaves while another reads its shared memory
        return;
    }
    SmRow row;
    row.lmax = hi;
    row.t = t;
    const float span = hi == lo ? 0.f : __fdiv_rn(hi - lo, t);
    row.step = fminf(SM_SPAN, fmaxf(1.01f * span, 1e-3f)) * (1.f / (SM_NB - 1));   // shorter spans stay off the last bin
    row.inv_bin = __fdiv_rn(1.f, row.step);
    const bool by_k = k > 1 && k < a.V, by_p = tp < 1.f;
    SmEntry cut{-INFINITY, 0x7fffffff};   // keep everything
    if (by_k || by_p) {
        for (int i = tid; i < n0; i += SM_THREADS) {
            const float l = x[i];
            if (!(l > -INFINITY)) continue;
            const float d = sm_dist(row, l);
            const int b = sm_bin(row, d);
            atomicAdd(&s->cnt[b], 1u);
            if (by_p) atomicAdd(&s->eps[b], sm_eps(row, b, d));
        }
        sm_combine<CL>(s);
        auto edge = [&](int b) { return b == SM_NB - 1 ? 0.f : sm_edge(row, b); };
        const double unit = (double)row.step / 8192.0;
        unsigned bn;
        double bm, total = -1.0;
        int kbin = SM_NB;
        unsigned kn = 0;
        if (by_k) {
            kbin = sm_find(s, true, (unsigned)k, 0.0, edge, unit, &bn, &bm);   // SM_NB: fewer than k tokens
            if (kbin < SM_NB) kn = s->cnt[kbin];
        }
        // the boundary search may reuse the histogram (bins of more than SM_CAP tokens): the bins of both cuts first
        if (!by_p) {
            if (kbin < SM_NB) sm_boundary<CL>(s, x, a, row, n0, kbin, kn, true, (unsigned)k, 0.0, bn, bm, &cut);
        } else {
            SmEntry kcut = cut;
            if (kbin < SM_NB) {
                total = sm_boundary<CL>(s, x, a, row, n0, kbin, kn, true, (unsigned)k, 0.0, bn, bm, &kcut);
                if (kn > SM_CAP) {   // the histogram was reused: make it again
                    for (int b = tid; b < SM_NB; b += SM_THREADS) s->cnt[b] = s->eps[b] = 0u;
                    __syncthreads();
                    for (int i = tid; i < n0; i += SM_THREADS) {
                        const float l = x[i];
                        if (!(l > -INFINITY)) continue;
                        const float d = sm_dist(row, l);
                        const int b = sm_bin(row, d);
                        atomicAdd(&s->cnt[b], 1u);
                        atomicAdd(&s->eps[b], sm_eps(row, b, d));
                    }
                    sm_combine<CL>(s);
                }
            } else {   // all tokens: their weight from the bins (a target no bin reaches)
                sm_find(s, false, 0u, 1e300, edge, unit, &bn, &bm);
                double all = 0.0;
                for (int w = 0; w < SM_THREADS / 32; ++w) all += s->scan[w];
                total = all;
                __syncthreads();
            }
            const double want = (double)tp * total;
            unsigned pn0;
            double pm0;
            const int pbin = sm_find(s, false, 0u, want, edge, unit, &pn0, &pm0);
            SmEntry pcut = cut;
            if (pbin < SM_NB)
                sm_boundary<CL>(s, x, a, row, n0, pbin, s->cnt[pbin], false, 0u, want, pn0, pm0, &pcut);
            cut = pcut.l > kcut.l || (pcut.l == kcut.l && pcut.i < kcut.i) ? pcut : kcut;
        }
    }
    // ---- the kept weight, by warp (contiguous pieces of the slice), block and row ----
    const float floor_w = fminf(mp, 1.f);
    auto kept = [&](int i) {   // weight of element i of the slice, 0 where it is not kept
        const float l = x[i];
        if (l < cut.l || (l == cut.l && first + i > cut.i)) return 0.f;
        const float w = sm_weight(sm_dist(row, l));
        return w >= floor_w ? w : 0.f;
    };
    const int nw = SM_THREADS / 32, piece = (n0 + nw - 1) / nw, i0 = min(n0, warp * piece), i1 = min(n0, i0 + piece);
    float part = 0.f;
    for (int i = i0 + lane; i < i1; i += 32) part += kept(i);
    part = warp_sum(part);
    if (lane == 0) s->wsum[warp] = (double)part;
    __syncthreads();
    if (tid == 0) {
        double m = 0.0;
        for (int w = 0; w < nw; ++w) m += s->wsum[w];
        s->sum = m;
    }
    row_sync<CL>();
    double ahead = 0.0, total = 0.0;
    int last = 0;   // the last block with any weight
#pragma unroll
    for (int r = 0; r < CL; ++r) {
        const double v = peer<CL>(&s->sum, r);
        if (r < rank) ahead += v;
        total += v;
        if (v > 0.0) last = r;
    }
    const double target = (double)u * total;
    // this block holds the token if the target falls into its part (the last one with weight takes rounding at the end)
    const double own = s->sum;
    if (own > 0.0 && ahead <= target && (target < ahead + own || rank == last) && warp == 0) {
        int w = 0, lw = 0;
        double m = ahead;
        for (int j = 0; j < nw; ++j) if (s->wsum[j] > 0.0) lw = j;
        while (w < lw && !(s->wsum[w] > 0.0 && target < m + s->wsum[w])) m += s->wsum[w++];
        const int a0 = min(n0, w * piece), a1 = min(n0, a0 + piece);
        int found = -1, back = -1;
        float fw = 0.f, bw = 0.f;
        for (int i = a0; i < a1 && found < 0; i += 32) {
            const float v = i + lane < a1 ? kept(i + lane) : 0.f;
            float inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float p = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += p;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, v > 0.f && m + (double)inc > target);
            const unsigned any = __ballot_sync(0xffffffffu, v > 0.f);
            if (hit) {
                const int b = __ffs(hit) - 1;
                found = i + b;
                fw = __shfl_sync(0xffffffffu, v, b);
            } else if (any) {
                const int b = 31 - __clz(any);
                back = i + b;
                bw = __shfl_sync(0xffffffffu, v, b);
            }
            m += (double)__shfl_sync(0xffffffffu, inc, 31);
        }
        if (found < 0) { found = back; fw = bw; }
        if (lane == 0) {
            a.token[rw] = first + found;
            if (a.prob) a.prob[rw] = (float)((double)fw / total);
        }
    }
    row_sync<CL>();
}

template <int DT, int CL> static int launch_sample(const SampleArgs& a, int B, int dev, cudaStream_t st) {
    auto kern = sample_kernel<DT, CL>;
    static std::once_flag once[kMaxDevices];
    static cudaError_t err[kMaxDevices];
    std::call_once(once[dev], [&] {
        err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)((sizeof(SmShared) + 15) / 16 * 16 + 4 * SM_MAX_SLICE));
    });
    if (err[dev] != cudaSuccess) return -(int)err[dev];
    const size_t smem = (sizeof(SmShared) + 15) / 16 * 16 + 4 * (size_t)a.slice;
    return launch_pdl(kern, dim3((unsigned)(B * CL)), dim3(SM_THREADS), smem, st, CL, a);
}

template <int DT> static int sample_cl(SampleArgs a, int B, int dev, cudaStream_t st) {
    // blocks per row: slices of a few thousand logits where the batch is small enough for the SMs, larger ones otherwise
    int cl = 1;
    while (cl < 8 && a.V > 4096 * cl) cl *= 2;
    a.slice = ((a.V + cl - 1) / cl + 7) / 8 * 8;
    if (a.slice > SM_MAX_SLICE) return VKB_EUNSUPPORTED;
    switch (cl) {
        case 1: return launch_sample<DT, 1>(a, B, dev, st);
        case 2: return launch_sample<DT, 2>(a, B, dev, st);
        case 4: return launch_sample<DT, 4>(a, B, dev, st);
        default: return launch_sample<DT, 8>(a, B, dev, st);
    }
}

}  // namespace vkb

using namespace vkb;

extern "C" int vkb_sample(int dt, const void* logits, long long ld, int B, int V, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                          float* prob, vkb_stream_t stream) {
    if (!dt_ok(dt) || B < 0 || V < 1 || ld < V) return VKB_EINVAL;
    if (B == 0) return 0;
    if (!logits || !u || !token || !aligned_to(logits, dt_size(dt))) return VKB_EINVAL;
    if (B > 0x7fffffff / 8) return VKB_EUNSUPPORTED;
    int dev = 0;
    if (int r = current_device(&dev)) return r;
    const SampleArgs a{logits, ld, temperature, top_k, top_p, min_p, u, token, prob, V, 0};
    cudaStream_t st = (cudaStream_t)stream;
    switch (dt) {
        case VKB_DT_F16: return sample_cl<VKB_DT_F16>(a, B, dev, st);
        case VKB_DT_BF16: return sample_cl<VKB_DT_BF16>(a, B, dev, st);
        default: return sample_cl<VKB_DT_F32>(a, B, dev, st);
    }
}
