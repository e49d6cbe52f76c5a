// vkb_sample: one token per row of logits, from given uniform random numbers.
//
// Order the tokens by (logit descending, index ascending). Top-k keeps the first k; top-p the shortest prefix of those
// whose weight reaches p of theirs, weight w = exp((logit - max) / temperature); min-p those with w >= min_p. The token
// is the first one, in index order, at which the running weight of the kept ones exceeds u times their sum.
//
// Both prefixes are cut at a boundary token, found without a sort. The row is read once, into the shared memory of a
// cluster of 1-8 blocks (a slice each). With a top-k of up to 3/5 of the cluster's threads, the k-th largest of the
// threads' own maxima bounds the k-th largest logit from below: the tokens above it (about 1.15 k of them for k a quarter
// of the threads) go to the first block, in index order, which finishes the row alone while the others make room for
// the next one. Rows without a top-k, or with a larger one, are finished by the whole cluster.
// Finishing: a histogram of (max - logit) / temperature (count and weight per bin) gives the bin of each boundary, and
// the few tokens of that bin are ranked against one another. A bin that holds more than SM_CAP tokens is split again
// by the bits of its logits (a bin of one repeated logit is cut by index).
//
// Measured on a B200, fp32: 256 x 151936 with mixed settings 249 us; all greedy 67 us (2.3 TB/s: a wave of clusters waits
// for its slowest read), all top-k 1000 with top-p 0.9 209 us, all top-p alone 528 us. Bound by the latency of a row's
// barriers and searches, with 33 clusters of 8 blocks on the device at a time.
//
// Deterministic: block-wide sums that atomics make are integers (counts; a bin's weight is its count times the weight at
// the bin's edge, less the sum of the tokens' distances to it in units of 2^-13 of the bin's width), the others have a
// fixed order. Weights below 2^-46 of the largest do not enter the top-p sums.
#include "step.cuh"

#include <mutex>

namespace vkb {

constexpr int SM_THREADS = 512;
constexpr int SM_NB = 1024;      // bins
constexpr int SM_CAP = 128;      // tokens of a boundary bin that are ranked directly (each against all: at 1024 the ranking of
                                 // a crowded bin, 600 tokens in 150000, took longer than splitting the bin)
constexpr float SM_SPAN = 46.f;  // bins cover distances up to this, in powers of two (the last bin: everything beyond)
constexpr int SM_LOCAL = 2048;   // candidates for the first block that one block can hold
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
    union {
        struct {
            SmEntry list[SM_CAP];   // this block's part of a boundary bin
            SmEntry all[SM_CAP];    // the row's
        };
        SmEntry cand[SM_LOCAL];     // this block's candidates, in index order
    };
    union {
        unsigned q[SM_CAP];         // weights of `all` in units of 2^-30 of the bin's edge
        float tmax[SM_THREADS];     // the threads' maxima
    };
    float2 range;               // this block's max and smallest finite logit
    int arg;                    // index of the max
    int nlist, ncand;
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
    float lmax, c;              // c: log2(e) / temperature
    float step, inv_bin;        // distance per bin, bins per unit of distance
};

// Distance (max - logit) / temperature in powers of two, >= 0; the weight is 2^-distance.
__device__ __forceinline__ float sm_dist(const SmRow& r, float l) { return l == r.lmax ? 0.f : (r.lmax - l) * r.c; }
__device__ __forceinline__ float sm_weight(float d) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(-d));
    return w;
}
__device__ __forceinline__ int sm_bin(const SmRow& r, float d) {
    return (int)fminf(d * r.inv_bin, (float)(SM_NB - 1));
}
// Weight at the near edge of a bin, and a token's relative distance to it in units of 2^-13 of a bin's width (0 for the
// last bin, whose weight does not count). SM_MAX_SLICE x 8 blocks x 2^13 < 2^32: a row's sum does not overflow.
__device__ __forceinline__ float sm_edge(const SmRow& r, int bin) {
    return bin == SM_NB - 1 ? 0.f : sm_weight((float)bin * r.step);
}
__device__ __forceinline__ unsigned sm_eps(const SmRow& r, int bin, float d) {
    if (bin == SM_NB - 1) return 0u;
    const float e = 1.f - sm_weight(fmaxf(d - (float)bin * r.step, 0.f));   // 1 - w / edge, in [0, step)
    return (unsigned)__float2int_rn(fminf(e * r.inv_bin, 1.f) * 8192.f);
}

// All threads: the first bin at which the running total of the bins' counts (by_count) or weights reaches the target,
// and the totals before it. cnt / eps: the row's summed histogram; edge >= 0: the edge weight of every bin (a bin of the
// row that was split), else each bin's own. The weights (before_m, total) are left out by_count over the row's own bins.
__device__ __noinline__ int sm_find(SmShared* s, const SmRow& row, bool by_count, unsigned tcount, double tmass,
                                    float edge, unsigned* before_n, double* before_m, double* total) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int PER = SM_NB / SM_THREADS, NW = SM_THREADS / 32;
    const double unit = (double)row.step / 8192.0;
    unsigned c[PER], csum = 0;
    double m[PER], msum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = tid * PER + j;
        c[j] = s->cnt[b];
        m[j] = c[j] && (!by_count || edge >= 0.f) ? (double)(edge >= 0.f ? edge : sm_edge(row, b)) * ((double)c[j] - (double)s->eps[b] * unit)
                                 : 0.0;
        csum += c[j];
        msum += m[j];
    }
    unsigned ci = csum;
    double mi = msum;
    const bool mass = !by_count || edge >= 0.f;   // the block together
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned p = __shfl_up_sync(0xffffffffu, ci, o);
        if (lane >= o) ci += p;
        if (mass) {
            const double q = __shfl_up_sync(0xffffffffu, mi, o);
            if (lane >= o) mi += q;
        }
    }
    if (lane == 31) { s->scan_n[warp] = ci; s->scan[warp] = mi; }
    if (tid == 0) s->out_i = SM_NB;
    __syncthreads();
    unsigned cb = 0;
    double mb = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) cb += s->scan_n[w];
        if (mass) {
            if (w < warp) mb += s->scan[w];
            all += s->scan[w];
        }
    }
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
    *total = all;
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

// The tokens that CL blocks finish: n0 of this block, logits x, in index order. List: their indices, null where they
// are consecutive from first.
struct SmSlice {
    const float* x;
    const int* list;
    int n0, first;
    __device__ __forceinline__ int index(int i) const { return list ? list[i] : first + i; }
};

// All blocks: counts (and, with mass, distances) per bin of the row.
template <int CL> __device__ __forceinline__ void sm_histogram(SmShared* s, const SmSlice& z, const SmRow& row, bool mass) {
    for (int b = threadIdx.x; b < SM_NB; b += SM_THREADS) s->cnt[b] = s->eps[b] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < z.n0; i += SM_THREADS) {
        const float l = z.x[i];
        if (!(l > -INFINITY)) continue;
        const float d = sm_dist(row, l);
        const int b = sm_bin(row, d);
        atomicAdd(&s->cnt[b], 1u);
        if (mass) atomicAdd(&s->eps[b], sm_eps(row, b, d));
    }
    sm_combine<CL>(s);
}

// All blocks: the boundary token within bin `bin` (before_n tokens of weight before_m come earlier in the order): the
// one that is number tcount of the row (by_count), or at which the running weight reaches tmass. Returns the weight up
// to and including it. n: tokens in the bin.
template <int CL>
__device__ __noinline__ double sm_boundary(SmShared* s, const SmSlice& z, const SmRow& row, int bin, unsigned n,
                                           bool by_count, unsigned tcount, double tmass, unsigned before_n,
                                           double before_m, SmEntry* cut) {
    const int tid = threadIdx.x;
    const int rank = CL > 1 ? (int)cluster_ctarank() : 0;
    const float edge = sm_edge(row, bin);
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
        for (int i = tid; i < z.n0; i += SM_THREADS)
            if (in(z.x[i])) { lo = min(lo, float_key(z.x[i])); hi = max(hi, float_key(z.x[i])); }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if ((tid & 31) == 0) { atomicMin(&s->kmin, lo); atomicMax(&s->kmax, hi); }
        for (int b = tid; b < SM_NB; b += SM_THREADS) s->cnt[b] = s->eps[b] = 0u;
        row_sync<CL>();
        lo = 0xffffffffu;
        hi = 0u;
#pragma unroll
        for (int r = 0; r < CL; ++r) { lo = min(lo, peer<CL>(&s->kmin, r)); hi = max(hi, peer<CL>(&s->kmax, r)); }
        klo = lo;
        khi = hi;
        if (lo == hi) break;
        const int shift = max(0, 32 - __clz(hi - lo) - 10);   // (hi - key) >> shift < 1024
        for (int i = tid; i < z.n0; i += SM_THREADS)
            if (in(z.x[i])) {
                const int b = (int)((hi - float_key(z.x[i])) >> shift);
                atomicAdd(&s->cnt[b], 1u);
                atomicAdd(&s->eps[b], sm_eps(row, bin, sm_dist(row, z.x[i])));
            }
        sm_combine<CL>(s);
        unsigned bn;
        double bm, total;
        int b = sm_find(s, row, by_count, tcount - before_n, tmass - before_m, edge, &bn, &bm, &total);
        if (b == SM_NB) {   // rounding: the target lies just past the bin's weight; its last part
            b = (int)((hi - lo) >> shift);
            bn = n - s->cnt[b];
            bm = total;
        }
        n = s->cnt[b];
        before_n += bn;
        before_m += bm;
        khi = hi - ((unsigned)b << shift);
        const unsigned width = (1u << shift) - 1u;
        klo = max(lo, khi > width ? khi - width : 0u);
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
        // occurrences in the blocks before this one, then per warp (contiguous pieces)
        const int lane = tid & 31, warp = tid >> 5, nw = SM_THREADS / 32;
        const int piece = (z.n0 + nw - 1) / nw, i0 = min(z.n0, warp * piece), i1 = min(z.n0, i0 + piece);
        unsigned mine = 0;
        for (int i = i0 + lane; i < i1; i += 32) mine += float_key(z.x[i]) == khi ? 1u : 0u;
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
            const bool hit = i + lane < i1 && float_key(z.x[i + lane]) == khi;
            const unsigned m = __ballot_sync(0xffffffffu, hit);
            const unsigned at = ahead + __popc(m & ((2u << lane) - 1u));
            if (hit && at == r) s->cut.i = z.index(i + lane);
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
    for (int i = tid; i < z.n0; i += SM_THREADS)
        if (in(z.x[i])) {
            const int at = atomicAdd(&s->nlist, 1);
            if (at < SM_CAP) s->list[at] = SmEntry{z.x[i], z.index(i)};
        }
    row_sync<CL>();
    const SmEntry* all = s->list;
    int m = s->nlist;
    if constexpr (CL > 1) {
        m = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
            const int c = min(peer<CL>(&s->nlist, r), SM_CAP - m);
            for (int i = tid; i < c; i += SM_THREADS) s->all[m + i] = peer<CL>(&s->list[i], r);
            m += c;
        }
        all = s->all;
        row_sync<CL>();
    }
    // weights in units of 2^-30 of the bin's edge: integers, whose sums do not depend on the order of the list
    const float up = edge > 0.f ? __fdiv_rn(1073741824.f, edge) : 0.f;
    if (!by_count || tmass >= 0.0) {
        for (int i = tid; i < m; i += SM_THREADS) s->q[i] = __float2uint_rn(sm_weight(sm_dist(row, all[i].l)) * up);
        __syncthreads();
    }
    // every token's number in the order, and the weight before it
    const unsigned want = by_count ? tcount - before_n : 0u;
    const double tgt = tmass - before_m, unit = (double)edge * (1.0 / 1073741824.0);
    for (int i = tid; i < m; i += SM_THREADS) {
        const SmEntry e = all[i];
        unsigned ahead = 0;
        unsigned long long mass = 0;
        if (!by_count || tmass >= 0.0) {
            for (int j = 0; j < m; ++j) {
                const SmEntry f = all[j];
                if (f.l > e.l || (f.l == e.l && f.i < e.i)) {
                    ++ahead;
                    mass += s->q[j];
                }
            }
        } else {
            for (int j = 0; j < m; ++j) {
                const SmEntry f = all[j];
                ahead += f.l > e.l || (f.l == e.l && f.i < e.i);
            }
        }
        const double before = (double)mass * unit, w = by_count && tmass < 0.0 ? 0.0 : (double)s->q[i] * unit;
        const bool hit = by_count ? ahead + 1 == want
                                  : (ahead == 0 || before < tgt) && ((int)ahead + 1 == m || before + w >= tgt);
        if (hit) {
            s->cut = e;
            s->cut_mass = before_m + before + w;
        }
    }
    __syncthreads();
    *cut = s->cut;
    const double cm = s->cut_mass;
    __syncthreads();
    return cm;
}

// All blocks: the last token that top-k and top-p keep, by histograms.
template <int CL>
__device__ __forceinline__ SmEntry sm_cut(SmShared* s, const SmSlice& z, const SmRow& row, int k, int held, float tp) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool by_k = k > 1 && k < held, by_p = tp < 1.f;
    SmEntry cut{-INFINITY, 0x7fffffff};   // keep everything
    if (by_k || by_p) {
        sm_histogram<CL>(s, z, row, by_p);
        unsigned bn;
        double bm, total;
        int kbin = SM_NB;
        unsigned kn = 0;
        if (by_k) {   // SM_NB: fewer than k tokens
            kbin = sm_find(s, row, true, (unsigned)k, 0.0, -1.f, &bn, &bm, &total);
            if (kbin < SM_NB) kn = s->cnt[kbin];
            __syncthreads();
        }
        if (!by_p) {
            if (kbin < SM_NB) sm_boundary<CL>(s, z, row, kbin, kn, true, (unsigned)k, -1.0, bn, 0.0, &cut);
        } else {
            SmEntry kcut = cut;
            if (kbin < SM_NB) {
                // the weight of the bins before the boundary's, then the weight up to the boundary
                double mine = 0.0;
                for (int b = tid; b < kbin; b += SM_THREADS)
                    if (s->cnt[b])
                        mine += (double)sm_edge(row, b) * ((double)s->cnt[b] - (double)s->eps[b] * ((double)row.step / 8192.0));
#pragma unroll
                for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
                if (lane == 0) s->scan[warp] = mine;
                __syncthreads();
                bm = 0.0;
#pragma unroll
                for (int w = 0; w < SM_THREADS / 32; ++w) bm += s->scan[w];
                __syncthreads();
                total = sm_boundary<CL>(s, z, row, kbin, kn, true, (unsigned)k, 0.0, bn, bm, &kcut);
                if (kn > SM_CAP) sm_histogram<CL>(s, z, row, true);   // the search used the histogram up
            } else {
                sm_find(s, row, false, 0u, 1e300, -1.f, &bn, &bm, &total);
            }
            const double want = (double)tp * total;
            unsigned pn;
            double pm;
            const int pbin = sm_find(s, row, false, 0u, want, -1.f, &pn, &pm, &total);
            const unsigned pcount = pbin < SM_NB ? s->cnt[pbin] : 0u;
            __syncthreads();
            SmEntry pcut = cut;
            if (pbin < SM_NB) sm_boundary<CL>(s, z, row, pbin, pcount, false, 0u, want, pn, pm, &pcut);
            cut = pcut.l > kcut.l || (pcut.l == kcut.l && pcut.i < kcut.i) ? pcut : kcut;
        }
    }
    return cut;
}

// All blocks: the token among those down to `cut` that weigh at least mp of the largest.
template <int CL>
__device__ __forceinline__ void sm_take(SmShared* s, const SmSlice& z, const SmRow& row, SmEntry cut, float mp, float u,
                                        int32_t* token, float* prob) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = CL > 1 ? (int)cluster_ctarank() : 0;
    // ---- the kept weight, by warp (contiguous pieces), block and row ----
    const float floor_w = fminf(mp, 1.f);
    auto kept = [&](int i) {   // weight of token i, 0 where it is not kept
        const float l = z.x[i], w = sm_weight(sm_dist(row, l));
        const bool in = l > cut.l || (l == cut.l && (cut.i == 0x7fffffff || z.index(i) <= cut.i));
        return in && w >= floor_w ? w : 0.f;
    };
    constexpr int nw = SM_THREADS / 32;
    const int piece = (z.n0 + nw - 1) / nw, i0 = min(z.n0, warp * piece), i1 = min(z.n0, i0 + piece);
    float part = 0.f;
#pragma unroll 4
    for (int i = i0 + lane; i < i1; i += 32) part += kept(i);
    part = warp_sum(part);
    if (lane == 0) s->wsum[warp] = (double)part;
    __syncthreads();
    double mine = 0.0, own = 0.0;   // warp 0: lane i has warp i's weight, and the block's
    if (warp == 0) {
        mine = lane < nw ? s->wsum[lane] : 0.0;
        own = mine;
#pragma unroll
        for (int o = 16; o; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    }
    double ahead = 0.0, total = own;
    int last = 0;   // the last block with any weight
    if constexpr (CL > 1) {
        if (tid == 0) s->sum = own;
        row_sync<CL>();
        if (warp == 0) {
            total = 0.0;
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                const double v = peer<CL>(&s->sum, r);
                if (r < rank) ahead += v;
                total += v;
                if (v > 0.0) last = r;
            }
        }
    }
    const double target = (double)u * total;
    // this block holds the token if the target falls into its part (the last one with weight takes rounding at the end)
    if (warp == 0 && own > 0.0 && ahead <= target && (target < ahead + own || rank == last)) {
        double inc = mine;
#pragma unroll
        for (int o = 1; o < nw; o <<= 1) {
            const double p = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += p;
        }
        // the warp's piece that the target falls into: the first that passes it, else the last with weight
        const unsigned pass = __ballot_sync(0xffffffffu, mine > 0.0 && target < ahead + inc);
        const unsigned any = __ballot_sync(0xffffffffu, mine > 0.0);
        const int w = pass ? __ffs(pass) - 1 : 31 - __clz(any);
        double m = ahead + __shfl_sync(0xffffffffu, inc - mine, w);
        const int a0 = min(z.n0, w * piece), a1 = min(z.n0, a0 + piece);
        int found = -1, back = -1;
        float fw = 0.f, bw = 0.f;
        for (int i = a0; i < a1 && found < 0; i += 32) {
            const float v = i + lane < a1 ? kept(i + lane) : 0.f;
            float run = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float p = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += p;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, v > 0.f && m + (double)run > target);
            const unsigned some = __ballot_sync(0xffffffffu, v > 0.f);
            if (hit) {
                const int b = __ffs(hit) - 1;
                found = i + b;
                fw = __shfl_sync(0xffffffffu, v, b);
            } else if (some) {
                const int b = 31 - __clz(some);
                back = i + b;
                bw = __shfl_sync(0xffffffffu, v, b);
            }
            m += (double)__shfl_sync(0xffffffffu, run, 31);
        }
        if (found < 0) { found = back; fw = bw; }
        if (lane == 0) {
            *token = z.index(found);
            if (prob) *prob = (float)((double)fw / total);
        }
    }
}

template <int DT, int CL>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const SampleArgs a) {
    using T = typename Elem<DT>::T;
    extern __shared__ __align__(16) uint8_t smem[];
    SmShared* s = reinterpret_cast<SmShared*>(smem);
    float* x = reinterpret_cast<float*>(smem + (sizeof(SmShared) + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = SM_THREADS / 32;
    const int rank = CL > 1 ? (int)cluster_ctarank() : 0, rw = blockIdx.x / CL;
    const int first = rank * a.slice, n0 = max(0, min(a.slice, a.V - first));
    pdl_trigger();
    pdl_wait();
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
        constexpr int UN = DT == VKB_DT_F32 ? 3 : 5;
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
    const float t = a.temperature ? a.temperature[rw] : 1.f, u = fminf(fmaxf(a.u[rw], 0.f), 1.f);   // NaN: 0
    const int k = a.top_k ? a.top_k[rw] : 0;
    const float tp = a.top_p ? a.top_p[rw] : 1.f, mp = a.min_p ? a.min_p[rw] : 0.f;
    s->tmax[tid] = hi;
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
    if (warp == 0) {
        const SmEntry e = lane < NW ? s->list[lane] : SmEntry{-INFINITY, 0x7fffffff};
        hi = e.l;
        arg = e.i;
        lo = lane < NW ? s->list[32 + lane].l : INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float h2 = __shfl_xor_sync(0xffffffffu, hi, o);
            const int a2 = __shfl_xor_sync(0xffffffffu, arg, o);
            if (h2 > hi || (h2 == hi && a2 < arg)) { hi = h2; arg = a2; }
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        if (lane == 0) {
            s->range = make_float2(hi, lo);
            s->arg = arg;
        }
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
    row.c = __fdiv_rn(1.4426950408889634f, t);
    const float span = hi == lo ? 0.f : (hi - lo) * row.c;
    row.step = fminf(SM_SPAN, fmaxf(1.01f * span, 1e-3f)) * (1.f / (SM_NB - 1));   // shorter spans stay off the last bin
    row.inv_bin = __fdiv_rn(1.f, row.step);
    if constexpr (CL > 1) {
        if (k > 1 && k <= SM_THREADS * CL / 5 * 3) {
            // ---- candidates: the tokens down to a logit that at least k threads' maxima reach ----
            for (int b = tid; b < SM_NB; b += SM_THREADS) s->cnt[b] = 0u;
            float m[CL];
#pragma unroll
            for (int r = 0; r < CL; ++r) m[r] = peer<CL>(&s->tmax[tid], r);
            __syncthreads();
#pragma unroll
            for (int r = 0; r < CL; ++r)
                if (m[r] > -INFINITY) atomicAdd(&s->cnt[sm_bin(row, sm_dist(row, m[r]))], 1u);
            if (tid == 0) s->kmin = 0xffffffffu;
            __syncthreads();
            unsigned bn;
            double bm, total;
            const int bin = sm_find(s, row, true, (unsigned)k, 0.0, -1.f, &bn, &bm, &total);
            unsigned low = 0xffffffffu;   // the smallest maximum down to that bin (all finite tokens: fewer than k maxima)
            if (bin < SM_NB - 1) {
#pragma unroll
                for (int r = 0; r < CL; ++r)
                    if (m[r] > -INFINITY && sm_bin(row, sm_dist(row, m[r])) <= bin) low = min(low, float_key(m[r]));
                low = __reduce_min_sync(0xffffffffu, low);
                if (lane == 0) atomicMin(&s->kmin, low);
            }
            __syncthreads();
            const unsigned kl = bin < SM_NB - 1 ? s->kmin : float_key(-INFINITY) + 1u;
            const float tau = __uint_as_float(kl ^ ((kl >> 31) ? 0x80000000u : 0xffffffffu));
            // this block's candidates, in index order: counted per warp (contiguous pieces), then written
            const int piece = (n0 + NW - 1) / NW, i0 = min(n0, warp * piece), i1 = min(n0, i0 + piece);
            unsigned c = 0;
            for (int i = i0 + lane; i < i1; i += 32) c += x[i] >= tau;
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0) s->scan_n[warp] = c;
            __syncthreads();
            unsigned at = 0, n = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                at += w < warp ? s->scan_n[w] : 0u;
                n += s->scan_n[w];
            }
            if (n <= SM_LOCAL)
                for (int i = i0; i < i1; i += 32) {   // whole warp
                    const bool hit = i + lane < i1 && x[i + lane] >= tau;
                    const unsigned b = __ballot_sync(0xffffffffu, hit);
                    if (hit) s->cand[at + __popc(b & ((1u << lane) - 1u))] = SmEntry{x[i + lane], first + i + lane};
                    at += __popc(b);
                }
            if (tid == 0) s->ncand = (int)n;
            row_sync<CL>();
            int count = 0;
            bool fits = true;
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                const int v = peer<CL>(&s->ncand, r);
                fits = fits && v <= SM_LOCAL;
                count += v;
            }
            fits = fits && 2 * count <= a.slice;   // logits and indices take the place of the first block's slice
            if (fits) {
                int* list = reinterpret_cast<int*>(x + count);
                if (rank == 0) {
                    int base = 0;
#pragma unroll
                    for (int r = 0; r < CL; ++r) {
                        const int v = peer<CL>(&s->ncand, r);
                        for (int i = tid; i < v; i += SM_THREADS) {
                            const SmEntry e = peer<CL>(&s->cand[i], r);
                            x[base + i] = e.l;
                            list[base + i] = e.i;
                        }
                        base += v;
                    }
                }
                row_sync<CL>();   // the others leave
                if (rank == 0) {
                    const SmSlice z{x, list, count, 0};
                    const SmEntry cut = sm_cut<1>(s, z, row, k, a.V, tp);
                    sm_take<1>(s, z, row, cut, mp, u, a.token + rw, a.prob ? a.prob + rw : nullptr);
                }
                return;
            }
            row_sync<CL>();   // the candidates' counts have been read
        }
    }
    const SmSlice z{x, nullptr, n0, first};
    sm_take<CL>(s, z, row, sm_cut<CL>(s, z, row, k, a.V, tp), mp, u, a.token + rw, a.prob ? a.prob + rw : nullptr);
    if constexpr (CL > 1) row_sync<CL>();
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
    // Blocks per row, by the row's length alone: up to 4096 logits each until there are eight, whatever the batch.
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
