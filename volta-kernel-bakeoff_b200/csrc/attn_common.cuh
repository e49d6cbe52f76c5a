// Attention over the paged 8-bit cache: the arguments, the division of the work over the SMs, and the joining of a
// query tile whose keys were split, shared by the two kernels (attn_token.cuh, attn_prompt.cuh).
//
// A work item is one sequence, one kv head and one tile of ROWS query rows; row r of a sequence is query token r / G,
// head h G + r % G (G = q heads per kv head), so that the heads sharing a kv head read its codes once. An item's units
// are its tiles of KT keys, from the first key that any of its rows sees to the last (an item that sees none has one
// empty unit, which writes its zeros). The units of all items, in order, are dealt out to the thread blocks in equal
// contiguous runs, worked out on the device from the lengths there: ragged batches balance, nothing is read back to
// the host, and a captured graph stays right as sequences grow. An item cut by a run's border is a "part" in each
// block: its unnormalised sums go to the workspace, and the block that arrives last joins the parts in block order
// (the result does not depend on which that is).
#pragma once

#include <type_traits>

#include "step.cuh"

namespace vkb {

struct AttnArgs {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    const float* ks;
    const float* vs;
    const void* q;
    void* out;
    float* part;          // [grid][2] parts: sums [DT / 4][ROWS][4], then {maximum, sum} [ROWS][2]
    unsigned* cnt;        // [grid] arrivals of the item that starts in this block; zero between calls
    long long ldq, ldo;
    float scale_log2;     // scale * log2(e)
    int B, T, heads, G, dim, pages, page_log2, table_ld, window;
};

struct AttnSeq {
    int len, n, q0;
};
// Sequence b: length with its new tokens, new tokens, first query row. Indices that do not fit the call or the table
// raise a status bit and leave the sequence out.
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int b) {
    AttnSeq s;
    s.len = a.lens[b];
    s.q0 = a.cu ? a.cu[b] : b;
    s.n = a.cu ? a.cu[b + 1] - s.q0 : 1;
    if (s.len < 0 || s.n < 0 || s.q0 < 0 || s.q0 > a.T - s.n || s.len > ((long long)a.table_ld << a.page_log2)) {
        raise_status(DEV_ERR_BAD_INDEX);
        s.len = s.n = 0;
    }
    return s;
}
// The key tiles [t0, t1) of rows [r0, r1) of a sequence (t1 <= t0: no row sees a key).
template <int KT> __device__ __forceinline__ void attn_tiles(const AttnArgs& a, const AttnSeq& s, int r0, int r1, int* t0, int* t1) {
    const int first = s.len - s.n + r0 / a.G, last = s.len - s.n + (r1 - 1) / a.G;   // token positions
    const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
    *t0 = lo / KT;
    *t1 = last >= 0 ? (last + KT) / KT : 0;
    if (*t1 < *t0) *t1 = *t0;
}
template <int KT> __device__ __forceinline__ int attn_units(const AttnArgs& a, const AttnSeq& s, int r0, int r1) {
    int t0, t1;
    attn_tiles<KT>(a, s, r0, r1, &t0, &t1);
    return max(1, t1 - t0);
}
// Units of one head of a sequence.
template <int ROWS, int KT> __device__ __forceinline__ long long attn_head_units(const AttnArgs& a, const AttnSeq& s) {
    const int rows = s.n * a.G;
    long long u = 0;
    for (int r = 0; r < rows; r += ROWS) u += attn_units<KT>(a, s, r, min(rows, r + ROWS));
    return u;
}

// A run of units: where it starts, and the walk over its segments.
struct AttnRun {
    long long u, u1, total;   // next unit, end of the run, units of the call
    int nb;                   // blocks with a run
    int b, h, r0, off;        // next item and the units of it that belong to earlier blocks
};
struct AttnSeg {
    int b, h, r0, rows;       // rows of the tile
    int pos0, q0;             // position of the sequence's first query token, its row in q and out
    int t0, t1;               // key tiles of this segment
    int len;
    long long iu0, iu1;       // the whole item's units
    bool whole;
};

// First unit of block c's run.
__device__ __forceinline__ long long attn_start(long long total, int nb, int c) { return total * c / nb; }
// The block whose run holds unit x.
__device__ __forceinline__ int attn_owner(long long total, int nb, long long x) {
    return (int)(((x + 1) * nb - 1) / total);
}

// All threads of the block: this block's run. sh: 2 + NT / 32 words of 8 bytes of shared memory.
template <int ROWS, int KT, int NT> __device__ __forceinline__ AttnRun attn_run(const AttnArgs& a, long long* sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NT / 32;
    AttnRun r;
    long long total = 0, mine0 = 0;
    for (int b = tid; b < a.B; b += NT) {
        const AttnSeq s = attn_seq(a, b);
        const long long u = a.heads * attn_head_units<ROWS, KT>(a, s);
        if (b == tid) mine0 = u;
        total += u;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) sh[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += sh[w];
    __syncthreads();
    r.total = total;
    r.nb = (int)min((long long)gridDim.x, total);
    r.u = r.u1 = 0;
    r.b = r.h = r.r0 = r.off = 0;
    if ((int)blockIdx.x >= r.nb) return r;
    r.u = attn_start(total, r.nb, blockIdx.x);
    r.u1 = attn_start(total, r.nb, blockIdx.x + 1);
    // the sequence that holds unit r.u: a scan, NT sequences at a time
    long long left = r.u;
    for (int base = 0; base < a.B; base += NT) {
        const int b = base + tid;
        long long u = mine0;
        if (base > 0) u = b < a.B ? a.heads * attn_head_units<ROWS, KT>(a, attn_seq(a, b)) : 0;
        long long inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) sh[warp] = inc;
        __syncthreads();
        long long before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            before += w < warp ? sh[w] : 0;
            all += sh[w];
        }
        const long long at = left - (before + inc - u);
        if (at >= 0 && at < u) {
            sh[NW] = b;
            sh[NW + 1] = at;
        }
        __syncthreads();
        if (left < all) break;
        left -= all;
    }
    r.b = (int)sh[NW];
    const AttnSeq s = attn_seq(a, r.b);
    const long long per = attn_head_units<ROWS, KT>(a, s);
    long long at = sh[NW + 1];
    r.h = (int)(at / per);
    at -= r.h * per;
    const int rows = s.n * a.G;
    for (;; r.r0 += ROWS) {
        const int u = attn_units<KT>(a, s, r.r0, min(rows, r.r0 + ROWS));
        if (at < u) break;
        at -= u;
    }
    r.off = (int)at;
    return r;
}

// The run's next segment; false at its end.
template <int ROWS, int KT> __device__ __forceinline__ bool attn_next(const AttnArgs& a, AttnRun& r, AttnSeg* g) {
    if (r.u >= r.u1) return false;
    AttnSeq s = attn_seq(a, r.b);
    while (s.n == 0) {   // sequences without query tokens have no unit
        if (r.b + 1 >= a.B) return false;
        s = attn_seq(a, ++r.b);
    }
    const int rows = s.n * a.G;
    g->b = r.b;
    g->h = r.h;
    g->r0 = r.r0;
    g->rows = min(ROWS, rows - r.r0);
    g->pos0 = s.len - s.n;
    g->q0 = s.q0;
    g->len = s.len;
    int t0, t1;
    attn_tiles<KT>(a, s, r.r0, r.r0 + g->rows, &t0, &t1);
    const int units = max(1, t1 - t0);
    const int take = (int)min((long long)(units - r.off), r.u1 - r.u);
    g->iu0 = r.u - r.off;
    g->iu1 = g->iu0 + units;
    g->whole = take == units;
    g->t0 = t0 + r.off;
    g->t1 = min(t1, g->t0 + take);
    r.u += take;
    r.off = 0;
    r.r0 += ROWS;
    if (r.r0 >= rows) {
        r.r0 = 0;
        if (++r.h == a.heads) {
            r.h = 0;
            ++r.b;
        }
    }
    return true;
}

// Where a part of this block goes: slot 1 for the item that starts in the block, 0 for one that started earlier.
__device__ __forceinline__ long long attn_slot(const AttnRun& r, const AttnSeg& g, int c) {
    return 2ll * c + (attn_owner(r.total, r.nb, g.iu0) == c ? 1 : 0);
}

// Output row of row r of a segment.
template <typename T> __device__ __forceinline__ T* attn_out(const AttnArgs& a, const AttnSeg& g, int r) {
    const int t = (g.r0 + r) / a.G, hq = g.h * a.G + (g.r0 + r) - t * a.G;
    return reinterpret_cast<T*>(a.out) + (g.q0 + t) * a.ldo + (long long)hq * a.dim;
}

// The threads tid of n (all of them, after the block's parts are written by them and a barrier among them): arrive for
// the segment's item, and where this block is the last, join its parts and write the output. bar: a barrier among the n
// threads. sh: a word of shared memory that they share.
template <int DT, int ROWS, typename T, typename Bar>
__device__ __forceinline__ void attn_join(const AttnArgs& a, const AttnRun& r, const AttnSeg& g, int tid, int n,
                                          volatile int* sh, Bar bar) {
    const int c0 = attn_owner(r.total, r.nb, g.iu0), c1 = attn_owner(r.total, r.nb, g.iu1 - 1), parts = c1 - c0 + 1;
    __threadfence();   // this thread's part, before the arrival
    bar();
    if (tid == 0) {
        __threadfence();
        *sh = atomicInc(&a.cnt[c0], (unsigned)(parts - 1)) == (unsigned)(parts - 1);   // wraps to zero
        __threadfence();
    }
    bar();
    if (!*sh) return;
    constexpr int PITCH = DT + 2;
    const float* base = a.part;
    auto slot = [&](int c) { return base + (2ll * c + (c == c0 ? 1 : 0)) * ROWS * PITCH; };
    // A thread takes four columns of a row; neighbouring threads neighbouring rows, as the parts lie.
    const int work = g.rows * (a.dim >> 2);
    for (int i = tid; i < work; i += n) {
        const int d4 = i / g.rows, row = i - d4 * g.rows;
        float m = -INFINITY;
#pragma unroll 8
        for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(slot(c) + ROWS * DT + 2 * row));
        if (m == -INFINITY) m = 0.f;   // no part saw a key
        float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int c = c0; c <= c1; ++c) {
            const float* p = slot(c);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + ROWS * DT + 2 * row));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p) + d4 * ROWS + row);
            const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
            l = fmaf(w, ml.y, l);
            o[0] = fmaf(w, v.x, o[0]);
            o[1] = fmaf(w, v.y, o[1]);
            o[2] = fmaf(w, v.z, o[2]);
            o[3] = fmaf(w, v.w, o[3]);
        }
        const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
        uint2 w;
        if constexpr (std::is_same<T, __half>::value)
            w = make_uint2(pack_f16(o[0] * inv, o[1] * inv), pack_f16(o[2] * inv, o[3] * inv));
        else
            w = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
        *reinterpret_cast<uint2*>(attn_out<T>(a, g, row) + 4 * d4) = w;
    }
}

}  // namespace vkb
