// Attention over the paged 8-bit cache: the arguments, the division of the work over the SMs, and the joining of a
// query tile whose keys were split, shared by the two kernels (attn_token.cuh, attn_prompt.cuh).
//
// A work item is one sequence, one kv head and one tile of ROWS query rows; row r of a sequence is query token r / G,
// head h G + r % G (G = q heads per kv head), so that the heads sharing a kv head read its codes once. An item's units
// are its tiles of KT keys, from the first key that any of its rows sees to the last (an item that sees none has one
// empty unit, which writes its zeros), and OV more in front of them, which stand for what an item costs beside its keys
// (q, the joining of the warps, the output; measured at 16 for both kernels: a batch of 64 sequences of 1 to 8192 tokens 168 us
// without, 111 us with them, ragged prompts through a window 906 and 483 us). The units of all items, in order, are dealt out to the thread blocks in equal
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
    int B, T, heads, G, dim, pages, page_log2, table_ld, window, max_len;
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
    if (s.len < 0 || s.n < 0 || s.q0 < 0 || s.q0 > a.T - s.n || s.len > a.max_len) {
        raise_status(DEV_ERR_BAD_INDEX);
        s.len = s.n = 0;
    }
    return s;
}
// The window's first key for a row at position p (at most 0: all). Rows before position 0 see no key; they count as position
// 0 here, so that no window, however wide, wraps around.
__device__ __forceinline__ int attn_window(const AttnArgs& a, int p) { return a.window > 0 ? max(p, 0) - a.window + 1 : 0; }
// The key tiles [t0, t1) of rows [r0, r1) of a sequence (t1 <= t0: no row sees a key).
template <int KT> __device__ __forceinline__ void attn_tiles(const AttnArgs& a, const AttnSeq& s, int r0, int r1, int* t0, int* t1) {
    const int first = s.len - s.n + r0 / a.G, last = s.len - s.n + (r1 - 1) / a.G;   // token positions
    *t0 = max(0, attn_window(a, first)) / KT;
    *t1 = last >= 0 ? (last + KT) / KT : 0;
    if (*t1 < *t0) *t1 = *t0;
}
template <int KT, int OV> __device__ __forceinline__ int attn_units(const AttnArgs& a, const AttnSeq& s, int r0, int r1) {
    int t0, t1;
    attn_tiles<KT>(a, s, r0, r1, &t0, &t1);
    return max(1, t1 - t0) + OV;
}
// Units of one head of a sequence.
template <int ROWS, int KT, int OV> __device__ __forceinline__ unsigned attn_head_units(const AttnArgs& a, const AttnSeq& s) {
    const int rows = s.n * a.G;
    unsigned u = 0;
    for (int r = 0; r < rows; r += ROWS) u += (unsigned) attn_units<KT, OV>(a, s, r, min(rows, r + ROWS));
    return u;
}

// A run of units: where it starts, and the walk over its segments. The host refuses calls whose spans could have 2^31 units if
// each row is in one span. Where offsets decrease from one sequence to the next (which raises a status bit), spans overlap and
// their units may pass 2^32: such a call is left out.
struct AttnRun {
    unsigned u, u1;           // next unit, end of the run
    unsigned per, rem;        // block c's run: per units from c per + min(c, rem) on, one more where c < rem
    int b, h, r0, off;        // next item and the units of it that belong to earlier blocks
};
struct AttnSeg {
    int b, h, r0, rows;       // rows of the tile
    int pos0, q0;             // position of the sequence's first query token, its row in q and out
    int t0, t1;               // key tiles of this segment
    int len;
    int c0, c1;               // blocks that hold the item (c0 == c1: this one, whole)
    bool whole;
};

__device__ __forceinline__ unsigned attn_start(const AttnRun& r, int c) { return c * r.per + min((unsigned)c, r.rem); }
// The block whose run holds unit x.
__device__ __forceinline__ int attn_owner(const AttnRun& r, unsigned x) {
    const unsigned big = r.rem * (r.per + 1);
    return (int)(x < big ? x / (r.per + 1) : r.rem + (x - big) / r.per);
}

// All threads of the block: this block's run. sh: 2 + NT / 32 words of shared memory. left_out: one more, whether the call is
// left out (through shared memory: kept as a value it cost the kernels' loops registers, 1.23 ms instead of 1.21 for a chunk of
// 4096 tokens).
template <int ROWS, int KT, int OV, int NT> __device__ __forceinline__ AttnRun attn_run(const AttnArgs& a, unsigned* sh, volatile int* left_out) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NT / 32;
    AttnRun r;
    unsigned total = 0, mine0 = 0;
    int overlap = 0;
    for (int b = tid; b < a.B; b += NT) {
        const AttnSeq s = attn_seq(a, b);
        const unsigned u = a.heads * attn_head_units<ROWS, KT, OV>(a, s);
        if (b == tid) mine0 = u;
        total += u;
        overlap |= a.cu && a.cu[b] > a.cu[b + 1];
    }
    total = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) sh[warp] = total;
    overlap = __syncthreads_or(overlap);
    *left_out = overlap;   // every thread the same
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += sh[w];
    __syncthreads();
    const unsigned nb = min(gridDim.x, total);
    r.u = r.u1 = r.rem = 0;
    r.per = 1;
    r.b = r.h = r.r0 = r.off = 0;
    if (blockIdx.x >= nb || *left_out) return r;
    r.per = total / nb;
    r.rem = total - r.per * nb;
    r.u = attn_start(r, blockIdx.x);
    r.u1 = attn_start(r, blockIdx.x + 1);
    // the sequence that holds unit r.u: a scan, NT sequences at a time
    unsigned left = r.u;
    for (int base = 0; base < a.B; base += NT) {
        const int b = base + tid;
        unsigned u = mine0;
        if (base > 0) u = b < a.B ? a.heads * attn_head_units<ROWS, KT, OV>(a, attn_seq(a, b)) : 0;
        unsigned inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) sh[warp] = inc;
        __syncthreads();
        unsigned before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            before += w < warp ? sh[w] : 0;
            all += sh[w];
        }
        before += inc - u;
        if (left >= before && left - before < u) {
            sh[NW] = (unsigned)b;
            sh[NW + 1] = left - before;
        }
        __syncthreads();
        if (left < all) break;
        left -= all;
    }
    r.b = (int)sh[NW];
    const AttnSeq s = attn_seq(a, r.b);
    const unsigned per = attn_head_units<ROWS, KT, OV>(a, s);
    unsigned at = sh[NW + 1];
    r.h = (int)(at / per);
    at -= r.h * per;
    const int rows = s.n * a.G;
    for (;; r.r0 += ROWS) {
        const unsigned u = (unsigned)attn_units<KT, OV>(a, s, r.r0, min(rows, r.r0 + ROWS));
        if (at < u) break;
        at -= u;
    }
    r.off = (int)at;
    return r;
}

// The run's next segment; false at its end.
template <int ROWS, int KT, int OV> __device__ __forceinline__ bool attn_next(const AttnArgs& a, AttnRun& r, AttnSeg* g) {
    for (;;) {
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
        const int units = max(1, t1 - t0) + OV;
        const int off = r.off, take = (int)min((unsigned)(units - off), r.u1 - r.u);
        const unsigned first = r.u - off;   // the item's first unit
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
        if (off + take <= OV) continue;   // nothing but the units in front: the next block has the item's first keys
        g->whole = off <= OV && off + take == units;
        g->c0 = g->c1 = blockIdx.x;
        if (!g->whole) {
            g->c0 = attn_owner(r, first + OV);
            g->c1 = attn_owner(r, first + units - 1);
        }
        g->t0 = t0 + max(0, off - OV);
        g->t1 = min(t1, t0 + off + take - OV);
        return true;
    }
}

// Where a part of block c goes: slot 1 for the item that starts in the block, 0 for one that started earlier.
__device__ __forceinline__ long long attn_slot(const AttnSeg& g, int c) { return 2ll * c + (g.c0 == c ? 1 : 0); }

// The first key that any row of the segment sees. Pages that end before it are not looked at: where a window has passed
// them the caller may have given them to another sequence.
__device__ __forceinline__ int attn_first_key(const AttnArgs& a, const AttnSeg& g) {
    return max(0, attn_window(a, g.pos0 + g.r0 / a.G));
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
__device__ __forceinline__ void attn_join(const AttnArgs& a, const AttnSeg& g, int tid, int n, volatile int* sh, Bar bar) {
    const int parts = g.c1 - g.c0 + 1;
    __threadfence();   // this thread's part, before the arrival
    bar();
    if (tid == 0) {
        __threadfence();
        *sh = atomicInc(&a.cnt[g.c0], (unsigned)(parts - 1)) == (unsigned)(parts - 1);   // wraps to zero
        __threadfence();
    }
    bar();
    if (!*sh) return;
    constexpr int PITCH = DT + 2, BATCH = 8;
    // A thread takes four columns of a row; neighbouring threads neighbouring rows, as the parts lie. Where there are
    // threads for it, four lanes share an item's parts and add their sums up (in a fixed order).
    const int work = g.rows * (a.dim >> 2), sp = parts > 4 && work * 4 <= n ? 4 : 1;
    for (int i0 = 0; i0 < work * sp; i0 += n) {   // every lane takes every turn: the lanes that share an item shuffle
        const int i = (i0 + tid) / sp, k = (i0 + tid) % sp;
        const bool on = i < work;
        const int d4 = on ? i / g.rows : 0, row = on ? i - d4 * g.rows : 0;
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = k; c < parts; c += BATCH * sp) {
            float2 ml[BATCH];
            float4 v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int p = c + j * sp;
                ml[j] = make_float2(-INFINITY, 0.f);
                v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p < parts) {
                    const float* at = a.part + attn_slot(g, g.c0 + p) * ROWS * PITCH;
                    ml[j] = __ldcg(reinterpret_cast<const float2*>(at + ROWS * DT + 2 * row));
                    v[j] = __ldcg(reinterpret_cast<const float4*>(at) + d4 * ROWS + row);
                }
            }
            float mn = m;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) mn = fmaxf(mn, ml[j].x);
            const float mu = mn == -INFINITY ? 0.f : mn, f = exp2f(m - mu);   // nothing seen so far: 0
            l *= f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] *= f;
            m = mn;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const float w = exp2f(ml[j].x - mu);
                l = fmaf(w, ml[j].y, l);
                o[0] = fmaf(w, v[j].x, o[0]);
                o[1] = fmaf(w, v[j].y, o[1]);
                o[2] = fmaf(w, v[j].z, o[2]);
                o[3] = fmaf(w, v[j].w, o[3]);
            }
        }
        if (sp == 4) {
            float mn = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
            const float f = exp2f(m - (mn == -INFINITY ? 0.f : mn));
            l *= f;
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] *= f;
                o[e] += __shfl_xor_sync(0xffffffffu, o[e], 1);
                o[e] += __shfl_xor_sync(0xffffffffu, o[e], 2);
            }
        }
        if (!on || k != 0) continue;
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
