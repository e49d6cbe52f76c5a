// Attention for few query rows per kv head (single tokens, drafted tokens): HBM-bound, the codes are read once and
// everything else hides behind that stream.
//
//   s_jr = (c_j . q_r) ks_j scale log2(e),  p'_jr = 2^(s_jr + log2(vs_j / V) - M_r + 8),
//   O'_r = sum_j p'_jr c'_j,   l_r = sum_j p'_jr (V / vs_j),   o_r = V O'_r / l_r
//
// with codes c, c', one scale per page for K (ks) and V (vs), and V the largest vs so far. One persistent block per SM
// (its run of units: attn_common.cuh), computing warps and four streaming ones, which take the units in turn (one alone
// issues a unit of 16 KB in about 650 cycles, all that an SM's share of HBM allows, and then waits for the ring too). A streaming warp brings, per unit of 64 keys, one TMA box of codes per page piece and 128-byte half for K and for V (128-byte swizzle), and the pages' scales
// with 4-byte asynchronous copies, into a ring of NS stages. Groups of four computing warps take the units in turn, 16
// keys per warp, each warp with its own M and sums, joined once per segment.
// Products are mma.sync.m16n8k16 on fp16 with the keys (or the dimensions) as the 16 rows and the queries as the 8
// columns: S^T = C q^T, then O^T += C'^T p^T, so that 8 query rows (a kv head's q heads) fill a tile; as the 16 rows of
// q C^T they left three quarters of it empty (192 us instead of 169 for 64 sequences of up to 8192 tokens, before the
// division of the work knew an item's own cost). The codes enter exactly (1024 + u as fp16, minus 1152), K through ldmatrix and V through
// transposing ldmatrix on byte pairs, so that a register of four codes gives two operand registers either way; p^T
// reaches the second product through movmatrix. tcgen05 has nothing to add: with 8 rows its tiles would be empty.
// p' is rounded once, to fp16, for the product. It is computed against the M of the keys before; only where one passes
// 2^(8 + 4) the warp finds the new maximum, rescales and computes it again. vs below 2^-30 V counts as that.
// Measured on a B200 (32 q heads on 8, dimension 128): 64 sequences of 1 to 8192 tokens 112 us, 4.5 TB/s of codes; one
// sequence of 131073, 24 heads on 4, 40 us, 3.4 TB/s; one of 777 tokens 9.5 us from the first block's start to the last's end.
// q: fp16 as it is; bf16 rows are scaled by a power of two into fp16's range first (exact but for values 2^-28 below the
// row's largest).
#pragma once

#include "attn_common.cuh"

namespace vkb {

constexpr int AT_KT = 64;                            // keys per unit
constexpr int TK_OV = 16;                            // an item's own cost in units
constexpr int TK_STREAMS = 4;                        // streaming warps
constexpr float TK_P_BIAS = 8.f;                     // p' is kept times 2^8

// The {K, V} scales of keys whose page does not exist.
static __device__ const float tk_no_page[2] = {-INFINITY, 0.f};

// DT: head dimension rounded up to 64, 128 or 256. NQ: tiles of 8 query rows per item.
template <int DT, int NQ> struct TkCfg {
    static constexpr int ROWS = 8 * NQ;
    static constexpr int OREG = DT * NQ / 4;                  // accumulator registers of a thread
    static constexpr int WARPS = OREG <= 32 ? 16 : 8;         // computing warps (groups of four)
    static constexpr int GROUPS = WARPS / 4;
    static constexpr int THREADS = 32 * (WARPS + 4);          // and the streaming warpgroup
    // registers: launched with LREG per thread; the streaming warpgroup keeps PREG, the computing ones have CREG
    static constexpr int LREG = WARPS == 16 ? 96 : 168, PREG = WARPS == 16 ? 32 : 40, CREG = WARPS == 16 ? 112 : 232;
    static_assert(128 * PREG + 32 * WARPS * CREG <= THREADS * LREG, "the split is of what the block is launched with");
    static constexpr bool QREGS = NQ == 1 && DT <= 128;       // q fragments in registers
    static constexpr int HB = DT < 128 ? DT : 128;            // bytes of a box row
    static constexpr int TILE = AT_KT * DT;                   // bytes of one tensor's codes in a stage
    static constexpr int STAGE = 2 * TILE;
    // Stages: a multiple of the streams and the groups, so that a stage always has the same streaming warp and the same
    // group, which take its units in order (a barrier's phase can be waited for only until the next one completes).
    static constexpr int NS = DT == 64 ? 16 : DT == 128 ? 8 : 4;
    static_assert(NS % TK_STREAMS == 0 && TK_STREAMS % GROUPS == 0, "stages belong to a stream and a group");
    static constexpr int Q = QREGS ? 0 : ROWS * DT * 2;       // q in B-fragment order
    static constexpr int MERGE = WARPS * 8 * 64 * 4;          // 64 columns of 8 rows of every warp
    // offsets from the 1024-aligned base
    static constexpr int q_off = NS * STAGE;
    static constexpr int merge_off = q_off + Q;
    static constexpr int ml_off = merge_off + MERGE;          // [warp][ROWS] {M, l}
    static constexpr int row_off = ml_off + WARPS * ROWS * 8; // [ROWS] factor of q
    static constexpr int sc_off = row_off + ROWS * 4;         // [NS][4 pieces]{k, v} scales
    static constexpr int bar_off = (sc_off + NS * 32 + 15) / 16 * 16;
    static constexpr int run_off = bar_off + 16 * NS;
    static constexpr int BYTES = run_off + 4 * (THREADS / 32 + 2) + 16 + 1024;
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The transpose of an 8 x 8 matrix of 16-bit elements, one row's neighbouring pair per thread.
__device__ __forceinline__ uint32_t movm(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// D += A B without volatile: the compiler may interleave independent products.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes (i, j) of v (codes + 128) as the exact fp16 pair of codes: 0x6400 | u is 1024 + u, minus 1152.
__device__ __forceinline__ uint32_t codes_f16(uint32_t v, uint32_t sel) {
    return h2_sub(prmt(v, 0x64646464u, sel), 0x64806480u);
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Larger of fp16 pairs; a NaN stays.
__device__ __forceinline__ uint32_t h2_max(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}
// The power of two that brings a row of largest magnitude m into [2^13, 2^14).
__device__ __forceinline__ float row_factor(float m) {
    const int e = (int)(__float_as_uint(m) >> 23) - 127;             // floor(log2 m); tiny: -127
    return m == 0.f ? 1.f : exp2f((float)min(126, max(-126, 13 - e)));
}

// Shared address of 16-byte chunk c of key row r of a stage's tile of codes (the TMA swizzles: 128-byte rows XOR the row's
// low three bits into the chunk, 64-byte rows bits 1-2 of the row).
template <int DT> __device__ __forceinline__ uint32_t code_addr(uint32_t tile, int r, int c) {
    if constexpr (DT == 64) return tile + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    else return tile + (c >> 3) * (AT_KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The B fragments of query row tile nq of a segment: {b0, b1} of k step ks hold elements 16 ks + 4 c .. + 3 of query
// 8 nq + lane / 4, the k order of the codes' registers. Returns the row's factor (bf16).
template <int DT, typename T>
__device__ __forceinline__ float tk_load_q(const AttnArgs& a, const AttnSeg& g, int nq, int lane, uint2 (&w)[DT / 16]) {
    const int r = 8 * nq + (lane >> 2), qc = lane & 3;
    const bool on = r < g.rows;
    const int t = (g.r0 + (on ? r : 0)) / a.G, hq = g.h * a.G + (g.r0 + (on ? r : 0)) - t * a.G;
    const T* q = reinterpret_cast<const T*>(a.q) + (g.q0 + t) * a.ldq + (long long)hq * a.dim + 4 * qc;
#pragma unroll
    for (int ks = 0; ks < DT / 16; ++ks) {
        w[ks] = make_uint2(0u, 0u);
        if (on && 16 * ks < a.dim) w[ks] = *reinterpret_cast<const uint2*>(q + 16 * ks);
    }
    float f = 1.f;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float m = 0.f;
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks)
            m = fmaxf(m, fmaxf(fmaxf(fabsf(__uint_as_float(w[ks].x << 16)), fabsf(__uint_as_float(w[ks].x & 0xffff0000u))),
                               fmaxf(fabsf(__uint_as_float(w[ks].y << 16)), fabsf(__uint_as_float(w[ks].y & 0xffff0000u)))));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        f = row_factor(m);
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) {
            w[ks].x = pack_f16(__uint_as_float(w[ks].x << 16) * f, __uint_as_float(w[ks].x & 0xffff0000u) * f);
            w[ks].y = pack_f16(__uint_as_float(w[ks].y << 16) * f, __uint_as_float(w[ks].y & 0xffff0000u) * f);
        }
    }
    return f;
}

template <int DT, int NQ, typename T>
__global__ void __launch_bounds__(TkCfg<DT, NQ>::THREADS, 1)
attn_token_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ AttnArgs a) {
    using C = TkCfg<DT, NQ>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::bar_off);
    uint64_t* empty = full + C::NS;
    float* scales = reinterpret_cast<float*>(sm + C::sc_off);
    unsigned* run_sh = reinterpret_cast<unsigned*>(sm + C::run_off);
    volatile int* join_sh = reinterpret_cast<volatile int*>(run_sh + C::THREADS / 32 + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&full[i], 1 + 32);   // the boxes' bytes, and the 32 lanes' scale copies
            mbar_init(&empty[i], 4);
        }
        fence_mbar_init();
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
    }
    pdl_wait();
    AttnRun run = attn_run<C::ROWS, AT_KT, TK_OV, C::THREADS>(a, run_sh, join_sh + 1);   // its barriers also publish the mbarriers
    AttnSeg g;

    if (warp >= C::WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::PREG));
        const int stream = warp - C::WARPS;
        // ===================== producer =====================
        const int pb = min(AT_KT, 1 << a.page_log2);   // keys per box
        int it = 0;
        bool ok = true;
        while (ok && attn_next<C::ROWS, AT_KT, TK_OV>(a, run, &g)) {
            const int32_t* row = a.table + (long long)g.b * a.table_ld;
            int have = -1, ids = -1;   // this lane's page id of pages [have, have + 32)
            const int first = attn_first_key(a, g) >> a.page_log2;   // pages before it: behind every row's window
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                if ((it & (TK_STREAMS - 1)) != stream) continue;
                const int st = it % C::NS;
                if (it >= C::NS) ok = __all_sync(0xffffffffu, wait_parity_sleep(&empty[st], (it / C::NS - 1) & 1));
                if (!ok) break;
                const int key0 = t * AT_KT, p0 = key0 >> a.page_log2;
                const int plast = min(key0 + AT_KT, g.len) - 1;          // last key of the unit that exists
                const int np = (plast >> a.page_log2) - p0 + 1;           // its pages: 1, 2 or 4
                if (have < 0 || p0 + np > have + 32) {
                    have = p0;
                    ids = p0 + lane < a.table_ld ? row[p0 + lane] : -1;
                }
                // lane i < np: piece i's page. For one that no row sees, or a page index outside the cache (which raises a
                // status bit), the boxes come from page 0, and the scales from a pair that tells the computing warps to
                // leave the keys out
                int id = __shfl_sync(0xffffffffu, ids, (p0 - have + min(lane, np - 1)) & 31);
                const bool unseen = p0 + lane < first, none = unseen || id < 0 || id >= a.pages;
                if (none) {
                    if (lane < np && !unseen) raise_status(DEV_ERR_BAD_INDEX);
                    id = 0;
                }
                uint8_t* dst = sm + st * C::STAGE;
                if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(np * pb * DT * 2));
                __syncwarp();
                if (lane < np) {
                    const long long ph = (long long)id * a.heads + g.h;
                    const int y = (int)((ph << a.page_log2) + (key0 & ((1 << a.page_log2) - 1)));
                    uint8_t* d = dst + lane * pb * C::HB;
#pragma unroll
                    for (int hf = 0; hf < DT / C::HB; ++hf) {
                        tma_load_2d(d + hf * AT_KT * 128, &tk, hf * 128, y, &full[st]);
                        tma_load_2d(d + C::TILE + hf * AT_KT * 128, &tv, hf * 128, y, &full[st]);
                    }
                    const uint32_t sd = smem_u32(scales + st * 8 + 2 * lane);
                    const float* ks = none ? tk_no_page : a.ks + ph;
                    const float* vs = none ? tk_no_page + 1 : a.vs + ph;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sd), "l"(ks) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sd + 4), "l"(vs) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
                __syncwarp();
            }
        }
        // drain: every copy of this warp has landed before it exits
        for (int i = max(0, it - C::NS); i < it; ++i)
            if ((i & (TK_STREAMS - 1)) == stream && !wait_parity_sleep(&full[i % C::NS], (i / C::NS) & 1, DEV_ERR_DRAIN_TIMEOUT)) break;
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // ===================== computing warps =====================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::CREG));
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    constexpr int KS = DT / 16, NT = 32 * C::WARPS;
    const int grp = warp >> 2, wk = (warp & 3) * 16;   // units this warp's group takes, first key of the unit it takes
    const int gr = lane >> 2, qc = lane & 3;           // fragment row (key or dimension) and column pair (query)
    auto bar = [] { named_sync(1, NT); };
    uint8_t* qs = sm + C::q_off;
    float* merge = reinterpret_cast<float*>(sm + C::merge_off);
    float2* ml = reinterpret_cast<float2*>(sm + C::ml_off);
    float* rowf = reinterpret_cast<float*>(sm + C::row_off);
    int it = 0;
    bool ok = true;
    while (attn_next<C::ROWS, AT_KT, TK_OV>(a, run, &g)) {
        // ---- q: registers of every warp, or shared memory ----
        uint2 qr[C::QREGS ? KS : 1];
        float qf[NQ][2];   // scale * log2(e) over the factor of this thread's queries 8 nq + 2 qc + {0, 1}
        if constexpr (C::QREGS) {
            const float f = tk_load_q<DT, T>(a, g, 0, lane, qr);
            qf[0][0] = __fdiv_rn(a.scale_log2, __shfl_sync(0xffffffffu, f, 8 * qc));
            qf[0][1] = __fdiv_rn(a.scale_log2, __shfl_sync(0xffffffffu, f, 8 * qc + 4));
        } else {
            if (warp < NQ) {
                uint2 w[KS];
                const float f = tk_load_q<DT, T>(a, g, warp, lane, w);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) reinterpret_cast<uint2*>(qs)[(warp * KS + ks) * 32 + lane] = w[ks];
                if (qc == 0) rowf[8 * warp + gr] = f;
            }
            bar();
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    qf[nq][e] = bf ? __fdiv_rn(a.scale_log2, rowf[8 * nq + 2 * qc + e]) : a.scale_log2;
        }
        // keys [klo, khi) that this thread's queries see
        int klo[NQ][2], khi[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * nq + 2 * qc + e, rr = min(r, g.rows - 1);
                const int p = g.pos0 + (g.r0 + rr) / a.G;
                khi[nq][e] = r < g.rows ? p + 1 : 0;
                klo[nq][e] = attn_window(a, p);
            }
        // keys that every row of the tile sees: no mask needed (rows past the tile's compute what is not written)
        const int all_hi = g.pos0 + g.r0 / a.G + 1;
        const int all_lo = attn_window(a, g.pos0 + (g.r0 + g.rows - 1) / a.G);

        float o[NQ][KS][4];   // O^T: dimension 16 j + 2 gr (and + 1: elements 2, 3), queries 2 qc, 2 qc + 1
        float M[NQ][2], l[NQ][2], V = 7.888609e-31f, vinv = 1.2676506e30f;   // 2^-100
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nq][j][e] = 0.f;
            M[nq][0] = M[nq][1] = -INFINITY;
            l[nq][0] = l[nq][1] = 0.f;
        }
        const int n = max(0, g.t1 - g.t0);
        // this group's units: it + i with (it + i) % GROUPS == grp
        for (int i = (grp - it) & (C::GROUPS - 1); i < n; i += C::GROUPS) {
            const int u = it + i, st = u % C::NS;
            if (ok) ok = __all_sync(0xffffffffu, wait_parity(&full[st], (u / C::NS) & 1));
            if (!ok) continue;   // the wait gave up (status bit): the walk goes on to the items' joins, whose barriers and counts
                                 // the other warps and blocks need (the streaming warps' waits give up too)
            const uint32_t kt = smem_u32(sm + st * C::STAGE), vt = kt + C::TILE;
            const int key0 = (g.t0 + i) * AT_KT + wk;
            const int piece = a.page_log2 >= 6 ? 0 : wk >> a.page_log2;   // one page's keys, or none that exist
            const float2 sc = *reinterpret_cast<const float2*>(scales + st * 8 + 2 * piece);
            if (key0 < g.len && sc.x != -INFINITY) {
                float s[NQ][4];
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nq][e] = 0.f;
#pragma unroll
                for (int c4 = 0; c4 < DT / 64; ++c4) {
                    uint32_t r0[4], r1[4];
                    ldsm_x4(r0, code_addr<DT>(kt, wk + (lane & 7), 4 * c4 + (lane >> 3)));
                    ldsm_x4(r1, code_addr<DT>(kt, wk + 8 + (lane & 7), 4 * c4 + (lane >> 3)));
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int ks = 4 * c4 + h;
                        const uint32_t a0 = codes_f16(r0[h], 0x4140u), a1 = codes_f16(r1[h], 0x4140u);
                        const uint32_t a2 = codes_f16(r0[h], 0x4342u), a3 = codes_f16(r1[h], 0x4342u);
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq) {
                            uint2 b;
                            if constexpr (C::QREGS) b = qr[ks];
                            else b = lds64(smem_u32(qs) + 8 * ((nq * KS + ks) * 32 + lane));
                            mma_f16(s[nq], a0, a1, a2, a3, b.x, b.y);
                        }
                    }
                }
                if (sc.y > V) {   // the reference of V's scales follows (the warp together)
                    const float f = V * __fdiv_rn(1.f, sc.y);
                    V = sc.y;
                    vinv = __fdiv_rn(1.f, V);
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int j = 0; j < KS; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nq][j][e] *= f;
                }
                const float ratio = fmaxf(sc.y * vinv, 9.313226e-10f);   // vs / V, at least 2^-30
                const float lv = __log2f(ratio), iv = __fdividef(1.f, ratio);
                const bool masked = key0 + 16 > all_hi || key0 < all_lo;
                uint32_t pk[NQ][2];   // p' of keys gr and gr + 8
                float add[NQ][2];
                auto weigh = [&] {
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq) {
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float kf = qf[nq][e] * sc.x, cg = lv - (M[nq][e] == -INFINITY ? 0.f : M[nq][e] - TK_P_BIAS);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float x = fmaf(s[nq][2 * h + e], kf, cg);
                                if (masked) {
                                    const int j = key0 + gr + 8 * h;
                                    if (j < klo[nq][e] || j >= khi[nq][e]) x = -INFINITY;
                                }
                                p[2 * h + e] = ex2(x);
                            }
                            add[nq][e] = p[e] + p[2 + e];
                        }
                        pk[nq][0] = pack_f16(p[0], p[1]);
                        pk[nq][1] = pack_f16(p[2], p[3]);
                    }
                };
                weigh();
                bool again = false;   // first keys of a row, or a p' past 2^12 (fp16 0x6c00; NaN, 0x7fff, too)
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                    const uint32_t top = h2_max(pk[nq][0], pk[nq][1]);
                    again |= (top & 0xffffu) > 0x6c00u || (top >> 16) > 0x6c00u;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        again |= M[nq][e] == -INFINITY && klo[nq][e] < key0 + 16 && khi[nq][e] > key0;
                }
                if (__any_sync(0xffffffffu, again)) {
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = -INFINITY;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int j = key0 + gr + 8 * h;
                                if (!masked || (j >= klo[nq][e] && j < khi[nq][e]))
                                    x = fmaxf(x, fmaf(s[nq][2 * h + e], qf[nq][e] * sc.x, lv));
                            }
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            const float mn = fmaxf(M[nq][e], x), al = M[nq][e] == -INFINITY ? 0.f : ex2(M[nq][e] - mn);
                            M[nq][e] = mn;
                            l[nq][e] *= al;
#pragma unroll
                            for (int j = 0; j < KS; ++j) {
                                o[nq][j][e] *= al;
                                o[nq][j][2 + e] *= al;
                            }
                        }
                    weigh();
                }
                uint32_t b[NQ][2];   // p'^T: keys as k, queries as columns
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                    l[nq][0] = fmaf(add[nq][0], iv, l[nq][0]);
                    l[nq][1] = fmaf(add[nq][1], iv, l[nq][1]);
                    b[nq][0] = movm(pk[nq][0]);
                    b[nq][1] = movm(pk[nq][1]);
                }
#pragma unroll
                for (int j2 = 0; j2 < DT / 32; ++j2) {
                    uint32_t r[4];
                    ldsm_x4_t(r, code_addr<DT>(vt, wk + 8 * ((lane >> 3) & 1) + (lane & 7), 2 * j2 + (lane >> 4)));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t a0 = codes_f16(r[2 * h], 0x4240u), a1 = codes_f16(r[2 * h], 0x4341u);
                        const uint32_t a2 = codes_f16(r[2 * h + 1], 0x4240u), a3 = codes_f16(r[2 * h + 1], 0x4341u);
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq) mma_f16(o[nq][2 * j2 + h], a0, a1, a2, a3, b[nq][0], b[nq][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        it += n;
        // ---- join the warps: O of a row = sum_w V_w O_w 2^(M_w - M), l likewise ----
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], d);
                if (gr == 0) ml[warp * C::ROWS + 8 * nq + 2 * qc + e] = make_float2(M[nq][e], l[nq][e]);
            }
        bar();
        const bool direct = g.whole;
        constexpr int PITCH = DT + 2;
        float* part = a.part + attn_slot(g, blockIdx.x) * C::ROWS * PITCH;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            float fac[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * nq + 2 * qc + e;
                // the eight lanes of a column pair take the warps' values between them
                const float2 v0 = ml[gr * C::ROWS + r];
                const float2 v1 = C::WARPS == 16 ? ml[((gr + 8) & (C::WARPS - 1)) * C::ROWS + r] : make_float2(-INFINITY, 0.f);
                float mm = fmaxf(v0.x, v1.x);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
                const float mu = mm == -INFINITY ? 0.f : mm;   // a warp that saw no key: 0
                float lsum = fmaf(v0.y, ex2(v0.x - mu), v1.y * ex2(v1.x - mu));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, d);
                fac[e] = M[nq][e] > -INFINITY ? ex2(M[nq][e] - mm) * V : 0.f;
                if (direct) fac[e] = lsum == 0.f ? 0.f : __fdiv_rn(fac[e], lsum);
                if (!direct && warp == 0 && gr == 0 && r < g.rows)
                    *reinterpret_cast<float2*>(part + C::ROWS * DT + 2 * r) = make_float2(mm, lsum);
            }
#pragma unroll
            for (int c = 0; c < DT / 64; ++c) {
                if (64 * c >= a.dim) break;
                // 64 columns, [warp][query][column]
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2*>(merge + (warp * 8 + 2 * qc + e) * 64 + 16 * jj + 2 * gr) =
                            make_float2(o[nq][4 * c + jj][e] * fac[e], o[nq][4 * c + jj][2 + e] * fac[e]);
                bar();
                // two columns of a row per thread of the first 256
                if (threadIdx.x < 256) {
                    const int r8 = threadIdx.x >> 5, d = 2 * (threadIdx.x & 31), r = 8 * nq + r8;
                    float2 v = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < C::WARPS; ++w) {
                        const float2 x = *reinterpret_cast<const float2*>(merge + (w * 8 + r8) * 64 + d);
                        v.x += x.x;
                        v.y += x.y;
                    }
                    if (r < g.rows && 64 * c + d < a.dim) {
                        if (direct) {
                            T* out = attn_out<T>(a, g, r) + 64 * c + d;
                            *reinterpret_cast<uint32_t*>(out) = bf ? pack_bf16(v.x, v.y) : pack_f16(v.x, v.y);
                        } else {
                            *reinterpret_cast<float2*>(part + ((16 * c + (d >> 2)) * C::ROWS + r) * 4 + (d & 3)) = v;
                        }
                    }
                }
                bar();
            }
        }
        if (!direct) attn_join<DT, C::ROWS, T>(a, g, threadIdx.x, NT, join_sh, bar);
    }
}

}  // namespace vkb
