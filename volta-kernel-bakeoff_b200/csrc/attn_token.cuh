// Attention for few query rows per kv head (single tokens, drafted tokens): HBM-bound, the codes are read once and
// everything else hides behind that stream.
//
//   s_rj = (q_r . c_j) ks_j scale, p_rj = exp(s_rj - m_r), o_r = sum_j p_rj vs_j c'_j / sum_j p_rj
//
// with codes c, c' and one scale per page for K (ks) and V (vs). One persistent block per SM (its run of units:
// attn_common.cuh), three warpgroups. Warp 8 streams: per unit of 64 keys, one TMA box of codes per page piece and 128-byte
// half for K and for V (128-byte swizzle), and the pages' scales with 4-byte asynchronous copies, into a ring of NS
// stages. Warps 0-3 compute the even units, warps 4-7 the odd ones, 16 keys per warp, each warp with its own running
// maximum and sum, joined once per segment. Products are mma.sync.m16n8k16 on fp16: the codes enter exactly (1024 + u as
// fp16, minus 1152), K through ldmatrix and V through transposing ldmatrix on byte pairs, so a register of four codes
// is one operand register pair either way; the scales are applied in fp32 (K) and folded into p before its one
// rounding to fp16 (V). tcgen05 has nothing to add here: with 16 rows the tensor work is an eighth of the time.
// p carries a factor 2^8 and the running maximum follows the true one lazily (by up to 2^4), so small p keep their
// fp16 precision: the smallest normal p is 2^-22 of the largest.
// q: fp16 as it is; bf16 rows are scaled by a power of two into fp16's range first (exact but for values 2^-28 below the
// row's largest).
#pragma once

#include "attn_common.cuh"

namespace vkb {

constexpr int AT_KT = 64;                            // keys per unit
constexpr int TK_WARPS = 8;                          // computing warps (two groups of four)
constexpr int TK_THREADS = 32 * (TK_WARPS + 4);      // and a warpgroup whose first warp streams
constexpr float TK_P_BIAS = 8.f;                     // p is kept times 2^8
constexpr float TK_LAZY = 4.f;                       // the reference maximum may lag the true one by 2^4

// DT: head dimension rounded up to 64, 128 or 256. MT: 16-row tiles per item.
template <int DT, int MT> struct TkCfg {
    static constexpr int ROWS = 16 * MT;
    static constexpr int HB = DT < 128 ? DT : 128;            // bytes of a box row
    static constexpr int TILE = AT_KT * DT;                   // bytes of one tensor's codes in a stage
    static constexpr int STAGE = 2 * TILE;
    static constexpr int NS = DT == 64 ? 12 : DT == 128 ? 8 : 5;
    static constexpr int Q = ROWS * DT * 2;                   // q in A-fragment order
    static constexpr int MERGE = TK_WARPS * 16 * 32 * 4;      // 32 columns of 16 rows of every warp
    // offsets from the 1024-aligned base
    static constexpr int q_off = NS * STAGE;
    static constexpr int merge_off = q_off + Q;
    static constexpr int ml_off = merge_off + MERGE;          // [warp][ROWS] {m, l}
    static constexpr int row_off = ml_off + TK_WARPS * ROWS * 8;   // [ROWS] factor of q
    static constexpr int sc_off = row_off + ROWS * 4;         // [NS][4 pieces]{k, v} scales
    static constexpr int bar_off = (sc_off + NS * 32 + 15) / 16 * 16;
    static constexpr int run_off = bar_off + 16 * NS;
    static constexpr int BYTES = run_off + 8 * (TK_THREADS / 32 + 2) + 16 + 1024;
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
// Bytes (i, j) of v (codes + 128) as the exact fp16 pair of codes: 0x6400 | u is 1024 + u, minus 1152.
__device__ __forceinline__ uint32_t codes_f16(uint32_t v, uint32_t sel) {
    return h2_sub(prmt(v, 0x64646464u, sel), 0x64806480u);
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Shared address of 16-byte chunk c of key row r of a stage's tile of codes (the TMA swizzles: 128-byte rows XOR the row's
// low three bits into the chunk, 64-byte rows bits 1-2 of the row).
template <int DT> __device__ __forceinline__ uint32_t code_addr(uint32_t tile, int r, int c) {
    if constexpr (DT == 64) return tile + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    else return tile + (c >> 3) * (AT_KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

template <int DT, int MT, typename T>
__global__ void __launch_bounds__(TK_THREADS, 1)
attn_token_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ AttnArgs a) {
    using C = TkCfg<DT, MT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::bar_off);
    uint64_t* empty = full + C::NS;
    float* scales = reinterpret_cast<float*>(sm + C::sc_off);
    long long* run_sh = reinterpret_cast<long long*>(sm + C::run_off);
    volatile int* join_sh = reinterpret_cast<volatile int*>(run_sh + TK_THREADS / 32 + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&full[i], 1 + 32);   // the boxes' bytes, and the 32 lanes' scale copies
            mbar_init(&empty[i], TK_WARPS / 2);
        }
        fence_mbar_init();
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
    }
    pdl_wait();
    AttnRun run = attn_run<C::ROWS, AT_KT, TK_THREADS>(a, run_sh);   // its barriers also publish the mbarriers
    AttnSeg g;

    // Registers: 384 threads are launched with 168 each (64512); the streaming warpgroup keeps 40, so that the computing
    // ones have 232 (128 x 40 + 256 x 232 = 64512).
    if (warp >= TK_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp > TK_WARPS) return;
        // ===================== producer =====================
        const int pb = min(AT_KT, 1 << a.page_log2);   // keys per box
        int it = 0;
        bool ok = true;
        while (ok && attn_next<C::ROWS, AT_KT>(a, run, &g)) {
            const int32_t* row = a.table + (long long)g.b * a.table_ld;
            int have = -1, ids = -1;   // this lane's page id of pages [have, have + 32)
            for (int t = g.t0; t < g.t1; ++t, ++it) {
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
                // lane i < np: piece i's page; a page index outside the cache reads page 0 and raises a status bit
                int id = __shfl_sync(0xffffffffu, ids, (p0 - have + min(lane, np - 1)) & 31);
                if (id < 0 || id >= a.pages) {
                    if (lane < np) raise_status(DEV_ERR_BAD_INDEX);
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
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sd), "l"(a.ks + ph) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sd + 4), "l"(a.vs + ph) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
                __syncwarp();
            }
        }
        // drain: every copy has landed before the block exits
        for (int i = max(0, it - C::NS); i < it; ++i)
            if (!wait_parity_sleep(&full[i % C::NS], (i / C::NS) & 1, DEV_ERR_DRAIN_TIMEOUT)) break;
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // ===================== computing warps =====================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int grp = warp >> 2, wk = (warp & 3) * 16;   // unit parity, first key of the unit that this warp takes
    const int gr = lane >> 2, qc = lane & 3;           // fragment row and quad column
    auto bar = [] { named_sync(1, 32 * TK_WARPS); };
    uint8_t* qs = sm + C::q_off;
    float* merge = reinterpret_cast<float*>(sm + C::merge_off);
    float2* ml = reinterpret_cast<float2*>(sm + C::ml_off);
    float* rowf = reinterpret_cast<float*>(sm + C::row_off);
    int it = 0;
    bool ok = true;
    while (attn_next<C::ROWS, AT_KT>(a, run, &g)) {
        // ---- q of the tile, in A-fragment order: {a0, a1, a2, a3} of k step ks, row tile mt at [mt][ks][lane]. The k
        // order of a step of 16 is that of the codes' registers: slots 2c, 2c + 1, 2c + 8, 2c + 9 hold 4c .. 4c + 3.
        {
            const int nt = 32 * TK_WARPS, tid = threadIdx.x;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                // a power of two that brings the row's largest magnitude into [2^13, 2^14)
                for (int r = tid >> 4; r < C::ROWS; r += nt >> 4) {
                    float m = 0.f;
                    if (r < g.rows) {
                        const int t = (g.r0 + r) / a.G, hq = g.h * a.G + (g.r0 + r) - t * a.G;
                        const T* q = reinterpret_cast<const T*>(a.q) + (g.q0 + t) * a.ldq + (long long)hq * a.dim;
                        for (int d = 2 * (tid & 15); d < a.dim; d += 32) {
                            const uint32_t w = *reinterpret_cast<const uint32_t*>(q + d);
                            m = fmaxf(m, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
                        }
                    }
#pragma unroll
                    for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    if ((tid & 15) == 0) {
                        const int e = (int)(__float_as_uint(m) >> 23) - 127;             // floor(log2 m); 0 or tiny: -127
                        rowf[r] = m == 0.f ? 1.f : exp2f((float)min(126, max(-126, 13 - e)));
                    }
                }
                bar();
            }
            constexpr int KS = DT / 16;
            for (int i = tid; i < MT * KS * 32; i += nt) {
                const int l = i & 31, ks = (i >> 5) % KS, mt = (i >> 5) / KS, d = 16 * ks + 4 * (l & 3);
                uint2 w[2];
#pragma unroll
                for (int hl = 0; hl < 2; ++hl) {
                    const int r = 16 * mt + (l >> 2) + 8 * hl;
                    w[hl] = make_uint2(0u, 0u);
                    if (r < g.rows && d < a.dim) {
                        const int t = (g.r0 + r) / a.G, hq = g.h * a.G + (g.r0 + r) - t * a.G;
                        const T* q = reinterpret_cast<const T*>(a.q) + (g.q0 + t) * a.ldq + (long long)hq * a.dim + d;
                        w[hl] = *reinterpret_cast<const uint2*>(q);
                        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                            const float f = rowf[r];
                            w[hl].x = pack_f16(__uint_as_float(w[hl].x << 16) * f, __uint_as_float(w[hl].x & 0xffff0000u) * f);
                            w[hl].y = pack_f16(__uint_as_float(w[hl].y << 16) * f, __uint_as_float(w[hl].y & 0xffff0000u) * f);
                        }
                    }
                }
                *reinterpret_cast<uint4*>(qs + 16 * i) = make_uint4(w[0].x, w[1].x, w[0].y, w[1].y);
            }
            bar();
        }
        // rows of this thread: 16 mt + gr + 8 hl; keys [klo, khi) that each sees
        int klo[MT][2], khi[MT][2];
        float qf[MT][2];   // scale * log2(e), and the inverse of the row's factor
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
                const int r = 16 * mt + gr + 8 * hl, rr = min(r, g.rows - 1);
                const int p = g.pos0 + (g.r0 + rr) / a.G;
                khi[mt][hl] = r < g.rows ? p + 1 : 0;
                klo[mt][hl] = a.window > 0 ? p - a.window + 1 : 0;
                qf[mt][hl] = a.scale_log2;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) qf[mt][hl] = __fdiv_rn(a.scale_log2, rowf[rr]);
            }
        // keys that every row of the tile sees: no mask needed
        const int all_hi = g.pos0 + g.r0 / a.G + 1;
        const int all_lo = a.window > 0 ? g.pos0 + (g.r0 + g.rows - 1) / a.G - a.window + 1 : 0;

        float o[MT][DT / 8][4], m[MT][2], l[MT][2], cref = 0.f;   // o of 16 columns j: even columns [2j], odd [2j + 1]
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int j = 0; j < DT / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
        }
        for (int t = g.t0; t < g.t1; ++t, ++it) {
            if ((it & 1) != grp) continue;
            const int st = it % C::NS;
            if (ok) ok = __all_sync(0xffffffffu, wait_parity(&full[st], (it / C::NS) & 1));
            if (!ok) continue;   // the wait gave up (status bit): the walk goes on so that every arrival is made
            const uint32_t kt = smem_u32(sm + st * C::STAGE), vt = kt + C::TILE;
            const int key0 = t * AT_KT + wk;
            const int piece = a.page_log2 >= 6 ? 0 : wk >> a.page_log2;
            if (key0 < g.len) {
                const float ks = scales[st * 8 + 2 * piece], vs = scales[st * 8 + 2 * piece + 1];
                float s[MT][2][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
                for (int c4 = 0; c4 < DT / 64; ++c4) {
                    uint32_t r0[4], r1[4];
                    ldsm_x4(r0, code_addr<DT>(kt, wk + (lane & 7), 4 * c4 + (lane >> 3)));
                    ldsm_x4(r1, code_addr<DT>(kt, wk + 8 + (lane & 7), 4 * c4 + (lane >> 3)));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t b0 = codes_f16(r0[i], 0x4140u), b1 = codes_f16(r0[i], 0x4342u);
                        const uint32_t b2 = codes_f16(r1[i], 0x4140u), b3 = codes_f16(r1[i], 0x4342u);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const uint4 qa = lds128(smem_u32(qs) + 16 * ((mt * (DT / 16) + 4 * c4 + i) * 32 + lane));
                            mma_16816(s[mt][0], qa.x, qa.y, qa.z, qa.w, b0, b1);
                            mma_16816(s[mt][1], qa.x, qa.y, qa.z, qa.w, b2, b3);
                        }
                    }
                }
                // ---- scores in the log2 domain, masks, running maximum ----
                const bool masked = key0 + 16 > all_hi || key0 < all_lo;
                bool grow = false;
                float top[MT][2];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int hl = 0; hl < 2; ++hl) {
                        const float f = qf[mt][hl] * ks;
                        float x = -INFINITY;
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float v = s[mt][nt][2 * hl + e] * f;
                                if (masked) {
                                    const int j = key0 + 8 * nt + 2 * qc + e;
                                    if (j < klo[mt][hl] || j >= khi[mt][hl]) v = -INFINITY;
                                }
                                s[mt][nt][2 * hl + e] = v;
                                x = fmaxf(x, v);
                            }
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                        top[mt][hl] = x;
                        grow |= x > m[mt][hl] + TK_LAZY || (x > -INFINITY && m[mt][hl] == -INFINITY);
                    }
                const bool cgrow = vs > cref;
                if (__any_sync(0xffffffffu, grow) || cgrow) {
                    const float cf = cgrow ? (cref > 0.f ? __fdiv_rn(cref, vs) : 0.f) : 1.f;
                    if (cgrow) cref = vs;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {
                            const float mn = fmaxf(m[mt][hl], top[mt][hl]);
                            const float al = m[mt][hl] == -INFINITY ? 0.f : ex2(m[mt][hl] - mn);
                            m[mt][hl] = mn;
                            l[mt][hl] *= al;
                            const float af = al * cf;
#pragma unroll
                            for (int j = 0; j < DT / 8; ++j) {
                                o[mt][j][2 * hl] *= af;
                                o[mt][j][2 * hl + 1] *= af;
                            }
                        }
                }
                const float vf = cref > 0.f ? __fdiv_rn(vs, cref) : 0.f;   // <= 1
                uint32_t pa[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int hl = 0; hl < 2; ++hl) {
                        const float mr = m[mt][hl] == -INFINITY ? 0.f : m[mt][hl] - TK_P_BIAS;
                        float p[4];
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                p[2 * nt + e] = ex2(s[mt][nt][2 * hl + e] - mr);
                                l[mt][hl] += p[2 * nt + e];
                            }
                        pa[mt][hl] = pack_f16(p[0] * vf, p[1] * vf);
                        pa[mt][2 + hl] = pack_f16(p[2] * vf, p[3] * vf);
                    }
                // ---- o += p c' ----
#pragma unroll
                for (int j2 = 0; j2 < DT / 32; ++j2) {
                    uint32_t r[4];
                    ldsm_x4_t(r, code_addr<DT>(vt, wk + 8 * ((lane >> 3) & 1) + (lane & 7), 2 * j2 + (lane >> 4)));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t e0 = codes_f16(r[2 * h], 0x4240u), e1 = codes_f16(r[2 * h + 1], 0x4240u);
                        const uint32_t d0 = codes_f16(r[2 * h], 0x4341u), d1 = codes_f16(r[2 * h + 1], 0x4341u);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma_16816(o[mt][2 * (2 * j2 + h)], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], e0, e1);
                            mma_16816(o[mt][2 * (2 * j2 + h) + 1], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], d0, d1);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        // ---- join the warps: o of row r = sum_w o_w c_w 2^(m_w - M), l likewise ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
                l[mt][hl] += __shfl_xor_sync(0xffffffffu, l[mt][hl], 1);
                l[mt][hl] += __shfl_xor_sync(0xffffffffu, l[mt][hl], 2);
                if (qc == 0) ml[warp * C::ROWS + 16 * mt + gr + 8 * hl] = make_float2(m[mt][hl], l[mt][hl]);
            }
        bar();
        const bool direct = g.whole;
        constexpr int PITCH = DT + 2;
        float* part = a.part + attn_slot(run, g, blockIdx.x) * C::ROWS * PITCH;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float mm[2], lsum[2], fac[2];
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
                const int r = 16 * mt + gr + 8 * hl;
                mm[hl] = -INFINITY;
#pragma unroll
                for (int w = 0; w < TK_WARPS; ++w) mm[hl] = fmaxf(mm[hl], ml[w * C::ROWS + r].x);
                lsum[hl] = 0.f;
#pragma unroll
                for (int w = 0; w < TK_WARPS; ++w) {
                    const float2 v = ml[w * C::ROWS + r];
                    if (v.x > -INFINITY) lsum[hl] = fmaf(v.y, ex2(v.x - mm[hl]), lsum[hl]);
                }
                fac[hl] = m[mt][hl] > -INFINITY ? ex2(m[mt][hl] - mm[hl]) * cref : 0.f;
                if (direct) fac[hl] = lsum[hl] == 0.f ? 0.f : __fdiv_rn(fac[hl], lsum[hl]);
                if (!direct && warp == 0 && qc == 0 && r < g.rows)
                    *reinterpret_cast<float2*>(part + C::ROWS * DT + 2 * r) = make_float2(mm[hl], lsum[hl]);
            }
#pragma unroll
            for (int c = 0; c < DT / 32; ++c) {
                if (32 * c >= a.dim) break;
                // 32 columns: two groups of 16, of which this thread holds 4 qc .. 4 qc + 3
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int hl = 0; hl < 2; ++hl) {
                        const float* e = o[mt][2 * (2 * c + jj)];
                        const float* d = o[mt][2 * (2 * c + jj) + 1];
                        float* x = merge + (warp * 16 + gr + 8 * hl) * 32 + 16 * jj + 4 * qc;
                        *reinterpret_cast<float4*>(x) = make_float4(e[2 * hl] * fac[hl], d[2 * hl] * fac[hl],
                                                                    e[2 * hl + 1] * fac[hl], d[2 * hl + 1] * fac[hl]);
                    }
                bar();
                {
                    const int r16 = threadIdx.x >> 4, d = 2 * (threadIdx.x & 15), r = 16 * mt + r16;
                    float2 v = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < TK_WARPS; ++w) {
                        const float2 x = *reinterpret_cast<const float2*>(merge + (w * 16 + r16) * 32 + d);
                        v.x += x.x;
                        v.y += x.y;
                    }
                    if (r < g.rows && 32 * c + d < a.dim) {
                        if (direct) {
                            T* out = attn_out<T>(a, g, r) + 32 * c + d;
                            *reinterpret_cast<uint32_t*>(out) =
                                std::is_same<T, __half>::value ? pack_f16(v.x, v.y) : pack_bf16(v.x, v.y);
                        } else {
                            *reinterpret_cast<float2*>(part + ((8 * c + (d >> 2)) * C::ROWS + r) * 4 + (d & 3)) = v;
                        }
                    }
                }
                bar();
            }
        }
        if (!direct) attn_join<DT, C::ROWS, T>(a, run, g, threadIdx.x, 32 * TK_WARPS, join_sh, bar);
    }
}

}  // namespace vkb
