// Attention for many query rows per kv head (prompts and prompt chunks), on the 5th-generation tensor cores.
//
// An item is a tile of NT x 128 query rows; per 128 keys S = Q K'^T and O += P V' are tcgen05.mma with fp32
// accumulators in tensor memory, K' and V' the codes as exact fp16 integers in shared memory, converted once for all
// rows of the tile. The scales never touch the codes: with x_j = s_j ks_j scale log2(e) + log2(vs_j / vs0),
//   p'_j = 2^(x_j - M + 8),   O' = sum_j p'_j c'_j,   l = sum_j p'_j (vs0 / vs_j),   o = vs0 O' / l,
// so a group of 16 keys (a page or part of one) costs one multiply-add per score and one multiply per group. p' is
// rounded once, to fp16, for the product; l sums it in fp32. M follows the running maximum of x lazily (by up to 2^4), so
// O' is rescaled only when a row's maximum grows by more. vs0: the largest V scale of the segment's first keys; scales
// below 2^-30 of the largest seen so far count as that.
//
// 16 warps, one block per SM (its run of units: attn_common.cuh):
//   warp 0        issues the MMAs. With two row tiles (NT = 2, dimensions up to 128): S_t(j + 1) goes out as soon as
//                 O_t += P_t(j) V(j) has read P_t(j), which lies in S_t's columns, while the other tile's rows are in
//                 their softmax. With one (NT = 1, dimension 256, where O takes half of tensor memory) S has two buffers.
//   warps 4-7     softmax of row tile 0, a row per thread (tensor memory lanes are rows): S is read twice (maximum, then
//                 exponentials), P goes back as fp16
//   warps 8-11    softmax of row tile 1 (NT = 2); convert codes (NT = 1)
//   warps 12-15   convert codes: global loads of 16 codes, a tile ahead in registers, to 128-byte swizzled fp16 tiles
//                 (K: K-major B operand; V: the same bytes are the MN-major B operand of P V)
// Bound by the exponentials (128 x 128 per row tile and key tile; 16 per clock and SM), which take twice the time of the
// MMAs at dimension 128.
#pragma once

#include "attn_common.cuh"
#include "tcgen05.cuh"

namespace vkb {

constexpr int PR_KT = 128;               // keys per unit
constexpr int PR_THREADS = 512;
constexpr float PR_BIAS = 8.f;           // p' carries 2^8
constexpr float PR_LAZY = 4.f;           // M may lag the true maximum by 2^4
constexpr int PR_SCT = 4;                // tiles of scale tables

template <int DT> struct PrCfg {
    static constexpr int NT = DT == 256 ? 1 : 2;
    static constexpr int ROWS = 128 * NT;
    static constexpr int NS = DT == 256 ? 1 : 2;                  // converted tiles of K and of V
    static constexpr int ND = NT == 1 ? 256 : 128;                // converting threads
    static constexpr int TILE = 128 * DT * 2;                     // bytes of a converted tile and of a row tile of q
    static constexpr int HALF = 128 * 128;                        // bytes of its 64-column pieces
    static constexpr int q_off = 0;
    static constexpr int k_off = NT * TILE;
    static constexpr int v_off = k_off + NS * TILE;
    static constexpr int sc_off = v_off + NS * TILE;              // [PR_SCT][8] {kf, lv, iv, vs0}
    static constexpr int row_off = sc_off + PR_SCT * 8 * 16;      // [ROWS] factor of q
    static constexpr int bar_off = row_off + ROWS * 4;
    static constexpr int NBAR = 1 + 4 * NS + 2 + 2 + 2 + PR_SCT;
    static constexpr int run_off = bar_off + NBAR * 8;
    static constexpr int BYTES = run_off + 8 * (PR_THREADS / 32 + 2) + 32 + 1024;
    static constexpr int o_col = 256;                             // O of row tile t at o_col + t DT; S at 0 and 128
};

// MN-major, 128B-swizzled operand of 16 k: rows of 64 elements (128 bytes), 8 rows to an atom, atoms 1024 bytes apart
// along k (stride byte offset), 64-element pieces HALF apart (leading byte offset).
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t saddr, uint32_t lbo) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

__device__ __forceinline__ float ex2_ftz(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Pairs of floats (one register pair, one instruction per operation).
__device__ __forceinline__ uint64_t f2_make(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// Maximum of x = s kf + lv over 32 scores (two groups of 16 keys, the first at key k0); MASK: keys outside [klo, khi) out.
template <bool MASK>
__device__ __forceinline__ float pr_max(const uint32_t (&s)[32], const float4* sc, float qinv, int k0, int klo, int khi,
                                        float mx) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __uint_as_float(s[16 * h + e + i]);
                if (MASK && (k0 + 16 * h + e + i < klo || k0 + 16 * h + e + i >= khi)) v[i] = -INFINITY;
            }
            m0 = fmaxf(fmaxf(m0, v[0]), v[1]);
            m1 = fmaxf(fmaxf(m1, v[2]), v[3]);
        }
        const float m = fmaxf(m0, m1);
        const float4 f = sc[h];
        if (!MASK || m > -INFINITY) mx = fmaxf(mx, fmaf(m, f.x * qinv, f.y));
    }
    return mx;
}
// p' of 32 scores as fp16 pairs, and their sum into l (two running halves).
template <bool MASK>
__device__ __forceinline__ void pr_exp(const uint32_t (&s)[32], uint32_t (&pk)[16], const float4* sc, float qinv, float mb,
                                       int k0, int klo, int khi, uint64_t& l) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 f = sc[h];
        const float kf = f.x * qinv, cg = f.y - mb;
        const uint64_t kf2 = f2_make(kf, kf), cg2 = f2_make(cg, cg);
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            float2 x = f2_get(f2_fma(f2_make(__uint_as_float(s[16 * h + e]), __uint_as_float(s[16 * h + e + 1])), kf2, cg2));
            if (MASK) {
                const int k = k0 + 16 * h + e;
                if (k < klo || k >= khi) x.x = -INFINITY;
                if (k + 1 < klo || k + 1 >= khi) x.y = -INFINITY;
            }
            x.x = ex2_ftz(x.x);
            x.y = ex2_ftz(x.y);
            const uint64_t p = f2_make(x.x, x.y);
            sum = e == 0 ? p : f2_add(sum, p);
            pk[8 * h + e / 2] = pack_f16(x.x, x.y);
        }
        l = f2_fma(sum, f2_make(f.z, f.z), l);
    }
}

// 32 lanes x 16 consecutive columns from registers (no wait: tmem_wait_st).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int DT, typename T>
__global__ void __launch_bounds__(PR_THREADS, 1) attn_prompt_kernel(const __grid_constant__ AttnArgs a,
                                                                    const uint8_t* __restrict__ kc,
                                                                    const uint8_t* __restrict__ vc) {
    using C = PrCfg<DT>;
    constexpr int NT = C::NT, NS = C::NS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float4* sct = reinterpret_cast<float4*>(sm + C::sc_off);
    float* rowf = reinterpret_cast<float*>(sm + C::row_off);
    uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + C::bar_off);   // q of the item written (NT * 4 warps)
    uint64_t* k_full = q_full + 1;        // [NS] K' tile and its scale table written (ND / 32 warps)
    uint64_t* k_empty = k_full + NS;      // [NS] the MMAs that read it done
    uint64_t* v_full = k_empty + NS;
    uint64_t* v_empty = v_full + NS;
    uint64_t* s_full = v_empty + NS;      // [2] S buffer written
    uint64_t* p_full = s_full + 2;        // [2] P written to the buffer (4 warps)
    uint64_t* o_full = p_full + 2;        // [2] O of row tile t updated
    uint64_t* sc_full = o_full + 2;       // [PR_SCT] scale table written. Its slot is free again: it is written for tile
                                          // J + PR_SCT only after the products of a tile whose P the softmax of J + 1 precedes
    long long* run_sh = reinterpret_cast<long long*>(sm + C::run_off);
    volatile int* join_sh = reinterpret_cast<volatile int*>(run_sh + PR_THREADS / 32 + 2);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(run_sh + PR_THREADS / 32 + 2) + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(q_full, NT * 4);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_full[i], C::ND / 32);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], C::ND / 32);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < PR_SCT; ++i) mbar_init(&sc_full[i], 1);
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc<1>(tmem_slot, 512);
    tc_fence_before();
    pdl_wait();
    AttnRun run = attn_run<C::ROWS, PR_KT, PR_THREADS>(a, run_sh);   // its barriers publish the above
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    AttnSeg g;
    bool ok = true;
    int jj = 0;          // key tiles so far, over all items of the run

    if (warp == 0) {
        // ===================== MMA issuer =====================
        const uint32_t id_s = umma_idesc_f16(PR_KT), id_o = umma_idesc_f16(DT) | (1u << 16);   // V': MN-major B
        const uint32_t sq = smem_u32(sm + C::q_off), sk = smem_u32(sm + C::k_off), sv = smem_u32(sm + C::v_off);
        int qn = 0;
        auto wait = [&](uint64_t* bar, int phase) {
            if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(bar, phase & 1));
        };
        // S of row tile t for tile j, after the O update of tile `prev`, which read the buffer's last P (the newest or the
        // one before the newest update: a barrier's phase can be waited for only until the next one completes)
        auto qk = [&](int t, int j, int prev) {
            const int buf = NT == 2 ? t : j & 1;
            if (prev >= 0) wait(&o_full[t], prev);
            if (t == 0) wait(&k_full[j % NS], j / NS);
            if (!ok) return;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < DT / 16; ++kk) {
                    const uint32_t o = (kk >> 2) * C::HALF + (kk & 3) * 32;
                    umma_f16(tmem + buf * 128, umma_desc_sw128(sq + t * C::TILE + o),
                             umma_desc_sw128(sk + (j % NS) * C::TILE + o), id_s, kk != 0);
                }
                umma_commit(&s_full[buf]);
                if (t == NT - 1) umma_commit(&k_empty[j % NS]);
            }
            __syncwarp();
        };
        while (ok && attn_next<C::ROWS, PR_KT>(a, run, &g)) {
            const int n = g.t1 - g.t0;
            if (n <= 0) continue;
            wait(q_full, qn++);
            for (int t = 0; t < NT; ++t) qk(t, jj, jj - 1);   // the last item's updates are done
            for (int j = 0; j < n && ok; ++j) {
                const int J = jj + j;
                if (NT == 1 && j + 1 < n) qk(0, J + 1, J - 1);
                for (int t = 0; t < NT && ok; ++t) {
                    const int buf = NT == 2 ? t : J & 1;
                    wait(&p_full[buf], NT == 2 ? J : J >> 1);
                    if (t == 0) wait(&v_full[J % NS], J / NS);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < PR_KT / 16; ++kk)
                            umma_f16_ts(tmem + C::o_col + t * DT, tmem + buf * 128 + kk * 8,
                                        umma_desc_sw128_mn(sv + (J % NS) * C::TILE + kk * 2048, C::HALF), id_o,
                                        (j | kk) != 0);
                        umma_commit(&o_full[t]);
                        if (t == NT - 1) umma_commit(&v_empty[J % NS]);
                    }
                    __syncwarp();
                    if (NT == 2 && j + 1 < n) qk(t, J + 1, J);
                }
            }
            jj += n;
        }
    } else if (warp >= 16 - C::ND / 32) {
        // ===================== convert codes =====================
        constexpr int CPR = DT / 16, EACH = PR_KT * CPR / C::ND;   // 16-code chunks per row; per thread and tile
        constexpr int BATCH = 8;
        static_assert(EACH % BATCH == 0 || EACH < BATCH, "whole batches");
        constexpr int NB = EACH < BATCH ? EACH : BATCH;
        const int dtid = threadIdx.x - (PR_THREADS - C::ND), pl = a.page_log2, pmask = (1 << pl) - 1;
        while (ok && attn_next<C::ROWS, PR_KT>(a, run, &g)) {
            const int n = g.t1 - g.t0;
            const int32_t* row = a.table + (long long)g.b * a.table_ld;
            float vs0 = 0.f, cmax = 0.f;   // reference and largest V scale of the segment
            for (int j = 0; j < n && ok; ++j) {
                const int J = jj + j, key0 = (g.t0 + j) * PR_KT;
                // lane i (mod 8): the page of keys 16 i .. 16 i + 15 of the tile, -1 where there is none
                const int gkey = key0 + 16 * (lane & 7);
                int id = -1;
                if (gkey < g.len) {
                    id = row[gkey >> pl];
                    if (id < 0 || id >= a.pages) {
                        raise_status(DEV_ERR_BAD_INDEX);
                        id = -1;
                    }
                }
                const long long ph = (long long)id * a.heads + g.h;
                float ks = 0.f, vs = 0.f;
                if (dtid < 32 && id >= 0) {
                    ks = a.ks[ph];
                    vs = a.vs[ph];
                }
                // codes of chunk e of this thread, 0 values where the key or the column does not exist
                auto load = [&](const uint8_t* codes, int e) {
                    const int x = dtid + e * C::ND, r = x / CPR, c = x % CPR;
                    const long long p = __shfl_sync(0xffffffffu, ph, r >> 4);
                    const int key = key0 + r;
                    uint4 v = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    if (p >= 0 && key < g.len && 16 * c < a.dim)
                        v = __ldg(reinterpret_cast<const uint4*>(codes + ((p << pl) + (key & pmask)) * a.dim + 16 * c));
                    return v;
                };
                auto store = [&](uint8_t* tile, int e, uint4 v) {
                    const int x = dtid + e * C::ND, r = x / CPR, c = x % CPR;
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t o[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[2 * i] = h2_sub(prmt(w[i], 0x64646464u, 0x4140u), 0x64806480u);
                        o[2 * i + 1] = h2_sub(prmt(w[i], 0x64646464u, 0x4342u), 0x64806480u);
                    }
                    // the two 16-byte chunks 2c, 2c + 1 of the row; lanes of the second 64 columns start with the other
                    // one, so that a row's lanes hit different banks
                    const uint32_t base = smem_u32(tile) + (c >> 2) * C::HALF + r * 128;
                    const int c0 = (2 * c) & 7, sw = r & 7, odd = (c >> 2) & 1;
                    const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
                    sts128(base + (((c0 + odd) ^ sw) << 4), odd ? hi : lo);
                    sts128(base + (((c0 + 1 - odd) ^ sw) << 4), odd ? lo : hi);
                };
                uint4 kr[NB], vr[NB];
#pragma unroll
                for (int e = 0; e < NB; ++e) kr[e] = load(kc, e);
                const int st = J % NS;
                if (J >= NS) ok = __all_sync(0xffffffffu, wait_parity_sleep(&k_empty[st], (J / NS - 1) & 1));
                uint8_t* kt = sm + C::k_off + st * C::TILE;
                uint8_t* vt = sm + C::v_off + st * C::TILE;
#pragma unroll
                for (int b = 0; b < EACH; b += NB) {
#pragma unroll
                    for (int e = 0; e < NB; ++e) {
                        store(kt, b + e, kr[e]);
                        if (b + NB < EACH) kr[e] = load(kc, b + NB + e);
                    }
                }
#pragma unroll
                for (int e = 0; e < NB; ++e) vr[e] = load(vc, e);
                if (dtid < 32) {   // the tile's scale table
                    float most = vs;
#pragma unroll
                    for (int o = 4; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    cmax = fmaxf(cmax, most);
                    if (j == 0) vs0 = fmaxf(most, 7.888609e-31f);   // 2^-100
                    const float ref = fmaxf(cmax, vs0) * 9.313226e-10f;   // 2^-30
                    const float lv = log2f(__fdiv_rn(fmaxf(vs, ref), vs0));
                    if (lane < 8) sct[(J % PR_SCT) * 8 + lane] = make_float4(ks * a.scale_log2, lv, exp2f(-lv), vs0);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[J % PR_SCT]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                if (ok && J >= NS) ok = __all_sync(0xffffffffu, wait_parity_sleep(&v_empty[st], (J / NS - 1) & 1));
#pragma unroll
                for (int b = 0; b < EACH; b += NB) {
#pragma unroll
                    for (int e = 0; e < NB; ++e) {
                        store(vt, b + e, vr[e]);
                        if (b + NB < EACH) vr[e] = load(vc, b + NB + e);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
            }
            jj += max(n, 0);
        }
    } else if (warp >= 4) {
        // ===================== softmax: a row per thread =====================
        const int t = (warp - 4) >> 2, q4 = warp & 3, r = 128 * t + 32 * q4 + lane;   // row tile, lane quarter, row
        const uint32_t tl = tmem + ((uint32_t)(32 * q4) << 16);
        const int nsm = 128 * NT, stid = threadIdx.x - 128;
        auto bar = [&] { named_sync(1, (uint32_t)nsm); };
        constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
        while (attn_next<C::ROWS, PR_KT>(a, run, &g)) {
            const int n = g.t1 - g.t0;
            if (n > 0) {
                // ---- this warp's 32 rows of q, 128-byte swizzled; bf16 rows times a power of two that brings their
                // largest magnitude into [2^13, 2^14), so that fp16 holds them ----
                constexpr int LPR = DT / 8, RPW = 32 / LPR > 0 ? 32 / LPR : 1;   // lanes per row (8 elements each)
                uint8_t* qt = sm + C::q_off + t * C::TILE;
                const int c = lane % LPR;
#pragma unroll 4
                for (int i = 0; i < 32; i += RPW) {
                    const int rl = 32 * q4 + i + lane / LPR, rr = 128 * t + rl;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (rr < g.rows && 8 * c < a.dim) {
                        const int tok = (g.r0 + rr) / a.G, hq = g.h * a.G + (g.r0 + rr) - tok * a.G;
                        v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (g.q0 + tok) * a.ldq +
                                                            (long long)hq * a.dim + 8 * c);
                    }
                    if constexpr (bf) {
                        Raw8<VKB_DT_BF16> raw;
                        raw.a = v;
                        float f[8], m = 0.f;
                        raw8_to<VKB_DT_BF16>(raw, f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
                        for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        const int e2 = (int)(__float_as_uint(m) >> 23) - 127;
                        const float fac = m == 0.f ? 1.f : exp2f((float)min(126, max(-126, 13 - e2)));
                        if (c == 0) rowf[rr] = fac;
                        v = make_uint4(pack_f16(f[0] * fac, f[1] * fac), pack_f16(f[2] * fac, f[3] * fac),
                                       pack_f16(f[4] * fac, f[5] * fac), pack_f16(f[6] * fac, f[7] * fac));
                    }
                    sts128(smem_u32(qt) + (c >> 3) * C::HALF + rl * 128 + (((c & 7) ^ (rl & 7)) << 4), v);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const int rr = min(r, g.rows - 1), pos = g.pos0 + (g.r0 + rr) / a.G;
            const int khi = r < g.rows ? pos + 1 : 0, klo = a.window > 0 ? pos - a.window + 1 : 0;
            const float qinv = bf && n > 0 ? __fdiv_rn(1.f, rowf[r]) : 1.f;
            const int all_hi = g.pos0 + g.r0 / a.G + 1;   // keys [all_lo, all_hi): every row of the item sees them
            const int all_lo = a.window > 0 ? g.pos0 + (g.r0 + g.rows - 1) / a.G - a.window + 1 : 0;
            float M = -INFINITY, vs0 = 0.f;
            uint64_t l2 = 0;   // the sum of p, two halves
            for (int j = 0; j < n; ++j) {
                const int J = jj + j, buf = NT == 2 ? t : J & 1, key0 = (g.t0 + j) * PR_KT;
                if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&s_full[buf], (NT == 2 ? J : J >> 1) & 1));
                if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&sc_full[J % PR_SCT], (J / PR_SCT) & 1));
                if (!ok) continue;   // the wait gave up (status bit): the walk goes on so that every arrival is made
                tc_fence_after();
                const float4* sc = sct + (J % PR_SCT) * 8;
                const uint32_t ts = tl + buf * 128;
                const bool masked = key0 + PR_KT > all_hi || key0 < all_lo || r >= g.rows;
                const bool wmask = __any_sync(0xffffffffu, masked);
                uint32_t s[32], s2[32];   // 32 scores each: one chunk is worked on while the next one is read
                // ---- maximum of x ----
                float mx = -INFINITY;
                auto max_of = [&](const uint32_t (&v)[32], int c) {
                    mx = wmask ? pr_max<true>(v, sc + 2 * c, qinv, key0 + 32 * c, klo, khi, mx)
                               : pr_max<false>(v, sc + 2 * c, qinv, 0, 0, 0, mx);
                };
                tmem_ld32_async(ts, s);
                tmem_wait_ld(s);
                tmem_ld32_async(ts + 32, s2);
                max_of(s, 0);
                tmem_wait_ld(s2);
                tmem_ld32_async(ts + 64, s);
                max_of(s2, 1);
                tmem_wait_ld(s);
                tmem_ld32_async(ts + 96, s2);
                max_of(s, 2);
                tmem_wait_ld(s2);
                max_of(s2, 3);
                vs0 = sc[0].w;
                const bool grow = mx > M + PR_LAZY || (mx > -INFINITY && M == -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = fmaxf(M, mx), al = M == -INFINITY ? 0.f : ex2_ftz(M - mn);
                    M = mn;
                    l2 = f2_fma(l2, f2_make(al, al), 0);
                    if (j > 0) {   // O of the tiles before this one, once its last MMA is done
                        if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&o_full[t], (J - 1) & 1));
                        tc_fence_after();
                        const uint32_t to = tl + C::o_col + t * DT;
#pragma unroll 1
                        for (int c = 0; c < DT / 32; ++c) {
                            tmem_ld32(to + 32 * c, s);
#pragma unroll
                            for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * al);
                            tmem_st32(to + 32 * c, s);
                        }
                    }
                }
                // ---- p' and its sum. P's columns 16 c .. 16 c + 15 lie in S's columns below 32 c + 32, which have been
                // read ----
                const float mb = M == -INFINITY ? 0.f : M - PR_BIAS;
                auto exp_of = [&](const uint32_t (&v)[32], int c) {
                    uint32_t pk[16];
                    if (wmask) pr_exp<true>(v, pk, sc + 2 * c, qinv, mb, key0 + 32 * c, klo, khi, l2);
                    else pr_exp<false>(v, pk, sc + 2 * c, qinv, mb, 0, 0, 0, l2);
                    tmem_st16(ts + 16 * c, pk);
                };
                tmem_ld32_async(ts, s);
                tmem_wait_ld(s);
                tmem_ld32_async(ts + 32, s2);
                exp_of(s, 0);
                tmem_wait_ld(s2);
                tmem_ld32_async(ts + 64, s);
                exp_of(s2, 1);
                tmem_wait_ld(s);
                tmem_ld32_async(ts + 96, s2);
                exp_of(s, 2);
                tmem_wait_ld(s2);
                exp_of(s2, 3);
                tmem_wait_st();
                // A barrier's phase can be waited for only until the next one completes: with one row tile this tile's S
                // does not follow from the last O update, so every update is waited for, before this P allows the next
                if (NT == 1 && j > 0 && ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&o_full[t], (J - 1) & 1));
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[buf]);
            }
            // ---- the item's part, or its output ----
            const float l = f2_get(l2).x + f2_get(l2).y;
            if (n > 0 && ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&o_full[t], (jj + n - 1) & 1));
            tc_fence_after();
            const uint32_t to = tl + C::o_col + t * DT;
            constexpr int PITCH = DT + 2;
            float* part = a.part + attn_slot(run, g, blockIdx.x) * C::ROWS * PITCH;
            const float inv = g.whole ? (l == 0.f ? 0.f : __fdiv_rn(vs0, l)) : vs0;
            const bool live = M > -INFINITY || M != M || l != 0.f;   // rows that saw a key
            T* out = attn_out<T>(a, g, rr);
            if (r < g.rows && !g.whole) *reinterpret_cast<float2*>(part + C::ROWS * DT + 2 * r) = make_float2(M, l);
#pragma unroll 1
            for (int c = 0; c < DT / 32; ++c) {
                uint32_t s[32];
                if (n > 0 && ok) tmem_ld32(to + 32 * c, s);
                if (r >= g.rows) continue;
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (32 * c + e >= a.dim) break;
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = n > 0 && live ? __uint_as_float(s[e + i]) * inv : 0.f;
                    if (g.whole) {
                        store8<std::is_same<T, __half>::value ? VKB_DT_F16 : VKB_DT_BF16>(out + 32 * c + e, f);
                    } else {
                        float2* p = reinterpret_cast<float2*>(part + (long long)r * DT + 32 * c + e);
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = make_float2(f[2 * i], f[2 * i + 1]);
                    }
                }
            }
            tc_fence_before();   // O and S are read before the next item's MMAs, which this thread's arrivals release
            jj += max(n, 0);
            if (!g.whole) attn_join<DT, C::ROWS, T>(a, run, g, stid, nsm, join_sh, bar);
        }
    }
    // The softmax warps have waited for the last O update, and so for every MMA, before tensor memory is freed
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc<1>(tmem, 512);
}

}  // namespace vkb
