// Attention for many query rows per kv head (prompts and prompt chunks), on the 5th-generation tensor cores.
//
// An item is a tile of NT x 128 query rows; per 64 keys S = Q K'^T and O += P V' are tcgen05.mma with fp32
// accumulators in tensor memory, K' and V' the codes as exact fp16 integers in shared memory, converted once for all
// rows of the tile. The scales never touch the codes: with x_j = s_j ks_j scale log2(e) + log2(vs_j / V),
//   p'_j = 2^(x_j - M + 8),   O' = sum_j p'_j c'_j,   l = sum_j p'_j (V / vs_j),   o = V O' / l,
// so a group of 16 keys (a page or part of one) costs one multiply-add per score and one multiply per group. p' is
// rounded once, to fp16, for the product; l sums it in fp32. M follows the running maximum of x lazily, so that O' is
// rescaled only when a p' might leave fp16's range. V is the power of two at or below the largest V scale seen so far (so
// that it seldom moves: O' is rescaled then too); scales below 2^-30 of that largest count as 2^-30 of it. V follows upwards
// because M would have to stand in for it otherwise: behind first keys of scale 0 M jumped past what 2^(M - M') holds, and
// their part of l was lost.
//
// 16 warps, one block per SM (its run of units: attn_common.cuh):
//   warp 0        issues the MMAs. S has two buffers of 64 columns per row tile, and P takes its S's place: S(j + 1) is
//                 issued before P(j) is there, so that the softmax goes from one tile to the next without waiting for
//                 an MMA (with one buffer of 128 keys the two waited for each other: 7700 cycles per 128 keys, the
//                 softmax busy for 3800 of them)
//   warp 1        makes the scale tables {ks scale log2(e), log2(vs / V), V / vs, V} of the groups of 16 keys
//   warps 4-7     softmax of row tile 0, a row per thread (tensor memory lanes are rows)
//   warps 8-11    softmax of row tile 1 (NT = 2: dimensions up to 128); convert codes (NT = 1: dimension 256, where O
//                 takes half of tensor memory)
//   warps 12-15   convert codes: global loads of 16 codes (past L1: each is read once), two tiles ahead in registers, to
//                 128-byte swizzled fp16 tiles (K: K-major B operand; V: the same bytes are the MN-major B operand of P V)
// Measured on a B200 (32 q heads on 8, dimension 128): 4096 tokens behind 12288 take 1.21 ms, 795 TFLOP/s on the causal
// pairs; the tensor pipe is busy for 36 % of it, the exponentials for a third, and a
// scheduler issues 0.41 instructions per cycle: bound by latency, two softmax warps per scheduler with one dependent chain per
// tile each (load of S, multiply-add, exponential, pack, store of P).
#pragma once

#include "attn_token.cuh"
#include "tcgen05.cuh"

namespace vkb {

constexpr int PR_KT = 64;                // keys per unit
constexpr int PR_OV = 16;                // an item's own cost in units
constexpr int PR_THREADS = 512;
constexpr float PR_BIAS = 8.f;           // p' carries 2^8
constexpr int PR_SCT = 16;               // tiles of scale tables: two batches of eight (a lane per group of 16 keys)

template <int DT> struct PrCfg {
    static constexpr int NT = DT == 256 ? 1 : 2;
    static constexpr int ROWS = 128 * NT;
    static constexpr int NS = DT == 256 ? 2 : 4;                  // converted tiles of K and of V
    static constexpr int ND = NT == 1 ? 256 : 128;                // converting threads
    static constexpr int TILE = PR_KT * DT * 2;                   // bytes of a converted tile
    static constexpr int HALF = PR_KT * 128;                      // bytes of its 64-column pieces
    static constexpr int QTILE = 128 * DT * 2, QHALF = 128 * 128; // a row tile of q, its pieces
    static constexpr int q_off = 0;
    static constexpr int k_off = NT * QTILE;
    static constexpr int v_off = k_off + NS * TILE;
    static constexpr int sc_off = v_off + NS * TILE;              // [PR_SCT][4] {kf, lv, iv, V}
    static constexpr int row_off = sc_off + PR_SCT * 4 * 16;      // [ROWS] factor of q
    static constexpr int bar_off = row_off + ROWS * 4;
    static constexpr int NBAR = 1 + 4 * NS + 4 + 4 + 4 + 4 + 1;
    static constexpr int run_off = bar_off + NBAR * 8;
    static constexpr int BYTES = run_off + 4 * (PR_THREADS / 32 + 2) + 16 + 1024;
    static constexpr int o_col = 256;                             // O of row tile t at o_col + t DT; its S buffers at
                                                                  // 128 t and 128 t + 64
};

// Low words of 128B-swizzled operand descriptors (shared memory ends below 2^18 bytes, so that a place further on is
// an addition to this word) and the high word both kinds share: 8-row atoms 1024 bytes apart (the stride byte offset).
//   K-major: rows of 64 k (128 bytes), 8 rows to an atom.
//   MN-major: 8 k, each a row of 64 elements (128 bytes), to an atom; 64-element pieces lbo apart (leading byte offset).
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;   // stride, version (sm_100), SWIZZLE_128B

// D += A B (accum 0: D = A B) with A from shared / tensor memory. Descriptors' low words only: what changes from one MMA to
// the next is one 32-bit addition, which keeps the issuing warp ahead of the tensor pipe.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accum), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accum), "n"(DESC_HI)
        : "memory");
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

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The factor of a group's scores: positive also where the page's scale is 0, so that a masked score stays -inf.
__device__ __forceinline__ float pr_factor(float4 f, float qinv) { return fmaxf(f.x * qinv, 1e-37f); }

// Maximum of x = s kf + lv over 32 scores (two groups of 16 keys).
__device__ __forceinline__ float pr_max(const uint32_t (&s)[32], const float4* sc, float qinv, float mx) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float m[2] = {__uint_as_float(s[16 * h]), __uint_as_float(s[16 * h + 1])};
#pragma unroll
        for (int e = 2; e < 14; e += 4) {
            m[0] = max3(m[0], __uint_as_float(s[16 * h + e]), __uint_as_float(s[16 * h + e + 1]));
            m[1] = max3(m[1], __uint_as_float(s[16 * h + e + 2]), __uint_as_float(s[16 * h + e + 3]));
        }
        m[0] = max3(m[0], __uint_as_float(s[16 * h + 14]), __uint_as_float(s[16 * h + 15]));
        const float4 f = sc[h];
        mx = fmaxf(mx, fmaf(fmaxf(m[0], m[1]), pr_factor(f, qinv), f.y));
    }
    return mx;
}
// p' of 32 scores as fp16 pairs, their sum into l (two running halves), and into top the largest sum of eight of them.
__device__ __forceinline__ void pr_exp(const uint32_t (&s)[32], uint32_t (&pk)[16], const float4* sc, float qinv, float mb,
                                       uint64_t& l, float& top) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 f = sc[h];
        const float kf = pr_factor(f, qinv), cg = f.y - mb;
        const uint64_t kf2 = f2_make(kf, kf), cg2 = f2_make(cg, cg);
        uint64_t sum[2];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            float2 x = f2_get(f2_fma(f2_make(__uint_as_float(s[16 * h + e]), __uint_as_float(s[16 * h + e + 1])), kf2, cg2));
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            const uint64_t p = f2_make(x.x, x.y);
            sum[(e >> 1) & 1] = e < 4 ? p : f2_add(sum[(e >> 1) & 1], p);
            pk[8 * h + e / 2] = pack_f16(x.x, x.y);
        }
        const uint64_t both = f2_add(sum[0], sum[1]);
        const float2 b = f2_get(both);
        top = max3(top, b.x, b.y);
        l = f2_fma(both, f2_make(f.z, f.z), l);
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

// Eight tiles from t on, a lane per group of 16 keys: whether any row may see the group (first: attn_first_key), and its
// page, -1 where none does.
__device__ __forceinline__ bool pr_seen(const AttnSeg& g, int first, int t, int lane) {
    const int key = (t + (lane >> 2)) * PR_KT + 16 * (lane & 3);
    return t + (lane >> 2) < g.t1 && key < g.len && key + 16 > first;
}
__device__ __forceinline__ int pr_page(const AttnArgs& a, const AttnSeg& g, int first, int t, int lane) {
    const int key = (t + (lane >> 2)) * PR_KT + 16 * (lane & 3);
    return pr_seen(g, first, t, lane) ? a.table[(long long)g.b * a.table_ld + (key >> a.page_log2)] : -1;
}

template <int DT, typename T>
__global__ void __launch_bounds__(PR_THREADS, 1) attn_prompt_kernel(const __grid_constant__ AttnArgs a,
                                                                    const uint8_t* kc,
                                                                    const uint8_t* vc) {
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
    uint64_t* s_full = v_empty + NS;      // [2 t + buffer] S written
    uint64_t* p_full = s_full + 4;        // [2 t + buffer] P written to it (4 warps)
    uint64_t* o_full = p_full + 4;        // [2 t + tile parity] O of the row tile updated
    uint64_t* sc_full = o_full + 4;       // [2] eight tiles' scale tables written
    uint64_t* sc_empty = sc_full + 2;     // [2] and read (NT * 4 warps)
    uint64_t* done = sc_empty + 2;        // every MMA of the block done
    unsigned* run_sh = reinterpret_cast<unsigned*>(sm + C::run_off);
    volatile int* join_sh = reinterpret_cast<volatile int*>(run_sh + PR_THREADS / 32 + 2);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(run_sh + PR_THREADS / 32 + 2) + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(q_full, NT * 4);
        mbar_init(done, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_full[i], C::ND / 32);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], C::ND / 32);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], NT * 4);
        }
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc<1>(tmem_slot, 512);
    tc_fence_before();
    pdl_wait();
    AttnRun run = attn_run<C::ROWS, PR_KT, PR_OV, PR_THREADS>(a, run_sh, join_sh + 2);   // its barriers publish the above
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    AttnSeg g;
    bool ok = true;
    int jj = 0;          // key tiles so far, over all items of the run

    // Registers: 512 threads are launched with 128 each (65536); the warpgroups take 56, 104 and 2 x 176 (65536), with NT = 1
    // 56, 2 x 128 and 192. The split stands at the head of each role, where the compiler counts from it. (160 for the softmax
    // and 128 to convert: 1.24 ms for the chunk of 4096 behind 12288 tokens, against 1.21.)
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
        // ===================== MMA issuer =====================
        const uint32_t id_s = umma_idesc_f16(PR_KT), id_o = umma_idesc_f16(DT) | (1u << 16);   // V': MN-major B
        const uint32_t dq = desc_k(smem_u32(sm + C::q_off)), dk = desc_k(smem_u32(sm + C::k_off));
        const uint32_t dv = desc_mn(smem_u32(sm + C::v_off), C::HALF);
        int qn = 0;
        auto wait = [&](uint64_t* bar, int phase) {
            if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(bar, phase & 1));
        };
        // S of row tile t for tile j, after the O update that read the buffer's last P
        auto qk = [&](int t, int j) {
            if (j > 1) wait(&o_full[2 * t + (j & 1)], (j - 2) >> 1);
            if (t == 0) wait(&k_full[j & (NS - 1)], j / NS);
            if (!ok) return;
            tc_fence_after();
            const uint32_t ds = tmem + 128 * t + 64 * (j & 1), aq = dq + t * (C::QTILE / 16), bk = dk + (j & (NS - 1)) * (C::TILE / 16);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < DT / 16; ++kk)   // 16 k: 32 bytes of a row
                    mma_ss(ds, aq + ((kk >> 2) * C::QHALF + (kk & 3) * 32) / 16, bk + ((kk >> 2) * C::HALF + (kk & 3) * 32) / 16,
                           id_s, kk != 0);
                umma_commit(&s_full[2 * t + (j & 1)]);
                if (t == NT - 1) umma_commit(&k_empty[j & (NS - 1)]);
            }
            __syncwarp();
        };
        while (ok && attn_next<C::ROWS, PR_KT, PR_OV>(a, run, &g)) {
            const int n = g.t1 - g.t0;
            if (n <= 0) continue;
            wait(q_full, qn++);
            for (int t = 0; t < NT; ++t) qk(t, jj);
            for (int j = 0; j < n && ok; ++j) {
                const int J = jj + j;
                for (int t = 0; t < NT && ok; ++t) {
                    if (j + 1 < n) qk(t, J + 1);
                    wait(&p_full[2 * t + (J & 1)], J >> 1);
                    if (t == 0) wait(&v_full[J & (NS - 1)], J / NS);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t dO = tmem + C::o_col + t * DT, ap = tmem + 128 * t + 64 * (J & 1);
                    const uint32_t bv = dv + (J & (NS - 1)) * (C::TILE / 16);
                    if (elect_one()) {
                        mma_ts(dO, ap, bv, id_o, j != 0);
#pragma unroll
                        for (int kk = 1; kk < PR_KT / 16; ++kk)   // 16 keys: 8 columns of P, 2 atoms of V'
                            mma_ts(dO, ap + 8 * kk, bv + kk * (2048 / 16), id_o, 1);
                        umma_commit(&o_full[2 * t + (J & 1)]);
                        if (t == NT - 1) umma_commit(&v_empty[J & (NS - 1)]);
                    }
                    __syncwarp();
                }
            }
            jj += n;
        }
        // drain: every MMA is done before tensor memory is freed, also where a wait gave up
        if (elect_one()) umma_commit(done);
        __syncwarp();
        wait_parity_sleep(done, 0, DEV_ERR_DRAIN_TIMEOUT);
        } else if (warp == 1) {
        // ===================== scale tables =====================
        int nb = 0;   // batches so far
        while (ok && attn_next<C::ROWS, PR_KT, PR_OV>(a, run, &g)) {
            const int n = g.t1 - g.t0, first = attn_first_key(a, g);
            float cmax = 7.888609e-31f;   // 2^-100, then the segment's largest V scale
            int next = pr_page(a, g, first, g.t0, lane);
            for (int j0 = 0; j0 < n && ok; j0 += 8, ++nb) {
                int id = next;
                next = pr_page(a, g, first, g.t0 + j0 + 8, lane);
                if (id >= a.pages) id = -1;
                float ks = 0.f, vs = 0.f;
                if (id >= 0) {
                    ks = __ldcg(a.ks + (long long)id * a.heads + g.h);
                    vs = __ldcg(a.vs + (long long)id * a.heads + g.h);
                }
                float most = fmaxf(vs, __shfl_xor_sync(0xffffffffu, vs, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {   // largest of this tile and the ones before it
                    const float v = __shfl_up_sync(0xffffffffu, most, o);
                    if (lane >= o) most = fmaxf(most, v);
                }
                most = fmaxf(most, cmax);
                cmax = __shfl_sync(0xffffffffu, most, 31);
                const float V = __uint_as_float(__float_as_uint(most) & 0x7f800000u);   // its power of two
                const float lv = log2f(__fdiv_rn(fmaxf(vs, most * 9.313226e-10f), V));    // 2^-30
                if (nb >= 2) ok = __all_sync(0xffffffffu, wait_parity_sleep(&sc_empty[nb & 1], ((nb >> 1) - 1) & 1));
                // keys of no page: weight 0, whatever their scores
                sct[(nb & 1) * 32 + lane] = id >= 0 ? make_float4(ks * a.scale_log2, lv, exp2f(-lv), V)
                                                    : make_float4(0.f, -INFINITY, 0.f, V);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_full[nb & 1]);
            }
        }
        }
    } else if (warp >= 16 - C::ND / 32) {
        if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // ===================== convert codes =====================
        constexpr int CPR = DT / 16, NB = PR_KT * CPR / C::ND;   // 16-code chunks per row; per thread and tile
        constexpr int RSTEP = C::ND / CPR;                        // rows between a thread's chunks (a multiple of 16)
        static_assert(RSTEP % 16 == 0 && NB == PR_KT / RSTEP, "the swizzle and the place in a group of 16 keys repeat");
        const int dtid = threadIdx.x - (PR_THREADS - C::ND), pl = a.page_log2, pmask = (1 << pl) - 1;
        // Thread to (row, 16 codes): eight lanes take four neighbouring chunks of two neighbouring rows, whose converted
        // halves (16-byte chunks 2c, then 2c + 1, of rows that differ in the swizzle's low bit) hit different banks.
        const int c = (lane & 3) + 4 * ((lane >> 3) % (CPR / 4));
        const int r0 = (dtid >> 5) * (32 / CPR) + ((lane >> 2) & 1) + 2 * ((lane >> 3) / (CPR / 4));
        const uint32_t st0 = (c >> 2) * C::HALF + r0 * 128 + (((2 * c) & 7) ^ (r0 & 7)) * 16, st1 = st0 ^ 16;
        const long long toff = (long long)(r0 & 15) * a.dim + 16 * c;   // within a group's 16 keys
        const bool col = 16 * c < a.dim;
        auto store = [&](uint32_t tile, const uint4 (&v)[NB]) {
#pragma unroll
            for (int e = 0; e < NB; ++e) {
                const uint32_t w[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
                uint32_t o[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[2 * i] = h2_sub(prmt(w[i], 0x64646464u, 0x4140u), 0x64806480u);
                    o[2 * i + 1] = h2_sub(prmt(w[i], 0x64646464u, 0x4342u), 0x64806480u);
                }
                sts128(tile + st0 + e * RSTEP * 128, make_uint4(o[0], o[1], o[2], o[3]));
                sts128(tile + st1 + e * RSTEP * 128, make_uint4(o[4], o[5], o[6], o[7]));
            }
        };
        struct Tile { uint4 k[NB], v[NB]; };   // a tile's codes on their way to shared memory
        while (ok && attn_next<C::ROWS, PR_KT, PR_OV>(a, run, &g)) {
            const int n = g.t1 - g.t0, first = attn_first_key(a, g);
            // eight tiles' groups, a lane each: where their codes start, -1 where there are none
            long long base = -1;
            int next = pr_page(a, g, first, g.t0, lane);
            auto enter = [&](int t) {
                int id = next;
                next = pr_page(a, g, first, t + 8, lane);
                if (id >= a.pages || (id < 0 && pr_seen(g, first, t, lane))) {
                    raise_status(DEV_ERR_BAD_INDEX);
                    id = -1;
                }
                base = -1;
                if (id >= 0)
                    base = ((((long long)id * a.heads + g.h) << pl) + (((t + (lane >> 2)) * PR_KT + 16 * (lane & 3)) & pmask)) * a.dim;
            };
            // tile j's loads (codes of value 0 where the key or the column does not exist)
            auto load = [&](Tile& x, int j) {
                if ((j & 7) == 0) enter(g.t0 + j);
                const int left = g.len - (g.t0 + j) * PR_KT - r0;
#pragma unroll
                for (int e = 0; e < NB; ++e) {
                    const long long p = __shfl_sync(0xffffffffu, base, 4 * (j & 7) + ((r0 + e * RSTEP) >> 4));
                    x.k[e] = x.v[e] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    if (p >= 0 && e * RSTEP < left && col) {
                        x.k[e] = __ldcg(reinterpret_cast<const uint4*>(kc + p + toff));
                        x.v[e] = __ldcg(reinterpret_cast<const uint4*>(vc + p + toff));
                    }
                }
            };
            auto convert = [&](const Tile& x, int j) {
                const int J = jj + j, st = J & (NS - 1);
                if (J >= NS) ok = __all_sync(0xffffffffu, wait_parity_sleep(&k_empty[st], (J / NS - 1) & 1));
                store(smem_u32(sm + C::k_off + st * C::TILE), x.k);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                if (ok && J >= NS) ok = __all_sync(0xffffffffu, wait_parity_sleep(&v_empty[st], (J / NS - 1) & 1));
                store(smem_u32(sm + C::v_off + st * C::TILE), x.v);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
            };
            // two tiles ahead: a load has the time of a whole tile
            Tile x0, x1;
            if (n > 0) load(x0, 0);
            if (n > 1) load(x1, 1);
            for (int j = 0; j < n && ok; j += 2) {
                convert(x0, j);
                if (j + 2 < n) load(x0, j + 2);
                if (j + 1 < n && ok) {
                    convert(x1, j + 1);
                    if (j + 3 < n) load(x1, j + 3);
                }
            }
            jj += max(n, 0);
        }
    } else {
        if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // ===================== softmax: a row per thread =====================
        const int t = (warp - 4) >> 2, q4 = warp & 3, r = 128 * t + 32 * q4 + lane;   // row tile, lane quarter, row
        const uint32_t tl = tmem + ((uint32_t)(32 * q4) << 16);
        int nb = 0;   // batches of scale tables so far
        const int nsm = 128 * NT, stid = threadIdx.x - 128;
        auto bar = [&] { named_sync(1, (uint32_t)nsm); };
        constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
        while (attn_next<C::ROWS, PR_KT, PR_OV>(a, run, &g)) {
            const int n = g.t1 - g.t0;
            if (n > 0) {
                // ---- this warp's 32 rows of q, 128-byte swizzled; bf16 rows times a power of two that brings their
                // largest magnitude into [2^13, 2^14), so that fp16 holds them ----
                constexpr int LPR = DT / 8, RPW = 32 / LPR > 0 ? 32 / LPR : 1;   // lanes per row (8 elements each)
                uint8_t* qt = sm + C::q_off + t * C::QTILE;
                const int c = lane % LPR;
                constexpr int QB = 32 / RPW < 16 ? 32 / RPW : 16;   // rows (per lane group) in flight
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += QB * RPW) {
                    uint4 v[QB];
#pragma unroll
                    for (int i = 0; i < QB; ++i) {
                        const int rr = 128 * t + 32 * q4 + i0 + i * RPW + lane / LPR;
                        v[i] = make_uint4(0u, 0u, 0u, 0u);
                        if (rr < g.rows && 8 * c < a.dim) {
                            const int tok = (g.r0 + rr) / a.G, hq = g.h * a.G + (g.r0 + rr) - tok * a.G;
                            v[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (g.q0 + tok) * a.ldq +
                                                                   (long long)hq * a.dim + 8 * c);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < QB; ++i) {
                        const int rl = 32 * q4 + i0 + i * RPW + lane / LPR;
                        if constexpr (bf) {
                            Raw8<VKB_DT_BF16> raw;
                            raw.a = v[i];
                            float f[8], m = 0.f;
                            raw8_to<VKB_DT_BF16>(raw, f);
#pragma unroll
                            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
                            for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                            const float fac = row_factor(m);
                            if (c == 0) rowf[128 * t + rl] = fac;
                            v[i] = make_uint4(pack_f16(f[0] * fac, f[1] * fac), pack_f16(f[2] * fac, f[3] * fac),
                                              pack_f16(f[4] * fac, f[5] * fac), pack_f16(f[6] * fac, f[7] * fac));
                        }
                        sts128(smem_u32(qt) + (c >> 3) * C::QHALF + rl * 128 + (((c & 7) ^ (rl & 7)) << 4), v[i]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const int rr = min(r, g.rows - 1), pos = g.pos0 + (g.r0 + rr) / a.G;
            const int khi = r < g.rows ? pos + 1 : 0, klo = attn_window(a, pos);
            const float qinv = bf && n > 0 ? __fdiv_rn(1.f, rowf[r]) : 1.f;
            const int all_hi = __reduce_min_sync(0xffffffffu, khi);   // keys [all_lo, all_hi): all the warp's rows see them
            const int all_lo = __reduce_max_sync(0xffffffffu, klo);
            float M = -INFINITY, V = 0.f;
            uint64_t l2 = 0;   // the sum of p, two halves
            for (int j = 0; j < n; ++j) {
                const int J = jj + j, buf = 2 * t + (J & 1), key0 = (g.t0 + j) * PR_KT;
                if (ok && (j & 7) == 0)
                    ok = __all_sync(0xffffffffu, wait_parity_sleep(&sc_full[nb & 1], (nb >> 1) & 1));
                if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&s_full[buf], (J >> 1) & 1));
                if (!ok) continue;   // the wait gave up (status bit): the walk goes on to the items' joins, whose barriers and
                                     // counts the other warps and blocks need (the pipeline's waits give up one after another)
                tc_fence_after();
                const float4* sc = sct + (nb & 1) * 32 + (j & 7) * 4;
                const uint32_t ts = tl + 64 * buf;
                const bool masked = key0 + PR_KT > all_hi || key0 < all_lo;
                uint32_t s[32], s2[32];   // the row's 64 scores
                auto read = [&] {
                    tmem_ld32_async(ts, s);
                    tmem_ld32_async(ts + 32, s2);
                    tmem_wait_ld(s);
                    tmem_wait_ld(s2);
                    if (masked) {   // keys that the row does not see (in the first and last tiles of an item)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (key0 + e < klo || key0 + e >= khi) s[e] = 0xff800000u;
                            if (key0 + 32 + e < klo || key0 + 32 + e >= khi) s2[e] = 0xff800000u;
                        }
                    }
                };
                const float v1 = sc[0].w;
                read();
                // ---- p' against the M of the tiles before this one, and its sum. Where eight p' of a row add up to more than
                // 2^15 (so that one of them might pass fp16's 65504), M is moved up to the maximum and the tile is done
                // again: the first tile that a row sees, the tiles where V moves, and few others, so that the maximum of the
                // scores is not taken ahead of everything else ----
                uint32_t pk[16], pk2[16];
                uint64_t sum = 0;
                float mb = M == -INFINITY ? 0.f : M - PR_BIAS, top = 0.f;
                pr_exp(s, pk, sc, qinv, mb, sum, top);
                pr_exp(s2, pk2, sc + 2, qinv, mb, sum, top);
                const bool unset = M == -INFINITY && klo < key0 + PR_KT && khi > key0;   // the row's first keys
                if (__any_sync(0xffffffffu, unset || top > 32768.f || v1 != V)) {
                    read();   // again, so that the scores need not stay in registers meanwhile
                    const float mx = pr_max(s2, sc + 2, qinv, pr_max(s, sc, qinv, -INFINITY));
                    const float mn = fmaxf(M, mx), al = M == -INFINITY ? 0.f : ex2(M - mn);
                    M = mn;
                    l2 = f2_fma(l2, f2_make(al, al), 0);
                    if (j > 0) {   // O of the tiles before this one, once its last MMA is done
                        if (ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&o_full[2 * t + ((J - 1) & 1)], ((J - 1) >> 1) & 1));
                        tc_fence_after();
                        const uint32_t to = tl + C::o_col + t * DT;
                        const float of = al * __fdiv_rn(V, v1);   // O' in units of the new V
#pragma unroll 1
                        for (int c = 0; c < DT / 32; ++c) {
                            tmem_ld32(to + 32 * c, s);
#pragma unroll
                            for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * of);
                            tmem_st32(to + 32 * c, s);
                        }
                        read();
                    }
                    V = v1;
                    sum = 0;
                    mb = M == -INFINITY ? 0.f : M - PR_BIAS;
                    pr_exp(s, pk, sc, qinv, mb, sum, top);
                    pr_exp(s2, pk2, sc + 2, qinv, mb, sum, top);
                }
                l2 = f2_add(l2, sum);
                tmem_st16(ts, pk);   // in place of S's first 32 columns
                tmem_st16(ts + 16, pk2);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[buf]);
                if ((j & 7) == 7 || j + 1 == n) {   // the batch's tables are done with
                    if (lane == 0) mbar_arrive(&sc_empty[nb & 1]);
                    ++nb;
                }
            }
            // ---- the item's part, or its output ----
            const float l = f2_get(l2).x + f2_get(l2).y;
            if (n > 0 && ok) ok = __all_sync(0xffffffffu, wait_parity_sleep(&o_full[2 * t + ((jj + n - 1) & 1)], ((jj + n - 1) >> 1) & 1));
            tc_fence_after();
            const uint32_t to = tl + C::o_col + t * DT;
            constexpr int PITCH = DT + 2;
            float* part = a.part + attn_slot(g, blockIdx.x) * C::ROWS * PITCH;
            const float inv = g.whole ? (l == 0.f ? 0.f : __fdiv_rn(V, l)) : V;
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
                        float4* p = reinterpret_cast<float4*>(part) + (8 * c + e / 4) * C::ROWS + r;
                        p[0] = make_float4(f[0], f[1], f[2], f[3]);
                        p[C::ROWS] = make_float4(f[4], f[5], f[6], f[7]);
                    }
                }
            }
            tc_fence_before();   // O and S are read before the next item's MMAs, which this thread's arrivals release
            jj += max(n, 0);
            if (!g.whole) attn_join<DT, C::ROWS, T>(a, g, stid, nsm, join_sh, bar);
        }
    }
    // The issuing warp has waited for every MMA, the softmax warps for their own loads, before tensor memory is freed
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc<1>(tmem, 512);
}

}  // namespace vkb
