// vkb_attention: argument checks, choice of the kernel, launch. The kernels: attn_token.cuh (few query rows per kv head),
// attn_prompt.cuh (many).
#include <mutex>

#include "attn_prompt.cuh"
#include "attn_token.cuh"

namespace vkb {

VKB_STATUS_ACCESSOR(status_take_attn)

int kv_cache_check(const vkb_kv_cache_t* c, const int32_t* table, int table_ld);   // kv_cache.cu

// Head dimension as the kernels hold it.
static int attn_dt(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// The largest partial result of a block: rows x (dimension, maximum and sum), of any variant.
static size_t attn_part_floats(int dt) {
    return (size_t)(dt == 256 ? 128 : 256) * (dt + 2);   // the prompt kernel's tile is the larger one
}

// Whether the kernels' 32-bit unit counts hold the call: an upper bound of its items times their units.
static bool units_fit(const vkb_kv_cache_t* c, const AttnArgs& a, int rows, int keys, int own) {
    const double items = (double)a.heads * ((double)a.T * a.G / rows + a.B);
    return items * ((double)a.table_ld * c->page / keys + 1 + own) <= 2147483647.0;
}

template <int DT, int NQ, typename T>
static int launch_token(const vkb_kv_cache_t* c, const AttnArgs& a, int dev, cudaStream_t st) {
    using C = TkCfg<DT, NQ>;
    if (!units_fit(c, a, C::ROWS, AT_KT, TK_OV)) return VKB_EUNSUPPORTED;
    auto kern = attn_token_kernel<DT, NQ, T>;
    static std::once_flag once[kMaxDevices];
    static cudaError_t err[kMaxDevices];
    std::call_once(once[dev], [&] {
        err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
        // the kernel's register split needs the registers that the block is launched with
        cudaFuncAttributes fa;
        if (err[dev] == cudaSuccess) err[dev] = cudaFuncGetAttributes(&fa, kern);
        if (err[dev] == cudaSuccess && fa.numRegs < C::LREG) err[dev] = cudaErrorInvalidConfiguration;
    });
    if (err[dev] != cudaSuccess) return -(int)err[dev];
    CUtensorMap tk, tv;
    const uint64_t rows = (uint64_t)c->pages * c->heads * c->page;
    const uint32_t pb = c->page < AT_KT ? c->page : AT_KT;
    const CUtensorMapSwizzle swz = DT == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    if (int r = get_tmap_2d(&tk, c->k, rows, c->dim, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, C::HB, pb, swz)) return r;
    if (int r = get_tmap_2d(&tv, c->v, rows, c->dim, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, C::HB, pb, swz)) return r;
    return launch_pdl(kern, dim3((unsigned)device_info(dev).sm_count), dim3(C::THREADS), C::BYTES, st, 1, tk, tv, a);
}

template <int DT, typename T>
static int launch_prompt(const vkb_kv_cache_t* c, const AttnArgs& a, int dev, cudaStream_t st) {
    using C = PrCfg<DT>;
    if (!units_fit(c, a, C::ROWS, PR_KT, PR_OV)) return VKB_EUNSUPPORTED;
    auto kern = attn_prompt_kernel<DT, T>;
    static std::once_flag once[kMaxDevices];
    static cudaError_t err[kMaxDevices];
    std::call_once(once[dev], [&] {
        err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
        // the kernel's register split needs the registers that the block is launched with
        cudaFuncAttributes fa;
        if (err[dev] == cudaSuccess) err[dev] = cudaFuncGetAttributes(&fa, kern);
        if (err[dev] == cudaSuccess && fa.numRegs != 128) err[dev] = cudaErrorInvalidConfiguration;
    });
    if (err[dev] != cudaSuccess) return -(int)err[dev];
    return launch_pdl(kern, dim3((unsigned)device_info(dev).sm_count), dim3(PR_THREADS), C::BYTES, st, 1, a,
                      (const uint8_t*)c->k, (const uint8_t*)c->v);
}

template <typename T>
static int attn_dispatch(const vkb_kv_cache_t* c, const AttnArgs& a, int dev, cudaStream_t st) {
    // Query rows per sequence and kv head, on average: the token kernel with the smallest tile that holds them. More rows
    // than its largest tile go to the prompt kernel, whose tile reads the keys once for 256 rows (128 at dimension 256), unless
    // the call is so small that the token kernel's many small items keep the SMs busier. Measured (token kernel against prompt
    // kernel, us, B200): 32 q heads on 8, dimension 128: one sequence of 8192 keys, 64 rows 39 against 50, 256 rows 79 against
    // 115, 512 rows 131 against 99; 16 sequences of 1500 keys, 36 rows 76 against 65, 64 rows 81 against 67. Dimension 64: one of
    // 8192 keys, 256 rows 65 against 66, 512 rows 108 against 64; 16 of 1500, 36 rows 62 against 54; 32 q heads on 2, 16 of 1500,
    // 64 rows 31 against 32, 128 rows 42 against 36. 16 q heads on 2, dimension 256: one of 8192 keys, 256 rows 48 against 214,
    // 16 of 1500 keys, 128 rows 72 against 101, 384 rows 174 against 107.
    // All of these are sequences alike. The lengths are on the device, so one kernel serves a call whose sequences differ, and
    // the mean says little there: 63 single tokens behind 4000 keys with a chunk of 2048 take 558 us (token kernel 1035), apart
    // 104 and 204; 255 behind 1000 with a prompt of 1024 556 us (prompt kernel 608), apart 151 and 76.
    const long long rows = ((long long)a.T + a.B - 1) / a.B * a.G;
    const bool few = (long long)a.T * a.G * a.heads <= (c->dim > 128 ? 4096 : 2560);
    switch (attn_dt(c->dim)) {
        case 64:
            if (rows <= 8) return launch_token<64, 1, T>(c, a, dev, st);
            if (rows <= 16) return launch_token<64, 2, T>(c, a, dev, st);
            return rows <= 32 || few ? launch_token<64, 4, T>(c, a, dev, st) : launch_prompt<64, T>(c, a, dev, st);
        case 128:
            if (rows <= 8) return launch_token<128, 1, T>(c, a, dev, st);
            if (rows <= 16) return launch_token<128, 2, T>(c, a, dev, st);
            return rows <= 32 || few ? launch_token<128, 4, T>(c, a, dev, st) : launch_prompt<128, T>(c, a, dev, st);
        default:
            if (rows <= 8) return launch_token<256, 1, T>(c, a, dev, st);
            return rows <= 16 || few ? launch_token<256, 2, T>(c, a, dev, st) : launch_prompt<256, T>(c, a, dev, st);
    }
}

constexpr size_t ATTN_CNT_BYTES = 4096;   // arrival counters: one per block of the grid (one per SM)

}  // namespace vkb

using namespace vkb;

extern "C" size_t vkb_attention_work_bytes(int dim) {
    int dev = 0;
    if (dim < 16 || dim > 256 || dim % 16 || current_device(&dev)) return 0;
    return ATTN_CNT_BYTES + (size_t)device_info(dev).sm_count * 2 * attn_part_floats(attn_dt(dim)) * sizeof(float);
}

extern "C" int vkb_attention(const vkb_kv_cache_t* c, const int32_t* table, int table_ld, const int32_t* lens,
                             const int32_t* cu, int B, int T, int dt, const void* q, long long ldq, void* out,
                             long long ldo, int q_heads, float scale, int window, void* work, size_t work_bytes,
                             vkb_stream_t stream) {
    if (int r = kv_cache_check(c, table, table_ld)) return r;
    if (!lens || B < 1 || T < 0 || (!cu && T != B) || window < 0 || !(scale >= 0.f)) return VKB_EINVAL;
    if (dt != VKB_DT_F16 && dt != VKB_DT_BF16) return dt == VKB_DT_F32 ? VKB_EUNSUPPORTED : VKB_EINVAL;
    if (q_heads < 1 || q_heads % c->heads) return VKB_EINVAL;
    if (T == 0) return 0;
    const long long row = (long long)q_heads * c->dim;
    if (!q || !out || ldq < row || ldo < row) return VKB_EINVAL;
    if (!work || !aligned_to(work, 16) || work_bytes < vkb_attention_work_bytes(c->dim)) return VKB_EINVAL;
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || ldq % 8 || ldo % 8) return VKB_EUNSUPPORTED;
    if ((long long)T * (q_heads / c->heads) > MAX_POSITIONS) return VKB_EUNSUPPORTED;
    int dev = 0;
    if (int r = current_device(&dev)) return r;
    if ((size_t)device_info(dev).sm_count * sizeof(unsigned) > ATTN_CNT_BYTES) return VKB_EUNSUPPORTED;
    AttnArgs a{};
    a.table = table; a.lens = lens; a.cu = cu;
    a.ks = c->k_scale; a.vs = c->v_scale;
    a.q = q; a.out = out;
    a.cnt = (unsigned*)work;
    a.part = (float*)((uint8_t*)work + ATTN_CNT_BYTES);
    a.ldq = ldq; a.ldo = ldo;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.B = B; a.T = T; a.heads = c->heads; a.G = q_heads / c->heads; a.dim = c->dim; a.pages = c->pages;
    a.page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    a.table_ld = table_ld; a.window = window; a.max_len = max_length(table_ld, c->page);
    cudaStream_t st = (cudaStream_t)stream;
    return dt == VKB_DT_F16 ? attn_dispatch<__half>(c, a, dev, st) : attn_dispatch<__nv_bfloat16>(c, a, dev, st);
}
