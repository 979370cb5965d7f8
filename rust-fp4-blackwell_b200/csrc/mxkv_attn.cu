// mxkv_attn.cu -- attention over the MX-quantised paged cache, with an optional
// prefix that all sequences of the batch share.
//
// For query row r of sequence b and KV head h, with keys k_t and values v_t of the
// prefix and of the sequence's own pages:
//   s_t = q . k_t / sqrt(hd),  out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),
// one pass with a running maximum m and sum; partial results of different warps
// join as (m, l, o).
#include "mxkv.cuh"

namespace fp4x {
namespace mxkv {

struct AttnParams {
    Cache c;
    uint32_t batch, n_heads, group, q_len, table_stride, max_len, prefix_len;
    const int32_t *prefix_pages, *page_table, *lens;
    const void *q;
    uint64_t q_stride;
    void *out;
    float scale;
};

template <uint32_t FMT, uint32_t HD>
__device__ __forceinline__ void row_values(const uint8_t *codes, const uint8_t *scales, uint32_t lane,
                                           float (&x)[HD / 32]) {
    constexpr uint32_t NB = HD / 32;
    const uint32_t g = lane >> 2, i = lane & 3;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        const uint32_t p = (g * NB + b) * 4 + i;
        uint32_t h;
        if (FMT == FMT_FP8)
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes[p]));
        else
            h = e2m1x2_to_f16x2((codes[p / 2] >> (4 * (p & 1))) & 15u);
        x[b] = __low2float(*reinterpret_cast<__half2 *>(&h)) * e8m0_to_f32(scales[b]);
    }
}

// One CTA of four warps per (sequence, query token, head); warps take positions in turn.
template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(128) attn_mx_kernel(AttnParams p) {
    constexpr uint32_t NB = HD / 32;
    const uint32_t row = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t head = row % p.n_heads, i = row / p.n_heads % p.q_len, b = row / p.n_heads / p.q_len;
    const uint32_t kvh = head / p.group;
    const int32_t len = min(max(p.lens[b], 0), (int32_t)p.max_len);
    const int32_t own = max(0, len - (int32_t)p.q_len + 1 + (int32_t)i);
    const uint32_t total = p.prefix_len + (uint32_t)own;
    const T *q = (const T *)p.q + ((uint64_t)b * p.q_len + i) * p.q_stride + head * HD;
    float qv[NB], o[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) qv[j] = (float)q[j * 32 + lane] * p.scale, o[j] = 0.0f;
    for (uint32_t t = warp; t < total; t += 4) {
        const uint32_t at = t < p.prefix_len ? t : t - p.prefix_len;
        const uint32_t idx = at >> p.c.page_shift, r = at & ((1u << p.c.page_shift) - 1);
        const int32_t page = t < p.prefix_len ? p.prefix_pages[idx] : p.page_table[(uint64_t)b * p.table_stride + idx];
        if (page < 0 || (uint32_t)page >= p.c.n_pages) {
            raise_device_error(DEVERR_BAD_ARG);
            continue;
        }
        const uint64_t co = code_off<FMT, HD>(p.c, page, kvh, r), so = scale_off<HD>(p.c, page, kvh, r);
        float kx[NB], vx[NB], s = 0.0f;
        row_values<FMT, HD>(p.c.k + co, p.c.ks + so, lane, kx);
#pragma unroll
        for (uint32_t j = 0; j < NB; ++j) s += qv[j] * kx[j];
        s = warp_sum(s);
        row_values<FMT, HD>(p.c.v + co, p.c.vs + so, lane, vx);
        const float mn = fmaxf(m, s), f = exp2f(m - mn), w = exp2f(s - mn);
        l = l * f + w;
#pragma unroll
        for (uint32_t j = 0; j < NB; ++j) o[j] = o[j] * f + w * vx[j];
        m = mn;
    }
    __shared__ float sm[4], sl[4], so[4][HD];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) so[warp][j * 32 + lane] = o[j];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        const float f = sm[w] == -INFINITY ? 0.0f : exp2f(sm[w] - top);
        sum += sl[w] * f, acc += so[w][threadIdx.x] * f;
    }
    const float y = sum == 0.0f ? 0.0f : acc / sum;
    ((T *)p.out)[(uint64_t)row * HD + threadIdx.x] = (T)y;
}

int launch_attn(const char *who, cudaStream_t st, const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                uint32_t q_len, const int32_t *prefix_pages, uint32_t prefix_len, const int32_t *page_table,
                uint32_t table_stride, const int32_t *lens, uint32_t max_len, uint32_t dtype, const void *q,
                uint64_t q_stride, void *out, void *workspace, size_t workspace_bytes) {
    AttnParams p;
    if (!view(who, cache, p.c)) return FP4X_EINVAL;
    const uint32_t hd = cache->head_dim;
    FP4X_REQUIRE(dtype == FP4X_F32 || dtype == FP4X_BF16, "%s: unknown dtype %u", who, dtype);
    FP4X_REQUIRE(n_heads && n_heads % p.c.n_kv == 0, "%s: n_heads %u is no multiple of n_kv_heads %u", who, n_heads,
                 p.c.n_kv);
    FP4X_REQUIRE(q_len >= 1 && q_len <= 64, "%s: q_len %u is not in 1..64", who, q_len);
    FP4X_REQUIRE(max_len < 0x7FFFFFFFu && prefix_len < 0x7FFFFFFFu && max_len + prefix_len < 0x7FFFFFFFu,
                 "%s: lengths must stay below 2^31", who);
    if (batch == 0) return FP4X_OK;
    const uint64_t rows = (uint64_t)batch * q_len * n_heads;
    FP4X_REQUIRE(rows <= 0x7FFFFFFFull / 2, "%s: too many query rows", who);
    FP4X_REQUIRE(q && out && lens, "%s: null pointer", who);
    FP4X_REQUIRE(max_len == 0 || page_table, "%s: null page table", who);
    FP4X_REQUIRE(prefix_len == 0 || prefix_pages, "%s: null prefix pages", who);
    FP4X_REQUIRE(((uint64_t)max_len + cache->page_size - 1) / cache->page_size <= table_stride,
                 "%s: table_stride %u holds fewer than max_len %u positions", who, table_stride, max_len);
    FP4X_REQUIRE(aligned(q, 16) && aligned(out, 16) && q_stride % (dtype == FP4X_F32 ? 4 : 8) == 0,
                 "%s: rows of q and out must be 16-byte aligned", who);
    FP4X_REQUIRE(q_stride >= (uint64_t)n_heads * hd, "%s: q_stride below n_heads * head_dim", who);
    const size_t need = llama_attn_mx_workspace_size(cache, batch, n_heads, q_len, prefix_len, max_len);
    FP4X_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))),
                 "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need, workspace_bytes);
    p.batch = batch, p.n_heads = n_heads, p.group = n_heads / p.c.n_kv, p.q_len = q_len;
    p.table_stride = table_stride, p.max_len = max_len, p.prefix_len = prefix_len;
    p.prefix_pages = prefix_pages, p.page_table = page_table, p.lens = lens;
    p.q = q, p.q_stride = q_stride, p.out = out;
    p.scale = 1.4426950408889634f / sqrtf((float)hd);
#define FP4X_LAUNCH(FMT, HD, T) attn_mx_kernel<FMT, HD, T><<<(uint32_t)rows, 128, 0, st>>>(p)
#define FP4X_PICK(FMT, HD)                              \
    if (dtype == FP4X_F32) FP4X_LAUNCH(FMT, HD, float); \
    else FP4X_LAUNCH(FMT, HD, __nv_bfloat16)
    if (cache->format == FP4X_MXFP8) {
        if (hd == 64) { FP4X_PICK(FMT_FP8, 64); } else { FP4X_PICK(FMT_FP8, 128); }
    } else {
        if (hd == 64) { FP4X_PICK(FMT_FP4, 64); } else { FP4X_PICK(FMT_FP4, 128); }
    }
#undef FP4X_PICK
#undef FP4X_LAUNCH
    return check_launch(who);
}

}  // namespace mxkv
}  // namespace fp4x

using namespace fp4x;

extern "C" size_t llama_attn_mx_workspace_size(const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                                               uint32_t q_len, uint32_t prefix_len, uint32_t max_len) {
    return 0;
}

extern "C" int llama_attn_paged_mx(fp4x_stream_t stream, const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                                   uint32_t q_len, const int32_t *page_table, uint32_t table_stride,
                                   const int32_t *lens, uint32_t max_len, uint32_t dtype, const void *q,
                                   uint64_t q_stride, void *out, void *workspace, size_t workspace_bytes) {
    return mxkv::launch_attn("llama_attn_paged_mx", (cudaStream_t)stream, cache, batch, n_heads, q_len, nullptr, 0,
                             page_table, table_stride, lens, max_len, dtype, q, q_stride, out, workspace,
                             workspace_bytes);
}

extern "C" int llama_attn_shared_mx(fp4x_stream_t stream, const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                                    uint32_t q_len, const int32_t *prefix_pages, uint32_t prefix_len,
                                    const int32_t *page_table, uint32_t table_stride, const int32_t *lens,
                                    uint32_t max_len, uint32_t dtype, const void *q, uint64_t q_stride, void *out,
                                    void *workspace, size_t workspace_bytes) {
    return mxkv::launch_attn("llama_attn_shared_mx", (cudaStream_t)stream, cache, batch, n_heads, q_len, prefix_pages,
                             prefix_len, page_table, table_stride, lens, max_len, dtype, q, q_stride, out, workspace,
                             workspace_bytes);
}
