// mxkv.cu -- writing and reading the MX-quantised paged KV cache.
//
// Quantisation of one 32-block (both formats): e = floor(log2 amax) - emax + 127
// clamped to 0..254 (emax 8 for E4M3, 2 for E2M1), codes = round(x * 2^(127 - e)).
// Scaling by a power of two is exact, so the only rounding is the one to the code.
#include "mxkv.cuh"

namespace fp4x {
namespace mxkv {

bool view(const char *who, const fp4x_mxkv *c, Cache &out) {
    if (!c) return set_error("%s: null cache", who), false;
    const uint32_t ps = c->page_size, hd = c->head_dim;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256)
        return set_error("%s: page_size %u is not 16, 32, 64, 128 or 256", who, ps), false;
    if (hd != 64 && hd != 128) return set_error("%s: head_dim %u is not 64 or 128", who, hd), false;
    if (c->format != FMT_FP8 && c->format != FMT_FP4)
        return set_error("%s: unknown cache format %u", who, c->format), false;
    if (c->n_kv_heads == 0 || c->n_pages == 0) return set_error("%s: empty cache", who), false;
    if ((uint64_t)c->n_pages * ps > 0x7FFFFFFFull)
        return set_error("%s: n_pages * page_size must stay below 2^31", who), false;
    if (!c->k || !c->v || !c->k_scales || !c->v_scales) return set_error("%s: null cache pointer", who), false;
    const uint64_t row = c->format == FMT_FP8 ? hd : hd / 2;
    if (c->page_stride < row * ps * c->n_kv_heads || c->scale_page_stride < (uint64_t)(hd / 32) * ps * c->n_kv_heads)
        return set_error("%s: pages overlap (strides below one page)", who), false;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % 16)
        return set_error("%s: codes and their page stride must be 16-byte aligned", who), false;
    if (!aligned(c->k_scales, 8) || !aligned(c->v_scales, 8) || c->scale_page_stride % 8)
        return set_error("%s: scales and their page stride must be 8-byte aligned", who), false;
    out.k = c->k, out.ks = c->k_scales, out.v = c->v, out.vs = c->v_scales;
    out.page_stride = c->page_stride, out.scale_stride = c->scale_page_stride;
    out.n_pages = c->n_pages, out.n_kv = c->n_kv_heads;
    out.page_shift = 31 - __builtin_clz(ps);
    return true;
}

// ---------------------------------------------------------------- append
__device__ __forceinline__ uint32_t e8m0_of(float amax, int emax) {
    if (!(amax > 0.0f)) return 127u;
    const uint32_t u = __float_as_uint(fminf(amax, 3.40282347e+38f));
    const int f = u >> 23 ? (int)(u >> 23) - 127 : (31 - __clz(u)) - 149;
    return (uint32_t)max(0, min(254, f - emax + 127));
}

// 2^(127 - e) as two factors, so that e = 254 and e = 0 stay exact.
__device__ __forceinline__ void inv_scale(uint32_t e, float &a, float &b) {
    const int h = 127 - (int)e, h0 = h / 2;
    a = __uint_as_float((uint32_t)(h0 + 127) << 23), b = __uint_as_float((uint32_t)(h - h0 + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Nearest E2M1 level, ties to the smaller magnitude; v < 0 sets the sign even when it rounds to 0.
__device__ __forceinline__ uint32_t e2m1_code(float v) {
    const float a = fabsf(v);
    const uint32_t c = (a > 0.25f) + (a > 0.75f) + (a > 1.25f) + (a > 1.75f) + (a > 2.5f) + (a > 3.5f) + (a > 5.0f);
    return c | (v < 0.0f ? 8u : 0u);
}

template <typename T>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float *p, float (&x)[4]) {
    const float4 f = __ldg(reinterpret_cast<const float4 *>(p));
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[4]) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xFFFF0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xFFFF0000u);
}

// One thread: dimensions 4g..4g+3 of one 32-block; eight neighbouring lanes share the block.
template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(256) kv_append_kernel(Cache c, uint32_t n, const int32_t *__restrict__ slots,
                                                        const T *__restrict__ k, uint64_t ks, const T *__restrict__ v,
                                                        uint64_t vs) {
    constexpr uint32_t NB = HD / 32;
    const uint64_t per = (uint64_t)c.n_kv * NB * 8, total = (uint64_t)n * 2 * per;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;  // whole groups of 8 lanes: per is a multiple of 8
    const uint32_t g = (uint32_t)(i & 7), b = (uint32_t)(i >> 3) % NB;
    const uint64_t r = i / (8 * NB);
    const uint32_t head = (uint32_t)(r % c.n_kv);
    const uint32_t is_v = (uint32_t)((r / c.n_kv) & 1);
    const uint32_t tok = (uint32_t)(r / c.n_kv / 2);
    float x[4];
    load4<T>((is_v ? v + tok * vs : k + tok * ks) + head * HD + b * 32 + g * 4, x);
    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    uint32_t nan = (x[0] != x[0]) | (x[1] != x[1]) | (x[2] != x[2]) | (x[3] != x[3]);
    const uint32_t mask = 0xFFu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
        amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
        nan |= __shfl_xor_sync(mask, nan, o);
    }
    uint32_t e = e8m0_of(amax, FMT == FMT_FP8 ? 8 : 2);
    float s0, s1;
    inv_scale(e, s0, s1);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = x[j] * s0 * s1;
    const int32_t slot = slots[tok];
    if (slot < 0) return;
    const uint32_t page = (uint32_t)slot >> c.page_shift, row = (uint32_t)slot & ((1u << c.page_shift) - 1);
    if (page >= c.n_pages) {
        raise_device_error(DEVERR_BAD_ARG);
        return;
    }
    uint8_t *dst = (is_v ? c.v : c.k) + code_off<FMT, HD>(c, page, head, row);
    if (FMT == FMT_FP8) {
        *reinterpret_cast<uint32_t *>(dst + (g * NB + b) * 4) = e4m3x2(x[0], x[1]) | (e4m3x2(x[2], x[3]) << 16);
    } else {
        *reinterpret_cast<uint16_t *>(dst + (g * NB + b) * 2) =
            (uint16_t)(e2m1_code(x[0]) | (e2m1_code(x[1]) << 4) | (e2m1_code(x[2]) << 8) | (e2m1_code(x[3]) << 12));
        if (nan) e = 255;
    }
    if (g == 0) ((is_v ? c.vs : c.ks) + scale_off<HD>(c, page, head, row))[b] = (uint8_t)e;
}

// ---------------------------------------------------------------- read
__device__ __forceinline__ void store4(float *p, const float (&x)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&x)[4]) {
    __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}

template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(Cache c, uint32_t n, const int32_t *__restrict__ slots,
                                                      T *__restrict__ k, T *__restrict__ v) {
    constexpr uint32_t NB = HD / 32;
    const uint64_t per = (uint64_t)c.n_kv * NB * 8, total = (uint64_t)n * 2 * per;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const uint32_t g = (uint32_t)(i & 7), b = (uint32_t)(i >> 3) % NB;
    const uint64_t r = i / (8 * NB);
    const uint32_t head = (uint32_t)(r % c.n_kv);
    const uint32_t is_v = (uint32_t)((r / c.n_kv) & 1);
    const uint32_t tok = (uint32_t)(r / c.n_kv / 2);
    const int32_t slot = slots[tok];
    const uint32_t page = (uint32_t)slot >> c.page_shift, row = (uint32_t)slot & ((1u << c.page_shift) - 1);
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (slot >= 0 && page < c.n_pages) {
        const uint8_t *src = (is_v ? c.v : c.k) + code_off<FMT, HD>(c, page, head, row);
        const float s = e8m0_to_f32(((is_v ? c.vs : c.ks) + scale_off<HD>(c, page, head, row))[b]);
        uint32_t h[2];
        if (FMT == FMT_FP8) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(src + (g * NB + b) * 4);
            h[0] = e4m3x2_to_f16x2(w & 0xFFFFu), h[1] = e4m3x2_to_f16x2(w >> 16);
        } else {
            const uint32_t w = *reinterpret_cast<const uint16_t *>(src + (g * NB + b) * 2);
            h[0] = e2m1x2_to_f16x2(w & 0xFFu), h[1] = e2m1x2_to_f16x2(w >> 8);
        }
        const float2 lo = __half22float2(*reinterpret_cast<__half2 *>(&h[0]));
        const float2 hi = __half22float2(*reinterpret_cast<__half2 *>(&h[1]));
        x[0] = lo.x * s, x[1] = lo.y * s, x[2] = hi.x * s, x[3] = hi.y * s;
    } else if (slot >= 0) {
        raise_device_error(DEVERR_BAD_ARG);
    }
    store4((is_v ? v : k) + ((uint64_t)tok * c.n_kv + head) * HD + b * 32 + g * 4, x);
}


}  // namespace mxkv
}  // namespace fp4x

using namespace fp4x;

extern "C" int llama_kv_append_mx(fp4x_stream_t stream, const fp4x_mxkv *cache, uint32_t n, const int32_t *slots,
                                  uint32_t dtype, const void *k, uint64_t k_stride, const void *v,
                                  uint64_t v_stride) {
    mxkv::Cache c;
    if (!mxkv::view("llama_kv_append_mx", cache, c)) return FP4X_EINVAL;
    FP4X_REQUIRE(dtype == FP4X_F32 || dtype == FP4X_BF16, "llama_kv_append_mx: unknown dtype %u", dtype);
    if (n == 0) return FP4X_OK;
    FP4X_REQUIRE(slots && k && v, "llama_kv_append_mx: null pointer");
    const uint32_t hd = cache->head_dim, vec = dtype == FP4X_F32 ? 4 : 8;
    FP4X_REQUIRE(mxkv::aligned(k, 16) && mxkv::aligned(v, 16) && k_stride % vec == 0 && v_stride % vec == 0,
                 "llama_kv_append_mx: rows of k and v must be 16-byte aligned");
    FP4X_REQUIRE(k_stride >= (uint64_t)c.n_kv * hd && v_stride >= (uint64_t)c.n_kv * hd,
                 "llama_kv_append_mx: row stride below n_kv_heads * head_dim");
    const uint64_t blocks = ((uint64_t)n * 2 * c.n_kv * (hd / 4) + 255) / 256;
    FP4X_REQUIRE(blocks <= 0x7FFFFFFFull, "llama_kv_append_mx: too many rows");
    cudaStream_t st = (cudaStream_t)stream;
#define FP4X_LAUNCH(FMT, HD, T)                                                                             \
    mxkv::kv_append_kernel<FMT, HD, T><<<(uint32_t)blocks, 256, 0, st>>>(c, n, slots, (const T *)k, k_stride, \
                                                                         (const T *)v, v_stride)
#define FP4X_PICK(FMT, HD)                                  \
    if (dtype == FP4X_F32) FP4X_LAUNCH(FMT, HD, float);     \
    else FP4X_LAUNCH(FMT, HD, __nv_bfloat16)
    if (cache->format == FP4X_MXFP8) {
        if (hd == 64) { FP4X_PICK(mxkv::FMT_FP8, 64); } else { FP4X_PICK(mxkv::FMT_FP8, 128); }
    } else {
        if (hd == 64) { FP4X_PICK(mxkv::FMT_FP4, 64); } else { FP4X_PICK(mxkv::FMT_FP4, 128); }
    }
#undef FP4X_PICK
#undef FP4X_LAUNCH
    return check_launch("llama_kv_append_mx");
}

extern "C" int llama_kv_read_mx(fp4x_stream_t stream, const fp4x_mxkv *cache, uint32_t n, const int32_t *slots,
                                uint32_t dtype, void *k_out, void *v_out) {
    mxkv::Cache c;
    if (!mxkv::view("llama_kv_read_mx", cache, c)) return FP4X_EINVAL;
    FP4X_REQUIRE(dtype == FP4X_F32 || dtype == FP4X_BF16, "llama_kv_read_mx: unknown dtype %u", dtype);
    if (n == 0) return FP4X_OK;
    FP4X_REQUIRE(slots && k_out && v_out, "llama_kv_read_mx: null pointer");
    FP4X_REQUIRE(mxkv::aligned(k_out, 16) && mxkv::aligned(v_out, 16),
                 "llama_kv_read_mx: outputs must be 16-byte aligned");
    const uint32_t hd = cache->head_dim;
    const uint64_t blocks = ((uint64_t)n * 2 * c.n_kv * (hd / 4) + 255) / 256;
    FP4X_REQUIRE(blocks <= 0x7FFFFFFFull, "llama_kv_read_mx: too many rows");
    cudaStream_t st = (cudaStream_t)stream;
#define FP4X_LAUNCH(FMT, HD, T) \
    mxkv::kv_read_kernel<FMT, HD, T><<<(uint32_t)blocks, 256, 0, st>>>(c, n, slots, (T *)k_out, (T *)v_out)
#define FP4X_PICK(FMT, HD)                                  \
    if (dtype == FP4X_F32) FP4X_LAUNCH(FMT, HD, float);     \
    else FP4X_LAUNCH(FMT, HD, __nv_bfloat16)
    if (cache->format == FP4X_MXFP8) {
        if (hd == 64) { FP4X_PICK(mxkv::FMT_FP8, 64); } else { FP4X_PICK(mxkv::FMT_FP8, 128); }
    } else {
        if (hd == 64) { FP4X_PICK(mxkv::FMT_FP4, 64); } else { FP4X_PICK(mxkv::FMT_FP4, 128); }
    }
#undef FP4X_PICK
#undef FP4X_LAUNCH
    return check_launch("llama_kv_read_mx");
}
