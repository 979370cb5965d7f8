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
    if (c->page_stride < row * ps * (uint64_t)c->n_kv_heads || c->scale_page_stride < (uint64_t)(hd / 32) * ps * c->n_kv_heads)
        return set_error("%s: pages overlap (strides below one page)", who), false;
    if (c->page_stride >> 32 || c->scale_page_stride >> 32)
        return set_error("%s: a page stride must stay below 4 GiB", who), false;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % 16)
        return set_error("%s: codes and their page stride must be 16-byte aligned", who), false;
    if (!aligned(c->k_scales, 8) || !aligned(c->v_scales, 8) || c->scale_page_stride % 8)
        return set_error("%s: scales and their page stride must be 8-byte aligned", who), false;
    out.k = c->k, out.ks = c->k_scales, out.v = c->v, out.vs = c->v_scales;
    out.page_stride = (uint32_t)c->page_stride, out.scale_stride = (uint32_t)c->scale_page_stride;
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

// 2^(127 - e): e is at most 252 (amax below 2^128), so this is a normal number.
__device__ __forceinline__ float inv_scale(uint32_t e) { return __uint_as_float((254u - e) << 23); }

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// x times 2^(127 - e) for the E2M1 conversion, which rounds ties to even where the rule is
// down, and with -0 as +0.  Every tie has at most two mantissa bits: one unit less in the
// last place turns ties (and exact levels, harmlessly) downwards.  An f32 value one unit
// above a tie must keep it, so the unit goes only where the low bits are zero; a bf16 value
// has no such neighbour, and a factor of 1 - 2^-24 in the scale does it for all.
template <typename T>
__device__ __forceinline__ float scaled_e2m1(float x, float s);
template <>
__device__ __forceinline__ float scaled_e2m1<__nv_bfloat16>(float x, float s) {
    return fmaf(x, s * 0.999999940395355224609375f, 0.0f);
}
template <>
__device__ __forceinline__ float scaled_e2m1<float>(float x, float s) {
    const uint32_t u = __float_as_uint(x * s);
    return __uint_as_float((u << 1) == 0 ? 0u : (u & 0x1FFFFFu) ? u : u - 1);
}
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
        : "=r"(r)
        : "f"(hi), "f"(lo));
    return r;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}

// Both kernels: four threads share a (K or V, token, head) row; thread t holds chunks
// 2t and 2t + 1, dimensions 8t..8t+7 of every 32-block, so it moves 16-byte pieces on
// both sides and a block's maximum takes two shuffles.  Bound by HBM: 131072 rows of
// 8 x 128 MXFP8 to bf16 take 124 us (0.98 of the measured rate), 16384 bf16 rows to MXFP4
// 19.8 us (85 MB, 4.3 TB/s), f32 rows to MXFP8 30.7 us (5.5 TB/s).  For MXFP4 the ALU comes
// first (65 % busy at 2.64 instructions a cycle and SM): 33 us with shuffles that name four lanes instead of the whole warp, 26 us with the
// f32 tie rule (below) for bf16 rows too.
template <uint32_t HD>
struct RowId {
    uint32_t t, head, is_v, token;
    __device__ __forceinline__ RowId(uint64_t i, uint32_t n_kv) {
        t = (uint32_t)(i & 3);
        const uint64_t r = i >> 2;
        const uint64_t tk = r / n_kv;
        head = (uint32_t)(r - tk * n_kv), is_v = (uint32_t)(tk & 1), token = (uint32_t)(tk >> 1);
    }
};

template <uint32_t WORDS>
__device__ __forceinline__ void store_words(uint8_t *p, const uint32_t (&w)[WORDS]) {
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < WORDS; i += 4)
            reinterpret_cast<uint4 *>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
}
template <uint32_t WORDS>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < WORDS; i += 4) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p) + i / 4);
            w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = u.x, w[1] = u.y;
    }
}

template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(256) kv_append_kernel(Cache c, uint32_t n, const int32_t *__restrict__ slots,
                                                        const T *__restrict__ k, uint64_t ks, const T *__restrict__ v,
                                                        uint64_t vs) {
    constexpr uint32_t NB = HD / 32, WORDS = Row<FMT, HD>::CHUNK / 2;
    // lanes past the end repeat the last row, so that the shuffles run with whole warps
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x, total = (uint64_t)n * 2 * c.n_kv * 4;
    const RowId<HD> id(i < total ? i : total - 4 + (i & 3), c.n_kv);
    const int32_t slot = slots[id.token];
    const T *src = (id.is_v ? v + id.token * vs : k + id.token * ks) + id.head * HD + id.t * 8;
    float x[NB][8];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) load8<T>(src + b * 32, x[b]);
    uint32_t w[WORDS], scales = 0;
#pragma unroll
    for (uint32_t j = 0; j < WORDS; ++j) w[j] = 0;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        float amax = 0.0f;
        uint32_t nan = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            amax = fmaxf(amax, fabsf(x[b][j]));
            if (FMT == FMT_FP4) nan |= x[b][j] != x[b][j];
        }
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
        uint32_t e = e8m0_of(amax, FMT == FMT_FP8 ? 8 : 2);
        const float s = inv_scale(e);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[b][j] = FMT == FMT_FP8 ? x[b][j] * s : scaled_e2m1<T>(x[b][j], s);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {  // chunk 2t + h: its four codes of block b at position 4 b
            const float *y = x[b] + 4 * h;
            if constexpr (FMT == FMT_FP8) {
                w[h * NB + b] = e4m3x2(y[0], y[1]) | (e4m3x2(y[2], y[3]) << 16);
            } else {
                const uint32_t half = e2m1x2(y[0], y[1]) | (e2m1x2(y[2], y[3]) << 8);
                w[(h * NB + b) / 2] |= half << (16 * (b & 1));
            }
        }
        if (FMT == FMT_FP4 && (__ballot_sync(~0u, nan) >> (threadIdx.x & 28) & 0xF)) e = 255;
        scales |= e << (8 * b);
    }
    if (slot < 0 || i >= total) return;
    const uint32_t page = (uint32_t)slot >> c.page_shift, row = (uint32_t)slot & ((1u << c.page_shift) - 1);
    if (page >= c.n_pages) {
        raise_device_error(DEVERR_BAD_ARG);
        return;
    }
    store_words<WORDS>((id.is_v ? c.v : c.k) + code_off<FMT, HD>(c, page, id.head, row) + id.t * WORDS * 4, w);
    if (id.t == 0) {
        uint8_t *dst = (id.is_v ? c.vs : c.ks) + scale_off<HD>(c, page, id.head, row);
        if (NB == 4)
            *reinterpret_cast<uint32_t *>(dst) = scales;
        else
            *reinterpret_cast<uint16_t *>(dst) = (uint16_t)scales;
    }
}

// ---------------------------------------------------------------- read
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}

template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(Cache c, uint32_t n, const int32_t *__restrict__ slots,
                                                      T *__restrict__ k, T *__restrict__ v) {
    constexpr uint32_t NB = HD / 32, WORDS = Row<FMT, HD>::CHUNK / 2;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (uint64_t)n * 2 * c.n_kv * 4) return;
    const RowId<HD> id(i, c.n_kv);
    const int32_t slot = slots[id.token];
    const uint32_t page = (uint32_t)slot >> c.page_shift, row = (uint32_t)slot & ((1u << c.page_shift) - 1);
    uint32_t w[WORDS], scales = 0;
#pragma unroll
    for (uint32_t j = 0; j < WORDS; ++j) w[j] = 0;
    if (slot >= 0 && page < c.n_pages) {
        load_words<WORDS>((id.is_v ? c.v : c.k) + code_off<FMT, HD>(c, page, id.head, row) + id.t * WORDS * 4, w);
        const uint8_t *src = (id.is_v ? c.vs : c.ks) + scale_off<HD>(c, page, id.head, row);
        scales = NB == 4 ? *reinterpret_cast<const uint32_t *>(src) : *reinterpret_cast<const uint16_t *>(src);
    } else if (slot >= 0) {
        raise_device_error(DEVERR_BAD_ARG);
    }
    T *dst = (id.is_v ? v : k) + ((uint64_t)id.token * c.n_kv + id.head) * HD + id.t * 8;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        const float s = e8m0_to_f32((scales >> (8 * b)) & 0xFF);
        float x[8];
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            uint32_t f[2];
            if constexpr (FMT == FMT_FP8) {
                const uint32_t y = w[h * NB + b];
                f[0] = e4m3x2_to_f16x2(y & 0xFFFFu), f[1] = e4m3x2_to_f16x2(y >> 16);
            } else {
                const uint32_t y = w[(h * NB + b) / 2] >> (16 * (b & 1));
                f[0] = e2m1x2_to_f16x2(y & 0xFF), f[1] = e2m1x2_to_f16x2((y >> 8) & 0xFF);
            }
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                const float2 z = __half22float2(*reinterpret_cast<const __half2 *>(&f[j]));
                x[4 * h + 2 * j] = z.x * s, x[4 * h + 2 * j + 1] = z.y * s;
            }
        }
        store8(dst + b * 32, x);
    }
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
    const uint64_t blocks = ((uint64_t)n * 2 * c.n_kv * 4 + 255) / 256;
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
    const uint64_t blocks = ((uint64_t)n * 2 * c.n_kv * 4 + 255) / 256;
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
