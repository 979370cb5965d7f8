// verify.cu -- verification of drafted tokens by speculative sampling with given
// random numbers.
//
// p_i = softmax(x_i / T) over the target's logits of position i.  Draft d_i is kept
// while u_i q_i(d_i) < p_i(d_i); the first rejected position samples from
// max(p - q, 0), a fully accepted draft from p_k.  Sampling by an exponential race:
// argmax_v w(v) / E(v) with E ~ Exp(1) picks v with probability w(v) / sum w, needs
// no normalised or running sums, and so does not hang on the order of a sum.
#include "common.cuh"

namespace fp4x {
namespace verify {

struct Params {
    uint32_t batch, k, vocab;
    const void *logits;
    uint64_t stride;
    const float *probs;
    const int32_t *drafts, *lens;
    const float *u, *noise, *temp;
    int32_t *accepted, *tokens;
    float *logprobs;
};

__device__ __forceinline__ float clean(float x) {  // NaN -> -inf, +inf -> the largest finite value
    return x != x ? -INFINITY : fminf(x, 3.40282347e+38f);
}
__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

struct Best {
    float v;
    uint32_t i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

__device__ Best block_best(Best x, Best *buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        x = better(x, Best{__shfl_xor_sync(~0u, x.v, o), __shfl_xor_sync(~0u, x.i, o)});
    __syncthreads();
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = x;
    __syncthreads();
    x = buf[0];
    for (uint32_t w = 1; w < blockDim.x / 32; ++w) x = better(x, buf[w]);
    return x;
}

// One CTA per sequence walks its rows.
template <typename T>
__global__ void __launch_bounds__(512) verify_kernel(Params p) {
    __shared__ Best buf[16];
    __shared__ float sums[16];
    const uint32_t b = blockIdx.x;
    const uint32_t n_draft = p.lens ? (uint32_t)min(max(p.lens[b], 0), (int32_t)p.k) : p.k;
    const float t = p.temp ? p.temp[b] : 1.0f;
    const bool greedy = !(t > 1e-30f);
    const float inv_t = greedy ? 1.0f : t;
    for (uint32_t i = 0;; ++i) {
        const T *x = (const T *)p.logits + ((uint64_t)b * (p.k + 1) + i) * p.stride;
        Best top{-INFINITY, 0xFFFFFFFFu};
        for (uint32_t v = threadIdx.x; v < p.vocab; v += blockDim.x) top = better(top, Best{clean(as_f32(x[v])), v});
        top = block_best(top, buf);
        if (top.v == -INFINITY) top.i = 0;
        float s = 0.0f;
        for (uint32_t v = threadIdx.x; v < p.vocab; v += blockDim.x) {
            const float y = clean(as_f32(x[v]));
            if (y > -INFINITY) s += expf((y - top.v) / inv_t);
        }
        s = warp_sum(s);
        __syncthreads();
        if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = s;
        __syncthreads();
        s = 0.0f;
        for (uint32_t w = 0; w < blockDim.x / 32; ++w) s += sums[w];
        const float *q = p.probs ? p.probs + ((uint64_t)b * p.k + i) * p.vocab : nullptr;
        int32_t tok;
        bool ok = false;
        if (i < n_draft) {
            tok = p.drafts[b * p.k + i];
            if ((uint32_t)tok < p.vocab) {
                const float y = clean(as_f32(x[tok]));
                const float pd = y > -INFINITY ? expf((y - top.v) / inv_t) / s : 0.0f;
                ok = greedy ? (uint32_t)tok == top.i : p.u[b * p.k + i] * (q ? q[tok] : 1.0f) < pd;
            }
        }
        if (!ok) {
            const bool residual = i < n_draft;
            const uint32_t d = (uint32_t)tok;
            if (greedy) {
                tok = (int32_t)top.i;
            } else {
                for (int pass = residual ? 0 : 1; pass < 2; ++pass) {
                    Best best{0.0f, 0xFFFFFFFFu};
                    for (uint32_t v = threadIdx.x; v < p.vocab; v += blockDim.x) {
                        const float y = clean(as_f32(x[v]));
                        float w = y > -INFINITY ? expf((y - top.v) / inv_t) / s : 0.0f;
                        if (pass == 0) w = fmaxf(w - (q ? q[v] : v == d ? 1.0f : 0.0f), 0.0f);
                        if (w > 0.0f) best = better(best, Best{w / p.noise[(uint64_t)b * p.vocab + v], v});
                    }
                    best = block_best(best, buf);
                    tok = (int32_t)(best.i == 0xFFFFFFFFu ? top.i : best.i);
                    if (best.i != 0xFFFFFFFFu) break;
                }
            }
        }
        if (threadIdx.x == 0) {
            p.tokens[b * (p.k + 1) + i] = tok;
            if (p.logprobs) p.logprobs[b * (p.k + 1) + i] = s > 0.0f ? (clean(as_f32(x[tok])) - top.v) / inv_t - logf(s) : -INFINITY;
        }
        if (!ok) {
            if (threadIdx.x == 0) p.accepted[b] = (int32_t)i;
            for (uint32_t j = i + 1 + threadIdx.x; j <= p.k; j += blockDim.x) {
                p.tokens[b * (p.k + 1) + j] = -1;
                if (p.logprobs) p.logprobs[b * (p.k + 1) + j] = 0.0f;
            }
            return;
        }
    }
}

}  // namespace verify
}  // namespace fp4x

using namespace fp4x;

extern "C" size_t llama_verify_workspace_size(uint32_t batch, uint32_t k, uint32_t vocab) { return 0; }

extern "C" int llama_verify_drafts(fp4x_stream_t stream, uint32_t batch, uint32_t k, uint32_t vocab, uint32_t dtype,
                                   const void *logits, uint64_t logits_stride, const float *draft_probs,
                                   const int32_t *drafts, const int32_t *draft_lens, const float *uniforms,
                                   const float *noise, const float *temperature, int32_t *accepted, int32_t *tokens,
                                   float *logprobs, void *workspace, size_t workspace_bytes) {
    FP4X_REQUIRE(dtype == FP4X_F32 || dtype == FP4X_BF16, "llama_verify_drafts: unknown dtype %u", dtype);
    FP4X_REQUIRE(vocab >= 1 && vocab < 0x7FFFFFFFu, "llama_verify_drafts: vocab must be in 1..2^31-2");
    FP4X_REQUIRE(k <= 255, "llama_verify_drafts: k %u above 255", k);
    FP4X_REQUIRE(logits_stride >= vocab, "llama_verify_drafts: logits_stride below vocab");
    if (batch == 0) return FP4X_OK;
    FP4X_REQUIRE(batch <= 65535, "llama_verify_drafts: batch %u above 65535", batch);
    FP4X_REQUIRE(logits && noise && accepted && tokens && (k == 0 || (drafts && uniforms)),
                 "llama_verify_drafts: null pointer");
    FP4X_REQUIRE(mxkv::aligned(logits, dtype == FP4X_F32 ? 4 : 2), "llama_verify_drafts: misaligned logits");
    const size_t need = llama_verify_workspace_size(batch, k, vocab);
    FP4X_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
                 "llama_verify_drafts: workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
                 workspace_bytes);
    verify::Params p{batch, k, vocab, logits, logits_stride, draft_probs, drafts, draft_lens, uniforms, noise,
                     temperature, accepted, tokens, logprobs};
    if (dtype == FP4X_F32)
        verify::verify_kernel<float><<<batch, 512, 0, (cudaStream_t)stream>>>(p);
    else
        verify::verify_kernel<__nv_bfloat16><<<batch, 512, 0, (cudaStream_t)stream>>>(p);
    return check_launch("llama_verify_drafts");
}
