// verify.cu -- verification of drafted tokens by speculative sampling with given
// random numbers.
//
// p_i = softmax(x_i / T) over the target's logits of position i.  Draft d_i is kept
// while u_i q_i(d_i) < p_i(d_i); the first rejected position samples from
// max(p - q, 0), a fully accepted draft from p_k.  Sampling by an exponential race:
// argmax_v w(v) / E(v) with E ~ Exp(1) picks v with probability w(v) / sum w, needs
// no normalised or running sums, and so does not hang on the order of a sum.
//
// Two kernels.  verify_stats_kernel reads every target row once (bound by HBM): each
// CTA takes a slice of one row and leaves (maximum, its index, sum of exp(x - max)).
// verify_choose_kernel, a cluster of eight CTAs per sequence, joins the slices, walks
// the drafts, and runs the race over the one row that decides: its logits, its draft
// probabilities and the noise, of which two thirds were not read before.  64 sequences of
// up to 5 drafts over 128256 f32 logits: 33 us (5.0 TB/s) and 25 us (98 MB), of which 6 are
// the chain before the race.  bf16 logits: 30 and 24 us, the statistics bound by their
// instructions per value (2.65 a cycle and SM; ALU 48 %, exponentials 43 %; 2.6 TB/s).
#include <cooperative_groups.h>

#include <type_traits>

#include "mxkv.cuh"

namespace fp4x {
namespace verify {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kCluster = 8;
constexpr uint32_t kMaxSlices = 32;  // slices of a row: one lane each when they are joined
constexpr float kLog2e = 1.4426950408889634f;

struct Stat {  // of a slice or row: max logit, sum of exp((x - max) / T), lowest index of the max (greedy)
    float m, s;
    uint32_t i, pad;
};

struct Params {
    uint32_t batch, k, vocab, slices;
    const void *logits;
    uint64_t stride;
    const float *probs;
    const int32_t *drafts, *lens;
    const float *u, *noise, *temp;
    int32_t *accepted, *tokens;
    float *logprobs;
    Stat *stats;  // [batch * (k + 1)][slices]
};

// NaN -> -inf (fmaxf returns the other operand), +inf -> the largest finite value.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), 3.40282347e+38f); }

__device__ __forceinline__ float load1(const float *p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

// Four consecutive values as they were loaded, past `hi` -inf: one 16- or 8-byte load where every row is
// aligned for it (VEC), else single ones.
template <typename T, bool VEC>
struct Raw {
    using Word = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
    Word w;
    __device__ __forceinline__ void load(const T *x, uint32_t v, uint32_t hi) {
        if (VEC && v + 4 <= hi) {
            w = __ldg(reinterpret_cast<const Word *>(x + v));
            return;
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (v < hi) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (v + e < hi) y[e] = load1(x + v + e);
        }
        set(y);
    }
    __device__ __forceinline__ void set(const float (&y)[4]) {
        if constexpr (sizeof(T) == 4)
            w = make_float4(y[0], y[1], y[2], y[3]);
        else
            w = make_uint2(mxkv::pack_bf16x2(y[0], y[1]), mxkv::pack_bf16x2(y[2], y[3]));
    }
    __device__ __forceinline__ void get(float (&y)[4]) const {
        if constexpr (sizeof(T) == 4) {
            y[0] = w.x, y[1] = w.y, y[2] = w.z, y[3] = w.w;
        } else {
            y[0] = __uint_as_float(w.x << 16), y[1] = __uint_as_float(w.x & 0xFFFF0000u);
            y[2] = __uint_as_float(w.y << 16), y[3] = __uint_as_float(w.y & 0xFFFF0000u);
        }
    }
};

__device__ __forceinline__ uint32_t drafts_of(const Params &p, uint32_t b) {
    return p.lens ? (uint32_t)min(max(p.lens[b], 0), (int32_t)p.k) : p.k;
}
// log2(e) / T, or log2(e) for greedy sequences (their log-probabilities are at T = 1).  Never 0: a temperature of +inf
// takes the smallest positive factor, with which a masked logit stays -inf (0 would make it NaN) and the others are alike.
__device__ __forceinline__ float factor_of(const Params &p, uint32_t b, bool &greedy) {
    const float t = p.temp ? p.temp[b] : 1.0f;
    greedy = !(t > 1e-30f);
    return greedy ? kLog2e : fmaxf(kLog2e / t, 1.401298464324817e-45f);
}

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b, float c) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    r.i = a.m > b.m || (a.m == b.m && a.i < b.i) ? a.i : b.i;
    r.s = r.m == -INFINITY ? 0.0f : a.s * exp2f((a.m - r.m) * c) + b.s * exp2f((b.m - r.m) * c);
    r.pad = 0;
    return r;
}
__device__ __forceinline__ Stat warp_join(Stat x, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stat y;
        y.m = __shfl_xor_sync(~0u, x.m, o), y.s = __shfl_xor_sync(~0u, x.s, o), y.i = __shfl_xor_sync(~0u, x.i, o);
        x = join(x, y, c);
    }
    return x;
}

// Slice of a row in units of four values.
__device__ __forceinline__ void slice_of(uint32_t vocab, uint32_t n, uint32_t s, uint32_t &lo, uint32_t &hi) {
    const uint32_t quads = (vocab + 3) / 4;
    lo = (uint32_t)((uint64_t)s * quads / n) * 4;
    hi = min(vocab, (uint32_t)((uint64_t)(s + 1) * quads / n) * 4);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) verify_stats_kernel(const __grid_constant__ Params p) {
    __shared__ Stat part[kThreads / 32];
    const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
    const uint32_t b = row / (p.k + 1), i = row % (p.k + 1);
    if (i > drafts_of(p, b)) return;
    bool greedy;
    const float c = factor_of(p, b, greedy);
    uint32_t lo, hi;
    slice_of(p.vocab, p.slices, slice, lo, hi);
    const T *x = (const T *)p.logits + (uint64_t)row * p.stride;
    Stat st{-INFINITY, 0.0f, 0xFFFFFFFFu, 0};
    // Two buffers of U loads in turn, kept as loaded until they are used: a conversion or
    // a move would wait for the data.
    constexpr uint32_t U = 4, STEP = kThreads * 4 * U;
    using R = Raw<T, VEC>;
    auto load = [&](R(&y)[U], uint32_t v0) {
#pragma unroll
        for (uint32_t j = 0; j < U; ++j) y[j].load(x, v0 + j * kThreads * 4, hi);
    };
    auto take = [&](const R(&raw)[U], uint32_t v0) {
        float y[U][4], mx = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < U; ++j) raw[j].get(y[j]);
#pragma unroll
        for (uint32_t j = 0; j < U; ++j)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) y[j][e] = clean(y[j][e]), mx = fmaxf(mx, y[j][e]);
        if (greedy && mx > st.m) {  // where the maximum is: greedy sequences only, the search costs more than the sum
#pragma unroll
            for (int j = U - 1; j >= 0; --j)
#pragma unroll
                for (int e = 3; e >= 0; --e)  // downwards: the lowest index stays
                    if (y[j][e] == mx) st.i = v0 + j * kThreads * 4 + e;
        }
        mx = fmaxf(mx, st.m);
        if (mx > -INFINITY) {
            st.s *= mxkv::ex2((st.m - mx) * c), st.m = mx;
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (uint32_t j = 0; j < U; ++j)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) s[e & 1] += mxkv::ex2((y[j][e] - st.m) * c);
            st.s += s[0] + s[1];
        }
    };
    R ya[U], yb[U];
    uint32_t v0 = lo + threadIdx.x * 4;
    load(ya, v0);
    for (; v0 < hi; v0 += 2 * STEP) {
        load(yb, v0 + STEP);
        take(ya, v0);
        load(ya, v0 + 2 * STEP);
        if (v0 + STEP < hi) take(yb, v0 + STEP);
    }
    st = warp_join(st, c);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = st;
    __syncthreads();
    if (threadIdx.x < 32) {
        st = threadIdx.x < kThreads / 32 ? part[threadIdx.x] : Stat{-INFINITY, 0.0f, 0xFFFFFFFFu, 0};
        st = warp_join(st, c);
        if (threadIdx.x == 0) p.stats[(uint64_t)row * p.slices + slice] = st;
    }
}

struct Best {
    float v;
    uint32_t i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }
__device__ __forceinline__ Best warp_best(Best x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        x = better(x, Best{__shfl_xor_sync(~0u, x.v, o), __shfl_xor_sync(~0u, x.i, o)});
    return x;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster, 1, 1)
    verify_choose_kernel(const __grid_constant__ Params p) {
    namespace cg = cooperative_groups;
    constexpr uint32_t W = kThreads / 32;
    __shared__ Stat rows[256];  // k + 1 <= 256
    __shared__ float pd[256];   // p_i(d_i) / q_i(d_i) test as 0 / 1
    __shared__ Best part[2][W], mine[2];
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t b = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t n_draft = drafts_of(p, b);
    bool greedy;
    const float c = factor_of(p, b, greedy);
    pdl_wait();
    const uint64_t first = (uint64_t)b * (p.k + 1);
    // ---- join the slices of every row, test the drafts
    for (uint32_t i = warp; i <= n_draft; i += W) {
        Stat st = lane < p.slices ? p.stats[(first + i) * p.slices + lane] : Stat{-INFINITY, 0.0f, 0xFFFFFFFFu, 0};
        st = warp_join(st, c);
        if (st.m == -INFINITY) st.i = 0;
        if (lane == 0) {
            rows[i] = st;
            bool ok = false;
            if (i < n_draft) {
                const int32_t d = p.drafts[(uint64_t)b * p.k + i];
                if ((uint32_t)d < p.vocab) {
                    if (greedy) {
                        ok = (uint32_t)d == st.i;
                    } else {
                        const float y = clean(load1((const T *)p.logits + (first + i) * p.stride + d));
                        const float pr = y > -INFINITY ? exp2f((y - st.m) * c) / st.s : 0.0f;
                        const float qr = p.probs ? p.probs[((uint64_t)b * p.k + i) * p.vocab + d] : 1.0f;
                        ok = p.u[(uint64_t)b * p.k + i] * qr < pr;
                    }
                }
            }
            pd[i] = ok ? 1.0f : 0.0f;
        }
    }
    __syncthreads();
    uint32_t at = 0;
    while (at < n_draft && pd[at] != 0.0f) ++at;
    const Stat st = rows[at];
    const T *x = (const T *)p.logits + (first + at) * p.stride;
    // ---- the race: over max(p - q, 0), and over p should that leave nothing
    Best best[2] = {{0.0f, 0xFFFFFFFFu}, {0.0f, 0xFFFFFFFFu}};
    if (!greedy && st.m > -INFINITY) {
        const bool rejected = at < n_draft;
        const float *q = rejected && p.probs ? p.probs + ((uint64_t)b * p.k + at) * p.vocab : nullptr;
        const uint32_t d = rejected && !p.probs ? (uint32_t)p.drafts[(uint64_t)b * p.k + at] : 0xFFFFFFFFu;
        const float *noise = p.noise + (uint64_t)b * p.vocab;
        const float inv = 1.0f / st.s;
        uint32_t lo, hi;
        slice_of(p.vocab, kCluster, rank, lo, hi);
        constexpr uint32_t U = 2;
        for (uint32_t v0 = lo + threadIdx.x * 4; v0 < hi; v0 += kThreads * 4 * U) {
            Raw<T, VEC> yr[U];
            Raw<float, VEC> qr[U], er[U];
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t v = v0 + j * kThreads * 4;
                yr[j].load(x, v, hi), er[j].load(noise, v, hi);
                if (q) qr[j].load(q, v, hi);
            }
            float y[U][4], qv[U][4], ev[U][4];
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                yr[j].get(y[j]), er[j].get(ev[j]);
                if (q) {
                    qr[j].get(qv[j]);
                } else {
                    qv[j][0] = qv[j][1] = qv[j][2] = qv[j][3] = 0.0f;
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < U; ++j)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t v = v0 + j * kThreads * 4 + e;
                    const float w = mxkv::ex2((clean(y[j][e]) - st.m) * c) * inv;
                    const float r = v == d ? 0.0f : fmaxf(w - qv[j][e], 0.0f);  // certain drafts: q = 1 at d
                    const float f = __fdividef(1.0f, ev[j][e]);
                    // indices ascend within a thread: a strict comparison keeps the lowest; w is 0 past the row's end
                    if (w > 0.0f && r * f > best[0].v) best[0] = Best{r * f, v};
                    if (w > 0.0f && w * f > best[1].v) best[1] = Best{w * f, v};
                }
        }
    }
#pragma unroll
    for (uint32_t z = 0; z < 2; ++z) {
        best[z] = warp_best(best[z]);
        if (lane == 0) part[z][warp] = best[z];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        Best r = part[threadIdx.x][0];
        for (uint32_t w = 1; w < W; ++w) r = better(r, part[threadIdx.x][w]);
        mine[threadIdx.x] = r;
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
        Best r[2];
#pragma unroll
        for (uint32_t z = 0; z < 2; ++z)
            r[z] = warp_best(lane < kCluster ? *cluster.map_shared_rank(&mine[z], lane) : Best{0.0f, 0xFFFFFFFFu});
        uint32_t pick = r[0].i != 0xFFFFFFFFu ? r[0].i : r[1].i != 0xFFFFFFFFu ? r[1].i : st.i;
        if (pick >= p.vocab) {  // nothing has any mass: the argmax
            pick = 0xFFFFFFFFu;
            for (uint32_t v = lane; v < p.vocab; v += 32)
                if (clean(load1(x + v)) == st.m) pick = min(pick, v);
            pick = __reduce_min_sync(~0u, pick);
        }
        const uint64_t out = (uint64_t)b * (p.k + 1);
        for (uint32_t i = lane; i <= p.k; i += 32) {
            const int32_t tok = i < at ? p.drafts[(uint64_t)b * p.k + i] : i == at ? (int32_t)pick : -1;
            p.tokens[out + i] = tok;
            if (p.logprobs) {
                float lp = 0.0f;
                if (i <= at) {
                    const Stat ri = rows[i];
                    const float y = clean(load1((const T *)p.logits + (first + i) * p.stride + tok));
                    lp = ri.s > 0.0f ? (y - ri.m) * c * 0.6931471805599453f - logf(ri.s) : -INFINITY;
                }
                p.logprobs[out + i] = lp;
            }
        }
        if (lane == 0) p.accepted[b] = (int32_t)at;
    }
    cluster.sync();  // no CTA leaves while its shared memory may be read
}

// Slices per row: enough CTAs for two waves of the 2048-thread SMs, and no slice below
// 2048 values (its join would cost as much as its reading).
inline uint32_t slices_of(uint64_t rows, uint32_t vocab) {
    const uint64_t want = (uint64_t)num_sms() * 8 / (rows ? rows : 1), most = vocab / 2048;
    const uint64_t n = want < most ? want : most;
    return (uint32_t)(n < 1 ? 1 : n > kMaxSlices ? kMaxSlices : n);
}

template <typename T, bool VEC>
int launch(cudaStream_t st, const Params &p) {
    const uint64_t ctas = (uint64_t)p.batch * (p.k + 1) * p.slices;
    verify_stats_kernel<T, VEC><<<(uint32_t)ctas, kThreads, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess)
        e = launch_pdl(verify_choose_kernel<T, VEC>, dim3(p.batch * kCluster), dim3(kThreads), 0, st, p);
    if (e != cudaSuccess) return set_error("llama_verify_drafts: %s", cudaGetErrorString(e)), FP4X_ECUDA;
    return FP4X_OK;
}

}  // namespace verify
}  // namespace fp4x

using namespace fp4x;

extern "C" size_t llama_verify_workspace_size(uint32_t batch, uint32_t k, uint32_t vocab) {
    const uint64_t rows = (uint64_t)batch * (k + 1);
    return (size_t)(rows * verify::slices_of(rows, vocab) * sizeof(verify::Stat));
}

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
    const uint32_t elem = dtype == FP4X_F32 ? 4 : 2;
    FP4X_REQUIRE(mxkv::aligned(logits, elem), "llama_verify_drafts: misaligned logits");
    const size_t need = llama_verify_workspace_size(batch, k, vocab);
    FP4X_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need,
                 "llama_verify_drafts: workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
                 workspace_bytes);
    const uint64_t rows = (uint64_t)batch * (k + 1);
    verify::Params p{batch, k, vocab, verify::slices_of(rows, vocab), logits, logits_stride, draft_probs, drafts,
                     draft_lens, uniforms, noise, temperature, accepted, tokens, logprobs,
                     (verify::Stat *)workspace};
    // four values per load where every row of every operand starts on a boundary of four
    const bool vec = vocab % 4 == 0 && logits_stride % 4 == 0 && mxkv::aligned(logits, 4 * elem) &&
                     aligned16(noise) && aligned16(draft_probs);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == FP4X_F32) return vec ? verify::launch<float, true>(st, p) : verify::launch<float, false>(st, p);
    return vec ? verify::launch<__nv_bfloat16, true>(st, p) : verify::launch<__nv_bfloat16, false>(st, p);
}
