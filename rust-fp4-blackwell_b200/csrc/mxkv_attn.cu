// mxkv_attn.cu -- attention over the MX-quantised paged cache, with an optional
// prefix that all sequences of the batch share.
//
// For query row r of sequence b and KV head h, with keys k_t and values v_t of the
// prefix and of the sequence's own pages:
//   s_t = q . k_t / sqrt(hd),  out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),
// one pass with a running maximum m and sum; partial results join as (m, l, o).
//
// attn_mx_kernel streams codes: a warp owns 16-position tiles, copies each lane's own
// codes with cp.async into a ring only that lane reads (no barrier in the loop), and
// contracts on mma.m16n8k16 f16 with the query rows as the 8 columns:
//   S^T = K q^T   in f16 per 32-block, times the block's K scale in f32;
//   O^T += V^T P^T in bf16 with the V scale of (position, block) multiplied into P^T.
// Codes are exact in f16 and bf16 and scales are powers of two, so the only roundings
// are P to two bf16 terms (16 bits; bf16 queries are exact in f16), or q to an f16 pair
// and P to three bf16 terms (f32 queries: 22 and 24 bits).  P takes bf16, not f16: its
// products with the scales, and probabilities far below the maximum, need the range (a
// dimension in which the largest position's code is 0 is made of those alone).
#include "mxkv.cuh"

namespace fp4x {
namespace mxkv {

constexpr uint32_t kWarps = 8;                 // warps per CTA
constexpr uint32_t kChunk = 16 * kWarps;       // positions of one step of a CTA
constexpr float kNoMax = -3.0e38f;             // running maximum before the first score
constexpr float kLag = 8.0f;                   // how far (in powers of two) a score may pass the running maximum

// One set of rows over one set of pages: the sequences of a batch over their own
// pages (n_seq = batch), or all rows of the batch over the shared prefix (n_seq = 1).
struct Job {
    uint32_t n_seq, rows, row_tiles, ctas;  // sequences, query rows per (sequence, KV head), tiles of them, grid
    const int32_t *pages, *lens;            // lens null: every sequence holds max_len positions
    uint32_t table_stride, max_len;
    float *slots;      // 2 per CTA: its part of a segment that began before it, and of one that it began
    float *row_slots;  // one per output row for segments of one CTA (null: written to out)
};

struct AttnParams {
    Cache c;
    uint32_t n_heads, group, q_len;
    const void *q;
    uint64_t q_stride;
    void *out;
    float scale;
    Job own, prefix;
};

__device__ __forceinline__ uint32_t seq_len(const Job &j, uint32_t s) {
    return j.lens ? (uint32_t)min(max(j.lens[s], 0), (int32_t)j.max_len) : j.max_len;
}
__device__ __forceinline__ uint32_t seq_chunks(const Job &j, uint32_t s) { return (seq_len(j, s) + kChunk - 1) / kChunk; }

// The work is a row of segments (sequence, row tile, head), dealt to the CTAs in equal
// contiguous parts so that ragged lengths load all CTAs alike.  A segment costs its
// chunks and kOpen more for reading its queries, filling the ring and joining the warps
// (measured with lengths up to 8192 of 64 sequences: without it the CTAs that got the
// short ones took 1.25 times the mean).  CTA c starts at cost floor(c * total / ctas).
constexpr uint32_t kOpen = 2;
__device__ __forceinline__ uint32_t seq_cost(const Job &j, uint32_t s) {
    const uint32_t n = seq_chunks(j, s);
    return n ? n + kOpen : 0;
}
__device__ __forceinline__ uint64_t cta_start(uint64_t c, uint64_t total, uint32_t ctas) { return c * total / ctas; }
__device__ __forceinline__ uint32_t cta_of(uint64_t at, uint64_t total, uint32_t ctas) {
    return (uint32_t)(((at + 1) * ctas - 1) / total);
}

// Block-wide scan of the sequences' costs (each `per` segments): the total, and the
// sequence in which CTA x starts (by_cta) or the cost before sequence x.
struct Located {
    uint64_t total, first;  // cost in all, cost before the located sequence
    uint32_t seq;
};
template <uint32_t THREADS>
__device__ Located locate(const Job &j, uint32_t per, bool by_cta, uint64_t x, uint64_t (&buf)[THREADS / 32 + 1],
                          Located &res) {
    const uint32_t each = (j.n_seq + THREADS - 1) / THREADS, s0 = min(threadIdx.x * each, j.n_seq),
                   s1 = min(s0 + each, j.n_seq);
    uint64_t mine = 0;
    for (uint32_t s = s0; s < s1; ++s) mine += (uint64_t)seq_cost(j, s) * per;
    uint64_t scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint64_t v = __shfl_up_sync(~0u, scan, o);
        if ((threadIdx.x & 31) >= (uint32_t)o) scan += v;
    }
    if ((threadIdx.x & 31) == 31) buf[threadIdx.x / 32] = scan;
    __syncthreads();
    uint64_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; ++w) {
        if (w < threadIdx.x / 32) before += buf[w];
        total += buf[w];
    }
    before += scan - mine;
    const uint64_t at = by_cta ? cta_start(x, total, j.ctas) : 0;
    if (threadIdx.x == 0) res = Located{total, 0, 0};
    __syncthreads();
    for (uint32_t s = s0; s < s1; ++s) {
        const uint64_t n = (uint64_t)seq_cost(j, s) * per;
        if (by_cta ? (before <= at && at < before + n) : s == x) res.first = before, res.seq = s;
        before += n;
    }
    __syncthreads();
    return res;
}

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, uint32_t size, uint32_t bytes) {
    if (size == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else if (size == 8)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four E4M3 codes of a word -> f16x2 of codes (0,1) and (2,3).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t bmul2(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
// Of values with at most eight significant bits (codes): the upper halves of their f32.
__device__ __forceinline__ uint32_t f16x2_to_bf16x2(uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
}
// Four E8M0 bytes -> bf16x2 of bytes (0,1) and (2,3).
__device__ __forceinline__ void e8m0x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.bf16x2.ue8m0x2 %0, l;\n\tcvt.rn.bf16x2.ue8m0x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
// Two E8M0 bytes (in the low half of w) -> two f32.
__device__ __forceinline__ void e8m0x2_to_f32(uint32_t w, float &lo, float &hi) {
    uint32_t y;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, l;\n\t}" : "=r"(y) : "r"(w));
    lo = __uint_as_float(y << 16), hi = __uint_as_float(y & 0xFFFF0000u);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Shapes of the streaming kernel's ring.  A tile is 16 positions; lane (g, t) copies
//   K: positions g and g + 8, the two chunks of each that hold its columns (t and t + 4,
//      or 2t and 2t + 1 where two chunks make one 16- or 8-byte copy);
//   V: positions 2t, 2t + 1, 2t + 8, 2t + 9, chunk g;
//   the scales of those positions.
template <uint32_t FMT, uint32_t HD>
struct Ring {
    static constexpr uint32_t NB = HD / 32, CHUNK = Row<FMT, HD>::CHUNK, CW = CHUNK / 4;
    static constexpr bool PAIR = CHUNK < 16;  // both K chunks of a position in one copy
    static constexpr uint32_t KCOPY = PAIR ? 2 * CHUNK : CHUNK, KN = PAIR ? 2 : 4;
    static constexpr uint32_t VS = 2 * NB;    // bytes of two positions' V scales
    static constexpr uint32_t LANE = KN * KCOPY + 4 * CHUNK + 2 * 4 + 2 * VS;
    static constexpr uint32_t STAGE = 32 * LANE;
    static constexpr uint32_t K_OFF = 0, V_OFF = 32 * KN * KCOPY, VS_OFF = V_OFF + 32 * 4 * CHUNK,
                              KS_OFF = VS_OFF + 32 * 2 * VS;
    // two CTAs per SM share 227 KB with their 16 or 32 KB merge buffers
    static constexpr uint32_t STAGES = STAGE > 3000 ? 2 : STAGE > 2000 ? 3 : 4;
};

template <uint32_t FMT, uint32_t HD, uint32_t NQ, bool F32>
struct Tile {
    using R = Ring<FMT, HD>;
    static constexpr uint32_t NB = HD / 32, MT = HD / 16, CW = R::CW, TERMS = F32 ? 2 : 1, PTERMS = F32 ? 3 : 2;
    static constexpr bool QREG = NQ == 1 && !F32;
    static constexpr uint32_t Q_BYTES = TERMS * 2 * NB * NQ * 32 * 8;  // [term][half][block][column tile][lane] 8 B
    static constexpr uint32_t MERGE_BYTES = kWarps * MT * 32 * 16;
    static constexpr uint32_t SMEM = kWarps * R::STAGES * R::STAGE + Q_BYTES + MERGE_BYTES;
    static constexpr uint32_t MIN_CTAS = NQ * HD <= 128 ? 2 : 1;

    float o[MT][NQ][4];
    float m[NQ][2], l[NQ][2];
    uint2 q[QREG ? 2 * NB : 1];

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (uint32_t i = 0; i < MT; ++i)
#pragma unroll
            for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) o[i][n][j] = 0.0f;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) m[n][0] = m[n][1] = kNoMax, l[n][0] = l[n][1] = 0.0f;
    }
};

template <uint32_t FMT, uint32_t HD>
__device__ __forceinline__ void issue_tile(const Cache &c, uint32_t ring, int32_t page, uint32_t head, uint32_t row0,
                                           uint32_t left, uint32_t lane) {
    using R = Ring<FMT, HD>;
    constexpr uint32_t B = Row<FMT, HD>::BYTES, NB = HD / 32;
    const uint32_t g = lane >> 2, t = lane & 3;
    const bool ok = (uint32_t)page < c.n_pages;
    const uint32_t p = ok ? (uint32_t)page : 0;
    const uint32_t n = ok ? left : 0;  // positions of the tile that exist
    const uint64_t co = code_off<FMT, HD>(c, p, head, row0), so = scale_off<HD>(c, p, head, row0);
    const uint8_t *k = c.k + co, *v = c.v + co, *ks = c.ks + so, *vs = c.vs + so;
#pragma unroll
    for (uint32_t i = 0; i < R::KN; ++i) {
        const uint32_t pos = g + 8 * (R::PAIR ? i : i / 2);
        const uint32_t off = R::PAIR ? t * R::KCOPY : (t + 4 * (i & 1)) * R::CHUNK;
        cp_async(ring + R::K_OFF + (i * 32 + lane) * R::KCOPY, k + pos * B + off, R::KCOPY, n ? R::KCOPY : 0);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t pos = 2 * t + (i & 1) + 8 * (i / 2);
        cp_async(ring + R::V_OFF + (i * 32 + lane) * R::CHUNK, v + pos * B + g * R::CHUNK, R::CHUNK,
                 pos < n ? R::CHUNK : 0);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t pos = 2 * t + 8 * i;
        cp_async(ring + R::VS_OFF + (i * 32 + lane) * R::VS, vs + pos * NB, R::VS,
                 pos < n ? min(n - pos, 2u) * NB : 0);
        const uint32_t kp = (g + 8 * i) * NB & ~3u;  // 64-wide heads: the two rows of a 4-byte piece
        cp_async(ring + R::KS_OFF + (i * 32 + lane) * 4, ks + kp, 4, n ? 4 : 0);
    }
}

template <uint32_t N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(addr));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// One block's V^T of a tile as the two 16-row A operands: dimensions 4g + 2j (row g)
// and 4g + 2j + 1 (row g + 8), columns = positions.
template <uint32_t FMT, uint32_t HD>
__device__ __forceinline__ void value_fragments(const uint32_t (&vw)[4][Ring<FMT, HD>::CW], uint32_t b,
                                                uint32_t (&a)[2][4]) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        uint32_t f[2][2];
        if constexpr (FMT == FMT_FP8) {
            const uint32_t x = vw[2 * h][b], y = vw[2 * h + 1][b];
            e4m3x4_to_f16(__byte_perm(x, y, 0x5140), f[0][0], f[0][1]);
            e4m3x4_to_f16(__byte_perm(x, y, 0x7362), f[1][0], f[1][1]);
        } else {
            const uint32_t x = vw[2 * h][b / 2], y = vw[2 * h + 1][b / 2];
            const uint32_t even = (x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u);
            const uint32_t odd = ((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u);
            uint32_t fe[4], fo[4];
            decode_word_f16(even, fe), decode_word_f16(odd, fo);
            f[0][0] = fe[2 * (b & 1)], f[0][1] = fo[2 * (b & 1)];
            f[1][0] = fe[2 * (b & 1) + 1], f[1][1] = fo[2 * (b & 1) + 1];
        }
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) a[j][2 * h + i] = f16x2_to_bf16x2(f[j][i]);
    }
}

// One tile from the ring into the running softmax.  `left` positions of the tile
// exist (0: a page outside the cache); lim[n][j] - first is the column's limit.
template <uint32_t FMT, uint32_t HD, uint32_t NQ, bool F32>
__device__ __forceinline__ void take_tile(Tile<FMT, HD, NQ, F32> &T, uint32_t ring, uint32_t qs, uint32_t left,
                                          bool masked, const int32_t *lim, int32_t first, const float *rf,
                                          uint32_t lane) {
    using R = Ring<FMT, HD>;
    using TT = Tile<FMT, HD, NQ, F32>;
    constexpr uint32_t NB = HD / 32, CW = R::CW, TERMS = TT::TERMS;
    const uint32_t g = lane >> 2;
    // ---- S^T = K q^T
    float s[NQ][4];
#pragma unroll
    for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) s[n][j] = 0.0f;
    {
        uint32_t kw[2][2 * CW];  // [position g, g + 8][chunk half][word]
        if constexpr (R::PAIR) {
            lds_words<2 * CW>(ring + R::K_OFF + lane * R::KCOPY, kw[0]);
            lds_words<2 * CW>(ring + R::K_OFF + (32 + lane) * R::KCOPY, kw[1]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                uint32_t w[CW];
                lds_words<CW>(ring + R::K_OFF + (i * 32 + lane) * R::KCOPY, w);
#pragma unroll
                for (uint32_t j = 0; j < CW; ++j) kw[i / 2][(i & 1) * CW + j] = w[j];
            }
        }
        uint32_t sc[2][1];
        lds_words<1>(ring + R::KS_OFF + lane * 4, sc[0]);
        lds_words<1>(ring + R::KS_OFF + (32 + lane) * 4, sc[1]);
        float ks[2][NB];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            if constexpr (NB == 4) {
                e8m0x2_to_f32(sc[i][0], ks[i][0], ks[i][1]);
                e8m0x2_to_f32(sc[i][0] >> 16, ks[i][2], ks[i][3]);
            } else {
                e8m0x2_to_f32(g & 1 ? sc[i][0] >> 16 : sc[i][0], ks[i][0], ks[i][1]);
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            uint32_t a[2][4];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    if constexpr (FMT == FMT_FP8) {
                        e4m3x4_to_f16(kw[i][h * CW + b], a[h][i], a[h][2 + i]);
                    } else {
                        uint32_t f[4];
                        decode_word_f16(kw[i][h * CW + b / 2], f);
                        a[h][i] = f[2 * (b & 1)], a[h][2 + i] = f[2 * (b & 1) + 1];
                    }
                }
#pragma unroll
            for (uint32_t n = 0; n < NQ; ++n) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t z = 0; z < TERMS; ++z)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        uint32_t qf[2];
                        if constexpr (TT::QREG)
                            qf[0] = T.q[h * NB + b].x, qf[1] = T.q[h * NB + b].y;
                        else
                            lds_words<2>(qs + ((((z * 2 + h) * NB + b) * NQ + n) * 32 + lane) * 8, qf);
                        mma_f16_16816(acc, a[h], qf[0], qf[1], acc);
                    }
                s[n][0] += acc[0] * ks[0][b], s[n][1] += acc[1] * ks[0][b];
                s[n][2] += acc[2] * ks[1][b], s[n][3] += acc[3] * ks[1][b];
            }
        }
    }
    // ---- running maximum, probabilities
    bool above = false;
#pragma unroll
    for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            s[n][j] *= rf[n * 2 + (j & 1)];
            if (masked) {
                const int32_t pos = (int32_t)(g + 8 * (j / 2));
                if (pos >= (int32_t)left || first + pos >= lim[n * 2 + (j & 1)]) s[n][j] = -INFINITY;
            }
            above |= s[n][j] > T.m[n][j & 1] + kLag;
        }
    if (__any_sync(~0u, above)) {
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                float x = fmaxf(s[n][j], s[n][2 + j]);
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                x = fmaxf(x, T.m[n][j]);
                const float f = ex2(T.m[n][j] - x);
                T.m[n][j] = x;
                T.l[n][j] *= f;
#pragma unroll
                for (uint32_t i = 0; i < TT::MT; ++i) T.o[i][n][j] *= f, T.o[i][n][2 + j] *= f;
            }
    }
    uint32_t p[TT::PTERMS][NQ][2];
#pragma unroll
    for (uint32_t n = 0; n < NQ; ++n) {
        float x[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            x[j] = ex2(s[n][j] - T.m[n][j & 1]);
            T.l[n][j & 1] += x[j];
        }
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t z = 0; z < TT::PTERMS; ++z) {
                const uint32_t y = pack_bf16x2(x[2 * h], x[2 * h + 1]);
                p[z][n][h] = movmatrix(y);
                x[2 * h] -= __uint_as_float(y << 16), x[2 * h + 1] -= __uint_as_float(y & 0xFFFF0000u);
            }
    }
    // ---- O^T += V^T (P scaled)^T
    uint32_t vw[4][CW], sc[2][NB];  // scales of positions (2t, 2t + 1) and (2t + 8, 2t + 9) as bf16 pairs
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) lds_words<CW>(ring + R::V_OFF + (i * 32 + lane) * R::CHUNK, vw[i]);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t w[R::VS / 4];
        lds_words<R::VS / 4>(ring + R::VS_OFF + (i * 32 + lane) * R::VS, w);
        e8m0x4_to_bf16(NB == 4 ? __byte_perm(w[0], w[R::VS / 4 - 1], 0x5140) : __byte_perm(w[0], 0, 0x3120), sc[i][0],
                       sc[i][1]);
        if constexpr (NB == 4) e8m0x4_to_bf16(__byte_perm(w[0], w[R::VS / 4 - 1], 0x7362), sc[i][2], sc[i][3]);
    }
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
        uint32_t a[2][4];
        value_fragments<FMT, HD>(vw, b, a);
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t z = 0; z < TT::PTERMS; ++z) {
                const uint32_t b0 = bmul2(p[z][n][0], sc[0][b]), b1 = bmul2(p[z][n][1], sc[1][b]);
                mma_bf16_16816(T.o[2 * b][n], a[0], b0, b1, T.o[2 * b][n]);
                mma_bf16_16816(T.o[2 * b + 1][n], a[1], b0, b1, T.o[2 * b + 1][n]);
            }
    }
}

// Row of q / out behind row r of a segment: its token and its head.
struct RowAt {
    uint32_t token, head, step;  // token = sequence * q_len + step
};
__device__ __forceinline__ RowAt row_at(const AttnParams &p, bool prefix, uint32_t seq, uint32_t kvh, uint32_t r) {
    const uint32_t tok = r / p.group;
    return RowAt{prefix ? tok : seq * p.q_len + tok, kvh * p.group + r % p.group, prefix ? 0u : tok};
}

template <typename T>
__device__ __forceinline__ void store2(T *p, float x, float y);
template <>
__device__ __forceinline__ void store2<float>(float *p, float x, float y) {
    *reinterpret_cast<float2 *>(p) = make_float2(x, y);
}
template <>
__device__ __forceinline__ void store2<__nv_bfloat16>(__nv_bfloat16 *p, float x, float y) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(x, y);
}

template <uint32_t FMT, uint32_t HD, uint32_t NQ, typename T>
__global__ void __launch_bounds__(kWarps * 32, Tile<FMT, HD, NQ, sizeof(T) == 4>::MIN_CTAS)
    attn_mx_kernel(const __grid_constant__ AttnParams p, bool prefix) {
    constexpr bool F32 = sizeof(T) == 4;
    using TT = Tile<FMT, HD, NQ, F32>;
    using R = Ring<FMT, HD>;
    constexpr uint32_t NB = HD / 32, ROWS = 8 * NQ;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t scan[kWarps + 1];
    __shared__ Located where;
    __shared__ float sm[kWarps][ROWS], sl[kWarps][ROWS], top[ROWS], sum[ROWS], rowf[ROWS];
    __shared__ int32_t limit[ROWS];
    const Job &job = prefix ? p.prefix : p.own;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * R::STAGES * R::STAGE;
    uint8_t *qbuf = smem + kWarps * R::STAGES * R::STAGE;
    float4 *merge = reinterpret_cast<float4 *>(qbuf + TT::Q_BYTES);
    const uint32_t per = p.c.n_kv * job.row_tiles;

    const Located loc = locate<kWarps * 32>(job, per, true, blockIdx.x, scan, where);
    uint64_t at = cta_start(blockIdx.x, loc.total, job.ctas);
    const uint64_t end = cta_start(blockIdx.x + 1, loc.total, job.ctas);
    uint32_t seq = loc.seq;
    uint64_t seq_first = loc.first;
    while (at < end) {
        uint32_t cost = seq_cost(job, seq);
        while (at >= seq_first + (uint64_t)cost * per) {
            seq_first += (uint64_t)cost * per;
            cost = seq_cost(job, ++seq);
        }
        const uint32_t len = seq_len(job, seq), chunks = cost - kOpen;
        const uint64_t in_seq = at - seq_first;
        const uint32_t unit = (uint32_t)(in_seq / cost), x0 = (uint32_t)(in_seq - (uint64_t)unit * cost);
        const uint32_t x1 = (uint32_t)min((uint64_t)cost, (uint64_t)x0 + (end - at));
        at += x1 - x0;
        const uint32_t c0 = max(x0, kOpen) - kOpen, c1 = max(x1, kOpen) - kOpen;
        if (c0 == c1) continue;
        const uint32_t head = unit % p.c.n_kv, r0 = unit / p.c.n_kv * ROWS;
        const uint32_t rows = min(ROWS, job.rows - r0);
        const int32_t *table = job.pages + (uint64_t)seq * job.table_stride;

        // this warp's tiles: c * kWarps + warp for c in [c0, c1), those that start below len
        const uint32_t tiles = (len + 15) / 16;
        uint32_t n_tiles = c1 - c0;
        while (n_tiles && (c0 + n_tiles - 1) * kWarps + warp >= tiles) --n_tiles;
        int32_t ids = 0;   // lane j: page of tile (j modulo 32)
        uint32_t bad = 0;  // bit s: the page of the tile in stage s is outside the cache
        auto load_ids = [&](uint32_t j0) {
            const uint32_t j = j0 + lane;
            ids = j < n_tiles ? table[((c0 + j) * kWarps + warp) * 16 >> p.c.page_shift] : 0;
        };
        auto issue = [&](uint32_t j) {
            if ((j & 31) == 0 && j < n_tiles) load_ids(j);
            if (j < n_tiles) {
                const uint32_t first = ((c0 + j) * kWarps + warp) * 16;
                const int32_t page = __shfl_sync(~0u, ids, j & 31);
                issue_tile<FMT, HD>(p.c, ring + j % R::STAGES * R::STAGE, page, head,
                                    first & ((1u << p.c.page_shift) - 1), min(16u, len - first), lane);
                const bool out = (uint32_t)page >= p.c.n_pages;
                bad = (bad & ~(1u << j % R::STAGES)) | ((uint32_t)out << j % R::STAGES);
                if (out && lane == 0) raise_device_error(DEVERR_BAD_ARG);
            }
            cp_async_commit();
        };
        __syncthreads();  // the previous segment's buffers are free
#pragma unroll
        for (uint32_t j = 0; j < R::STAGES; ++j) issue(j);
        // ---- query rows: scaled to a maximum in [2^14, 2^15), f16 (and the remainder's f16), fragment order
        for (uint32_t r = warp; r < ROWS; r += kWarps) {
            float x[HD / 32], amax = 0.0f;
            const RowAt ra = row_at(p, prefix, seq, head, r0 + min(r, rows - 1));
            const T *src = (const T *)p.q + (uint64_t)ra.token * p.q_stride + ra.head * HD;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) x[b] = r < rows ? (float)src[b * 32 + lane] : 0.0f, amax = fmaxf(amax, fabsf(x[b]));
            amax = warp_max(amax);
            const int e = amax > 0.0f ? max(-112, min(127, (int)(__float_as_uint(amax) >> 23) - 127)) : 0;
            const float up = pow2(14 - e);
            if (lane == 0) {
                rowf[r] = p.scale * pow2(max(e - 14, -126));
                limit[r] = prefix ? (int32_t)len
                                  : (int32_t)len - (int32_t)p.q_len + 1 + (int32_t)ra.step;
            }
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                // dimension 32 b + lane: chunk c = lane / 4, code i = lane % 4 -> lane t, half, position in the fragment
                const uint32_t c = lane >> 2, i = lane & 3;
                const uint32_t tt = R::PAIR ? c / 2 : c & 3, h = R::PAIR ? c & 1 : c >> 2;
                float y = x[b] * up;
#pragma unroll
                for (uint32_t z = 0; z < TT::TERMS; ++z) {
                    const __half hy = __float2half_rn(y);
                    y -= __half2float(hy);
                    const uint32_t idx = ((((z * 2 + h) * NB + b) * NQ + r / 8) * 32 + (r % 8) * 4 + tt) * 4 + i;
                    reinterpret_cast<__half *>(qbuf)[idx] = hy;
                }
            }
        }
        __syncthreads();
        TT tile;
        tile.reset();
        float rf[2 * NQ];
        int32_t lim[2 * NQ], lowest = 0x7FFFFFFF;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                rf[n * 2 + j] = rowf[n * 8 + 2 * t + j];
                lim[n * 2 + j] = limit[n * 8 + 2 * t + j];
                lowest = min(lowest, lim[n * 2 + j]);
            }
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, 1));
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, 2));
        if constexpr (TT::QREG) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * NB; ++i) tile.q[i] = reinterpret_cast<const uint2 *>(qbuf)[i * 32 + lane];
        }
        uint32_t stage = 0;
        for (uint32_t j = 0; j < n_tiles; ++j) {
            const uint32_t first = ((c0 + j) * kWarps + warp) * 16;
            cp_async_wait<R::STAGES - 1>();
            uint32_t left = min(16u, len - first);
            bool masked = (int32_t)(first + 16) > lowest || left < 16;
            if ((bad >> stage) & 1) left = 0, masked = true;
            take_tile<FMT, HD, NQ, F32>(tile, ring + stage * R::STAGE, smem_u32(qbuf), left, masked, lim,
                                        (int32_t)first, rf, lane);
            stage = stage + 1 == R::STAGES ? 0 : stage + 1;
            issue(j + R::STAGES);
        }
        // ---- join the warps
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                float l = tile.l[n][j];
                l += __shfl_xor_sync(~0u, l, 4);
                l += __shfl_xor_sync(~0u, l, 8);
                l += __shfl_xor_sync(~0u, l, 16);
                if (g == 0) sm[warp][n * 8 + 2 * t + j] = tile.m[n][j], sl[warp][n * 8 + 2 * t + j] = l;
            }
        __syncthreads();
        if (threadIdx.x < ROWS) {
            float mx = kNoMax, l = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w][threadIdx.x]);
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) l += sl[w][threadIdx.x] * exp2f(sm[w][threadIdx.x] - mx);
            top[threadIdx.x] = mx, sum[threadIdx.x] = l;
        }
        __syncthreads();
        const bool whole = c0 == 0 && c1 == chunks;
        float *slot = nullptr;
        if (!whole) {
            slot = job.slots + (uint64_t)(2 * blockIdx.x + (c0 == 0)) * ROWS * (HD + 2);
            if (threadIdx.x < ROWS) slot[2 * threadIdx.x] = top[threadIdx.x], slot[2 * threadIdx.x + 1] = sum[threadIdx.x];
            slot += 2 * ROWS;
        } else if (job.row_slots && threadIdx.x < rows) {
            const RowAt ra = row_at(p, prefix, seq, head, r0 + threadIdx.x);
            float *rs = job.row_slots + ((uint64_t)ra.token * p.n_heads + ra.head) * (HD + 2);
            rs[HD] = top[threadIdx.x], rs[HD + 1] = sum[threadIdx.x];
        }
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) {
            if (n) __syncthreads();
            float f[2];
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) f[j] = exp2f(tile.m[n][j] - top[n * 8 + 2 * t + j]);
#pragma unroll
            for (uint32_t i = 0; i < TT::MT; ++i)
                merge[(warp * TT::MT + i) * 32 + lane] = make_float4(tile.o[i][n][0] * f[0], tile.o[i][n][1] * f[1],
                                                                     tile.o[i][n][2] * f[0], tile.o[i][n][3] * f[1]);
            __syncthreads();
            if (warp < TT::MT) {
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) {
                    const float4 x = merge[(w * TT::MT + warp) * 32 + lane];
                    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
                }
                const uint32_t d = 32 * (warp / 2) + 4 * g + 2 * (warp & 1);
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    const uint32_t r = n * 8 + 2 * t + j;
                    if (r >= rows) continue;
                    const float y0 = j ? acc.y : acc.x, y1 = j ? acc.w : acc.z;
                    if (!whole) {
                        store2<float>(slot + r * HD + d, y0, y1);
                        continue;
                    }
                    const RowAt ra = row_at(p, prefix, seq, head, r0 + r);
                    const uint64_t row = (uint64_t)ra.token * p.n_heads + ra.head;
                    if (job.row_slots) {
                        store2<float>(job.row_slots + row * (HD + 2) + d, y0, y1);
                    } else {
                        const float inv = sum[r] > 0.0f ? 1.0f / sum[r] : sum[r] == 0.0f ? 0.0f : sum[r];
                        store2<T>((T *)p.out + row * HD + d, y0 * inv, y1 * inv);
                    }
                }
            }
        }
    }
}

// Joins the partial results of one output row: those of the CTAs that shared its
// segment, and with a prefix those of both jobs.  A CTA of HD threads per row, each
// warp takes every fourth (second) partial.
template <uint32_t HD, typename T>
__global__ void __launch_bounds__(HD) attn_mx_join_kernel(const __grid_constant__ AttnParams p, uint32_t tile_rows) {
    constexpr uint32_t W = HD / 32;
    __shared__ uint64_t scan[W + 1];
    __shared__ Located where;
    __shared__ float sm[W], sl[W], so[W][HD];
    pdl_wait();
    const uint32_t row = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t token = row / p.n_heads, head = row % p.n_heads, kvh = head / p.group;
    float m = kNoMax, l = 0.0f, o[W];  // lane holds dimensions lane * W ..
#pragma unroll
    for (uint32_t i = 0; i < W; ++i) o[i] = 0.0f;
    auto take = [&](const float *ml, const float *po) {
        const float pm = ml[0], pl = ml[1], mn = fmaxf(m, pm), f0 = exp2f(m - mn), f1 = exp2f(pm - mn);
        l = l * f0 + pl * f1;
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) o[i] = o[i] * f0 + po[lane * W + i] * f1;
        m = mn;
    };
    bool direct = false;
#pragma unroll 1
    for (uint32_t which = 0; which < 2; ++which) {
        const Job &job = which ? p.prefix : p.own;
        if (which && !job.ctas) break;
        const uint32_t seq = which ? 0 : token / p.q_len;
        const uint32_t r = which ? token * p.group + head % p.group : token % p.q_len * p.group + head % p.group;
        if (job.ctas == 0) {  // no positions of their own in the whole batch
            direct = false;
            continue;
        }
        const uint32_t per = p.c.n_kv * job.row_tiles;
        const Located loc = locate<HD>(job, per, false, seq, scan, where);
        const uint32_t chunks = seq_chunks(job, seq);
        if (chunks == 0) continue;
        const uint64_t first = loc.first + (uint64_t)(r / tile_rows * p.c.n_kv + kvh) * (chunks + kOpen) + kOpen;
        const uint32_t ca = cta_of(first, loc.total, job.ctas), cb = cta_of(first + chunks - 1, loc.total, job.ctas);
        if (ca == cb) {
            if (!job.row_slots) {
                direct = true;
            } else if (warp == 0) {
                const float *rs = job.row_slots + (uint64_t)row * (HD + 2);
                take(rs + HD, rs);
            }
            continue;
        }
        for (uint32_t c = ca + warp; c <= cb; c += W) {
            if (c != ca && cta_start(c, loc.total, job.ctas) == cta_start(c + 1, loc.total, job.ctas)) continue;
            const float *slot = job.slots + (uint64_t)(2 * c + (c == ca)) * tile_rows * (HD + 2);
            take(slot + 2 * (r % tile_rows), slot + 2 * tile_rows + r % tile_rows * HD);
        }
    }
    if (direct) return;
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (uint32_t i = 0; i < W; ++i) so[warp][lane * W + i] = o[i];
    __syncthreads();
    float mx = kNoMax, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) mx = fmaxf(mx, sm[w]);
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        const float f = exp2f(sm[w] - mx);
        sum += sl[w] * f, acc += so[w][threadIdx.x] * f;
    }
    ((T *)p.out)[(uint64_t)row * HD + threadIdx.x] = (T)(sum == 0.0f ? 0.0f : acc / sum);
}

// ---------------------------------------------------------------- host
// Columns of a row tile: 8 per mma; up to 32 rows share one read of the codes.
inline uint32_t column_tiles(uint64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

struct Plan {
    uint32_t nq;                   // column tiles of both jobs
    uint32_t own_ctas, prefix_ctas;
    uint64_t own_slots, prefix_slots, row_slots;  // floats
};
inline uint32_t min_ctas(uint32_t hd, uint32_t nq) { return nq * hd <= 128 ? 2 : 1; }

Plan make_plan(uint32_t n_kv, uint32_t hd, uint32_t batch, uint32_t n_heads, uint32_t q_len, uint32_t prefix_len,
               uint32_t max_len) {
    Plan pl = {};
    const uint64_t group = n_heads / n_kv, rows = group * q_len, all = rows * batch;
    pl.nq = column_tiles(prefix_len ? all : rows);
    const uint32_t sms = (uint32_t)num_sms(), slots = sms * min_ctas(hd, pl.nq);
    const uint64_t tr = 8 * pl.nq;
    auto chunks = [](uint32_t n) { return ((uint64_t)n + kChunk - 1) / kChunk; };  // CTAs beyond the chunks would idle
    const uint64_t own = chunks(max_len) * batch * n_kv * ((rows + tr - 1) / tr);
    pl.own_ctas = (uint32_t)(own < slots ? own : slots);
    pl.own_slots = 2ull * pl.own_ctas * tr * (hd + 2);
    if (prefix_len) {
        const uint64_t pre = chunks(prefix_len) * n_kv * ((all + tr - 1) / tr);
        pl.prefix_ctas = (uint32_t)(pre < slots ? pre : slots);
        pl.prefix_slots = 2ull * pl.prefix_ctas * tr * (hd + 2);
        pl.row_slots = (uint64_t)batch * q_len * n_heads * (hd + 2);
    }
    return pl;
}

template <uint32_t FMT, uint32_t HD, uint32_t NQ, typename T>
int launch_job(const char *who, cudaStream_t st, const AttnParams &p, bool prefix) {
    using TT = Tile<FMT, HD, NQ, sizeof(T) == 4>;
    auto kernel = attn_mx_kernel<FMT, HD, NQ, T>;
    static bool ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TT::SMEM);
        if (e != cudaSuccess) return set_error("%s: %s", who, cudaGetErrorString(e)), FP4X_ECUDA;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    kernel<<<(prefix ? p.prefix : p.own).ctas, kWarps * 32, TT::SMEM, st>>>(p, prefix);
    return check_launch(who);
}

template <uint32_t FMT, uint32_t HD, typename T>
int launch_all(const char *who, cudaStream_t st, const AttnParams &p, uint32_t nq, uint64_t rows) {
    int rc = FP4X_OK;
    for (int prefix = 1; prefix >= 0 && rc == FP4X_OK; --prefix) {
        if (!(prefix ? p.prefix : p.own).ctas) continue;
        rc = nq == 1   ? launch_job<FMT, HD, 1, T>(who, st, p, prefix)
             : nq == 2 ? launch_job<FMT, HD, 2, T>(who, st, p, prefix)
                       : launch_job<FMT, HD, 4, T>(who, st, p, prefix);
    }
    if (rc != FP4X_OK) return rc;
    const cudaError_t e = launch_pdl(attn_mx_join_kernel<HD, T>, dim3((uint32_t)rows), dim3(HD), 0, st, p, 8 * nq);
    if (e != cudaSuccess) return set_error("%s: %s", who, cudaGetErrorString(e)), FP4X_ECUDA;
    return check_launch(who);
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
    FP4X_REQUIRE(rows <= 0x3FFFFFFFull, "%s: too many query rows", who);
    FP4X_REQUIRE(q && out && lens, "%s: null pointer", who);
    FP4X_REQUIRE(max_len == 0 || page_table, "%s: null page table", who);
    FP4X_REQUIRE(prefix_len == 0 || prefix_pages, "%s: null prefix pages", who);
    FP4X_REQUIRE(((uint64_t)max_len + cache->page_size - 1) / cache->page_size <= table_stride,
                 "%s: table_stride %u holds fewer than max_len %u positions", who, table_stride, max_len);
    FP4X_REQUIRE(aligned(q, 16) && aligned(out, 16) && q_stride % (dtype == FP4X_F32 ? 4 : 8) == 0,
                 "%s: rows of q and out must be 16-byte aligned", who);
    FP4X_REQUIRE(q_stride >= (uint64_t)n_heads * hd, "%s: q_stride below n_heads * head_dim", who);
    const Plan pl = make_plan(p.c.n_kv, hd, batch, n_heads, q_len, prefix_len, max_len);
    const size_t need = (pl.own_slots + pl.prefix_slots + pl.row_slots * 2) * sizeof(float);
    FP4X_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))),
                 "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need, workspace_bytes);
    float *ws = (float *)workspace;
    p.n_heads = n_heads, p.group = n_heads / p.c.n_kv, p.q_len = q_len;
    p.q = q, p.q_stride = q_stride, p.out = out;
    p.scale = 1.4426950408889634f / sqrtf((float)hd);
    const uint32_t tr = 8 * pl.nq, own_rows = p.group * q_len, all = own_rows * batch;
    p.own = Job{batch, own_rows, (own_rows + tr - 1) / tr, pl.own_ctas, page_table, lens, table_stride, max_len, ws,
                prefix_len ? ws + pl.own_slots + pl.prefix_slots : nullptr};
    p.prefix = Job{1, all, (all + tr - 1) / tr, pl.prefix_ctas, prefix_pages, nullptr, 0, prefix_len,
                   ws + pl.own_slots, ws + pl.own_slots + pl.prefix_slots + pl.row_slots};
    const bool f32 = dtype == FP4X_F32;
    if (cache->format == FP4X_MXFP8) {
        if (hd == 64) return f32 ? launch_all<FMT_FP8, 64, float>(who, st, p, pl.nq, rows) : launch_all<FMT_FP8, 64, __nv_bfloat16>(who, st, p, pl.nq, rows);
        return f32 ? launch_all<FMT_FP8, 128, float>(who, st, p, pl.nq, rows) : launch_all<FMT_FP8, 128, __nv_bfloat16>(who, st, p, pl.nq, rows);
    }
    if (hd == 64) return f32 ? launch_all<FMT_FP4, 64, float>(who, st, p, pl.nq, rows) : launch_all<FMT_FP4, 64, __nv_bfloat16>(who, st, p, pl.nq, rows);
    return f32 ? launch_all<FMT_FP4, 128, float>(who, st, p, pl.nq, rows) : launch_all<FMT_FP4, 128, __nv_bfloat16>(who, st, p, pl.nq, rows);
}

}  // namespace mxkv
}  // namespace fp4x

using namespace fp4x;

extern "C" size_t llama_attn_mx_workspace_size(const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                                               uint32_t q_len, uint32_t prefix_len, uint32_t max_len) {
    if (!cache || !cache->n_kv_heads || n_heads < cache->n_kv_heads) return 0;
    const mxkv::Plan pl =
        mxkv::make_plan(cache->n_kv_heads, cache->head_dim, batch, n_heads, q_len, prefix_len, max_len);
    return (size_t)((pl.own_slots + pl.prefix_slots + pl.row_slots * 2) * sizeof(float));
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
