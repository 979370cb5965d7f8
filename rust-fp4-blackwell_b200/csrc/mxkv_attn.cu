// mxkv_attn.cu -- attention over the MX-quantised paged cache, with an optional
// prefix that all sequences of the batch share.
//
// For query row r of sequence b and KV head h, with keys k_t and values v_t of the
// prefix and of the sequence's own pages:
//   s_t = q . k_t / sqrt(hd),  out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),
// one pass with a running maximum m and sum; partial results join as (m, l, o).
//
// attn_mx_kernel streams codes: a warp owns 16-position tiles, copies them with cp.async
// into a ring of its own (no barrier of the CTA in the loop), and contracts on mma.sync
// with the query rows as the 8 columns:
//   S^T = K q^T   in f16 per 32-block, times the block's K scale in f32;
//   O^T += V^T P^T in bf16 with the V scale of (position, block) multiplied into P^T.
// Codes are exact in f16 and bf16 and scales are powers of two, so the only roundings
// are P to two bf16 terms (16 bits; bf16 queries are exact in f16), or q to an f16 pair
// and P to three bf16 terms (f32 queries: 22 and 24 bits).  P takes bf16, not f16: its
// products with the scales, and probabilities far below the maximum, need the range (a
// dimension in which the largest position's code is 0 is made of those alone).  Bound by
// HBM: 64 sequences of up to 16384 positions, 8 KV heads x 128, MXFP8, take 216 us,
// 6.1 TB/s (0.93 of the measured rate); one of 32768 17 us, most of it opening and joining.
#include "mxkv.cuh"
#include "tc05.cuh"

namespace fp4x {
namespace mxkv {

constexpr uint32_t kWarps = 8;                 // warps per CTA
constexpr uint32_t kChunk = 16 * kWarps;       // positions of one step of a CTA
constexpr float kNoMax = -3.0e38f;             // running maximum before the first score
constexpr float kLag = 16.0f;                  // how far (in powers of two) a score may pass the running maximum

// One set of rows over one set of pages: the sequences of a batch over their own
// pages (n_seq = batch), or all rows of the batch over the shared prefix (n_seq = 1).
struct Job {
    uint32_t n_seq, rows, row_tiles, ctas;  // sequences, query rows per (sequence, KV head), tiles of them, grid
    uint32_t tile_rows;                     // 8, 16 or 32: attn_mx_kernel; 128: attn_mx_tile_kernel
    const int32_t *pages, *lens;            // lens null: every sequence holds max_len positions
    uint32_t table_stride, max_len;
    float *slots;      // 2 per CTA: its part of a segment that began before it, and of one that it began
    float *row_slots;  // one per output row for segments of one CTA (null: written to out)
    uint64_t *starts;  // cost before every sequence, then the total: for the join (null: one sequence)
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

// The own positions' kernel may run beside the prefix's, which waited for the stream's
// earlier work: it reads nothing of it, and ends after it, so that the join waits for both.
__device__ __forceinline__ bool beside(const AttnParams &p, bool prefix) { return !prefix && p.prefix.ctas; }
__device__ __forceinline__ void begin_kernel(const AttnParams &p, bool prefix) {
    if (!beside(p, prefix)) pdl_wait();
}
__device__ __forceinline__ void end_kernel(const AttnParams &p, bool prefix) {
    if (beside(p, prefix)) pdl_wait();
}

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
__device__ __forceinline__ uint64_t div(uint64_t a, uint64_t b) {  // a 64-bit division costs some hundred cycles
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}
__device__ __forceinline__ uint64_t cta_start(uint64_t c, uint64_t total, uint32_t ctas) { return div(c * total, ctas); }
__device__ __forceinline__ uint32_t cta_of(uint64_t at, uint64_t total, uint32_t ctas) {
    return (uint32_t)div((at + 1) * ctas - 1, total);
}

// Block-wide scan of the sequences' costs (each `per` segments): the total, and the
// sequence in which this CTA starts.
struct Located {
    uint64_t total, first;  // cost in all, cost before the located sequence
    uint32_t seq;
};
template <uint32_t THREADS>
__device__ Located locate(const Job &j, uint32_t per, uint64_t (&buf)[THREADS / 32 + 1], Located &res) {
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
    const uint64_t at = cta_start(blockIdx.x, total, j.ctas);
    if (threadIdx.x == 0) {
        res = Located{total, 0, 0};
        if (j.starts && blockIdx.x == 0) j.starts[j.n_seq] = total;
    }
    __syncthreads();
    for (uint32_t s = s0; s < s1; ++s) {
        const uint64_t n = (uint64_t)seq_cost(j, s) * per;
        if (before <= at && at < before + n) res.first = before, res.seq = s;
        if (j.starts && blockIdx.x == 0) j.starts[s] = before;
        before += n;
    }
    __syncthreads();
    return res;
}

// The segments of one CTA in turn.
struct Segment {
    uint32_t seq, head, r0, rows;  // first query row of the tile and how many it has
    uint32_t c0, c1, chunks, len;  // this CTA's chunks of the sequence's
    __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == chunks; }
};
struct Segments {
    uint64_t at, end, seq_first;
    uint32_t seq, per;
    Segments() = default;
    __device__ __forceinline__ Segments(const Job &j, uint32_t n_kv, const Located &loc) {
        at = cta_start(blockIdx.x, loc.total, j.ctas), end = cta_start(blockIdx.x + 1, loc.total, j.ctas);
        seq_first = loc.first, seq = loc.seq, per = n_kv * j.row_tiles;
    }
    __device__ __forceinline__ bool next(const Job &j, uint32_t n_kv, Segment &s) {
        while (at < end) {
            uint32_t cost = seq_cost(j, seq);
            while (at >= seq_first + (uint64_t)cost * per) {
                seq_first += (uint64_t)cost * per;
                cost = seq_cost(j, ++seq);
            }
            const uint64_t in_seq = at - seq_first;
            const uint32_t unit = (uint32_t)div(in_seq, cost), x0 = (uint32_t)(in_seq - (uint64_t)unit * cost);
            const uint32_t x1 = (uint32_t)min((uint64_t)cost, (uint64_t)x0 + (end - at));
            at += x1 - x0;
            s.c0 = max(x0, kOpen) - kOpen, s.c1 = max(x1, kOpen) - kOpen;
            if (s.c0 == s.c1) continue;
            s.seq = seq, s.len = seq_len(j, seq), s.chunks = cost - kOpen;
            s.head = unit % n_kv, s.r0 = unit / n_kv * j.tile_rows, s.rows = min(j.tile_rows, j.rows - s.r0);
            return true;
        }
        return false;
    }
};

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
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// The streaming kernel's ring.  A tile is 16 positions: their K codes, V codes and
// scales are four contiguous pieces of a page, copied 16 (scales: 8) bytes per lane in
// address order.  (Copied by the lanes that use them, V's pieces asked the L2 for single
// sectors, and the kernel stopped at 5.0 TB/s with all arithmetic taken out.)  Lane
// (g, t) uses
//   K: positions g and g + 8, two chunks of each: t and t + 4, or 2t and 2t + 1 where two
//      chunks make one 16- or 8-byte load;
//   V: positions 2t, 2t + 1, 2t + 8, 2t + 9, chunk g.
// at() places a row's 16-byte pieces so that both kinds of loads touch every bank once.
template <uint32_t FMT, uint32_t HD>
struct Ring {
    static constexpr uint32_t NB = HD / 32, B = Row<FMT, HD>::BYTES, CHUNK = Row<FMT, HD>::CHUNK, CW = CHUNK / 4;
    static constexpr bool PAIR = CHUNK < 16;  // both K chunks of a position in one load
    static constexpr uint32_t K_OFF = 0, V_OFF = 16 * B, KS_OFF = 32 * B, VS_OFF = KS_OFF + 16 * NB;
    static constexpr uint32_t STAGE = VS_OFF + 16 * NB;
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t piece) {
        if (B == 128) return row * B + ((piece ^ (row & 6) ^ ((row & 1) << 2)) << 4);
        const uint32_t slot = row ^ ((row >> 2) & 1);
        return slot * B + ((B == 64 ? piece ^ (row & 2) : piece) << 4);
    }
};

__device__ __forceinline__ float lds1(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts1(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ float4 lds4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts4(uint32_t a, float4 v) {
    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// CTAs of attn_mx_kernel that share an SM, by its rows / 8 x dimensions: two while O and, for f32 queries, the sums of
// it (Tile::SUMS) leave room for a second one.
__host__ __device__ constexpr bool two_ctas(uint32_t nq_hd, bool f32) { return nq_hd < 256 || (nq_hd == 256 && !f32); }

template <uint32_t FMT, uint32_t HD, uint32_t NQ, bool F32>
struct Tile {
    using R = Ring<FMT, HD>;
    static constexpr uint32_t NB = HD / 32, MT = HD / 16, CW = R::CW, TERMS = F32 ? 2 : 1, PTERMS = F32 ? 3 : 2;
    static constexpr bool QREG = NQ == 1 && !F32;
    static constexpr uint32_t Q_BYTES = TERMS * 2 * NB * NQ * 32 * 8;  // [term][half][block][column tile][lane] 8 B
    static constexpr int Q_TOP = 14;  // queries are scaled to a maximum in [2^14, 2^15): f16 keeps 2^-38 of it
    static constexpr uint32_t MERGE_BYTES = kWarps * MT * 32 * 16;  // O of one column tile, all warps
    static constexpr uint32_t MIN_CTAS = two_ctas(NQ * HD, F32) ? 2 : 1;
    // The MMA's accumulator cuts off what it adds (up to an ulp, always towards zero): over the 768 dependent
    // additions of 32768 positions that took 6.0e-6 of an f32 result, over 131072 positions 3.1e-5.  So every PERIOD
    // tiles (48 additions, 32 for bf16 queries) O moves to an f32 sum that each lane keeps in shared memory, where the
    // warps' results meet later: 5.9e-7 at any length.  It costs 1.5 % at 8 rows x 128 (64 sequences of up to 16384,
    // MXFP8, bf16: 219 -> 222 us) and 11 % where f32 queries give up the second CTA for it (16 rows x 128, 64 of up to
    // 8192: 214 -> 238 us; sums after every tile instead, in registers: 287 us).  bf16 queries with 256 row-dimensions
    // keep the second CTA (184 us; 204 with one) and the chain: 2 additions a tile, up to 1e-4 of a result over 131072
    // positions in one CTA, where bf16 has steps of 4e-3 to 8e-3 of it.
    static constexpr bool SUMS = !(MIN_CTAS == 2 && NQ * HD == 256);
    // The loop over the tiles in blocks of PERIOD, or a test in every tile: 222 against 231 us at 8 rows (as above), 288
    // against 302 at 32 rows x 64, but 451 against 422 at 32 rows x 128 (f32 queries, 64 of up to 8192).
    static constexpr bool BLOCKS = SUMS && (NQ == 1 || NQ * HD == 256);
    static constexpr uint32_t PERIOD = 16, SUM_BYTES = (SUMS ? NQ : 1) * MERGE_BYTES;
    static constexpr uint32_t STAGES = MIN_CTAS == 1 && NQ * HD == 256 ? 4 : R::STAGE > 3000 ? 2 : R::STAGE > 2000 ? 3 : 4;
    static constexpr uint32_t SMEM = kWarps * STAGES * R::STAGE + Q_BYTES + SUM_BYTES;
    static_assert((SMEM + 5120) * MIN_CTAS <= 228 * 1024, "the CTAs of an SM share its memory (5 KB: static and reserved)");

    float o[MT][NQ][4];
    float m[NQ][2], l[NQ][2];
    uint2 q[QREG ? 2 * NB : 1];

    // This lane's part of a sum, by column tile and 16-row tile of O.
    static __device__ __forceinline__ uint32_t sum_at(uint32_t qs, uint32_t n, uint32_t i) {
        return qs + Q_BYTES + (((n * kWarps + threadIdx.x / 32) * MT + i) * 32 + threadIdx.x % 32) * 16;
    }
    __device__ __forceinline__ void to_sum(uint32_t qs, bool add) {
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t i = 0; i < MT; ++i) {
                const uint32_t at = sum_at(qs, n, i);
                float4 y = make_float4(o[i][n][0], o[i][n][1], o[i][n][2], o[i][n][3]);
                if (add) {
                    const float4 z = lds4(at);
                    y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                }
                sts4(at, y);
                o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
            }
    }
    __device__ __forceinline__ void from_sum(uint32_t qs) {
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t i = 0; i < MT; ++i) {
                const float4 z = lds4(sum_at(qs, n, i));
                o[i][n][0] += z.x, o[i][n][1] += z.y, o[i][n][2] += z.z, o[i][n][3] += z.w;
            }
    }
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
    constexpr uint32_t NB = HD / 32, PIECES = R::B / 16;  // of a row
    const bool ok = (uint32_t)page < c.n_pages;
    const uint32_t p = ok ? (uint32_t)page : 0;
    const uint32_t n = ok ? left : 0;  // positions of the tile that exist
    const uint64_t co = code_off<FMT, HD>(c, p, head, row0) + lane * 16, so = scale_off<HD>(c, p, head, row0);
    const uint8_t *k = c.k + co, *v = c.v + co;
#pragma unroll
    for (uint32_t i = 0; i < PIECES / 2; ++i) {
        const uint32_t x = i * 32 + lane, row = x / PIECES, dst = ring + R::at(row, x % PIECES);
        cp_async(dst + R::K_OFF, k + i * 512, 16, n ? 16 : 0);
        cp_async(dst + R::V_OFF, v + i * 512, 16, row < n ? 16 : 0);  // V of positions that do not exist: zeros
    }
    constexpr uint32_t PER = 16 * NB / 8;  // 8-byte pieces of the tile's K (and of its V) scales
    if (lane < 2 * PER) {
        const uint32_t x = lane % PER * 8, have = lane < PER ? (n ? 8 : 0) : min(8u, n * NB - min(n * NB, x));
        cp_async(ring + R::KS_OFF + lane * 8, (lane < PER ? c.ks : c.vs) + so + x, 8, have);
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
// exist (0: a page outside the cache); lim[8 n + j] is the limit of column 2 t + j of tile n.
template <uint32_t FMT, uint32_t HD, uint32_t NQ, bool F32>
__device__ __forceinline__ void take_tile(Tile<FMT, HD, NQ, F32> &T, uint32_t ring, uint32_t qs, bool summed,
                                          uint32_t left, bool masked, const int32_t *lim, int32_t first, const float *rf,
                                          uint32_t lane) {
    using R = Ring<FMT, HD>;
    using TT = Tile<FMT, HD, NQ, F32>;
    constexpr uint32_t NB = HD / 32, CW = R::CW, TERMS = TT::TERMS;
    const uint32_t g = lane >> 2, t = lane & 3;
    // ---- S^T = K q^T
    float s[NQ][4];
#pragma unroll
    for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) s[n][j] = 0.0f;
    {
        uint32_t kw[2][2 * CW];  // [position g, g + 8][chunk half][word]
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t row = g + 8 * i;
            if constexpr (R::PAIR) {
                lds_words<2 * CW>(ring + R::K_OFF + R::at(row, t * CW / 2) + t * CW * 8 % 16, kw[i]);
            } else {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t w[CW];
                    lds_words<CW>(ring + R::K_OFF + R::at(row, t + 4 * h), w);
#pragma unroll
                    for (uint32_t j = 0; j < CW; ++j) kw[i][h * CW + j] = w[j];
                }
            }
        }
        uint32_t sc[2][1];  // 64-wide heads: the word of two rows
        lds_words<1>(ring + R::KS_OFF + (g * NB & ~3u), sc[0]);
        lds_words<1>(ring + R::KS_OFF + ((g + 8) * NB & ~3u), sc[1]);
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
                if (pos >= (int32_t)left || first + pos >= lim[n * 8 + (j & 1)]) s[n][j] = -INFINITY;
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
                if (TT::SUMS && summed) {
#pragma unroll 1
                    for (uint32_t i = 0; i < TT::MT; ++i) {
                        const uint32_t at = TT::sum_at(qs, n, i) + 4 * j;
                        sts1(at, lds1(at) * f), sts1(at + 8, lds1(at + 8) * f);
                    }
                }
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
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = 2 * t + (i & 1) + 8 * (i / 2);
        lds_words<CW>(ring + R::V_OFF + R::at(row, g * R::CHUNK / 16) + g * R::CHUNK % 16, vw[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t w[NB / 2];
        lds_words<NB / 2>(ring + R::VS_OFF + (2 * t + 8 * i) * NB, w);
        e8m0x4_to_bf16(NB == 4 ? __byte_perm(w[0], w[NB / 2 - 1], 0x5140) : __byte_perm(w[0], 0, 0x3120), sc[i][0],
                       sc[i][1]);
        if constexpr (NB == 4) e8m0x4_to_bf16(__byte_perm(w[0], w[NB / 2 - 1], 0x7362), sc[i][2], sc[i][3]);
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
    begin_kernel(p, prefix);
    pdl_launch_dependents();
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
    const uint32_t ring = smem_u32(smem) + warp * TT::STAGES * R::STAGE;
    uint8_t *qbuf = smem + kWarps * TT::STAGES * R::STAGE;
    float4 *merge = reinterpret_cast<float4 *>(qbuf + TT::Q_BYTES);
    const Located loc = locate<kWarps * 32>(job, p.c.n_kv * job.row_tiles, scan, where);
    // The walk over the segments lives in shared memory, one copy per warp: its state
    // would hold some thirty registers through the loop over the tiles.
    __shared__ Segments walk[kWarps];
    __shared__ Segment segs[kWarps][2];
    if (lane == 0) walk[warp] = Segments(job, p.c.n_kv, loc);
    __syncwarp();
    // The segment that copies are issued for: this warp's tiles are c * kWarps + warp for
    // c in [c0, c1), those that start below len.
    uint32_t c0 = 0, len = 0, head = 0, n_tiles = 0;
    uint32_t bad = 0;  // bit s: the page of the tile in stage s is outside the cache
    int32_t ids = 0;   // lane j: page of tile (j modulo 32)
    const int32_t *table = nullptr;
    auto issue = [&](uint32_t j) {
        if (j < n_tiles) {
            if ((j & 31) == 0) ids = j + lane < n_tiles ? table[((c0 + j + lane) * kWarps + warp) * 16 >> p.c.page_shift] : 0;
            const uint32_t first = ((c0 + j) * kWarps + warp) * 16;
            const int32_t page = __shfl_sync(~0u, ids, j & 31);
            issue_tile<FMT, HD>(p.c, ring + j % TT::STAGES * R::STAGE, page, head,
                                first & ((1u << p.c.page_shift) - 1), min(16u, len - first), lane);
            const bool out = (uint32_t)page >= p.c.n_pages;
            bad = (bad & ~(1u << j % TT::STAGES)) | ((uint32_t)out << j % TT::STAGES);
            if (out && lane == 0) raise_device_error(DEVERR_BAD_ARG);
        }
        cp_async_commit();
    };
    auto open = [&](uint32_t slot) {  // the next segment and its first copies
        Segments it = walk[warp];
        Segment sg = {};
        const bool any = it.next(job, p.c.n_kv, sg);
        __syncwarp();
        if (lane == 0) walk[warp] = it, segs[warp][slot] = sg;
        __syncwarp();
        if (!any) return false;
        c0 = sg.c0, len = sg.len, head = sg.head;
        table = job.pages + (uint64_t)sg.seq * job.table_stride;
        const uint32_t tiles = (len + 15) / 16;
        n_tiles = sg.c1 - c0;
        while (n_tiles && (c0 + n_tiles - 1) * kWarps + warp >= tiles) --n_tiles;
#pragma unroll
        for (uint32_t j = 0; j < TT::STAGES; ++j) issue(j);
        return true;
    };
    uint32_t slot_of = 0;
    for (bool more = open(0); more;) {
        const Segment &cur = segs[warp][slot_of];
        slot_of ^= 1;
        // ---- query rows: scaled by a power of two, in terms, fragment order
        for (uint32_t r = warp; r < ROWS; r += kWarps) {
            float x[HD / 32], amax = 0.0f;
            const RowAt ra = row_at(p, prefix, cur.seq, cur.head, cur.r0 + min(r, cur.rows - 1));
            const T *src = (const T *)p.q + (uint64_t)ra.token * p.q_stride + ra.head * HD;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) x[b] = r < cur.rows ? (float)src[b * 32 + lane] : 0.0f, amax = fmaxf(amax, fabsf(x[b]));
            amax = warp_max(amax);
            const int e = amax > 0.0f ? max(-112, min(127, (int)(__float_as_uint(amax) >> 23) - 127)) : 0;
            const float up = pow2(TT::Q_TOP - e);
            if (lane == 0) {
                rowf[r] = p.scale * pow2(max(e - TT::Q_TOP, -126));
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
        int32_t lowest = 0x7FFFFFFF;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                rf[n * 2 + j] = rowf[n * 8 + 2 * t + j];
                lowest = min(lowest, limit[n * 8 + 2 * t + j]);
            }
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, 1));
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, 2));
        if constexpr (TT::QREG) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * NB; ++i) tile.q[i] = reinterpret_cast<const uint2 *>(qbuf)[i * 32 + lane];
        }
        uint32_t stage = 0;
        bool summed = false;
        for (uint32_t j = 0; j < n_tiles;) {
            const uint32_t to = TT::BLOCKS ? min(n_tiles, j + TT::PERIOD) : n_tiles;
            for (; j < to; ++j) {
                if (TT::SUMS && !TT::BLOCKS && j && j % TT::PERIOD == 0) tile.to_sum(smem_u32(qbuf), summed), summed = true;
                const uint32_t first = ((c0 + j) * kWarps + warp) * 16;
                cp_async_wait<TT::STAGES - 1>();
                __syncwarp();  // every lane's copies of the tile have landed
                uint32_t left = min(16u, len - first);
                bool masked = (int32_t)(first + 16) > lowest || left < 16;
                if ((bad >> stage) & 1) left = 0, masked = true;
                take_tile<FMT, HD, NQ, F32>(tile, ring + stage * R::STAGE, smem_u32(qbuf), summed, left, masked, limit + 2 * t,
                                            (int32_t)first, rf, lane);
                stage = stage + 1 == TT::STAGES ? 0 : stage + 1;
                __syncwarp();  // every lane has read the stage
                issue(j + TT::STAGES);
            }
            if (TT::BLOCKS && j < n_tiles) tile.to_sum(smem_u32(qbuf), summed), summed = true;
        }
        if (summed) tile.from_sum(smem_u32(qbuf));
        more = open(slot_of);  // its first copies run under the joining of this one
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
        const bool whole = cur.whole();
        float *slot = nullptr;
        if (!whole) {
            slot = job.slots + (uint64_t)(2 * blockIdx.x + (cur.c0 == 0)) * ROWS * (HD + 2);
            if (threadIdx.x < ROWS) slot[2 * threadIdx.x] = top[threadIdx.x], slot[2 * threadIdx.x + 1] = sum[threadIdx.x];
            slot += 2 * ROWS;
        } else if (job.row_slots && threadIdx.x < cur.rows) {
            const RowAt ra = row_at(p, prefix, cur.seq, cur.head, cur.r0 + threadIdx.x);
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
                    if (r >= cur.rows) continue;
                    const float y0 = j ? acc.y : acc.x, y1 = j ? acc.w : acc.z;
                    if (!whole) {
                        store2<float>(slot + r * HD + d, y0, y1);
                        continue;
                    }
                    const RowAt ra = row_at(p, prefix, cur.seq, cur.head, cur.r0 + r);
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
    end_kernel(p, prefix);
}

// ---------------------------------------------------------------- many rows: tcgen05
// attn_mx_tile_kernel: 128 query rows of a KV head against tiles of TN positions on
// tcgen05.  The codes are dequantised once per tile for all 128 rows:
//   warps 8-15  codes -> bf16 (exact: at most four significant bits times a power of
//               two) in shared memory, rows of 128 bytes with the 128-byte swizzle; the
//               same image serves K (K-major) and V (MN-major);
//   warp 16     S = Q K^T and O += P V, S of the next tile ahead of P V;
//   warps 0-7   two threads per row, half of the columns each: maximum (exchanged
//               through shared memory), exp2, row sum; P as two bf16 terms (16 bits; f32
//               queries: Q and P as three, 24 bits) back into tensor memory, from where
//               it is the A operand.  O is rescaled only when a row's maximum grows by
//               more than kLag powers of two, and moved to a sum every FLUSH tiles.
// Bound by the instructions of the two: 96 x 4 rows x 8 heads on 32768 positions (MXFP8,
// bf16) take 118 us, 4500 cycles a tile, 1536 of them MMAs.
template <uint32_t HD, bool F32>
struct Big {
    static constexpr uint32_t TN = F32 ? 64 : 128, QT = F32 ? 3 : 1, PT = F32 ? 3 : 2;
    static constexpr uint32_t REG = HD / 64;  // 64-dimension regions of an operand
    static constexpr uint32_t Q_BYTES = QT * REG * 128 * 128, KV_BYTES = REG * TN * 128;
    static constexpr uint32_t SMEM = Q_BYTES + 4 * KV_BYTES + 1024;
    static constexpr uint32_t THREADS = 17 * 32, DEQ = 256;
    // tensor memory columns: two S buffers (P takes the place of S), then O, then the sum of earlier O
    static constexpr uint32_t S_COLS = F32 ? 96 : 128, O_COL = 2 * S_COLS, SUM_COL = O_COL + HD, COLS = 512;
    // O is added to a sum of its own every FLUSH tiles, because the MMA's accumulator cuts off what it adds (see
    // Tile::SUMS).  f32: 24 additions a time, 4.3e-7 of sums of one sign (every 8 tiles: 5.0e-6; every tile: 4.0e-7
    // for up to 3 % of the time).  bf16, 96 x 4 rows on 32768 positions: 64 additions, 0.12 % of the results on the other
    // side of a rounding edge than the 64-bit ones (plain f32 arithmetic: 0.15 %); every 8 tiles 0.14 % and 2 % less
    // time, every 2 tiles 0.11 % and 5 % more, never 0.3 % and 3.5 % less.
    static constexpr uint32_t FLUSH = F32 ? 2 : 4;
    // first column of term z of P for positions 16 ks .. 16 ks + 15 (8 columns), from the buffer's start
    static __device__ __forceinline__ uint32_t p_col(uint32_t z, uint32_t ks) {
        return F32 ? 32 * z + 8 * ks : 32 * (ks / 2) + 16 * z + 8 * (ks & 1);
    }
};

__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// kind::f16 instruction descriptor: bf16 x bf16 -> f32, M = 128; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t idesc_bf16(uint32_t n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

#define FP4X_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define FP4X_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : FP4X_R8(v, 0), FP4X_R8(v, 8), FP4X_R8(v, 16), FP4X_R8(v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : FP4X_R8(v, 0), FP4X_R8(v, 8)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        FP4X_I8(v, 0), FP4X_I8(v, 8)
        : "memory");
}
#undef FP4X_R8
#undef FP4X_I8
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Codes of one thread's task: chunks 2 pair and 2 pair + 1 of a position, and its scales.
template <uint32_t FMT, uint32_t HD>
struct Codes {
    static constexpr uint32_t W = Row<FMT, HD>::CHUNK / 2, NB = HD / 32;
    uint32_t w[W], scales;
    __device__ __forceinline__ void load(const uint8_t *codes, const uint8_t *sc) {
        load_words<W>(codes, w);
        scales = NB == 4 ? __ldg(reinterpret_cast<const uint32_t *>(sc)) : __ldg(reinterpret_cast<const uint16_t *>(sc));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) w[i] = 0;
        scales = 0;
    }
    // -> the position's row in an operand image at `base` (region stride TN * 128 bytes)
    template <uint32_t TN>
    __device__ __forceinline__ void store(uint8_t *base, uint32_t pos, uint32_t pair) const {
        uint32_t sc[NB / 2];
#pragma unroll
        for (uint32_t i = 0; i < NB / 2; ++i)
            asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, l;\n\t}"
                : "=r"(sc[i])
                : "r"(i ? scales >> 16 : scales));
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            const uint32_t s2 = __byte_perm(sc[b / 2], 0, b & 1 ? 0x3232 : 0x1010);
            uint32_t f[4], y[4];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                if constexpr (FMT == FMT_FP8) {
                    e4m3x4_to_f16(w[h * NB + b], f[2 * h], f[2 * h + 1]);
                } else {
                    uint32_t d[4];
                    decode_word_f16(w[(h * NB + b) / 2], d);
                    f[2 * h] = d[2 * (b & 1)], f[2 * h + 1] = d[2 * (b & 1) + 1];
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) y[i] = bmul2(f16x2_to_bf16x2(f[i]), s2);
            const uint32_t c = ((b & 1) * 4 + pair) ^ (pos & 7);
            *reinterpret_cast<uint4 *>(base + (b / 2) * TN * 128 + pos * 128 + c * 16) =
                make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
};

// True in one lane of a converged warp (always the same one).
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

// A bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase) {
    return __all_sync(~0u, mbar_wait_bounded(bar, phase));
}

template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(Big<HD, sizeof(T) == 4>::THREADS, 1)
    attn_mx_tile_kernel(const __grid_constant__ AttnParams p, bool prefix) {
    constexpr bool F32 = sizeof(T) == 4;
    using BG = Big<HD, F32>;
    constexpr uint32_t TN = BG::TN, ROWS = 128;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t scan[BG::THREADS / 32 + 1];
    __shared__ Located where;
    __shared__ __align__(8) uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pready[2], pvdone[2], done;
    // Byte w, bit i: positions 64 i + 8 w .. of the tile lie in no page.  Four deep: tile t + 4 is written after S of
    // tile t + 2, which waits for P V of tile t and so for the softmax warps that read tile t's bytes.
    __shared__ __align__(8) uint8_t no_page[4][8];
    __shared__ uint32_t tmem_base;
    __shared__ float halfmax[2][2][ROWS], halfsum[2][ROWS];
    __shared__ uint32_t lost[4];  // a wait of either warp of these 32 rows ran out at a segment's end
    uint8_t *smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    uint8_t *qs = smem, *ks = smem + BG::Q_BYTES, *vs = ks + 2 * BG::KV_BYTES;
    const Job &job = prefix ? p.prefix : p.own;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&kfull[i], BG::DEQ / 32), mbar_init(&vfull[i], BG::DEQ / 32);
            mbar_init(&kempty[i], 1), mbar_init(&vempty[i], 1), mbar_init(&sfull[i], 1), mbar_init(&pvdone[i], 1);
            mbar_init(&pready[i], 8);
        }
        mbar_init(&done, 1);
        lost[0] = lost[1] = lost[2] = lost[3] = 0;
        fence_mbar_init();
    }
    if (warp == 16) {
        tc::tmem_alloc(&tmem_base, BG::COLS);
        tc::tmem_relinquish();
    }
    begin_kernel(p, prefix);
    const Located loc = locate<BG::THREADS>(job, p.c.n_kv * job.row_tiles, scan, where);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    pdl_launch_dependents();  // not before this CTA has its tensor memory: a dependent may be this kernel again
    const uint32_t tmem = tmem_base;
    Segments segments(job, p.c.n_kv, loc);
    Segment sg = {};
    bool ok = true;    // a bounded wait ran out: leave (the others' waits run out too)
    uint32_t tile = 0;  // tiles taken so far, over all segments

    if (warp < 8) {
        // ================================================= softmax
        const uint32_t quad = warp & 3, half = warp >> 2, row = quad * 32 + lane, lanes = (quad * 32) << 16;
        constexpr uint32_t CH = TN / 64;  // 32-column pieces of a thread
        // the two warps of 32 rows meet here; a failed wait is passed on as a NaN, so that both leave
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(quad + 1) : "memory"); };
        while (ok && segments.next(job, p.c.n_kv, sg)) {
            const RowAt ra = row_at(p, prefix, sg.seq, sg.head, sg.r0 + min(row, sg.rows - 1));
            const int32_t limit =
                prefix ? (int32_t)sg.len : (int32_t)sg.len - (int32_t)p.q_len + 1 + (int32_t)ra.step;
            const int32_t low = __reduce_min_sync(~0u, limit);
            const uint32_t stop = min(sg.c1 * kChunk, sg.len);
            float m = kNoMax, l = 0.0f;
            bool good = true;
            uint32_t taken = 0;  // tiles of the segment so far
            for (uint32_t pos = sg.c0 * kChunk; pos < stop; pos += TN, ++tile, ++taken) {
                const uint32_t buf = tile & 1, ph = (tile >> 1) & 1, sb = tmem + lanes + buf * BG::S_COLS;
                good = good && warp_wait(&sfull[buf], ph);
                tc::fence_after_sync();
                const uint64_t bad = *(volatile uint64_t *)no_page[tile & 3];
                const bool masked = (int32_t)(pos + TN) > low || bad;
                const int32_t left = limit - (int32_t)pos;
                auto load = [&](uint32_t(&x)[32], uint32_t c) {
                    tmem_ld32(sb + c * 32, x);
                    if (masked) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i)
                            if ((int32_t)(c * 32 + i) >= left || (bad >> ((c % 2 * 4 + i / 8) * 8 + c / 2)) & 1)
                                x[i] = __float_as_uint(-INFINITY);
                    }
                };
                uint32_t x[32];  // the last piece stays for the exponentials
                float mx = -INFINITY;
#pragma unroll
                for (uint32_t c = 0; c < CH; ++c) {
                    load(x, half * CH + c);
                    float mz[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 2)
                        mz[i / 2 % 4] = fmaxf(mz[i / 2 % 4], fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                    mx = fmaxf(fmaxf(mz[0], mz[1]), fmaxf(mz[2], mz[3]));
                }
                halfmax[tile & 1][half][row] = good ? mx : __uint_as_float(0x7FC00000u);
                meet();
                const float other = halfmax[tile & 1][half ^ 1][row];
                if (__any_sync(~0u, !good || other != other)) {
                    ok = false;
                    break;
                }
                mx = fmaxf(mx, other) * p.scale;
                const bool grow = mx > m + kLag, any = __any_sync(~0u, grow);
                const bool flush = taken && taken % BG::FLUSH == 0, summed = taken > BG::FLUSH;
                const float mn = grow ? mx : m, f = any ? ex2(m - mn) : 1.0f;
                m = mn, l *= f;
                if ((any && taken) || flush) {  // O rescaled, or moved to the sum
                    const uint32_t pt = tile - 1;
                    good = warp_wait(&pvdone[pt & 1], (pt >> 1) & 1);
                    tc::fence_after_sync();
#pragma unroll 1
                    for (uint32_t c = 0; c < HD / 32; ++c) {
                        const uint32_t at = tmem + lanes + half * (HD / 2) + c * 16;
                        uint32_t y[16];
                        tmem_ld16(at + BG::O_COL, y);
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                        if (!flush) tmem_st16(at + BG::O_COL, y);
                        if (summed) {
                            uint32_t z[16];
                            tmem_ld16(at + BG::SUM_COL, z);
#pragma unroll
                            for (uint32_t i = 0; i < 16; ++i)
                                y[i] = __float_as_uint(fmaf(__uint_as_float(z[i]), f, flush ? __uint_as_float(y[i]) : 0.0f));
                        }
                        if (summed || flush) tmem_st16(at + BG::SUM_COL, y);
                    }
                }
#pragma unroll
                for (uint32_t cc = 0; cc < CH; ++cc) {
                    const uint32_t c = half * CH + (CH - 1 - cc);
                    if (cc) load(x, c);
                    float2 part = {0.0f, 0.0f};
                    const float2 sc2 = {p.scale, p.scale}, m2 = {-m, -m};
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 2) {
                        float2 e = fma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, m2);
                        e = make_float2(ex2(e.x), ex2(e.y));
                        part = add2(part, e);
                        x[i] = __float_as_uint(e.x), x[i + 1] = __float_as_uint(e.y);
                    }
                    l += part.x + part.y;
#pragma unroll
                    for (uint32_t z = 0; z < BG::PT; ++z) {
                        uint32_t y[16];
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) {
                            const float2 e = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
                            y[i] = pack_bf16x2(e.x, e.y);
                            if (z + 1 < BG::PT) {
                                const float2 r = add2(e, make_float2(__uint_as_float((y[i] << 16) ^ 0x80000000u),
                                                                     __uint_as_float((y[i] & 0xFFFF0000u) ^ 0x80000000u)));
                                x[2 * i] = __float_as_uint(r.x), x[2 * i + 1] = __float_as_uint(r.y);
                            }
                        }
                        tmem_st16(sb + BG::p_col(z, 2 * c), y);
                    }
                }
                tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pready[buf]);
            }
            if (!ok) break;
            const uint32_t pt = tile - 1;
            good = good && warp_wait(&pvdone[pt & 1], (pt >> 1) & 1);
            tc::fence_after_sync();
            halfsum[half][row] = l;
            if (!good && lane == 0) lost[quad] = 1;
            meet();
            l = halfsum[0][row] + halfsum[1][row];
            ok = *(volatile uint32_t *)&lost[quad] == 0;  // both leave or neither
            const uint64_t out_row = (uint64_t)ra.token * p.n_heads + ra.head;
            const bool whole = sg.whole(), live = row < sg.rows;
            float *dst = nullptr;
            if (!whole) {
                dst = job.slots + (uint64_t)(2 * blockIdx.x + (sg.c0 == 0)) * ROWS * (HD + 2);
                if (live && !half) dst[2 * row] = m, dst[2 * row + 1] = l;
                dst += 2 * ROWS + row * HD;
            } else if (job.row_slots) {
                dst = job.row_slots + out_row * (HD + 2);
                if (live && !half) dst[HD] = m, dst[HD + 1] = l;
            }
            const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll 1
            for (uint32_t c = half * (HD / 64); c < (half + 1) * (HD / 64); ++c) {
                uint32_t x[32];
                tmem_ld32(tmem + lanes + BG::O_COL + c * 32, x);
                if (taken > BG::FLUSH) {
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        uint32_t z[16];
                        tmem_ld16(tmem + lanes + BG::SUM_COL + c * 32 + h * 16, z);
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i)
                            x[h * 16 + i] = __float_as_uint(__uint_as_float(x[h * 16 + i]) + __uint_as_float(z[i]));
                    }
                }
                if (live) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 2) {
                        const float a = __uint_as_float(x[i]), b = __uint_as_float(x[i + 1]);
                        if (dst)
                            store2<float>(dst + c * 32 + i, a, b);
                        else
                            store2<T>((T *)p.out + out_row * HD + c * 32 + i, a * inv, b * inv);
                    }
                }
            }
            tc::fence_before_sync();
        }
    } else if (warp < 16) {
        // ================================================= codes -> bf16 images
        const uint32_t id = threadIdx.x - 256, pair = id & 3;
        // eight lanes of a store phase hold positions x and x + 4: all 32 banks
        const uint32_t sub = (lane >> 2) & 7, pos0 = (id / 32) * 8 + (sub >> 1) + (sub & 1) * 4;
        constexpr uint32_t TASKS = TN / 64;
        const uint32_t off = pair * Codes<FMT, HD>::W * 4;
        while (ok && segments.next(job, p.c.n_kv, sg)) {
            const int32_t *table = job.pages + (uint64_t)sg.seq * job.table_stride;
            const uint32_t start = sg.c0 * kChunk, stop = min(sg.c1 * kChunk, sg.len);
            Codes<FMT, HD> kc[TASKS], vc[TASKS];
            // where a position's row lies, in K and V alike; not in the cache or past the end: no row
            struct Place {
                uint64_t codes, scales;
                bool row, bad;
            } next[TASKS];
            uint32_t kbad = 0;  // bit i: the positions of kc[i] lie in no page
            int32_t ids[TASKS];
            auto page_of = [&](uint32_t pos) { return pos < stop ? table[pos >> p.c.page_shift] : 0; };
            auto place = [&](uint32_t pos, int32_t page) {
                const uint32_t r = pos & ((1u << p.c.page_shift) - 1);
                return Place{code_off<FMT, HD>(p.c, (uint32_t)page, sg.head, r) + off,
                             scale_off<HD>(p.c, (uint32_t)page, sg.head, r), pos < stop && (uint32_t)page < p.c.n_pages,
                             pos < stop && (uint32_t)page >= p.c.n_pages};
            };
            auto fetch = [&](Codes<FMT, HD> &cd, const uint8_t *codes, const uint8_t *scales, const Place &a) {
                if (a.row)
                    cd.load(codes + a.codes, scales + a.scales);
                else
                    cd.clear();
            };
            auto fetch_k = [&](const Place(&a)[TASKS]) {
                kbad = 0;
#pragma unroll
                for (uint32_t i = 0; i < TASKS; ++i) fetch(kc[i], p.c.k, p.c.ks, a[i]), kbad |= (uint32_t)a[i].bad << i;
            };
            // K of tile t (the codes are in kc): the image, and which positions lie in no page
            auto put_k = [&](uint32_t t) {
                const uint32_t st = t & 1;
                if (t >= 2 && !warp_wait(&kempty[st], ((t >> 1) - 1) & 1)) return false;
#pragma unroll
                for (uint32_t i = 0; i < TASKS; ++i)
                    kc[i].template store<TN>(ks + st * BG::KV_BYTES, pos0 + 64 * i, pair);
                const uint32_t bits = __reduce_or_sync(~0u, kbad);
                if (lane == 0) {
                    no_page[t & 3][warp - 8] = (uint8_t)bits;
                    if (bits) raise_device_error(DEVERR_BAD_ARG);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&kfull[st]);
                return true;
            };
#pragma unroll
            for (uint32_t i = 0; i < TASKS; ++i) {
                const uint32_t pos = start + pos0 + 64 * i;
                next[i] = place(pos, page_of(pos));
                fetch(vc[i], p.c.v, p.c.vs, next[i]);
            }
            fetch_k(next);
#pragma unroll
            for (uint32_t i = 0; i < TASKS; ++i) {
                const uint32_t pos = start + pos0 + 64 * i;
                next[i] = place(pos + TN, page_of(pos + TN));
                ids[i] = page_of(pos + 2 * TN);
            }
            // ---- query rows: after the previous segment's last S
            if (tile && !(ok = warp_wait(&kempty[(tile - 1) & 1], ((tile - 1) >> 1) & 1))) break;
            for (uint32_t i = id; i < ROWS * (HD / 8); i += BG::DEQ) {
                const uint32_t r = i / (HD / 8), c = i % (HD / 8);
                float x[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) x[j] = 0.0f;
                if (r < sg.rows) {
                    const RowAt ra = row_at(p, prefix, sg.seq, sg.head, sg.r0 + r);
                    load8<T>((const T *)p.q + (uint64_t)ra.token * p.q_stride + ra.head * HD + c * 8, x);
                }
#pragma unroll
                for (uint32_t z = 0; z < BG::QT; ++z) {
                    uint32_t y[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        y[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
                        x[2 * j] -= __uint_as_float(y[j] << 16), x[2 * j + 1] -= __uint_as_float(y[j] & 0xFFFF0000u);
                    }
                    *reinterpret_cast<uint4 *>(qs + (z * BG::REG + c / 8) * 128 * 128 + r * 128 +
                                               ((c & 7) ^ (r & 7)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
                // K runs one tile ahead of V, so that S of the next tile does not wait for P V of the last
            if (!(ok = put_k(tile))) break;
            fetch_k(next);
            for (uint32_t pos = start; pos < stop; pos += TN, ++tile) {
                const uint32_t st = tile & 1;
                Place after[TASKS];
#pragma unroll
                for (uint32_t i = 0; i < TASKS; ++i) after[i] = place(pos + 2 * TN + pos0 + 64 * i, ids[i]);
                if (pos + TN < stop) {
                    if (!(ok = put_k(tile + 1))) break;
                    fetch_k(after);
#pragma unroll
                    for (uint32_t i = 0; i < TASKS; ++i) ids[i] = page_of(pos + 3 * TN + pos0 + 64 * i);
                }
                if (tile >= 2 && !(ok = warp_wait(&vempty[st], ((tile >> 1) - 1) & 1))) break;
#pragma unroll
                for (uint32_t i = 0; i < TASKS; ++i) {
                    vc[i].template store<TN>(vs + st * BG::KV_BYTES, pos0 + 64 * i, pair);
                    fetch(vc[i], p.c.v, p.c.vs, next[i]);
                    next[i] = after[i];
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&vfull[st]);
            }
        }
    } else {
        // ================================================= the MMAs
        // The whole warp runs the loop and one elected lane issues: the operands then are
        // warp-uniform values.  Issued from a branch on the lane number, an MMA took some
        // 200 cycles instead of its 64.
        const uint32_t qa = smem_u32(qs), ka = smem_u32(ks), va = smem_u32(vs);
        constexpr uint32_t ID_S = idesc_bf16(TN, false), ID_O = idesc_bf16(HD, true);
        uint32_t pv = 0;  // tiles whose P V has been issued
        bool pending = false, opens = false;  // a tile waits for its P V; it is its segment's first
        auto issue_pv = [&]() {
            const uint32_t st = pv & 1, ph = (pv >> 1) & 1;
            if (!warp_wait(&vfull[st], ph) || !warp_wait(&pready[st], ph)) return false;
            tc::fence_after_sync();
            const uint32_t sb = tmem + st * BG::S_COLS;
            const uint64_t bd = tc::smem_desc(va + st * BG::KV_BYTES, TN * 128, 1024, tc::kLayoutSw128);
            if (elect_one()) {
#pragma unroll
                for (uint32_t k = 0; k < TN / 16; ++k)
#pragma unroll
                    for (uint32_t z = 0; z < BG::PT; ++z)
                        mma_bf16_ts(tmem + BG::O_COL, sb + BG::p_col(z, k), bd + k * (2048 >> 4), ID_O,
                                    k || z ? 1u : !opens);
                tc::commit(&vempty[st]);
                tc::commit(&pvdone[st]);
            }
            __syncwarp();
            ++pv;
            return true;
        };
        while (ok && segments.next(job, p.c.n_kv, sg)) {
            const uint32_t start = sg.c0 * kChunk, stop = min(sg.c1 * kChunk, sg.len);
            for (uint32_t pos = start; pos < stop; pos += TN, ++tile) {
                const uint32_t st = tile & 1, ph = (tile >> 1) & 1;
                // the S buffer holds the P of two tiles ago until its P V is done
                if (tile >= 2 && !(ok = warp_wait(&pvdone[st], ((tile >> 1) - 1) & 1))) break;
                if (!(ok = warp_wait(&kfull[st], ph))) break;
                tc::fence_after_sync();
                const uint64_t ad = tc::desc_sw128(qa), bd = tc::desc_sw128(ka + st * BG::KV_BYTES);
                if (elect_one()) {
#pragma unroll
                    for (uint32_t z = 0; z < BG::QT; ++z)
#pragma unroll
                        for (uint32_t k = 0; k < HD / 16; ++k)
                            mma_bf16_ss(tmem + st * BG::S_COLS,
                                        ad + (((z * BG::REG + k / 4) * 128 * 128 + (k & 3) * 32) >> 4),
                                        bd + (((k / 4) * TN * 128 + (k & 3) * 32) >> 4), ID_S, z || k);
                    tc::commit(&kempty[st]);
                    tc::commit(&sfull[st]);
                }
                __syncwarp();
                if (pending && !(ok = issue_pv())) break;
                pending = true, opens = (pos - start) / TN % BG::FLUSH == 0;
            }
        }
        if (ok && pending) ok = issue_pv();
        // everything issued has finished before tensor memory is given back
        if (elect_one()) tc::commit(&done);
        __syncwarp();
        warp_wait(&done, 0);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == 16) tc::tmem_dealloc(tmem, BG::COLS);
    end_kernel(p, prefix);
}

// ---------------------------------------------------------------- hidden positions that are not finite
// Of the last q_len positions of a sequence some queries see only the first ones.  The kernels above give the others the
// probability 0, and 0 times a NaN (or a value past 2^128) in V is NaN.  That is rare, so they do not look: the join
// does where a result is NaN, and if such a position holds one, it computes the row anew from what the row sees, with
// plain f32 arithmetic (a CTA for one row, 128 positions at a time).

// Dimension d of a cached row.
template <uint32_t FMT, uint32_t HD>
__device__ __forceinline__ float value_at(const uint8_t *codes, const uint8_t *scales, uint32_t d) {
    const uint32_t at = (d % 32 / 4 * (HD / 32) + d / 32) * 4 + d % 4;
    const uint32_t h = FMT == FMT_FP8 ? e4m3x2_to_f16x2(codes[at]) : e2m1x2_to_f16x2(codes[at / 2] >> (at % 2 * 4) & 15);
    return __half2float(__ushort_as_half((unsigned short)h)) * e8m0_to_f32(scales[d / 32]);
}

// The page of position t of a row that sees the prefix and then `own` positions.
__device__ __forceinline__ uint32_t page_of(const AttnParams &p, uint32_t seq, uint32_t t, uint32_t &row) {
    const uint32_t before = p.prefix.ctas ? p.prefix.max_len : 0, u = t < before ? t : t - before;
    row = u & ((1u << p.c.page_shift) - 1);
    return t < before ? p.prefix.pages[u >> p.c.page_shift]
                      : p.own.pages[(uint64_t)seq * p.own.table_stride + (u >> p.c.page_shift)];
}

template <uint32_t FMT, uint32_t HD, typename T>
__device__ __noinline__ void redo_row(const AttnParams &p, uint32_t token, uint32_t head) {
    __shared__ float qf[HD], prob[128], red[4];
    const uint32_t seq = token / p.q_len, kvh = head / p.group, tid = threadIdx.x;
    const uint32_t before = p.prefix.ctas ? p.prefix.max_len : 0, len = seq_len(p.own, seq);
    const uint32_t seen = (uint32_t)max((int32_t)len - (int32_t)p.q_len + 1 + (int32_t)(token % p.q_len), 0), n = before + seen;
    uint32_t row;
    bool bad = false;
    for (uint32_t i = tid; i < (len - seen) * HD; i += 128) {
        const uint32_t page = page_of(p, seq, n + i / HD, row);
        if (page >= p.c.n_pages) continue;
        const float v = value_at<FMT, HD>(p.c.v + code_off<FMT, HD>(p.c, page, kvh, row),
                                          p.c.vs + scale_off<HD>(p.c, page, kvh, row), i % HD);
        bad |= !(fabsf(v) <= 3.40282347e+38f);
    }
    if (!__syncthreads_or(bad)) return;  // the NaN is the row's own
    if (tid < HD) qf[tid] = (float)((const T *)p.q)[token * p.q_stride + head * HD + tid] * p.scale;
    float m = kNoMax, l = 0.0f, o = 0.0f;
    for (uint32_t t0 = 0; t0 < n; t0 += 128) {
        __syncthreads();
        float s = -INFINITY;
        uint32_t page = t0 + tid < n ? page_of(p, seq, t0 + tid, row) : ~0u;
        if (page < p.c.n_pages) {
            const uint8_t *codes = p.c.k + code_off<FMT, HD>(p.c, page, kvh, row), *scales = p.c.ks + scale_off<HD>(p.c, page, kvh, row);
            s = 0.0f;
            for (uint32_t d = 0; d < HD; ++d) s = fmaf(qf[d], value_at<FMT, HD>(codes, scales, d), s);
        }
        const float mw = warp_max(s);
        if (tid % 32 == 0) red[tid / 32] = mw;
        __syncthreads();
        const float mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), f = exp2f(m - mx);
        prob[tid] = exp2f(s - mx);
        __syncthreads();
        m = mx, l *= f, o *= f;
        for (uint32_t i = 0; i < min(128u, n - t0); ++i) {
            l += prob[i];
            page = page_of(p, seq, t0 + i, row);
            if (page < p.c.n_pages && tid < HD)
                o += prob[i] * value_at<FMT, HD>(p.c.v + code_off<FMT, HD>(p.c, page, kvh, row),
                                                 p.c.vs + scale_off<HD>(p.c, page, kvh, row), tid);
        }
    }
    if (tid < HD) ((T *)p.out)[((uint64_t)token * p.n_heads + head) * HD + tid] = (T)(l == 0.0f ? 0.0f : o / l);
}

// Joins the partial results of one output row: those of the CTAs that shared its
// segment, and with a prefix those of both jobs.  The places of all partials are worked
// out first, so that four warps can have four loads each in flight; a row that one CTA
// wrote whole has nothing to join.
template <uint32_t FMT, uint32_t HD, typename T>
__global__ void __launch_bounds__(128) attn_mx_join_kernel(const __grid_constant__ AttnParams p) {
    constexpr uint32_t W = 4, V = HD / 32, U = 4, LIST = 64;  // a lane holds V dimensions
    __shared__ float sm[W], sl[W], so[W][HD];
    __shared__ const float *ml_of[LIST], *o_of[LIST];
    const uint32_t row = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t token = row / p.n_heads, head = row % p.n_heads, kvh = head / p.group;
    const bool hides = p.q_len > 1 && p.own.ctas;  // some positions from some queries
    T *out = (T *)p.out + (uint64_t)row * HD + threadIdx.x;
    pdl_wait();
    // partials of each job: the row's slot, or its place in the slots of CTAs first..last
    uint32_t n = 0, from[2], count[2], in_tile[2];
    uint64_t total[2];
#pragma unroll
    for (uint32_t which = 0; which < 2; ++which) {
        const Job &job = which ? p.prefix : p.own;
        count[which] = 0, from[which] = 0, total[which] = 0;
        const uint32_t seq = which ? 0 : token / p.q_len;
        const uint32_t r = which ? token * p.group + head % p.group : token % p.q_len * p.group + head % p.group;
        in_tile[which] = job.ctas ? r % job.tile_rows : 0;
        if (!job.ctas) continue;
        const uint32_t chunks = seq_chunks(job, seq);
        if (chunks == 0) continue;
        total[which] = which ? (uint64_t)seq_cost(job, 0) * p.c.n_kv * job.row_tiles : job.starts[job.n_seq];
        const uint64_t at = (which ? 0 : job.starts[seq]) +
                            (uint64_t)(r / job.tile_rows * p.c.n_kv + kvh) * (chunks + kOpen) + kOpen;
        from[which] = cta_of(at, total[which], job.ctas);
        count[which] = cta_of(at + chunks - 1, total[which], job.ctas) - from[which] + 1;
        if (count[which] == 1 && !job.row_slots) {  // written whole (without a prefix)
            if (hides) {
                const float y = threadIdx.x < HD ? (float)*out : 0.0f;
                if (__syncthreads_or(y != y)) redo_row<FMT, HD, T>(p, token, head);
            }
            return;
        }
        n += count[which];
    }
    float m = kNoMax, l = 0.0f, o[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) o[i] = 0.0f;
    for (uint32_t base = 0; base < n; base += LIST) {
        const uint32_t here = min(LIST, n - base);
        if (base) __syncthreads();
        for (uint32_t i = threadIdx.x; i < here; i += 128) {
            const uint32_t k = base + i, which = k >= count[0];
            const Job &job = which ? p.prefix : p.own;
            const uint32_t at = which ? k - count[0] : k, cnt = which ? count[1] : count[0];
            if (cnt == 1) {
                o_of[i] = job.row_slots + (uint64_t)row * (HD + 2), ml_of[i] = o_of[i] + HD;
            } else {
                const uint32_t c = (which ? from[1] : from[0]) + at, tr = job.tile_rows, r = which ? in_tile[1] : in_tile[0];
                const uint64_t tot = which ? total[1] : total[0];
                const float *slot = job.slots + (uint64_t)(2 * c + (at == 0)) * tr * (HD + 2);
                // with more CTAs than cost some have no work
                const bool idle = at && tot < job.ctas && cta_start(c, tot, job.ctas) == cta_start(c + 1, tot, job.ctas);
                ml_of[i] = idle ? nullptr : slot + 2 * r, o_of[i] = slot + 2 * tr + r * HD;
            }
        }
        __syncthreads();
        for (uint32_t k0 = warp; k0 < here; k0 += W * U) {
            float2 ml[U], po[U][V / 2];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t k = min(k0 + u * W, here - 1);
                const bool take = k0 + u * W < here && ml_of[k];
                ml[u] = take ? *reinterpret_cast<const float2 *>(ml_of[k]) : make_float2(kNoMax, 0.0f);
#pragma unroll
                for (uint32_t i = 0; i < V / 2; ++i)
                    po[u][i] = take ? reinterpret_cast<const float2 *>(o_of[k])[lane * (V / 2) + i]
                                    : make_float2(0.0f, 0.0f);
            }
            float mn = m;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
            const float f = exp2f(m - mn);
            l *= f, m = mn;
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) o[i] *= f;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const float g = exp2f(ml[u].x - mn);
                l += ml[u].y * g;
#pragma unroll
                for (uint32_t i = 0; i < V / 2; ++i) o[2 * i] += po[u][i].x * g, o[2 * i + 1] += po[u][i].y * g;
            }
        }
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) so[warp][lane * V + i] = o[i];
    __syncthreads();
    float mx = kNoMax, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) mx = fmaxf(mx, sm[w]);
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        const float f = exp2f(sm[w] - mx);
        sum += sl[w] * f, acc += so[w][threadIdx.x % HD] * f;
    }
    const float y = sum == 0.0f ? 0.0f : acc / sum;
    if (threadIdx.x < HD) *out = (T)y;
    if (hides && __syncthreads_or(y != y)) redo_row<FMT, HD, T>(p, token, head);
}

// ---------------------------------------------------------------- host
// Rows of a tile: 8 per mma column tile; up to 32 rows share one read of the codes in attn_mx_kernel, 128 in
// attn_mx_tile_kernel.  Time on the GPU of calls with MXFP8 (MXFP4 within 6 % of it), 4 KV heads, 24 sequences of up
// to 6001 positions (in brackets one of 32768):
//   rows                    20 or 40 in attn_mx_kernel     in attn_mx_tile_kernel
//   40 x 64, bf16 / f32     72 (37) / 90 (40) us           52 (29) / 70 (37) us
//   40 x 128, bf16 / f32    108 (47) / 135 (59)            62 (35) / 93 (47)
//   20 x 64, bf16 / f32     45 (33) / 53 (29)              48 (29) / 66 (37)
//   20 x 128, bf16 / f32    64 (33) / 77 (41)              58 (33) / 88 (46)
inline uint32_t tile_rows_of(uint64_t rows, uint32_t hd, bool f32) {
    const uint32_t most = hd == 128 && !f32 ? 16 : 32;
    return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= most ? 32 : 128;
}

struct Plan {
    uint32_t own_rows, prefix_rows;  // per tile
    uint32_t own_ctas, prefix_ctas;
    uint64_t own_slots, prefix_slots, row_slots, starts;  // floats
};
// CTAs of a job that run at once per SM.
inline uint32_t ctas_per_sm(uint32_t hd, uint32_t tile_rows, bool f32) { return two_ctas(tile_rows / 8 * hd, f32) ? 2 : 1; }

// The plan for bf16 queries needs at least the workspace of that for f32 (it has at least the CTAs, and their rows).
Plan make_plan(uint32_t n_kv, uint32_t hd, uint32_t batch, uint32_t n_heads, uint32_t q_len, uint32_t prefix_len,
               uint32_t max_len, bool f32) {
    Plan pl = {};
    const uint64_t rows = (uint64_t)(n_heads / n_kv) * q_len, all = rows * batch;
    const uint32_t sms = (uint32_t)num_sms();
    auto job = [&](uint32_t seqs, uint32_t len, uint64_t r, uint32_t &tile_rows, uint32_t &ctas, uint64_t &slots) {
        tile_rows = tile_rows_of(r, hd, f32);
        const uint64_t chunks = ((uint64_t)len + kChunk - 1) / kChunk * seqs * n_kv * ((r + tile_rows - 1) / tile_rows);
        const uint64_t room = (uint64_t)sms * ctas_per_sm(hd, tile_rows, f32);
        ctas = (uint32_t)(chunks < room ? chunks : room);  // more would idle
        slots = 2ull * ctas * tile_rows * (hd + 2);
    };
    job(batch, max_len, rows, pl.own_rows, pl.own_ctas, pl.own_slots);
    pl.starts = ((uint64_t)batch + 2) / 2 * 4;
    if (prefix_len) {
        job(1, prefix_len, all, pl.prefix_rows, pl.prefix_ctas, pl.prefix_slots);
        pl.row_slots = (uint64_t)batch * q_len * n_heads * (hd + 2);
    }
    return pl;
}

template <typename K>
int launch_with_smem(const char *who, cudaStream_t st, K kernel, bool (&ready)[64], uint32_t ctas, uint32_t threads,
                     uint32_t smem, const AttnParams &p, bool prefix) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return set_error("%s: %s", who, cudaGetErrorString(e)), FP4X_ECUDA;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const cudaError_t e = launch_pdl(kernel, dim3(ctas), dim3(threads), smem, st, p, prefix);
    if (e != cudaSuccess) return set_error("%s: %s", who, cudaGetErrorString(e)), FP4X_ECUDA;
    return check_launch(who);
}

template <uint32_t FMT, uint32_t HD, uint32_t NQ, typename T>
int launch_stream(const char *who, cudaStream_t st, const AttnParams &p, bool prefix) {
    using TT = Tile<FMT, HD, NQ, sizeof(T) == 4>;
    static bool ready[64] = {};
    return launch_with_smem(who, st, attn_mx_kernel<FMT, HD, NQ, T>, ready, (prefix ? p.prefix : p.own).ctas,
                            kWarps * 32, TT::SMEM, p, prefix);
}
template <uint32_t FMT, uint32_t HD, typename T>
int launch_tile(const char *who, cudaStream_t st, const AttnParams &p, bool prefix) {
    using BG = Big<HD, sizeof(T) == 4>;
    static bool ready[64] = {};
    return launch_with_smem(who, st, attn_mx_tile_kernel<FMT, HD, T>, ready, (prefix ? p.prefix : p.own).ctas,
                            BG::THREADS, BG::SMEM, p, prefix);
}

template <uint32_t FMT, uint32_t HD, typename T>
int launch_all(const char *who, cudaStream_t st, const AttnParams &p, uint64_t rows) {
    int rc = FP4X_OK;
    for (int prefix = 1; prefix >= 0 && rc == FP4X_OK; --prefix) {
        const Job &job = prefix ? p.prefix : p.own;
        if (!job.ctas) continue;
        if (job.tile_rows == 8)
            rc = launch_stream<FMT, HD, 1, T>(who, st, p, prefix);
        else if (job.tile_rows == 16)
            rc = launch_stream<FMT, HD, 2, T>(who, st, p, prefix);
        else if (job.tile_rows == 128)
            rc = launch_tile<FMT, HD, T>(who, st, p, prefix);
        else if constexpr (HD == 64 || sizeof(T) == 4)
            rc = launch_stream<FMT, HD, 4, T>(who, st, p, prefix);
    }
    if (rc != FP4X_OK) return rc;
    const cudaError_t e = launch_pdl(attn_mx_join_kernel<FMT, HD, T>, dim3((uint32_t)rows), dim3(128), 0, st, p);
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
    // the end of the tile in which a sequence ends is a 32-bit signed position too
    constexpr uint32_t kMost = 0x7FFFFFFFu - 2 * kChunk;
    FP4X_REQUIRE(max_len <= kMost && prefix_len <= kMost && max_len + prefix_len <= kMost,
                 "%s: lengths must stay below 2^31 - 256", who);
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
    const Plan pl = make_plan(p.c.n_kv, hd, batch, n_heads, q_len, prefix_len, max_len, dtype == FP4X_F32);
    const size_t need = (pl.starts + pl.own_slots + pl.prefix_slots + pl.row_slots * 2) * sizeof(float);
    FP4X_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace, 16))),
                 "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need, workspace_bytes);
    float *ws = (float *)workspace + pl.starts;
    p.n_heads = n_heads, p.group = n_heads / p.c.n_kv, p.q_len = q_len;
    p.q = q, p.q_stride = q_stride, p.out = out;
    p.scale = 1.4426950408889634f / sqrtf((float)hd);
    const uint32_t own_rows = p.group * q_len, all = own_rows * batch;
    p.own = Job{batch, own_rows, (own_rows + pl.own_rows - 1) / pl.own_rows, pl.own_ctas, pl.own_rows, page_table, lens,
                table_stride, max_len, ws, prefix_len ? ws + pl.own_slots + pl.prefix_slots : nullptr, (uint64_t *)workspace};
    p.prefix = Job{};
    if (prefix_len)
        p.prefix = Job{1, all, (all + pl.prefix_rows - 1) / pl.prefix_rows, pl.prefix_ctas, pl.prefix_rows,
                       prefix_pages, nullptr, 0, prefix_len, ws + pl.own_slots,
                       ws + pl.own_slots + pl.prefix_slots + pl.row_slots, nullptr};
    const bool f32 = dtype == FP4X_F32;
    if (cache->format == FP4X_MXFP8) {
        if (hd == 64) return f32 ? launch_all<FMT_FP8, 64, float>(who, st, p, rows) : launch_all<FMT_FP8, 64, __nv_bfloat16>(who, st, p, rows);
        return f32 ? launch_all<FMT_FP8, 128, float>(who, st, p, rows) : launch_all<FMT_FP8, 128, __nv_bfloat16>(who, st, p, rows);
    }
    if (hd == 64) return f32 ? launch_all<FMT_FP4, 64, float>(who, st, p, rows) : launch_all<FMT_FP4, 64, __nv_bfloat16>(who, st, p, rows);
    return f32 ? launch_all<FMT_FP4, 128, float>(who, st, p, rows) : launch_all<FMT_FP4, 128, __nv_bfloat16>(who, st, p, rows);
}

}  // namespace mxkv
}  // namespace fp4x

using namespace fp4x;

extern "C" size_t llama_attn_mx_workspace_size(const fp4x_mxkv *cache, uint32_t batch, uint32_t n_heads,
                                               uint32_t q_len, uint32_t prefix_len, uint32_t max_len) {
    if (!cache || !cache->n_kv_heads || n_heads < cache->n_kv_heads) return 0;
    const mxkv::Plan pl =
        mxkv::make_plan(cache->n_kv_heads, cache->head_dim, batch, n_heads, q_len, prefix_len, max_len, false);
    return (size_t)((pl.starts + pl.own_slots + pl.prefix_slots + pl.row_slots * 2) * sizeof(float));
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
