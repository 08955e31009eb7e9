// attention_rows.cu -- attention of few query rows (a decode step, a few drafted tokens) over the paged
// cache: row tiles of 8 or 16, bound by the bytes of the cache.
//
// Arithmetic: mma.sync m16n8k16 with fp32 sums, transposed so that the keys, not the few queries,
// fill the 16 rows of a product: S^T = K Q^T (16 keys x 8 queries), then the weights by a reference that
// is raised when one grows large, and their sum, then O^T += V^T P^T.  P is rounded to the products' 16-bit type (fp16
// 2^-11, bf16 2^-8 of each weight) and a quantised value to fp16 (2^-11).  That is a choice: the tensor cores' floats
// have no more bits than fp16's, and operands in two halves would take two or three products for each.  With fp16
// outputs the error against 64 bits is then 3.4e-4 of the outputs' norm, where their own rounding is 2.1e-4.  Scores of
// quantised keys are of exact codes; scores, references, sums and outputs are fp32.  A tile of 8 queries costs half the
// products, exponentials and registers that a 16-row tile of queries would, and widening the codes, which dominates, is
// done once for all queries.  The legacy tensor path is enough: it works a fifth of the time at the rate at which
// HBM delivers keys, and tcgen05's smallest tile has 64 rows, of which a decode step fills 8.
//
// What bounds it: 48 sequences of 300 to 9000 tokens in Q8_0 (573 MB) take 115 us, 76% of the measured HBM rate, and 124 to 129
// once it has run for some milliseconds, when the card's 1000 W cap holds its clock (1725 MHz).  Q4_0
// carries twice the values a byte, and there the instructions that widen them bound it: one row over 120000
// keys (138 MB) takes 64 us, 33%, of which some 8 are the join and the launches.  A decode step of 4 short
// sequences takes 9 us, which is latency: finding its share, one ring, the join.
//
// Loads: each warp owns a ring of stages of 16 keys, filled by cp.async.  Pages of 16 keys and more
// hold whole steps, whose rows are one run of memory; in smaller pages each key's row is looked up
// and handed to the lanes that copy it.  (One bulk copy a row was tried: the instruction takes
// uniform operands, so 32 of them become a loop of 400 instructions a step.)  Rows are padded by 16
// bytes, which makes the reads below free of bank conflicts.  Codes are widened straight from the ring into
// MMA operands: the order of a product's inner dimension is free as long as both operands share it,
// so a lane feeds the contiguous values of its key to consecutive MMAs, and the query's operands
// are gathered to match once; the same holds for the order of the head's dimensions in O^T, which
// are put in order when the outputs are stored.
//
// The four warps of a CTA take turns at the steps of a unit and keep maxima, sums and outputs of
// their own, joined through shared memory at the end of the unit.
#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "attention.cuh"

namespace anvil {

constexpr int kRowsWarps = 4;
constexpr int kRowsStep = 16;   // keys of a warp's step
constexpr int kRowsKeys = 64;   // keys of a key tile: one step of each warp
constexpr float kRowsSlack = 60000.0f;  // the largest weight: fp16 ends at 65504
constexpr int kRowsCost = 0;    // beginning and ending a unit, in key tiles

template <int KIND, int D, int NT> struct RowsShape {
    static constexpr int rows = 8 * NT;                     // query rows of a unit
    static constexpr int rb = KvRow<KIND, D>::bytes;
    static constexpr int ch = rb / 16;                      // 16-byte chunks of a row
    static constexpr int sb = KvRow<KIND, D>::scales * 2;   // bytes of a row's scales
    static constexpr int kst = KIND == kKvQ8_0 ? rb + 32 : rb + 16;  // row strides in the ring: distinct banks
    static constexpr int vst = rb + 16;
    static constexpr int off_v = kRowsStep * kst, off_s = off_v + kRowsStep * vst;
    static constexpr int off_bad = off_s + 2 * kRowsStep * sb;
    static constexpr int stage = off_bad + 16;
    // two stages keep 16 keys of every warp in flight while 16 are worked on; rows of up to 80 bytes take three
    static constexpr int stages = stage <= 3000 ? 3 : 2;
    static constexpr int ring = stage * stages;             // of one warp
    static constexpr int join = rows * (D + 4) * 4 + rows * 8;  // of one warp, reuses the ring
    static constexpr int per_warp = ((ring > join ? ring : join) + 15) & ~15;
    static constexpr int smem = kRowsWarps * per_warp;
    static constexpr bool bf16 = KIND == kKvBF16;
    static constexpr bool quant = KIND == kKvQ8_0 || KIND == kKvQ4_0;
    // CTAs of an SM that the registers are cut for: O^T takes D NT / 4 of them
    static constexpr int min_ctas = D * NT <= 128 ? 4 : D * NT <= 256 ? 3 : 2;
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Copies 16 bytes to shared memory, of which the first n are read and the others zero.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// Transposes an 8 x 8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Codes to fp16 pairs: a byte or nibble below the exponent of 1024 (or 16 times a nibble) is an fp16
// number that differs from the code by a constant, taken off exactly.
__device__ __forceinline__ uint32_t q8_pair(uint32_t u, uint32_t sel) {  // bytes are code + 128
    return h2sub(__byte_perm(u, 0x64646464u, sel), 0x64806480u);
}
__device__ __forceinline__ uint32_t q4_low(uint32_t u) { return (u & 0x000F000Fu) | 0x64006400u; }
__device__ __forceinline__ uint32_t q4_high(uint32_t u) { return (u & 0x00F000F0u) | 0x64006400u; }
__device__ __forceinline__ uint32_t q4_fix_low(uint32_t h) { return h2sub(h, 0x64086408u); }            // - 1032
__device__ __forceinline__ uint32_t q4_fix_high(uint32_t h) { return h2fma(h, 0x2C002C00u, 0xD480D480u); }  // / 16 - 72

// ---- the dimension that a lane's operand stands for -------------------------------------------

// First of the 4 dimensions of QK step s for quad lane c; the operands hold (d, d+1), (d+2, d+3), or
// for Q4_0, whose nibbles come in pairs two bytes apart, (d, d+2), (d+1, d+3).  Of a quantised row two steps
// cover a block of 32 values; 16-bit rows are read in chunks of 8 values, chunk j of a lane 8 (j / 2) + 2 c + j % 2.
__device__ __forceinline__ int k_chunk(int j, int c) { return 8 * (j >> 1) + 2 * c + (j & 1); }
template <int KIND> __device__ __forceinline__ int k_dim(int s, int c) {
    if constexpr (KIND == kKvQ8_0) return 32 * (s >> 1) + 8 * c + 4 * (s & 1);
    else if constexpr (KIND == kKvQ4_0) return 32 * (s >> 1) + 4 * c + 16 * (s & 1);
    else return 8 * k_chunk(s >> 1, c) + 4 * (s & 1);
}

// The i-th (of D / 8) dimension that lane group g (0..7) owns in O^T.
template <int KIND, int D> __device__ __forceinline__ int v_dim(int i, int g) {
    if constexpr (KIND == kKvQ8_0) {
        if constexpr (D == 64) return 8 * g + i;
        else return 16 * (g + 8 * (i >> 4)) + (i & 15);
    } else if constexpr (KIND == kKvQ4_0) {
        // word i / 8, then low and high nibbles, each in the order 0, 2, 1, 3
        const int w = i >> 3, r = i & 7, e = ((r & 1) << 1) | ((r >> 1) & 1), d = 4 * w + 16 * (r >> 2) + e;
        if constexpr (D == 64) return 32 * (g >> 2) + 4 * (g & 3) + d;
        else if constexpr (D == 128) return 32 * (g >> 1) + 8 * (g & 1) + d;
        else return 32 * g + d;
    } else return 8 * (g + 8 * (i >> 3)) + (i & 7);
}

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(kRowsWarps * 32, RowsShape<KIND, D, NT>::min_ctas)
    attn_rows_kernel(KvCacheView c, KvBatchView bt, AttnIO io) {
    using S = RowsShape<KIND, D, NT>;
    constexpr int ROWS = S::rows;
    constexpr int NS = D / 16;   // QK steps
    constexpr int MT = D / 16;   // tiles of 16 dimensions
    constexpr bool BF = S::bf16;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ AttnScratch sc;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cq = lane & 3;
    uint8_t *ring = smem + warp * S::per_warp;
    const bool whole = c.page_shift >= 4;

    const int64_t work = attn_locate<ROWS, kRowsKeys, kRowsCost>(
        c, bt, io, &sc, [&](const AttnShares &s) { return s.begin(min(int(blockIdx.x), s.ctas - 1)); }, blockIdx.x == 0);
    pdl_launch_dependents();
    attn_zero_rest<D>(bt, io);
    const AttnShares shares(work, gridDim.x);
    // what is to be joined: nothing, unless the last unit is left unfinished below
    if (io.part && threadIdx.x == 0) attn_open<ROWS, D>(io.part, gridDim.x)[blockIdx.x].parts = 0;
    if (int(blockIdx.x) >= shares.ctas) return;
    const int64_t lo = shares.begin(blockIdx.x), hi = shares.begin(blockIdx.x + 1);
    AttnPos p = sc.pos;
    KvSeq kseq = load_seq(bt, c, p.b);
    int slot = 0, fill = 0;     // ring slots: next to be worked on, next to be filled

    while (p.b < bt.batch && p.unit0 < hi) {
        const AttnSeq<ROWS, kRowsKeys> q(kseq, io);
        const int ntiles = q.key_tiles(p.mt), nkeys = q.keys(p.mt);
        const int t0 = int(max(lo - p.unit0, int64_t(0))), t1 = int(min(hi - p.unit0, int64_t(ntiles)));
        const int key_end = min(t1 * kRowsKeys, nkeys);
        const int nrows = int(min(int64_t(ROWS), int64_t(unsigned(q.n) * unsigned(io.group) - unsigned(p.mt) * ROWS)));

        // ---- the ring: step s covers keys 16 s .. 16 s + 15
        const int step0 = t0 * 4 + warp, steps = (key_end + kRowsStep - 1) / kRowsStep;
        // Cache row of key 16 s + lane % 16 (-1: no page, -2: no key); where pages hold 16 keys and more, and so
        // whole steps, the row of key 16 s on every lane.
        auto row_of = [&](int s) -> int64_t {
            const int key = s * kRowsStep + (whole ? 0 : lane & 15);
            if (s >= steps || key >= key_end) return -2;
            return kv_lookup(bt, c, p.b, key, p.head);
        };
        auto issue = [&](int s, int64_t row) {
            if (s < steps) {
                uint8_t *st = ring + fill * S::stage;
                const uint32_t dst = smem_u32(st) + (lane / S::ch) * S::kst + (lane % S::ch) * 16;
                const uint32_t dst_v = smem_u32(st) + S::off_v + (lane / S::ch) * S::vst + (lane % S::ch) * 16;
                uint32_t bad;
                if (whole) {
                    const int live = row < 0 ? 0 : min(kRowsStep, key_end - s * kRowsStep);
                    bad = row == -1 ? 0xFFFFu : 0;
                    const int64_t off = max(row, int64_t(0)) * S::rb + lane * 16;
#pragma unroll
                    for (int j = 0; j < S::ch / 2; ++j) {
                        const int n = lane / S::ch + j * (32 / S::ch) < live ? 16 : 0;  // 0: zeros are written
                        cp_async16(dst + j * (32 / S::ch) * S::kst, c.k + off + j * 512, n);
                        cp_async16(dst_v + j * (32 / S::ch) * S::vst, c.v + off + j * 512, n);
                    }
                    if constexpr (S::quant) {  // 16 rows' scales: sb chunks of 16 bytes of each tensor
                        if (lane < 2 * S::sb) {
                            const int i = lane & (S::sb - 1);
                            const uint8_t *src = reinterpret_cast<const uint8_t *>(lane < S::sb ? c.ks : c.vs);
                            // (a chunk of scales may cover rows behind the last: bytes, not chunks, are cut)
                            const int n = max(0, min(16, live * S::sb - i * 16));
                            cp_async16(smem_u32(st) + S::off_s + lane * 16,
                                       src + max(row, int64_t(0)) * S::sb + i * 16, n);
                        }
                    }
                } else {
                    bad = __ballot_sync(0xffffffffu, row == -1) & 0xFFFFu;
#pragma unroll
                    for (int j = 0; j < S::ch / 2; ++j) {
                        const int64_t rw = __shfl_sync(0xffffffffu, row, lane / S::ch + j * (32 / S::ch));
                        const int64_t off = max(rw, int64_t(0)) * S::rb + (lane % S::ch) * 16;
                        cp_async16(dst + j * (32 / S::ch) * S::kst, c.k + off, rw < 0 ? 0 : 16);
                        cp_async16(dst_v + j * (32 / S::ch) * S::vst, c.v + off, rw < 0 ? 0 : 16);
                    }
                    if constexpr (S::quant) {
                        const uint8_t *src = reinterpret_cast<const uint8_t *>(lane < 16 ? c.ks : c.vs);
                        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(
                                         smem_u32(st) + S::off_s + lane * S::sb),
                                     "l"(src + max(row, int64_t(0)) * S::sb), "n"(S::sb), "r"(row < 0 ? 0 : S::sb)
                                     : "memory");
                    }
                }
                if (lane == 0) {
                    *reinterpret_cast<uint32_t *>(st + S::off_bad) = bad;
                    if (bad) flag_bad_page();
                }
                if (++fill == S::stages) fill = 0;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        int64_t next = row_of(step0);
#pragma unroll
        for (int i = 0; i < S::stages - 1; ++i) {
            const int64_t row = next;
            next = row_of(step0 + 4 * (i + 1));
            issue(step0 + 4 * i, row);
        }

        // ---- the query's operands.  Lane group g gathers rows 8 t + g; a lane's scores are of the rows
        // 8 t + 2 cq + e, whose keys seen and score factors come from the lanes that gathered them.
        int seen[NT][2];
        float fac[NT][2];
        uint32_t qb[NT][NS][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = 8 * t + g;
            const unsigned rr = unsigned(p.mt) * ROWS + r;
            const int tok = int(by_group(io, rr)), h = p.head * io.group + int(rr - unsigned(tok) * io.group);
            const bool live = r < nrows;
            const int my_seen = live ? kv_seen(tok, q.n, q.s.kv, io.causal) : 0;
            const uint16_t *src = static_cast<const uint16_t *>(io.q) + (q.s.q0 + int64_t(tok)) * io.q_row + h * io.q_head;
            uint32_t m = 0;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                uint2 w = make_uint2(0, 0);
                if (live) w = __ldg(reinterpret_cast<const uint2 *>(src + k_dim<KIND>(s, cq)));
                qb[t][s][0] = w.x;
                qb[t][s][1] = w.y;
                if (S::quant) {
                    m = max(max(m, w.x & 0x7FFFu), (w.x >> 16) & 0x7FFFu);
                    m = max(max(m, w.y & 0x7FFFu), (w.y >> 16) & 0x7FFFu);
                }
            }
            int ex = 0;
            if (S::quant && io.q_bf16) {
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                ex = q_exponent(m << 16);
                const float f = pow2i(ex);
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = qb[t][s][i];
                        qb[t][s][i] = pack_half(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xFFFF0000u) * f);
                    }
            }
            if (KIND == kKvQ4_0)
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const uint32_t x = qb[t][s][0], y = qb[t][s][1];
                    qb[t][s][0] = __byte_perm(x, y, 0x5410);
                    qb[t][s][1] = __byte_perm(x, y, 0x7632);
                }
            // A negative scale: -q, so that the largest score stays the largest.  Above zero, so that a masked score stays -inf.
            if (io.scale_log2 < 0.0f)
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    qb[t][s][0] ^= 0x80008000u;
                    qb[t][s][1] ^= 0x80008000u;
                }
            const float my_fac = fmaxf(fabsf(io.scale_log2) * pow2i(-ex), 1e-36f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                seen[t][e] = min(__shfl_sync(0xffffffffu, my_seen, (2 * cq + e) * 4), key_end);
                fac[t][e] = __shfl_sync(0xffffffffu, my_fac, (2 * cq + e) * 4);
            }
        }
        // every row of the unit sees the keys below this: no mask is needed there
        const int free_end = min(key_end, kv_seen(int(by_group(io, unsigned(p.mt) * ROWS)), q.n, q.s.kv, io.causal));

        // m: references; nb: their negatives, 0 for none; fresh: some row has none
        float o[NT][MT][4], m[NT][2], l[NT][2], nb[NT][2];
        bool fresh = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t][i][j] = 0.0f;
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = nb[t][0] = nb[t][1] = 0.0f;
        }

        for (int s = step0; s < steps; s += 4) {
            {   // the slot that the last step freed
                const int64_t row = next;
                next = row_of(s + 4 * S::stages);
                __syncwarp();
                issue(s + 4 * (S::stages - 1), row);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(S::stages - 1) : "memory");
            __syncwarp();
            uint8_t *sk = ring + slot * S::stage, *sv = sk + S::off_v;
            __half *ks = reinterpret_cast<__half *>(sk + S::off_s);
            __half *vs = ks + kRowsStep * KvRow<KIND, D>::scales;
            const uint32_t bad = *reinterpret_cast<const uint32_t *>(sk + S::off_bad);
            (void)ks;
            (void)vs;

            // ---- S^T = K Q^T: sc2[t]: keys g (0, 1) and g + 8 (2, 3), rows 8 t + 2 cq + (0, 1)
            float sc2[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc2[t][j] = 0.0f;
            const uint8_t *k0 = sk + g * S::kst, *k1 = k0 + 8 * S::kst;
            if constexpr (S::quant) {
                // Codes are whole numbers of fp16, taken exactly; a block's sum is multiplied by its scale in fp32.  (The
                // scale times the codes, rounded to fp16, was the largest error of the scores, and more instructions.)
                constexpr int NB = D / 32;
                uint32_t dw[2][NB / 2];  // scales of keys g and g + 8
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const __half *at = ks + (g + 8 * i) * NB;
                    if constexpr (NB == 2) dw[i][0] = *reinterpret_cast<const uint32_t *>(at);
                    else
#pragma unroll
                        for (int j = 0; j < NB / 4; ++j)
                            *reinterpret_cast<uint2 *>(&dw[i][2 * j]) = *reinterpret_cast<const uint2 *>(at + 4 * j);
#pragma unroll
                    for (int j = 0; j < NB / 2; ++j) dw[i][j] = usable_scales<KIND>(dw[i][j]);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float x[NT][4] = {};
                    uint32_t lo[4], hi[4];  // the block's two steps
                    if constexpr (KIND == kKvQ8_0) {
                        uint2 u = *reinterpret_cast<const uint2 *>(k0 + b * 32 + cq * 8), v = *reinterpret_cast<const uint2 *>(k1 + b * 32 + cq * 8);
                        u.x ^= 0x80808080u, u.y ^= 0x80808080u, v.x ^= 0x80808080u, v.y ^= 0x80808080u;
                        lo[0] = q8_pair(u.x, 0x4140), lo[1] = q8_pair(v.x, 0x4140), lo[2] = q8_pair(u.x, 0x4342), lo[3] = q8_pair(v.x, 0x4342);
                        hi[0] = q8_pair(u.y, 0x4140), hi[1] = q8_pair(v.y, 0x4140), hi[2] = q8_pair(u.y, 0x4342), hi[3] = q8_pair(v.y, 0x4342);
                    } else {
                        const uint32_t u = *reinterpret_cast<const uint32_t *>(k0 + b * 16 + cq * 4), v = *reinterpret_cast<const uint32_t *>(k1 + b * 16 + cq * 4);
                        const uint32_t u8 = u >> 8, v8 = v >> 8;
                        lo[0] = q4_fix_low(q4_low(u)), lo[1] = q4_fix_low(q4_low(v)), lo[2] = q4_fix_low(q4_low(u8)), lo[3] = q4_fix_low(q4_low(v8));
                        hi[0] = q4_fix_high(q4_high(u)), hi[1] = q4_fix_high(q4_high(v)), hi[2] = q4_fix_high(q4_high(u8)), hi[3] = q4_fix_high(q4_high(v8));
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma16816<BF>(x[t], lo, qb[t][2 * b][0], qb[t][2 * b][1]);
                        mma16816<BF>(x[t], hi, qb[t][2 * b + 1][0], qb[t][2 * b + 1][1]);
                    }
                    float d[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        d[i] = __half2float(__ushort_as_half(uint16_t(dw[i][b >> 1] >> (16 * (b & 1)))));
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc2[t][j] = fmaf(x[t][j], d[j >> 1], sc2[t][j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < S::ch / 4; ++j) {
                    const int at = k_chunk(j, cq) * 16;
                    const uint4 u = *reinterpret_cast<const uint4 *>(k0 + at), v = *reinterpret_cast<const uint4 *>(k1 + at);
                    const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma16816<BF>(sc2[t], a0, qb[t][2 * j][0], qb[t][2 * j][1]);
                        mma16816<BF>(sc2[t], a1, qb[t][2 * j + 1][0], qb[t][2 * j + 1][1]);
                    }
                }
            }

            // ---- weights by the rows' references m.  Only where one exceeds 60000, or where there is
            // no reference yet, is the step's maximum looked for, made the reference, and the step taken again.
            const int key0 = s * kRowsStep;
            const bool masked = key0 + kRowsStep > free_end || bad != 0;
            if (masked) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = g + 8 * (j >> 1);
                        if (key0 + k >= seen[t][j & 1] || ((bad >> k) & 1)) sc2[t][j] = -INFINITY;
                    }
            }
            uint32_t pb[NT][2];
            float e[NT][4];
            for (bool first = true;; first = false) {
                bool raise = false;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[t][j] = ex2(fmaf(sc2[t][j], fac[t][j & 1], nb[t][j & 1]));
                        raise |= e[t][j] > kRowsSlack;
                    }
                if (!__any_sync(0xffffffffu, (raise || fresh) && first)) break;
                fresh = false;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        float x = fmaxf(sc2[t][d], sc2[t][2 + d]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) * fac[t][d] - kAttnHead<BF>;
                        const float mn = fmaxf(m[t][d], x);
                        const float a = mn == -INFINITY ? 1.0f : ex2(m[t][d] - mn);
                        fresh |= mn == -INFINITY;  // a row without keys so far
                        l[t][d] *= a;
                        m[t][d] = mn;
                        nb[t][d] = mn == -INFINITY ? 0.0f : -mn;
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            o[t][i][d] *= a;
                            o[t][i][2 + d] *= a;
                        }
                    }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = e[t][2 * i], y = e[t][2 * i + 1];
                    l[t][0] += x;
                    l[t][1] += y;
                    pb[t][i] = transpose8(BF ? pack_bf16(x, y) : pack_half(x, y));
                }

            if (masked) {
                // A value that some row of the tile does not see must not reach it, and 0 x NaN would: a
                // non-finite value is added by hand to the rows that see it and leaves the product.
                bool odd = false;
                if constexpr (S::quant) {
                    if (lane < 16)
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) {
                            const uint32_t y = usable_scales<KIND>(__half_as_ushort(vs[lane * (D / 32) + i]));
                            odd |= (y & 0x7FFFu) >= kOddScale<KIND>;
                        }
                } else {
                    for (int i = lane; i < kRowsStep * S::ch; i += 32) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(sv + (i / S::ch) * S::vst + (i % S::ch) * 16);
                        odd |= (nonfinite2<BF>(w.x) | nonfinite2<BF>(w.y) | nonfinite2<BF>(w.z) | nonfinite2<BF>(w.w)) != 0;
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            const int dim = v_dim<KIND, D>(2 * i + d, g);
                            for (int k = 0; k < kRowsStep; ++k) {
                                const int at = KIND == kKvQ4_0 ? (dim / 32) * 16 + (dim & 15) : S::quant ? dim : 2 * dim;
                                const uint8_t *b = sv + k * S::vst + at;
                                float x;
                                if constexpr (S::quant)
                                    x = __half2float(__ushort_as_half(
                                        uint16_t(usable_scales<KIND>(__half_as_ushort(vs[k * (D / 32) + dim / 32])))));
                                else if constexpr (BF) x = __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t *>(b)) << 16);
                                else x = __half2float(*reinterpret_cast<const __half *>(b));
                                if constexpr (KIND == kKvQ8_0) x *= float(*reinterpret_cast<const int8_t *>(b));
                                if constexpr (KIND == kKvQ4_0) x *= float(int((dim & 16) ? *b >> 4 : *b & 15) - 8);
                                if (fabsf(x) < INFINITY) continue;
#pragma unroll
                                for (int t = 0; t < NT; ++t)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        if (key0 + k < seen[t][e]) o[t][i][2 * d + e] += x;
                            }
                        }
                    __syncwarp();
                    if constexpr (S::quant) {
                        for (int i = lane; i < kRowsStep * (D / 32); i += 32) {
                            const uint32_t y = usable_scales<KIND>(__half_as_ushort(vs[i]));
                            if ((y & 0x7FFFu) >= kOddScale<KIND>)
                                vs[i] = __ushort_as_half(uint16_t(KIND == kKvQ8_0 && (y & 0x7FFFu) == 0x6000u ? y - 1 : 0));
                        }
                    } else {
                        for (int i = lane; i < kRowsStep * S::ch * 4; i += 32) {
                            uint32_t *w = reinterpret_cast<uint32_t *>(sv + (i / (4 * S::ch)) * S::vst + (i % (4 * S::ch)) * 4);
                            *w &= ~nonfinite2<BF>(*w);
                        }
                    }
                    __syncwarp();
                }
            }

            // ---- O^T += V^T P^T
            auto pv = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                const uint32_t a[4] = {a0, a1, a2, a3};
#pragma unroll
                for (int t = 0; t < NT; ++t) mma16816<BF>(o[t][i], a, pb[t][0], pb[t][1]);
            };
            const int r4[4] = {2 * cq, 2 * cq + 1, 2 * cq + 8, 2 * cq + 9};  // the lane's keys
            uint32_t d01 = 0, d23 = 0;
            auto v_scales = [&](int dim) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = __half_as_ushort(vs[r4[j] * (D / 32) + dim / 32]);
                d01 = usable_scales<KIND>(h[0] | (h[1] << 16));
                d23 = usable_scales<KIND>(h[2] | (h[3] << 16));
            };
            auto q8_word = [&](int i, const uint32_t (&w)[4]) {  // 4 owned dimensions: tiles i, i + 1
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = __byte_perm(w[0], w[1], k ? 0x7362 : 0x5140) ^ 0x80808080u;
                    const uint32_t y = __byte_perm(w[2], w[3], k ? 0x7362 : 0x5140) ^ 0x80808080u;
                    pv(i + k, h2mul(q8_pair(x, 0x4140), d01), h2mul(q8_pair(x, 0x4342), d01),
                       h2mul(q8_pair(y, 0x4140), d23), h2mul(q8_pair(y, 0x4342), d23));
                }
            };
            auto q4_word = [&](int i, const uint32_t (&w)[4]) {  // 8 owned dimensions: tiles i .. i + 3
#pragma unroll
                for (int hi4 = 0; hi4 < 2; ++hi4)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t x[4], a[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[j] = hi4 ? q4_high(w[j] >> (8 * k)) : q4_low(w[j] >> (8 * k));
                        a[0] = __byte_perm(x[0], x[1], 0x5410);
                        a[1] = __byte_perm(x[0], x[1], 0x7632);
                        a[2] = __byte_perm(x[2], x[3], 0x5410);
                        a[3] = __byte_perm(x[2], x[3], 0x7632);
#pragma unroll
                        for (int j = 0; j < 4; ++j) a[j] = h2mul(hi4 ? q4_fix_high(a[j]) : q4_fix_low(a[j]), j < 2 ? d01 : d23);
                        pv(i + 2 * hi4 + k, a[0], a[1], a[2], a[3]);
                    }
            };
            if constexpr (KIND == kKvQ4_0 && D == 64) {
                v_scales(v_dim<KIND, D>(0, g));
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t *>(sv + r4[j] * S::vst + g * 4);
                q4_word(0, w);
            } else if constexpr ((KIND == kKvQ4_0 && D == 128) || (KIND == kKvQ8_0 && D == 64)) {
                v_scales(v_dim<KIND, D>(0, g));
                uint2 w2[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w2[j] = *reinterpret_cast<const uint2 *>(sv + r4[j] * S::vst + g * 8);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t w[4] = {k ? w2[0].y : w2[0].x, k ? w2[1].y : w2[1].x, k ? w2[2].y : w2[2].x,
                                           k ? w2[3].y : w2[3].x};
                    if constexpr (KIND == kKvQ4_0) q4_word(4 * k, w);
                    else q8_word(2 * k, w);
                }
            } else {
#pragma unroll
                for (int j8 = 0; j8 < S::ch / 8; ++j8) {
                    uint32_t w4[4][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(sv + r4[j] * S::vst + (g + 8 * j8) * 16);
                        w4[0][j] = x.x;
                        w4[1][j] = x.y;
                        w4[2][j] = x.z;
                        w4[3][j] = x.w;
                    }
                    if constexpr (S::quant) v_scales(v_dim<KIND, D>(j8 * (KIND == kKvQ8_0 ? 16 : 32), g));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t(&w)[4] = w4[k];
                        if constexpr (KIND == kKvQ8_0) q8_word(8 * j8 + 2 * k, w);
                        else if constexpr (KIND == kKvQ4_0) q4_word(16 * j8 + 4 * k, w);
                        else
                            pv(4 * j8 + k, __byte_perm(w[0], w[1], 0x5410), __byte_perm(w[0], w[1], 0x7632),
                               __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[2], w[3], 0x7632));
                    }
                }
            }
            if (++slot == S::stages) slot = 0;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- join the four warps: maxima and sums, then the outputs by rows
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
            }
        __syncthreads();  // the rings are free
        float *so = reinterpret_cast<float *>(ring), *sm = so + ROWS * (D + 4), *sl = sm + ROWS;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * t + 2 * cq + e;
                if (g == 0) {
                    sm[r] = m[t][e];
                    sl[r] = l[t][e];
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int d = 0; d < 2; ++d) so[r * (D + 4) + v_dim<KIND, D>(2 * i + d, g)] = o[t][i][2 * d + e];
            }
        __syncthreads();
        const bool begun = p.unit0 < lo, unfinished = p.unit0 + ntiles > hi;
        float *part = AttnPart<ROWS, D>::slot(io.part, blockIdx.x, begun ? 0 : 1);
        if (unfinished && !begun && threadIdx.x == 0)
            attn_open<ROWS, D>(io.part, gridDim.x)[blockIdx.x] =
                AttnOpen{shares.owner(p.unit0 + ntiles - 1) - int(blockIdx.x) + 1, q.s.q0, p.head * io.group, p.mt * ROWS, nrows, {}};
        for (int r = warp; r < nrows; r += kRowsWarps) {
            float mw[kRowsWarps], mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                mw[w] = reinterpret_cast<float *>(smem + w * S::per_warp)[ROWS * (D + 4) + r];
                mx = fmaxf(mx, mw[w]);
            }
            const float bs = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                mw[w] = ex2(mw[w] - bs);
                sum += mw[w] * reinterpret_cast<float *>(smem + w * S::per_warp)[ROWS * (D + 4) + ROWS + r];
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const unsigned rr = unsigned(p.mt) * ROWS + r;
            const int tok = int(by_group(io, rr)), h = p.head * io.group + int(rr - unsigned(tok) * io.group);
            uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(io.out) +
                                                         ((int64_t(q.s.q0) + tok) * io.heads + h) * D);
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kRowsWarps; ++w) {
                    const float2 y = *reinterpret_cast<const float2 *>(
                        reinterpret_cast<float *>(smem + w * S::per_warp) + r * (D + 4) + j * 64 + lane * 2);
                    x.x += mw[w] * y.x;
                    x.y += mw[w] * y.y;
                }
                if (begun || unfinished)
                    *reinterpret_cast<float2 *>(part + r * D + j * 64 + lane * 2) = x;
                else
                    dst[j * 32 + lane] = io.q_bf16 ? pack_bf16(x.x * inv, x.y * inv) : pack_half(x.x * inv, x.y * inv);
            }
            if ((begun || unfinished) && lane == 0) {
                part[ROWS * D + r] = mx;
                part[ROWS * D + ROWS + r] = sum;
            }
        }
        __syncthreads();  // before the rings are filled again
        attn_next<ROWS, kRowsKeys, kRowsCost>(c, bt, io, p, kseq);
    }
}

// CTAs of one SM: as many as its shared memory holds (1 KB of it goes to each CTA, and the kernel's
// static arrays) and its registers.
template <int KIND, int D, int NT> static constexpr int rows_occ() {
    using S = RowsShape<KIND, D, NT>;
    return std::min(S::min_ctas, 228 * 1024 / (S::smem + 2048));
}

template <int KIND, int D, int NT> struct RowsOps {
    using S = RowsShape<KIND, D, NT>;
    static int launch(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas, bool join,
                      cudaStream_t stream) {
        static std::atomic<uint64_t> allowed{0};
        cudaError_t e = attn_allow_smem(attn_rows_kernel<KIND, D, NT>, S::smem, &allowed);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        attn_rows_kernel<KIND, D, NT><<<ctas, kRowsWarps * 32, S::smem, stream>>>(c, bt, io);
        if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "paged_attention launch");
        return join ? attn_join_launch<S::rows, D>(io, ctas, stream) : ANVIL_OK;
    }
};

// The instance for a cache kind, head size and row tile (8 or 16): f.template operator()<KIND, D, NT>().
template <typename F> static auto rows_pick(int kind, int D, int nt, F f) {
#define ANVIL_ROWS_D(K)                                                                              \
    switch (D * 2 + nt - 1) {                                                                        \
    case 128: return f.template operator()<K, 64, 1>();                                              \
    case 129: return f.template operator()<K, 64, 2>();                                              \
    case 256: return f.template operator()<K, 128, 1>();                                             \
    case 257: return f.template operator()<K, 128, 2>();                                             \
    case 512: return f.template operator()<K, 256, 1>();                                             \
    default: return f.template operator()<K, 256, 2>();                                              \
    }
    switch (kind) {
    case kKvF16: ANVIL_ROWS_D(kKvF16)
    case kKvBF16: ANVIL_ROWS_D(kKvBF16)
    case kKvQ8_0: ANVIL_ROWS_D(kKvQ8_0)
    default: ANVIL_ROWS_D(kKvQ4_0)
    }
#undef ANVIL_ROWS_D
}

struct RowsOcc {
    template <int K, int D, int NT> int operator()() const { return rows_occ<K, D, NT>(); }
};
struct RowsLaunch {
    const KvCacheView &c;
    const KvBatchView &bt;
    const AttnIO &io;
    int ctas;
    bool join;
    cudaStream_t s;
    template <int K, int D, int NT> int operator()() const {
        return RowsOps<K, D, NT>::launch(c, bt, io, ctas, join, s);
    }
};

AttnTiles attn_rows_tiles(int kind, int D, int nt) {
    return AttnTiles{8 * nt, kRowsKeys, rows_pick(kind, D, nt, RowsOcc{})};
}

int attn_rows_launch(int kind, int D, int nt, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                     bool join, cudaStream_t s) {
    return rows_pick(kind, D, nt, RowsLaunch{c, bt, io, ctas, join, s});
}

int attn_rows_take_status() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_anvil_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (cudaMemcpyToSymbol(g_anvil_device_status, &z, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace anvil
