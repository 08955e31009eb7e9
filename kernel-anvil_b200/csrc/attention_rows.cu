// attention_rows.cu -- attention of few query rows (a decode step, a few drafted tokens) over the paged
// cache: row tiles of 16, bound by the bytes of the cache.
//
// Arithmetic: mma.sync m16n8k16 with fp32 sums.  S = Q K^T over 16 rows x 16 keys a warp and step,
// then the running maximum and sum, then O += P V with P rounded to the products' 16-bit type.  The
// legacy tensor path is enough here: at 16 rows a key costs 8 K flops against 272 bytes (Q8_0, D =
// 128), a third of what the path gives at the rate at which HBM delivers keys; tcgen05's smallest
// tile is 64 rows, of which a decode step fills 8.
//
// Loads: each warp owns a ring of stages of 16 keys (codes and scales of keys and values) filled
// by cp.async, 16 bytes a lane, through the page table, so that pages of any size look alike.  The
// ring keeps 48 KB and more in flight on an SM, without registers.  Codes are widened straight
// from the ring into MMA operands: the order of a product's inner dimension is free as long as
// both operands share it, so a lane takes 16 contiguous bytes of its key and feeds them to
// consecutive MMAs, and the query's operands are gathered to match once; for P V the same holds
// for the columns (a lane's values of V are contiguous, and the outputs' columns are put in order
// when they are stored).  Chunks are swizzled by row so that these reads hit every bank once.
//
// The four warps of a CTA take turns at the steps of a unit and keep maxima, sums and outputs of
// their own, joined through shared memory at the end of the unit.
#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "attention.cuh"

namespace anvil {

constexpr int kRowsTile = 16;   // query rows of a unit
constexpr int kRowsWarps = 4;
constexpr int kRowsStep = 16;   // keys of a warp's step
constexpr int kRowsKeys = 64;   // keys of a key tile: one step of each warp

template <int KIND, int D> struct RowsShape {
    static constexpr int rb = KvRow<KIND, D>::bytes;
    static constexpr int ch = rb / 16;                      // 16-byte chunks of a row
    static constexpr int sb = KvRow<KIND, D>::scales * 2;   // bytes of a row's scales
    static constexpr int stage = 2 * kRowsStep * (rb + sb) + 16;
    // as many stages as keep a CTA of four warps at about a third of an SM's shared memory (D = 256
    // in 16 bits: two stages are 132 KB), so that two or three CTAs stay resident
    static constexpr int stages = stage <= 2400 ? 6 : stage <= 4500 ? 4 : stage <= 8800 ? 3 : 2;
    static constexpr int ring = stage * stages;             // of one warp
    static constexpr int join = kRowsTile * (D + 4) * 4 + kRowsTile * 8;  // of one warp, reuses the ring
    static constexpr int per_warp = (ring > join ? ring : join + 15) & ~15;
    static constexpr int smem = kRowsWarps * per_warp;
    static constexpr bool bf16 = KIND == kKvBF16;
    static constexpr bool quant = KIND == kKvQ8_0 || KIND == kKvQ4_0;
    static constexpr bool q_in_regs = D <= 128;
};

__device__ __forceinline__ int k_chunk(int ch, int row, int chunk) { return ch >= 8 ? chunk ^ ((row & 1) << 2) : chunk; }
__device__ __forceinline__ int v_chunk(int ch, int row, int chunk) {
    return ch >= 8 ? chunk ^ (((row >> 1) & 3) << 1) : chunk;
}

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

__device__ __forceinline__ uint32_t h2sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t h2mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t h2fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t dup16(uint32_t x) { return __byte_perm(x, x, 0x1010); }

// ---- the dimension that a lane's operand stands for -------------------------------------------

// First of the 4 dimensions of QK step s for quad lane c; the operands hold (d, d+1), (d+2, d+3), or
// for Q4_0, whose nibbles come in pairs two bytes apart, (d, d+2), (d+1, d+3).
template <int KIND, int D> __device__ __forceinline__ int k_dim(int s, int c) {
    if constexpr (KIND == kKvQ8_0) return 16 * (c + 4 * (s >> 2)) + 4 * (s & 3);
    else if constexpr (KIND == kKvQ4_0) {
        if constexpr (D == 64) return 32 * (c >> 1) + 8 * (c & 1) + 4 * (s >> 1) + 16 * (s & 1);
        else return 32 * (c + 4 * (s >> 3)) + 4 * ((s & 7) >> 1) + 16 * (s & 1);
    } else return 8 * (c + 4 * (s >> 1)) + 4 * (s & 1);
}

// Dimension of PV column tile i for lane group g (0..7).
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

template <int KIND, int D>
__global__ void __launch_bounds__(kRowsWarps * 32, D == 256 ? 2 : 3)
    attn_rows_kernel(KvCacheView c, KvBatchView bt, AttnIO io) {
    using S = RowsShape<KIND, D>;
    constexpr int NS = D / 16;   // QK steps
    constexpr int NT = D / 8;    // PV column tiles
    constexpr bool BF = S::bf16;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ AttnScratch sc;
    __shared__ __align__(16) uint32_t sq[S::q_in_regs ? 1 : NS * 32 * 4];  // query operands where registers are short

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cq = lane & 3;
    uint8_t *ring = smem + warp * S::per_warp;
    const uint32_t ring_u = smem_u32(ring);

    const int64_t work = attn_locate<kRowsTile, kRowsKeys>(
        c, bt, io, &sc,
        [&](int64_t w) {
            const int n = attn_ctas(w, gridDim.x);
            return attn_share(w, min(int(blockIdx.x), n - 1), n);
        },
        blockIdx.x == 0);
    pdl_launch_dependents();
    const int ctas = attn_ctas(work, gridDim.x);
    if (int(blockIdx.x) >= ctas) return;
    const int64_t lo = attn_share(work, blockIdx.x, ctas), hi = attn_share(work, blockIdx.x + 1, ctas);
    AttnPos p = sc.pos;

    while (p.b < bt.batch && p.unit0 < hi) {
        const AttnSeq<kRowsTile, kRowsKeys> q(load_seq(bt, c, p.b), io);
        const int ntiles = q.key_tiles(p.mt), nkeys = q.keys(p.mt);
        const int t0 = int(max(lo - p.unit0, int64_t(0))), t1 = int(min(hi - p.unit0, int64_t(ntiles)));
        const int key_end = min(t1 * kRowsKeys, nkeys);
        const int nrows = int(min(int64_t(kRowsTile), int64_t(q.n) * q.group - int64_t(p.mt) * kRowsTile));

        // ---- the query's operands; seen[i], fac[i]: keys and score factor of rows g and g + 8
        int seen[2];
        float fac[2];
        uint32_t qa[S::q_in_regs ? NS : 1][4];
        {
            const uint16_t *src[2];
            int ex[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = g + 8 * i;
                const int64_t rr = int64_t(p.mt) * kRowsTile + r;
                const int tok = int(rr / q.group), h = p.head * q.group + int(rr - int64_t(tok) * q.group);
                seen[i] = r < nrows ? kv_seen(tok, q.n, q.s.kv, q.causal) : 0;
                src[i] = r < nrows ? static_cast<const uint16_t *>(io.q) + (q.s.q0 + tok) * io.q_row + h * io.q_head
                                   : nullptr;
            }
            if (S::quant && io.q_bf16) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t m = 0;
                    if (src[i])
#pragma unroll 4
                        for (int s = 0; s < NS; ++s) {
                            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(src[i] + k_dim<KIND, D>(s, cq)));
                            m = max(max(m, w.x & 0x7FFFu), (w.x >> 16) & 0x7FFFu);
                            m = max(max(m, w.y & 0x7FFFu), (w.y >> 16) & 0x7FFFu);
                        }
                    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    ex[i] = q_exponent(m << 16);
                }
            }
            if (!S::q_in_regs) __syncthreads();
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (!S::q_in_regs && (s & 3) != warp) continue;  // the warps share the gathering
                uint32_t a[4] = {};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint2 w = make_uint2(0, 0);
                    if (src[i]) w = __ldg(reinterpret_cast<const uint2 *>(src[i] + k_dim<KIND, D>(s, cq)));
                    if (S::quant && io.q_bf16) {
                        const float f = pow2i(ex[i]);
                        w.x = pack_half(__uint_as_float(w.x << 16) * f, __uint_as_float(w.x & 0xFFFF0000u) * f);
                        w.y = pack_half(__uint_as_float(w.y << 16) * f, __uint_as_float(w.y & 0xFFFF0000u) * f);
                    }
                    a[i] = KIND == kKvQ4_0 ? __byte_perm(w.x, w.y, 0x5410) : w.x;
                    a[2 + i] = KIND == kKvQ4_0 ? __byte_perm(w.x, w.y, 0x7632) : w.y;
                }
                if constexpr (S::q_in_regs) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) qa[s][i] = a[i];
                } else {
                    *reinterpret_cast<uint4 *>(&sq[(s * 32 + lane) * 4]) = make_uint4(a[0], a[1], a[2], a[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) fac[i] = io.scale_log2 * pow2i(-ex[i]);
            if (!S::q_in_regs) __syncthreads();
        }
        // every row of the unit sees the keys below this: no mask is needed there
        const int free_end = kv_seen(int(int64_t(p.mt) * kRowsTile / q.group), q.n, q.s.kv, q.causal);

        // ---- the ring
        const int step0 = t0 * 4 + warp;                   // step s covers keys 16 s .. 16 s + 15
        const int steps = (key_end + kRowsStep - 1) / kRowsStep;
        auto row_of = [&](int s) -> int64_t {              // cache row of key 16 s + lane, lanes 0..15
            const int key = s * kRowsStep + (lane & 15);
            if (s >= steps || key >= key_end) return -2;
            return kv_lookup(bt, c, p.b, key, p.head);
        };
        auto issue = [&](int s, int slot, int64_t row) {
            if (s < steps) {
                const uint32_t st = ring_u + slot * S::stage;
                const uint32_t bad = __ballot_sync(0xffffffffu, row == -1) & 0xFFFFu;
                if (lane == 0) {
                    *reinterpret_cast<uint32_t *>(ring + slot * S::stage + 2 * kRowsStep * (S::rb + S::sb)) = bad;
                    if (bad) flag_bad_page();
                }
#pragma unroll
                for (int j = 0; j < kRowsStep * S::ch / 32; ++j) {
                    const int i = lane + 32 * j, r = i / S::ch, ch = i % S::ch;
                    const int64_t rw = __shfl_sync(0xffffffffu, row, r);
                    const int64_t off = rw < 0 ? 0 : rw * S::rb + ch * 16;
                    const int n = rw < 0 ? 0 : 16;  // 0: the 16 bytes are zero-filled
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                     st + r * S::rb + k_chunk(S::ch, r, ch) * 16),
                                 "l"(c.k + off), "r"(n) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                     st + kRowsStep * S::rb + r * S::rb + v_chunk(S::ch, r, ch) * 16),
                                 "l"(c.v + off), "r"(n) : "memory");
                }
                if constexpr (S::quant) {
                    const int64_t rw = __shfl_sync(0xffffffffu, row, lane & 15);
                    const uint8_t *src = reinterpret_cast<const uint8_t *>(lane < 16 ? c.ks : c.vs);
                    const uint32_t dst = st + 2 * kRowsStep * S::rb + lane * S::sb;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst),
                                 "l"(src + (rw < 0 ? 0 : rw * S::sb)), "n"(S::sb), "r"(rw < 0 ? 0 : S::sb)
                                 : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

        int64_t next = row_of(step0);
#pragma unroll
        for (int i = 0; i < S::stages - 1; ++i) {
            const int64_t row = next;
            next = row_of(step0 + 4 * (i + 1));
            issue(step0 + 4 * i, i, row);
        }
        int slot = 0, fill = S::stages - 1;
        for (int s = step0; s < steps; s += 4) {
            {   // the slot that the last step freed
                const int64_t row = next;
                next = row_of(s + 4 * S::stages);
                __syncwarp();
                issue(s + 4 * (S::stages - 1), fill, row);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(S::stages - 1) : "memory");
            __syncwarp();
            const uint8_t *sk = ring + slot * S::stage, *sv = sk + kRowsStep * S::rb;
            const __half *ks = reinterpret_cast<const __half *>(sk + 2 * kRowsStep * S::rb);
            const __half *vs = ks + kRowsStep * KvRow<KIND, D>::scales;
            const uint32_t bad = *reinterpret_cast<const uint32_t *>(sk + 2 * kRowsStep * (S::rb + S::sb));
            (void)ks;
            (void)vs;

            // ---- S = Q K^T: sc2[t] are keys 8 t + 2 cq, + 1 for rows g and g + 8
            float sc2[2][4] = {};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = 8 * t + g;
                auto mul = [&](int s2, uint32_t b0, uint32_t b1) {
                    if constexpr (S::q_in_regs) {
                        mma16816<BF>(sc2[t], qa[s2], b0, b1);
                    } else {
                        const uint4 w = *reinterpret_cast<const uint4 *>(&sq[(s2 * 32 + lane) * 4]);
                        const uint32_t a[4] = {w.x, w.y, w.z, w.w};
                        mma16816<BF>(sc2[t], a, b0, b1);
                    }
                };
                auto scale_of = [&](int dim) {
                    return dup16(__half_as_ushort(ks[row * (D / 32) + dim / 32]));
                };
                if constexpr (KIND == kKvQ4_0 && D == 64) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(sk + row * S::rb + cq * 8);
                    const uint32_t d = scale_of(k_dim<KIND, D>(0, cq));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t u = j ? w.y : w.x;
                        mul(2 * j, h2mul(h2sub((u & 0x000F000Fu) | 0x64006400u, 0x64086408u), d),
                            h2mul(h2sub(((u >> 8) & 0x000F000Fu) | 0x64006400u, 0x64086408u), d));
                        mul(2 * j + 1, h2mul(h2fma((u & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u), d),
                            h2mul(h2fma(((u >> 8) & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u), d));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < S::ch / 4; ++j) {
                        const uint4 w4 = *reinterpret_cast<const uint4 *>(sk + row * S::rb + k_chunk(S::ch, row, cq + 4 * j) * 16);
                        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                        if constexpr (KIND == kKvQ8_0) {
                            const uint32_t d = scale_of(k_dim<KIND, D>(4 * j, cq));
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t u = w[i] ^ 0x80808080u;
                                mul(4 * j + i, h2mul(h2sub(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u), d),
                                    h2mul(h2sub(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u), d));
                            }
                        } else if constexpr (KIND == kKvQ4_0) {
                            const uint32_t d = scale_of(k_dim<KIND, D>(8 * j, cq));
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t u = w[i], u8 = u >> 8;
                                mul(8 * j + 2 * i, h2mul(h2sub((u & 0x000F000Fu) | 0x64006400u, 0x64086408u), d),
                                    h2mul(h2sub((u8 & 0x000F000Fu) | 0x64006400u, 0x64086408u), d));
                                mul(8 * j + 2 * i + 1, h2mul(h2fma((u & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u), d),
                                    h2mul(h2fma((u8 & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u), d));
                            }
                        } else {
                            mul(2 * j, w[0], w[1]);
                            mul(2 * j + 1, w[2], w[3]);
                        }
                    }
                }
            }

            // ---- scores, running maximum and sum
            const int key0 = s * kRowsStep;
            const bool masked = key0 + kRowsStep > free_end || bad != 0 || key0 + kRowsStep > key_end;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc2[t][j] *= fac[j >> 1];
            if (masked) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = 8 * t + 2 * cq + (j & 1);
                        if (key0 + k >= min(seen[j >> 1], key_end) || ((bad >> k) & 1)) sc2[t][j] = -INFINITY;
                    }
            }
            float mn[2], base[2];
            bool grew = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = fmaxf(fmaxf(sc2[0][2 * i], sc2[0][2 * i + 1]), fmaxf(sc2[1][2 * i], sc2[1][2 * i + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                mn[i] = fmaxf(m[i], x);
                base[i] = mn[i] == -INFINITY ? 0.0f : mn[i];
                grew |= mn[i] > m[i];
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = ex2(m[i] - base[i]);
                    l[i] *= a;
                    m[i] = mn[i];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[n][2 * i] *= a;
                        o[n][2 * i + 1] *= a;
                    }
                }
            }
            uint32_t pa[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = ex2(sc2[t][2 * i] - base[i]), y = ex2(sc2[t][2 * i + 1] - base[i]);
                    l[i] += x + y;
                    pa[2 * t + i] = BF ? pack_bf16(x, y) : pack_half(x, y);
                }

            // ---- O += P V.  Values that some row does not see must not reach it through 0 x NaN: in
            // a masked step non-finite values are taken out of the product and added by hand.
            uint32_t odd = 0;
            auto pv = [&](int i, uint32_t b0, uint32_t b1) {
                if (masked) {
                    const uint32_t n0 = nonfinite2<BF>(b0), n1 = nonfinite2<BF>(b1);
                    odd |= n0 | n1;
                    b0 &= ~n0;
                    b1 &= ~n1;
                }
                mma16816<BF>(o[i], pa, b0, b1);
            };
            const int r4[4] = {2 * cq, 2 * cq + 1, 2 * cq + 8, 2 * cq + 9};
            uint32_t d01 = 0, d23 = 0;
            auto v_scales = [&](int dim) {  // of the lane's four keys
                uint16_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = __half_as_ushort(vs[r4[j] * (D / 32) + dim / 32]);
                d01 = h[0] | (uint32_t(h[1]) << 16);
                d23 = h[2] | (uint32_t(h[3]) << 16);
            };
            auto q8_word = [&](int i, const uint32_t (&w)[4]) {  // column tiles i .. i + 3
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = __byte_perm(w[0], w[1], k ? 0x7362 : 0x5140) ^ 0x80808080u;
                    const uint32_t y = __byte_perm(w[2], w[3], k ? 0x7362 : 0x5140) ^ 0x80808080u;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t sel = e ? 0x4342u : 0x4140u;
                        pv(i + 2 * k + e, h2mul(h2sub(__byte_perm(x, 0x64646464u, sel), 0x64806480u), d01),
                           h2mul(h2sub(__byte_perm(y, 0x64646464u, sel), 0x64806480u), d23));
                    }
                }
            };
            auto q4_word = [&](int i, const uint32_t (&w)[4]) {  // column tiles i .. i + 7
#pragma unroll
                for (int hi = 0; hi < 2; ++hi)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t x[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[j] = ((w[j] >> (8 * k)) & (hi ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t sel = e ? 0x7632u : 0x5410u;
                            uint32_t b0 = __byte_perm(x[0], x[1], sel), b1 = __byte_perm(x[2], x[3], sel);
                            b0 = hi ? h2fma(b0, 0x2C002C00u, 0xD480D480u) : h2sub(b0, 0x64086408u);
                            b1 = hi ? h2fma(b1, 0x2C002C00u, 0xD480D480u) : h2sub(b1, 0x64086408u);
                            pv(i + 4 * hi + 2 * k + e, h2mul(b0, d01), h2mul(b1, d23));
                        }
                    }
            };
            if constexpr (KIND == kKvQ4_0 && D == 64) {
                v_scales(v_dim<KIND, D>(0, g));
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t *>(sv + r4[j] * S::rb + g * 4);
                q4_word(0, w);
            } else if constexpr ((KIND == kKvQ4_0 && D == 128) || (KIND == kKvQ8_0 && D == 64)) {
                v_scales(v_dim<KIND, D>(0, g));
                uint2 w2[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w2[j] = *reinterpret_cast<const uint2 *>(sv + r4[j] * S::rb + g * 8);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = k ? w2[j].y : w2[j].x;
                    if constexpr (KIND == kKvQ4_0) q4_word(8 * k, w);
                    else q8_word(4 * k, w);
                }
            } else {
#pragma unroll
                for (int j8 = 0; j8 < S::ch / 8; ++j8) {
                    uint4 w4[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w4[j] = *reinterpret_cast<const uint4 *>(sv + r4[j] * S::rb + v_chunk(S::ch, r4[j], g + 8 * j8) * 16);
                    if constexpr (S::quant) v_scales(v_dim<KIND, D>(j8 * (KIND == kKvQ8_0 ? 16 : 32), g));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = k == 0 ? w4[j].x : k == 1 ? w4[j].y : k == 2 ? w4[j].z : w4[j].w;
                        if constexpr (KIND == kKvQ8_0) q8_word(16 * j8 + 4 * k, w);
                        else if constexpr (KIND == kKvQ4_0) q4_word(32 * j8 + 8 * k, w);
                        else {
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                pv(8 * j8 + 2 * k + e, __byte_perm(w[0], w[1], e ? 0x7632 : 0x5410),
                                   __byte_perm(w[2], w[3], e ? 0x7632 : 0x5410));
                        }
                    }
                }
            }
            if (masked && __any_sync(0xffffffffu, odd != 0)) {
                // rare: every output of a row adds the non-finite values that the row sees, key by key
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int dim = v_dim<KIND, D>(i, 2 * cq + e);
                        for (int k = 0; k < kRowsStep; ++k) {
                            float x;
                            const int at = KIND == kKvQ4_0 ? (dim / 32) * 16 + (dim & 15) : S::quant ? dim : 2 * dim;
                            const uint8_t *b = sv + k * S::rb + v_chunk(S::ch, k, at >> 4) * 16 + (at & 15);
                            if constexpr (S::quant) x = __half2float(vs[k * (D / 32) + dim / 32]);
                            else if constexpr (BF) x = __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t *>(b)) << 16);
                            else x = __half2float(*reinterpret_cast<const __half *>(b));
                            if constexpr (KIND == kKvQ8_0) x *= float(*reinterpret_cast<const int8_t *>(b));
                            if constexpr (KIND == kKvQ4_0) x *= float(int((dim & 16) ? *b >> 4 : *b & 15) - 8);
                            // (what fp16 rounds to infinity is one in the product too)
                            if (!BF && fabsf(x) >= 65520.0f) x = copysignf(INFINITY, x);
                            if (!(fabsf(x) < INFINITY) && !((bad >> k) & 1))
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    if (key0 + k < min(seen[j], key_end)) o[i][2 * j + e] += x;
                        }
                    }
            }
            if (++slot == S::stages) slot = 0;
            if (++fill == S::stages) fill = 0;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- join the four warps: maxima and sums, then the outputs by rows
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        __syncthreads();  // the rings are free
        float *so = reinterpret_cast<float *>(ring), *sm = so + kRowsTile * (D + 4), *sl = sm + kRowsTile;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = g + 8 * i;
            if (cq == 0) {
                sm[r] = m[i];
                sl[r] = l[i];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) so[r * (D + 4) + v_dim<KIND, D>(n, 2 * cq + e)] = o[n][2 * i + e];
        }
        __syncthreads();
        const bool begun = p.unit0 < lo, unfinished = p.unit0 + ntiles > hi;
        float *part = AttnPart<kRowsTile, D>::slot(io.part, blockIdx.x, begun ? 0 : 1);
        for (int r = warp; r < nrows; r += kRowsWarps) {
            float mw[kRowsWarps], mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                mw[w] = reinterpret_cast<float *>(smem + w * S::per_warp)[kRowsTile * (D + 4) + r];
                mx = fmaxf(mx, mw[w]);
            }
            const float bs = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                mw[w] = ex2(mw[w] - bs);
                sum += mw[w] * reinterpret_cast<float *>(smem + w * S::per_warp)[kRowsTile * (D + 4) + kRowsTile + r];
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int64_t rr = int64_t(p.mt) * kRowsTile + r;
            const int tok = int(rr / q.group), h = p.head * q.group + int(rr - int64_t(tok) * q.group);
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
                part[kRowsTile * D + r] = mx;
                part[kRowsTile * D + kRowsTile + r] = sum;
            }
        }
        __syncthreads();  // before the rings are filled again
        attn_next(c, bt, io, p, q);
    }
}

template <int KIND, int D> static int launch_rows(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io,
                                                  int ctas, bool join, cudaStream_t stream) {
    using S = RowsShape<KIND, D>;
    const void *fn = reinterpret_cast<const void *>(attn_rows_kernel<KIND, D>);
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    attn_rows_kernel<KIND, D><<<ctas, kRowsWarps * 32, S::smem, stream>>>(c, bt, io);
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "paged_attention launch");
    if (!join) return ANVIL_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, kRowsTile / 4);
    cfg.blockDim = 128;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attn_join_kernel<kRowsTile, kRowsKeys, D>, c, bt, io);
    return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "paged_attention join launch");
}

// CTAs of one SM: as many as its shared memory holds (1 KB of it goes to each CTA, and the kernel's
// static arrays), at most 3 of the kernels' 168 registers or 2 of D = 256's 255.
template <int KIND, int D> static int rows_ctas_per_sm() {
    using S = RowsShape<KIND, D>;
    return std::min(D == 256 ? 2 : 3, 228 * 1024 / (S::smem + 2048 + (S::q_in_regs ? 0 : D * 32)));
}

template <int KIND> static int rows_dim(int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                                        bool join, cudaStream_t s) {
    return D == 64 ? launch_rows<KIND, 64>(c, bt, io, ctas, join, s)
         : D == 128 ? launch_rows<KIND, 128>(c, bt, io, ctas, join, s)
                    : launch_rows<KIND, 256>(c, bt, io, ctas, join, s);
}
template <int KIND> static int rows_occ(int D) {
    return D == 64 ? rows_ctas_per_sm<KIND, 64>() : D == 128 ? rows_ctas_per_sm<KIND, 128>() : rows_ctas_per_sm<KIND, 256>();
}

int attn_rows_ctas_per_sm(int kind, int D) {
    return kind == kKvF16 ? rows_occ<kKvF16>(D) : kind == kKvBF16 ? rows_occ<kKvBF16>(D)
         : kind == kKvQ8_0 ? rows_occ<kKvQ8_0>(D) : rows_occ<kKvQ4_0>(D);
}
int64_t attn_rows_part_bytes(int D) { return int64_t(kRowsTile) * (D + 2) * 4 * 2; }  // per CTA

int attn_rows_launch(int kind, int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                     bool join, cudaStream_t s) {
    switch (kind) {
    case kKvF16: return rows_dim<kKvF16>(D, c, bt, io, ctas, join, s);
    case kKvBF16: return rows_dim<kKvBF16>(D, c, bt, io, ctas, join, s);
    case kKvQ8_0: return rows_dim<kKvQ8_0>(D, c, bt, io, ctas, join, s);
    default: return rows_dim<kKvQ4_0>(D, c, bt, io, ctas, join, s);
    }
}

int attn_rows_take_status() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_anvil_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (cudaMemcpyToSymbol(g_anvil_device_status, &z, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace anvil
