// attention_tile.cu -- attention of many query rows (chunks and whole prompts) over the paged cache on
// the fifth-generation tensor cores.
//
// A CTA, one per SM, works on a unit of 256 query rows (two tiles of 128; one tile where head_dim is
// 256) against tiles of 128 keys (64), with S and O in tensor memory:
//   S = Q K^T          tcgen05.mma, both operands in shared memory
//   P = 2^(S f - m)    one thread a row: no shuffles; P goes back over S in 16 bits
//   O += P V           tcgen05.mma with P from tensor memory, V transposed by its descriptor
// Warp roles: warps 0-3 and 4-7 are the softmax of the two row tiles, which alternate so that one
// tile's exponentials run under the other's products; warps 8-11 bring keys and values through
// the page table into a ring of buffers in the 128-byte swizzled layout, widening quantised codes
// to fp16 on the way; warp 12 issues every product.  All hand-over is by mbarriers; each wait is
// bounded and a failure makes the later ones return at once.
//
// The running maximum is only raised when it grew by more than 2^8 (weights may then reach 2^8, which
// fp16 and fp32 hold without loss), so that O is rescaled a few times a row instead of at every tile.
#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "attention.cuh"

namespace anvil {

constexpr int kTileThreads = 512;
constexpr int kTileCost = 4;        // beginning and ending a unit, in key tiles
constexpr float kTileSlack = 8.0f;  // log2 of how far weights may exceed 1

template <int KIND, int D> struct TileShape {
    static constexpr int nq = D == 256 ? 1 : 2;         // row tiles of 128
    static constexpr int rows = 128 * nq;
    static constexpr int keys = D == 256 ? 64 : 128;
    static constexpr int blocks = D / 64;               // 64-value column blocks of an operand
    static constexpr int q_bytes = rows * D * 2;
    static constexpr int buf = keys * D * 2;            // one buffer: keys or values of a tile
    static constexpr int nbuf = D == 64 ? 6 : 4;
    static constexpr int smem = 1024 + q_bytes + nbuf * buf;
    static constexpr bool bf16 = KIND == kKvBF16;
    static constexpr bool quant = KIND == kKvQ8_0 || KIND == kKvQ4_0;
    // tensor memory columns: S of the two tiles (or two turns of one), then O
    static constexpr int s_cols = keys, o_col = 2 * keys, o_cols = D;
};

// ---- tcgen05 ----------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    // start, leading and stride byte offsets in 16-byte units; version 1; 128-byte swizzle
    return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(lbo >> 4) << 16) | (uint64_t(sbo >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of this thread's row
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
                 "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : R8(v, 0), R8(v, 8), R8(v, 16), R8(v, 24) : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
                 "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::W8(v, 0), W8(v, 8), W8(v, 16), W8(v, 24), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::W8(v, 0),
                 W8(v, 8), "r"(addr)
                 : "memory");
}
#undef R8
#undef W8

// ---- hand-over --------------------------------------------------------------------------------

struct TileShared {
    AttnScratch sc;
    uint64_t full[6], empty[6], q_full[2], s_full[2], p_full[2], pv_done[2], drain;
    uint32_t tmem;
    int failed;             // a wait gave up: later ones do not wait
    int dirty[8];           // [unit % 8] = unit where non-finite values were taken out of its value tiles
    uint32_t bad[4][4];     // [tile % 4]: keys without a page
    int64_t row[2][128];    // loader: cache rows of a key tile, by parity
};

// try_wait that may sleep for up to 20 us: 13 warps that poll take issue slots from the softmax
__device__ __forceinline__ bool mbar_try_wait_long(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ void tile_wait(TileShared *sh, uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
    if (mbar_try_wait_long(bar, parity)) return;
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait_long(bar, parity)) {
        if (*reinterpret_cast<volatile int *>(&sh->failed)) return;
        if (global_timer_ns() - t0 > limit_ns) {
            *reinterpret_cast<volatile int *>(&sh->failed) = 1;
            atomicOr(&g_anvil_device_status, kStatusMbarTimeout);
            return;
        }
    }
}
__device__ __forceinline__ void loader_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A unit's share of this CTA: key tiles [t0, t1) and the limits of its masks.
template <int KIND, int D> struct TileUnit {
    using S = TileShape<KIND, D>;
    AttnSeq<S::rows, S::keys> q;
    int ntiles, t0, t1, key_end, nrows, free_end;
    __device__ __forceinline__ TileUnit(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, const AttnPos &p,
                                        int64_t lo, int64_t hi)
        : q(load_seq(bt, c, p.b), io) {
        ntiles = q.key_tiles(p.mt);
        t0 = int(max(lo - p.unit0, int64_t(0)));
        t1 = int(min(hi - p.unit0, int64_t(ntiles)));
        key_end = min(t1 * S::keys, q.keys(p.mt));
        nrows = int(min(int64_t(S::rows), int64_t(unsigned(q.n) * unsigned(q.group) - unsigned(p.mt) * S::rows)));
        // every row of the unit sees the keys below this
        free_end = min(key_end, kv_seen(int(unsigned(p.mt) * S::rows / unsigned(q.group)), q.n, q.s.kv, q.causal));
    }
};

template <int KIND, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attn_tile_kernel(KvCacheView c, KvBatchView bt, AttnIO io, uint64_t limit_ns) {
    using S = TileShape<KIND, D>;
    constexpr bool BF = S::bf16;
    extern __shared__ uint8_t dyn[];
    __shared__ TileShared sh;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
    uint8_t *sq = base, *sbuf = base + S::q_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int64_t work = attn_locate<S::rows, S::keys, kTileCost>(
        c, bt, io, &sh.sc, [&](const AttnShares &s) { return s.begin(min(int(blockIdx.x), s.ctas - 1)); }, blockIdx.x == 0);
    pdl_launch_dependents();
    const AttnShares shares(work, gridDim.x);
    if (int(blockIdx.x) >= shares.ctas) return;
    const int64_t lo = shares.begin(blockIdx.x), hi = shares.begin(blockIdx.x + 1);
    AttnPos p = sh.sc.pos;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::nbuf; ++i) {
            mbar_init(&sh.full[i], 4);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 4);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.pv_done[i], 1);
        }
        mbar_init(&sh.drain, 1);
        mbar_fence_init();
        sh.failed = 0;
        for (int i = 0; i < 8; ++i) sh.dirty[i] = 0;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sh.tmem);

    if (warp < 8) {
        // ================= softmax: thread = row of tile w ==========================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        const int w = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        uint32_t ns[2] = {0, 0}, npv = 0;   // completions waited for: S by buffer, PV of this tile
        int unit = 0, seq = 0;              // units and key tiles so far, counted alike in every role
        if (w < S::nq)
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(c, bt, io, p, lo, hi);
                ++unit;
                if (w * 128 < u.nrows) {
                    // ---- this row's query, into the swizzled operand
                    const int ur = w * 128 + r;
                    const bool live = ur < u.nrows;
                    const unsigned rr = unsigned(p.mt) * S::rows + ur;
                    const int tok = int(rr / unsigned(u.q.group)), h = p.head * u.q.group + int(rr - unsigned(tok) * u.q.group);
                    const int seen = live ? min(u.key_end, kv_seen(tok, u.q.n, u.q.s.kv, u.q.causal)) : 0;
                    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(io.q) +
                                                                       (u.q.s.q0 + int64_t(tok)) * io.q_row + h * io.q_head);
                    int ex = 0;
                    if (S::quant && io.q_bf16 && live) {
                        uint32_t m = 0;
#pragma unroll 8
                        for (int i = 0; i < D / 8; ++i) {
                            const uint4 x = __ldg(src + i);
                            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) m = max(max(m, y[j] & 0x7FFFu), (y[j] >> 16) & 0x7FFFu);
                        }
                        ex = q_exponent(m << 16);
                    }
                    const float up = pow2i(ex);
                    uint8_t *dq = sq + w * 128 * 128 + r * 128;
#pragma unroll 8
                    for (int i = 0; i < D / 8; ++i) {
                        uint4 x = live ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
                        if (S::quant && io.q_bf16) {
                            uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                y[j] = pack_half(__uint_as_float(y[j] << 16) * up, __uint_as_float(y[j] & 0xFFFF0000u) * up);
                            x = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                        if (io.scale_log2 < 0.0f) {  // a negative scale: -q, so that the largest score stays the largest
                            x.x ^= 0x80008000u;
                            x.y ^= 0x80008000u;
                            x.z ^= 0x80008000u;
                            x.w ^= 0x80008000u;
                        }
                        *reinterpret_cast<uint4 *>(dq + (i >> 3) * (S::rows * 128) + (((i & 7) ^ (r & 7)) << 4)) = x;
                    }
                    // (above zero, so that a masked score stays -inf)
                    const float fac = fmaxf(fabsf(io.scale_log2) * pow2i(-ex), 1e-36f);
                    fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.q_full[w]);

                    float m = -INFINITY, l = 0.0f;
                    for (int t = u.t0; t < u.t1; ++t) {
                        const int x = S::nq == 2 ? w : (t - u.t0) & 1;
                        const uint32_t ts = tmem + lanes + x * S::s_cols, to = tmem + lanes + S::o_col + (S::nq == 2 ? w * S::o_cols : 0);
                        tile_wait(&sh, &sh.s_full[x], ns[x]++ & 1, limit_ns);
                        __syncwarp();
                        fence_after();
                        const int key0 = t * S::keys;
                        uint32_t any_bad = 0;
#pragma unroll
                        for (int i = 0; i < S::keys / 32; ++i) any_bad |= sh.bad[(seq + t - u.t0) & 3][i];
                        const bool masked = key0 + S::keys > u.free_end || any_bad;
                        // 32 scores of this row; S is read twice rather than held in 128 registers
                        auto mask = [&](uint32_t *s, int i) {
                            const uint32_t bad = sh.bad[(seq + t - u.t0) & 3][i];
                            const int left = seen - key0 - 32 * i;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j >= left || ((bad >> j) & 1)) s[j] = 0xFF800000u;
                        };
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < S::keys / 32; i += 2) {
                            uint32_t s[64];
                            tmem_ld32(ts + 32 * i, s);
                            tmem_ld32(ts + 32 * i + 32, s + 32);
                            wait_ld();
                            if (masked) {
                                mask(s, i);
                                mask(s + 32, i + 1);
                            }
#pragma unroll
                            for (int j = 0; j < 64; j += 2)
                                mx[(j >> 1) & 3] = max3(mx[(j >> 1) & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
                        }
                        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        const float mt = top * fac;
                        const bool first = t == u.t0;
                        const bool raise = mt > m + kTileSlack || (m == -INFINITY && mt > m);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float mn = raise ? mt : m;
                            const float a = raise ? ex2(m - mn) : 1.0f;
                            if (!first) {
                                tile_wait(&sh, &sh.pv_done[w], (npv - 1) & 1, limit_ns);
                                __syncwarp();
                                fence_after();
#pragma unroll 1
                                for (int i = 0; i < D / 32; ++i) {
                                    uint32_t v[32];
                                    tmem_ld32(to + 32 * i, v);
                                    wait_ld();
#pragma unroll
                                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * a);
                                    tmem_st32(to + 32 * i, v);
                                }
                            }
                            l *= a;
                            m = mn;
                        }
                        const float nb = m == -INFINITY ? 0.0f : -m;
                        const uint64_t fac2 = pack2(fac, fac), nb2 = pack2(nb, nb);
                        uint64_t sum[2] = {0, 0};
                        uint32_t s[2][32];
                        tmem_ld32(ts, s[0]);
#pragma unroll
                        for (int i = 0; i < S::keys / 32; ++i) {
                            uint32_t *x = s[i & 1];
                            wait_ld();
                            if (i + 1 < S::keys / 32) tmem_ld32(ts + 32 * (i + 1), s[(i + 1) & 1]);
                            if (masked) mask(x, i);
                            uint32_t y[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float e0, e1;
                                unpack2(fma2(pack2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), fac2, nb2), e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                                sum[j & 1] = add2(sum[j & 1], pack2(e0, e1));
                                y[j] = BF ? pack_bf16(e0, e1) : pack_half(e0, e1);
                            }
                            tmem_st16(ts + 16 * i, y);  // over scores already read
                        }
                        {
                            float a0, a1;
                            unpack2(add2(sum[0], sum[1]), a0, a1);
                            l += a0 + a1;
                        }
                        wait_st();
                        // A wait on a parity holds only while the phase before is known to be over.  Where scores run
                        // ahead of the last tile's P V (one row tile) nothing else has shown that yet.
                        if (S::nq == 1 && !first) tile_wait(&sh, &sh.pv_done[w], (npv - 1) & 1, limit_ns);
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_full[w]);
                        ++npv;
                    }

                    // ---- the unit's outputs, or this share's part of them
                    tile_wait(&sh, &sh.pv_done[w], (npv - 1) & 1, limit_ns);
                    fence_after();
                    const uint32_t to = tmem + lanes + S::o_col + (S::nq == 2 ? w * S::o_cols : 0);
                    const bool begun = p.unit0 < lo, unfinished = p.unit0 + u.ntiles > hi;
                    const bool dirty = *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) == unit;
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    float *part = AttnPart<S::rows, D>::slot(io.part, blockIdx.x, begun ? 0 : 1);
                    uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(io.out) +
                                                                 ((int64_t(u.q.s.q0) + tok) * io.heads + h) * D);
#pragma unroll 1
                    for (int i = 0; i < D / 32; ++i) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld32(to + 32 * i, v);
                        wait_ld();
                        if (dirty) {
                            // non-finite values of the masked tiles, which left the product: to the rows that see them
                            for (int k = max(u.t0, u.free_end / S::keys) * S::keys; k < seen; ++k) {
                                const int64_t row = kv_lookup(bt, c, p.b, k, p.head);
#pragma unroll 1
                                for (int j = 0; j < 32 && row >= 0; ++j) {
                                    const float y = kv_value<KIND, D>(c.v, c.vs, row, 32 * i + j);
                                    if (!(fabsf(y) < INFINITY)) {
#pragma unroll
                                        for (int e = 0; e < 32; ++e)
                                            if (e == j) v[e] = __float_as_uint(__uint_as_float(v[e]) + y);
                                    }
                                }
                            }
                        }
                        if (live && (begun || unfinished)) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *reinterpret_cast<uint4 *>(part + ur * D + 32 * i + 4 * j) =
                                    make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        } else if (live) {
                            uint32_t y[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float e0 = __uint_as_float(v[2 * j]) * inv, e1 = __uint_as_float(v[2 * j + 1]) * inv;
                                y[j] = io.q_bf16 ? pack_bf16(e0, e1) : pack_half(e0, e1);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                *reinterpret_cast<uint4 *>(dst + 16 * i + 4 * j) =
                                    make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                        }
                    }
                    if (live && (begun || unfinished)) {
                        part[S::rows * D + ur] = m;
                        part[S::rows * D + S::rows + ur] = l;
                    }
                    fence_before();
                }
                seq += u.t1 - u.t0;
                attn_next<S::rows, S::keys, kTileCost>(c, bt, p, u.q);
            }
    } else if (warp < 12) {
        // ================= loader: 128 threads, keys then values of each tile ========================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        const int tid = threadIdx.x - 256;
        uint32_t nb = 0;        // buffers filled
        int pending = -1;       // buffer whose copies were not announced yet
        int unit = 0, seq = 0;
        auto announce = [&](int b) {
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.full[b]);
        };
        while (p.b < bt.batch && p.unit0 < hi) {
            const TileUnit<KIND, D> u(c, bt, io, p, lo, hi);
            ++unit;
            for (int t = u.t0; t < u.t1; ++t, ++seq) {
                // rows of this tile's keys
                const int key = t * S::keys + tid;
                int64_t row = -2;
                if (tid < S::keys && key < u.key_end) row = kv_lookup(bt, c, p.b, key, p.head);
                if (tid < S::keys) sh.row[seq & 1][tid] = row;
                const uint32_t bad = __ballot_sync(0xffffffffu, row == -1);
                if (lane == 0) {
                    sh.bad[seq & 3][tid >> 5] = bad;
                    if (bad) flag_bad_page();
                }
                loader_sync();
                const bool check = t * S::keys + S::keys > u.free_end;
                for (int kv = 0; kv < 2; ++kv, ++nb) {
                    const int b = nb % S::nbuf;
                    if (nb >= S::nbuf) {
                        const uint32_t parity = (nb / S::nbuf - 1) & 1;
                        // (a product may wait for the pending buffer before it frees this one)
                        if (!S::quant && pending >= 0 && !__all_sync(0xffffffffu, mbar_try_wait(&sh.empty[b], parity))) {
                            asm volatile("cp.async.wait_group 0;" ::: "memory");
                            announce(pending);
                            pending = -1;
                        }
                        tile_wait(&sh, &sh.empty[b], parity, limit_ns);
                    }
                    uint8_t *dst = sbuf + b * S::buf;
                    const uint8_t *src = kv ? c.v : c.k;
                    if constexpr (!S::quant) {
                        constexpr int CH = D / 8;  // chunks of a row
#pragma unroll 4
                        for (int i = tid; i < S::keys * CH; i += 128) {
                            const int r = i / CH, ch = i % CH;
                            const int64_t rw = sh.row[seq & 1][r];
                            const uint32_t to = smem_u32(dst + (ch >> 3) * (S::keys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to),
                                         "l"(src + max(rw, int64_t(0)) * (2 * D) + ch * 16), "r"(rw < 0 ? 0 : 16)
                                         : "memory");
                        }
                        asm volatile("cp.async.commit_group;" ::: "memory");
                        if (kv && check) {
                            // a masked tile's values: what is not finite leaves the product (see the outputs)
                            asm volatile("cp.async.wait_group 0;" ::: "memory");
                            for (int i = tid; i < S::keys * CH; i += 128) {
                                const int r = i / CH, ch = i % CH;
                                uint32_t *w4 = reinterpret_cast<uint32_t *>(dst + (ch >> 3) * (S::keys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint32_t bits = nonfinite2<BF>(w4[j]);
                                    if (bits) {
                                        w4[j] &= ~bits;
                                        *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) = unit;
                                    }
                                }
                            }
                        }
                        if (pending >= 0) {
                            asm volatile("cp.async.wait_group 1;" ::: "memory");
                            announce(pending);
                        }
                        pending = b;
                    } else {
                        // 16 bytes of codes a turn: 16 (Q8_0) or 32 (Q4_0) values, two or four chunks
                        constexpr int RB = KvRow<KIND, D>::bytes, CH = RB / 16, N = S::keys * CH / 128;
                        constexpr int OUT = KIND == kKvQ8_0 ? 2 : 4, VALS = 8 * OUT;
                        const __half *scales = kv ? c.vs : c.ks;
                        // eight lanes store two rows of four chunks where rows have them: distinct banks
                        const int in = tid % (2 * CH);
                        const int ch = CH >= 8 ? (in & 3) | ((in >> 3) << 2) : tid % CH;
                        const int r0 = CH >= 8 ? tid / (2 * CH) * 2 + ((in >> 2) & 1) : tid / CH;
                        uint4 w[N];
                        uint16_t d[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const int64_t rw = sh.row[seq & 1][r0 + i * (128 / CH)];
                            w[i] = make_uint4(0, 0, 0, 0);
                            d[i] = 0;
                            if (rw >= 0) {
                                w[i] = __ldg(reinterpret_cast<const uint4 *>(src + rw * RB + ch * 16));
                                d[i] = __ldg(reinterpret_cast<const unsigned short *>(scales) + rw * (D / 32) + ch * VALS / 32);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const int r = r0 + i * (128 / CH);
                            uint32_t d2 = d[i] | (uint32_t(d[i]) << 16);
                            if (kv && check && nonfinite2<false>(d2)) {
                                d2 = 0;
                                *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) = unit;
                            }
                            const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                            uint32_t y[4 * OUT];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if constexpr (KIND == kKvQ8_0) {
                                    const uint32_t v = x[j] ^ 0x80808080u;
                                    y[2 * j] = h2mul(h2sub(__byte_perm(v, 0x64646464u, 0x4140), 0x64806480u), d2);
                                    y[2 * j + 1] = h2mul(h2sub(__byte_perm(v, 0x64646464u, 0x4342), 0x64806480u), d2);
                                } else {
                                    const uint32_t a = x[j] & 0x0F0F0F0Fu, e = (x[j] >> 4) & 0x0F0F0F0Fu;
                                    y[2 * j] = h2mul(h2sub(__byte_perm(a, 0x64646464u, 0x4140), 0x64086408u), d2);
                                    y[2 * j + 1] = h2mul(h2sub(__byte_perm(a, 0x64646464u, 0x4342), 0x64086408u), d2);
                                    y[8 + 2 * j] = h2mul(h2sub(__byte_perm(e, 0x64646464u, 0x4140), 0x64086408u), d2);
                                    y[8 + 2 * j + 1] = h2mul(h2sub(__byte_perm(e, 0x64646464u, 0x4342), 0x64086408u), d2);
                                }
                            }
#pragma unroll
                            for (int j = 0; j < OUT; ++j) {
                                const int oc = ch * OUT + j;
                                *reinterpret_cast<uint4 *>(dst + (oc >> 3) * (S::keys * 128) + r * 128 + (((oc & 7) ^ (r & 7)) << 4)) =
                                    make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                            }
                        }
                        announce(b);
                    }
                }
            }
            attn_next<S::rows, S::keys, kTileCost>(c, bt, p, u.q);
        }
        if (!S::quant && pending >= 0) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            announce(pending);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 12 && lane == 0) {
            // ================= products ================================================================
            constexpr uint32_t fmt = BF ? 1 : 0;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
            constexpr uint32_t id_qk = idesc0 | (uint32_t(S::keys / 8) << 17);
            constexpr uint32_t id_pv = idesc0 | (1u << 16) | (uint32_t(D / 8) << 17);  // V: its columns are contiguous
            uint32_t nb = 0, nq[2] = {0, 0}, np[2] = {0, 0};
            auto qk = [&](int w, int x, uint32_t b) {
                const uint32_t a = smem_u32(sq) + w * 128 * 128, k = smem_u32(sbuf) + b * S::buf;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    mma_ss(tmem + x * S::s_cols, smem_desc(a + (i >> 2) * (S::rows * 128) + (i & 3) * 32, 16, 1024),
                           smem_desc(k + (i >> 2) * (S::keys * 128) + (i & 3) * 32, 16, 1024), id_qk, i > 0);
                mma_commit(&sh.s_full[x]);
            };
            auto pv = [&](int w, int x, uint32_t b, bool acc) {
                const uint32_t v = smem_u32(sbuf) + b * S::buf;
#pragma unroll
                for (int i = 0; i < S::keys / 16; ++i)
                    mma_ts(tmem + S::o_col + (S::nq == 2 ? w * S::o_cols : 0), tmem + x * S::s_cols + i * 8,
                           smem_desc(v + i * 2048, S::keys * 128, 1024), id_pv, acc || i > 0);
                mma_commit(&sh.pv_done[w]);
            };
            auto wait_full = [&](uint32_t n) {
                tile_wait(&sh, &sh.full[n % S::nbuf], (n / S::nbuf) & 1, limit_ns);
                fence_after();
            };
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(c, bt, io, p, lo, hi);
                const int tiles = u.t1 - u.t0, active = S::nq == 2 && u.nrows > 128 ? 2 : 1;
#pragma unroll
                for (int w = 0; w < S::nq; ++w)
                    if (w < active) tile_wait(&sh, &sh.q_full[w], nq[w]++ & 1, limit_ns);
                wait_full(nb);
#pragma unroll
                for (int w = 0; w < S::nq; ++w)
                    if (w < active) qk(w, w, nb % S::nbuf);
                mma_commit(&sh.empty[nb % S::nbuf]);
                for (int i = 0; i < tiles; ++i) {
                    const uint32_t bv = nb + 2 * i + 1, bk = bv + 1;
                    const bool more = i + 1 < tiles;
                    if (S::nq == 1 && more) {  // the next scores go to the other turn's columns
                        wait_full(bk);
                        qk(0, (i + 1) & 1, bk % S::nbuf);
                        mma_commit(&sh.empty[bk % S::nbuf]);
                    }
#pragma unroll
                    for (int w = 0; w < S::nq; ++w) {
                        if (w >= active) continue;
                        if (w == 0) wait_full(bv);
                        tile_wait(&sh, &sh.p_full[w], np[w]++ & 1, limit_ns);
                        fence_after();
                        pv(w, S::nq == 2 ? w : i & 1, bv % S::nbuf, i > 0);
                        if (S::nq == 2 && more) {
                            if (w == 0) wait_full(bk);
                            qk(w, w, bk % S::nbuf);
                        }
                    }
                    mma_commit(&sh.empty[bv % S::nbuf]);
                    if (S::nq == 2 && more) mma_commit(&sh.empty[bk % S::nbuf]);
                }
                nb += 2 * tiles;
                attn_next<S::rows, S::keys, kTileCost>(c, bt, p, u.q);
            }
            mma_commit(&sh.drain);
            tile_wait(&sh, &sh.drain, 0, limit_ns);
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (warp == 12) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

template <int KIND, int D> static int launch_tile(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                                                  bool join, cudaStream_t stream) {
    using S = TileShape<KIND, D>;
    cudaError_t e = cudaFuncSetAttribute(attn_tile_kernel<KIND, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    attn_tile_kernel<KIND, D><<<ctas, kTileThreads, S::smem, stream>>>(c, bt, io, wait_limit_ns());
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "paged_attention launch");
    return join ? attn_join_launch<S::rows, S::keys, kTileCost, D>(c, bt, io, ctas, stream) : ANVIL_OK;
}

template <int KIND> static int tile_dim(int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                                        bool join, cudaStream_t s) {
    return D == 64 ? launch_tile<KIND, 64>(c, bt, io, ctas, join, s)
         : D == 128 ? launch_tile<KIND, 128>(c, bt, io, ctas, join, s)
                    : launch_tile<KIND, 256>(c, bt, io, ctas, join, s);
}

AttnTiles attn_tile_tiles(int D) { return D == 256 ? AttnTiles{128, 64, 1} : AttnTiles{256, 128, 1}; }

int attn_tile_launch(int kind, int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas, bool join,
                     cudaStream_t s) {
    switch (kind) {
    case kKvF16: return tile_dim<kKvF16>(D, c, bt, io, ctas, join, s);
    case kKvBF16: return tile_dim<kKvBF16>(D, c, bt, io, ctas, join, s);
    case kKvQ8_0: return tile_dim<kKvQ8_0>(D, c, bt, io, ctas, join, s);
    default: return tile_dim<kKvQ4_0>(D, c, bt, io, ctas, join, s);
    }
}

int attn_tile_take_status() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_anvil_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (cudaMemcpyToSymbol(g_anvil_device_status, &z, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace anvil
