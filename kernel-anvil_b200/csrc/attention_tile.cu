// attention_tile.cu -- attention of many query rows (chunks and whole prompts) over the paged cache on
// the fifth-generation tensor cores.
//
// A CTA, one per SM, works on a unit of 256 query rows (two tiles of 128; one tile where head_dim is
// 256) against tiles of 64 keys, with S and O in tensor memory:
//   S = Q K^T          tcgen05.mma, both operands in shared memory
//   P = 2^(S f - m)    one thread a row: no shuffles; P goes back over S in 16 bits
//   O += P V           tcgen05.mma with P from tensor memory, V transposed by its descriptor
// S has two turns of 64 columns a row tile, so the scores of the next keys are there when the weights of
// the last ones are done, and the softmax never waits for a product that waits for it.  (Tiles of 128
// keys fill tensor memory with one turn, P over S: the chain softmax, P V, Q K^T, softmax then left
// both sides idle half of the time: 2.68 against 2.19 ms for 2048 rows of 64 heads over 30049 keys of Q8_0.)
// Warp roles: warps 0-3 and 4-7 are the softmax of the two row tiles; warps 8-11 bring keys and values
// through the page table into a ring of buffers in the 128-byte swizzled layout, widening quantised
// codes to fp16 on the way, and a unit's queries while the softmax is at the unit before; warps 12 and 13
// issue the products of a row tile each (one warp for both took 1900 cycles a tile to issue and
// hand over, more than the products took); warp 14 fetches quantised codes.  All hand-over is by mbarriers;
// each wait is bounded and a failure makes the later ones return at once.
//
// Weights are taken by a reference, which a row's first tile sets near its maximum; it is raised, and O rescaled,
// only when a tile's weights sum to more than fp16 holds, which the sum that is taken anyway shows: most tiles are
// never searched for their maximum.  P is rounded to the products' 16-bit type (fp16 2^-11, bf16 2^-8 of each weight) and
// quantised keys and values to fp16 (2^-11); scores, sums and outputs are fp32.  That is a choice: the tensor cores' floats
// have no more bits than fp16's (tf32 rounds alike), P has V's type, as the instruction wants it, and operands in two halves
// would take two or three products for each.  With fp16 outputs the error against 64 bits is 2 to 3 times the output's own
// rounding (5.7e-4 against 2.1e-4, Q8_0), with a BF16 cache 1.3 times (2.1e-3 against 1.6e-3).
//
// What bounds it: the softmax, some 2000 cycles for the 64 keys of 256 rows (64 exponentials, as many roundings and the moves
// from and to tensor memory a thread, four warps a scheduler); the products take about 1300.  No pipe is full
// (tcgen05 59%, exponentials 50%, issue slots 39%): the two wait for one another.  7993 rows of 32 heads of 128 over themselves, BF16,
// take 0.55 ms, 950 TFLOP/s or 57% of the measured GEMM rate; 2048 rows of 64 heads over 30049 keys of Q8_0 2.2 ms, 880 TFLOP/s.
// Short sequences pay kTileCost for each unit: 12 sequences of 1 to 600 new tokens 0.36 ms, 490 TFLOP/s.
#include <cuda.h>

#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "attention.cuh"

namespace anvil {

constexpr int kTileThreads = 512;   // 128 registers a thread at launch, divided anew by warp group below
constexpr int kTileLoaders = 128;   // threads of the four loading warps
// Beginning and ending a unit, in key tiles.  Counted as 2 / 4 / 8 / 12: 644 / 592 / 564 / 577 us for a prompt of 7993
// tokens, 463 / 389 / 393 / 435 for 12 sequences of 1 to 600 new ones.
constexpr int kTileCost = 8;
// Quantised pages of 16 keys and more, whose scales are whole 16-byte pieces, come by bulk copies: 1000 rows of 32 heads over
// 16000 keys in pages of 16 take 326 us (Q8_0) and 357 (Q4_0), by plain loads 440 and 383.  (16-bit pages of 8 keys
// and more by TMA: 382 us at 8 and 283 at 16 keys a page, by cp.async 551.)
constexpr int kTileBulkShift = 4;
constexpr float kTileSlack = 60000.0f;  // the largest sum of a tile's weights, and so weight: fp16 ends at 65504

template <int KIND, int D> struct TileShape {
    static constexpr int nq = D == 256 ? 1 : 2;         // row tiles of 128
    static constexpr int rows = 128 * nq;
    static constexpr int keys = 64;
    static constexpr int blocks = D / 64;               // 64-value column blocks of an operand
    static constexpr int q_bytes = rows * D * 2;
    static constexpr int buf = keys * D * 2;            // one buffer: keys or values of a tile
    static constexpr bool bf16 = KIND == kKvBF16;
    static constexpr bool quant = KIND == kKvQ8_0 || KIND == kKvQ4_0;
    static constexpr int nbuf = D == 256 ? 2 : D == 128 && quant ? 3 : 4;  // buffers of keys, and of values
    // A tile's keys and values are loaded and freed together where there are buffers for more than two tiles; else
    // they are a job each, so that the next keys come while the last values are in use.
    static constexpr int jobs = D == 256 ? 2 : 1;
    // quantised: a job's codes and scales as they are in the cache
    static constexpr int rb = KvRow<KIND, D>::bytes, sb = KvRow<KIND, D>::scales * 2;
    // (of Q8_0 with head_dim 256 half a job: one whole job has room beside the operands, and waiting for every job's
    // copies took twice the time)
    static constexpr int halves = D == 256 && KIND == kKvQ8_0 ? 2 : 1;
    static constexpr int raw_keys = keys / halves;
    static constexpr int raw = quant ? raw_keys * (rb + sb) * 2 / jobs : 0;
    static constexpr int nraw = 3;
    static constexpr int smem = 1024 + q_bytes + 2 * nbuf * buf + nraw * raw;
    // tensor memory columns: two turns of S for each row tile, then O
    static constexpr int s_cols = keys, o_col = 4 * keys, o_cols = D;
};

// ---- tcgen05 ----------------------------------------------------------------------------------

// A shared-memory operand in the 128-byte swizzle: low word start and leading byte offset, high word stride
// byte offset 1024 (eight rows), version 1 and the swizzle; offsets in 16-byte units.
__device__ __forceinline__ uint32_t smem_desc_lo(uint32_t addr, uint32_t lbo) {
    return ((addr & 0x3FFFF) >> 4) | ((lbo >> 4) << 16);
}
__device__ __forceinline__ uint64_t smem_desc(uint32_t lo) {
    constexpr uint32_t hi = (1024 >> 4) | (1u << 14) | (2u << 29);
    return uint64_t(lo) | (uint64_t(hi) << 32);
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

// One lane of the warp.  (Code under this predicate keeps the operands of the instructions below in uniform
// registers; under lane == 0 every one of them is moved there first: 85 cycles a product to issue.)
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e != 0;
}

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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : R8(v, 0), R8(v, 8) : "r"(addr));
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
    uint64_t full[2][4], empty[2][4], raw_full[3], raw_empty[3], partial[4], q_full, q_free,  // [job][buffer]
         s_full[2][2], p_full[2][2], pv_done[2][2], drain[2];  // [row tile][turn]
    float fac[2][256];      // [unit % 2]: what a row's scores are multiplied by
    uint32_t tmem;
    int failed;             // a wait gave up: later ones do not wait
    int dirty[8];           // [unit % 8] = unit where non-finite values were taken out of its value tiles
    uint32_t bad[8][2];     // [tile % 8]: keys without a page
};

// Bounded by the wall clock, which is only looked at after some hundred polls: reading it takes longer
// than most waits.
__device__ __forceinline__ void tile_wait(TileShared *sh, uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
    uint64_t t0 = 0;
    for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
        if (i & 255) continue;
        if (*reinterpret_cast<volatile int *>(&sh->failed)) return;
        const uint64_t now = global_timer_ns();
        if (t0 == 0) {
            t0 = now;
        } else if (now - t0 > limit_ns) {
            *reinterpret_cast<volatile int *>(&sh->failed) = 1;
            atomicOr(&g_anvil_device_status, kStatusMbarTimeout);
            return;
        }
    }
}
__device__ __forceinline__ void loaders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kTileLoaders) : "memory"); }
// Whether a phase is over, without the wait that try_wait may take.
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// Loads that leave no line in L1, which is small beside this kernel's shared memory and holds what registers do not.
__device__ __forceinline__ uint4 ld_stream(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_stream16(const uint8_t *p) {
    uint16_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
// 0 * a + c of 16-bit pairs
template <bool BF> __device__ __forceinline__ uint32_t zero_times(uint32_t a, uint32_t c) {
    uint32_t r;
    if constexpr (BF) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0u), "r"(c));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0u), "r"(c));
    return r;
}
// Stores of 32 bytes, a whole sector a lane.
__device__ __forceinline__ void st32(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// A box of 64 columns from (x, y) of a tensor of 16-bit rows into the 128-byte swizzled layout.
__device__ __forceinline__ void tma_box(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A unit's share of this CTA: key tiles [t0, t1) and the limits of its masks.
template <int KIND, int D> struct TileUnit {
    using S = TileShape<KIND, D>;
    AttnSeq<S::rows, S::keys> q;
    int ntiles, t0, t1, key_end, nrows, free_end;
    __device__ __forceinline__ TileUnit(const KvSeq &seq, const AttnIO &io, const AttnPos &p, int64_t lo, int64_t hi)
        : q(seq, io) {
        ntiles = q.key_tiles(p.mt);
        t0 = int(max(lo - p.unit0, int64_t(0)));
        t1 = int(min(hi - p.unit0, int64_t(ntiles)));
        key_end = min(t1 * S::keys, q.keys(p.mt));
        nrows = int(min(int64_t(S::rows), int64_t(unsigned(q.n) * unsigned(io.group) - unsigned(p.mt) * S::rows)));
        // every row of the unit sees the keys below this
        free_end = min(key_end, kv_seen(int(by_group(io, unsigned(p.mt) * S::rows)), q.n, q.s.kv, io.causal));
    }
};

template <int KIND, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attn_tile_kernel(KvCacheView c, KvBatchView bt, AttnIO io, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, int box, uint64_t limit_ns) {
    using S = TileShape<KIND, D>;
    constexpr bool BF = S::bf16;
    extern __shared__ uint8_t dyn[];
    __shared__ TileShared sh;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
    uint8_t *sq = base, *sbuf = base + S::q_bytes, *sraw = sbuf + 2 * S::nbuf * S::buf;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int64_t work = attn_locate<S::rows, S::keys, kTileCost>(
        c, bt, io, &sh.sc, [&](const AttnShares &s) { return s.begin(min(int(blockIdx.x), s.ctas - 1)); }, blockIdx.x == 0);
    pdl_launch_dependents();
    attn_zero_rest<D>(bt, io);
    const AttnShares shares(work, gridDim.x);
    AttnOpen *const note = io.part ? attn_open<S::rows, D>(io.part, gridDim.x) + blockIdx.x : nullptr;
    if (int(blockIdx.x) >= shares.ctas) {
        if (note && threadIdx.x == 0) *note = AttnOpen{};
        return;
    }
    const int64_t lo = shares.begin(blockIdx.x), hi = shares.begin(blockIdx.x + 1);
    AttnPos p = sh.sc.pos;
    KvSeq kseq = load_seq(bt, c, p.b);

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::nbuf; ++i)
            for (int kv = 0; kv < 2; ++kv) {
                mbar_init(&sh.full[kv][i], kTileLoaders / 32);
                mbar_init(&sh.empty[kv][i], S::nq);
            }
        for (int i = 0; i < S::nraw; ++i) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_empty[i], kTileLoaders / 32);
        }
        for (int i = 0; i < 2; ++i) {
            for (int x = 0; x < 2; ++x) {
                mbar_init(&sh.s_full[i][x], 1);
                mbar_init(&sh.p_full[i][x], 4);
                mbar_init(&sh.pv_done[i][x], 1);
            }
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sh.partial[i], 1);
        mbar_init(&sh.q_full, (S::quant ? kTileLoaders : kTileLoaders - 32) / 32);
        mbar_init(&sh.q_free, S::nq);
        for (int i = 0; i < 2; ++i) mbar_init(&sh.drain[i], 1);
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

    // Registers by warp group: 2 x 152 + 136 + 72 = 4 x 128, what the CTA was launched with.
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    else if (warp < 12) asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp < 8) {
        // ================= softmax: thread = row of tile w ==========================================
        const int w = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        // Tiles so far on each turn.  S, P and P V of a tile use its turn's barriers: a side may be a whole tile
        // ahead of the other, and a parity tells one phase from the next only.
        uint32_t n0 = 0, n1 = 0;
        int unit = 0, seq = 0;              // units and key tiles so far, counted alike in every role
        bool noted = false;
        if (w < S::nq)
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                ++unit;
                if (w * 128 < u.nrows) {
                    const int ur = w * 128 + r;
                    const bool live = ur < u.nrows;
                    const unsigned rr = unsigned(p.mt) * S::rows + ur;
                    const int tok = int(by_group(io, rr)), h = p.head * io.group + int(rr - unsigned(tok) * io.group);
                    const int seen = live ? min(u.key_end, kv_seen(tok, u.q.n, u.q.s.kv, io.causal)) : 0;
                    float fac = 0.0f;
                    float m = -INFINITY, l = 0.0f;
                    const uint32_t to = tmem + lanes + S::o_col + w * S::o_cols;
                    for (int t = u.t0; t < u.t1; ++t) {
                        const int x = (t - u.t0) & 1;
                        const uint32_t ts = tmem + lanes + (w * 2 + x) * S::s_cols;
                        tile_wait(&sh, &sh.s_full[w][x], (x ? n1 : n0) & 1, limit_ns);
                        __syncwarp();
                        fence_after();
                        if (t == u.t0) fac = sh.fac[unit & 1][ur];  // written with the query
                        uint32_t s[64];
                        tmem_ld32(ts, s);
                        tmem_ld32(ts + 32, s + 32);
                        const uint32_t bad[2] = {sh.bad[(seq + t - u.t0) & 7][0], sh.bad[(seq + t - u.t0) & 7][1]};
                        wait_ld();
                        if ((t + 1) * 64 > u.free_end || (bad[0] | bad[1])) {
                            const int left = seen - t * 64;
#pragma unroll
                            for (int i = 0; i < 64; ++i)
                                if (i >= left || ((bad[i >> 5] >> (i & 31)) & 1)) s[i] = 0xFF800000u;
                        }
                        // The weights of this tile by the row's reference m so far; only where their sum shows that one may
                        // be too large, or where there is no reference yet, is the maximum looked for, the reference set by
                        // it, and the tile taken again.
                        float sum = 0.0f;
                        uint32_t y[32];
                        bool raise = m == -INFINITY;
                        for (int pass = 0;; ++pass) {
                            if (__any_sync(0xffffffffu, raise)) {
                                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int i = 0; i < 64; i += 2)
                                    mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                                const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * fac - kAttnHead<BF>;
                                const float mn = raise && mt > m ? mt : m;
                                const float a = mn > m ? ex2(m - mn) : 1.0f;
                                if (t > u.t0) {
                                    tile_wait(&sh, &sh.pv_done[w][x ^ 1], ((x ? n0 : n1) - 1) & 1, limit_ns);  // the last tile's P V
                                    __syncwarp();
                                    fence_after();
#pragma unroll 1
                                    for (int i = 0; i < D / 16; ++i) {
                                        uint32_t v[16];
                                        tmem_ld16(to + 16 * i, v);
                                        wait_ld();
#pragma unroll
                                        for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * a);
                                        tmem_st16(to + 16 * i, v);
                                    }
                                }
                                l *= a;
                                m = mn;
                            }
                            const float nb = m == -INFINITY ? 0.0f : -m;
                            const uint64_t fac2 = pack2(fac, fac), nb2 = pack2(nb, nb);
                            uint64_t sums[2] = {0, 0};
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                float e0, e1;
                                unpack2(fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), fac2, nb2), e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                                sums[i & 1] = add2(sums[i & 1], pack2(e0, e1));
                                y[i] = BF ? pack_bf16(e0, e1) : pack_half(e0, e1);
                            }
                            float a0, a1;
                            unpack2(add2(sums[0], sums[1]), a0, a1);
                            sum = a0 + a1;
                            raise = pass == 0 && sum > kTileSlack;
                            if (!__any_sync(0xffffffffu, raise)) break;
                        }
                        l += sum;
                        tmem_st32(ts, y);
                        wait_st();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.p_full[w][x]);
                        (x ? n1 : n0) += 1;
                    }

                    // ---- the unit's outputs, or this share's part of them
                    const int xl = (u.t1 - 1 - u.t0) & 1;  // the last tile's turn; its P V ends after all others
                    tile_wait(&sh, &sh.pv_done[w][xl], ((xl ? n1 : n0) - 1) & 1, limit_ns);
                    __syncwarp();
                    fence_after();
                    const bool begun = p.unit0 < lo, unfinished = p.unit0 + u.ntiles > hi;
                    if (unfinished && !begun && threadIdx.x == 0) {
                        noted = true;
                        *note = AttnOpen{shares.owner(p.unit0 + u.ntiles - 1) - int(blockIdx.x) + 1, u.q.s.q0, p.head * io.group, p.mt * S::rows, u.nrows, {}};
                    }
                    const bool dirty = *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) == unit;
                    const bool wide = reinterpret_cast<uintptr_t>(io.out) % 32 == 0;
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
                            for (int j = 0; j < 4; ++j) st32(part + ur * D + 32 * i + 8 * j, v + 8 * j);
                        } else if (live) {
                            uint32_t y[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float e0 = __uint_as_float(v[2 * j]) * inv, e1 = __uint_as_float(v[2 * j + 1]) * inv;
                                y[j] = io.q_bf16 ? pack_bf16(e0, e1) : pack_half(e0, e1);
                            }
                            // (out is 16-byte aligned, 32 only where its allocation is)
                            if (wide) {
                                st32(dst + 16 * i, y);
                                st32(dst + 16 * i + 8, y + 8);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    *reinterpret_cast<uint4 *>(dst + 16 * i + 4 * j) =
                                        make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                            }
                        }
                    }
                    if (live && (begun || unfinished)) {
                        part[S::rows * D + ur] = m;
                        part[S::rows * D + S::rows + ur] = l;
                    }
                    fence_before();
                }
                seq += u.t1 - u.t0;
                attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
            }
        if (threadIdx.x == 0 && note && !noted) *note = AttnOpen{};
    } else if (warp < 12) {
        // ================= loaders: keys and values of a tile together ===============================
        constexpr int LT = kTileLoaders;
        const int tid = threadIdx.x - 256;
        int unit = 0, seq = 0;  // units and tiles begun
        auto announce = [&](int job, int b) {
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.full[job][b]);
        };
        // Page of a key (0 behind the last one), looked up a tile ahead of its use; and the key's cache row, -1 where
        // there is no page and -2 behind the last key.
        auto page_of = [&](const TileUnit<KIND, D> &u, int key) {
            return key < u.key_end ? __ldg(bt.table + p.b * bt.table_stride + (key >> c.page_shift)) : 0;
        };
        auto row_of = [&](const TileUnit<KIND, D> &u, int key, int page) -> int64_t {
            return key < u.key_end
                       ? kv_row(page, c.num_pages, p.head, c.kv_heads, key & ((1 << c.page_shift) - 1), c.page_shift)
                       : -2;
        };
        // keys of the tile without a page, for the softmax (each of the first two warps knows 32 of them)
        auto share_bad = [&](bool none) {
            const uint32_t bad = __ballot_sync(0xffffffffu, none);
            if (tid < S::keys && lane == 0) {
                sh.bad[seq & 7][tid >> 5] = bad;
                if (bad) flag_bad_page();
            }
        };
        // A unit's query rows into the swizzled operand, while the softmax is still at the unit before: once that one's
        // scores are all taken.  Rows that are none are zeros.  (16-bit caches: by warps 9-11.)
        auto load_q = [&](const TileUnit<KIND, D> &u) {
            constexpr int CHQ = D / 8, QT = S::quant ? LT : LT - 32, FLY = 8;
            const int qt = tid - (LT - QT);
            if (unit > 1) {
                tile_wait(&sh, &sh.q_free, unit & 1, limit_ns);
                __syncwarp();
            }
            const int all = (u.nrows > 128 ? S::rows : 128) * CHQ;
            auto row_at = [&](int ur) {
                const unsigned rr = unsigned(p.mt) * S::rows + ur;
                const int tok = int(by_group(io, rr)), h = p.head * io.group + int(rr - unsigned(tok) * io.group);
                return static_cast<const uint16_t *>(io.q) + (u.q.s.q0 + int64_t(tok)) * io.q_row + h * io.q_head;
            };
            auto place_q = [&](int ur, int ch) { return sq + (ch >> 3) * (S::rows * 128) + ur * 128 + (((ch & 7) ^ (ur & 7)) << 4); };
            // (above zero, so that a masked score stays -inf)
            auto put_fac = [&](int ur, int ex) { sh.fac[unit & 1][ur] = fmaxf(fabsf(io.scale_log2) * pow2i(-ex), 1e-36f); };
            // a negative scale: -q, so that the largest score stays the largest
            const uint32_t sign = io.scale_log2 < 0.0f ? 0x80008000u : 0;
            if (sign == 0 && !(S::quant && io.q_bf16)) {
                const int ch = qt % CHQ;  // of every row of this thread
#pragma unroll 4
                for (int ur = qt / CHQ; ur < all / CHQ; ur += QT / CHQ) {
                    const bool live = ur < u.nrows;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(place_q(ur, ch))),
                                 "l"(live ? row_at(ur) + ch * 8 : io.q), "r"(live ? 16 : 0)
                                 : "memory");
                    if (ch == 0) put_fac(ur, 0);
                }
                asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
            } else {
                for (int at0 = qt; at0 < all + qt; at0 += FLY * QT) {  // (every lane the same number of times)
                    uint4 x[FLY];
#pragma unroll
                    for (int f = 0; f < FLY; ++f) {
                        const int at = at0 + f * QT, ur = at / CHQ, ch = at % CHQ;
                        x[f] = at < all && ur < u.nrows ? __ldg(reinterpret_cast<const uint4 *>(row_at(ur)) + ch) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int f = 0; f < FLY; ++f) {
                        const int at = at0 + f * QT, ur = at / CHQ, ch = at % CHQ;
                        uint32_t y[4] = {x[f].x, x[f].y, x[f].z, x[f].w};
                        int ex = 0;
                        if (S::quant && io.q_bf16) {
                            uint32_t m = 0;
#pragma unroll
                            for (int j = 0; j < 4; ++j) m = max(max(m, y[j] & 0x7FFFu), (y[j] >> 16) & 0x7FFFu);
#pragma unroll
                            for (int o = CHQ / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                            ex = q_exponent(m << 16);
                            const float up = pow2i(ex);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                y[j] = pack_half(__uint_as_float(y[j] << 16) * up, __uint_as_float(y[j] & 0xFFFF0000u) * up);
                        }
                        if (at < all) {
                            *reinterpret_cast<uint4 *>(place_q(ur, ch)) = make_uint4(y[0] ^ sign, y[1] ^ sign, y[2] ^ sign, y[3] ^ sign);
                            if (ch == 0) put_fac(ur, ex);
                        }
                    }
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
        };
        // place of 16-byte chunk oc of key r in a buffer
        auto place = [&](int kv, int b, int r, int oc) {
            return sbuf + (kv * S::nbuf + b) * S::buf + (oc >> 3) * (S::keys * 128) + r * 128 + (((oc & 7) ^ (r & 7)) << 4);
        };
        if constexpr (!S::quant) {
            // 16-bit rows go straight to their places: from pages of 8 keys and more by TMA, boxes of up to 64 keys of one
            // page and 64 columns; from smaller ones by cp.async, a tile announced when the next one's copies are on their way.
            // Of a tile that lacks pages, or keys behind the last, what is no key leaves the values first; of one that some row
            // does not see whole, what is not finite too (the outputs bring it back to the rows that see it).
            constexpr int CH = D / 8;
            auto clean = [&](const TileUnit<KIND, D> &u, int t, int b, int from) {  // by threads `from` and up
                const int left = u.key_end - t * S::keys;
                const uint32_t bad[2] = {sh.bad[seq & 7][0], sh.bad[seq & 7][1]};
                const int step = (LT - from) / CH, ch = (tid - from) % CH, first = (tid - from) / CH;
                if (left < S::keys || (bad[0] | bad[1])) {
                    for (int r = first; r < S::keys; r += step)
                        if (r >= left || ((bad[r >> 5] >> (r & 31)) & 1))
                            *reinterpret_cast<uint4 *>(place(1, b, r, ch)) = make_uint4(0, 0, 0, 0);
                }
                if ((t + 1) * S::keys <= u.free_end) return;  // only a page was missing: every row sees the other keys
                // 0 x value summed: NaN if any value is not finite
                uint32_t odd = 0;
#pragma unroll 4
                for (int r = first; r < S::keys; r += step) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(place(1, b, r, ch));
                    odd = zero_times<BF>(x.x, zero_times<BF>(x.y, zero_times<BF>(x.z, zero_times<BF>(x.w, odd))));
                }
                if (nonfinite2<BF>(odd)) {
                    for (int r = first; r < S::keys; r += step) {
                        uint4 *w4 = reinterpret_cast<uint4 *>(place(1, b, r, ch));
                        const uint4 x = *w4;
                        *w4 = make_uint4(x.x & ~nonfinite2<BF>(x.x), x.y & ~nonfinite2<BF>(x.y), x.z & ~nonfinite2<BF>(x.z),
                                         x.w & ~nonfinite2<BF>(x.w));
                    }
                    *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) = unit;
                }
                __syncwarp();
            };
            auto wait_empty = [&](int job, int b) {
                if (seq >= S::nbuf) tile_wait(&sh, &sh.empty[job][b], (seq / S::nbuf - 1) & 1, limit_ns);
                __syncwarp();
            };
            if (box) {
                // Warp 8 issues the copies; the other three load the queries and clean, and do not hold it up.
                const int boxes = S::keys / box;  // of a tile's keys
                uint32_t partial = 0;             // bit b: parity of the next partial tile in buffer b
                while (p.b < bt.batch && p.unit0 < hi) {
                    const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                    ++unit;
                    if (warp > 8) load_q(u);
                    // lane i: the page of box i
                    int page = lane < boxes ? page_of(u, u.t0 * S::keys + lane * box) : 0;
                    for (int t = u.t0; t < u.t1; ++t, ++seq) {
                        const int64_t row = lane < boxes ? row_of(u, t * S::keys + lane * box, page) : -2;
                        if (lane < boxes && t + 1 < u.t1) page = page_of(u, (t + 1) * S::keys + lane * box);
                        const uint32_t live = __ballot_sync(0xffffffffu, row >= 0), none = __ballot_sync(0xffffffffu, row == -1);
                        const bool whole = (t + 1) * S::keys <= u.free_end && !none;
                        const int b = seq % S::nbuf;
#pragma unroll
                        for (int job = 0; job < S::jobs; ++job) {
                            const bool keys = job == 0, values = job == S::jobs - 1;
                            const bool direct = whole || !values;  // (keys need no cleaning: they are masked)
                            wait_empty(job, b);
                            if (warp == 8) {
                                uint64_t *bar = direct ? &sh.full[job][b] : &sh.partial[b];
                                if (lane == 0) {
                                    if (job == 0) {
                                        uint64_t bad = 0;
                                        for (int i = 0; none && i < boxes; ++i)
                                            if ((none >> i) & 1) bad |= (box == 64 ? ~uint64_t(0) : (uint64_t(1) << box) - 1) << (i * box);
                                        sh.bad[seq & 7][0] = uint32_t(bad);
                                        sh.bad[seq & 7][1] = uint32_t(bad >> 32);
                                        if (bad) flag_bad_page();
                                    }
                                    mbar_arrive_expect_tx(bar, __popc(live) * box * D * 2 * (int(keys) + int(values)));
                                    if (!direct) mbar_arrive(&sh.full[job][b]);
                                }
                                __syncwarp();
                                for (int i = 0; i < boxes; ++i) {
                                    const int y = int(__shfl_sync(0xffffffffu, row, i));
                                    if (y >= 0 && elect_one()) {
#pragma unroll
                                        for (int j = 0; j < S::blocks; ++j) {
                                            if (keys) tma_box(place(0, b, i * box, 8 * j), &map_k, 64 * j, y, bar);
                                            if (values) tma_box(place(1, b, i * box, 8 * j), &map_v, 64 * j, y, bar);
                                        }
                                    }
                                    __syncwarp();
                                }
                            } else if (direct) {
                                if (lane == 0) mbar_arrive(&sh.full[job][b]);
                            } else {
                                tile_wait(&sh, &sh.partial[b], (partial >> b) & 1, limit_ns);
                                __syncwarp();
                                partial ^= 1u << b;
                                clean(u, t, b, 32);
                                announce(job, b);
                            }
                        }
                    }
                    attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
                }
            } else {
                constexpr int ALL = 2 * S::keys * CH, depth = S::nbuf > 2 ? 2 : 1;
                int pending = 0;
                auto settle = [&](int left) {  // announces all but the newest `left` tiles, whose copies are done
                    for (; pending > left; --pending)
                        for (int job = 0; job < S::jobs; ++job) announce(job, (seq - pending) % S::nbuf);
                };
                while (p.b < bt.batch && p.unit0 < hi) {
                    const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                    ++unit;
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    settle(0);
                    if (warp > 8) load_q(u);
                    for (int t = u.t0; t < u.t1; ++t) {
                        const int b = seq % S::nbuf;
                        // (a product may wait for a pending tile before it frees this one's buffers)
                        if (pending && seq >= S::nbuf &&
                            !__all_sync(0xffffffffu, mbar_test(&sh.empty[S::jobs - 1][b], (seq / S::nbuf - 1) & 1))) {
                            asm volatile("cp.async.wait_group 0;" ::: "memory");
                            settle(0);
                        }
                        for (int job = 0; job < S::jobs; ++job) wait_empty(job, b);
                        const int key = t * S::keys + tid;
                        share_bad(tid < S::keys && row_of(u, key, page_of(u, key)) == -1);
#pragma unroll 8
                        for (int at = tid; at < ALL; at += LT) {
                            const int kv = at / (ALL / 2), r = at / CH % S::keys, ch = at % CH;
                            const int64_t rw = row_of(u, t * S::keys + r, page_of(u, t * S::keys + r));
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(place(kv, b, r, ch))),
                                         "l"((kv ? c.v : c.k) + max(rw, int64_t(0)) * (2 * D) + ch * 16), "r"(rw < 0 ? 0 : 16)
                                         : "memory");
                        }
                        asm volatile("cp.async.commit_group;" ::: "memory");
                        if ((t + 1) * S::keys > u.free_end) {
                            asm volatile("cp.async.wait_group 0;" ::: "memory");
                            settle(0);
                            loaders_sync();  // a thread cleans what others copied, by the mask that others wrote
                            clean(u, t, b, 0);
                            for (int job = 0; job < S::jobs; ++job) announce(job, b);
                            ++seq;
                        } else {
                            ++seq;
                            if (++pending == depth) {
                                asm volatile("cp.async.wait_group %0;" ::"n"(depth - 1) : "memory");
                                settle(depth - 1);
                            }
                        }
                    }
                    attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                settle(0);
            }
        } else {
            // 16 bytes of codes a turn: 16 (Q8_0) or 32 (Q4_0) values, two or four chunks; a thread has one chunk of R
            // keys, 128 / CH apart.  Pages of 16 keys and more come through raw buffers that warp 14 fills by bulk copies:
            // beside 200 KB of shared memory L1 is too small to have many plain loads on their way.
            constexpr int RB = S::rb, CH = RB / 16, R = S::keys * CH / LT, STEP = LT / CH;
            constexpr int jobs = S::jobs, N = 2 * R / jobs;
            constexpr int OUT = KIND == kKvQ8_0 ? 2 : 4, VALS = 8 * OUT;
            // eight lanes store two rows of four chunks where rows have them: distinct banks
            const int in = tid % (2 * CH);
            const int ch = CH >= 8 ? (in & 3) | ((in >> 3) << 2) : tid % CH;
            const int r0 = CH >= 8 ? tid / (2 * CH) * 2 + ((in >> 2) & 1) : tid / CH;
            const bool bulk = c.page_shift >= kTileBulkShift;
            uint4 w[N], wn[N];
            uint32_t d[N], dn[N], gone = 0;  // gone: bits of the fetched keys that are not there
            int pages[R];                    // pages of the next fetch's keys
            uint32_t taken = 0;              // jobs taken from the raw buffers
            auto look = [&](const TileUnit<KIND, D> &u, int t) {
#pragma unroll
                for (int i = 0; i < R; ++i) pages[i] = page_of(u, t * S::keys + r0 + i * STEP);
            };
            constexpr uint32_t flip = KIND == kKvQ8_0 ? 0x80808080u : 0;
            // a job's codes from the raw buffer that warp 14 had filled
            auto from_raw = [&](const TileUnit<KIND, D> &u, int t, int half) {
                const int slot = taken % S::nraw;
                tile_wait(&sh, &sh.raw_full[slot], (taken / S::nraw) & 1, limit_ns);
                __syncwarp();
                const uint8_t *raw = sraw + slot * S::raw;
                const int left = u.key_end - t * S::keys;
                const uint32_t bad[2] = {sh.bad[seq & 7][0], sh.bad[seq & 7][1]};
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i * S::halves / N != half) continue;
                    const int r = r0 + i % R * STEP, v = i / R, at = v * S::raw_keys + r - half * S::raw_keys;
                    const uint4 x = *reinterpret_cast<const uint4 *>(raw + at * RB + ch * 16);
                    const uint32_t y = *reinterpret_cast<const uint16_t *>(raw + N / R * S::raw_keys * RB + at * S::sb + ch * VALS / 32 * 2);
                    w[i] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
                    d[i] = r >= left || ((bad[r >> 5] >> (r & 31)) & 1) ? 0 : dup16(y);
                }
            };
            // Loads without a condition (of the pool's first row where there is none): loads in branches would be
            // waited for one after the other.
            auto fetch = [&](const TileUnit<KIND, D> &u, int t, int job) {
                const uint8_t *pk = job ? c.v : c.k, *pv = c.v;
                const uint8_t *sk = reinterpret_cast<const uint8_t *>(job ? c.vs : c.ks), *sv = reinterpret_cast<const uint8_t *>(c.vs);
                const int co = ch * 16, so = ch * VALS / 32 * 2;
                auto get = [&](int i, int64_t row) {
                    wn[i] = ld_stream(pk + row * RB + co);
                    dn[i] = ld_stream16(sk + row * (D / 16) + so);
                    if constexpr (jobs == 1) {
                        wn[R + i] = ld_stream(pv + row * RB + co);
                        dn[R + i] = ld_stream16(sv + row * (D / 16) + so);
                    }
                };
                gone = 0;
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int64_t row = row_of(u, t * S::keys + r0 + i * STEP, pages[i]);
                    gone |= row < 0 ? 1u << i : 0;
                    get(i, max(row, int64_t(0)));
                }
            };
            auto take = [&]() {  // the fetched codes, that is, waits for them
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    w[i] = make_uint4(wn[i].x ^ flip, wn[i].y ^ flip, wn[i].z ^ flip, wn[i].w ^ flip);
                    d[i] = (gone >> (i % R)) & 1 ? 0 : dup16(dn[i]);
                }
            };
            auto widen = [&](int job, bool check) {
                const int b = seq % S::nbuf;
                if (seq >= S::nbuf) tile_wait(&sh, &sh.empty[job][b], (seq / S::nbuf - 1) & 1, limit_ns);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int kv = jobs == 1 ? i / R : job, r = r0 + i % R * STEP;
                    uint32_t d2 = usable_scales<KIND>(d[i]);  // (beside the loads above it took 13% of a chunk's time)
                    if (check && kv && (d2 & 0x7FFFu) >= kOddScale<KIND>) {
                        const bool whole = KIND == kKvQ8_0 && (d2 & 0x7FFFu) == 0x6000u;
                        if (!whole) *reinterpret_cast<volatile int *>(&sh.dirty[unit & 7]) = unit;
                        d2 = whole ? d2 - 0x00010001u : 0;
                    }
                    const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                    uint32_t y[4 * OUT];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (KIND == kKvQ8_0) {  // x: codes + 128
                            y[2 * j] = h2mul(h2sub(__byte_perm(x[j], 0x64646464u, 0x4140), 0x64806480u), d2);
                            y[2 * j + 1] = h2mul(h2sub(__byte_perm(x[j], 0x64646464u, 0x4342), 0x64806480u), d2);
                        } else {
                            const uint32_t a = x[j] & 0x0F0F0F0Fu, e = (x[j] >> 4) & 0x0F0F0F0Fu;
                            y[2 * j] = h2mul(h2sub(__byte_perm(a, 0x64646464u, 0x4140), 0x64086408u), d2);
                            y[2 * j + 1] = h2mul(h2sub(__byte_perm(a, 0x64646464u, 0x4342), 0x64086408u), d2);
                            y[8 + 2 * j] = h2mul(h2sub(__byte_perm(e, 0x64646464u, 0x4140), 0x64086408u), d2);
                            y[8 + 2 * j + 1] = h2mul(h2sub(__byte_perm(e, 0x64646464u, 0x4342), 0x64086408u), d2);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < OUT; ++j)
                        *reinterpret_cast<uint4 *>(place(kv, b, r, ch * OUT + j)) =
                            make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                }
                announce(job, b);
            };
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                ++unit;
                load_q(u);
                if (bulk) {
                    for (int t = u.t0; t < u.t1; ++t, ++seq)
                        for (int job = 0; job < jobs; ++job) {
                            // (Raw buffers are given back when their codes are in registers where they hold half a job, else
                            // after the widening, which took 4% less.)
#pragma unroll
                            for (int half = 0; half < S::halves; ++half) {
                                from_raw(u, t, half);
                                if (S::halves == 1) break;
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&sh.raw_empty[taken % S::nraw]);
                                ++taken;
                            }
                            widen(job, job == jobs - 1 && (t + 1) * S::keys > u.free_end);
                            if (S::halves == 1) {
                                if (lane == 0) mbar_arrive(&sh.raw_empty[taken % S::nraw]);
                                ++taken;
                            }
                        }
                } else {
                    // pages of a few keys: every thread fetches its own, a job ahead of the widening
                    look(u, u.t0);
                    fetch(u, u.t0, 0);
                    int page = page_of(u, u.t0 * S::keys + tid);  // of key `tid` of the tile
                    if (jobs == 1) look(u, u.t0 + 1);
                    for (int t = u.t0; t < u.t1; ++t, ++seq) {
                        const bool check = (t + 1) * S::keys > u.free_end, more = t + 1 < u.t1;
                        share_bad(tid < S::keys && row_of(u, t * S::keys + tid, page) == -1);
                        if (tid < S::keys) page = page_of(u, (t + 1) * S::keys + tid);
                        take();
                        if (jobs == 2) {
                            fetch(u, t, 1);
                            look(u, t + 1);
                            widen(0, false);
                            take();
                        }
                        if (more) {
                            fetch(u, t + 1, 0);
                            if (jobs == 1) look(u, t + 2);
                        }
                        widen(jobs - 1, check);
                    }
                }
                attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
            }
        }
    } else {
        const int w = warp - 12;  // row tile of the products that warp 12 or 13 issues
        if (w < S::nq && elect_one()) {
            // ================= products ================================================================
            constexpr uint32_t fmt = BF ? 1 : 0;
            constexpr uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
            constexpr uint32_t id_qk = idesc0 | (uint32_t(S::keys / 8) << 17);
            constexpr uint32_t id_pv = idesc0 | (1u << 16) | (uint32_t(D / 8) << 17);  // V: its columns are contiguous
            uint32_t nb = 0, units = 0, np[2] = {0, 0};  // tiles, units, tiles by turn
            const uint32_t q0 = smem_desc_lo(smem_u32(sq + w * 128 * 128), 16), k0 = smem_desc_lo(smem_u32(sbuf), 16),
                           v0 = smem_desc_lo(smem_u32(sbuf + S::nbuf * S::buf), S::keys * 128);
            const uint32_t ts = tmem + w * 2 * S::s_cols, to = tmem + S::o_col + w * S::o_cols;
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                const int tiles = u.t1 - u.t0;
                const bool on = w * 128 < u.nrows;  // (else this warp only keeps step)
                auto wait_full = [&](int job, int i) {
                    tile_wait(&sh, &sh.full[job][(nb + i) % S::nbuf], ((nb + i) / S::nbuf) & 1, limit_ns);
                    fence_after();
                };
                auto done = [&](uint64_t *bar) {
                    if (on) mma_commit(bar);
                    else mbar_arrive(bar);
                };
                auto scores = [&](int i) {  // S of tile i, once its keys are there
                    wait_full(0, i);
                    const uint32_t k = k0 + (nb + i) % S::nbuf * (S::buf >> 4), d = ts + (i & 1) * S::s_cols;
                    if (on) {
#pragma unroll
                        for (int j = 0; j < D / 16; ++j)
                            mma_ss(d, smem_desc(q0 + (((j >> 2) * (S::rows * 128) + (j & 3) * 32) >> 4)),
                                   smem_desc(k + (((j >> 2) * (S::keys * 128) + (j & 3) * 32) >> 4)), id_qk, j > 0);
                        mma_commit(&sh.s_full[w][i & 1]);
                    }
                    if (S::jobs == 2) done(&sh.empty[0][(nb + i) % S::nbuf]);
                    if (i + 1 == tiles) done(&sh.q_free);
                };
                auto outputs = [&](int i) {  // O += P V of tile i, once its weights are there
                    if (S::jobs == 2) wait_full(1, i);
                    if (on) {
                        if (i & 1) tile_wait(&sh, &sh.p_full[w][1], np[1]++ & 1, limit_ns);
                        else tile_wait(&sh, &sh.p_full[w][0], np[0]++ & 1, limit_ns);
                        fence_after();
                        const uint32_t v = v0 + (nb + i) % S::nbuf * (S::buf >> 4), a = ts + (i & 1) * S::s_cols;
#pragma unroll
                        for (int j = 0; j < S::keys / 16; ++j)
                            mma_ts(to, a + j * 8, smem_desc(v + ((j * 2048) >> 4)), id_pv, i > 0 || j > 0);
                        mma_commit(&sh.pv_done[w][i & 1]);
                    }
                    done(&sh.empty[S::jobs - 1][(nb + i) % S::nbuf]);
                };
                tile_wait(&sh, &sh.q_full, units++ & 1, limit_ns);
                if constexpr (S::jobs == 1) {
                    // Two tiles ahead of the softmax: when P V of tile i is issued, its columns take the scores of tile
                    // i + 2, while the softmax works on those of i + 1.
                    for (int i = 0; i < min(tiles, 2); ++i) scores(i);
                    for (int i = 0; i < tiles; ++i) {
                        outputs(i);
                        if (i + 2 < tiles) scores(i + 2);
                    }
                } else {
                    // One tile ahead (two buffers): S of tile i + 1 goes to the other turn's columns, whose P was read by the
                    // products of tile i - 1, which were issued before.
                    scores(0);
                    for (int i = 0; i < tiles; ++i) {
                        if (i + 1 < tiles) scores(i + 1);
                        outputs(i);
                    }
                }
                nb += tiles;
                attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
            }
            mma_commit(&sh.drain[w]);
            tile_wait(&sh, &sh.drain[w], 0, limit_ns);
        }
        if (warp == 14 && S::quant && c.page_shift >= kTileBulkShift) {
            // ================= raw buffers: bulk copies, page by page ====================================
            const int per = min(S::raw_keys, 1 << c.page_shift), parts = S::keys / per;  // keys of a copy, copies of a tile
            uint32_t filled = 0;
            int seq = 0;
            while (p.b < bt.batch && p.unit0 < hi) {
                const TileUnit<KIND, D> u(kseq, io, p, lo, hi);
                auto page_of = [&](int t) {  // lane i: the page of part i
                    const int key = t * S::keys + lane * per;
                    return lane < parts && key < u.key_end ? __ldg(bt.table + p.b * bt.table_stride + (key >> c.page_shift)) : -1;
                };
                int page = page_of(u.t0);
                for (int t = u.t0; t < u.t1; ++t, ++seq) {
                    const int key = t * S::keys + lane * per;
                    const bool here = lane < parts && key < u.key_end;
                    const int64_t row = here ? kv_row(page, c.num_pages, p.head, c.kv_heads, key & ((1 << c.page_shift) - 1), c.page_shift) : -1;
                    page = page_of(t + 1);
                    const uint32_t live = __ballot_sync(0xffffffffu, row >= 0), none = __ballot_sync(0xffffffffu, here && row < 0);
                    for (int piece = 0; piece < S::jobs * S::halves; ++piece, ++filled) {
                        const int job = piece / S::halves, half = piece % S::halves, i0 = half * (parts / S::halves), i1 = i0 + parts / S::halves;
                        const int slot = filled % S::nraw;
                        if (filled >= S::nraw) tile_wait(&sh, &sh.raw_empty[slot], (filled / S::nraw - 1) & 1, limit_ns);
                        __syncwarp();
                        if (lane == 0) {
                            if (piece == 0) {
                                uint64_t bad = 0;
                                for (int i = 0; i < parts; ++i)
                                    if ((none >> i) & 1) bad |= (per == 64 ? ~uint64_t(0) : (uint64_t(1) << per) - 1) << (i * per);
                                sh.bad[seq & 7][0] = uint32_t(bad);
                                sh.bad[seq & 7][1] = uint32_t(bad >> 32);
                                if (bad) flag_bad_page();
                            }
                            mbar_arrive_expect_tx(&sh.raw_full[slot], __popc(live >> i0 << (32 - i1 + i0)) * per * (S::rb + S::sb) * 2 / S::jobs);
                        }
                        __syncwarp();
                        uint8_t *raw = sraw + slot * S::raw;
                        for (int i = i0; i < i1; ++i) {
                            const int64_t first = __shfl_sync(0xffffffffu, row, i);
                            if (first >= 0 && elect_one()) {
#pragma unroll
                                for (int v = 0; v < 2 / S::jobs; ++v) {
                                    const bool values = S::jobs == 2 ? job == 1 : v == 1;
                                    bulk_copy_g2s(raw + (v * S::raw_keys + (i - i0) * per) * S::rb, (values ? c.v : c.k) + first * S::rb,
                                                  per * S::rb, &sh.raw_full[slot]);
                                    bulk_copy_g2s(raw + 2 / S::jobs * S::raw_keys * S::rb + (v * S::raw_keys + (i - i0) * per) * S::sb,
                                                  reinterpret_cast<const uint8_t *>(values ? c.vs : c.ks) + first * S::sb, per * S::sb,
                                                  &sh.raw_full[slot]);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
                attn_next<S::rows, S::keys, kTileCost>(c, bt, io, p, kseq);
            }
            // (every copy has landed before the loaders, and so the CTA, are done)
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    // a wait gave up: what is still on its way to shared memory gets a millisecond to land
    if (*reinterpret_cast<volatile int *>(&sh.failed))
        for (const uint64_t t = global_timer_ns(); global_timer_ns() - t < 1000000;) __nanosleep(1000);
    __syncthreads();
    if (warp == 12) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Tensor map of a 16-bit cache tensor as rows of D values, read in boxes of `box` rows and 64 columns.
static int tile_map(CUtensorMap *map, void *data, int D, int64_t rows, int box) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) == cudaSuccess &&
                       found == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<Encode>(f)
                   : nullptr;
    }();
    if (!encode) return fail(ANVIL_ERR_CUDA, "cuTensorMapEncodeTiled not found");
    const cuuint64_t dims[2] = {cuuint64_t(D), cuuint64_t(rows)}, strides[1] = {cuuint64_t(2 * D)};
    const cuuint32_t boxes[2] = {64, cuuint32_t(box)}, steps[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, data, dims, strides, boxes, steps,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ANVIL_OK : fail(ANVIL_ERR_CUDA, "cuTensorMapEncodeTiled: error %d", int(r));
}

template <int KIND, int D> static int launch_tile(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                                                  bool join, cudaStream_t stream) {
    using S = TileShape<KIND, D>;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = attn_allow_smem(attn_tile_kernel<KIND, D>, S::smem, &allowed);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    // The warp groups' shares of the registers add up to 128 a thread: a build with fewer must not be launched
    // (the group that asks for more would wait for ever).
    static const int regs = [] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, attn_tile_kernel<KIND, D>) == cudaSuccess ? a.numRegs : 0;
    }();
    if (regs <= 120) return fail(ANVIL_ERR_UNSUPPORTED, "attention tile kernel built with %d registers", regs);
    CUtensorMap mk = {}, mv = {};
    const int64_t rows = (int64_t(c.num_pages) * c.kv_heads) << c.page_shift;
    int box = 0;  // TMA takes 16-bit rows, whole swizzle atoms of 8 keys, and 31-bit row numbers
    if (!S::quant && c.page_shift >= 3 && rows <= 0x7fffffff) {
        box = std::min(S::keys, 1 << c.page_shift);
        if (int st = tile_map(&mk, c.k, D, rows, box)) return st;
        if (int st = tile_map(&mv, c.v, D, rows, box)) return st;
    }
    attn_tile_kernel<KIND, D><<<ctas, kTileThreads, S::smem, stream>>>(c, bt, io, mk, mv, box, wait_limit_ns());
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "paged_attention launch");
    return join ? attn_join_launch<S::rows, D>(io, ctas, stream) : ANVIL_OK;
}

template <int KIND> static int tile_dim(int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                                        bool join, cudaStream_t s) {
    return D == 64 ? launch_tile<KIND, 64>(c, bt, io, ctas, join, s)
         : D == 128 ? launch_tile<KIND, 128>(c, bt, io, ctas, join, s)
                    : launch_tile<KIND, 256>(c, bt, io, ctas, join, s);
}

AttnTiles attn_tile_tiles(int D) { return D == 256 ? AttnTiles{128, 64, 1} : AttnTiles{256, 64, 1}; }

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
