// attention.cuh -- what the attention kernels share: the call's arguments, the division of a ragged
// batch over a fixed grid, and small helpers.
//
// Division.  The query rows of a sequence that read one key/value head (q_len x group of them:
// row r is token r / group, head r % group) are cut into row tiles; a (sequence, head, row tile)
// is a unit, and a unit's keys are cut into key tiles.  All key tiles of all units, in the order
// sequence, head, row tile, key tile, are dealt to the grid's CTAs in equal contiguous shares, so
// every CTA has the same work whatever the lengths, and neighbouring CTAs read the same keys.  A
// unit that lies in one share is finished there; a unit that spans shares leaves one partial
// result (unnormalised output, maximum, sum) per share, and a second kernel joins them in the
// order of the shares, so results do not depend on timing.  Lengths are read on the device; the
// grid depends on the batch's outer sizes alone, so a captured graph replays with other lengths.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "kv_cache.cuh"

namespace anvil {

struct AttnIO {
    const void *q;
    int64_t q_row, q_head;  // in values
    void *out;              // (total, heads, D)
    int heads, group;       // group: query heads per key/value head
    float scale_log2;       // scale * log2(e): scores are kept in powers of two
    int causal;
    int q_bf16;             // q and out are bf16 (else fp16)
    float *part;            // partial results, see AttnPart
};

// Partial results of CTA c: slot 2 c (the unit it found begun) and 2 c + 1 (the unit it left
// unfinished), each ROWS x (D + 2) floats: the rows' outputs, then maxima, then sums.
template <int ROWS, int D> struct AttnPart {
    static constexpr int floats = ROWS * (D + 2);
    static __device__ __forceinline__ float *slot(float *part, int cta, int which) {
        return part + (int64_t(cta) * 2 + which) * floats;
    }
};

// One sequence's units: row tiles and their key tiles.
template <int ROWS, int KEYS> struct AttnSeq {
    KvSeq s;
    int n, group, causal, tiles;  // new tokens; row tiles

    __device__ __forceinline__ AttnSeq(const KvSeq &seq, const AttnIO &io)
        : s(seq), n(seq.q1 - seq.q0), group(io.group), causal(io.causal),
          tiles(int((int64_t(n) * io.group + ROWS - 1) / ROWS)) {}

    // Keys that some row of tile mt sees (its last token's), and their key tiles: at least one,
    // so that rows without keys are visited and get their zeros.
    __device__ __forceinline__ int keys(int mt) const {
        const int last = min(n - 1, int((int64_t(mt + 1) * ROWS - 1) / group));
        return kv_seen(last, n, s.kv, causal);
    }
    __device__ __forceinline__ int key_tiles(int mt) const { return max(1, (keys(mt) + KEYS - 1) / KEYS); }
    __device__ __forceinline__ int64_t head_work() const {  // key tiles of one head
        if (!causal) return int64_t(tiles) * key_tiles(0);
        int64_t w = 0;
        for (int mt = 0; mt < tiles; ++mt) w += key_tiles(mt);
        return w;
    }
};

// A place in the order of all key tiles.
struct AttnPos {
    int b, head, mt, tile;  // key tile `tile` of the unit
    int64_t unit0;          // global number of the unit's first key tile
};

// CTAs that work: each has at least one key tile.
__device__ __forceinline__ int attn_ctas(int64_t work, int grid) { return int(min(work, int64_t(grid))); }
// CTA c's share of `work` key tiles is [share(c), share(c + 1)).
__device__ __forceinline__ int64_t attn_share(int64_t work, int c, int ctas) { return work * c / ctas; }
// The CTA whose share holds key tile t: the last c with share(c) <= t.
__device__ __forceinline__ int attn_owner(int64_t work, int64_t t, int ctas) {
    return int(((t + 1) * ctas - 1) / work);
}

// All threads: the total work, and the position of key tile `share(cta) + ahead` (valid where that
// is below the work).  scratch: blockDim.x / 32 + 1 words of 64 bits and an AttnPos in shared memory.
struct AttnScratch {
    int64_t warp[33];
    AttnPos pos;
};

__device__ __forceinline__ int64_t block_scan(int64_t x, AttnScratch *sc, int64_t *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int64_t y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    __syncthreads();
    if (lane == 31) sc->warp[w] = y;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < nw; ++i) {
        const int64_t v = sc->warp[i];
        if (i < w) before += v;
        all += v;
    }
    *total = all;
    return before + y - x;  // exclusive
}

template <int ROWS, int KEYS, typename PickTile>
__device__ __forceinline__ int64_t attn_locate(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io,
                                               AttnScratch *sc, PickTile pick, bool report) {
    // pass 1: the total (and, for batches of one chunk, each sequence's work in a register)
    int64_t work = 0, mine = 0;
    for (int b0 = 0; b0 < bt.batch; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        mine = 0;
        if (b < bt.batch) {
            const KvSeq s = load_seq(bt, c, b);
            if (s.bad && report) flag_bad_page();
            if (s.q1 > s.q0) mine = AttnSeq<ROWS, KEYS>(s, io).head_work() * c.kv_heads;
        }
        int64_t t;
        block_scan(mine, sc, &t);
        work += t;
    }
    if (threadIdx.x == 0) sc->pos.b = -1;
    const int64_t want = work ? pick(work) : 0;  // uniform
    int64_t before = 0;
    for (int b0 = 0; b0 < bt.batch && work; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        if (bt.batch > blockDim.x) {
            mine = 0;
            if (b < bt.batch) {
                const KvSeq s = load_seq(bt, c, b);
                if (s.q1 > s.q0) mine = AttnSeq<ROWS, KEYS>(s, io).head_work() * c.kv_heads;
            }
        }
        int64_t t;
        const int64_t at = before + block_scan(mine, sc, &t);
        if (mine && at <= want && want < at + mine) {
            const AttnSeq<ROWS, KEYS> q(load_seq(bt, c, b), io);
            const int64_t per = mine / c.kv_heads, head = (want - at) / per;
            int64_t rest = want - at - head * per;
            int mt = 0;
            while (rest >= q.key_tiles(mt)) rest -= q.key_tiles(mt++);
            sc->pos = AttnPos{b, int(head), mt, int(rest), want - rest};
        }
        before += t;
    }
    __syncthreads();
    return work;
}

// The unit behind p's (p is moved to its first key tile); b reaches bt.batch behind the last.
template <int ROWS, int KEYS>
__device__ __forceinline__ void attn_next(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io,
                                          AttnPos &p, const AttnSeq<ROWS, KEYS> &q) {
    p.unit0 += q.key_tiles(p.mt);
    p.tile = 0;
    if (++p.mt < q.tiles) return;
    p.mt = 0;
    if (++p.head < c.kv_heads) return;
    p.head = 0;
    for (++p.b; p.b < bt.batch; ++p.b) {
        const KvSeq s = load_seq(bt, c, p.b);
        if (s.q1 > s.q0) return;
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The exponent of 2 that the row of a bf16 query is multiplied by so that it fits fp16 (its
// largest magnitude in [2^13, 2^14)); 0 for zeros, infinities and NaN.  Bounded so that the
// factor and its inverse are fp32 numbers.
__device__ __forceinline__ int q_exponent(uint32_t amax_bits) {
    const int e = int(amax_bits >> 23);
    if (amax_bits == 0 || e == 255) return 0;
    return max(-100, min(100, 127 + 13 - e));
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Which of the two 16-bit floats of w are infinite or NaN, as a mask of their bits.
template <bool BF16> __device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
    constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
    return ((w & E) == E ? 0xFFFFu : 0u) | (((w >> 16) & E) == E ? 0xFFFF0000u : 0u);
}

// Value e of a cache row.
template <int KIND, int D>
__device__ __forceinline__ float kv_value(const uint8_t *data, const __half *scales, int64_t row, int e) {
    if constexpr (KIND == kKvF16) {
        return __half2float(reinterpret_cast<const __half *>(data)[row * D + e]);
    } else if constexpr (KIND == kKvBF16) {
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(data)[row * D + e]);
    } else if constexpr (KIND == kKvQ8_0) {
        return float(reinterpret_cast<const int8_t *>(data)[row * D + e]) *
               __half2float(scales[row * (D / 32) + e / 32]);
    } else {
        const uint8_t w = data[row * (D / 2) + (e / 32) * 16 + (e % 16)];
        return float(int((e % 32) < 16 ? w & 15 : w >> 4) - 8) * __half2float(scales[row * (D / 32) + e / 32]);
    }
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

// Joins the partial results of the unit that CTA `blockIdx.x` of the attention kernel began and did
// not finish, every gridDim.y-th four rows of it: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.
template <int ROWS, int KEYS, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(KvCacheView c, KvBatchView bt, AttnIO io) {
    __shared__ AttnScratch sc;
    const int cta = blockIdx.x;
    const int64_t work = attn_locate<ROWS, KEYS>(
        c, bt, io, &sc,
        [&](int64_t w) {
            const int n = attn_ctas(w, gridDim.x);
            return attn_share(w, min(cta + 1, n), n) - 1;  // the share's last key tile
        },
        false);
    pdl_wait();  // the partial results are the kernel before's; waited for by every CTA
    const int ctas = attn_ctas(work, gridDim.x);
    if (cta >= ctas) return;
    const AttnPos p = sc.pos;
    const int64_t lo = attn_share(work, cta, ctas), hi = attn_share(work, cta + 1, ctas);
    if (p.unit0 < lo) return;  // begun elsewhere
    const AttnSeq<ROWS, KEYS> q(load_seq(bt, c, p.b), io);
    const int64_t end = p.unit0 + q.key_tiles(p.mt);
    if (end <= hi) return;  // finished where it was begun
    const int last = attn_owner(work, end - 1, ctas);
    const int lane = threadIdx.x & 31;
    using P = AttnPart<ROWS, D>;
    for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < ROWS; row += 4 * gridDim.y) {
        const int64_t r = int64_t(p.mt) * ROWS + row;
        if (r >= int64_t(q.n) * q.group) return;
        float m = -INFINITY;
        for (int i = cta + lane; i <= last; i += 32) m = fmaxf(m, P::slot(io.part, i, i == cta)[ROWS * D + row]);
        m = warp_max(m);
        const float base = m == -INFINITY ? 0.0f : m;
        constexpr int V = D / 32;
        float o[V] = {}, l = 0.0f;
        for (int i = cta; i <= last; ++i) {
            const float *s = P::slot(io.part, i, i == cta);
            const float a = ex2(s[ROWS * D + row] - base);
            l += a * s[ROWS * D + ROWS + row];
            if constexpr (V == 2) {
                const float2 x = *reinterpret_cast<const float2 *>(s + row * D + lane * 2);
                o[0] += a * x.x;
                o[1] += a * x.y;
            } else {
#pragma unroll
                for (int j = 0; j < V / 4; ++j) {
                    const float4 x = *reinterpret_cast<const float4 *>(s + row * D + j * 128 + lane * 4);
                    o[4 * j] += a * x.x;
                    o[4 * j + 1] += a * x.y;
                    o[4 * j + 2] += a * x.z;
                    o[4 * j + 3] += a * x.w;
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int token = q.s.q0 + int(r / q.group), h = p.head * q.group + int(r % q.group);
        uint32_t *out = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(io.out) +
                                                     (int64_t(token) * io.heads + h) * D);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const int at = V == 2 ? lane : (j / 2) * 64 + lane * 2 + (j & 1);
            out[at] = io.q_bf16 ? pack_bf16(o[2 * j] * inv, o[2 * j + 1] * inv)
                                : pack_half(o[2 * j] * inv, o[2 * j + 1] * inv);
        }
    }
}

// Host side: a kernel's row tile, key tile and resident CTAs of an SM.
struct AttnTiles {
    int rows, keys, occ;
};

template <int ROWS, int KEYS, int D>
static int attn_join_launch(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                            cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, std::min(ROWS / 4, 8));
    cfg.blockDim = 128;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_join_kernel<ROWS, KEYS, D>, c, bt, io);
    return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "paged_attention join launch");
}

}  // namespace anvil
