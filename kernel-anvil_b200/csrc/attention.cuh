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
// order of the shares, so results do not depend on timing; a note of each CTA says which units there
// are to join (with a search for them by the joining CTAs a decode batch of 48 took 130 us, with the
// notes 113).  Lengths are read on the device; the grid depends on the batch's outer sizes alone, so a
// captured graph replays with other lengths.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "anvil.h"
#include "anvil_host.h"
#include "kv_cache.cuh"

namespace anvil {

// How far (in powers of two) a row's reference lies below the largest score when it is chosen, where weights are
// fp16: those lose bits below 2^-14 and end at 2^-25, so that with 2^6 for the largest, keys of 2^-31 of it still count and
// a first key with a high score does not drown thousands of low ones.  (bf16 weights have fp32's range.)
template <bool BF16> constexpr float kAttnHead = BF16 ? 0.0f : 6.0f;

struct AttnIO {
    const void *q;
    int64_t q_row, q_head;  // in values
    void *out;              // (total, heads, D)
    int heads, group;       // group: query heads per key/value head
    uint32_t group_mul;     // n / group = n * group_mul / 2^(32 + group_shift) for n < 2^31 (group 1: group_mul 0)
    int group_shift;
    float scale_log2;       // scale * log2(e): scores are kept in powers of two
    int causal;
    int q_bf16;             // q and out are bf16 (else fp16)
    int zero_rest;          // rows of no sequence become zeros (else they stay as they were)
    float *part;            // partial results, see AttnPart
};

// n / group without a division (group is the call's, and dozens of instructions as a divisor): with l the least
// power 2^l >= group and M = floor(2^(31+l) / group) + 1, M group exceeds 2^(31+l) by at most 2^l, so n M / 2^(31+l)
// exceeds n / group by less than 1 / group.
__device__ __forceinline__ unsigned by_group(const AttnIO &io, unsigned n) {
    return io.group_mul ? __umulhi(n, io.group_mul) >> io.group_shift : n;
}
inline void set_group(AttnIO &io, int group) {
    io.group = group;
    int l = 0;
    while ((int64_t(1) << l) < group) ++l;
    io.group_mul = group == 1 ? 0 : uint32_t((uint64_t(1) << (31 + l)) / group + 1);
    io.group_shift = l - 1;
}

// Partial results of CTA c: slot 2 c (the unit it found begun) and 2 c + 1 (the unit it left
// unfinished), each ROWS x (D + 2) floats: the rows' outputs, then maxima, then sums.
template <int ROWS, int D> struct AttnPart {
    static constexpr int floats = ROWS * (D + 2);
    static __device__ __forceinline__ float *slot(float *part, int cta, int which) {
        return part + (int64_t(cta) * 2 + which) * floats;
    }
};

// What CTA c says of slot 2 c + 1, behind all slots: the unit it began and did not finish.
struct alignas(16) AttnOpen {
    int parts;               // CTAs that have a part of it, c and the next ones; 0: none
    int token0, head0, row0; // its sequence's first packed row, its first query head, its first row
    int rows, pad[3];        // rows of the unit
};
template <int ROWS, int D> __device__ __forceinline__ AttnOpen *attn_open(float *part, int ctas) {
    return reinterpret_cast<AttnOpen *>(AttnPart<ROWS, D>::slot(part, ctas, 0));
}

// One sequence's units: row tiles and their key tiles.  Rows are counted in 32 bits (the host refuses
// batches of 2^31 query rows).
template <int ROWS, int KEYS> struct AttnSeq {
    KvSeq s;
    int n, tiles;  // new tokens; row tiles
    const AttnIO &io;

    __device__ __forceinline__ AttnSeq(const KvSeq &seq, const AttnIO &io)
        : s(seq), n(seq.q1 - seq.q0), tiles(int((unsigned(n) * unsigned(io.group) + ROWS - 1) / ROWS)), io(io) {}

    // Keys that some row of tile mt sees (its last token's), and their key tiles: at least one,
    // so that rows without keys are visited and get their zeros.
    __device__ __forceinline__ int keys(int mt) const {
        if (!io.causal) return s.kv;
        const int last = min(n - 1, int(by_group(io, unsigned(mt + 1) * ROWS - 1)));
        return kv_seen(last, n, s.kv, true);
    }
    __device__ __forceinline__ int key_tiles(int mt) const { return max(1, (keys(mt) + KEYS - 1) / KEYS); }
};

// A place in the order of all key tiles.  A unit counts COST places before its first key tile, what it
// takes to begin and end one in terms of a key tile's time.
struct AttnPos {
    int b, head, mt;
    int64_t unit0;  // place of the unit's first key tile
};

// a / b without the long 64-bit division where both are short
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : int64_t(unsigned(a) / unsigned(b));
}

// The division of `work` places over the grid: the first `more` CTAs get per + 1, the others per.
// CTAs that work: each has at least one place.
struct AttnShares {
    int64_t per;
    int ctas, more;
    __device__ __forceinline__ AttnShares(int64_t work, int grid) {
        ctas = int(min(work, int64_t(grid)));
        per = ctas ? div64(work, ctas) : 0;
        more = int(work - per * ctas);
    }
    __device__ __forceinline__ int64_t begin(int c) const { return per * c + min(c, more); }
    __device__ __forceinline__ int owner(int64_t place) const {  // the CTA whose share holds it
        const int64_t cut = (per + 1) * more;
        return place < cut ? int(div64(place, per + 1)) : more + int(div64(place - cut, per));
    }
};

struct AttnScratch {
    int64_t warp[33];
    int64_t at;     // place of the found sequence's first unit
    int b;          // the sequence that holds the place looked for
    AttnPos pos;
};

// Places of one head of a sequence; the lanes of a warp that called with `many` set get theirs from the
// whole warp, one after the other.
template <int ROWS, int KEYS, int COST>
__device__ __forceinline__ int64_t attn_head_work(const AttnSeq<ROWS, KEYS> &q, bool live) {
    int64_t w = 0;
    const bool many = live && q.io.causal && q.tiles > 2;
    if (live && !many) {
        w = q.tiles ? int64_t(q.tiles) * (q.key_tiles(0) + COST) : 0;
        if (q.io.causal && q.tiles == 2) w += q.key_tiles(1) - q.key_tiles(0);
    }
    for (uint32_t rest = __ballot_sync(0xffffffffu, many); rest; rest &= rest - 1) {
        const int src = __ffs(rest) - 1, lane = threadIdx.x & 31;
        AttnSeq<ROWS, KEYS> x = q;
        x.n = __shfl_sync(0xffffffffu, q.n, src);
        x.s.kv = __shfl_sync(0xffffffffu, q.s.kv, src);
        x.tiles = __shfl_sync(0xffffffffu, q.tiles, src);
        int sum = 0;  // of at most 2^31 / ROWS tiles of 2^31 / KEYS keys: split where it could overflow
        int64_t all = 0;
        for (int mt = lane; mt < x.tiles; mt += 32) {
            sum += x.key_tiles(mt);
            if (sum > (1 << 29)) {
                all += sum;
                sum = 0;
            }
        }
        all += sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        if (lane == src) w = all + int64_t(x.tiles) * COST;
    }
    return w;
}

// All threads: the total work; sc->pos becomes the unit that holds place pick(shares), for which its
// first key tile may lie before or behind that place.
template <int ROWS, int KEYS, int COST, typename Pick>
__device__ __forceinline__ int64_t attn_locate(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io,
                                               AttnScratch *sc, Pick pick, bool report) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int64_t work = 0, want = -1;
    // one pass where the batch fits the block; else one for the total and one to find the place
    const bool once = bt.batch <= int(blockDim.x);
    for (int pass = once ? 1 : 0; pass < 2; ++pass) {
        int64_t before = 0;
        for (int b0 = 0; b0 < bt.batch; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            KvSeq s{0, 0, 0, false};
            if (b < bt.batch) {
                s = load_seq(bt, c, b);
                if (s.bad && report && pass == 1) flag_bad_page();
            }
            const AttnSeq<ROWS, KEYS> q(s, io);
            const int64_t head = attn_head_work<ROWS, KEYS, COST>(q, q.n > 0);
            const int64_t mine = head * c.kv_heads;
            int64_t y = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) y += z;
            }
            __syncthreads();
            if (lane == 31) sc->warp[w] = y;
            __syncthreads();
            int64_t all = 0;
            int64_t at = before + y - mine;
            for (int i = 0; i < nw; ++i) {
                const int64_t v = sc->warp[i];
                if (i < w) at += v;
                all += v;
            }
            before += all;
            if (once) {
                work = all;
                want = work ? pick(AttnShares(work, gridDim.x)) : -1;
            }
            if (pass == 1 && mine && at <= want && want < at + mine) {
                sc->b = b;
                sc->at = at;
                sc->warp[32] = head;
            }
        }
        if (pass == 0) {
            work = before;
            want = work ? pick(AttnShares(work, gridDim.x)) : -1;
        }
    }
    __syncthreads();
    if (work == 0) return 0;
    if (w == 0) {
        // the unit within the sequence: every lane of warp 0 takes a row tile of the head
        const int b = sc->b;
        const AttnSeq<ROWS, KEYS> q(load_seq(bt, c, b), io);
        const int64_t per = sc->warp[32], head = div64(want - sc->at, per);
        int64_t unit = sc->at + head * per;  // place of the unit of row tile m0
        const int64_t rest = want - unit;
        AttnPos p{b, int(head), 0, 0};
        if (!io.causal || q.tiles == 1) {
            const int one = q.key_tiles(0) + COST;
            p.mt = int(rest / one);
            p.unit0 = unit + int64_t(p.mt) * one + COST;
        } else {
            for (int m0 = 0;; m0 += 32) {
                const int n = m0 + lane < q.tiles ? q.key_tiles(m0 + lane) + COST : 0;
                int64_t y = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
                    if (lane >= o) y += z;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, unit + y > want);
                if (hit || m0 + 32 >= q.tiles) {
                    const int l = hit ? __ffs(hit) - 1 : 31;
                    p.mt = m0 + l;
                    p.unit0 = unit + __shfl_sync(0xffffffffu, y - n, l) + COST;
                    break;
                }
                unit += __shfl_sync(0xffffffffu, y, 31);
            }
        }
        if (lane == 0) sc->pos = p;
    }
    __syncthreads();
    return work;
}

// The unit behind p's; b reaches bt.batch behind the last.  seq: p's sequence, looked up again only where it changes.
template <int ROWS, int KEYS, int COST>
__device__ __forceinline__ void attn_next(const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, AttnPos &p, KvSeq &seq) {
    const AttnSeq<ROWS, KEYS> q(seq, io);
    p.unit0 += q.key_tiles(p.mt) + COST;
    if (++p.mt < q.tiles) return;
    p.mt = 0;
    if (++p.head < c.kv_heads) return;
    p.head = 0;
    for (++p.b; p.b < bt.batch; ++p.b) {
        seq = load_seq(bt, c, p.b);
        if (seq.q1 > seq.q0) return;
    }
}

// Zeros for the rows before the first sequence and behind the last one, by the last warp of every CTA: the others need not
// wait for the starts (a decode step of one sequence takes 8.7 us, with all warps 8.8, without zeros 8.6).
template <int D>
__device__ __forceinline__ void attn_zero_rest(const KvBatchView &bt, const AttnIO &io) {
    const int lane = int(threadIdx.x) - int(blockDim.x) + 32;
    if (!io.zero_rest || lane < 0) return;
    const int64_t row = int64_t(io.heads) * (D / 8);  // 16-byte pieces
    const int64_t begin = min(max(bt.start[0], 0), bt.total) * row, end = min(max(bt.start[bt.batch], 0), bt.total) * row;
    const int64_t rest = begin + (bt.total * row - end);
    uint4 *out = static_cast<uint4 *>(io.out);
    for (int64_t i = int64_t(blockIdx.x) * 32 + lane; i < rest; i += int64_t(gridDim.x) * 32)
        out[i < begin ? i : i - begin + end] = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 operations at once
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The exponent of 2 that the row of a bf16 query is multiplied by so that it fits fp16: its largest magnitude goes to
// [2^13, 2^14), as far as the factor and its inverse are normal fp32 numbers, from 2^-114 to 2^126 (which brings the
// smallest normal magnitude to 1).  0 for zeros, infinities and NaN.
__device__ __forceinline__ int q_exponent(uint32_t amax_bits) {
    const int e = int(amax_bits >> 23);
    if (amax_bits == 0 || e == 255) return 0;
    return min(126, 127 + 13 - e);
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

// Two blocks' scales as the products take them: NaN where a block's largest value could pass fp16, above 512 (Q8_0, codes
// of up to 127) or 8188 (Q4_0, of up to 8), which a cache that anvil_kv_write filled does not have.  Products of such
// scales would be infinite in some places only, and zero weights times them NaN in rows that do not see them; so the block is
// one with a non-finite scale, of which the kernels take care.  The largest allowed scale times the factor is 65504, the
// next one's product rounds to infinity, and zero times that is NaN.
template <int KIND> __device__ __forceinline__ uint32_t usable_scales(uint32_t d) {
    constexpr uint32_t factor = KIND == kKvQ8_0 ? 0x57FF57FFu : 0x48004800u;  // 127.9375, 8
    return h2fma(h2mul(d, factor), 0u, d);
}
// From here on, in bits of the magnitude, a usable scale needs care in tiles that some row does not see: NaN; and 512, which
// with the code -128 (not of the type, but a tensor may hold it) passes fp16, while 511.75, 2^-11 less, does not.
template <int KIND> constexpr uint32_t kOddScale = KIND == kKvQ8_0 ? 0x6000 : 0x7C00;

// Value e of a cache row, as the products take it.
template <int KIND, int D>
__device__ __forceinline__ float kv_value(const uint8_t *data, const __half *scales, int64_t row, int e) {
    auto scale = [&] {
        const uint32_t d = usable_scales<KIND>(__half_as_ushort(scales[row * (D / 32) + e / 32]));
        return __half2float(__ushort_as_half(uint16_t(d)));
    };
    if constexpr (KIND == kKvF16) {
        return __half2float(reinterpret_cast<const __half *>(data)[row * D + e]);
    } else if constexpr (KIND == kKvBF16) {
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(data)[row * D + e]);
    } else if constexpr (KIND == kKvQ8_0) {
        return float(reinterpret_cast<const int8_t *>(data)[row * D + e]) * scale();
    } else {
        const uint8_t w = data[row * (D / 2) + (e / 32) * 16 + (e % 16)];
        return float(int((e % 32) < 16 ? w & 15 : w >> 4) - 8) * scale();
    }
}

// Joins the partial results of the unit that CTA `blockIdx.x` of the attention kernel began and did
// not finish: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.  A row's parts are shared by 1, 2, 4 or 8 of the
// eight warps, at most 8 parts a warp where there are that many; the order of the sums is fixed by the parts.
// Bound by latency (launch, note, parts): 3 to 10 us, the most where one sequence was cut into hundreds of parts.
constexpr int kJoinWarps = 8;
template <int ROWS, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(AttnIO io) {
    __shared__ __align__(16) float so[kJoinWarps][D];
    __shared__ float sl[kJoinWarps];
    const int cta = blockIdx.x;
    pdl_wait();  // the partial results are the kernel before's; waited for by every CTA
    const AttnOpen open = attn_open<ROWS, D>(io.part, gridDim.x)[cta];
    const int np = open.parts;
    if (np == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = np > 32 ? 8 : np > 16 ? 4 : np > 8 ? 2 : 1;  // warps of a row
    const int sub = warp % share, rows = kJoinWarps / share;        // rows at once
    const int nrows = open.rows;
    using P = AttnPart<ROWS, D>;
    constexpr int V = D / 32;
    for (int r0 = blockIdx.y * rows; r0 < nrows; r0 += rows * gridDim.y) {
        const int row = r0 + warp / share;
        const bool live = row < nrows;
        float o[V] = {}, l = 0.0f;
        if (live) {
            float m = -INFINITY;
            for (int i = lane; i < np; i += 32) m = fmaxf(m, P::slot(io.part, cta + i, i == 0)[ROWS * D + row]);
            m = warp_max(m);
            const float base = m == -INFINITY ? 0.0f : m;
            for (int i0 = sub * 8; i0 < np; i0 += share * 8) {
                // eight parts at a time: their weights on lanes 0..7, their loads in flight together
                float a = 0.0f, pl = 0.0f;
                if (lane < 8 && i0 + lane < np) {
                    const float *s = P::slot(io.part, cta + i0 + lane, i0 + lane == 0) + ROWS * D + row;
                    a = ex2(s[0] - base);
                    pl = a * s[ROWS];
                }
                float x[8][V];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i0 + i < np) {
                        const float *s = P::slot(io.part, cta + i0 + i, i0 + i == 0) + row * D + lane * V;
#pragma unroll
                        for (int j = 0; j < V; j += 2) {
                            const float2 y = *reinterpret_cast<const float2 *>(s + j);
                            x[i][j] = y.x;
                            x[i][j + 1] = y.y;
                        }
                    }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i0 + i < np) {
                        const float ai = __shfl_sync(0xffffffffu, a, i);
                        l += __shfl_sync(0xffffffffu, pl, i);
#pragma unroll
                        for (int j = 0; j < V; ++j) o[j] += ai * x[i][j];
                    }
            }
        }
        if (share > 1) {  // uniform: the warps of a row meet
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) so[warp][lane * V + j] = o[j];
            if (lane == 0) sl[warp] = l;
            __syncthreads();
            if (sub == 0)
                for (int i = 1; i < share; ++i) {
                    l += sl[warp + i];
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] += so[warp + i][lane * V + j];
                }
        }
        if (!live || sub) continue;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const unsigned r = unsigned(open.row0) + row;
        const int tok = int(by_group(io, r)), token = open.token0 + tok, h = open.head0 + int(r - unsigned(tok) * io.group);
        uint32_t *out = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(io.out) +
                                                     (int64_t(token) * io.heads + h) * D) + lane * (V / 2);
#pragma unroll
        for (int j = 0; j < V / 2; ++j)
            out[j] = io.q_bf16 ? pack_bf16(o[2 * j] * inv, o[2 * j + 1] * inv)
                               : pack_half(o[2 * j] * inv, o[2 * j + 1] * inv);
    }
}

// Lets `fn` use `bytes` of dynamic shared memory, once for each device (up to 64; beyond, every time).
template <typename F> static cudaError_t attn_allow_smem(F *fn, int bytes, std::atomic<uint64_t> *done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done->load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Host side: a kernel's row tile, key tile and resident CTAs of an SM.
struct AttnTiles {
    int rows, keys, occ;
};

template <int ROWS, int D> static int attn_join_launch(const AttnIO &io, int ctas, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, std::min(ROWS / 2, 8));
    cfg.blockDim = kJoinWarps * 32;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_join_kernel<ROWS, D>, io);
    return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "paged_attention join launch");
}

}  // namespace anvil
