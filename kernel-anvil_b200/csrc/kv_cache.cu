// kv_cache.cu -- the paged key/value cache's write and read: quantising new tokens' keys and
// values as they are put into their pages, and bringing cached rows back as values.
//
// Write, blocks of 32 along a head's values (x exact, M = the block's largest magnitude):
//   Q8_0: d = M / 127, code = 127 x / M to the nearest integer, halves away from zero
//   Q4_0: d = top / -8 (top: the value of largest magnitude, the first of equals),
//         nibble = min(15, floor(x / d + 8.5))
// and the stored scale is fp16(d), rounded once.  Codes are those of exact arithmetic: the fp32
// quotient picks a candidate, and where it lies near a border the sign of an exactly evaluated
// remainder decides (fma), so the result does not depend on how a quotient was rounded.
// Magnitudes above kKvMax = 127 * 512 are stored as kKvMax in the quantised kinds, so that
// every stored value is a finite fp16; a block that holds a NaN gets a NaN scale.
//
// Both kernels move each byte once.  7993 bf16 tokens of 8 heads of 128: F16 written in 8 us (the L2 takes them), read in 8;
// Q8_0 18 and 9, Q4_0 24 and 11: the write of the quantised kinds is bound by the instructions that find the
// codes.  Reading 32801 tokens of Q8_0 as bf16 (206 MB) takes 40 us, 78% of the measured HBM rate, and a decode
// step's 48 rows 3 us each way, which is the launch.  (Two, three or four rows a thread in the read, for more loads on
// their way, took 43 to 44 us, and a decode step 1 to 2 us more.)  One lane handles 8 values of a row (16 bytes of a 16-bit input), so a
// block is four neighbouring lanes and its maximum is two shuffles; keys and values of a row are
// handled by the same lanes, which keeps two independent streams of loads in flight.
#include <cuda_runtime.h>

#include <algorithm>

#include "anvil.h"
#include "anvil_host.h"
#include "kv_cache.cuh"

namespace anvil {

constexpr float kKvMax = 65024.0f;  // 127 * 512

struct KvIO {
    // write: the new rows (strides in values); read: the destination (contiguous)
    const void *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    void *ok, *ov;
    const int *first;  // read: position of each sequence's first row (null: 0)
    int zero_rest;     // read: rows of no sequence become zeros (else they stay as they were)
};

// ---- input / output of 8 values ---------------------------------------------------------

template <typename T> struct Vec8;
template <> struct Vec8<float> {
    static __device__ __forceinline__ void load(const void *p, int64_t at, float (&x)[8]) {
        const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        const float4 a = __ldg(q), b = __ldg(q + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void store(void *p, int64_t at, const float (&x)[8]) {
        float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + at);
        __stcs(q, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(q + 1, make_float4(x[4], x[5], x[6], x[7]));
    }
};
template <> struct Vec8<__half> {
    static __device__ __forceinline__ void load(const void *p, int64_t at, float (&x)[8]) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __half *>(p) + at));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ void store(void *p, int64_t at, const float (&x)[8]) {
        __stcs(reinterpret_cast<uint4 *>(static_cast<__half *>(p) + at), pack(x));
    }
};
template <> struct Vec8<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const void *p, int64_t at, float (&x)[8]) {
        const uint4 w =
            __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p) + at));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ void store(void *p, int64_t at, const float (&x)[8]) {
        __stcs(reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p) + at), pack(x));
    }
};

// ---- quantising 8 values of a 32-value block (lanes 4m..4m+3) -----------------------------

// Largest magnitude of the block as fp32 bits; NaN (bits above infinity's) wins.
__device__ __forceinline__ uint32_t block_amax_bits(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        m = __vimax3_u32(m, __float_as_uint(x[i]) & 0x7FFFFFFFu, __float_as_uint(x[i + 1]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

__device__ __forceinline__ float clamp_kv(float x) { return fminf(fmaxf(x, -kKvMax), kKvMax); }

// A value's code takes five fp32 operations; one that lies near a border between two codes is then decided
// exactly.  (With the exact decision inlined for every value the write of 7993 tokens took 31 us for Q4_0 and 25 for
// Q8_0, now 24 and 18; inputs of 16 bits lie on borders of Q4_0 often, so that recomputing a lane's eight values for one
// of them was no better.)
constexpr float kKvMagic = 12582912.0f;  // 1.5 * 2^23: x + kKvMagic holds round(x) in its last bits
constexpr float kKvNear = 0.4999f;       // |x - round(x)| from here on: near a border

// fp16(M / 127) where the product with 1 / 127 (off by 2 units in the last place at most) is not near a border
// between two halves; else and for subnormal halves, exactly.
__device__ __forceinline__ __half q8_scale_half(float M);
__device__ __forceinline__ __half q8_scale_fast(float M) {
    const float q = M * (1.0f / 127.0f);
    const uint32_t rest = __float_as_uint(q) & 0x1FFFu;
    if (q < 0x1p-13f || (rest > 0x1000u - 8 && rest < 0x1000u + 8)) return q8_scale_half(M);
    return __float2half_rn(q);
}

// fp16(M / 127), rounded once: the truncated quotient with a sticky last bit (set when the
// remainder M - q 127, which fma gives exactly, is not zero) rounds to fp16 as M / 127 does.
__device__ __forceinline__ __half q8_scale_half(float M) {
    const float q = __fdiv_rz(M, 127.0f);
    const uint32_t sticky = fmaf(-q, 127.0f, M) != 0.0f ? 1u : 0u;
    return __float2half_rn(__uint_as_float(__float_as_uint(q) | sticky));
}

// round_half_away(127 x / M) where t = 127 x / M to within 1e-4 and k = round(t) are known and t lies near a border
// of k, b = |k| +- 1/2: the sign of 127 |x| - b M decides.  p + e is 127 |x| exactly, and p - b M is exact this near
// to zero.
__device__ __noinline__ float q8_border(float x, float M, float t, float k) {
    const float a = fabsf(x), b = fabsf(k) + (fabsf(t) > fabsf(k) ? 0.5f : -0.5f);
    const float p = a * 127.0f, e = fmaf(a, 127.0f, -p);
    return copysignf(b + (fmaf(-b, M, p) + e >= 0.0f ? 0.5f : -0.5f), x);
}

__device__ __forceinline__ uint2 quant8_q8(const float (&x)[8], __half &d) {
    const uint32_t mb = block_amax_bits(x);
    uint2 w = make_uint2(0, 0);
    if (mb > 0x7F800000u) {  // a NaN: the whole block reads back as NaN
        d = __ushort_as_half(0x7FFF);
        return w;
    }
    const float M = fminf(__uint_as_float(mb), kKvMax);
    d = q8_scale_fast(M);
    if (M == 0.0f) return w;
    // below 2^-100 M is scaled up with its block (exactly), so that no quotient or remainder
    // is subnormal; such a block's scale is zero in fp16 and its codes stand for zeros
    const float up = M < 0x1p-100f ? 0x1p100f : 1.0f, Ms = M * up;
    const float inv = __fdividef(127.0f, Ms);  // 127 x / M off by less than 1e-4
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = clamp_kv(x[i]) * up, t = c * inv, m = t + kKvMagic, k = m - kKvMagic;
        r[i] = __float_as_uint(m);
        if (fabsf(t - k) >= kKvNear) r[i] = __float_as_uint(q8_border(c, Ms, t, k) + kKvMagic);
    }
    w.x = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
    return w;
}

// floor(t + 1/2) for t = -8 x / top, known to within 1e-5, where it lies near a border b = k +- 1/2 of k = round(t):
// t - b = (-8 x - b top) / top, and the numerator's sign is that of one fma.
__device__ __noinline__ float q4_border(float x, float top, float t, float k) {
    const float b = k + (t > k ? 0.5f : -0.5f), s = fmaf(-b, top, -8.0f * x);
    return b + (s == 0.0f || ((s > 0.0f) == (top > 0.0f)) ? 0.5f : -0.5f);
}

__device__ __forceinline__ uint32_t quant8_q4(const float (&x)[8], __half &d) {
    const uint32_t mb = block_amax_bits(x);
    const float M = mb > 0x7F800000u ? 0.0f : fminf(__uint_as_float(mb), kKvMax);
    // the first value of the block whose magnitude is M decides the sign
    int key = 1 << 20;
#pragma unroll
    for (int i = 7; i >= 0; --i)
        if (fabsf(x[i]) >= M) key = (((threadIdx.x & 3) * 8 + i) << 1) | (x[i] < 0.0f ? 1 : 0);
    key = min(key, __shfl_xor_sync(0xffffffffu, key, 1));
    key = min(key, __shfl_xor_sync(0xffffffffu, key, 2));
    if (mb > 0x7F800000u) {  // after the shuffles, which every lane of the warp takes part in
        d = __ushort_as_half(0x7FFF);
        return 0;
    }
    const float top = (key & 1) ? -M : M;
    d = __float2half_rn(top / -8.0f);
    if (M == 0.0f) {
        d = __float2half_rn(0.0f);
        return 0x88888888u;
    }
    // nibble = min(15, floor(t + 8.5)), t = -8 x / top within [-8, 8]; from 7.25 on it is 15
    const float up = M < 0x1p-100f ? 0x1p100f : 1.0f, ts = top * up;
    const float inv = __fdividef(-8.0f, ts);
    uint32_t w = 0;  // nibble i = value i
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = clamp_kv(x[i]) * up, t = fminf(c * inv, 7.25f), m = t + (kKvMagic + 8.0f), k = m - (kKvMagic + 8.0f);
        uint32_t r = __float_as_uint(m);
        if (fabsf(t - k) >= kKvNear) r = __float_as_uint(q4_border(c, ts, t, k) + (kKvMagic + 8.0f));
        w |= (r & 15u) << (4 * i);
    }
    return w;
}

// Nibbles of 4 values (bits 4i) spread to the low nibbles of 4 bytes.
__device__ __forceinline__ uint32_t spread4(uint32_t n) {
    n = (n | (n << 8)) & 0x00FF00FFu;
    return (n | (n << 4)) & 0x0F0F0F0Fu;
}

// Stores one row's 8 values of this lane (values 8 l .. 8 l + 7 of the row at `row`).  All lanes
// of a block take part; `row` < 0 stores nothing.
template <int KIND, int D>
__device__ __forceinline__ void store_row(uint8_t *data, __half *scales, int64_t row, int l,
                                          const float (&x)[8]) {
    if constexpr (KIND == kKvF16) {
        if (row >= 0)
            *reinterpret_cast<uint4 *>(data + row * (2 * D) + l * 16) = Vec8<__half>::pack(x);
    } else if constexpr (KIND == kKvBF16) {
        if (row >= 0)
            *reinterpret_cast<uint4 *>(data + row * (2 * D) + l * 16) = Vec8<__nv_bfloat16>::pack(x);
    } else if constexpr (KIND == kKvQ8_0) {
        __half d;
        const uint2 w = quant8_q8(x, d);
        if (row >= 0) {
            *reinterpret_cast<uint2 *>(data + row * D + l * 8) = w;
            if ((l & 3) == 0) scales[row * (D / 32) + (l >> 2)] = d;
        }
    } else {
        __half d;
        const uint32_t w = quant8_q4(x, d);
        // bytes 0..7 of the block pair values 0..7 with 16..23 (lanes 0 and 2), bytes 8..15
        // values 8..15 with 24..31 (lanes 1 and 3): the lower lane of a pair stores four bytes,
        // the upper one the other four
        const uint32_t o = __shfl_xor_sync(0xffffffffu, w, 2);
        const int up = (l >> 1) & 1;
        const uint32_t lo = up ? o : w, hi = up ? w : o;
        const uint32_t bytes = spread4((lo >> (16 * up)) & 0xFFFFu) |
                               (spread4((hi >> (16 * up)) & 0xFFFFu) << 4);
        if (row >= 0) {
            *reinterpret_cast<uint32_t *>(data + row * (D / 2) + (l >> 2) * 16 + (l & 1) * 8 +
                                          up * 4) = bytes;
            if ((l & 3) == 0) scales[row * (D / 32) + (l >> 2)] = d;
        }
    }
}

template <int KIND, int D>
__device__ __forceinline__ void load_row(const uint8_t *data, const __half *scales, int64_t row,
                                         int l, float (&x)[8]) {
    if constexpr (KIND == kKvF16) {
        Vec8<__half>::load(data, row * D + l * 8, x);
    } else if constexpr (KIND == kKvBF16) {
        Vec8<__nv_bfloat16>::load(data, row * D + l * 8, x);
    } else if constexpr (KIND == kKvQ8_0) {
        const uint2 w = __ldg(reinterpret_cast<const uint2 *>(data + row * D + l * 8));
        const float d = __half2float(__ldg(scales + row * (D / 32) + (l >> 2)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // code + 128 in the last byte of 2^23
            const uint32_t b = __byte_perm((i < 4 ? w.x : w.y) ^ 0x80808080u, 0x4B000000u, 0x7650 | (i & 3));
            x[i] = (__uint_as_float(b) - 8388736.0f) * d;
        }
    } else {
        const uint2 w =
            __ldg(reinterpret_cast<const uint2 *>(data + row * (D / 2) + (l >> 2) * 16 + (l & 1) * 8));
        const float d = __half2float(__ldg(scales + row * (D / 32) + (l >> 2)));
        const int sh = (l & 2) ? 4 : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // the nibble in the last byte of 2^23
            const uint32_t n = ((i < 4 ? w.x : w.y) >> (8 * (i & 3) + sh)) & 15u;
            x[i] = (__uint_as_float(n | 0x4B000000u) - 8388616.0f) * d;
        }
    }
}

// ---- kernels ------------------------------------------------------------------------------

// The sequence that packed row t belongs to, or -1.  One token a sequence (a decode step) is
// guessed first; else a binary search over the starts.
__device__ __forceinline__ int seq_of_row(const KvBatchView &bt, int t) {
    int b = min(t, bt.batch - 1);
    if (bt.start[b] <= t && t < bt.start[b + 1]) return b;
    int lo = 0, hi = bt.batch;  // the last b with start[b] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (bt.start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return bt.start[lo] <= t && t < bt.start[lo + 1] ? lo : -1;
}

// By the grid's first CTA: reports every start and length out of range, of sequences without rows in this call too.
__device__ __forceinline__ void report_bad_entries(const KvCacheView &c, const KvBatchView &bt) {
    if (blockIdx.x || blockIdx.y) return;
    bool bad = false;
    for (int b = threadIdx.x; b < bt.batch; b += blockDim.x) bad |= load_seq(bt, c, b).bad;
    if (bad) flag_bad_page();
}

constexpr int kKvThreads = 256;

template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(KvCacheView c, KvBatchView bt, KvIO io) {
    constexpr int LPR = D / 8;  // lanes of a row
    const int64_t t = int64_t(blockIdx.x) * (kKvThreads / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR, h = blockIdx.y;
    int64_t row = -1;
    const bool live = t < bt.total;
    float k[8] = {}, v[8] = {};
    if (live) {
        Vec8<T>::load(io.k, t * io.k_row + h * io.k_head + l * 8, k);
        Vec8<T>::load(io.v, t * io.v_row + h * io.v_head + l * 8, v);
        const int b = seq_of_row(bt, int(t));
        if (b >= 0) {
            // (cut entries would name other positions, with tokens that are to stay)
            const KvSeq s = load_seq(bt, c, b);
            const int pos = s.kv - (s.q1 - s.q0) + (int(t) - s.q0);
            if (pos >= 0 && !s.bad) row = kv_lookup(bt, c, b, pos, h);
            if (row < 0 && l == 0) flag_bad_page();
        }
    }
    store_row<KIND, D>(c.k, c.ks, row, l, k);
    store_row<KIND, D>(c.v, c.vs, row, l, v);
    report_bad_entries(c, bt);
}

template <typename T, int KIND, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(KvCacheView c, KvBatchView bt, KvIO io) {
    constexpr int LPR = D / 8;
    const int64_t t = int64_t(blockIdx.x) * (kKvThreads / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR, h = blockIdx.y;
    report_bad_entries(c, bt);
    if (t >= bt.total) return;
    const int b = seq_of_row(bt, int(t));
    const int64_t at = (t * c.kv_heads + h) * D + l * 8;
    float k[8] = {}, v[8] = {};
    if (b < 0) {  // a row of no sequence
        if (io.zero_rest) {
            Vec8<T>::store(io.ok, at, k);
            Vec8<T>::store(io.ov, at, v);
        }
        return;
    }
    const int64_t pos = t - bt.start[b] + (io.first ? io.first[b] : 0);
    int64_t row = -1;
    if (pos >= 0 && pos < kv_capacity(bt, c)) row = kv_lookup(bt, c, b, int(pos), h);
    if (row >= 0) {
        load_row<KIND, D>(c.k, c.ks, row, l, k);
        load_row<KIND, D>(c.v, c.vs, row, l, v);
    } else if (l == 0) {
        flag_bad_page();
    }
    Vec8<T>::store(io.ok, at, k);
    Vec8<T>::store(io.ov, at, v);
}

using KvKernel = void (*)(KvCacheView, KvBatchView, KvIO);

template <typename T, int KIND> static KvKernel pick_dim(bool write, int D) {
    switch (D) {
    case 64: return write ? kv_write_kernel<T, KIND, 64> : kv_read_kernel<T, KIND, 64>;
    case 128: return write ? kv_write_kernel<T, KIND, 128> : kv_read_kernel<T, KIND, 128>;
    default: return write ? kv_write_kernel<T, KIND, 256> : kv_read_kernel<T, KIND, 256>;
    }
}

template <typename T> static KvKernel pick_kind(bool write, int kind, int D) {
    switch (kind) {
    case kKvF16: return pick_dim<T, kKvF16>(write, D);
    case kKvBF16: return pick_dim<T, kKvBF16>(write, D);
    case kKvQ8_0: return pick_dim<T, kKvQ8_0>(write, D);
    default: return pick_dim<T, kKvQ4_0>(write, D);
    }
}

// ---- argument checks shared with the attention ----------------------------------------------

static bool aligned(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int kv_check(const anvil_kv_cache *c, const anvil_kv_batch *b, KvCacheView *cv, KvBatchView *bv) {
    if (!c || !b) return fail(ANVIL_ERR_INVALID, "null cache or batch");
    const bool quant = c->kind == kKvQ8_0 || c->kind == kKvQ4_0;
    if (!quant && c->kind != kKvF16 && c->kind != kKvBF16)
        return fail(ANVIL_ERR_UNSUPPORTED, "cache kind %d (F16, BF16, Q8_0 and Q4_0 are)", c->kind);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(ANVIL_ERR_UNSUPPORTED, "head_dim=%d (64, 128 and 256 are)", c->head_dim);
    if (c->page_size < 1 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(ANVIL_ERR_INVALID, "page_size=%d is not a power of two up to 1024", c->page_size);
    if (c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 65535)
        return fail(ANVIL_ERR_INVALID, "num_pages=%d kv_heads=%d", c->num_pages, c->kv_heads);
    if (!c->k || !c->v || (quant && (!c->k_scale || !c->v_scale)))
        return fail(ANVIL_ERR_INVALID, "null cache tensor");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || (quant && (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))))
        return fail(ANVIL_ERR_ALIGN, "cache tensors must be 16-byte aligned");
    if (b->batch < 0 || b->total < 0 || b->max_pages < 0 || b->page_table_stride < b->max_pages)
        return fail(ANVIL_ERR_INVALID, "batch=%d total=%d max_pages=%d stride=%lld", b->batch, b->total,
                    b->max_pages, (long long)b->page_table_stride);
    if (b->batch && b->total && (!b->start || (b->max_pages && !b->page_table)))
        return fail(ANVIL_ERR_INVALID, "null page table or starts");
    if (!aligned(b->page_table, 4) || !aligned(b->start, 4) || !aligned(b->kv_len, 4))
        return fail(ANVIL_ERR_ALIGN, "page table, starts and lengths must be 4-byte aligned");
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    *cv = KvCacheView{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v),
                      static_cast<__half *>(c->k_scale), static_cast<__half *>(c->v_scale),
                      c->num_pages, c->kv_heads, shift};
    *bv = KvBatchView{b->page_table, b->page_table_stride, b->max_pages, b->start, b->kv_len,
                      b->batch, b->total};
    return ANVIL_OK;
}

static int run_kv(bool write, const anvil_kv_cache *c, const KvCacheView &cv, const KvBatchView &bv,
                  int dtype, const KvIO &io, cudaStream_t stream) {
    if (bv.total == 0 || bv.batch == 0) return ANVIL_OK;
    KvKernel fn;
    switch (dtype) {
    case kKvF32: fn = pick_kind<float>(write, c->kind, c->head_dim); break;
    case kKvF16: fn = pick_kind<__half>(write, c->kind, c->head_dim); break;
    case kKvBF16: fn = pick_kind<__nv_bfloat16>(write, c->kind, c->head_dim); break;
    default: return fail(ANVIL_ERR_UNSUPPORTED, "dtype %d (F32, F16 and BF16 are)", dtype);
    }
    const int rows = kKvThreads / (c->head_dim / 8);  // of one head, per CTA
    const dim3 grid(unsigned((int64_t(bv.total) + rows - 1) / rows), unsigned(cv.kv_heads));
    fn<<<grid, kKvThreads, 0, stream>>>(cv, bv, io);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, write ? "kv_write launch" : "kv_read launch");
}

int kv_take_status() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_anvil_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (cudaMemcpyToSymbol(g_anvil_device_status, &z, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace anvil

using namespace anvil;

extern "C" int anvil_kv_write(const anvil_kv_cache *cache, const anvil_kv_batch *batch, int dtype, const void *k,
                              int64_t k_row_stride, int64_t k_head_stride, const void *v,
                              int64_t v_row_stride, int64_t v_head_stride, anvil_stream_t stream) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    if (bv.batch && bv.total) {
        if (!k || !v || !bv.kv_len) return fail(ANVIL_ERR_INVALID, "null k, v or kv_len");
        const int n = dtype == kKvF32 ? 4 : 8;  // values in 16 bytes
        if (!aligned(k, 16) || !aligned(v, 16) || k_row_stride % n || k_head_stride % n || v_row_stride % n ||
            v_head_stride % n)
            return fail(ANVIL_ERR_ALIGN, "rows of k and v must start on 16-byte boundaries");
    }
    KvIO io{k, v, k_row_stride, k_head_stride, v_row_stride, v_head_stride, nullptr, nullptr, nullptr, 0};
    return run_kv(true, cache, cv, bv, dtype, io, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int anvil_kv_read(const anvil_kv_cache *cache, const anvil_kv_batch *batch, const int32_t *first,
                             int dtype, void *k, void *v, anvil_stream_t stream) {
    return anvil_kv_read_ex(cache, batch, first, dtype, k, v, 0, stream);
}

extern "C" int anvil_kv_read_ex(const anvil_kv_cache *cache, const anvil_kv_batch *batch, const int32_t *first,
                                int dtype, void *k, void *v, unsigned flags, anvil_stream_t stream) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    if (flags & ~unsigned(ANVIL_FLAG_ZERO_REST)) return fail(ANVIL_ERR_INVALID, "flags=0x%x", flags);
    bv.kv_len = nullptr;  // lengths are no part of a read
    if (bv.total && (bv.batch || flags)) {
        if (dtype != kKvF32 && dtype != kKvF16 && dtype != kKvBF16)
            return fail(ANVIL_ERR_UNSUPPORTED, "dtype %d (F32, F16 and BF16 are)", dtype);
        if (!k || !v) return fail(ANVIL_ERR_INVALID, "null k or v");
        if (!aligned(k, 16) || !aligned(v, 16) || !aligned(first, 4))
            return fail(ANVIL_ERR_ALIGN, "k and v must be 16-byte aligned, first 4-byte");
    }
    if (bv.batch == 0 && bv.total && flags) {  // all rows are of no sequence
        const size_t n = size_t(bv.total) * cv.kv_heads * cache->head_dim * (dtype == kKvF32 ? 4 : 2);
        cudaError_t e = cudaMemsetAsync(k, 0, n, reinterpret_cast<cudaStream_t>(stream));
        if (e == cudaSuccess) e = cudaMemsetAsync(v, 0, n, reinterpret_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "kv_read memset");
    }
    KvIO io{nullptr, nullptr, 0, 0, 0, 0, k, v, first, flags != 0};
    return run_kv(false, cache, cv, bv, dtype, io, reinterpret_cast<cudaStream_t>(stream));
}
