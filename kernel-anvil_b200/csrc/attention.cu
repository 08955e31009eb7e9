// attention.cu -- attention of new tokens over the paged key/value cache.
//
// For row i of sequence b (q_len new tokens, kv cached ones), query head h and its key/value
// head h / (heads / kv_heads):
//   s_j = scale q . k_j,  j < seen(i)  (kv, or min(kv, kv - q_len + i + 1) when causal)
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j;  o = 0 where nothing is seen.
// Keys are visited once with a running maximum and sum (fp32).
#include <algorithm>
#include <cmath>

#include "anvil.h"
#include "anvil_host.h"
#include "attention.cuh"

namespace anvil {

int kv_check(const anvil_kv_cache *c, const anvil_kv_batch *b, KvCacheView *cv, KvBatchView *bv);

AttnTiles attn_rows_tiles(int kind, int D, int nt);
int attn_rows_launch(int kind, int D, int nt, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas,
                     bool join, cudaStream_t s);
int attn_rows_take_status();
AttnTiles attn_tile_tiles(int D);
int attn_tile_launch(int kind, int D, const KvCacheView &c, const KvBatchView &bt, const AttnIO &io, int ctas, bool join,
                     cudaStream_t s);
int attn_tile_take_status();

int attn_take_status() {
    const int a = attn_rows_take_status(), b = attn_tile_take_status();
    return a < 0 ? a : b < 0 ? b : a | b;
}

// The grid: every resident slot, or fewer where the batch cannot have that many key tiles.  It
// follows from the batch's outer sizes, not from lengths, which are on the device.
// (A constant, so that the workspace can be asked for without a device and the order of the sums is the same on every one; on
// a part with fewer multiprocessors the CTAs take turns.)
constexpr int kAttnSms = 148;
struct AttnPlan {
    int nt;         // row tile of the rows kernel in eighths; 0: the tile kernel
    int ctas;
    bool join;      // some unit may span CTAs
    int64_t bytes;  // of partial results
};

static AttnPlan attn_plan(const anvil_kv_cache *c, const KvCacheView &cv, const KvBatchView &bv, int heads) {
    const int group = heads / cv.kv_heads;
    AttnPlan p;
    const int64_t rows = int64_t(bv.total) * group;
    // Few rows a sequence go to the rows kernel, in tiles of 8 or 16; the tile kernel, whose tiles have 128 rows,
    // takes the others.  Where they cross, 16 sequences of 6000 keys in 8 heads of 128, us by rows a sequence and head:
    //                 8: 8 / 16 / tile     16: 8 / 16 / tile     32: 16 / tile     48: 16 / tile
    //   F16              83 /  84 /  95      141 /  87 /  94       149 /  97         216 /  98
    //   Q8_0             52 /  60 / 113       86 /  63 / 113       106 / 115         152 / 117
    //   Q4_0             52 /  63 / 152       87 /  66 / 152       111 / 154         159 / 156
    // (a second tile of rows reads a 16-bit cache, which is what bounds it, once more, and widens quantised codes once
    // more, which the tile kernel does more slowly: through shared memory).  head_dim 256 and 4000 keys, 32 rows: Q8_0 133 /
    // 253, Q4_0 170 / 144.  Averages over the batch: the lengths are on the device.
    const int64_t few = int64_t(bv.batch) * (c->kind == kKvQ8_0 || (c->kind == kKvQ4_0 && c->head_dim < 256) ? 32 : 16);
    p.nt = rows <= int64_t(bv.batch) * 8 ? 1 : rows <= few ? 2 : 0;
    const AttnTiles t = p.nt ? attn_rows_tiles(c->kind, c->head_dim, p.nt) : attn_tile_tiles(c->head_dim);
    const int64_t capacity = kv_capacity(bv, cv);
    const int64_t units = int64_t(cv.kv_heads) * (int64_t(bv.total) * group / t.rows + std::min(bv.batch, bv.total));
    const int64_t per = std::max<int64_t>(1, (capacity + t.keys - 1) / t.keys);
    const int64_t slots = int64_t(kAttnSms) * t.occ;
    p.ctas = int(per > slots / std::max<int64_t>(units, 1) ? slots : std::min(slots, units * per));
    p.join = per > 1;
    p.bytes = p.join ? (int64_t(t.rows) * (c->head_dim + 2) * 8 + int64_t(sizeof(AttnOpen))) * p.ctas : 0;
    return p;
}

}  // namespace anvil

using namespace anvil;

extern "C" int64_t anvil_paged_attention_workspace(const anvil_kv_cache *cache, const anvil_kv_batch *batch,
                                                   int heads) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    if (heads < 1 || heads % cv.kv_heads)
        return fail(ANVIL_ERR_INVALID, "heads=%d is not a multiple of kv_heads=%d", heads, cv.kv_heads);
    if (bv.batch == 0 || bv.total == 0) return 0;
    return attn_plan(cache, cv, bv, heads).bytes;
}

extern "C" int anvil_paged_attention(const anvil_kv_cache *cache, const anvil_kv_batch *batch, int dtype,
                                     const void *q, int64_t q_row_stride, int64_t q_head_stride, int heads,
                                     float scale, int causal, void *out, void *workspace,
                                     int64_t workspace_bytes, anvil_stream_t stream) {
    return anvil_paged_attention_ex(cache, batch, dtype, q, q_row_stride, q_head_stride, heads, scale, causal, out,
                                    workspace, workspace_bytes, 0, stream);
}

extern "C" int anvil_paged_attention_ex(const anvil_kv_cache *cache, const anvil_kv_batch *batch, int dtype,
                                        const void *q, int64_t q_row_stride, int64_t q_head_stride, int heads,
                                        float scale, int causal, void *out, void *workspace,
                                        int64_t workspace_bytes, unsigned flags, anvil_stream_t stream) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    if (dtype != kKvF16 && dtype != kKvBF16)
        return fail(ANVIL_ERR_UNSUPPORTED, "q is F16 or BF16, not type %d", dtype);
    if ((cache->kind == kKvF16 || cache->kind == kKvBF16) && cache->kind != dtype)
        return fail(ANVIL_ERR_UNSUPPORTED, "an unquantised cache takes q of its own type");
    if (heads < 1 || heads % cv.kv_heads)
        return fail(ANVIL_ERR_INVALID, "heads=%d is not a multiple of kv_heads=%d", heads, cv.kv_heads);
    if (int64_t(bv.total) * heads > 0x7fffffff - 1024)
        return fail(ANVIL_ERR_UNSUPPORTED, "%d rows of %d heads are too many for one call", bv.total, heads);
    if (flags & ~unsigned(ANVIL_FLAG_ZERO_REST)) return fail(ANVIL_ERR_INVALID, "flags=0x%x", flags);
    if (bv.total == 0 || (bv.batch == 0 && !flags)) return ANVIL_OK;
    if (bv.batch == 0) {  // all rows are of no sequence
        if (!out) return fail(ANVIL_ERR_INVALID, "null out");
        const cudaError_t e = cudaMemsetAsync(out, 0, size_t(bv.total) * heads * cache->head_dim * 2,
                                              reinterpret_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "paged_attention memset");
    }
    if (!q || !out || !bv.kv_len) return fail(ANVIL_ERR_INVALID, "null q, out or kv_len");
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return fail(ANVIL_ERR_INVALID, "scale=%g is not finite in powers of two", double(scale));
    const auto mis = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
    if (mis(q) || mis(out) || q_row_stride % 8 || q_head_stride % 8)
        return fail(ANVIL_ERR_ALIGN, "q, its rows and out must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(workspace) % 32) return fail(ANVIL_ERR_ALIGN, "the workspace must be 32-byte aligned");
    const AttnPlan p = attn_plan(cache, cv, bv, heads);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes))
        return fail(ANVIL_ERR_INVALID, "a workspace of %lld bytes is needed, got %lld", (long long)p.bytes,
                    (long long)(workspace ? workspace_bytes : 0));
    // (the kernels write notes wherever there is a place for parts, so a call without joins has none, whatever the
    // caller's pointer)
    AttnIO io{q, q_row_stride, q_head_stride, out, heads, 0, 0, 0, scale_log2,
              causal != 0, dtype == kKvBF16, (flags & ANVIL_FLAG_ZERO_REST) != 0, p.join ? static_cast<float *>(workspace) : nullptr};
    set_group(io, heads / cv.kv_heads);
    if (!p.nt)
        return attn_tile_launch(cache->kind, cache->head_dim, cv, bv, io, p.ctas, p.join,
                                reinterpret_cast<cudaStream_t>(stream));
    return attn_rows_launch(cache->kind, cache->head_dim, p.nt, cv, bv, io, p.ctas, p.join,
                            reinterpret_cast<cudaStream_t>(stream));
}
