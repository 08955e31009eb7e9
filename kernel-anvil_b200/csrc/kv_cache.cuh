// kv_cache.cuh -- views of the paged key/value cache and of a ragged batch, as the kernels
// that write it (kv_cache.cu) and read it (kv_cache.cu, attention*.cu) take them.
//
// A cache tensor (keys or values) is (num_pages, kv_heads, page_size, row), row-major, so the
// tokens of one head that share a page are one run of memory.  A row holds head_dim values:
//   F16 / BF16  head_dim 16-bit values
//   Q8_0        head_dim int8 codes; scales in a tensor of their own (fp16, one per 32 values)
//   Q4_0        head_dim / 2 bytes: 16 bytes per 32 values, value e < 16 in the low nibble of
//               byte e, value e >= 16 in the high nibble of byte e - 16; scales as Q8_0
// These are the blocks of the GGUF types with the scale kept apart, so that the codes of a row
// start on a 16-byte boundary and move in 16-byte pieces.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "anvil_common.cuh"
#include "kv_index.h"

namespace anvil {

constexpr int kKvF32 = 0;    // ggml type ids
constexpr int kKvF16 = 1;
constexpr int kKvQ4_0 = 2;
constexpr int kKvQ8_0 = 8;
constexpr int kKvBF16 = 30;

// Device status flag: a page number, length or start was out of range (cut or skipped).
constexpr int kStatusBadPage = 2;

// Bytes of one row's codes.
template <int KIND, int D> struct KvRow {
    static constexpr int bytes = KIND == kKvQ8_0 ? D : KIND == kKvQ4_0 ? D / 2 : 2 * D;
    static constexpr int scales = (KIND == kKvQ8_0 || KIND == kKvQ4_0) ? D / 32 : 0;
};

struct KvCacheView {
    uint8_t *k, *v;
    __half *ks, *vs;  // null for F16 / BF16
    int num_pages, kv_heads, page_shift;
};

struct KvBatchView {
    const int *table;  // (batch, max_pages)
    int64_t table_stride;
    int max_pages;
    const int *start;   // batch + 1
    const int *kv_len;  // batch
    int batch, total;
};

// Tokens of a sequence at most: positions of the tiles behind the last one are still ints.
constexpr int64_t kKvMaxTokens = 0x7ffff000;

// Tokens that a sequence's row of the page table can name.
__host__ __device__ __forceinline__ int64_t kv_capacity(const KvBatchView &bt, const KvCacheView &c) {
    const int64_t n = int64_t(bt.max_pages) << c.page_shift;
    return n > kKvMaxTokens ? kKvMaxTokens : n;
}

__device__ __forceinline__ KvSeq load_seq(const KvBatchView &bt, const KvCacheView &c, int b) {
    return kv_seq(bt.start[b], bt.start[b + 1], bt.kv_len ? bt.kv_len[b] : 0, bt.total,
                  kv_capacity(bt, c));
}

// Cache row of position `pos` of sequence b for `head`, or -1; pos is within the capacity.
__device__ __forceinline__ int64_t kv_lookup(const KvBatchView &bt, const KvCacheView &c, int b,
                                             int pos, int head) {
    const int page = bt.table[b * bt.table_stride + (pos >> c.page_shift)];
    return kv_row(page, c.num_pages, head, c.kv_heads, pos & ((1 << c.page_shift) - 1),
                  c.page_shift);
}

__device__ __forceinline__ void flag_bad_page() {
    atomicOr(&g_anvil_device_status, kStatusBadPage);
}

}  // namespace anvil
