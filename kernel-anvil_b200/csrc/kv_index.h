// kv_index.h -- index arithmetic of the paged key/value cache, shared by its kernels and, as
// plain C++, by the CPU tests.  Every value that comes from device memory (sequence starts,
// lengths, page numbers) passes through here before it becomes an address: what is out of
// range is cut to the range or reported, never followed.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define ANVIL_HD __host__ __device__ __forceinline__
#else
#define ANVIL_HD inline
#endif

namespace anvil {

// One sequence of a ragged batch: its rows are [q0, q1) of the packed rows, and `kv` tokens of
// it are in the cache.  bad: something had to be cut to its range.
struct KvSeq {
    int q0, q1, kv;
    bool bad;
};

// start0 / start1: two neighbouring entries of the starts; total: packed rows; capacity: tokens
// that the sequence's row of the page table can name.
ANVIL_HD KvSeq kv_seq(int start0, int start1, int kv_len, int total, int64_t capacity) {
    KvSeq s;
    s.q0 = start0 < 0 ? 0 : start0 > total ? total : start0;
    s.q1 = start1 < s.q0 ? s.q0 : start1 > total ? total : start1;
    s.kv = kv_len < 0 ? 0 : int64_t(kv_len) > capacity ? int(capacity) : kv_len;
    s.bad = s.q0 != start0 || s.q1 != start1 || s.kv != kv_len;
    return s;
}

// Row of a cache tensor (num_pages, kv_heads, page_size, ...) that holds the token at offset
// `off` of page `page` for head `head`; -1 where there is no such page.  64 bits: a long cache
// has more than 2^31 values, and may have more than 2^31 rows.
ANVIL_HD int64_t kv_row(int page, int num_pages, int head, int kv_heads, int off, int page_shift) {
    if (page < 0 || page >= num_pages) return -1;
    return (((int64_t(page) * kv_heads + head) << page_shift) + off);
}

// Cached tokens that the row `i` (of n) of a sequence with `kv` cached tokens sees.  Causal: row
// i stands at position kv - n + i and sees itself and what is before it; 0 (a row with nothing to
// see) where the sequence has fewer cached tokens than rows after it.
ANVIL_HD int kv_seen(int i, int n, int kv, bool causal) {
    if (!causal) return kv;
    const int seen = kv - n + i + 1;
    return seen < 0 ? 0 : seen > kv ? kv : seen;
}

}  // namespace anvil
