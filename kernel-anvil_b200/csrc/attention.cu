// attention.cu -- attention of new tokens over the paged key/value cache.
//
// For row i of sequence b (q_len new tokens, kv cached ones), query head h and its key/value
// head h / (heads / kv_heads):
//   s_j = scale q . k_j,  j < seen(i)  (kv, or min(kv, kv - q_len + i + 1) when causal)
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j;  o = 0 where nothing is seen.
// Keys are visited once with a running maximum and sum (fp32).
#include <cuda_runtime.h>

#include "anvil.h"
#include "anvil_host.h"
#include "kv_cache.cuh"

namespace anvil {

int kv_check(const anvil_kv_cache *c, const anvil_kv_batch *b, KvCacheView *cv, KvBatchView *bv);

struct AttnIO {
    const void *q;
    int64_t q_row, q_head;  // in values
    void *out;              // (total, heads, D)
    int heads;
    float scale;
    int causal;
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

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

// One CTA per (packed row, query head): four warps share the keys, a lane owns D / 32 dimensions.
template <typename T, int KIND, int D>
__global__ void __launch_bounds__(128) attn_simple_kernel(KvCacheView c, KvBatchView bt, AttnIO io) {
    constexpr int E = D / 32;
    __shared__ float sm[4], sl[4], so[4][D];
    const int t = blockIdx.x, h = blockIdx.y, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b = -1;
    for (int i = 0; i < bt.batch; ++i) {
        const KvSeq x = load_seq(bt, c, i);
        if (x.bad && threadIdx.x == 0) flag_bad_page();
        if (x.q0 <= t && t < x.q1) b = i;
    }
    if (b < 0) return;
    const KvSeq s = load_seq(bt, c, b);
    const int kvh = h / (io.heads / c.kv_heads);
    const int seen = kv_seen(t - s.q0, s.q1 - s.q0, s.kv, io.causal);
    const T *q = static_cast<const T *>(io.q) + t * io.q_row + h * io.q_head;
    float qv[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = to_f(q[lane + 32 * e]) * io.scale;
        o[e] = 0.0f;
    }
    for (int j = w; j < seen; j += 4) {
        const int64_t row = kv_lookup(bt, c, b, j, kvh);
        if (row < 0) {
            if (lane == 0) flag_bad_page();
            continue;
        }
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) dot += qv[e] * kv_value<KIND, D>(c.k, c.ks, row, lane + 32 * e);
        dot = warp_sum(dot);
        const float mn = fmaxf(m, dot);
        const float base = mn == -INFINITY ? 0.0f : mn;  // a NaN score stays one: fmaxf passes it by
        const float a = expf(m - base), p = expf(dot - base);
        l = l * a + p;
#pragma unroll
        for (int e = 0; e < E; ++e)
            o[e] = o[e] * a + p * kv_value<KIND, D>(c.v, c.vs, row, lane + 32 * e);
        m = mn;
    }
    if (lane == 0) {
        sm[w] = m;
        sl[w] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) so[w][lane + 32 * e] = o[e];
    __syncthreads();
    const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    for (int e = threadIdx.x; e < D; e += 128) {
        float num = 0.0f, den = 0.0f;
        for (int i = 0; i < 4; ++i) {
            const float a = mx == -INFINITY ? 0.0f : expf(sm[i] - mx);
            num += a * so[i][e];
            den += a * sl[i];
        }
        static_cast<T *>(io.out)[(int64_t(t) * io.heads + h) * D + e] = from_f<T>(den == 0.0f ? 0.0f : num / den);
    }
}

using AttnKernel = void (*)(KvCacheView, KvBatchView, AttnIO);

template <typename T, int KIND> static AttnKernel simple_dim(int D) {
    return D == 64 ? attn_simple_kernel<T, KIND, 64> : D == 128 ? attn_simple_kernel<T, KIND, 128>
                                                               : attn_simple_kernel<T, KIND, 256>;
}

int attn_take_status() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_anvil_device_status, sizeof(int)) != cudaSuccess) return -1;
    if (cudaMemcpyToSymbol(g_anvil_device_status, &z, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace anvil

using namespace anvil;

extern "C" int64_t anvil_paged_attention_workspace(const anvil_kv_cache *cache, const anvil_kv_batch *batch,
                                                   int heads) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    return 0;
}

extern "C" int anvil_paged_attention(const anvil_kv_cache *cache, const anvil_kv_batch *batch, int dtype,
                                     const void *q, int64_t q_row_stride, int64_t q_head_stride, int heads,
                                     float scale, int causal, void *out, void *workspace,
                                     int64_t workspace_bytes, anvil_stream_t stream) {
    KvCacheView cv;
    KvBatchView bv;
    if (int s = kv_check(cache, batch, &cv, &bv)) return s;
    if (dtype != kKvF16 && dtype != kKvBF16)
        return fail(ANVIL_ERR_UNSUPPORTED, "q is F16 or BF16, not type %d", dtype);
    if ((cache->kind == kKvF16 || cache->kind == kKvBF16) && cache->kind != dtype)
        return fail(ANVIL_ERR_UNSUPPORTED, "an unquantised cache takes q of its own type");
    if (heads < 1 || heads % cv.kv_heads)
        return fail(ANVIL_ERR_INVALID, "heads=%d is not a multiple of kv_heads=%d", heads, cv.kv_heads);
    if (bv.batch == 0 || bv.total == 0) return ANVIL_OK;
    if (!q || !out || !bv.kv_len) return fail(ANVIL_ERR_INVALID, "null q, out or kv_len");
    const auto mis = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
    if (mis(q) || mis(out) || mis(workspace) || q_row_stride % 8 || q_head_stride % 8)
        return fail(ANVIL_ERR_ALIGN, "q, its rows, out and the workspace must be 16-byte aligned");
    AttnIO io{q, q_row_stride, q_head_stride, out, heads, scale, causal};
    const int D = cache->head_dim;
    AttnKernel fn = nullptr;
    switch (cache->kind) {
    case kKvF16: fn = simple_dim<__half, kKvF16>(D); break;
    case kKvBF16: fn = simple_dim<__nv_bfloat16, kKvBF16>(D); break;
    case kKvQ8_0: fn = dtype == kKvF16 ? simple_dim<__half, kKvQ8_0>(D) : simple_dim<__nv_bfloat16, kKvQ8_0>(D); break;
    default: fn = dtype == kKvF16 ? simple_dim<__half, kKvQ4_0>(D) : simple_dim<__nv_bfloat16, kKvQ4_0>(D); break;
    }
    fn<<<dim3(bv.total, heads), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(cv, bv, io);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ANVIL_OK : cuda_fail(e, "paged_attention launch");
}
