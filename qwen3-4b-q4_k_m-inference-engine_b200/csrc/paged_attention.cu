// q4k_paged_attention: causal grouped-query attention of a batch's new tokens
// over the pages of their sequences. Per query row,
//   s_k = scale q . k,  o = sum_k e^(s_k - m) v_k / l,  l = sum_k e^(s_k - m),
//   lse = m + log l,    m = max_k s_k,
// over the keys k <= p (the row's position) of its sequence's cached tokens,
// with a window of w also k > p - w. A row with no key gets o = 0, lse = -inf.
#include <math_constants.h>

#include "paged.h"
#include "paged_device.cuh"

namespace q4k {
namespace {

using namespace paged_dev;

// One CTA per (row, query head): four warps take every fourth key with an
// online softmax of their own and are joined at the end.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const __grid_constant__ PagedAttentionArgs a) {
    constexpr int V = D / 32;
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int s = 0;
    for (int i = 0; i < a.batch.sequences; i += 128)
        s += __syncthreads_count(i + tid < a.batch.sequences && __ldg(a.batch.q_start + i + tid + 1) <= t);
    if (s >= a.batch.sequences) return;
    const int len = __ldg(a.batch.kv_len + s);
    const int position = len - __ldg(a.batch.q_start + s + 1) + t;
    const long long held = (long long)a.batch.table_width << a.cache.page_shift;
    const int end = (int)min((long long)position + 1, held);
    const int begin = a.window > 0 ? max(position - a.window + 1, 0) : 0;
    const int kvh = h / (a.heads / a.cache.kv_heads);
    const T* q = static_cast<const T*>(a.q) + t * a.ld_q + (size_t)h * D + lane * V;
    float x[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = to_float<T>(q[i]) * a.scale;
        o[i] = 0.0f;
    }
    float m = -CUDART_INF_F, l = 0.0f;
    for (int p = begin + warp; p < end; p += 4) {
        const int page = __ldg(a.batch.page_table + (size_t)s * a.batch.table_stride + (p >> a.cache.page_shift));
        if (page < 0 || page >= a.cache.pages) continue;
        const long long at = page * a.cache.page_stride + kvh * a.cache.head_stride +
                             (p & (a.cache.page_size - 1)) * a.cache.row_stride + lane * V;
        const C* k = reinterpret_cast<const C*>(a.cache.k) + at;
        const C* v = reinterpret_cast<const C*>(a.cache.v) + at;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) dot += x[i] * to_float<C>(k[i]);
        dot = warp_sum(dot);
        const float mn = fmaxf(m, dot);
        const float r = expf(m - mn), e = expf(dot - mn);
        l = l * r + e;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = o[i] * r + e * to_float<C>(v[i]);
        m = mn;
    }
    __shared__ float wm[4], wl[4], wo[4][D];
    if (lane == 0) {
        wm[warp] = m;
        wl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) wo[warp][lane * V + i] = o[i];
    __syncthreads();
    if (tid >= D) return;
    float top = wm[0], total = 0.0f, sum = 0.0f;
    for (int w = 1; w < 4; ++w) top = fmaxf(top, wm[w]);
    for (int w = 0; w < 4; ++w) {
        if (!(wl[w] > 0.0f)) continue;
        const float f = expf(wm[w] - top);
        total += f * wl[w];
        sum += f * wo[w][tid];
    }
    static_cast<T*>(a.out)[t * a.ld_out + (size_t)h * D + tid] = from_float<T>(total > 0.0f ? sum / total : 0.0f);
    if (tid == 0 && a.lse) a.lse[(size_t)t * a.heads + h] = total > 0.0f ? top + logf(total) : -CUDART_INF_F;
}

template <typename T, typename C>
void launch(const PagedAttentionArgs& a, cudaStream_t s) {
    const dim3 grid(a.batch.tokens, a.heads);
    if (a.cache.head_dim == 128)
        paged_attention_kernel<T, C, 128><<<grid, 128, 0, s>>>(a);
    else
        paged_attention_kernel<T, C, 64><<<grid, 128, 0, s>>>(a);
}

}  // namespace

size_t paged_attention_workspace_bytes(int, int, int, int) { return 0; }

cudaError_t paged_attention(const PagedAttentionArgs& a, cudaStream_t s) {
    if (a.f32)
        launch<float, __half>(a, s);
    else if (a.cache.bf16)
        launch<__nv_bfloat16, __nv_bfloat16>(a, s);
    else
        launch<__half, __half>(a, s);
    return cudaGetLastError();
}

}  // namespace q4k
