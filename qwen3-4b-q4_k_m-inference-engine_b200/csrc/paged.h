// A paged KV cache and the batch of sequences that lives in it: the host-side
// arguments of the append (paged_append.cu) and attention (paged_attention.cu)
// kernels behind q4k_paged_append and q4k_paged_attention.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace q4k {

// A kernel's shared-memory limit (and, for clusters of 16, leave to use them) on
// the current device, set at its first launch there: attributes are a device's.
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<unsigned long long>& done, bool big_clusters = false) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (e != cudaSuccess || (done.load() & bit)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && big_clusters)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

// Element (page, head, row, dim) of K or V is at page * page_stride + head *
// head_stride + row * row_stride + dim, in 2-byte elements.
struct PagedCache {
    uint16_t* k = nullptr;
    uint16_t* v = nullptr;
    bool bf16 = false;  // else fp16
    int kv_heads = 0, head_dim = 0, page_size = 0;
    int page_shift = 0;  // page_size = 1 << page_shift
    long long pages = 0;
    long long page_stride = 0, head_stride = 0, row_stride = 0;
};

struct PagedBatch {
    int sequences = 0;
    const int* q_start = nullptr;     // [sequences + 1]
    const int* kv_len = nullptr;      // [sequences]
    const int* page_table = nullptr;  // [sequences][table_stride], table_width of them used
    long long table_stride = 0;
    int table_width = 0;
    int max_new = 0;
    int tokens = 0;  // rows of q, k, v and the outputs
};

struct PagedAppendArgs {
    PagedCache cache;
    PagedBatch batch;
    bool f32 = false;  // activations are fp32 (else of the cache's type)
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    void* q_out = nullptr;
    long long ld_q = 0, ld_k = 0, ld_v = 0, ld_q_out = 0;  // elements between token rows
    int heads = 0;
    const float* q_gamma = nullptr;
    const float* k_gamma = nullptr;
    float eps = 1e-6f;
    double rope_base = 1e6;
};
cudaError_t paged_append(const PagedAppendArgs& a, cudaStream_t s);

struct PagedAttentionArgs {
    PagedCache cache;
    PagedBatch batch;
    bool f32 = false;
    const void* q = nullptr;
    void* out = nullptr;
    float* lse = nullptr;  // optional, [tokens][heads]
    long long ld_q = 0, ld_out = 0;
    int heads = 0;
    float scale = 0.0f;
    int window = 0;  // 0: none
    void* workspace = nullptr;
};
size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int max_new);
cudaError_t paged_attention(const PagedAttentionArgs& a, cudaStream_t s);

// Sampling (sample.cu).
struct SampleArgs {
    const void* logits = nullptr;
    int type = 0;  // Q4K_TYPE_F32, _F16 or _BF16
    long long ld = 0;
    int rows = 0, vocab = 0;
    const float* temperature = nullptr;
    const int* top_k = nullptr;
    const float* top_p = nullptr;
    const float* min_p = nullptr;
    const float* uniform = nullptr;
    int* tokens = nullptr;
    float* logprob = nullptr;
};
cudaError_t sample(const SampleArgs& a, cudaStream_t s);

}  // namespace q4k
