// Bounded waits of the paged attention kernels and of the sampler that run out:
// the kernels are compiled here with copies that can be left out, so that what
// waits for them gives up after its limit. Rows whose work met that are NaN (a
// sampled row: token -1, logprob NaN), all others keep their results to the bit,
// and the next call is right again. No other access changes.
#define kWaitLimitNs kLibraryWaitLimitNs
#include "q4k_device.cuh"
#undef kWaitLimitNs
namespace q4k {
constexpr uint64_t kWaitLimitNs = 20000000ull;  // of the attention kernels' waits; others keep the library's 2 s
}
#include "paged_tc.cuh"

namespace q4k {
__device__ int lost_page = -1;                // of KV head 0
__device__ unsigned long long lost_source = 0;  // address, of a bulk copy
namespace paged_dev {
__device__ __forceinline__ void tma_load_4d_or_not(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                                   uint64_t* bar) {
    if (w == lost_page && z == 0) return;
    tma_load_4d(dst, map, x, y, z, w, bar);
}
}  // namespace paged_dev
__device__ __forceinline__ void bulk_g2s_or_not(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    if (reinterpret_cast<unsigned long long>(src) != lost_source) bulk_g2s(dst, src, bytes, bar);
}
}  // namespace q4k
#define tma_load_4d tma_load_4d_or_not
#include "paged_attention.cu"
#undef tma_load_4d
#define bulk_g2s bulk_g2s_or_not
#include "sample.cu"
#undef bulk_g2s

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

namespace q4k {
int sm_count() {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, 0);
    return n;
}
void* tensor_map_encoder() {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r);
    return p;
}
}  // namespace q4k

static void must(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return;
    std::printf("%s: %s\n", what, cudaGetErrorString(e));
    std::exit(1);
}

template <typename T>
static T* device(const std::vector<T>& v) {
    T* p = nullptr;
    must(cudaMalloc(&p, v.size() * sizeof(T)), "malloc");
    must(cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice), "copy");
    return p;
}
template <typename T>
static std::vector<T> host(const T* p, size_t n) {
    std::vector<T> v(n);
    must(cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost), "read");
    return v;
}

static uint16_t half_of(float x, bool bf16) {
    if (bf16) {
        uint32_t b;
        std::memcpy(&b, &x, 4);
        return (uint16_t)(b >> 16);
    }
    const __half h = __float2half(x);
    uint16_t r;
    std::memcpy(&r, &h, 2);
    return r;
}
static bool is_nan(uint32_t bits, int size, bool bf16) {
    if (size == 4) return (bits & 0x7fffffffu) > 0x7f800000u;
    return bf16 ? (bits & 0x7fffu) > 0x7f80u : (bits & 0x7fffu) > 0x7c00u;
}

// sequences of `ctx` cached and `fresh` new tokens each; the first page of the first one is lost
static int attention(const char* name, bool f32, bool bf16, int d, int sequences, int fresh, int ctx, int heads, int kv) {
    const int page = 16, width = (ctx + page - 1) / page, pages = sequences * width, tokens = sequences * fresh;
    const int size = f32 ? 4 : 2;
    std::mt19937 rng(7);
    std::normal_distribution<float> normal;
    std::vector<uint16_t> cache((size_t)pages * kv * page * d);
    for (auto& x : cache) x = half_of(normal(rng), bf16);
    std::vector<uint8_t> queries((size_t)tokens * heads * d * size);
    for (size_t i = 0; i < queries.size() / size; ++i) {
        const float x = normal(rng);
        const uint16_t h = half_of(x, bf16);
        std::memcpy(&queries[i * size], f32 ? (const void*)&x : (const void*)&h, size);
    }
    std::vector<int> q_start(sequences + 1), kv_len(sequences, ctx), table(pages);
    for (int i = 0; i <= sequences; ++i) q_start[i] = i * fresh;
    for (int i = 0; i < pages; ++i) table[i] = i;

    q4k::PagedAttentionArgs a;
    a.cache.k = device(cache);
    std::rotate(cache.begin(), cache.begin() + 12345 % cache.size(), cache.end());
    a.cache.v = device(cache);
    a.cache.bf16 = bf16;
    a.cache.kv_heads = kv, a.cache.head_dim = d, a.cache.page_size = page, a.cache.page_shift = 4, a.cache.pages = pages;
    a.cache.row_stride = d, a.cache.head_stride = page * d, a.cache.page_stride = (long long)kv * page * d;
    a.batch.sequences = sequences, a.batch.table_stride = a.batch.table_width = width;
    a.batch.q_start = device(q_start), a.batch.kv_len = device(kv_len), a.batch.page_table = device(table);
    a.batch.max_new = fresh, a.batch.tokens = tokens;
    a.f32 = f32;
    a.q = device(queries);
    uint8_t* out = nullptr;
    must(cudaMalloc(&out, queries.size()), "malloc");
    must(cudaMalloc(&a.lse, (size_t)tokens * heads * 4), "malloc");
    must(cudaMalloc(&a.workspace, q4k::paged_attention_workspace_bytes(heads, kv, d, 0)), "malloc");
    a.out = out;
    a.ld_q = a.ld_out = heads * d;
    a.heads = heads, a.scale = 0.08f;

    auto run = [&](int lost) {
        must(cudaMemcpyToSymbol(q4k::lost_page, &lost, sizeof lost), "symbol");
        must(cudaMemset(out, 0, queries.size()), "clear");
        must(cudaMemset(a.lse, 0, (size_t)tokens * heads * 4), "clear");
        must(q4k::paged_attention(a, nullptr), "launch");
        must(cudaDeviceSynchronize(), "run");
    };
    run(-1);
    const auto good = host(out, queries.size());
    const auto good_lse = host(a.lse, (size_t)tokens * heads);
    run(0);
    const auto bad = host(out, queries.size());
    const auto bad_lse = host(a.lse, (size_t)tokens * heads);
    run(-1);
    int wrong = host(out, queries.size()) != good || host(a.lse, (size_t)tokens * heads) != good_lse;
    int nans = 0, same = 0;
    for (int t = 0; t < tokens; ++t)
        for (int h = 0; h < heads; ++h) {
            const size_t row = (size_t)t * heads + h;
            const uint8_t *x = &bad[row * d * size], *y = &good[row * d * size];
            uint32_t lse;
            std::memcpy(&lse, &bad_lse[row], 4);
            bool all = is_nan(lse, 4, false);
            for (int i = 0; i < d; ++i) {
                uint32_t v = 0;
                std::memcpy(&v, x + i * size, size);
                all &= is_nan(v, size, bf16);
            }
            const bool equal = !std::memcmp(x, y, (size_t)d * size) && !std::memcmp(&bad_lse[row], &good_lse[row], 4);
            nans += all, same += equal;
            wrong += !all && !equal;                                // nothing in between
            wrong += t < fresh && h < heads / kv && !all;           // these need the page
            wrong += is_nan(*(const uint32_t*)&good_lse[row], 4, false);
        }
    std::printf("%s: %d rows NaN, %d as before, %d wrong\n", name, nans, same, wrong);
    return wrong + (same == 0);
}

static int sampling() {
    const int rows = 3, vocab = 40000;
    std::mt19937 rng(9);
    std::normal_distribution<float> normal;
    std::vector<float> logits((size_t)rows * vocab), uniform(rows, 0.4f);
    for (auto& x : logits) x = normal(rng);
    q4k::SampleArgs a;
    const float* l = device(logits);
    a.logits = l, a.type = Q4K_TYPE_F32, a.ld = vocab, a.rows = rows, a.vocab = vocab;
    a.uniform = device(uniform);
    a.tokens = device(std::vector<int>(rows));
    a.logprob = device(std::vector<float>(rows));
    std::vector<int> tokens[3];
    std::vector<float> logprob[3];
    for (int i = 0; i < 3; ++i) {
        const unsigned long long lost = i == 1 ? reinterpret_cast<unsigned long long>(l + vocab) : 0;  // the first stretch of row 1
        must(cudaMemcpyToSymbol(q4k::lost_source, &lost, sizeof lost), "symbol");
        must(q4k::sample(a, nullptr), "launch");
        must(cudaDeviceSynchronize(), "run");
        tokens[i] = host(a.tokens, rows), logprob[i] = host(a.logprob, rows);
    }
    int wrong = tokens[0] != tokens[2] || logprob[0] != logprob[2];
    for (int r = 0; r < rows; ++r)
        wrong += r == 1 ? tokens[1][r] != -1 || logprob[1][r] == logprob[1][r]
                        : tokens[1][r] != tokens[0][r] || logprob[1][r] != logprob[0][r];
    std::printf("sampling: tokens %d %d %d, %d wrong\n", tokens[1][0], tokens[1][1], tokens[1][2], wrong);
    return wrong;
}

int main() {
    int wrong = 0;
    // tiles shared by many CTAs, then tiles of one CTA, of both kernels
    wrong += attention("decode, long", true, false, 128, 2, 1, 6000, 8, 2);
    wrong += attention("decode, many", true, false, 64, 120, 1, 200, 8, 2);
    wrong += attention("decode, 16 rows", false, true, 128, 3, 4, 3000, 8, 2);
    wrong += attention("chunk, fp32", true, false, 128, 2, 200, 3000, 8, 2);
    wrong += attention("chunk, bf16", false, true, 128, 40, 70, 300, 16, 4);
    wrong += attention("chunk, fp16", false, false, 64, 3, 90, 700, 10, 2);
    wrong += sampling();
    std::printf("%d wrong in all\n", wrong);
    return wrong != 0;
}
