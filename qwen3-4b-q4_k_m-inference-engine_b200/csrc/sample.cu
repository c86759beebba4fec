// q4k_sample: one token per row of logits. With x_i = (l_i - max l) / T and
// w_i = e^(x_i), the tokens are ordered by logit (ties: the lowest index
// first); top-k keeps the first k, top-p the shortest prefix of those that
// holds p of their weight, min-p those with w_i >= min_p. The token drawn is
// the first, in index order, whose running sum of kept weights exceeds u
// times their total.
//
// Weights are whole numbers, round(w 2^S), from an fp64 exponential, so that
// every sum is exact: it does not depend on the order of its atomics and
// parts, and two calls (or two launch shapes) give the same token. A weight's
// rounding, 2^-(S+1) of the largest, is below the fp64 rounding of a running
// sum over a vocabulary.
#include <math_constants.h>

#include "paged_device.cuh"

namespace q4k {
namespace {

using namespace paged_dev;
using u64 = unsigned long long;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;

// Whole numbers in the order of the floats; NaN and -inf (never drawn) are 0.
__device__ __forceinline__ uint32_t key_of(float l) {
    if (!(l > -CUDART_INF_F)) return 0u;
    const uint32_t b = __float_as_uint(l + 0.0f);  // -0 and 0 are ties
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// One row per CTA.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a, int shift) {
    __shared__ u64 bin_w[256];
    __shared__ uint32_t bin_n[256];
    __shared__ u64 part[kSampleWarps];
    __shared__ u64 found_w;
    __shared__ uint32_t found_bin;
    __shared__ int found_index;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = a.vocab;
    const T* logits = static_cast<const T*>(a.logits) + row * a.ld;
    auto key_at = [&](int i) { return key_of(to_float<T>(logits[i])); };

    auto block_sum = [&](u64 v) {
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) part[warp] = v;
        __syncthreads();
        u64 t = 0;
        for (int w = 0; w < kSampleWarps; ++w) t += part[w];
        return t;
    };

    // the largest logit and its lowest index
    u64 best = 0;
    for (int i = tid; i < vocab; i += kSampleThreads) {
        const u64 c = (u64)key_at(i) << 32 | (uint32_t)(~i);
        best = c > best ? c : best;
    }
    for (int o = 16; o > 0; o >>= 1) {
        const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
        best = c > best ? c : best;
    }
    if (lane == 0) part[warp] = best;
    __syncthreads();
    for (int w = 0; w < kSampleWarps; ++w) best = part[w] > best ? part[w] : best;
    const uint32_t top = (uint32_t)(best >> 32);
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    if (top == 0 || !(temperature > 0.0f)) {
        if (tid == 0) {
            a.tokens[row] = top == 0 ? -1 : (int)~(uint32_t)best;
            if (a.logprob) a.logprob[row] = top == 0 ? -CUDART_INF_F : 0.0f;
        }
        return;
    }
    const double most = (double)logit_of(top), inv = 1.0 / (double)temperature, unit = ldexp(1.0, shift);
    auto exponent = [&](uint32_t key) { return key == top ? 0.0 : ((double)logit_of(key) - most) * inv; };
    auto weight = [&](uint32_t key) -> u64 { return key == 0 ? 0 : (u64)__double2ll_rn(exp(exponent(key)) * unit); };

    // kept: keys above cut, and those equal to it up to index cut_index
    uint32_t cut = 1;
    int cut_index = vocab - 1;
    auto kept = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= cut_index); };

    // Moves the cut to the shortest prefix of the kept that has `want`
    // tokens (by_weight: `want` of weight): 8 bits of the key at a time, the
    // bin where the running total passes, then the index among equal keys.
    auto narrow = [&](bool by_weight, u64 want) {
        uint32_t prefix = 0;
        u64 above = 0;
        for (int level = 24; level >= 0; level -= 8) {
            __syncthreads();
            if (tid < 256) bin_w[tid] = 0, bin_n[tid] = 0;
            __syncthreads();
            for (int i = tid; i < vocab; i += kSampleThreads) {
                const uint32_t key = key_at(i);
                if (key == 0 || !kept(key, i) || (level < 24 && key >> (level + 8) != prefix)) continue;
                const uint32_t b = key >> level & 255u;
                atomicAdd(&bin_n[b], 1u);
                if (by_weight) atomicAdd(&bin_w[b], weight(key));
            }
            __syncthreads();
            if (tid == 0) {
                u64 sum = above;
                int b = 255;
                for (; b > 0; --b) {
                    const u64 w = by_weight ? bin_w[b] : bin_n[b];
                    if (sum + w >= want) break;
                    sum += w;
                }
                found_bin = b;
                found_w = sum;
            }
            __syncthreads();
            above = found_w;
            prefix = prefix << 8 | found_bin;
        }
        // of the keys equal to prefix, the first n by index
        const u64 each = by_weight ? weight(prefix) : 1;
        const u64 n = each ? (want - above + each - 1) / each : 1;
        u64 seen = 0;
        for (int base = 0; base < vocab; base += kSampleThreads) {
            const int i = base + tid;
            const bool mine = i < vocab && key_at(i) == prefix && kept(prefix, i);
            const unsigned ballot = __ballot_sync(0xffffffffu, mine);
            __syncthreads();
            if (lane == 0) part[warp] = __popc(ballot);
            __syncthreads();
            u64 before = seen, all = seen;
            for (int w = 0; w < kSampleWarps; ++w) {
                if (w < warp) before += part[w];
                all += part[w];
            }
            if (mine && before + __popc(ballot & ((1u << lane) - 1u)) + 1 == n) found_index = i;
            seen = all;
            if (seen >= n) break;
        }
        __syncthreads();
        cut = prefix;
        cut_index = found_index;
        __syncthreads();
    };
    auto kept_weight = [&](double least) {
        u64 sum = 0;
        for (int i = tid; i < vocab; i += kSampleThreads) {
            const uint32_t key = key_at(i);
            if (key && kept(key, i) && (least <= 0.0 || exp(exponent(key)) >= least)) sum += weight(key);
        }
        return block_sum(sum);
    };

    u64 tokens = 0;
    for (int i = tid; i < vocab; i += kSampleThreads) tokens += key_at(i) != 0;
    tokens = block_sum(tokens);
    const int top_k = a.top_k ? a.top_k[row] : 0;
    if (top_k > 0 && (u64)top_k < tokens) narrow(false, (u64)top_k);
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    if (top_p < 1.0f) {
        const u64 all = kept_weight(0.0);
        const double want = ceil((double)top_p * (double)all);
        narrow(true, want >= 1.0 ? (u64)want : 1ull);
    }
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const double least = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
    const u64 total = kept_weight(least);
    const double u = (double)a.uniform[row];
    // the first running sum above floor(u total) is the first above u total
    u64 target = u > 0.0 ? (u64)(u * (double)total) : 0ull;
    target = target < total ? target : total - 1;
    u64 seen = 0;
    for (int base = 0; base < vocab; base += kSampleThreads) {
        const int i = base + tid;
        u64 w = 0;
        if (i < vocab) {
            const uint32_t key = key_at(i);
            if (key && kept(key, i) && (least <= 0.0 || exp(exponent(key)) >= least)) w = weight(key);
        }
        u64 run = w;
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        __syncthreads();
        if (lane == 31) part[warp] = run;
        __syncthreads();
        u64 before = seen, all = seen;
        for (int k = 0; k < kSampleWarps; ++k) {
            if (k < warp) before += part[k];
            all += part[k];
        }
        run += before;
        if (w && run > target && run - w <= target) {
            a.tokens[row] = i;
            if (a.logprob) a.logprob[row] = (float)(exponent(key_at(i)) - log((double)total / unit));
        }
        seen = all;
        if (seen > target) break;
    }
}

}  // namespace

cudaError_t sample(const SampleArgs& a, cudaStream_t s) {
    int bits = 1;  // vocab < 2^bits
    while ((1ll << bits) <= a.vocab) ++bits;
    const int shift = 62 - bits;
    if (a.type == Q4K_TYPE_F32)
        sample_kernel<float><<<a.rows, kSampleThreads, 0, s>>>(a, shift);
    else if (a.type == Q4K_TYPE_F16)
        sample_kernel<__half><<<a.rows, kSampleThreads, 0, s>>>(a, shift);
    else
        sample_kernel<__nv_bfloat16><<<a.rows, kSampleThreads, 0, s>>>(a, shift);
    return cudaGetLastError();
}

}  // namespace q4k
