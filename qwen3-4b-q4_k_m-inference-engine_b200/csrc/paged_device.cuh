// Device routines over a batch of sequences in a paged cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "q4k_device.cuh"

namespace q4k {
namespace paged_dev {

// A sequence of the batch as the kernels see it. Whatever stands in the
// device arrays, first_row and rows stay inside the batch's rows and keys
// inside the page table, so that no access depends on their values being
// sensible.
struct Sequence {
    int first_row;  // of q, k, v and the outputs
    int rows;       // new tokens
    int position;   // of the first new token (negative: rows before the cache's start)
};

__device__ __forceinline__ Sequence sequence_of(const PagedBatch& b, int s) {
    Sequence r;
    const int q0 = __ldg(b.q_start + s), q1 = __ldg(b.q_start + s + 1), len = max(__ldg(b.kv_len + s), 0);
    r.first_row = min(max(q0, 0), b.tokens);
    r.rows = max(min(q1, b.tokens) - r.first_row, 0);
    r.position = len - r.rows;
    return r;
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// N consecutive values to memory aligned to their size, at most 16 bytes.
template <typename T, int N>
__device__ __forceinline__ void store_values(T* p, const float (&x)[N]) {
    constexpr int kBytes = N * (int)sizeof(T);
    static_assert(kBytes == 8 || kBytes % 16 == 0, "8 bytes or whole 16-byte words");
    alignas(16) T t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = from_float<T>(x[j]);
    if constexpr (kBytes == 8) {
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
    }
}

}  // namespace paged_dev
}  // namespace q4k
