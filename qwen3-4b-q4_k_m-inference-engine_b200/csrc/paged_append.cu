// q4k_paged_append: the new tokens of a batch of sequences enter a paged KV
// cache. Per token and head, y = x * rsqrt(mean(x^2) + eps) * gamma (queries
// and keys, where a gamma is given), then the pair (y_j, y_{j + d/2}) is
// turned by the angle position * base^(-2j/d); queries go to q_out, keys and
// values (values as they are) to the page row of the token's position.
//
// HBM-bound: each row is read once and written once. A thread holds 16 bytes
// of each half of a row (4 fp32 or 8 16-bit values), so that a pair never
// leaves its thread and every access is a whole 16-byte word (8-byte stores
// where fp32 rows become fp16); a row takes 4 to 16 neighbouring lanes, whose
// sum of squares is a few shuffles. A CTA works on rows of one token, which
// share their angles.
//
// Angles: far positions need more bits than fp32 has (position 1e5 has an
// fp32 angle error of 4e-3 rad), so the turns position * (base^(-2j/d) / 2 pi)
// are taken in fp64 (the frequencies come from the host), reduced to [-1/2,
// 1/2] exactly, and only the fraction goes to fp32: its rounding is 2^-25 of
// a turn, 2e-7 rad.
#include <cmath>

#include "paged.h"
#include "paged_device.cuh"

namespace q4k {
namespace {

using namespace paged_dev;

constexpr int kAppendThreads = 256;
constexpr int kMaxHalf = 64;  // pairs of a head

struct Frequencies {
    double turns[kMaxHalf];  // base^(-2j/d) / (2 pi)
};

template <typename T, typename C, int HALF>
__global__ void __launch_bounds__(kAppendThreads)
    paged_append_kernel(const __grid_constant__ PagedAppendArgs a, const __grid_constant__ Frequencies f) {
    constexpr int kVec = 16 / sizeof(T);
    constexpr int kLanes = HALF / kVec;             // lanes of a row
    constexpr int kRows = kAppendThreads / kLanes;  // rows a CTA holds at a time
    constexpr int D = 2 * HALF;
    __shared__ float cosines[HALF], sines[HALF];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int heads = a.heads, kv = a.cache.kv_heads, rows = heads + 2 * kv;
    const int j0 = tid % kLanes * kVec;
    const int first = blockIdx.y * kRows + tid / kLanes, step = gridDim.y * kRows;

    // row r of the token: its queries, then keys, then values
    auto row = [&](int r) -> const T* {
        if (r < heads) return static_cast<const T*>(a.q) + t * a.ld_q + (size_t)r * D;
        if (r < heads + kv) return static_cast<const T*>(a.k) + t * a.ld_k + (size_t)(r - heads) * D;
        return static_cast<const T*>(a.v) + t * a.ld_v + (size_t)(r - heads - kv) * D;
    };
    float x0[kVec], x1[kVec];
    if (first < rows) {
        load_values(row(first) + j0, x0);
        load_values(row(first) + j0 + HALF, x1);
    }
    // the sequences that end at or before row t are those before its own
    int s = 0;
    for (int i = 0; i < a.batch.sequences; i += kAppendThreads)
        s += __syncthreads_count(i + tid < a.batch.sequences && __ldg(a.batch.q_start + i + tid + 1) <= t);
    if (s >= a.batch.sequences) return;  // a row behind the last sequence
    const int position = __ldg(a.batch.kv_len + s) - __ldg(a.batch.q_start + s + 1) + t;
    const int column = position >> a.cache.page_shift;
    // the token's page; -1 for a position that no page holds
    int page = -1;
    if (position >= 0 && column < a.batch.table_width)
        page = __ldg(a.batch.page_table + (size_t)s * a.batch.table_stride + column);
    if (page >= a.cache.pages) page = -1;
    if (tid < HALF) {
        const double turns = (double)position * f.turns[tid];
        sincospif(2.0f * (float)(turns - rint(turns)), &sines[tid], &cosines[tid]);
    }
    __syncthreads();

    for (int r = first; r < rows; r += step) {
        const bool is_v = r >= heads + kv;
        float y0[kVec], y1[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            y0[i] = x0[i];
            y1[i] = x1[i];
        }
        if (r + step < rows) {
            load_values(row(r + step) + j0, x0);
            load_values(row(r + step) + j0 + HALF, x1);
        }
        if (!is_v) {
            const float* gamma = r < heads ? a.q_gamma : a.k_gamma;
            if (gamma) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < kVec; ++i) ss += y0[i] * y0[i] + y1[i] * y1[i];
                // the row's lanes are neighbours, and all of them are here
                const unsigned mask = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << ((tid & 31) / kLanes * kLanes));
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float inv = rsqrtf(ss / (float)D + a.eps);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    y0[i] = y0[i] * inv * __ldg(gamma + j0 + i);
                    y1[i] = y1[i] * inv * __ldg(gamma + j0 + HALF + i);
                }
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float c = cosines[j0 + i], sn = sines[j0 + i], u = y0[i], w = y1[i];
                y0[i] = u * c - w * sn;
                y1[i] = u * sn + w * c;
            }
        }
        if (r < heads) {
            T* o = static_cast<T*>(a.q_out) + t * a.ld_q_out + (size_t)r * D + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        } else if (page >= 0) {
            const int h = is_v ? r - heads - kv : r - heads;
            C* o = reinterpret_cast<C*>(is_v ? a.cache.v : a.cache.k) + page * a.cache.page_stride +
                   h * a.cache.head_stride + (position & (a.cache.page_size - 1)) * a.cache.row_stride + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        }
    }
}

template <typename T, typename C>
void launch(const PagedAppendArgs& a, const Frequencies& f, dim3 grid, cudaStream_t s) {
    if (a.cache.head_dim == 128)
        paged_append_kernel<T, C, 64><<<grid, kAppendThreads, 0, s>>>(a, f);
    else
        paged_append_kernel<T, C, 32><<<grid, kAppendThreads, 0, s>>>(a, f);
}

}  // namespace

cudaError_t paged_append(const PagedAppendArgs& a, cudaStream_t s) {
    const int d = a.cache.head_dim, half = d / 2;
    Frequencies f = {};
    // powers by products: 64 roundings of 2^-53 are 1e-7 of a turn at position 2^30
    const double ratio = std::pow(a.rope_base, -2.0 / d);
    f.turns[0] = 1.0 / 6.283185307179586476925;
    for (int j = 1; j < half; ++j) f.turns[j] = f.turns[j - 1] * ratio;
    const int rows = a.heads + 2 * a.cache.kv_heads;
    const int held = kAppendThreads / (half / (a.f32 ? 4 : 8));
    const dim3 grid(a.batch.tokens, (rows + held - 1) / held);
    if (a.f32)
        launch<float, __half>(a, f, grid, s);
    else if (a.cache.bf16)
        launch<__nv_bfloat16, __nv_bfloat16>(a, f, grid, s);
    else
        launch<__half, __half>(a, f, grid, s);
    return cudaGetLastError();
}

}  // namespace q4k
