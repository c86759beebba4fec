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
// sum of squares is a few shuffles. A CTA takes kTokens tokens: one with few
// tokens (a decode step), so that its rows spread over several CTAs; with many
// as many as give every thread one angle to work out, which also spreads the
// search for the token's sequence and page over more bytes.
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

template <typename T, typename C, int HALF, int kTokens>
__global__ void __launch_bounds__(kAppendThreads)
    paged_append_kernel(const __grid_constant__ PagedAppendArgs a, const __grid_constant__ Frequencies f) {
    constexpr int kVec = 16 / sizeof(T);
    constexpr int kLanes = HALF / kVec;             // lanes of a row
    constexpr int kRows = kAppendThreads / kLanes;  // rows a CTA holds at a time
    constexpr int D = 2 * HALF;
    constexpr int kWarps = kAppendThreads / 32;
    static_assert(kTokens <= kWarps, "a warp finds a token's place");
    __shared__ float cosines[kTokens][HALF], sines[kTokens][HALF];
    __shared__ long long places[kTokens];  // cache offset of head 0's row; -1: none; -2: a row of no sequence
    __shared__ int positions[kTokens];
    const int t0 = blockIdx.x * kTokens, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int heads = a.heads, kv = a.cache.kv_heads, rows = heads + 2 * kv;
    const int tokens = min(kTokens, a.batch.tokens - t0);
    const int j0 = tid % kLanes * kVec;
    // work items: rows of token 0, of token 1, ...
    const int items = tokens * rows, step = gridDim.y * kRows;
    int item = blockIdx.y * kRows + tid / kLanes;

    // row r of a token: its queries, then keys, then values
    auto row = [&](int t, int r) -> const T* {
        if (r < heads) return static_cast<const T*>(a.q) + (t0 + t) * a.ld_q + (size_t)r * D;
        if (r < heads + kv) return static_cast<const T*>(a.k) + (t0 + t) * a.ld_k + (size_t)(r - heads) * D;
        return static_cast<const T*>(a.v) + (t0 + t) * a.ld_v + (size_t)(r - heads - kv) * D;
    };
    uint4 x[2];
    auto fetch = [&](int i) {
        if (i >= items) return;
        const int t = kTokens == 1 ? 0 : i / rows;
        const T* p = row(t, i - t * rows) + j0;
        x[0] = __ldg(reinterpret_cast<const uint4*>(p));
        x[1] = __ldg(reinterpret_cast<const uint4*>(p + HALF));
    };
    fetch(item);
    if (warp < tokens) {
        // the sequences that end at or before a token's row are those before its own
        const int t = t0 + warp;
        int s = 0;
        for (int i = 0; i < a.batch.sequences; i += 32)
            s += __popc(__ballot_sync(0xffffffffu, i + lane < a.batch.sequences && __ldg(a.batch.q_start + i + lane + 1) <= t));
        if (lane == 0) {
            long long place = -2;
            int position = 0;
            // (rows before the first sequence are nobody's either)
            if (s < a.batch.sequences && t >= __ldg(a.batch.q_start + s)) {
                position = max(__ldg(a.batch.kv_len + s), 0) - __ldg(a.batch.q_start + s + 1) + t;
                const int column = position >> a.cache.page_shift;
                place = -1;  // a position that no page holds
                if (position >= 0 && column < a.batch.table_width) {
                    const int page = __ldg(a.batch.page_table + (size_t)s * a.batch.table_stride + column);
                    if (page >= 0 && page < a.cache.pages)
                        place = page * a.cache.page_stride + (position & (a.cache.page_size - 1)) * a.cache.row_stride;
                }
            }
            places[warp] = place;
            positions[warp] = position;
        }
    }
    __syncthreads();
    for (int i = tid; i < tokens * HALF; i += kAppendThreads) {
        const double turns = (double)positions[i / HALF] * f.turns[i % HALF];
        sincospif(2.0f * (float)(turns - rint(turns)), &sines[i / HALF][i % HALF], &cosines[i / HALF][i % HALF]);
    }
    __syncthreads();

    for (; item < items; item += step) {
        const int t = kTokens == 1 ? 0 : item / rows, r = item - t * rows;
        float y0[kVec], y1[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            y0[i] = to_float<T>(reinterpret_cast<const T*>(&x[0])[i]);
            y1[i] = to_float<T>(reinterpret_cast<const T*>(&x[1])[i]);
        }
        fetch(item + step);
        const long long place = places[t];
        const bool is_v = r >= heads + kv;
        if (!is_v) {
            const float* gamma = r < heads ? a.q_gamma : a.k_gamma;
            if (gamma) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < kVec; ++i) ss += y0[i] * y0[i] + y1[i] * y1[i];
                // the row's lanes are neighbours, and all of them are here
                const unsigned mask = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (lane / kLanes * kLanes);
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float inv = rsqrtf(ss / (float)D + a.eps);
                float g0[kVec], g1[kVec];
#pragma unroll
                for (int i = 0; i < kVec; i += 4) {
                    *reinterpret_cast<float4*>(g0 + i) = __ldg(reinterpret_cast<const float4*>(gamma + j0 + i));
                    *reinterpret_cast<float4*>(g1 + i) = __ldg(reinterpret_cast<const float4*>(gamma + j0 + HALF + i));
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    y0[i] = y0[i] * inv * g0[i];
                    y1[i] = y1[i] * inv * g1[i];
                }
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float c = cosines[t][j0 + i], sn = sines[t][j0 + i], u = y0[i], w = y1[i];
                y0[i] = u * c - w * sn;
                y1[i] = u * sn + w * c;
            }
        }
        if (place == -2) continue;
        if (r < heads) {
            T* o = static_cast<T*>(a.q_out) + (t0 + t) * a.ld_q_out + (size_t)r * D + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        } else if (place >= 0) {
            const int h = is_v ? r - heads - kv : r - heads;
            C* o = reinterpret_cast<C*>(is_v ? a.cache.v : a.cache.k) + place + h * a.cache.head_stride + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        }
    }
}

template <typename T, typename C, int HALF>
void launch(const PagedAppendArgs& a, const Frequencies& f, cudaStream_t s) {
    constexpr int kHeld = kAppendThreads / (HALF / (16 / (int)sizeof(T)));  // rows of a CTA at a time
    constexpr int kMany = kAppendThreads / HALF;
    const int rows = a.heads + 2 * a.cache.kv_heads;
    // few tokens: a token's rows over several CTAs; measured equal near 2 tokens per SM
    if (a.batch.tokens <= 2 * sm_count())
        paged_append_kernel<T, C, HALF, 1>
            <<<dim3(a.batch.tokens, (rows + kHeld - 1) / kHeld), kAppendThreads, 0, s>>>(a, f);
    else
        paged_append_kernel<T, C, HALF, kMany>
            <<<dim3((a.batch.tokens + kMany - 1) / kMany, 1), kAppendThreads, 0, s>>>(a, f);
}

template <typename T, typename C>
void launch_dim(const PagedAppendArgs& a, const Frequencies& f, cudaStream_t s) {
    if (a.cache.head_dim == 128)
        launch<T, C, 64>(a, f, s);
    else
        launch<T, C, 32>(a, f, s);
}

}  // namespace

cudaError_t paged_append(const PagedAppendArgs& a, cudaStream_t s) {
    const int d = a.cache.head_dim, half = d / 2;
    Frequencies f = {};
    // powers by products: 64 roundings of 2^-53 are 1e-7 of a turn at position 2^30
    const double ratio = std::pow(a.rope_base, -2.0 / d);
    f.turns[0] = 1.0 / 6.283185307179586476925;
    for (int j = 1; j < half; ++j) f.turns[j] = f.turns[j - 1] * ratio;
    if (a.f32)
        launch_dim<float, __half>(a, f, s);
    else if (a.cache.bf16)
        launch_dim<__nv_bfloat16, __nv_bfloat16>(a, f, s);
    else
        launch_dim<__half, __half>(a, f, s);
    return cudaGetLastError();
}

}  // namespace q4k
