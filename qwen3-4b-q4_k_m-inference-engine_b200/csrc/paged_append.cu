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
// tokens (a decode step), so that its rows spread over several CTAs; up to eight
// with many, a warp finding each token's sequence and page, so that this chain of
// loads (2 us) and the angles are spread over more bytes. Measured: 8252 bf16
// tokens of 32 + 2 x 8 heads of 128 in 40.8 us, 4.7 TB/s (1 token a CTA: 107 us,
// 2: 43.7, 4: 41.6); 64 fp32 tokens 3.7 us, which is the launch and that chain.
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
    __shared__ __align__(16) float cosines[kTokens][HALF], sines[kTokens][HALF], gammas[2][D];
    __shared__ long long places[kTokens];  // cache offset of head 0's row; -1: none; -2: a row of no sequence
    __shared__ int positions[kTokens];
    const int t0 = blockIdx.x * kTokens, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int heads = a.heads, kv = a.cache.kv_heads, rows = heads + 2 * kv;
    const int tokens = min(kTokens, a.batch.tokens - t0);
    const int j0 = tid % kLanes * kVec;
    // work items: rows of token 0, of token 1, ...; this thread's next is row r of token t
    const int step = gridDim.y * kRows;
    int t = 0, r = blockIdx.y * kRows + tid / kLanes;
    auto settle = [&] {
        while (r >= rows && t < tokens) {
            r -= rows;
            ++t;
        }
    };
    uint4 x[2];
    // the item's halves: a query's, key's or value's
    auto fetch = [&] {
        if (t >= tokens) return;
        const T* p;
        if (r < heads)
            p = static_cast<const T*>(a.q) + (t0 + t) * a.ld_q + (size_t)r * D;
        else if (r < heads + kv)
            p = static_cast<const T*>(a.k) + (t0 + t) * a.ld_k + (size_t)(r - heads) * D;
        else
            p = static_cast<const T*>(a.v) + (t0 + t) * a.ld_v + (size_t)(r - heads - kv) * D;
        x[0] = __ldg(reinterpret_cast<const uint4*>(p + j0));
        x[1] = __ldg(reinterpret_cast<const uint4*>(p + j0 + HALF));
    };
    settle();
    fetch();
    for (int i = tid; i < 2 * D; i += kAppendThreads) {
        const float* g = i < D ? a.q_gamma : a.k_gamma;
        gammas[i / D][i % D] = g ? __ldg(g + i % D) : 1.0f;
    }
    if (warp < tokens) {
        // the sequences that end at or before a token's row are those before its own
        const int at = t0 + warp;
        int s = 0;
        for (int i = 0; i < a.batch.sequences; i += 32)
            s += __popc(
                __ballot_sync(0xffffffffu, i + lane < a.batch.sequences && __ldg(a.batch.q_start + i + lane + 1) <= at));
        if (lane == 0) {
            long long place = -2;
            int position = 0;
            // (rows before the first sequence are nobody's either)
            if (s < a.batch.sequences && at >= __ldg(a.batch.q_start + s)) {
                position = max(__ldg(a.batch.kv_len + s), 0) - __ldg(a.batch.q_start + s + 1) + at;
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

    while (t < tokens) {
        const int token = t, row = r;
        float y0[kVec], y1[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            y0[i] = to_float<T>(reinterpret_cast<const T*>(&x[0])[i]);
            y1[i] = to_float<T>(reinterpret_cast<const T*>(&x[1])[i]);
        }
        r += step;
        settle();
        fetch();
        const long long place = places[token];
        const bool is_q = row < heads, is_v = row >= heads + kv;
        if (!is_v) {
            if (is_q ? a.q_gamma : a.k_gamma) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < kVec; ++i) ss += y0[i] * y0[i] + y1[i] * y1[i];
                // the row's lanes are neighbours, and all of them are here
                const unsigned mask = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (lane / kLanes * kLanes);
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float inv = rsqrtf(ss * (1.0f / (float)D) + a.eps);
                const float* g = gammas[is_q ? 0 : 1] + j0;
#pragma unroll
                for (int i = 0; i < kVec; i += 4) {
                    const float4 g0 = *reinterpret_cast<const float4*>(g + i);
                    const float4 g1 = *reinterpret_cast<const float4*>(g + HALF + i);
                    y0[i] *= inv * g0.x, y0[i + 1] *= inv * g0.y, y0[i + 2] *= inv * g0.z, y0[i + 3] *= inv * g0.w;
                    y1[i] *= inv * g1.x, y1[i + 1] *= inv * g1.y, y1[i + 2] *= inv * g1.z, y1[i + 3] *= inv * g1.w;
                }
            }
            float c[kVec], sn[kVec];
#pragma unroll
            for (int i = 0; i < kVec; i += 4) {
                *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(&cosines[token][j0 + i]);
                *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(&sines[token][j0 + i]);
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float u = y0[i], w = y1[i];
                y0[i] = u * c[i] - w * sn[i];
                y1[i] = u * sn[i] + w * c[i];
            }
        }
        if (place == -2) continue;
        if (is_q) {
            T* o = static_cast<T*>(a.q_out) + (t0 + token) * a.ld_q_out + (size_t)row * D + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        } else if (place >= 0) {
            const int h = is_v ? row - heads - kv : row - heads;
            C* o = reinterpret_cast<C*>(is_v ? a.cache.v : a.cache.k) + place + h * a.cache.head_stride + j0;
            store_values(o, y0);
            store_values(o + HALF, y1);
        }
    }
}

template <typename T, typename C, int HALF>
void launch(const PagedAppendArgs& a, const Frequencies& f, cudaStream_t s) {
    constexpr int kHeld = kAppendThreads / (HALF / (16 / (int)sizeof(T)));  // rows of a CTA at a time
    const int rows = a.heads + 2 * a.cache.kv_heads, n = a.batch.tokens, per_sm = n / sm_count();
    // Tokens a CTA, by how many there are (us with 1 / 2 / 4 / 8 of them, fp32 rows of 32 + 2 x 8 heads of 128):
    //   300 tokens 6.9 / 7.4 / 9.7 / 15.5, 1000 20.2 / 15.5 / 18.1 / 24.9, 2000 41.3 / 29.3 / 27.3 / 33.0,
    //   4000 90.3 / 51.2 / 54.9 / 49.8; bf16 the same way (1000: 14.3 / 10.0 / 10.6 / 13.0)
    if (per_sm < 2)  // a token's rows over several CTAs
        paged_append_kernel<T, C, HALF, 1><<<dim3(n, (rows + kHeld - 1) / kHeld), kAppendThreads, 0, s>>>(a, f);
    else if (per_sm < 8)
        paged_append_kernel<T, C, HALF, 2><<<(n + 1) / 2, kAppendThreads, 0, s>>>(a, f);
    else if (per_sm < 16)
        paged_append_kernel<T, C, HALF, 4><<<(n + 3) / 4, kAppendThreads, 0, s>>>(a, f);
    else
        paged_append_kernel<T, C, HALF, 8><<<(n + 7) / 8, kAppendThreads, 0, s>>>(a, f);
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
