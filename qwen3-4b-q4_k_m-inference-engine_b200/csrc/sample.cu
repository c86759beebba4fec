// q4k_sample: one token per row of logits. With x_i = (l_i - max l) / T and
// w_i = e^(x_i), the tokens are ordered by logit (ties: the lowest index
// first); top-k keeps the first k, top-p the shortest prefix of those that
// holds p of their weight, min-p those with w_i >= min_p. The token drawn is
// the first, in index order, whose running sum of kept weights exceeds u
// times their total.
//
// Weights are whole numbers, round(w 2^S), so that every sum is exact: it
// does not depend on the order of atomics or on how a row is cut, and two
// calls (or two launch shapes) give the same token. S leaves room for a
// vocabulary of ones in 62 bits (44 for 2^18 tokens); a weight's rounding,
// 2^-(S+1) of the largest, moves the draw's boundaries by about 1e-12.
//
// No sorting: a row's threshold is found by histograms. A cluster of 1 to 16
// CTAs holds the row in shared memory, each CTA a slice, so that the logits
// are read from HBM once; the passes over them (maximum, 2048 equal bins of
// the distance to the maximum, 2048 bins of the bin where the running total
// passes, the draw) run from there, and only bins and totals cross the
// cluster. Equal keys in the last bin end the search; otherwise (values
// closer than 2^-22 of the range) their bits are gone through, 11 at a time.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <mutex>

#include "paged_device.cuh"

namespace q4k {
namespace {

using namespace paged_dev;
namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 16;
constexpr int kVec = 4;                               // consecutive logits of a thread
constexpr int kStride = kSampleThreads * kVec;        // logits of one step of the CTA
// Logits of one CTA: 80 KB of them, so that two CTAs fit an SM; 25000 fp32 ones
// of a vocabulary of 400000 in 16 CTAs (one to an SM).
constexpr int kSliceBytes = 80 * 1024;
template <typename T>
constexpr int kMaxSlice = kSliceBytes / sizeof(T) > 25600 ? kSliceBytes / sizeof(T) : 25600;
constexpr int kMaxSteps = (kMaxSlice<uint16_t> + kStride - 1) / kStride;
constexpr int kTable = 64;

// Whole numbers in the order of the floats.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);  // -0 and 0 are ties
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Crossing {
    u64 above, inside;  // the total above the bin, and in it
    int bin;
};

struct alignas(16) SampleShared {
    uint32_t lo[kBins], hi[kBins];  // a histogram of 64-bit sums
    double table[kTable];           // 2^(j/64)
    u64 chunk[kMaxSteps * kSampleWarps];
    u64 warp_sum[kSampleWarps];
    u64 total[kMaxCluster];  // one word from every CTA of the cluster
    float bound[2][kMaxCluster];
    Crossing crossing;
    int place;
};

// w(l) = round(2^(S + (l - top) log2(e) / T)). The exponent t is taken as a
// sum of two floats (the subtraction's and the product's own roundings kept),
// 2^-46 of it; 2^frac(t) is 2^(j/64) times a Taylor polynomial in fp64 where w
// needs the bits, ex2.approx (2^-22) below 2^-26, where 2^-48 of the largest
// weight is all that is lost.
struct Weights {
    float top, c_hi, c_lo, cutoff;
    int S;
    const double* table;

    __device__ __forceinline__ u64 operator()(float l) const {
        if (l == top) return 1ull << S;
        const float d = l - top, bb = d - l;
        const float err = (l - (d - bb)) - (top + bb);
        const float t = d * c_hi;
        if (!(t > cutoff)) return 0;
        const float t_lo = fmaf(d, c_hi, -t) + fmaf(d, c_lo, err * c_hi);
        const float n = rintf(t), f = t - n;
        if (t < -26.0f) {
            float p;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(f + t_lo));
            return __float2ull_rn(p * __uint_as_float((uint32_t)(127 + (int)n + S) << 23));
        }
        // f = j / 64 + r
        const float j = rintf(f * 64.0f);
        const double r = ((double)fmaf(j, -1.0f / 64.0f, f) + (double)t_lo) * 0.693147180559945309417;
        const int ji = (int)j;
        double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        const int e = (int)n + S + (ji >> 6);  // ji in [-32, 32]
        const double scale = __hiloint2double((1023 + e) << 20, 0);
        return (u64)__double2ll_rn(p * table[ji & 63] * scale);
    }
};

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2)
    sample_kernel(const __grid_constant__ SampleArgs a, int S, int slice) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
    T* held = reinterpret_cast<T*>(smem + sizeof(SampleShared));
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = min(rank * slice, a.vocab);         // this CTA's logits: base .. base + count - 1
    const int count = min(slice, a.vocab - base);
    const int steps = (count + kStride - 1) / kStride;
    const T* src = static_cast<const T*>(a.logits) + row * a.ld + base;

    if (tid < kTable) sh.table[tid] = exp2(tid / 64.0);
    float most = -CUDART_INF_F;
    if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
        constexpr int kWide = 16 / sizeof(T);
#pragma unroll 4
        for (int i = tid * kWide; i + kWide <= count; i += kSampleThreads * kWide) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src + i));
            *reinterpret_cast<uint4*>(held + i) = w;
            const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int j = 0; j < kWide; ++j) most = fmaxf(most, to_float<T>(t[j]));
        }
        const int i = count / kWide * kWide + tid;
        if (i < count) {
            held[i] = src[i];
            most = fmaxf(most, to_float<T>(src[i]));
        }
    } else {
#pragma unroll 4
        for (int i = tid; i < count; i += kSampleThreads) {
            const T v = src[i];
            held[i] = v;
            most = fmaxf(most, to_float<T>(v));
        }
    }
    // what lies behind the slice, up to a whole step, is never drawn
    for (int i = count + tid; i < steps * kStride; i += kSampleThreads) held[i] = from_float<T>(-CUDART_INF_F);

    // The largest and smallest of a value over the cluster.
    auto cluster_bounds = [&](float high, float low) {
        high = warp_max(high);
        low = -warp_max(-low);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = (u64)__float_as_uint(low) << 32 | __float_as_uint(high);
        __syncthreads();
        if (tid < ranks) {
            for (int w = 0; w < kSampleWarps; ++w) {
                high = fmaxf(high, __uint_as_float((uint32_t)sh.warp_sum[w]));
                low = fminf(low, __uint_as_float((uint32_t)(sh.warp_sum[w] >> 32)));
            }
            float* to = cluster.map_shared_rank(&sh.bound[0][0], tid);
            to[rank] = high;
            to[kMaxCluster + rank] = low;
        }
        cluster.sync();
        for (int r = 0; r < ranks; ++r) {
            high = fmaxf(high, sh.bound[0][r]);
            low = fminf(low, sh.bound[1][r]);
        }
        return make_float2(high, low);
    };
    const float top = cluster_bounds(most, most).x;

    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    const double c = 1.44269504088896340736 / (double)(greedy ? 1.0f : temperature);
    const float c_hi = (float)c;
    const Weights weight = {top, c_hi, (float)(c - (double)c_hi), -(float)S - 1.0f, S, sh.table};

    // kept: logits above cut, and those equal to it up to index cut_index
    float cut = -CUDART_INF_F;
    int cut_index = -1;
    auto kept = [&](float l, int i) { return l > cut || (l == cut && i <= cut_index); };

    // f(logit, index) for all of the CTA's logits, four at a time
    auto for_each = [&](auto&& f) {
        for (int s = 0; s < steps; ++s) {
            const int at = s * kStride + tid * kVec;
            T v[kVec];
            if constexpr (sizeof(T) == 4)
                *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(held + at);
            else
                *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(held + at);
#pragma unroll
            for (int j = 0; j < kVec; ++j) f(to_float<T>(v[j]), base + at + j, s);
        }
    };

    auto clear = [&] {
        for (int i = tid; i < kBins; i += kSampleThreads) sh.lo[i] = sh.hi[i] = 0;
        __syncthreads();
    };
    auto add = [&](int bin, u64 v) {
        const uint32_t low = (uint32_t)v, old = atomicAdd(&sh.lo[bin], low);
        const uint32_t high = (uint32_t)(v >> 32) + (old + low < old);
        if (high) atomicAdd(&sh.hi[bin], high);
    };
    // The inclusive running sum over the CTA's threads, and the CTA's total.
    auto block_scan = [&](u64 v, u64& all) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = v;
        __syncthreads();
        all = 0;
        u64 before = 0;
        for (int w = 0; w < kSampleWarps; ++w) {
            if (w < warp) before += sh.warp_sum[w];
            all += sh.warp_sum[w];
        }
        return v + before;
    };
    // Of the cluster's histograms together: the bin where the running total,
    // from `above`, first reaches `want`. Each CTA adds up a share of the bins.
    auto cross = [&](u64 above, u64 want) {
        cluster.sync();
        const int per = kBins / ranks, q = (per + kSampleThreads - 1) / kSampleThreads;
        u64 mine[kBins / kSampleThreads], sum = 0;
#pragma unroll
        for (int j = 0; j < kBins / kSampleThreads; ++j) {
            mine[j] = 0;
            if (j < q && tid * q + j < per) {
                const int bin = rank * per + tid * q + j;
                for (int r = 0; r < ranks; ++r)
                    mine[j] += ((u64)cluster.map_shared_rank(sh.hi, r)[bin] << 32) + cluster.map_shared_rank(sh.lo, r)[bin];
                sum += mine[j];
            }
        }
        u64 all;
        const u64 run = block_scan(sum, all) - sum;
        if (tid < ranks) cluster.map_shared_rank(sh.total, tid)[rank] = all;
        cluster.sync();
        u64 before = above + run;
        for (int r = 0; r < rank; ++r) before += sh.total[r];
        if (before < want && want <= before + sum) {
#pragma unroll
            for (int j = 0; j < kBins / kSampleThreads; ++j) {
                if (before < want && want <= before + mine[j]) {
                    const Crossing found = {before, mine[j], rank * per + tid * q + j};
                    for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&sh.crossing, r) = found;
                }
                before += mine[j];
            }
        }
        cluster.sync();
        return sh.crossing;
    };
    // Index of the first logit, in index order, at which the running sum of
    // value(logit, index) over the row exceeds target(total); -1 if none does.
    auto locate = [&](auto&& value, auto&& target, u64& total) {
        u64 mine = 0, step_sum = 0;
        int step = 0;
        auto close = [&] {
            u64 v = step_sum;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == 0) sh.chunk[step * kSampleWarps + warp] = v;
            mine += step_sum;
            step_sum = 0;
        };
        for_each([&](float l, int i, int s) {
            if (s != step) {
                close();
                step = s;
            }
            step_sum += value(l, i);
        });
        if (steps > 0) close();
        u64 all;
        block_scan(mine, all);
        if (tid == 0) sh.place = -1;
        if (tid < ranks) cluster.map_shared_rank(sh.total, tid)[rank] = all;
        cluster.sync();
        total = 0;
        u64 before = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r < rank) before += sh.total[r];
            total += sh.total[r];
        }
        const u64 goal = target(total);
        if (warp == 0 && before <= goal && goal < before + all) {
            // the chunk of 128 logits, 32 chunks at a time, then the logit
            u64 at = goal - before;
            int chunk = 0;
            for (int b = 0; b < steps * kSampleWarps; b += 32) {
                const u64 v = b + lane < steps * kSampleWarps ? sh.chunk[b + lane] : 0;
                u64 run = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 u = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += u;
                }
                const unsigned past = __ballot_sync(0xffffffffu, run > at);
                if (past) {
                    const int first = __ffs(past) - 1;
                    at -= __shfl_sync(0xffffffffu, run - v, first);
                    chunk = b + first;
                    break;
                }
                at -= __shfl_sync(0xffffffffu, run, 31);
            }
            const int i0 = chunk / kSampleWarps * kStride + chunk % kSampleWarps * 32 * kVec + lane * kVec;
            u64 v[kVec], sum = 0;
#pragma unroll
            for (int j = 0; j < kVec; ++j) sum += v[j] = value(to_float<T>(held[i0 + j]), base + i0 + j);
            u64 run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 u = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += u;
            }
            run -= sum;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                if (run <= at && at < run + v[j])
                    for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&sh.place, r) = base + i0 + j;
                run += v[j];
            }
        }
        cluster.sync();
        return sh.place;
    };

    // Moves the cut to the shortest prefix of the kept that has `want` of
    // value(logit), `range` being the distance from the top that the first
    // bins resolve.
    auto narrow = [&](auto&& value, u64 want, float range) {
        const float scale = (float)kBins / range;
        auto bin_of = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * scale, (float)(kBins - 1)); };
        clear();
        for_each([&](float l, int i, int) {
            if (kept(l, i)) add(bin_of(l), value(l));
        });
        Crossing x = cross(0, want);
        const int bin = x.bin;
        auto fine = [&](float l) {
            return (int)fminf(fmaxf(((top - l) * scale - (float)bin) * (float)kBins, 0.0f), (float)(kBins - 1));
        };
        clear();
        for_each([&](float l, int i, int) {
            if (kept(l, i) && bin_of(l) == bin) add(fine(l), value(l));
        });
        x = cross(x.above, want);
        const int sub = x.bin;
        float high = -CUDART_INF_F, low = CUDART_INF_F;
        for_each([&](float l, int i, int) {
            if (kept(l, i) && bin_of(l) == bin && fine(l) == sub) high = fmaxf(high, l), low = fminf(low, l);
        });
        const float2 ends = cluster_bounds(high, low);
        float key = ends.x;
        if (ends.x != ends.y) {
            uint32_t prefix = 0;
#pragma unroll 1
            for (int level = 0; level < 3; ++level) {
                const int down = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
                const uint32_t mask = (1u << bits) - 1u;
                clear();
                for_each([&](float l, int i, int) {
                    if (!(kept(l, i) && bin_of(l) == bin && fine(l) == sub)) return;
                    const uint32_t k = key_of(l);
                    if (level == 0 || k >> (down + bits) == prefix) add((int)(mask - (k >> down & mask)), value(l));
                });
                x = cross(x.above, want);
                prefix = prefix << bits | (mask - (uint32_t)x.bin);
            }
            key = logit_of(prefix);
        }
        // of the logits equal to key, the first n by index
        const u64 each = value(key), n = each ? (want - x.above + each - 1) / each : 1;
        const float old = cut;
        const int old_index = cut_index;
        cut = key;
        cut_index = a.vocab;
        if (n * each < x.inside) {
            u64 total;
            cut_index = locate(
                [&](float l, int i) -> u64 { return l == key && (l > old || (l == old && i <= old_index)); },
                [&](u64) { return n - 1; }, total);
        } else if (key == old) {
            cut_index = old_index;
        }
    };

    if (top == -CUDART_INF_F || greedy) {
        u64 total;
        const int i = locate([&](float l, int) -> u64 { return l == top && l > -CUDART_INF_F; },
                             [](u64) { return 0ull; }, total);
        if (rank == 0 && tid == 0) {
            a.tokens[row] = i;
            if (a.logprob) a.logprob[row] = i < 0 ? -CUDART_INF_F : 0.0f;
        }
        return;  // the last cluster.sync is behind every access of another CTA's memory
    }
    const int top_k = a.top_k ? a.top_k[row] : 0;
    if (top_k > 0 && top_k < a.vocab) {
        u64 tokens;
        const float none = -CUDART_INF_F;
        locate([&](float l, int) -> u64 { return l > none; }, [](u64) { return ~0ull; }, tokens);
        // logits of language models lie within 64 of their largest
        if ((u64)top_k < tokens) narrow([](float) -> u64 { return 1; }, (u64)top_k, 64.0f);
    }
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    if (top_p < 1.0f) {
        u64 all;
        locate([&](float l, int i) -> u64 { return kept(l, i) ? weight(l) : 0; }, [](u64) { return ~0ull; }, all);
        const double want = ceil((double)top_p * (double)all);
        // weights end 2^-(S + 1) below the largest
        narrow(weight, want >= 1.0 ? (u64)want : 1ull, fminf(fmaxf(32.0f * temperature, 1e-30f), 1e30f));
    }
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const u64 least = min_p > 0.0f ? (u64)ceil(fmin((double)min_p, 1.0) * (double)(1ull << S)) : 0ull;
    const double u = (double)a.uniform[row];
    u64 total;
    const int token = locate(
        [&](float l, int i) -> u64 {
            if (!kept(l, i)) return 0;
            const u64 w = weight(l);
            return w >= least ? w : 0;
        },
        [&](u64 all) {
            // the first running sum above floor(u total) is the first above u total
            const u64 t = u > 0.0 ? (u64)fmin(u * (double)all, 9e18) : 0ull;
            return t < all ? t : all - 1;
        },
        total);
    if (rank == 0 && tid == 0) {
        a.tokens[row] = token;
        if (a.logprob) {
            const float l = to_float<T>(static_cast<const T*>(a.logits)[row * a.ld + token]);
            const double x = l == top ? 0.0 : ((double)l - (double)top) / (double)temperature;
            a.logprob[row] = (float)(x - log((double)total / (double)(1ull << S)));
        }
    }
}

template <typename T>
cudaError_t launch(const SampleArgs& a, cudaStream_t s) {
    static std::once_flag once;
    static cudaError_t attr = cudaSuccess;
    auto kernel = sample_kernel<T>;
    constexpr int kMost = (int)sizeof(SampleShared) +
                          (kMaxSlice<T> + kStride - 1) / kStride * kStride * (int)sizeof(T);
    static_assert(kMost <= 227 * 1024, "shared memory of one CTA");
    std::call_once(once, [&] {
        attr = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (attr == cudaSuccess) attr = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (attr != cudaSuccess) return attr;
    // CTAs per row: as few as leave two CTAs to an SM (80 KB of logits each),
    // more while the rows leave SMs idle and a CTA has a step of its own
    int ranks = 1;
    while (ranks < kMaxCluster && (long long)ranks * (kSliceBytes / (int)sizeof(T)) < a.vocab) ranks *= 2;
    while (ranks < kMaxCluster && 2ll * ranks * a.rows <= sm_count() && ranks * kStride < a.vocab) ranks *= 2;
    const int slice = ((a.vocab + ranks - 1) / ranks + 7) / 8 * 8;  // whole 16-byte words
    if (slice > kMaxSlice<T>) return cudaErrorInvalidValue;
    int bits = 1;  // vocab < 2^bits
    while ((1ll << bits) <= a.vocab) ++bits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * ranks);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)((slice + kStride - 1) / kStride) * kStride * sizeof(T);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, 62 - bits, slice);
}

}  // namespace

cudaError_t sample(const SampleArgs& a, cudaStream_t s) {
    if (a.type == Q4K_TYPE_F32) return launch<float>(a, s);
    return a.type == Q4K_TYPE_F16 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
}

}  // namespace q4k
