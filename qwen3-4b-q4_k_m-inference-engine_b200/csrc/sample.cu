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
// vocabulary of ones in 62 bits (44 up to 2^18 tokens); a weight's rounding,
// 2^-(S+1) of the largest, moves the draw's boundaries by about 1e-12.
//
// No sorting: a row's threshold is found by histograms. A cluster of 1 to 16
// CTAs holds the row in shared memory, each CTA a slice, so that the logits
// are read from HBM once; the passes over them run from there, and only bins,
// totals and candidates cross the cluster. The first pass takes the maximum,
// the second 2048 equal bins of the distance to it: of counts (top-k) or of
// weights (top-p). The tokens down to the bin where the running total reaches
// what is wanted are the candidates. Up to kList of them (the usual case) are
// brought to one CTA, which ranks them by comparing all with all, applies the
// filters in turn and draws. With more of them, the crossing bin's are ranked
// that way, if they are kList at most, and the draw is made by one more pass
// where the logits are. Else the bin is cut into 2048 again, then by the keys'
// bits, 11 at a time, until equal logits are left, of which the lowest indexes
// are kept.
//
// Measured, rows of 151936 fp32 logits: 1 row with all filters 14.4 us, a chain of
// passes over 9496 logits a CTA and barriers of its cluster; 257 flat rows with
// top-p 0.9 (about 90000 tokens kept of each) 299 us: issue slots are 55% busy, of
// which the fp64 weights, worked out twice, are most, HBM 7%.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <cmath>

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
constexpr int kVec = 4;  // consecutive logits of a lane
constexpr int kStep = 32 * kVec;
constexpr int kList = kSampleThreads;
// Logits of one CTA: 80 KB of them, so that two CTAs fit an SM; 25088 fp32
// ones of a vocabulary of 400000 in 16 CTAs (one to an SM).
constexpr int kSliceBytes = 80 * 1024;
template <typename T>
constexpr int kMaxSlice = kSliceBytes / sizeof(T) > 25600 ? kSliceBytes / sizeof(T) : 25600;
constexpr int kTable = 64;
constexpr int kCopies = 4;  // a slice's copies, each of a quarter of the warps' stretches

// Whole numbers in the order of the floats.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);  // -0 and 0 are ties
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^(j/64), from the host.
struct ExpTable {
    double v[kTable];
};

struct Crossing {
    u64 above, inside, all;  // the total above the bin, in it, and of every bin
    int bin;
};

struct alignas(16) SampleShared {
    uint32_t lo[kBins], hi[kBins];  // a histogram of 64-bit sums
    u64 list_key[kList];            // candidates: key, then the complement of the index
    u64 list_w[kList];
    double table[kTable];           // 2^(j/64)
    u64 warp_sum[kSampleWarps];
    u64 total[kMaxCluster];  // one word from every CTA of the cluster
    float bound[2][kMaxCluster];
    Crossing crossing;
    u64 last, chosen;
    int place, listed, members;
    uint64_t landed[kCopies];
};

// w(l) = round(2^(S + t)), t = (l - top) log2(e) / T, in fp64: l - top is exact,
// 64 t = i + r with i whole, 2^t = 2^(i/64) (the table, its exponent moved) times
// the Taylor polynomial of e^(r ln 2 / 64), |r| <= 1/2, whose fifth term is below
// 4e-14. Whole numbers are split off by adding 1.5 2^52 and w is read from the
// mantissa after adding 2^52 (w < 2^45): conversion instructions would cost
// more than all the arithmetic.
struct Weights {
    float top, c, cutoff;
    double top64, c64;  // 64 log2(e) / T
    int S;
    const double* table;

    __device__ __forceinline__ u64 operator()(float l) const {
        constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52
        const double d = (double)l - top64;
        const double z = fma(d, c64, kWhole);
        const double r = fma(d, c64, kWhole - z);
        constexpr double k = 0.693147180559945309417 / 64.0;
        double p = fma(r, k * k * k * k / 24.0, k * k * k / 6.0);
        p = fma(p, r, k * k / 2.0);
        p = fma(p, r, k);
        p = fma(p, r, 1.0);
        const int i = __double2loint(z);
        const double v = table[i & 63];
        const double w = p * __hiloint2double(__double2hiint(v) + (((i >> 6) + S) << 20), __double2loint(v));
        const u64 n = (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
        // a select, not a branch: four of these run side by side
        return (l - top) * c > cutoff ? n : 0;
    }
};

// All CTAs of the cluster have started once each has arrived: only then may one
// touch another's shared memory.
__device__ __forceinline__ void cluster_started_arrive() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_started_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2)
    sample_kernel(const __grid_constant__ SampleArgs a, const __grid_constant__ ExpTable table, int S, int slice) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
    T* held = reinterpret_cast<T*>(smem + sizeof(SampleShared));
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = min(rank * slice, a.vocab);  // this CTA's logits: base .. base + count - 1
    const int count = min(slice, a.vocab - base);
    const T* src = static_cast<const T*>(a.logits) + row * a.ld + base;

    cluster_started_arrive();
    // The slice into shared memory: bulk copies where rows start on 16-byte
    // words, all in flight at once.
    const int stretch = slice / kSampleWarps;  // a warp's logits, a multiple of 8
    if (tid == 0) {
        for (int i = 0; i < kCopies; ++i) mbar_init(&sh.landed[i], 1);
        mbar_fence_init();
    }
    __syncthreads();
    const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0;
    constexpr int kWide = 16 / sizeof(T);
    const int copied = aligned ? count / kWide * kWide : 0;
    if (tid == 0) {
        const int part = slice / kCopies;
        for (int i = 0; i < kCopies; ++i) {
            const int n = min(max(copied - i * part, 0), part);
            mbar_arrive_expect_tx(&sh.landed[i], n * (int)sizeof(T));
            if (n > 0) bulk_g2s(held + i * part, src + i * part, n * (int)sizeof(T), &sh.landed[i]);
        }
    }
    if (tid < kTable) sh.table[tid] = table.v[tid];
#pragma unroll 4
    for (int i = copied + tid; i < count; i += kSampleThreads) held[i] = src[i];
    // what lies behind the vocabulary is never drawn
    for (int i = count + tid; i < slice; i += kSampleThreads) held[i] = from_float<T>(-CUDART_INF_F);

    // f(logits, index of the first) for all of the CTA's logits, kVec at a time;
    // a warp's are consecutive, so that its sums are of one stretch of the
    // index order
    auto for_each = [&](auto&& f) {
        for (int s = lane * kVec; s < stretch; s += kStep) {
            const int at = warp * stretch + s;
            T v[kVec];
            if constexpr (sizeof(T) == 4)
                *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(held + at);
            else
                *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(held + at);
            float l[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) l[j] = to_float<T>(v[j]);
            f(l, base + at);
        }
    };
    __syncthreads();
    const bool lost = !mbar_wait_bounded(&sh.landed[warp / (kSampleWarps / kCopies)], 0, nullptr, 0);
    float most = -CUDART_INF_F, least_logit = CUDART_INF_F;
    for_each([&](const float(&l)[kVec], int) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            most = fmaxf(most, l[j]);
            least_logit = fminf(least_logit, l[j] > -CUDART_INF_F ? l[j] : CUDART_INF_F);
        }
    });

    // The largest and smallest of a value over the cluster; NaN if any thread says `bad`.
    auto cluster_bounds = [&](float high, float low, bool bad = false) {
        high = warp_max(high);
        low = -warp_max(-low);
        bad = __syncthreads_or(bad);
        if (lane == 0) sh.warp_sum[warp] = (u64)__float_as_uint(low) << 32 | __float_as_uint(high);
        __syncthreads();
        if (tid < ranks) {
            for (int w = 0; w < kSampleWarps; ++w) {
                high = fmaxf(high, __uint_as_float((uint32_t)sh.warp_sum[w]));
                low = fminf(low, __uint_as_float((uint32_t)(sh.warp_sum[w] >> 32)));
            }
            float* to = cluster.map_shared_rank(&sh.bound[0][0], tid);
            to[rank] = bad ? CUDART_NAN_F : high;
            to[kMaxCluster + rank] = low;
        }
        cluster.sync();
        for (int r = 0; r < ranks; ++r) {
            bad |= sh.bound[0][r] != sh.bound[0][r];
            high = fmaxf(high, sh.bound[0][r]);
            low = fminf(low, sh.bound[1][r]);
        }
        return make_float2(bad ? CUDART_NAN_F : high, low);
    };
    cluster_started_wait();
    const float2 extent = cluster_bounds(most, least_logit, lost);
    float top = extent.x;
    if (top != top) {  // a part of the row has not arrived, here or in another CTA
        for (int i = 0; i < kCopies; ++i) mbar_wait_bounded(&sh.landed[i], 0, nullptr, 0);
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprob) a.logprob[row] = CUDART_NAN_F;
        }
        return;
    }
    if (top == CUDART_INF_F) {
        // infinite logits share the row: as equal finite ones
        for (int i = tid; i < slice; i += kSampleThreads)
            held[i] = from_float<T>(to_float<T>(held[i]) == CUDART_INF_F ? 0.0f : -CUDART_INF_F);
        top = 0.0f;
        __syncthreads();
    }

    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    // (a temperature below 1e-37 would make 0 / T of the top itself NaN)
    const double c = 1.44269504088896340736 / (double)(greedy ? 1.0f : fmaxf(temperature, 1e-37f));
    const Weights weight = {top, (float)c, -(float)S - 1.0f, (double)top, 64.0 * c, S, sh.table};

    // kept: logits above cut, and those equal to it up to index cut_index
    float cut = -CUDART_INF_F;
    int cut_index = -1;
    auto kept = [&](float l, int i) { return l > cut || (l == cut && i <= cut_index); };

    auto clear = [&] {
        for (int i = tid; i < kBins; i += kSampleThreads) sh.lo[i] = sh.hi[i] = 0;
        __syncthreads();
    };
    auto add = [&](int bin, u64 v) {
        const uint32_t low = (uint32_t)v, old = atomicAdd(&sh.lo[bin], low);
        const uint32_t high = (uint32_t)(v >> 32) + (old + low < old);
        if (high) atomicAdd(&sh.hi[bin], high);
    };
    auto warp_total = [&](u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    auto warp_scan = [&](u64 v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        return v;
    };
    auto block_total = [&](u64 v) {
        v = warp_total(v);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = v;
        __syncthreads();
        v = 0;
        for (int w = 0; w < kSampleWarps; ++w) v += sh.warp_sum[w];
        return v;
    };
    // Of the cluster's histograms together: the bin where the running total,
    // from `above`, first reaches want(total of all bins). Each CTA adds up a
    // share of the bins.
    auto cross = [&](u64 above, auto&& wanted) {
        cluster.sync();
        const int per = kBins / ranks, q = (per + kSampleThreads - 1) / kSampleThreads;
        u64 mine[kBins / kSampleThreads], sum = 0;
#pragma unroll
        for (int j = 0; j < kBins / kSampleThreads; ++j) {
            mine[j] = 0;
            if (j < q && tid * q + j < per) {
                const int bin = rank * per + tid * q + j;
                // eight CTAs' loads at a time
                for (int r0 = 0; r0 < ranks; r0 += 8) {
                    uint32_t low[8], high[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        low[r] = r0 + r < ranks ? cluster.map_shared_rank(sh.lo, r0 + r)[bin] : 0;
                        high[r] = r0 + r < ranks ? cluster.map_shared_rank(sh.hi, r0 + r)[bin] : 0;
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) mine[j] += ((u64)high[r] << 32) + low[r];
                }
                sum += mine[j];
            }
        }
        const u64 run = warp_scan(sum);
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = run;
        __syncthreads();
        u64 before = above + run - sum, all = 0;
        for (int w = 0; w < kSampleWarps; ++w) {
            if (w < warp) before += sh.warp_sum[w];
            all += sh.warp_sum[w];
        }
        if (tid < ranks) cluster.map_shared_rank(sh.total, tid)[rank] = all;
        cluster.sync();
        all = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r < rank) before += sh.total[r];
            all += sh.total[r];
        }
        const u64 want = wanted(all);
        if (before < want && want <= before + sum) {
#pragma unroll
            for (int j = 0; j < kBins / kSampleThreads; ++j) {
                if (before < want && want <= before + mine[j]) {
                    const Crossing found = {before, mine[j], all, rank * per + tid * q + j};
                    for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&sh.crossing, r) = found;
                }
                before += mine[j];
            }
        }
        cluster.sync();
        return sh.crossing;
    };
    // found(index, logit, total) for the first logit, in index order, at which
    // the running sum of value(logit), over the row's logits with in(logit,
    // index), exceeds target(total).
    auto locate = [&](auto&& in, auto&& value, auto&& target, auto&& found) {
        u64 mine = 0;
        for_each([&](const float(&l)[kVec], int i) {
            bool is_in[kVec], any = false;
#pragma unroll
            for (int j = 0; j < kVec; ++j) any |= is_in[j] = in(l[j], i + j);
            if (!any) return;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const u64 v = value(l[j]);
                mine += is_in[j] ? v : 0;
            }
        });
        mine = warp_total(mine);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = mine;
        __syncthreads();
        u64 before = 0, all = 0;
        for (int w = 0; w < kSampleWarps; ++w) {
            if (w < warp) before += sh.warp_sum[w];
            all += sh.warp_sum[w];
        }
        if (tid < ranks) cluster.map_shared_rank(sh.total, tid)[rank] = all;
        cluster.sync();
        u64 total = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r < rank) before += sh.total[r];
            total += sh.total[r];
        }
        const u64 goal = target(total);
        // `before` is the sum before this CTA from here on
        for (int w = 0; w < warp; ++w) before -= sh.warp_sum[w];
        if (before <= goal && goal < before + all) {
            // the stretch, then all threads over it: a few consecutive logits each
            u64 at = goal - before;
            int owner = 0;
            while (at >= sh.warp_sum[owner]) at -= sh.warp_sum[owner++];
            __syncthreads();  // the sums are read: they are written again below
            constexpr int kEach = (kMaxSlice<T> / kSampleWarps + kSampleThreads - 1) / kSampleThreads;
            const int each = (stretch + kSampleThreads - 1) / kSampleThreads;
            const int i0 = owner * stretch + tid * each;
            u64 v[kEach], sum = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const bool there = j < each && tid * each + j < stretch;
                const float l = to_float<T>(held[there ? i0 + j : 0]);
                v[j] = there && in(l, base + i0 + j) ? value(l) : 0;
                sum += v[j];
            }
            u64 run = warp_scan(sum);
            if (lane == 31) sh.warp_sum[warp] = run;
            __syncthreads();
            for (int w = 0; w < warp; ++w) run += sh.warp_sum[w];
            run -= sum;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                if (run <= at && at < run + v[j]) found(base + i0 + j, to_float<T>(held[i0 + j]), total);
                run += v[j];
            }
        }
    };
    // the same, its index known to every CTA of the cluster
    auto locate_all = [&](auto&& in, auto&& value, auto&& target) {
        locate(in, value, target, [&](int i, float, u64) {
            for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&sh.place, r) = i;
        });
        cluster.sync();
        return sh.place;
    };

    const double u = (double)a.uniform[row];
    // the first running sum above floor(u total) is the first above u total
    auto goal_of = [&](u64 all) {
        const u64 t = u > 0.0 ? (u64)fmin(u * (double)all, 9e18) : 0ull;
        return t < all ? t : all - 1;
    };
    auto answer = [&](int token, float l, u64 total) {
        a.tokens[row] = token;
        if (a.logprob) {
            const double x = ((double)l - (double)top) / (double)fmaxf(temperature, 1e-37f);
            a.logprob[row] = token < 0 ? -CUDART_INF_F : (float)(x - log((double)total / (double)(1ull << S)));
        }
    };

    if (top == -CUDART_INF_F || greedy) {
        if (rank == 0 && tid == 0 && top == -CUDART_INF_F) answer(-1, top, 0);
        locate([&](float l, int) { return l == top && l > -CUDART_INF_F; }, [](float) { return 1ull; },
               [](u64) { return 0ull; }, [&](int i, float l, u64) { answer(i, l, 1ull << S); });
        return;  // the last cluster.sync is behind every access of another CTA's memory
    }
    int top_k = a.top_k ? a.top_k[row] : 0;
    if (top_k <= 0 || top_k > a.vocab) top_k = a.vocab;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    const bool by_weight = top_p < 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const u64 least = min_p > 0.0f ? (u64)ceil(fmin((double)min_p, 1.0) * (double)(1ull << S)) : 0ull;
    auto share_of = [&](u64 all) {
        const double want = ceil((double)top_p * (double)all);
        return want >= 1.0 ? (u64)want : 1ull;
    };
    // distances from the top that the first bins resolve: the row's extent (the
    // more bins its logits fall into, the fewer atomics meet), but logits of
    // language models lie within 64 of their largest, where masks need not;
    // weights end 2^-(S+1) below theirs
    const float span = fminf(fmaxf(top - extent.y, 1e-30f), 1e30f);
    const float count_range = fminf(span, 64.0f),
                weight_range = fminf(span, fmaxf(32.0f * temperature, 1e-30f));

    // the distance from the top in bins, and the nearest whole number of one below 2^22
    auto distance = [&](float l, float scale) { return fminf((top - l) * scale, (float)(kBins - 1)); };
    auto whole = [](float x) { return (int)(__float_as_uint(x + 8388608.0f) & 0x3fffffu); };
    auto bin_in = [&](float l, float scale) { return whole(distance(l, scale)); };

    // The first bins: of counts where top_k cuts, else of weights
    const bool counting = top_k < a.vocab;
    Crossing first = {0, 0, 0, kBins - 1};
    bool narrowed = false;  // the first filter's cut has been found
    const float first_scale = (float)kBins / (counting ? count_range : weight_range);
    if (counting || by_weight) {
        clear();
        if (counting)
            for_each([&](const float(&l)[kVec], int) {
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (l[j] > -CUDART_INF_F) atomicAdd(&sh.lo[bin_in(l[j], first_scale)], 1u);
            });
        else
            for_each([&](const float(&l)[kVec], int) {
                u64 w[kVec];
#pragma unroll
                for (int j = 0; j < kVec; ++j) w[j] = weight(l[j]);
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (w[j]) add(bin_in(l[j], first_scale), w[j]);
            });
        if (tid == 0) sh.listed = sh.members = sh.place = 0;
        // fewer tokens than top_k: the last of them ends the prefix
        first = cross(0, [&](u64 all) { return counting ? min((u64)top_k, all) : share_of(all); });
        // To CTA 0: the candidates if they are few, else those of the last bin.
        // How many there are the counts have told; under weights it takes a pass,
        // which brings the last bin's on the way.
        auto send = [&](u64* list, int* counter, float l, int i) {
            const int n = atomicAdd(cluster.map_shared_rank(counter, 0), 1);
            if (n < kList) cluster.map_shared_rank(list, 0)[n] = (u64)key_of(l) << 32 | (uint32_t)~i;
        };
        u64* const member = reinterpret_cast<u64*>(sh.lo);  // the histogram's place
        u64 n = first.above + first.inside;
        if (!counting) {
            u64 mine = 0;
            for_each([&](const float(&l)[kVec], int i) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const int bin = bin_in(l[j], first_scale);
                    const bool in = bin <= first.bin && l[j] > -CUDART_INF_F;
                    mine += in;
                    // (one too many tells of an overflow as well as all of them)
                    if (in && bin == first.bin && *reinterpret_cast<volatile int*>(&sh.place) <= kList &&
                        atomicAdd(&sh.place, 1) <= kList)
                        send(member, &sh.members, l[j], i + j);
                }
            });
            mine = block_total(mine);
            if (tid < ranks) cluster.map_shared_rank(sh.total, tid)[rank] = mine;
            cluster.sync();
            n = 0;
            for (int r = 0; r < ranks; ++r) n += sh.total[r];
        }
        if (n <= kList || (counting && first.inside <= kList)) {
            const bool all = n <= kList;
            for_each([&](const float(&l)[kVec], int i) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const int bin = bin_in(l[j], first_scale);
                    if ((all ? bin <= first.bin : bin == first.bin) && l[j] > -CUDART_INF_F) {
                        if (all)
                            send(sh.list_key, &sh.listed, l[j], i + j);
                        else
                            send(member, &sh.members, l[j], i + j);
                    }
                }
            });
            cluster.sync();
        }
        if (n <= kList) {
            if (rank != 0) return;
            const u64 key = tid < (int)n ? sh.list_key[tid] : 0;
            const float l = logit_of((uint32_t)(key >> 32));
            const int index = (int)~(uint32_t)key;
            u64 w = tid < (int)n ? weight(l) : 0;
            sh.list_w[tid] = w;
            __syncthreads();
            // rank and weight of those before it
            int ahead = 0;
            u64 ahead_w = 0;
            const int listed = (int)n;
            if (tid < listed)
#pragma unroll 4
                for (int j = 0; j < listed; ++j)
                    if (sh.list_key[j] > key) {
                        ++ahead;
                        ahead_w += sh.list_w[j];
                    }
            if (ahead >= top_k) w = 0;
            const u64 all = counting ? block_total(w) : first.all;
            if ((by_weight && ahead_w >= share_of(all)) || w < least) w = 0;
            const u64 total = block_total(w);  // its barriers end the loop above
            sh.list_w[tid] = w;
            __syncthreads();
            const u64 goal = goal_of(total);
            if (w) {
                u64 run = 0;
#pragma unroll 4
                for (int j = 0; j < listed; ++j)
                    if ((uint32_t)sh.list_key[j] > (uint32_t)key) run += sh.list_w[j];  // lower indexes
                if (run <= goal && goal < run + w) answer(index, l, total);
            }
            return;
        }
        const int members = counting ? (int)min(first.inside, (u64)kList + 1) : *cluster.map_shared_rank(&sh.members, 0);
        if (members <= kList) {
            // the last one to keep, found in one CTA and told to all
            if (rank == 0) {
                const u64 key = tid < members ? member[tid] : 0;
                const float l = logit_of((uint32_t)(key >> 32));
                const u64 w = tid >= members ? 0 : counting ? 1 : weight(l);
                // kSampleThreads parts of the bin, then all with all within the part
                // where the total passes
                const float edge = (float)first.bin - 0.5f;
                const int part = whole(fminf(fmaxf((distance(l, first_scale) - edge) * (float)kSampleThreads, 0.0f),
                                             (float)(kSampleThreads - 1)));
                __syncthreads();
                clear();
                if (w) add(part, w);
                if (tid == 0) sh.listed = 0;
                __syncthreads();
                const u64 mine_w = ((u64)sh.hi[tid] << 32) + sh.lo[tid];
                u64 run = warp_scan(mine_w);
                if (lane == 31) sh.warp_sum[warp] = run;
                __syncthreads();
                for (int i = 0; i < warp; ++i) run += sh.warp_sum[i];
                run += first.above - mine_w;
                const u64 want = counting ? min((u64)top_k, first.all) : share_of(first.all);
                if (run < want && want <= run + mine_w) {
                    sh.place = tid;
                    sh.last = run;
                }
                __syncthreads();
                const bool passing = w && part == sh.place;
                u64 ahead = sh.last;
                if (passing) {
                    const int n = atomicAdd(&sh.listed, 1);
                    sh.list_key[n] = key;
                    sh.list_w[n] = w;
                }
                __syncthreads();
                if (passing)
                    for (int j = 0; j < sh.listed; ++j)
                        if (sh.list_key[j] > key) ahead += sh.list_w[j];
                if (passing && ahead < want && want <= ahead + w)
                    for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&sh.chosen, r) = key;
            }
            cluster.sync();
            cut = logit_of((uint32_t)(sh.chosen >> 32));
            cut_index = (int)~(uint32_t)sh.chosen;
            narrowed = true;
        }
    }

    // Moves the cut to the shortest prefix of the kept that has wanted(total)
    // of value(logit); x: the crossing of the first bins.
    auto narrow = [&](auto&& value, Crossing x, float scale, u64 want) {
        const int bin = x.bin;
        const float low_edge = (float)bin - 0.5f;
        auto fine = [&](float l) {
            return whole(fminf(fmaxf((distance(l, scale) - low_edge) * (float)kBins, 0.0f), (float)(kBins - 1)));
        };
        auto level = [&](u64) { return want; };
        // the bin's ends (sub < 0), or those of its finer bin `sub`
        int sub = -1;
        auto among = [&](float l, int i) { return bin_in(l, scale) == bin && (sub < 0 || fine(l) == sub) && kept(l, i); };
        auto ends_of = [&] {
            float high = -CUDART_INF_F, low = CUDART_INF_F;
            for_each([&](const float(&l)[kVec], int i) {
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (among(l[j], i + j)) high = fmaxf(high, l[j]), low = fminf(low, l[j]);
            });
            __syncthreads();
            cluster.sync();  // the last bounds have been read
            return cluster_bounds(high, low);
        };
        float2 ends = ends_of();
        if (ends.x != ends.y) {
            clear();
            for_each([&](const float(&l)[kVec], int i) {
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (among(l[j], i + j)) add(fine(l[j]), value(l[j]));
            });
            x = cross(x.above, level);
            sub = x.bin;
            ends = ends_of();
        }
        float key = ends.x;
        if (ends.x != ends.y) {
            uint32_t prefix = 0;
#pragma unroll 1
            for (int step = 0; step < 3; ++step) {
                const int down = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
                const uint32_t mask = (1u << bits) - 1u;
                clear();
                for_each([&](const float(&l)[kVec], int i) {
#pragma unroll 1
                    for (int j = 0; j < kVec; ++j) {
                        if (!among(l[j], i + j)) continue;
                        const uint32_t k = key_of(l[j]);
                        if (step == 0 || k >> (down + bits) == prefix)
                            add((int)(mask - (k >> down & mask)), value(l[j]));
                    }
                });
                x = cross(x.above, level);
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
            cut_index = locate_all(
                [&](float l, int i) { return l == key && (key > old || (key == old && i <= old_index)); },
                [](float) { return 1ull; }, [&](u64) { return n - 1; });
        } else if (key == old) {
            cut_index = old_index;
        }
    };
    if (counting) {
        if (!narrowed) narrow([](float) -> u64 { return 1; }, first, first_scale, min((u64)top_k, first.all));
        if (by_weight) {
            const float scale = (float)kBins / weight_range;
            clear();
            for_each([&](const float(&l)[kVec], int i) {
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (kept(l[j], i + j)) add(bin_in(l[j], scale), weight(l[j]));
            });
            first = cross(0, share_of);
            narrow(weight, first, scale, share_of(first.all));
        }
    } else if (by_weight && !narrowed) {
        narrow(weight, first, first_scale, share_of(first.all));
    }
    locate(
        kept,
        [&](float l) {
            const u64 w = weight(l);
            return w >= least ? w : 0ull;
        },
        goal_of, answer);
}

template <typename T>
cudaError_t launch(const SampleArgs& a, cudaStream_t s) {
    auto kernel = sample_kernel<T>;
    constexpr int kMost = (int)sizeof(SampleShared) + kMaxSlice<T> * (int)sizeof(T);
    static_assert(kMost <= 227 * 1024, "shared memory of one CTA");
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = allow_shared(kernel, kMost, allowed, true);
    if (e != cudaSuccess) return e;
    // CTAs per row: as few as hold it two to an SM, then twice as many while they
    // take half of the SMs at most (beyond that the clusters do not all fit at
    // once: 9 rows of 32000 17.5 us in clusters of 8, 20.9 in 16; 18 rows of them
    // 20.8 in 4, 32.2 in 16) and a CTA has 2048 logits of its own (1 row of 4000
    // 14.9 us, 17.9 if 8192 are asked for)
    int ranks = 1;
    while (ranks < kMaxCluster && (long long)ranks * (kSliceBytes / (int)sizeof(T)) < a.vocab) ranks *= 2;
    while (ranks < kMaxCluster && 4ll * ranks * a.rows <= sm_count() && ranks * 2048 < a.vocab) ranks *= 2;
    constexpr int kUnit = 8 * kSampleWarps;  // whole 16-byte words, for every warp
    const int slice = (a.vocab + ranks * kUnit - 1) / (ranks * kUnit) * kUnit;
    if (slice > kMaxSlice<T>) return cudaErrorInvalidValue;
    int bits = 18;  // vocab < 2^bits
    while ((1ll << bits) <= a.vocab) ++bits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * ranks);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)slice * sizeof(T);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ExpTable table;
    for (int j = 0; j < kTable; ++j) table.v[j] = std::exp2(j / (double)kTable);
    return cudaLaunchKernelEx(&cfg, kernel, a, table, 62 - bits, slice);
}

}  // namespace

cudaError_t sample(const SampleArgs& a, cudaStream_t s) {
    if (a.type == Q4K_TYPE_F32) return launch<float>(a, s);
    return a.type == Q4K_TYPE_F16 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
}

}  // namespace q4k
