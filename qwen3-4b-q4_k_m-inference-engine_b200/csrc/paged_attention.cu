// q4k_paged_attention: causal grouped-query attention of a batch's new tokens
// over the pages of their sequences. Per query row,
//   s_k = scale q . k,  o = sum_k e^(s_k - m) v_k / l,  l = sum_k e^(s_k - m),
//   lse = m + log l,    m = max_k s_k,
// over the keys k <= p (the row's position) of its sequence's cached tokens,
// with a window of w also k > p - w. A row with no key gets o = 0, lse = -inf.
#include <math_constants.h>

#include "ops.h"
#include "paged_plan.cuh"
#include "paged_tc.cuh"

namespace q4k {
namespace {

using namespace paged_dev;

enum class Kind { kF32, kF16, kBf16 };

constexpr int kTileRows = 256;  // two MMA tiles of 128 query rows
constexpr int kBlockKeys = 128;
constexpr int kSoftmaxWarps = 16;  // two warpgroups per MMA tile, a thread per row and half of its keys
constexpr int kTcThreads = (kSoftmaxWarps + 3) * 32;  // and a TMA, an MMA and a piece-walking warp
// A tile's queries and outputs take about as long as 4 of its blocks (chunk of 512
// at 4096: 87.0 us with 2 to 4, 89.6 with 6; longer prompts the same with 2 to 6),
// and a share is at least that.
constexpr int kTileCost = 4;
constexpr int kMinUnits = 4;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
// The reference point of a row's exponentials moves only when its maximum
// has grown by more than 2^8: probabilities stay below 256, far inside
// fp16, and the accumulator is rescaled a few times per row instead of at
// every block.
constexpr float kLazy = 8.0f;
// fp16 probabilities are kept 2^7 times larger, at most 2^15: fp16 ends at
// 2^-24, so that one of 2^-32 of the row's largest still has its low part.
template <Kind K>
constexpr float kBias = K == Kind::kBf16 ? 0.0f : 7.0f;
// The tensor cores truncate their fp32 sums: each MMA takes on average half a
// last place, kTruncation of the sum so far (2^-24 of the mean of 1 / mantissa),
// off O, and addends are truncated too (values of one sign lose 1.7 times as much):
// 7e-6 after 4500 keys, 6e-4 after 131072. So O leaves TMEM every kFlush blocks for
// a sum in the workspace: 128 MMAs for fp32 activations, who are also given back
// kTruncation of it (2.5e-6 left for values of mean and spread 1, whatever the
// context), 1024 for 16-bit ones, whose outputs' rounding hides the 3e-5 left.
constexpr float kTruncation = 0.7213f / 16777216.0f;
template <Kind K>
constexpr int kFlush = K == Kind::kF32 ? 8 : 64;

template <Kind K>
struct Types {
    using Act = __half;
};
template <>
struct Types<Kind::kF32> {
    using Act = float;
};
template <>
struct Types<Kind::kBf16> {
    using Act = __nv_bfloat16;
};

// A piece as the softmax warps need it, written by a warp that walks ahead of
// them: the walk's state and divisions take none of their registers and time.
struct PieceInfo {
    int count;  // blocks; 0: no more pieces
    int first_row, position, row0, rows;  // the tile's query rows: of the batch, of the sequence
    int h;
    int begin, key_first, key_end;  // first key of the piece; keys that any row sees
    int all_first, all_last;        // keys that every row sees
    // Keys with values that are not finite, of those that only some rows see: bit
    // i of [0] is key_first + i (below all_first), of [1] all_last + 1 + i. A tile
    // has kTileRows tokens at most, so that neither has as many bits.
    uint32_t poison[2][kTileRows / 32];
    int poisoned;                   // there are such keys
    int twin;                       // tile 0: where tile 1's info is (-1: it has no rows)
    int whole, slot;                // slot: which of the CTA's two partial sums
    JoinNote note;
};

struct TcBars {
    uint64_t full[6], empty[6];
    uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], done;
    uint64_t piece_full[2][2], piece_empty[2][2];
    uint32_t tmem;
    int dead;
    Share share;
    int run[2][128];  // per row of each tile: what its two threads tell each other
    PieceInfo piece[2][2];  // per tile, in turn
};
constexpr int kBarBytes = 1024 + 896;
static_assert(sizeof(TcBars) <= kBarBytes, "barrier area");

// Shared memory: Q (per MMA tile: the fp16 high and, for fp32 activations,
// low parts; 64-dim halves of 128 rows x 128 bytes), the ring of K and V
// blocks in the same layout, and where Q is too small for them the outputs on
// their way out (4 KB a softmax warp).
template <Kind K, int D>
struct Layout {
    static constexpr int kParts = K == Kind::kF32 ? 2 : 1;  // of Q
    static constexpr int kHalf = 128 * 128;
    static constexpr int kMat = D / 64 * kHalf;  // 128 rows of D 16-bit values
    static constexpr int kStages = D == 64 ? 6 : K == Kind::kF32 ? 3 : 5;
    static constexpr int kRing = 2 * kParts * kMat;
    static constexpr bool kOutInQ = kParts * kMat >= 8 * 4096;
    static constexpr int kOut = kOutInQ ? 0 : kRing + kStages * kMat;
    static constexpr int kOutTile = kOutInQ ? kParts * kMat : 8 * 4096;
    static constexpr int kBars = kRing + kStages * kMat + (kOutInQ ? 0 : 2 * kOutTile);
    static constexpr int kBytes = kBars + kBarBytes + 1024;  // alignment slack
    static_assert(kBytes <= 227 * 1024, "shared memory of one CTA");
};

// The workspace: a note per CTA and piece, then per CTA and piece the rows'
// (m, l) and unnormalised outputs.
struct Partials {
    JoinNote* notes;  // [ctas][2]
    float2* ml;        // [ctas][2][kTileRows]
    float* o;          // [ctas][2][kTileRows][D]
    float4* flushed;   // [ctas][D / 4][kTileRows]: sums over a long piece
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <Kind K>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (K == Kind::kBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Whether 8 16-bit values are all finite: none has an exponent of ones.
template <Kind K>
__device__ __forceinline__ bool finite16(uint4 v) {
    constexpr uint32_t kExp = K == Kind::kBf16 ? 0x7f807f80u : 0x7c007c00u;
    // a half's exponent bits are all set where their complement is 0
    auto hit = [](uint32_t w) { return __vcmpeq2(w & kExp, kExp); };
    return (hit(v.x) | hit(v.y) | hit(v.z) | hit(v.w)) == 0;
}

// hi, lo: 16-bit parts of (a, b); hi + lo is within 2^-22 of each (bf16: 2^-16).
template <Kind K>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2<K>(a, b);
    if constexpr (K == Kind::kBf16) {
        lo = pack2<K>(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        lo = pack2<K>(a - f.x, b - f.y);
    }
}

// The power of two, as two factors, that brings a row of largest magnitude
// `most` to below 2^8 (any fp32 row then fits fp16 parts), and c divided by it:
// at least the smallest normal number, whose products with scores, below 2^31,
// are 0 to the exponential as well, and which leaves masked scores at -infinity.
__device__ __forceinline__ void row_scale(float most, float c, float& f1, float& f2, float& c_out) {
    const int e = min(max((int)(__float_as_uint(most) >> 23) - 126, -100), 127);  // most < 2^e
    const int e1 = (8 - e) / 2, e2 = 8 - e - e1;
    f1 = __uint_as_float((uint32_t)(127 + e1) << 23);
    f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
    c_out = fmaxf(c * __uint_as_float((uint32_t)(127 - e1) << 23) * __uint_as_float((uint32_t)(127 - e2) << 23),
                  1.17549435e-38f);
}

// Signed whole numbers in the order of the floats.
__device__ __forceinline__ int ordered(float v) {
    const int b = __float_as_int(v);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// ---------------------------------------------------------------------------
// Many query rows (prompt chunks): bound by the tensor cores (6 x 512 cycles per
// block of 256 rows x 128 keys x 128 dims; fp32 activations 8 x 512) and the
// exponentials (2048 cycles at 16 per cycle and SM). One MMA-issuing thread
// alternates between two tiles of 128 rows, so that one tile's products run under
// the other's softmax: S = Q K^T from shared memory into TMEM, probabilities back
// over S as 16-bit high and low parts, O += P V with P from TMEM, the first half
// of the products under the second half of their own exponentials (bf16 prompt of
// 8192: 739 us, 766 with all after them). High parts alone would take 524 us, but
// leave 16-bit outputs 1.4 times the error of their own rounding. Two threads share a row, each
// with half of a block's keys and half of the row's output: with one thread to
// a row the two warps of an SM sub-partition could not hide their own latencies
// (2300 cycles for a softmax of 1024 cycles of exponentials). Measured: 8192
// bf16 tokens of 32 / 8 heads of 128 in 720 to 790 us by the clocks of the moment
// (853 in sustained calls), 730 TFLOP/s of 1100 in the products; tensor pipe 54%,
// exponentials 36%, issue 43% busy: the latencies of a tile's softmax between its
// own products, and the power limit.
// ---------------------------------------------------------------------------
template <Kind K, int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_attention_tc_kernel(const __grid_constant__ PagedAttentionArgs a, const __grid_constant__ CUtensorMap kmap,
                              const __grid_constant__ CUtensorMap vmap, const Partials part) {
    using L = Layout<K, D>;
    using Act = typename Types<K>::Act;
    using Walk = Pieces<kTileRows, kBlockKeys, kTileCost>;
    constexpr int kStages = L::kStages;
    constexpr uint32_t kIdescS = idesc_f16(K == Kind::kBf16, 128, kBlockKeys, false);
    constexpr uint32_t kIdescO = idesc_f16(K == Kind::kBf16, 128, D, true);
    // TMEM columns: S (its probabilities written over it: of 32 of them 16 columns
    // of high parts, two to a column, then 16 of low parts) and O of each MMA tile
    constexpr uint32_t kS = 0, kO = 256, kPStep = 32;
    constexpr int kTmaWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1, kWalkWarp = kSoftmaxWarps + 2;

    extern __shared__ __align__(1024) uint8_t smem_dyn[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    TcBars& bar = *reinterpret_cast<TcBars*>(smem + L::kBars);
    volatile int* dead = &bar.dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.heads / a.cache.kv_heads;
    const int held = a.batch.table_width << a.cache.page_shift;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bar.full[i], 1);
            mbar_init(&bar.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.q_full[i], kSoftmaxWarps / 2);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i][0], kSoftmaxWarps / 2);
            mbar_init(&bar.p_full[i][1], kSoftmaxWarps / 2);
            mbar_init(&bar.o_full[i], 1);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&bar.piece_full[i][j], 1);
                mbar_init(&bar.piece_empty[i][j], kSoftmaxWarps / 2);
            }
        }
        mbar_init(&bar.done, 1);
        bar.dead = 0;
        mbar_fence_init();
    }
    if (warp == kMmaWarp) tmem_alloc(&bar.tmem, 512);
    tc_fence_before();
    plan_share<kTileRows, kBlockKeys, kTileCost>(a.batch, group, a.cache.kv_heads, a.window, held, kMinUnits,
                                                 reinterpret_cast<unsigned long long*>(smem + L::kRing), &bar.share);
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    fence_proxy_async();  // the plan's words, before the ring's copies land on them
    __syncthreads();

    // The walking and the softmax warps go through all pieces even after a wait has
    // given up, as their rows have to be written: a piece then takes 2 s at most.
    auto piece_wait = [&](uint64_t* b, uint32_t parity) {
        bool ok = false;
        for (int i = 0; i < 4 && !ok; ++i) ok = mbar_wait_bounded(b, parity, nullptr, 0);
        return ok;
    };

    if (warp == kTmaWarp) {
        // ---------------- TMA: K and V blocks, page by page, a lane per (page, half)
        Walk pc(a.batch, group, a.cache.kv_heads, a.window, held, bar.share);
        const int box = min(a.cache.page_size, kBlockKeys);
        const int boxes = kBlockKeys / box;
        const int page_in_block = lane / (D / 64), half = lane % (D / 64);
        const uint32_t box_bytes = (uint32_t)box * D * 2;
        int n = 0;
        bool ok = true;
        for (; pc.valid() && ok; pc.next()) {
            const int* const table = a.batch.page_table + (size_t)pc.s * a.batch.table_stride;
            auto page_of = [&](int key) {  // of this lane's box of the block
                key += page_in_block * box;
                return page_in_block < boxes && key < pc.tile.key_end ? __ldg(table + (key >> a.cache.page_shift)) : -1;
            };
            int next_page = page_of(pc.tile.key_begin + pc.b * kBlockKeys);
            for (int i = 0; i < pc.count && ok; ++i) {
                const int key0 = pc.tile.key_begin + (pc.b + i) * kBlockKeys;
                const int live = min(max((pc.tile.key_end - key0 + box - 1) / box, 0), boxes);
                const int page = next_page;
                if (i + 1 < pc.count) next_page = page_of(key0 + kBlockKeys);  // a block ahead
                for (int kv = 0; kv < 2 && ok; ++kv, ++n) {
                    const int st = n % kStages;
                    // (once a wait has given up no stage is filled again: one whose copy is
                    // missing may have been given back in that copy's phase)
                    ok = wait_or_dead(&bar.empty[st], ((n / kStages) & 1) ^ 1, dead) && !*dead;
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&bar.full[st], live * box_bytes);
                    __syncwarp();
                    if (page_in_block < live)
                        tma_load_4d(smem + L::kRing + st * L::kMat + half * L::kHalf + page_in_block * box * 128,
                                    kv ? &vmap : &kmap, half * 64, key0 & (a.cache.page_size - 1), pc.h, page,
                                    &bar.full[st]);
                }
            }
        }
        // every copy issued has landed before the CTA can exit
        for (int i = max(n - kStages, 0); i < n; ++i)
            mbar_wait_bounded(&bar.full[i % kStages], (i / kStages) & 1, nullptr, 0);
        __syncwarp();
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            // ---------------- MMA issue
            Walk pc(a.batch, group, a.cache.kv_heads, a.window, held, bar.share);
            int n = 0;
            uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
            bool ok = true;
            const uint32_t ring = smem_addr(smem + L::kRing);
            const uint64_t q_desc = desc_k_major(smem_addr(smem)), k_desc = desc_k_major(ring);
            const uint64_t v_desc = desc_mn_major(ring, L::kHalf);
            auto wait_stage = [&](int i) { return wait_or_dead(&bar.full[i % kStages], (i / kStages) & 1, dead); };
            auto score = [&](int t, int stage) {
                const uint64_t k = k_desc + (stage % kStages) * (L::kMat >> 4);
                // the low parts first, while the sum is small: each MMA truncates it
                uint64_t q = q_desc + (t + 1) * L::kParts * (L::kMat >> 4);
#pragma unroll
                for (int pt = 0; pt < L::kParts; ++pt) {
                    q -= L::kMat >> 4;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((kk / 4) * L::kHalf + (kk % 4) * 32) >> 4;
                        mma_ss(tmem + kS + 128 * t, q + off, k + off, kIdescS, (pt | kk) != 0);
                    }
                }
                tc_commit(&bar.s_full[t]);
            };
            // O += P V over the first or second 32 of each thread's 64 keys
            auto value = [&](int t, int stage, int part, bool accumulate) {
                const uint64_t v = v_desc + (stage % kStages) * (L::kMat >> 4) + 2 * part * (2048 >> 4);
                const uint32_t p = tmem + kS + 128 * t + kPStep * part;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                        for (int pt = 0; pt < 2; ++pt)
                            mma_ts(tmem + kO + 128 * t, p + 2 * kPStep * h + 16 * pt + 8 * kk,
                                   v + (4 * h + kk) * (2048 >> 4), kIdescO, accumulate || (pt | kk | h) != 0);
            };
            for (; pc.valid() && ok; pc.next()) {
                const int tiles = pc.tile.rows > 128 ? 2 : 1;
                int k_stage = n++;
                ok = wait_stage(k_stage);
                for (int t = 0; t < tiles && ok; ++t) {
                    ok = wait_or_dead(&bar.q_full[t], q_phase[t]++ & 1, dead);
                    if (!ok) break;
                    tc_fence_after();
                    score(t, k_stage);
                }
                tc_commit(&bar.empty[k_stage % kStages]);
                for (int i = 0; i < pc.count && ok; ++i) {
                    const bool more = i + 1 < pc.count;
                    const int v_stage = n++;
                    if (more) k_stage = n++;
                    for (int t = 0; t < tiles && ok; ++t) {
                        const uint32_t phase = p_phase[t]++ & 1;
                        // Either part waits for both threads of every row: each MMA
                        // reads and writes all of O's columns, and either thread may
                        // have rescaled its half of them before its first part
                        ok = wait_stage(v_stage);
                        for (int part = 0; part < 2 && ok; ++part) {
                            ok = wait_or_dead(&bar.p_full[t][part], phase, dead);
                            if (!ok) break;
                            tc_fence_after();
                            value(t, v_stage, part, i % kFlush<K> > 0 || part > 0);
                        }
                        if (!ok) break;
                        if (more) {
                            ok = wait_stage(k_stage);
                            if (!ok) break;
                            tc_fence_after();
                            score(t, k_stage);
                        } else {
                            tc_commit(&bar.o_full[t]);
                        }
                    }
                    tc_commit(&bar.empty[v_stage % kStages]);
                    if (more) tc_commit(&bar.empty[k_stage % kStages]);
                }
            }
        }
        __syncwarp();
    } else if (warp == kWalkWarp) {
        if (lane == 0) {
            // ---------------- the pieces, for the softmax warps of each tile; a count of 0 ends them
            Walk pc(a.batch, group, a.cache.kv_heads, a.window, held, bar.share);
            uint32_t turn[2] = {0, 0};
            bool ok = true;
            for (bool more = true; more && ok; pc.next()) {
                more = pc.valid();
                // (tile 1's first: tile 0's warps write into it)
                for (int t = 1; t >= 0 && ok; --t) {
                    if (more && pc.tile.rows <= 128 * t) continue;
                    const uint32_t slot = turn[t] & 1;
                    ok = piece_wait(&bar.piece_empty[t][slot], (turn[t] >> 1 & 1) ^ 1);
                    if (!ok) break;
                    ++turn[t];
                    PieceInfo& pi = bar.piece[t][slot];
                    pi.count = more ? pc.count : 0;
                    pi.first_row = pc.seq.first_row;
                    pi.position = pc.seq.position;
                    pi.row0 = pc.tile.row0 + 128 * t;
                    pi.rows = pc.tile.rows - 128 * t;
                    pi.h = pc.h;
                    pi.begin = pc.tile.key_begin + pc.b * kBlockKeys;
                    pi.key_first = pc.tile.key_first;
                    pi.key_end = pc.tile.key_end;
                    pi.all_first = pc.tile.all_first;
                    pi.all_last = pc.tile.all_last;
                    for (int i = 0; i < 2 * kTileRows / 32; ++i) (&pi.poison[0][0])[i] = 0;
                    pi.poisoned = 0;
                    pi.twin = pc.tile.rows > 128 ? (int)(turn[1] - 1 & 1) : -1;
                    pi.whole = pc.whole();
                    pi.slot = pc.index > 0;
                    pi.note = note_of(pc);
                    mbar_arrive(&bar.piece_full[t][slot]);
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------- softmax: MMA tile t, half h of a block's keys, a thread per query row
        const int t = warp >> 3, h = warp >> 2 & 1, quad = warp & 3, row = 32 * quad + lane;
        const int pair_barrier = 1 + 4 * t + quad, tile_barrier = 9 + t;
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        const uint32_t s_addr = tmem + kS + 128 * t + lanes, o_addr = tmem + kO + 128 * t + lanes + h * (D / 2);
        int* run = &bar.run[t][row];  // the row's largest score so far, ordered()
        uint8_t* const qs = smem + t * L::kParts * L::kMat;
        uint8_t* const out_stage =
            smem + (L::kOutInQ ? t * L::kParts * L::kMat : L::kOut + t * L::kOutTile) + (warp & 7) * 4096;
        int n = 1;  // ring number of the block's V
        uint32_t phase = 0;
        int left = 0;  // bit i: partial sum i has been left
        // (a wait that gives up is not acted on within a piece: every warp goes
        // through the same barriers, and once one wait has given up the others
        // return at once; the rows of that piece and of later ones become NaN)
        for (uint32_t items = 0;; ++items) {
            PieceInfo& pi = bar.piece[t][items & 1];
            const bool there = piece_wait(&bar.piece_full[t][items & 1], items >> 1 & 1);
            // and the last piece's outputs have left the shared memory
            if (named_barrier_or(tile_barrier, 256, !there)) break;
            const int count = pi.count;
            if (count == 0) break;
            const int r = pi.row0 + row;
            float c = a.scale * kLog2e;
            {
                // Q into shared memory, 16 rows a warp, whole rows at a time
                constexpr int kChunks = D * (int)sizeof(Act) / 16;  // 16-byte words of a row
                constexpr int kAtOnce = 32 / kChunks;               // rows of one load
                constexpr int kBatch = 4;                           // loads in flight
                static_assert(16 % (kBatch * kAtOnce) == 0, "whole passes");
                const int chunk = lane % kChunks;
                // where the warp's rows are: lanes 0 .. 15 know theirs (null: past the tile)
                const int r0 = 16 * (warp & 7), rq = pi.row0 + r0 + (lane & 15);
                const Act* q = static_cast<const Act*>(a.q) + ((size_t)pi.first_row + rq / group) * a.ld_q +
                               (size_t)(pi.h * group + rq % group) * D;
                const unsigned long long mine =
                    r0 + (lane & 15) < pi.rows ? reinterpret_cast<unsigned long long>(q) : 0ull;
#pragma unroll 1
                for (int it = 0; it < 16; it += kBatch * kAtOnce) {
                    uint4 x[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const unsigned long long from =
                            __shfl_sync(0xffffffffu, mine, it + j * kAtOnce + lane / kChunks);
                        x[j] = make_uint4(0u, 0u, 0u, 0u);
                        if (from) x[j] = __ldg(reinterpret_cast<const uint4*>(from) + chunk);
                    }
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const int rr = r0 + it + j * kAtOnce + lane / kChunks;
                        if constexpr (K == Kind::kF32) {
                            // scaled by a power of two to below 2^8, as high and low parts
                            float v[4] = {__uint_as_float(x[j].x), __uint_as_float(x[j].y), __uint_as_float(x[j].z),
                                          __uint_as_float(x[j].w)};
                            float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
                            for (int o = kChunks / 2; o > 0; o >>= 1)
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                            float f1, f2, row_c;
                            row_scale(most, c, f1, f2, row_c);
                            uint2 hi, lo;
                            split2<K>(v[0] * f1 * f2, v[1] * f1 * f2, hi.x, lo.x);
                            split2<K>(v[2] * f1 * f2, v[3] * f1 * f2, hi.y, lo.y);
                            uint8_t* at = qs + (chunk >> 4) * L::kHalf + swz128(rr, chunk >> 1 & 7) + (chunk & 1) * 8;
                            *reinterpret_cast<uint2*>(at) = hi;
                            *reinterpret_cast<uint2*>(at + L::kMat) = lo;
                            if (chunk == 0) bar.run[t][rr] = __float_as_int(row_c);
                        } else {
                            *reinterpret_cast<uint4*>(qs + (chunk >> 3) * L::kHalf + swz128(rr, chunk & 7)) = x[j];
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.q_full[t]);
                if constexpr (K == Kind::kF32) {
                    named_barrier(tile_barrier, 256);
                    c = __int_as_float(*run);
                    named_barrier(pair_barrier, 64);
                }
                if (h == 0) *run = ordered(-CUDART_INF_F);
                named_barrier(pair_barrier, 64);
            }
            // keys this row sees, from this thread's first key of the piece on
            const int position = pi.position + r / group;
            int hi = (row < pi.rows ? min(position, held - 1) : -1) - pi.begin - 64 * h;
            int lo = (a.window > 0 ? max(position - a.window + 1, 0) : 0) - pi.begin - 64 * h;
            float m = -CUDART_INF_F, l = 0.0f;
            // sums since the last flush of O are l and steps, those before it
            // l_flushed, its reference point m_flushed
            // (16-bit: l is of all blocks)
            constexpr bool kBack = K == Kind::kF32;
            float steps = 0.0f, l_flushed = 0.0f, m_flushed = -CUDART_INF_F;
            float4* const flushed = part.flushed + ((size_t)blockIdx.x * (D / 4) + h * (D / 8)) * kTileRows + 128 * t + row;
            // The sums so far being O l' / l, with l' the row's sum then, the 16 MMAs
            // of a block have taken 16 kTruncation sum(l') / l of O.
            auto give_back = [&] { return kBack && l > 0.0f ? 1.0f + 16.0f * kTruncation * steps / l : 1.0f; };
            auto flushed_factor = [&] { return m_flushed == m ? 1.0f : exp2_fast(m_flushed - m); };
            for (int i = 0; i < count; ++i, ++phase, hi -= kBlockKeys, lo -= kBlockKeys) {
                if (t == 0 && h == 0) {
                    const int key0 = pi.begin + i * kBlockKeys;
                    if (key0 < pi.all_first || key0 + kBlockKeys - 1 > pi.all_last) {
                        // V holds keys that some rows do not see, whose 0 times
                        // what is not finite would not be 0. What no row sees (it may
                        // never have been loaded) becomes zeros. A row of V that
                        // is not finite becomes zeros too, and the rows that see it
                        // NaN at the end.
                        const int v_stage = n + 2 * i;
                        wait_or_dead(&bar.full[v_stage % kStages], (v_stage / kStages) & 1, dead);
                        const int key = key0 + row;
                        uint8_t* v = smem + L::kRing + (v_stage % kStages) * L::kMat;
                        bool clear = key < pi.key_first || key >= pi.key_end;
                        if (!clear && (key < pi.all_first || key > pi.all_last)) {
#pragma unroll 4
                            for (int j = 0; j < D / 8; ++j)
                                clear |= !finite16<K>(*reinterpret_cast<const uint4*>(v + (j >> 3) * L::kHalf +
                                                                                      swz128(row, j & 7)));
                            if (clear) {
                                const int side = key > pi.all_last;
                                const int bit = key - (side ? pi.all_last + 1 : pi.key_first);
                                auto note = [&](PieceInfo& info) {
                                    atomicOr(&info.poison[side][bit >> 5], 1u << (bit & 31));
                                    info.poisoned = 1;
                                };
                                note(pi);
                                if (pi.twin >= 0) note(bar.piece[1][pi.twin]);
                            }
                        }
                        if (clear)
#pragma unroll 4
                            for (int j = 0; j < D / 8; ++j)
                                *reinterpret_cast<uint4*>(v + (j >> 3) * L::kHalf + swz128(row, j & 7)) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        fence_proxy_async();
                    }
                }
                wait_or_dead(&bar.s_full[t], phase & 1, dead);
                __syncwarp();
                tc_fence_after();
                bool fresh = i == 0;  // O begins anew with this block
                if (i > 0 && i % kFlush<K> == 0) {
                    // the score MMAs of this block were committed after the last
                    // block's value MMAs: O is at rest
                    const float back = give_back(), f = i == kFlush<K> ? 0.0f : flushed_factor();
#pragma unroll 1
                    for (int j = 0; j < D / 2; j += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + j, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            float4* const at = flushed + (size_t)((j + e) / 4) * kTileRows;
                            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (i > kFlush<K>) v = *at;
                            v.x = fmaf(v.x, f, back * __uint_as_float(o[e]));
                            v.y = fmaf(v.y, f, back * __uint_as_float(o[e + 1]));
                            v.z = fmaf(v.z, f, back * __uint_as_float(o[e + 2]));
                            v.w = fmaf(v.w, f, back * __uint_as_float(o[e + 3]));
                            *at = v;
                        }
                    }
                    m_flushed = m;
                    if (kBack) {
                        l_flushed += l;
                        l = steps = 0.0f;
                    }
                    fresh = true;
                }
                uint32_t s[2][32];
                tmem_ld32(s_addr + 64 * h, s[0]);
                tmem_ld32(s_addr + 64 * h + 32, s[1]);
                tmem_wait_ld();
                if (__any_sync(0xffffffffu, hi < 63 || lo > 0)) {
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (j < lo || j > hi) s[j >> 5][j & 31] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) mx[j] = __uint_as_float(s[j >> 1][16 * (j & 1)]);
#pragma unroll
                for (int e = 1; e < 15; e += 2)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mx[j] = max3(mx[j], __uint_as_float(s[j >> 1][16 * (j & 1) + e]),
                                     __uint_as_float(s[j >> 1][16 * (j & 1) + e + 1]));
#pragma unroll
                for (int j = 0; j < 4; ++j) mx[j] = fmaxf(mx[j], __uint_as_float(s[j >> 1][16 * (j & 1) + 15]));
                // both halves' largest, and so far
                atomicMax(run, ordered(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c));
                named_barrier(pair_barrier, 64);
                const float top = from_ordered(*reinterpret_cast<volatile int*>(run));
                if (__any_sync(0xffffffffu, top > m + kLazy)) {
                    const float mn = top > m + kLazy ? top : m;
                    const float f = mn == m ? 1.0f : exp2_fast(m - mn);
                    if (kBack) l_flushed *= f;
                    if (!kBack || !fresh) l *= f;
                    if (!fresh) {
                        if (kBack) steps *= f;
                        // (at rest, as above)
#pragma unroll 1
                        for (int j = 0; j < D / 16; j += 2) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + 8 * j, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(o_addr + 8 * j, o);
                        }
                    }
                    m = mn;
                }
                const float shift = m == -CUDART_INF_F ? 0.0f : m - kBias<K>;
                const uint64_t c2 = pack_f32x2(c, c), shift2 = pack_f32x2(-shift, -shift);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // 16 probabilities: 8 words of high and 8 of low parts
                    uint32_t w[8], low[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int at = 16 * (j & 1) + 2 * e;
                        const uint64_t x = fma_f32x2(
                            pack_f32x2(__uint_as_float(s[j >> 1][at]), __uint_as_float(s[j >> 1][at + 1])), c2, shift2);
                        float p0, p1;
                        unpack_f32x2(x, p0, p1);
                        p0 = exp2_fast(p0);
                        p1 = exp2_fast(p1);
                        sum[e & 1] = add_f32x2(sum[e & 1], pack_f32x2(p0, p1));
                        split2<K>(p0, p1, w[e], low[e]);
                    }
                    const uint32_t col = s_addr + kPStep * (2 * h + (j >> 1)) + 8 * (j & 1);
                    tmem_st8(col, w);
                    tmem_st8(col + 16, low);
                    if (j == 1) {  // half of them: their products run under the other half's exponentials
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.p_full[t][0]);
                    }
                }
                float sum0, sum1;
                unpack_f32x2(add_f32x2(sum[0], sum[1]), sum0, sum1);
                if (kBack) steps += fmaf(0.5f, sum0 + sum1, l);
                l += sum0 + sum1;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.p_full[t][1]);
            }
            wait_or_dead(&bar.o_full[t], items & 1, dead);
            __syncwarp();
            tc_fence_after();
            n += 2 * count;
            const float back = give_back();
            const bool was_flushed = count > kFlush<K>;
            const float before = was_flushed ? flushed_factor() : 0.0f;
            if (kBack) l += l_flushed;
            // the row's sum, from both halves
            if (h == 1) *run = __float_as_int(l);
            named_barrier(pair_barrier, 64);
            if (h == 0) {
                l += __int_as_float(*run);
                *run = __float_as_int(l);
            }
            named_barrier(pair_barrier, 64);
            const bool lost = *dead != 0;
            l = lost ? CUDART_NAN_F : __int_as_float(*run);
            const bool whole = pi.whole;
            const size_t slot = ((size_t)blockIdx.x * 2 + pi.slot) * kTileRows + 128 * t;
            const float inv = whole ? (l > 0.0f ? 1.0f / l : 0.0f) : 1.0f;
            const bool none = whole && !(l != 0.0f);
            bool poisoned = lost;
            if (pi.poisoned) {
                const int oldest = a.window > 0 ? max(position - a.window + 1, 0) : 0;
#pragma unroll 1
                for (int i = 0; i < 2 * kTileRows / 32; ++i) {
                    const int word = i % (kTileRows / 32), side = i / (kTileRows / 32);
                    const int key = (side ? pi.all_last + 1 : pi.key_first) + 32 * word;  // of the word's first bit
                    const int from = max(oldest - key, 0), to = min(position - key, 31);
                    if (from <= to) poisoned |= (pi.poison[side][word] >> from << from & 0xffffffffu >> (31 - to)) != 0;
                }
            }
            const int rows = pi.rows;
            const int head = pi.h * group + r % group;
            const size_t out_row = (size_t)pi.first_row + r / group;
            Act* const out = static_cast<Act*>(a.out) + out_row * a.ld_out + (size_t)head * D + h * (D / 2);
#pragma unroll 1
            for (int j = 0; j < D / 64; ++j) {
                uint32_t o[32];
                tmem_ld32(o_addr + 32 * j, o);
                tmem_wait_ld();
                if (kBack || was_flushed) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (was_flushed) v = flushed[(size_t)(8 * j + e / 4) * kTileRows];
                        o[e] = __float_as_uint(fmaf(v.x, before, back * __uint_as_float(o[e])));
                        o[e + 1] = __float_as_uint(fmaf(v.y, before, back * __uint_as_float(o[e + 1])));
                        o[e + 2] = __float_as_uint(fmaf(v.z, before, back * __uint_as_float(o[e + 2])));
                        o[e + 3] = __float_as_uint(fmaf(v.w, before, back * __uint_as_float(o[e + 3])));
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                if (poisoned)
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0x7fffffffu;
                // 32 columns of 32 rows, turned in shared memory so that rows are
                // written whole
                if (sizeof(Act) == 2 && whole) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        *reinterpret_cast<uint4*>(out_stage + lane * 64 + ((x ^ (lane >> 1 & 3)) << 4)) = make_uint4(
                            pack2<K>(__uint_as_float(o[8 * x]), __uint_as_float(o[8 * x + 1])),
                            pack2<K>(__uint_as_float(o[8 * x + 2]), __uint_as_float(o[8 * x + 3])),
                            pack2<K>(__uint_as_float(o[8 * x + 4]), __uint_as_float(o[8 * x + 5])),
                            pack2<K>(__uint_as_float(o[8 * x + 6]), __uint_as_float(o[8 * x + 7])));
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int rr = it * 8 + lane / 4, x = lane & 3;
                        const unsigned long long to = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), rr);
                        const uint4 v = *reinterpret_cast<const uint4*>(out_stage + rr * 64 + ((x ^ (rr >> 1 & 3)) << 4));
                        if (32 * quad + rr < rows) reinterpret_cast<uint4*>(to)[4 * j + x] = v;
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        *reinterpret_cast<uint4*>(out_stage + lane * 128 + ((x ^ (lane & 7)) << 4)) =
                            make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int rr = it * 4 + lane / 8, x = lane & 7;
                        unsigned long long to = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), rr);
                        if (!whole)
                            to = reinterpret_cast<unsigned long long>(part.o + (slot + 32 * quad + rr) * D + h * (D / 2));
                        const uint4 v = *reinterpret_cast<const uint4*>(out_stage + rr * 128 + ((x ^ (rr & 7)) << 4));
                        if (32 * quad + rr < rows) reinterpret_cast<uint4*>(to)[8 * j + x] = v;
                    }
                }
                __syncwarp();
            }
            if (h == 0 && row < rows) {
                if (!whole)
                    part.ml[slot + row] = make_float2(m - kBias<K>, l);
                else if (a.lse)
                    a.lse[out_row * a.heads + head] = none ? -CUDART_INF_F : (m - kBias<K> + log2f(l)) * kLn2;
            }
            if (!whole) {
                left |= 1 << pi.slot;
                if (tid == 0) part.notes[blockIdx.x * 2 + pi.slot] = pi.note;
            }
            // O has been read before the next piece's first value MMA
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.piece_empty[t][items & 1]);
        }
        if (tid == 0)
            for (int i = 0; i < 2; ++i)
                if (!(left >> i & 1)) part.notes[blockIdx.x * 2 + i] = {0, 0, 0, 0, 0};
    }
    pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        if (*dead && lane == 0) {  // the MMAs in flight end before the TMEM is freed
            tc_commit(&bar.done);
            mbar_wait_bounded(&bar.done, 0, nullptr, 0);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Few query rows per sequence and KV head (decode steps, draft tokens): the
// keys and values are read once from HBM and that bounds the call. A producer
// warp streams 64-key blocks (K and V) through a ring of shared memory; each
// of kWarps warps takes every kWarps-th block by itself (mma.sync m16n8k16,
// its own running maximum, sum and output), so no barrier stands in the loop,
// and the warps are joined once per piece. kWarps divides the ring's stages:
// all uses of a stage are one warp's, which therefore never waits on a stage
// whose phase before its own is still another's. Probabilities enter the products as
// 16-bit high and low parts, fp32 activations' queries too: in rows 0-7 and 8-15
// of one MMA tile when those are fp32 and 8 rows suffice, else in two MMAs.
// ---------------------------------------------------------------------------
constexpr int kDecodeKeys = 64;
// Shares of one block: 1 sequence of 500 in 11.1 us; of two 11.5, of four 14.0.
constexpr int kDecodeMinUnits = 1;
constexpr int kDecodeCost = 1;
// A warp's blocks between two drains of its outputs from the MMA's sums, which are
// truncated, to fp32 ones in shared memory (see kTruncation; 4 or 8 MMAs a block
// here): without them fp32 activations would lose 3e-5 over 32768 keys of values
// of mean and spread 1, and 1.3e-4 over 131072.
template <Kind K>
constexpr int kDrain = K == Kind::kF32 ? 8 : 64;

template <Kind K, int D, int ROWS>
struct DecodeLayout {
    static constexpr int kHalf = kDecodeKeys * 128;  // 64 dims of a block
    static constexpr int kMat = D / 64 * kHalf;
    static constexpr int kStage = 2 * kMat;
    static constexpr int kWarps = D == 64 || ROWS == 8 ? 6 : 5;
    static constexpr int kStages = D == 64 ? 2 * kWarps : kWarps;
    static constexpr int kThreads = (kWarps + 1) * 32;
    static_assert(kStages % kWarps == 0, "a stage belongs to one warp");
    static constexpr int kJoin = kStages * kStage;  // [kWarps][ROWS][D] floats, then (m, l)
    static constexpr int kBars = kJoin + kWarps * ROWS * (D + 2) * 4;
    static constexpr int kBytes = kBars + 512 + 1024;
    static_assert(kBytes <= 227 * 1024, "shared memory of one CTA");
};

struct DecodeBars {
    uint64_t full[12], empty[12];
    int dead;
    Share share;
};
static_assert(sizeof(DecodeBars) <= 512, "barrier area");

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <Kind K>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (K == Kind::kBf16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <Kind K, int D, int ROWS>
__global__ void __launch_bounds__((DecodeLayout<K, D, ROWS>::kThreads), 1)
    paged_attention_decode_kernel(const __grid_constant__ PagedAttentionArgs a, const __grid_constant__ CUtensorMap kmap,
                                  const __grid_constant__ CUtensorMap vmap, const Partials part) {
    using L = DecodeLayout<K, D, ROWS>;
    using Act = typename Types<K>::Act;
    constexpr int kStages = L::kStages, kWarps = L::kWarps;
    constexpr bool kStacked = ROWS == 8;           // fp32: low parts in rows 8-15
    constexpr bool kSplit = K == Kind::kF32;
    constexpr int kParts = kSplit && !kStacked ? 2 : 1;
    static_assert(!kStacked || kSplit, "16-bit rows take all 16 MMA rows");
    constexpr int kR = kStacked ? 1 : 2;  // query rows of a lane: g (and g + 8)

    extern __shared__ uint8_t smem_dyn[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    DecodeBars& bar = *reinterpret_cast<DecodeBars*>(smem + L::kBars);
    float* join_o = reinterpret_cast<float*>(smem + L::kJoin);
    float2* join_ml = reinterpret_cast<float2*>(join_o + kWarps * ROWS * D);
    volatile int* dead = &bar.dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.heads / a.cache.kv_heads;
    const int held = a.batch.table_width << a.cache.page_shift;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bar.full[i], 1);
            mbar_init(&bar.empty[i], 1);
        }
        bar.dead = 0;
        mbar_fence_init();
    }
    plan_share<ROWS, kDecodeKeys, kDecodeCost>(a.batch, group, a.cache.kv_heads, a.window, held, kDecodeMinUnits,
                                  reinterpret_cast<unsigned long long*>(smem), &bar.share);
    fence_proxy_async();  // the plan's words, before the ring's copies land on them
    __syncthreads();
    Pieces<ROWS, kDecodeKeys, kDecodeCost> pc(a.batch, group, a.cache.kv_heads, a.window, held, bar.share);

    if (warp == kWarps) {
        // ---------------- TMA: a lane per (K or V, page, half)
        const int box = min(a.cache.page_size, kDecodeKeys);
        const int boxes = kDecodeKeys / box;
        const int half = lane % (D / 64), kv = lane / (D / 64) & 1, page_in_block = lane / (D / 64 * 2);
        const uint32_t box_bytes = (uint32_t)box * D * 2 * 2;
        int n = 0;
        bool ok = true;
        for (; pc.valid() && ok; pc.next()) {
            const int* const table = a.batch.page_table + (size_t)pc.s * a.batch.table_stride;
            auto page_of = [&](int key) {  // of this lane's box of the block
                key += page_in_block * box;
                return page_in_block < boxes && key < pc.tile.key_end ? __ldg(table + (key >> a.cache.page_shift)) : -1;
            };
            // two blocks ahead
            int page = page_of(pc.tile.key_begin + pc.b * kDecodeKeys);
            int next_page = page_of(pc.tile.key_begin + (pc.b + 1) * kDecodeKeys);
            for (int i = 0; i < pc.count; ++i, ++n) {
                const int key0 = pc.tile.key_begin + (pc.b + i) * kDecodeKeys;
                const int live = min(max((pc.tile.key_end - key0 + box - 1) / box, 0), boxes);
                const int far_page = page_of(key0 + 2 * kDecodeKeys);
                const int st = n % kStages;
                ok = wait_or_dead(&bar.empty[st], ((n / kStages) & 1) ^ 1, dead);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&bar.full[st], live * box_bytes);
                __syncwarp();
                if (page_in_block < live)
                    tma_load_4d(smem + st * L::kStage + kv * L::kMat + half * L::kHalf + page_in_block * box * 128,
                                kv ? &vmap : &kmap, half * 64, key0 & (a.cache.page_size - 1), pc.h, page,
                                &bar.full[st]);
                page = next_page;
                next_page = far_page;
            }
        }
        for (int i = max(n - kStages, 0); i < n; ++i)
            mbar_wait_bounded(&bar.full[i % kStages], (i / kStages) & 1, nullptr, 0);
        __syncwarp();
    } else {
        // ---------------- attention
        const int g = lane >> 2, t = lane & 3;
        int n0 = 0;  // ring number of the piece's first block
        bool ok = true, left[2] = {false, false};
        for (; pc.valid(); pc.next()) {
            const Tile& tl = pc.tile;
            // Q: MMA A fragments of every 16-dim step; rows g and g + 8
            uint32_t qf[D / 16][kParts][4];
            float c[kR], m[kR], l[kR];
            int first[kR], last[kR];
#pragma unroll
            for (int y = 0; y < kR; ++y) {
                const int row = g + 8 * y;
                const bool live = row < tl.rows;
                const int r = tl.row0 + (live ? row : 0);
                const int token = r / group, head = pc.h * group + r % group;
                const int position = pc.seq.position + token;
                last[y] = live ? min(position, held - 1) : -1;
                first[y] = a.window > 0 ? max(position - a.window + 1, 0) : 0;
                c[y] = a.scale * kLog2e;
                m[y] = -CUDART_INF_F;
                l[y] = 0.0f;
                const Act* q = static_cast<const Act*>(a.q) + ((size_t)pc.seq.first_row + token) * a.ld_q + (size_t)head * D;
                if constexpr (kSplit) {
                    float2 x[D / 16][2];
                    float most = 0.0f;
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            x[s][e] = __ldg(reinterpret_cast<const float2*>(q + 16 * s + 8 * e + 2 * t));
                            most = fmaxf(most, fmaxf(fabsf(x[s][e].x), fabsf(x[s][e].y)));
                        }
                    float f1, f2;
                    row_scale(quad_max(most), c[y], f1, f2, c[y]);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t hi, lo;
                            split2<K>(x[s][e].x * f1 * f2, x[s][e].y * f1 * f2, hi, lo);
                            if constexpr (kStacked) {
                                qf[s][0][2 * e] = hi;
                                qf[s][0][2 * e + 1] = lo;
                            } else {
                                qf[s][0][2 * e + y] = hi;
                                qf[s][1][2 * e + y] = lo;
                            }
                        }
                } else {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            qf[s][0][2 * e + y] = __ldg(reinterpret_cast<const uint32_t*>(q + 16 * s + 8 * e + 2 * t));
                }
            }
            float o[D / 8][4];
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
            // o to the join area, onto what is there of this piece (its reference
            // point: m_drained)
            int undrained = 0;
            bool drained = false;
            float m_drained[kR];
            auto drain = [&] {
#pragma unroll
                for (int y = 0; y < kR; ++y) {
                    float* dst = join_o + (warp * ROWS + g + 8 * y) * D + 2 * t;
                    const float f = m_drained[y] == m[y] ? 1.0f : exp2_fast(m_drained[y] - m[y]);
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        float2 v;
                        if constexpr (kStacked)
                            v = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
                        else
                            v = make_float2(o[j][2 * y], o[j][2 * y + 1]);
                        if (drained) {
                            const float2 u = *reinterpret_cast<const float2*>(dst + 8 * j);
                            v = make_float2(fmaf(u.x, f, v.x), fmaf(u.y, f, v.y));
                        }
                        *reinterpret_cast<float2*>(dst + 8 * j) = v;
                    }
                    m_drained[y] = m[y];
                }
#pragma unroll
                for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
                drained = true;
            };
#pragma unroll
            for (int y = 0; y < kR; ++y) m_drained[y] = 0.0f;

            // this warp's blocks of the piece
            for (int i = (warp - n0 % kWarps + kWarps) % kWarps; i < pc.count && ok; i += kWarps) {
                const int n = n0 + i, st = n % kStages;
                ok = wait_or_dead(&bar.full[st], (n / kStages) & 1, dead);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                const int key0 = tl.key_begin + (pc.b + i) * kDecodeKeys;
                const uint32_t kbase = smem_addr(smem + st * L::kStage), vbase = kbase + L::kMat;
                // keys that some rows do not see: as in the other kernel, zeros for
                // what no row sees and for what is not finite, and NaN for the
                // rows that see the latter
                const bool edge = key0 < tl.all_first || key0 + kDecodeKeys - 1 > tl.all_last;
                bool nan[kR] = {};
                if (edge) {
                    uint8_t* v = smem + st * L::kStage + L::kMat;
                    for (int row = lane; row < kDecodeKeys; row += 32) {
                        const int key = key0 + row;
                        const bool unseen = key < tl.key_first || key >= tl.key_end;
                        bool poison = false;
                        if (!unseen && (key < tl.all_first || key > tl.all_last))
#pragma unroll 4
                            for (int j = 0; j < D / 8; ++j)
                                poison |= !finite16<K>(
                                    *reinterpret_cast<const uint4*>(v + (j >> 3) * L::kHalf + swz128(row, j & 7)));
                        if (unseen || poison)
#pragma unroll 4
                            for (int j = 0; j < D / 8; ++j)
                                *reinterpret_cast<uint4*>(v + (j >> 3) * L::kHalf + swz128(row, j & 7)) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        for (unsigned bad = __ballot_sync(0xffffffffu, poison); bad; bad &= bad - 1) {
                            const int bad_key = key - lane + __ffs(bad) - 1;
#pragma unroll
                            for (int y = 0; y < kR; ++y) nan[y] |= bad_key >= first[y] && bad_key <= last[y];
                        }
                    }
                    __syncwarp();
                }
                // S = Q K^T: scores of 8 keys at a time
                float s[kDecodeKeys / 8][2 * kR];
#pragma unroll
                for (int j = 0; j < kDecodeKeys / 8; ++j) {
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int d = 0; d < D / 16; d += 2) {
                        uint32_t b[4];
                        const int chunk = 2 * d + (lane >> 3);
                        ldsm_x4(kbase + (chunk >> 3) * L::kHalf + swz128(8 * j + (lane & 7), chunk & 7), b);
#pragma unroll
                        for (int p = 0; p < kParts; ++p) {
                            mma16816<K>(acc, qf[d][p], b[0], b[1]);
                            mma16816<K>(acc, qf[d + 1][p], b[2], b[3]);
                        }
                    }
                    if constexpr (kStacked) {
                        s[j][0] = acc[0] + acc[2];
                        s[j][1] = acc[1] + acc[3];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[j][e] = acc[e];
                    }
                }
                float top[kR];
#pragma unroll
                for (int y = 0; y < kR; ++y) {
                    const int lo = first[y] - key0 - 2 * t, hi = last[y] - key0 - 2 * t;
                    if (__any_sync(0xffffffffu, first[y] > key0 || last[y] < key0 + kDecodeKeys - 1)) {
#pragma unroll
                        for (int j = 0; j < kDecodeKeys / 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (8 * j + e < lo || 8 * j + e > hi) s[j][2 * y + e] = -CUDART_INF_F;
                    }
                    float mx = -CUDART_INF_F;
#pragma unroll
                    for (int j = 0; j < kDecodeKeys / 8; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * y], s[j][2 * y + 1]));
                    top[y] = quad_max(mx) * c[y];
                }
                bool moves = false;
#pragma unroll
                for (int y = 0; y < kR; ++y) moves |= top[y] > m[y] + kLazy;
                if (__any_sync(0xffffffffu, moves)) {
                    float f[kR];
#pragma unroll
                    for (int y = 0; y < kR; ++y) {
                        const float mn = top[y] > m[y] + kLazy ? top[y] : m[y];
                        f[y] = mn == m[y] ? 1.0f : exp2_fast(m[y] - mn);
                        l[y] *= f[y];
                        m[y] = mn;
                    }
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        o[j][0] *= f[0];
                        o[j][1] *= f[0];
                        o[j][2] *= f[kR - 1];
                        o[j][3] *= f[kR - 1];
                    }
                }
                // O += P V, 16 keys at a time: their probabilities go straight into
                // the A fragments, as 16-bit high and low parts (the products are
                // cheap here: 16-bit activations then only round their outputs)
                float shift[kR];
#pragma unroll
                for (int y = 0; y < kR; ++y) shift[y] = m[y] == -CUDART_INF_F ? 0.0f : m[y] - kBias<K>;
#pragma unroll
                for (int kk = 0; kk < kDecodeKeys / 16; ++kk) {
                    uint32_t pf[kStacked ? 1 : 2][4];
#pragma unroll
                    for (int y = 0; y < kR; ++y)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {  // keys 0-7 of the 16, keys 8-15
                            const float p0 = exp2_fast(fmaf(s[2 * kk + e][2 * y], c[y], -shift[y]));
                            const float p1 = exp2_fast(fmaf(s[2 * kk + e][2 * y + 1], c[y], -shift[y]));
                            l[y] += p0 + p1;  // this lane's keys; the quad's are added at the end
                            uint32_t hi, lo;
                            split2<K>(p0, p1, hi, lo);
                            if constexpr (kStacked) {
                                pf[0][2 * e] = hi;
                                pf[0][2 * e + 1] = lo;
                            } else {
                                pf[0][2 * e + y] = hi;
                                pf[1][2 * e + y] = lo;
                            }
                        }
#pragma unroll
                    for (int j = 0; j < D / 8; j += 2) {
                        uint32_t b[4];
                        const int row = 16 * kk + (lane & 15), chunk = j + (lane >> 4);
                        ldsm_x4_t(vbase + (chunk >> 3) * L::kHalf + swz128(row, chunk & 7), b);
#pragma unroll
                        for (int p = 0; p < (kStacked ? 1 : 2); ++p) {
                            mma16816<K>(o[j], pf[p], b[0], b[1]);
                            mma16816<K>(o[j + 1], pf[p], b[2], b[3]);
                        }
                    }
                }
                if (edge) {
                    fence_proxy_async();  // the zeros, before the next copy into this stage
#pragma unroll
                    for (int y = 0; y < kR; ++y)
                        if (nan[y])
#pragma unroll
                            for (int j = 0; j < D / 8; ++j) o[j][2 * y] = o[j][2 * y + 1] = __uint_as_float(0x7fffffffu);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.empty[st]);
                if (++undrained == kDrain<K>) {
                    drain();
                    undrained = 0;
                }
            }
            n0 += pc.count;

            // join the warps
            drain();
#pragma unroll
            for (int y = 0; y < kR; ++y) {
                const int row = g + 8 * y;
                l[y] = quad_sum(l[y]);
                if (t == 0) join_ml[warp * ROWS + row] = make_float2(m[y], l[y]);
            }
            // (once a wait has given up, this piece's rows and those of later ones are NaN)
            ok = !named_barrier_or(1, kWarps * 32, !ok);
            const bool whole = pc.whole();
            const size_t slot = ((size_t)blockIdx.x * 2 + (pc.index > 0)) * ROWS;
            for (int x = tid; x < tl.rows * (D / 4); x += kWarps * 32) {
                const int row = x / (D / 4), d = x % (D / 4) * 4;
                float mx = -CUDART_INF_F;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, join_ml[w * ROWS + row].x);
                float sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 ml = join_ml[w * ROWS + row];
                    if (!(ml.y != 0.0f)) continue;
                    const float f = exp2_fast(ml.x - mx);
                    const float4 u = *reinterpret_cast<const float4*>(join_o + (w * ROWS + row) * D + d);
                    sum += f * ml.y;
                    v[0] += f * u.x;
                    v[1] += f * u.y;
                    v[2] += f * u.z;
                    v[3] += f * u.w;
                }
                if (!ok) sum = CUDART_NAN_F;
                const int r = tl.row0 + row;
                const int head = pc.h * group + r % group;
                const size_t out_row = (size_t)pc.seq.first_row + r / group;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = sum != 0.0f ? v[e] / sum : 0.0f;
                    store_values<Act, 4>(static_cast<Act*>(a.out) + out_row * a.ld_out + (size_t)head * D + d, v);
                    if (d == 0 && a.lse)
                        a.lse[out_row * a.heads + head] = sum != 0.0f ? (mx - kBias<K> + log2f(sum)) * kLn2 : -CUDART_INF_F;
                } else {
                    store_values<float, 4>(part.o + (slot + row) * D + d, v);
                    if (d == 0) part.ml[slot + row] = make_float2(mx - kBias<K>, sum);
                }
            }
            if (!whole) {
                left[pc.index > 0] = true;
                if (tid == 0)
                    part.notes[blockIdx.x * 2 + (pc.index > 0)] = note_of(pc);
            }
            named_barrier(1, kWarps * 32);  // the join area may be written again
        }
        if (tid == 0)
            for (int i = 0; i < 2; ++i)
                if (!left[i]) part.notes[blockIdx.x * 2 + i] = {0, 0, 0, 0, 0};
    }
    pdl_launch_dependents();
}

// The tiles that several CTAs share: block c of this grid joins the tile that
// begins in CTA c's share and ends in a later one's, in the order of the CTAs.
// A row's pieces are spread over as many warps as the block's rows leave (a
// decode step over a long context: a few rows of dozens of pieces).
constexpr int kJoinWarps = 8;
// Rows of a block: 16 of a tile of 256 (chunk of 512 at 4096 86.9 us, with 64
// 94.6), 2 of a decode tile (2 sequences of 131071 56.7 us, with 8 59.0).
constexpr int kJoinRows = 16;
constexpr int kJoinDecodeRows = 2;
template <typename Act, int D, int kRows>
__global__ void __launch_bounds__(kJoinWarps * 32)
    paged_attention_join_kernel(const __grid_constant__ PagedAttentionArgs a, const Partials part, int rows_per_block) {
    constexpr int V = D / 32;
    __shared__ float sums[kJoinWarps][D + 1];
    pdl_wait();
    const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const JoinNote first = part.notes[2 * c0], second = part.notes[2 * c0 + 1];
    const int own = second.pieces > 0;
    const JoinNote n = own ? second : first;
    const int begin = blockIdx.y * rows_per_block, end = min(begin + rows_per_block, n.rows);
    if (n.pieces == 0 || begin >= end) return;
    int spread = 1;  // warps of a row
    while (2 * spread * (end - begin) <= kJoinWarps && 2 * spread <= n.pieces) spread *= 2;
    const int group = a.heads / a.cache.kv_heads;
    // where (piece, row) is in the workspace
    auto at = [&](int i, int row) { return ((size_t)2 * (c0 + i) + (i == 0 ? own : 0)) * kRows + row; };
    for (int row0 = begin; row0 < end; row0 += kJoinWarps / spread) {
        const int row = row0 + warp / spread, part_of = warp % spread;
        const bool live = row < end;
        float m = -CUDART_INF_F, l = 0.0f, o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.0f;
        if (live) {
            for (int i = lane; i < n.pieces; i += 32) m = fmaxf(m, part.ml[at(i, row)].x);
            m = warp_max(m);
#pragma unroll 4
            for (int i = part_of; i < n.pieces; i += spread) {
                const float2 ml = part.ml[at(i, row)];
                const float* src = part.o + at(i, row) * D + lane * V;
                float v[V];
                if constexpr (V == 4)
                    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
                else
                    *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
                const float f = ml.y != 0.0f ? exp2_fast(ml.x - m) : 0.0f;
                l += f * ml.y;
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] += f != 0.0f ? f * v[j] : 0.0f;
            }
        }
        if (spread > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = o[j];
            if (lane == 0) sums[warp][D] = l;
            __syncthreads();
            if (part_of == 0)
                for (int w = 1; w < spread; ++w) {
                    l += sums[warp + w][D];
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] += sums[warp + w][lane * V + j];
                }
        }
        if (!live || part_of) continue;
        const int r = n.row0 + row;
        const int head = n.head + r % group;
        const size_t out_row = (size_t)n.first_row + r / group;
        Act* out = static_cast<Act*>(a.out) + out_row * a.ld_out + (size_t)head * D + lane * V;
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = from_float<Act>(l != 0.0f ? o[j] / l : 0.0f);
        if (lane == 0 && a.lse)
            a.lse[out_row * a.heads + head] = l != 0.0f ? (m + log2f(l)) * kLn2 : -CUDART_INF_F;
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// K or V pages as (dim, row, head, page): boxes of 64 dims and up to `rows`
// rows of a page. A page number outside the cache reads as zeros.
bool page_map(const PagedCache& c, const uint16_t* base, int rows, CUtensorMap* map) {
    const EncodeTiled encode = reinterpret_cast<EncodeTiled>(tensor_map_encoder());
    if (!encode) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads,
                                (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.row_stride * 2, (cuuint64_t)c.head_stride * 2,
                                   (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(c.page_size < rows ? c.page_size : rows), 1, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return encode(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  const_cast<uint16_t*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t partial_bytes(int ctas, int rows, int head_dim) {
    const size_t partial = 32 + (size_t)rows * (sizeof(float2) + sizeof(float) * head_dim);
    const size_t flushed = rows == kTileRows ? (size_t)rows * sizeof(float) * head_dim : 0;
    return (size_t)ctas * (2 * partial + flushed);
}

Partials partials(void* workspace, int ctas, int rows, int head_dim) {
    static_assert(sizeof(JoinNote) <= 32, "notes");
    Partials p;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    p.notes = reinterpret_cast<JoinNote*>(w);
    p.ml = reinterpret_cast<float2*>(w + (size_t)ctas * 2 * 32);
    p.o = reinterpret_cast<float*>(w + (size_t)ctas * 2 * (32 + (size_t)rows * sizeof(float2)));
    p.flushed = reinterpret_cast<float4*>(p.o + (size_t)ctas * 2 * rows * head_dim);
    return p;
}

template <Kind K, int D>
cudaError_t launch_tc(const PagedAttentionArgs& a, cudaStream_t s) {
    using L = Layout<K, D>;
    auto kernel = paged_attention_tc_kernel<K, D>;
    static std::atomic<unsigned long long> allowed{0};
    cudaError_t e = allow_shared(kernel, L::kBytes, allowed);
    if (e != cudaSuccess) return e;
    CUtensorMap km, vm;
    if (!page_map(a.cache, a.cache.k, kBlockKeys, &km) || !page_map(a.cache, a.cache.v, kBlockKeys, &vm))
        return cudaErrorInvalidValue;
    const int ctas = sm_count();
    const Partials part = partials(a.workspace, ctas, kTileRows, D);
    kernel<<<ctas, kTcThreads, L::kBytes, s>>>(a, km, vm, part);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_pdl(paged_attention_join_kernel<typename Types<K>::Act, D, kTileRows>, dim3(ctas, kTileRows / kJoinRows),
                      dim3(kJoinWarps * 32), 0, s, a, part, kJoinRows);
}

template <Kind K, int D, int ROWS>
cudaError_t launch_decode(const PagedAttentionArgs& a, cudaStream_t s) {
    using L = DecodeLayout<K, D, ROWS>;
    auto kernel = paged_attention_decode_kernel<K, D, ROWS>;
    static std::atomic<unsigned long long> allowed{0};
    cudaError_t e = allow_shared(kernel, L::kBytes, allowed);
    if (e != cudaSuccess) return e;
    CUtensorMap km, vm;
    if (!page_map(a.cache, a.cache.k, kDecodeKeys, &km) || !page_map(a.cache, a.cache.v, kDecodeKeys, &vm))
        return cudaErrorInvalidValue;
    const int ctas = sm_count();
    const Partials part = partials(a.workspace, ctas, ROWS, D);
    kernel<<<ctas, L::kThreads, L::kBytes, s>>>(a, km, vm, part);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_pdl(paged_attention_join_kernel<typename Types<K>::Act, D, ROWS>, dim3(ctas, ROWS / kJoinDecodeRows),
                      dim3(kJoinWarps * 32), 0, s, a, part, kJoinDecodeRows);
}

// Which kernel, by the query rows per sequence and KV head. Up to the decode
// kernel's 16 MMA rows it is ahead everywhere (us, decode / chunk kernel, 32 and 8
// heads of 128: 1 sequence of 500 with 4 rows 10.8 / 25.0, 32 of 2000 53.8 / 125,
// with 16 rows 73.8 / 131, bf16 57.9 / 103 and 64.1 / 109, 2 of 131071 with 4 rows
// 160 / 402, bf16 169 / 323). Up to 32 rows it reads the keys twice, which it can
// afford with head_dim 64 (1 sequence of 131071 with 32 rows 93 / 176, 256 of 1000
// 260 / 374; bf16 90 / 163 and 219 / 328) and up to two tiles an SM, whatever the
// context. With 32 rows of 128 in bf16: 1 sequence of 500 14.0 / 21.8, of 32000 47 /
// 70, of 131071 173 / 179; 4 of 4000 30 / 40, of 32000 168 / 166, of 131071 627 / 649;
// 16 of 500 30.6 / 28.7, of 4000 100 / 104; 32 of 500 49 / 41, of 4000 181 / 181.
// fp32: 1 of 500 15.5 / 25.9, of 131071 195 / 221; 8 of 32000 358 / 400; 32 of 500
// 58 / 50, of 4000 211 / 223. With more tiles it is behind more often than ahead
// (64 of 1000 143 / 140, of 4000 398 / 415, 256 of 1000 524 / 453; bf16 116 / 119 and
// 419 / 385 at 1000).
constexpr int kDecodeRows = 16;

bool few_rows(const PagedAttentionArgs& a, long long rows) {
    const long long tiles = (long long)a.batch.sequences * a.cache.kv_heads;
    return rows <= kDecodeRows || (rows <= 2 * kDecodeRows &&
                                   (a.cache.head_dim == 64 || tiles <= 2 * sm_count()));
}

template <Kind K, int D>
cudaError_t launch_dim(const PagedAttentionArgs& a, cudaStream_t s) {
    const long long rows = (long long)a.batch.max_new * (a.heads / a.cache.kv_heads);
    if (!few_rows(a, rows)) return launch_tc<K, D>(a, s);
    // (fp32, 4 rows: 11.0 us against 13.0 with 16 rows at 1 sequence of 500, 58.6 against 69.0 at 32 of 2000)
    if constexpr (K == Kind::kF32)
        if (rows <= 8) return launch_decode<K, D, 8>(a, s);
    return launch_decode<K, D, 16>(a, s);
}

template <Kind K>
cudaError_t launch(const PagedAttentionArgs& a, cudaStream_t s) {
    return a.cache.head_dim == 128 ? launch_dim<K, 128>(a, s) : launch_dim<K, 64>(a, s);
}

}  // namespace

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int max_new) {
    const bool few = max_new > 0 && (long long)max_new * (heads / kv_heads) <= kDecodeRows;
    return partial_bytes(sm_count(), few ? kDecodeRows : kTileRows, head_dim);
}

cudaError_t paged_attention(const PagedAttentionArgs& a, cudaStream_t s) {
    if (a.f32) return launch<Kind::kF32>(a, s);
    return a.cache.bf16 ? launch<Kind::kBf16>(a, s) : launch<Kind::kF16>(a, s);
}

}  // namespace q4k
