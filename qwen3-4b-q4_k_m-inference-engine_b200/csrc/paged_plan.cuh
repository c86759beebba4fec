// How attention's work over a batch of sequences is cut: the same plan is
// worked out by every CTA from the lengths on the device, so that a captured
// launch follows them.
//
// A tile is kRows query rows (new token x query head of one KV head) of one
// sequence and KV head; its keys are cut into blocks of kBlock positions. The
// blocks of all tiles, in the order sequence, KV head, tile, block, are dealt
// out in contiguous shares of equal cost, one per CTA, a tile costing kCost
// blocks on top of its own (its queries and outputs): lengths of any
// raggedness keep every CTA busy, long contexts with few rows are split over
// many CTAs, and a CTA has at most two tiles that it shares with others (its
// first and its last). Those leave partial sums in the workspace, which a second kernel
// joins in the order of the CTAs.
#pragma once
#include "paged_device.cuh"

namespace q4k {
namespace paged_dev {

// Rows and keys of tile r of a sequence.
struct Tile {
    int row0, rows;        // query rows row0 .. row0 + rows - 1 of the sequence (row = token * group + head)
    int key_begin;         // first key any row sees, rounded down to a block
    int key_first;         // first key any row sees
    int key_end;           // past the last key any row sees
    int all_first;         // keys that every row sees: all_first ..
    int all_last;          // .. all_last
    int blocks;            // at least 1 (its outputs have to be written)
};

template <int kRows, int kBlock>
__device__ __forceinline__ Tile tile_of(const Sequence& q, int r, int group, int window, int held) {
    Tile t;
    t.row0 = r * kRows;
    t.rows = min(q.rows * group - t.row0, kRows);
    const int first = q.position + t.row0 / group, last = q.position + (t.row0 + t.rows - 1) / group;
    t.key_end = max(min(last, held - 1) + 1, 0);
    t.key_first = window > 0 ? max(first - window + 1, 0) : 0;
    t.all_first = window > 0 ? max(last - window + 1, 0) : 0;
    t.all_last = min(first, held - 1);
    t.key_begin = t.key_first & ~(kBlock - 1);
    t.blocks = max((t.key_end - t.key_begin + kBlock - 1) / kBlock, 1);
    return t;
}

template <int kRows>
__device__ __forceinline__ int tiles_of(const Sequence& q, int group) {
    return (q.rows * group + kRows - 1) / kRows;
}

// Where a CTA's share begins, and how many blocks it is.
struct Share {
    int s, h, r;
    int at;     // in the tile's units: kCost, then its blocks
    int units;
    unsigned long long start, all;  // among all units
    int ctas;                       // that have a share
};

// Worked out by all threads; per_seq ([sequences] words of shared memory) and
// out are free to use and reuse once it returns. Ends with a barrier.
template <int kRows, int kBlock, int kCost>
__device__ __forceinline__ void plan_share(const PagedBatch& b, int group, int kv_heads, int window, int held,
                                           int min_units, unsigned long long* per_seq, Share* out) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    // a thread per sequence; the tiles of a sequence of many, a lane each
    for (int base = 32 * warp; base < b.sequences; base += 32 * warps) {
        const int s = base + lane;
        Sequence q = {};
        if (s < b.sequences) q = sequence_of(b, s);
        const int n = tiles_of<kRows>(q, group);
        unsigned long long sum = 0;
        constexpr int kFew = 2;
        if (n <= kFew)
            for (int r = 0; r < n; ++r) sum += tile_of<kRows, kBlock>(q, r, group, window, held).blocks + kCost;
        for (unsigned many = __ballot_sync(0xffffffffu, n > kFew); many; many &= many - 1) {
            const int from = __ffs(many) - 1;
            const Sequence one = {__shfl_sync(0xffffffffu, q.first_row, from), __shfl_sync(0xffffffffu, q.rows, from),
                                  __shfl_sync(0xffffffffu, q.position, from)};
            const int tiles = __shfl_sync(0xffffffffu, n, from);
            unsigned long long part = 0;
            for (int r = lane; r < tiles; r += 32)
                part += tile_of<kRows, kBlock>(one, r, group, window, held).blocks + kCost;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
            if (lane == from) sum = part;
        }
        if (s < b.sequences) per_seq[s] = sum;
    }
    __syncthreads();
    if (warp == 0) {
        unsigned long long all = 0;
        for (int s = lane; s < b.sequences; s += 32) all += per_seq[s];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        all *= kv_heads;
        const int ctas = all >= (unsigned long long)gridDim.x * min_units ? (int)gridDim.x
                                                                          : ((int)all + min_units - 1) / min_units;
        Share v = {0, 0, 0, 0, 0, 0, all, ctas};
        if ((int)blockIdx.x < ctas) {
            // (32-bit divisions where they do: the 64-bit ones take hundreds of cycles)
            const bool small = all < (1ull << 32) / (gridDim.x + 1);
            auto divide = [&](unsigned long long x, unsigned long long y) {
                return small ? (unsigned long long)((uint32_t)x / (uint32_t)y) : x / y;
            };
            unsigned long long at = divide(all * blockIdx.x, ctas);
            v.start = at;
            v.units = (int)(divide(all * (blockIdx.x + 1), ctas) - at);
            // the sequence, 32 at a time
            for (int base = 0; base < b.sequences; base += 32) {
                const unsigned long long mine = base + lane < b.sequences ? per_seq[base + lane] * kv_heads : 0;
                unsigned long long run = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long u = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += u;
                }
                const unsigned past = __ballot_sync(0xffffffffu, run > at);
                if (past) {
                    const int l = __ffs(past) - 1;
                    at -= __shfl_sync(0xffffffffu, run - mine, l);
                    v.s = base + l;
                    break;
                }
                at -= __shfl_sync(0xffffffffu, run, 31);
            }
            const unsigned long long head = per_seq[v.s];
            v.h = (int)divide(at, head);
            at -= v.h * head;
            // the tile, 32 at a time
            const Sequence q = sequence_of(b, v.s);
            const int n = tiles_of<kRows>(q, group);
            for (int base = 0; base < n; base += 32) {
                const unsigned long long mine =
                    base + lane < n ? tile_of<kRows, kBlock>(q, base + lane, group, window, held).blocks + kCost : 0;
                unsigned long long run = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long u = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += u;
                }
                const unsigned past = __ballot_sync(0xffffffffu, run > at);
                if (past) {
                    const int l = __ffs(past) - 1;
                    at -= __shfl_sync(0xffffffffu, run - mine, l);
                    v.r = base + l;
                    break;
                }
                at -= __shfl_sync(0xffffffffu, run, 31);
            }
            v.at = (int)at;
        }
        if (lane == 0) *out = v;
    }
    __syncthreads();
}

// A share's pieces in turn: blocks [b, b + count) of `tile`, the index-th piece.
template <int kRows, int kBlock, int kCost>
struct Pieces {
    const PagedBatch& batch;
    int group, kv_heads, window, held;
    int s, h, r, at, left, b, count, index;
    Sequence seq = {};
    Tile tile = {};
    unsigned long long start, all;
    int ctas, units;

    __device__ __forceinline__ Pieces(const PagedBatch& batch, int group, int kv_heads, int window, int held,
                                      const Share& share)
        : batch(batch), group(group), kv_heads(kv_heads), window(window), held(held), s(share.s), h(share.h),
          r(share.r), at(share.at), left(share.units), b(0), count(0), index(0), start(share.start), all(share.all),
          ctas(share.ctas), units(share.units) {
        if (left <= 0) return;
        seq = sequence_of(batch, s);
        take();
        if (count == 0) step();
    }
    __device__ __forceinline__ void take() {
        tile = tile_of<kRows, kBlock>(seq, r, group, window, held);
        const int units = min(tile.blocks + kCost - at, left);
        b = max(at - kCost, 0);
        count = max(at + units - kCost, 0) - b;
        left -= units;
    }
    // to the next tile that has blocks in this share
    __device__ __forceinline__ void step() {
        count = 0;
        while (left > 0 && count == 0) {
            at = 0;
            if (++r >= tiles_of<kRows>(seq, group)) {
                r = 0;
                if (++h == kv_heads) {
                    h = 0;
                    do {  // a sequence with work follows, as units are left
                        ++s;
                        seq = sequence_of(batch, s);
                    } while (seq.rows == 0 && s + 1 < batch.sequences);
                }
            }
            take();
        }
    }
    __device__ __forceinline__ bool valid() const { return count > 0; }
    __device__ __forceinline__ bool whole() const { return b == 0 && count == tile.blocks; }
    __device__ __forceinline__ void next() {
        ++index;
        step();
    }
};

// What the joining kernel has to know of a tile that several CTAs share, left
// by the one where it begins (pieces 0: nothing begins here). CTA c shares
// units [all c / ctas, all (c + 1) / ctas), so unit x is CTA
// ((x + 1) ctas - 1) / all's.
struct JoinNote {
    int pieces;               // of consecutive CTAs, this one's first
    int first_row, row0, rows;  // of the batch, of the sequence, in the tile
    int head;                 // the KV head's first query head
};

template <int kRows, int kBlock, int kCost>
__device__ __forceinline__ JoinNote note_of(const Pieces<kRows, kBlock, kCost>& p) {
    if (p.whole() || p.b != 0) return {0, 0, 0, 0, 0};
    const unsigned long long end = p.start + (p.units - p.left) + (p.tile.blocks - p.count);
    const int last = (int)((end * p.ctas - 1) / p.all);
    return {last - (int)blockIdx.x + 1, p.seq.first_row, p.tile.row0, p.tile.rows, p.h * p.group};
}

}  // namespace paged_dev
}  // namespace q4k
