// How the attention over a paged cache (cache.cu) cuts a call's work into runs of equal cost.  The lengths
// are the device's, so it does this itself; the arithmetic compiles for the host as well.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LSX_RUNS __host__ __device__ __forceinline__
#else
#define LSX_RUNS inline
#endif

namespace lsx {

constexpr int kCellTokens = 16;  // positions of a cell
constexpr int kPairTokens = 2 * kCellTokens;
// Cost that a block takes at least, where there is little: a tile and two pairs a warp.
constexpr int kLeastRun = 20;
// What a tile costs beside its pairs (the first copies' latency, the queries, the sums), in
// pairs: it counts so many more when the runs are cut (61 sequences of about 5000 positions, f16: 70 us
// with 1, 61 with 4, 45 with 12).
constexpr int kTileCost = 12;

struct SequenceRows {
    int table;   // row of the tables, -1 when the list names none
    int first;   // its first row of the call
    int count;   // its rows
    int length;  // its positions, those of the rows last
};

template <typename N>
LSX_RUNS N least_of(N a, N b) {
    return a < b ? a : b;
}
template <typename N>
LSX_RUNS N most_of(N a, N b) {
    return a < b ? b : a;
}

// A call's pairs of cells in order.  Tile k of a sequence holds its rows' positions k * tokens and on;
// a tile without visible positions counts as one pair, so that its rows get written.
LSX_RUNS int tile_count(const SequenceRows& s, int tokens) { return (s.count + tokens - 1) / tokens; }

LSX_RUNS int tile_pairs(const SequenceRows& s, int tokens, int k) {
    const int seen = s.length - s.count + least_of(s.count, (k + 1) * tokens);  // positions that its last row sees
    return seen <= kPairTokens ? 1 : ((seen - 1) >> 5) + 1;
}

// Sum of floor(i / m) over i = 0 .. n.
LSX_RUNS long long sum_of_quotients(long long n, int m) {
    if (n < 0) return 0;
    const long long q = n / m, r = n % m;
    return m * q * (q - 1) / 2 + q * (r + 1);
}

// Cost of the tiles before k (k below the tile count), kTileCost and their pairs each: the sum of
// floor((base + 31 + (i + 1) tokens) / 32), with base = length - count, over the tiles that see anything, and 1 for
// those that do not.  tokens is a power of two that divides 32.
LSX_RUNS long long cost_before(const SequenceRows& s, int tokens, int k) {
    if (k == 0) return 0;
    const int base = s.length - s.count;
    const int blind = s.length <= 0 ? k : base >= 0 ? 0 : least_of(k, -base / tokens);
    const long long fixed = (long long)k * kTileCost;
    if (k <= blind) return fixed + k;
    int shift = 0;
    while (tokens >> (shift + 1)) ++shift;
    const int m = kPairTokens >> shift;
    const long long y = ((long long)base + kPairTokens - 1) >> shift;  // a length may be 2^31 - 1
    return fixed + blind + sum_of_quotients(y + k, m) - sum_of_quotients(y + blind, m);
}

LSX_RUNS long long sequence_cost(const SequenceRows& s, int tokens) {
    const int tiles = tile_count(s, tokens);
    return tiles ? cost_before(s, tokens, tiles - 1) + kTileCost + tile_pairs(s, tokens, tiles - 1) : 0;
}

// What is left of a block's run.
struct Run {
    long long at, end;  // cost of the call before the next and before what follows the run
    uint32_t sequence;  // the next is a part of its tiles,
    long long offset;   // this far into them
};

struct RunTile {
    uint32_t head;    // key head, and part of its query heads, as the call numbers them
    int k;            // tile of the sequence's rows
    int first, last;  // pairs of it that the run holds
    int pairs;        // all of them
};

// The run's next part of a tile, where sequence run.sequence, of these rows, has one; `heads` tiles for each k.
// `whole`: tiles are not shared, each is the run's in which it begins.
LSX_RUNS bool next_tile(Run& run, const SequenceRows& s, int tokens, uint32_t heads, bool whole, RunTile& tile) {
    const long long one = sequence_cost(s, tokens);
    if (run.offset >= one * heads) {
        ++run.sequence;
        run.offset = 0;
        return false;
    }
    // 32 bits where both fit; a long prompt behind many positions costs 2^32 and more
    tile.head = (run.offset | one) >> 32 ? (uint32_t)(run.offset / one) : (uint32_t)run.offset / (uint32_t)one;
    const long long rest = run.offset - tile.head * one;
    tile.k = 0;
    for (int high = tile_count(s, tokens); high - tile.k > 1;) {  // cost_before(k) <= rest
        const int middle = tile.k + (high - tile.k) / 2;
        if (cost_before(s, tokens, middle) <= rest)
            tile.k = middle;
        else
            high = middle;
    }
    // the first kTileCost of a tile's cost stand for no pair
    tile.pairs = tile_pairs(s, tokens, tile.k);
    const long long all = (long long)tile.pairs + kTileCost, from = rest - cost_before(s, tokens, tile.k);
    const long long to = whole ? all : least_of(all, from + run.end - run.at);
    run.at += to - from;
    run.offset += to - from;
    if (to <= kTileCost || (whole && from > 0)) return false;
    tile.first = (int)most_of(from - kTileCost, 0ll);
    tile.last = (int)(to - kTileCost);
    return true;
}

}  // namespace lsx
