// Division of attention over a paged cache into pieces of equal work. Arithmetic only, for the kernels and for the host.
//
// An item is a tile of query rows of one sequence and KV head: the rows of a sequence and KV head are its new tokens times the
// query heads that share the KV head, row = token * group + head, cut into tiles of 1 << row_shift. Its cost is the number of key
// tiles that hold a key some row of it sees, at least one (an item without keys still writes its output), and `item_cost`
// more for its start and end. Items follow each other by sequence, KV head, tile; their costs, laid end to end, are cut into
// equal ranges, one per block of the launch. A range ends where it ends, inside an item as well, so that lengths which differ
// leave no block idle and a single long context is spread over all SMs; an item whose key tiles are cut this way leaves
// partial results that a second launch joins. Short contexts are not worth that launch: `even` items cost 1 each, whatever their
// length, and no range ends inside one.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define QS3_HD __host__ __device__ __forceinline__
#else
#define QS3_HD inline
#endif

namespace qs3 {

// n / d for n < 2^31 by a multiplication: with s = ceil(log2 d), m = ceil(2^(31+s) / d) has an error below d / 2^(31+s), which
// times n stays below 1/d.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor)
    {
        uint32_t s = 0;
        while ((1ull << s) < divisor)
            ++s;
        mul = static_cast<uint32_t>(((1ull << (31 + s)) + divisor - 1) / divisor);
        shift = s;
    }
    QS3_HD uint32_t div(uint32_t n) const
    {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> (31 + shift));
    }
};

struct AttnTiling {
    FastDiv group;      // by the query heads per KV head
    uint32_t row_shift; // log2 of the rows of an item
    uint32_t key_shift; // log2 of the keys of a key tile
    uint32_t kv_heads;
    uint32_t window;    // 0: none
    uint32_t causal;
    uint32_t item_cost; // in key tiles
    uint32_t even = 0;
};

struct KeyTiles {
    uint32_t first, end; // end > first
};

// Row tiles of a sequence with `fresh` new tokens. (Rows, and positions, stay below 2^31 by the limits of the entry point.)
QS3_HD uint32_t row_tiles(const AttnTiling& a, uint32_t fresh)
{
    return (fresh * a.group.d + (1u << a.row_shift) - 1) >> a.row_shift;
}

// Keys [lo, hi) that new token `i` of `fresh` sees in a cache of `length` tokens (its own position: length - fresh + i).
QS3_HD void visible_keys(const AttnTiling& a, uint32_t fresh, uint32_t length, uint32_t i, uint32_t* lo, uint32_t* hi)
{
    const int64_t pos = static_cast<int64_t>(length) - fresh + i;
    const int64_t h = a.causal ? pos + 1 : static_cast<int64_t>(length);
    *hi = h > 0 ? static_cast<uint32_t>(h) : 0;
    const int64_t l = a.window != 0 ? pos - a.window + 1 : 0;
    *lo = l <= 0 ? 0 : l < h ? static_cast<uint32_t>(l) : *hi;
}

// `room`: the first keys of the sequence, which are there to be seen.
QS3_HD KeyTiles key_tiles(const AttnTiling& a, uint32_t fresh, uint32_t length, uint32_t tile, uint32_t room = 0xffffffffu)
{
    const uint32_t rows = fresh * a.group.d, r0 = tile << a.row_shift, next = r0 + (1u << a.row_shift);
    const uint32_t r1 = (next < rows ? next : rows) - 1;
    uint32_t lo, hi, unused;
    visible_keys(a, fresh, length, a.group.div(r0), &lo, &unused);
    visible_keys(a, fresh, length, a.group.div(r1), &unused, &hi);
    hi = hi < room ? hi : room;
    lo = lo < room ? lo : room;
    KeyTiles k;
    k.first = lo >> a.key_shift;
    k.end = (hi + (1u << a.key_shift) - 1) >> a.key_shift;
    if (k.end <= k.first)
        k.end = k.first + 1;
    return k;
}

QS3_HD uint32_t cost_of(const AttnTiling& a, uint32_t tiles) { return a.even ? 1 : a.item_cost + tiles; }

// Blocks that get work: every one at least `least` key tiles, as far as there are any.
QS3_HD uint32_t active_blocks(uint64_t total, uint32_t blocks, uint32_t least)
{
    const uint64_t n = (total + least - 1) / least;
    return n < blocks ? static_cast<uint32_t>(n) : blocks;
}

// Where the range of block `c` of `blocks` begins. (c * total stays below 2^63: total <= 2^52 and blocks < 2^11 by the limits of the entry point.)
QS3_HD uint64_t block_begin(uint64_t total, uint32_t blocks, uint32_t c) { return total * c / blocks; }

// The last block whose range begins before `end`.
QS3_HD uint32_t block_of_end(uint64_t total, uint32_t blocks, uint64_t end)
{
    // total * c / blocks < end exactly when total * c < end * blocks
    return static_cast<uint32_t>((end * blocks - 1) / total);
}

// Key tiles of an item that lie before a position `offset` from its beginning.
QS3_HD uint32_t tiles_before(const AttnTiling& a, uint64_t offset, uint32_t tiles)
{
    if (a.even)
        return offset > 0 ? tiles : 0;
    const uint64_t t = offset > a.item_cost ? offset - a.item_cost : 0;
    return t < tiles ? static_cast<uint32_t>(t) : tiles;
}

// Where a position in the row of all items lies.
struct AttnPlace {
    uint32_t seq, head, tile;
    uint32_t offset; // from the item's beginning
};

} // namespace qs3
