// What the attention kernels over a paged cache share: parameters, the search for a block's range of key tiles, and the layout
// of the partial results that the joining launch reads.
#pragma once

#include "paged.cuh"

namespace qs3 {

struct AttnParams {
    PagedView view;
    AttnTiling tiling;
    const uint8_t* q; // strides in bytes
    int64_t q_token, q_head;
    uint8_t* out;
    int64_t out_token, out_head;
    float* lse; // elements
    int64_t lse_token, lse_head;
    const int32_t* q_indptr;
    uint32_t rows, heads;
    float scale_log2;            // sm_scale * log2(e)
    uint32_t blocks;             // of the launch
    uint32_t least;              // key tiles of a block
    // Partial results. Block c has two slots of [rows of an item, head_dim] f32 weighted sums and [rows] maxima (in units of log2) and
    // sums: 0 for an item that began in an earlier block, 1 for one that begins here and goes on in the next.
    float* part_o;
    float2* part_ml;
    struct SplitNote* notes; // [blocks]
    uint32_t* err;
};

// What block c leaves for the joining launch when its range begins inside the key tiles of an item and no earlier block's does:
// the item, and how many blocks after c - 1 hold parts of it. 0: nothing to join here.
struct SplitNote {
    uint32_t seq, head, tile, parts;
};

#ifdef __CUDACC__

// Rows of the new tokens of a sequence, kept inside the tensors whatever the tables hold.
struct SeqRows {
    uint32_t row0, fresh;
};

__device__ __forceinline__ SeqRows seq_rows(const AttnParams& p, uint32_t seq)
{
    if (p.q_indptr == nullptr)
        return SeqRows { seq, 1 };
    const int32_t a = p.q_indptr[seq], b = p.q_indptr[seq + 1];
    const uint32_t lo = a > 0 ? min(static_cast<uint32_t>(a), p.rows) : 0;
    const uint32_t hi = b > 0 ? min(static_cast<uint32_t>(b), p.rows) : 0;
    return SeqRows { lo, hi > lo ? hi - lo : 0 };
}

// The search for where a block's range begins. `cost` [batch] is shared memory that nothing else uses meanwhile; every thread of
// the block takes part and gets the same answer, warps at their own time (a barrier comes before `cost` is used again).
struct BlockRange {
    uint64_t begin, end;
    uint64_t total;
    uint32_t active;
    AttnPlace place;     // of `begin`
};

// Cost of the items of a (sequence, KV head), by one warp.
__device__ __forceinline__ uint64_t warp_tiles_cost(const AttnTiling& a, uint32_t fresh, const SeqPages& s, uint32_t tiles)
{
    uint64_t sum = 0;
    for (uint32_t t = threadIdx.x & 31; t < tiles; t += 32) {
        const KeyTiles k = key_tiles(a, fresh, s.length, t, s.room);
        sum += cost_of(a, k.end - k.first);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

constexpr uint64_t kUnknown = ~0ull;
constexpr uint32_t kSerialTiles = 4; // row tiles of a sequence up to which one thread adds up their cost

template <uint32_t THREADS>
__device__ BlockRange find_range(const AttnParams& p, uint64_t* cost, uint32_t block)
{
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t batch = p.view.batch;
    for (uint32_t b = tid; b < batch; b += THREADS) {
        const uint32_t fresh = seq_rows(p, b).fresh, tiles = row_tiles(p.tiling, fresh);
        uint64_t sum = 0;
        if (tiles <= kSerialTiles) {
            const SeqPages s = seq_pages(p.view, b);
#pragma unroll 1
            for (uint32_t t = 0; t < tiles; ++t) { // (short, and once a block)
                const KeyTiles k = key_tiles(p.tiling, fresh, s.length, t, s.room);
                sum += cost_of(p.tiling, k.end - k.first);
            }
        } else {
            sum = kUnknown;
        }
        cost[b] = sum;
    }
    __syncthreads();
    for (uint32_t b = warp; b < batch; b += THREADS / 32) {
        if (cost[b] == kUnknown) {
            const uint32_t fresh = seq_rows(p, b).fresh;
            const uint64_t sum = warp_tiles_cost(p.tiling, fresh, seq_pages(p.view, b), row_tiles(p.tiling, fresh));
            __syncwarp();
            if (lane == 0)
                cost[b] = sum;
        }
    }
    __syncthreads();
    // every warp adds the costs up for itself, 32 sequences at a time, and stops at the one that holds `begin`
    uint64_t sum = 0;
    for (uint32_t b = lane; b < batch; b += 32)
        sum += cost[b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    BlockRange r;
    r.total = sum * p.view.kv_heads;
    r.active = active_blocks(r.total, p.blocks, p.least);
    r.place = AttnPlace { 0, 0, 0, 0 };
    if (block >= r.active) {
        r.begin = r.end = r.total;
        return r;
    }
    r.begin = block_begin(r.total, r.active, block);
    r.end = block_begin(r.total, r.active, block + 1);
    uint64_t before = 0;
    uint32_t seq = 0;
    for (uint32_t b0 = 0; b0 < batch; b0 += 32) {
        const uint64_t mine = b0 + lane < batch ? cost[b0 + lane] * p.view.kv_heads : 0;
        uint64_t run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= static_cast<uint32_t>(o))
                run += up;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, before + run > r.begin);
        if (beyond != 0) {
            const uint32_t at = __ffs(beyond) - 1;
            seq = b0 + at;
            before += __shfl_sync(0xffffffffu, run - mine, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
    uint64_t inside = r.begin - before;
    const uint64_t per_head = cost[seq];
    r.place.seq = seq;
    r.place.head = static_cast<uint32_t>(inside / per_head);
    uint64_t rest = inside - r.place.head * per_head;
    const uint32_t fresh = seq_rows(p, seq).fresh;
    const SeqPages pages = seq_pages(p.view, seq);
    const uint32_t tiles = row_tiles(p.tiling, fresh);
    for (uint32_t t0 = 0; t0 < tiles; t0 += 32) {
        uint32_t mine = 0;
        if (t0 + lane < tiles) {
            const KeyTiles k = key_tiles(p.tiling, fresh, pages.length, t0 + lane, pages.room);
            mine = cost_of(p.tiling, k.end - k.first);
        }
        uint64_t run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= static_cast<uint32_t>(o))
                run += up;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, run > rest);
        if (beyond != 0) {
            const uint32_t at = __ffs(beyond) - 1;
            r.place.tile = t0 + at;
            r.place.offset = static_cast<uint32_t>(rest - __shfl_sync(0xffffffffu, run - mine, at));
            break;
        }
        rest -= __shfl_sync(0xffffffffu, run, 31);
    }
    return r;
}

// What becomes of a row without a score above -infinity: zeros (and a log-sum-exp of -infinity) where it sees no key, NaN where it
// sees some, of which no softmax exists.
__device__ __forceinline__ float without_scores(const AttnParams& p, uint32_t fresh, const SeqPages& s, uint32_t row)
{
    uint32_t lo, hi;
    visible_keys(p.tiling, fresh, s.length, p.tiling.group.div(row), &lo, &hi);
    return lo < min(hi, s.room) ? __int_as_float(0x7fffffff) : 0.0f;
}

// The item after the one at `at`; sequences without new tokens have none.
__device__ __forceinline__ void next_item(const AttnParams& p, AttnPlace* at, uint32_t tiles)
{
    at->offset = 0;
    if (++at->tile < tiles)
        return;
    at->tile = 0;
    if (++at->head < p.view.kv_heads)
        return;
    at->head = 0;
    do
        ++at->seq;
    while (at->seq < p.view.batch && seq_rows(p, at->seq).fresh == 0);
}

// By one thread of every block.
__device__ __forceinline__ void note_split(const AttnParams& p, const BlockRange& r)
{
    SplitNote n { r.place.seq, r.place.head, r.place.tile, 0 };
    if (r.begin < r.end && r.place.offset > p.tiling.item_cost) { // (never with even items, which have an offset of 0)
        const uint64_t item = r.begin - r.place.offset;
        const SeqPages s = seq_pages(p.view, n.seq);
        const KeyTiles k = key_tiles(p.tiling, seq_rows(p, n.seq).fresh, s.length, n.tile, s.room);
        if (block_begin(r.total, r.active, blockIdx.x - 1) <= item + p.tiling.item_cost) // (block 0 begins with an item)
            n.parts = block_of_end(r.total, r.active, item + p.tiling.item_cost + (k.end - k.first)) - blockIdx.x + 1;
    }
    p.notes[blockIdx.x] = n;
}

// A block's part of an item. `at` moves along the block's range with `left`; false: the range is through.
struct Segment {
    uint32_t seq = 0xffffffffu; // of rows and pages
    SeqRows rows;
    SeqPages pages;
    uint32_t row0, nrows;  // of the item, among the sequence's
    uint32_t tile0, count; // key tiles
    uint32_t tiles;        // of the item
    bool starts, whole;    // with the item's first key tile; with all of them
};

// KEEP: rows and pages of a sequence are held from item to item, where registers are left for them. In the chunk kernel, whose 128
// are all taken, each role looks them up again instead: mixed batch 127.2 us held, 125.6 looked up, 8192 tokens 569 and 561, 1021 tokens
// over an e4m3 cache 693 and 682.
template <bool KEEP>
__device__ __forceinline__ bool this_segment(const AttnParams& p, const AttnPlace& at, uint64_t left, Segment* s)
{
    if (left == 0 || at.seq >= p.view.batch)
        return false;
    if (!KEEP || s->seq != at.seq) {
        s->seq = at.seq;
        s->rows = seq_rows(p, at.seq);
        s->pages = seq_pages(p.view, at.seq);
    }
    if (s->rows.fresh == 0)
        return false;
    const KeyTiles keys = key_tiles(p.tiling, s->rows.fresh, s->pages.length, at.tile, s->pages.room);
    const uint32_t tiles = s->tiles = keys.end - keys.first;
    const uint32_t from = tiles_before(p.tiling, at.offset, tiles), to = tiles_before(p.tiling, at.offset + left, tiles);
    if (from >= to)
        return false; // the range ends before the item's first key tile
    s->count = to - from;
    s->tile0 = keys.first + from;
    s->starts = from == 0;
    s->whole = s->count == tiles;
    s->row0 = at.tile << p.tiling.row_shift;
    s->nrows = min(1u << p.tiling.row_shift, s->rows.fresh * p.tiling.group.d - s->row0);
    return true;
}

__device__ __forceinline__ void next_segment(const AttnParams& p, const Segment& s, AttnPlace* at, uint64_t* left)
{
    const uint64_t rest = cost_of(p.tiling, s.tiles) - at->offset;
    *left = *left > rest ? *left - rest : 0;
    next_item(p, at, row_tiles(p.tiling, s.rows.fresh));
}

#endif

cudaError_t launch_attn_stream(const AttnParams& p, bool fp8, cudaStream_t stream);
cudaError_t launch_attn_prefill(const AttnParams& p, bool fp8, cudaStream_t stream);
cudaError_t launch_attn_join(const AttnParams& p, cudaStream_t stream);
// Rows of an item of the streaming kernel: 8 or 16; blocks that fit the device at once.
uint32_t attn_stream_rows(uint32_t rows_per_seq);
uint32_t attn_prefill_rows(uint32_t head_dim); // and of the kernel for chunks; keys of its key tile: 128
uint32_t attn_stream_blocks(uint32_t tile_rows, uint32_t head_dim, bool fp8);

} // namespace qs3
