// Attention of chunks of new tokens over a paged KV cache, on the tensor cores with accumulators in tensor memory.
//
// A block holds 128 query rows (heads of 256 elements) or two tiles of 128 (smaller heads); a row is a new token and one of the
// query heads that share a KV head, so that a short chunk still fills a tile. Keys pass by 128 at a time:
//   S = Q K^T           tcgen05.mma 128 x 128, both operands in shared memory
//   P = exp2(c S - m)   a thread per row: tensor memory -> registers -> tensor memory, where P (16 bits) takes the place of S
//   O += P V            tcgen05.mma 128 x head_dim, P from tensor memory, V as it lies in the cache (its rows along k)
// Two score tiles are under way at a time, so that the products of one run beside the exponentials of the other: the next key
// tile's with one query tile, the other query tile's with two. m follows the row's maximum only when that has grown by 2^8
// (the weights stay below 256, the sums take the difference): tiles that rescale O in tensor memory are then few.
//
// Four warps fetch: K in panels of 64 elements, V in groups of keys, both in pieces of 16 KB through one ring, with cp.async
// rather than TMA, because a page may hold any number of tokens and end anywhere inside a tile, and 16 bytes are the unit in
// which every page size, stride and swizzled place works. Keys that no row sees are filled with zeros.
#include "paged_attention.cuh"
#include "tcgen05.cuh"

#include <cmath>
#include <type_traits>

namespace qs3 {

namespace {

using namespace tc;

constexpr uint32_t kRowTile = 128;
constexpr uint32_t kKeyTile = 128;
constexpr uint32_t kPiece = 16384;
constexpr uint32_t kPieces = 9;   // of the ring
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kNone = 0xffffffffu;
constexpr float kGrowth = 8.0f; // of a row's maximum, in powers of two, before O is rescaled

enum : uint32_t {
    ERR_PF_EMPTY_WAIT = 0x5a000001u,
    ERR_PF_FULL_WAIT = 0x5a000002u,
    ERR_PF_QUERY_WAIT = 0x5a000003u,
    ERR_PF_SCORE_WAIT = 0x5a000004u,
    ERR_PF_WEIGHT_WAIT = 0x5a000005u,
    ERR_PF_SUM_WAIT = 0x5a000006u,
};

template <uint32_t D> struct PrefillShape {
    static constexpr uint32_t kTiles = D == 256 ? 1 : 2; // query tiles
    static constexpr uint32_t kRows = kTiles * kRowTile;
    static constexpr uint32_t kPanels = D / 64;                     // pieces of a K tile, and of a V tile
    static constexpr uint32_t kPieceKeys = kPiece / (2 * D);        // keys of a piece of V
    static constexpr uint32_t kQ = kRows * D * 2;
    static constexpr uint32_t kSoftmaxWarps = 4 * kTiles;
    static constexpr uint32_t kLoadWarp = kSoftmaxWarps;            // first of four
    static constexpr uint32_t kMmaWarp = kSoftmaxWarps + 4;
    static constexpr uint32_t kThreads = (kSoftmaxWarps + 5) * 32;
    static constexpr uint32_t kSmem = 1024 + kQ + kPieces * kPiece + 512;
    static_assert(kSmem <= 227 * 1024, "shared memory of a block");
    static_assert(kPieces * kPiece >= kMaxBatch * 8, "the search for the block's range uses the ring");
};

struct Barriers {
    uint64_t full[kPieces], empty[kPieces];
    uint64_t q_full, q_free;
    uint64_t s_full[2], p_full[2], pv_done[2], o_free[2];
    uint64_t drain;
    uint32_t tmem;
    volatile uint32_t abort;
};

__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

// V as the B operand with its n side contiguous: panels of 64 elements (`panel` bytes apart), keys 128 bytes apart, groups of
// eight keys 1024, 128-byte swizzle.
__device__ __forceinline__ uint64_t value_desc(uint32_t smem_addr, uint32_t panel)
{
    return static_cast<uint64_t>((smem_addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(panel >> 4) << 16)
        | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t* r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22,"
                 " %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
                   "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}

// Waits for loads from tensor memory, of which `r` is the last: what is computed from the registers stays behind the wait only
// because they pass through it.
__device__ __forceinline__ void tc_ld_wait32(uint32_t* r)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16],"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// What every role of the block has to know of its next piece of work: it follows the items for itself.
struct Segment {
    SeqRows rows;
    SeqPages pages;
    uint32_t row0, nrows; // of the item, among the sequence's
    uint32_t tile0, count; // key tiles
    uint32_t item_tiles;
    bool second; // the second query tile has rows
};

template <uint32_t ROWS>
__device__ __forceinline__ bool next_segment(const AttnParams& p, const AttnPlace& at, uint64_t left, Segment* s)
{
    if (left == 0 || at.seq >= p.view.batch)
        return false;
    s->rows = seq_rows(p, at.seq);
    s->pages = seq_pages(p.view, at.seq);
    if (s->rows.fresh == 0)
        return false;
    const KeyTiles keys = key_tiles(p.tiling, s->rows.fresh, s->pages.length, at.tile);
    s->item_tiles = keys.end - keys.first;
    if (at.offset >= s->item_tiles)
        return false; // (the tables changed under the kernel)
    s->count = static_cast<uint32_t>(min(static_cast<uint64_t>(s->item_tiles - at.offset), left));
    s->tile0 = keys.first + at.offset;
    s->row0 = at.tile * ROWS;
    s->nrows = static_cast<uint32_t>(min(static_cast<uint64_t>(ROWS), static_cast<uint64_t>(s->rows.fresh) * p.tiling.group - s->row0));
    s->second = s->nrows > kRowTile;
    return true;
}

// Pieces of a segment in the order in which they are fetched: K 0, K 1, V 0, K 2, V 1, ... V n-1.
__device__ __forceinline__ uint32_t k_piece(uint32_t i, uint32_t panels) { return i == 0 ? 0 : panels * (2 * i - 1); }
__device__ __forceinline__ uint32_t v_piece(uint32_t i, uint32_t n, uint32_t panels)
{
    return panels * (i + 1 < n ? 2 * i + 2 : 2 * i + 1);
}

// The copies of a warp that are under way. What they wrote has to be handed to the tensor core by the threads that copied, so a
// piece is reported when the warp's next one is out, or before a wait.
struct Copies {
    uint64_t* bar = nullptr;
    __device__ __forceinline__ void report()
    {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if ((threadIdx.x & 31) == 0)
            mbar_arrive(bar);
        bar = nullptr;
    }
    __device__ __forceinline__ void push(uint64_t* b)
    {
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (bar != nullptr) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            report();
        }
        bar = b;
    }
    __device__ __forceinline__ void drain()
    {
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (bar != nullptr)
            report();
    }
};

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int slot, int head, int page)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(slot), "r"(head), "r"(page)
                 : "memory");
}

template <uint32_t D>
__global__ void __launch_bounds__(PrefillShape<D>::kThreads, 1)
attn_prefill_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map, const uint32_t k_box, const uint32_t v_box)
{
    using Shape = PrefillShape<D>;
    constexpr uint32_t TILES = Shape::kTiles, PANELS = Shape::kPanels, PIECE_KEYS = Shape::kPieceKeys;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const ring = smem + Shape::kQ;
    Barriers& bar = *reinterpret_cast<Barriers*>(ring + kPieces * kPiece);
    static_assert(sizeof(Barriers) <= 512, "room for the barriers");
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;

    if (tid == 0) {
        for (uint32_t i = 0; i < kPieces; ++i) {
            mbar_init(&bar.full[i], 1);
            mbar_init(&bar.empty[i], 1);
        }
        mbar_init(&bar.q_full, 4);
        mbar_init(&bar.q_free, 1);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 4);
            mbar_init(&bar.pv_done[i], 1);
            mbar_init(&bar.o_free[i], 4);
        }
        mbar_init(&bar.drain, 1);
        bar.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == Shape::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    const auto o_col = [&](uint32_t q) { return tmem + q * D; };
    const auto s_col = [&](uint32_t slot) { return tmem + 256 + slot * kKeyTile; };
    chain_begin();

    const BlockRange range = find_range<Shape::kThreads>(p, reinterpret_cast<uint64_t*>(ring), blockIdx.x);
    __syncthreads();
    uint64_t left = range.end - range.begin;
    AttnPlace at = range.place;
    Segment seg;
    if (tid == 0) {
        const bool work = next_segment<Shape::kRows>(p, at, left, &seg);
        note_split(p, range, work ? seg.item_tiles : 0);
    }

    if (warp >= Shape::kLoadWarp && warp < Shape::kLoadWarp + 4) {
        // ------------------------------------------------------------------------------ fetching --
        // A piece is one warp's, so that a warp looks up the pages of its next piece while the others copy.
        const uint32_t w = warp - Shape::kLoadWarp;
        Copies copies;
        uint32_t piece = 0, segments = 0;
        bool ok = true;
        const auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
            if (__all_sync(0xffffffffu, mbar_test_wait(b, parity)))
                return true;
            copies.drain();
            return __all_sync(0xffffffffu, mbar_wait(b, parity, &bar.abort, p.err, code)) != 0;
        };
        while (ok && next_segment<Shape::kRows>(p, at, left, &seg)) {
            uint32_t seen_lo, seen_hi, unused;
            visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, p.group_div.div(seg.row0), &seen_lo, &unused);
            visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, p.group_div.div(seg.row0 + seg.nrows - 1), &unused, &seen_hi);
            seen_hi = min(seen_hi, seg.pages.length);

            ok = wait(&bar.q_free, (segments & 1) ^ 1, ERR_PF_QUERY_WAIT);
            if (!ok)
                break;
#pragma unroll 1
            for (uint32_t j = 0; j < Shape::kRows / 16; ++j) {
                const uint32_t r = w * 4 + lane / 8 + 16 * j, in_tile = r & (kRowTile - 1);
                const bool there = r < seg.nrows;
                const uint32_t flat = seg.row0 + (there ? r : 0), token = p.group_div.div(flat);
                const uint8_t* src = p.q + (seg.rows.row0 + token) * p.q_token
                    + (at.head * p.tiling.group + flat - token * p.tiling.group) * p.q_head + (lane & 7) * 16;
                const uint32_t dst = smem_u32(smem) + (r / kRowTile) * (kRowTile * D * 2) + in_tile * 128 + (((lane & 7) ^ (r & 7)) * 16);
#pragma unroll
                for (uint32_t panel = 0; panel < PANELS; ++panel)
                    cp_async16z(dst + panel * kPiece, src + panel * 128, there);
            }
            copies.push(&bar.q_full);

            // KEYS keys from `key0` on, UNITS units of 16 bytes of each from `skip` bytes on, to panels of 64 elements
            const auto load = [&](const PagedPool& pool, const CUtensorMap& map, uint32_t box, uint32_t key0, auto keys, auto units,
                                  uint32_t skip) {
                constexpr uint32_t KEYS = decltype(keys)::value, UNITS = decltype(units)::value, AT_ONCE = 32 / UNITS;
                const uint32_t s = piece % kPieces;
                if (box != 0 && key0 >= seen_lo && key0 + KEYS <= seg.pages.length) {
                    // whole boxes of cached tokens: a lane each
                    const uint32_t per_panel = KEYS / box, boxes = per_panel * (UNITS / 8);
                    const uint32_t panel = lane / per_panel, first = (lane - panel * per_panel) * box;
                    uint32_t slot = 0;
                    int32_t page = 0;
                    if (lane < boxes)
                        page = page_of(p.view, seg.pages, key0 + first, &slot);
                    if (__all_sync(0xffffffffu, page >= 0)) {
                        if (!wait(&bar.empty[s], ((piece / kPieces) & 1) ^ 1, ERR_PF_EMPTY_WAIT))
                            return false;
                        if (lane == 0)
                            mbar_expect_tx(&bar.full[s], kPiece);
                        __syncwarp();
                        if (lane < boxes)
                            tma_load_page(smem_u32(ring) + s * kPiece + panel * (KEYS * 128) + first * 128, &map, &bar.full[s],
                                          static_cast<int>(skip / 2 + panel * 64), static_cast<int>(slot), static_cast<int>(at.head), page);
                        return true;
                    }
                }
                // where the rows of keys lane + 32 a begin, in units of 16 bytes; none: zeros
                uint32_t row[KEYS / 32];
#pragma unroll
                for (uint32_t a = 0; a < KEYS / 32; ++a) {
                    const uint32_t key = key0 + a * 32 + lane;
                    row[a] = kNone;
                    if (key >= seen_lo && key < seen_hi) {
                        uint32_t slot;
                        const int32_t page = page_of(p.view, seg.pages, key, &slot);
                        if (page >= 0)
                            row[a] = static_cast<uint32_t>((page * pool.page_stride + slot * pool.slot_stride) >> 4);
                    }
                }
                if (!wait(&bar.empty[s], ((piece / kPieces) & 1) ^ 1, ERR_PF_EMPTY_WAIT))
                    return false;
                const uint8_t* const from = pool.data + at.head * pool.head_stride + skip + (lane % UNITS) * 16;
                const uint32_t to = smem_u32(ring) + s * kPiece + (lane % UNITS / 8) * (KEYS * 128);
#pragma unroll
                for (uint32_t j = 0; j < KEYS / AT_ONCE; ++j) {
                    const uint32_t key = j * AT_ONCE + lane / UNITS;
                    const uint32_t r = __shfl_sync(0xffffffffu, row[j * AT_ONCE / 32], key & 31);
                    cp_async16z(to + key * 128 + (((lane & 7) ^ (key & 7)) * 16),
                                from + static_cast<uint64_t>(r == kNone ? 0 : r) * 16, r != kNone);
                }
                copies.push(&bar.full[s]);
                return true;
            };
            const auto load_k = [&](uint32_t tile) {
#pragma unroll 1
                for (uint32_t panel = 0; panel < PANELS; ++panel, ++piece)
                    if ((piece & 3) == w
                        && !load(p.view.k, k_map, k_box, (seg.tile0 + tile) * kKeyTile, std::integral_constant<uint32_t, kKeyTile> {},
                                 std::integral_constant<uint32_t, 8> {}, panel * 128))
                        return false;
                return true;
            };
            const auto load_v = [&](uint32_t tile) {
#pragma unroll 1
                for (uint32_t v = 0; v < PANELS; ++v, ++piece)
                    if ((piece & 3) == w
                        && !load(p.view.v, v_map, v_box, (seg.tile0 + tile) * kKeyTile + v * PIECE_KEYS,
                                 std::integral_constant<uint32_t, PIECE_KEYS> {}, std::integral_constant<uint32_t, D / 8> {}, 0))
                        return false;
                return true;
            };
            ok = load_k(0);
            for (uint32_t i = 0; ok && i < seg.count; ++i) {
                if (i + 1 < seg.count)
                    ok = load_k(i + 1);
                ok = ok && load_v(i);
            }
            ++segments;
            left -= seg.count;
            next_item(p, &at, row_tiles(p.tiling, seg.rows.fresh));
        }
        copies.drain();
    } else if (warp == Shape::kMmaWarp) {
        // ------------------------------------------------------------------------------- products --
        if (elect_one()) {
            constexpr uint32_t kFormat = (1u << 4) | (1u << 7) | (1u << 10) | ((kRowTile >> 4) << 24); // bf16 x bf16 -> f32
            constexpr uint32_t kScores = kFormat | ((kKeyTile >> 3) << 17);
            constexpr uint32_t kSums = kFormat | ((D >> 3) << 17) | (1u << 16);
            uint32_t piece0 = 0, segments = 0, tiles[TILES] = {}, segs[TILES] = {}, weights[2] = {};
            bool ok = true;
            const auto wait_full = [&](uint32_t piece) {
                const bool r = mbar_wait<true>(&bar.full[piece % kPieces], (piece / kPieces) & 1, &bar.abort, p.err, ERR_PF_FULL_WAIT);
                tc_fence_after();
                return r;
            };
            // scores of key tile i; the last query tile to use K lets go of it
            const auto scores = [&](uint32_t i, uint32_t q, uint32_t slot, bool release) {
                const uint32_t first = piece0 + k_piece(i, PANELS);
#pragma unroll 1
                for (uint32_t panel = 0; panel < PANELS; ++panel) {
                    if (!wait_full(first + panel))
                        return false;
                    const uint32_t s = (first + panel) % kPieces;
                    const uint64_t a = operand_desc(smem_u32(smem) + q * (kRowTile * D * 2) + panel * kPiece);
                    const uint64_t b = operand_desc(smem_u32(ring) + s * kPiece);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        tc_mma_bf16(s_col(slot), a + 2 * j, b + 2 * j, kScores, panel > 0 || j > 0);
                    if (release)
                        tc_commit(&bar.empty[s]);
                }
                tc_commit(&bar.s_full[slot]);
                return true;
            };
            const auto sums = [&](uint32_t i, uint32_t n, uint32_t q, uint32_t slot, bool release) {
                if (!mbar_wait<true>(&bar.p_full[slot], weights[slot] & 1, &bar.abort, p.err, ERR_PF_WEIGHT_WAIT))
                    return false;
                ++weights[slot];
                if (i == 0 && !mbar_wait<true>(&bar.o_free[q], (segs[q] & 1) ^ 1, &bar.abort, p.err, ERR_PF_SUM_WAIT))
                    return false;
                tc_fence_after();
                const uint32_t first = piece0 + v_piece(i, n, PANELS);
#pragma unroll 1
                for (uint32_t v = 0; v < PANELS; ++v) {
                    if (!wait_full(first + v))
                        return false;
                    const uint32_t s = (first + v) % kPieces;
                    const uint64_t b = value_desc(smem_u32(ring) + s * kPiece, PIECE_KEYS * 128);
                    constexpr uint32_t STEPS = PIECE_KEYS / 16;
#pragma unroll
                    for (uint32_t j = 0; j < STEPS; ++j) // 16 keys: 2048 bytes of V, eight columns of P
                        mma_ts(o_col(q), s_col(slot) + (v * STEPS + j) * 8, b + j * (2048 >> 4), kSums, i > 0 || v > 0 || j > 0);
                    if (release)
                        tc_commit(&bar.empty[s]);
                }
                tc_commit(&bar.pv_done[q]);
                return true;
            };
            while (ok && next_segment<Shape::kRows>(p, at, left, &seg)) {
                const uint32_t n = seg.count;
                ok = mbar_wait<true>(&bar.q_full, segments & 1, &bar.abort, p.err, ERR_PF_QUERY_WAIT);
                tc_fence_after();
                if constexpr (TILES == 1) {
                    ok = ok && scores(0, 0, tiles[0] & 1, true);
                    for (uint32_t i = 0; ok && i < n; ++i, ++tiles[0]) {
                        if (i + 1 < n)
                            ok = scores(i + 1, 0, (tiles[0] + 1) & 1, true);
                        if (i + 2 == n || n == 1) // the segment's last scores are on their way
                            tc_commit(&bar.q_free);
                        ok = ok && sums(i, n, 0, tiles[0] & 1, true);
                    }
                } else {
                    const bool second = seg.second;
                    ok = ok && scores(0, 0, 0, !second);
                    if (second)
                        ok = ok && scores(0, 1, 1, true);
                    for (uint32_t i = 0; ok && i < n; ++i) {
                        const bool more = i + 1 < n;
                        if (!more)
                            tc_commit(&bar.q_free);
                        ok = sums(i, n, 0, 0, !second);
                        if (more)
                            ok = ok && scores(i + 1, 0, 0, !second);
                        if (second) {
                            ok = ok && sums(i, n, 1, 1, true);
                            if (more)
                                ok = ok && scores(i + 1, 1, 1, true);
                        }
                    }
                    if (second)
                        ++segs[TILES - 1];
                }
                ++segs[0];
                ++segments;
                piece0 += 2 * n * PANELS;
                left -= n;
                next_item(p, &at, row_tiles(p.tiling, seg.rows.fresh));
            }
            // whatever was issued is complete before the tensor memory goes back
            volatile uint32_t never = 0;
            tc_commit(&bar.drain);
            mbar_wait<true>(&bar.drain, 0, &never, p.err, ERR_PF_SUM_WAIT);
        }
        __syncwarp();
    } else if (warp < Shape::kSoftmaxWarps) {
        // -------------------------------------------------------------------------------- weights --
        const uint32_t q = warp / 4;
        const uint32_t lanes = (warp & 3) << 21; // this warp's 32 lanes of tensor memory
        uint32_t tiles = 0;
        bool ok = true;
        while (ok && next_segment<Shape::kRows>(p, at, left, &seg)) {
            const uint32_t n = seg.count;
            if (q == 0 || seg.second) {
                const uint32_t r = q * kRowTile + (warp & 3) * 32 + lane;
                const bool live = r < seg.nrows;
                const uint32_t flat = seg.row0 + (live ? r : 0), token = p.group_div.div(flat);
                uint32_t lo = 0, hi = 0xffffffffu; // (rows past the last one need no mask)
                if (live) {
                    visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, token, &lo, &hi);
                    hi = min(hi, seg.pages.length);
                }
                float m = -INFINITY, l = 0.0f;
                for (uint32_t i = 0; i < n; ++i, ++tiles) {
                    const uint32_t slot = TILES == 1 ? tiles & 1 : q;
                    const uint32_t parity = TILES == 1 ? (tiles >> 1) & 1 : tiles & 1;
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar.s_full[slot], parity, &bar.abort, p.err, ERR_PF_SCORE_WAIT));
                    if (!ok)
                        break;
                    tc_fence_after();
                    const uint32_t s_addr = s_col(slot) + lanes;
                    const uint32_t key0 = (seg.tile0 + i) * kKeyTile;
                    const bool part = __any_sync(0xffffffffu, lo > key0 || hi < key0 + kKeyTile);

                    uint32_t x[32];
                    // both passes once with and once without the mask: a test inside them costs a branch per element
                    const auto largest = [&](auto masked) {
                        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
                        for (uint32_t c = 0; c < kKeyTile / 32; ++c) {
                            tc_ld32(s_addr + c * 32, x);
                            tc_ld_wait32(x);
#pragma unroll
                            for (uint32_t j = 0; j < 32; j += 2) {
                                float a = __uint_as_float(x[j]), b = __uint_as_float(x[j + 1]);
                                if constexpr (decltype(masked)::value) {
                                    const uint32_t key = key0 + c * 32 + j;
                                    a = key >= lo && key < hi ? a : -INFINITY;
                                    b = key + 1 >= lo && key + 1 < hi ? b : -INFINITY;
                                }
                                if ((j & 2) == 0)
                                    top0 = fmaxf(top0, fmaxf(a, b));
                                else
                                    top1 = fmaxf(top1, fmaxf(a, b));
                            }
                        }
                        return fmaxf(top0, top1);
                    };
                    float top = part ? largest(std::true_type {}) : largest(std::false_type {});
                    top *= p.scale_log2;
                    const bool grow = top > m + kGrowth; // (m = -inf: whenever something is seen)
                    if (__any_sync(0xffffffffu, grow)) {
                        const float next = grow ? top : m;
                        const float keep = grow ? exp2_approx(m - next) : 1.0f;
                        m = next;
                        l *= keep;
                        if (i > 0) { // O holds the sums up to tile i - 1 once its product is through
                            ok = __all_sync(0xffffffffu, mbar_wait(&bar.pv_done[q], (tiles - 1) & 1, &bar.abort, p.err, ERR_PF_SUM_WAIT));
                            if (!ok)
                                break;
                            tc_fence_after();
#pragma unroll 1
                            for (uint32_t c = 0; c < D / 32; ++c) {
                                tc_ld32(o_col(q) + lanes + c * 32, x);
                                tc_ld_wait32(x);
#pragma unroll
                                for (uint32_t j = 0; j < 32; ++j)
                                    x[j] = __float_as_uint(__uint_as_float(x[j]) * keep);
                                tc_st16(o_col(q) + lanes + c * 32, x);
                                tc_st16(o_col(q) + lanes + c * 32 + 16, x + 16);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const auto weights = [&](auto masked) {
                        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                        for (uint32_t c = 0; c < kKeyTile / 32; ++c) {
                            tc_ld32(s_addr + c * 32, x);
                            tc_ld_wait32(x);
                            uint32_t w[16];
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) {
                                float a = fmaf(__uint_as_float(x[2 * j]), p.scale_log2, -base);
                                float b = fmaf(__uint_as_float(x[2 * j + 1]), p.scale_log2, -base);
                                if constexpr (decltype(masked)::value) {
                                    const uint32_t key = key0 + c * 32 + 2 * j;
                                    a = key >= lo && key < hi ? a : -INFINITY;
                                    b = key + 1 >= lo && key + 1 < hi ? b : -INFINITY;
                                }
                                a = exp2_approx(a);
                                b = exp2_approx(b);
                                sum0 += a;
                                sum1 += b;
                                w[j] = pack_bf16x2(a, b);
                            }
                            tc_st16(s_addr + c * 16, w);
                        }
                        return sum0 + sum1;
                    };
                    l += part ? weights(std::true_type {}) : weights(std::false_type {});
                    tc_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar.p_full[slot]);
                }
                if (!ok)
                    break;
                // The last two products: a barrier's parity tells one phase from the next only, and with one query tile the
                // scores that were waited for last are issued before the product of the tile before.
                if (TILES == 1 && n > 1)
                    ok = __all_sync(0xffffffffu, mbar_wait(&bar.pv_done[q], (tiles - 2) & 1, &bar.abort, p.err, ERR_PF_SUM_WAIT));
                ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar.pv_done[q], (tiles - 1) & 1, &bar.abort, p.err, ERR_PF_SUM_WAIT));
                if (!ok)
                    break;
                tc_fence_after();
                const bool whole = n == seg.item_tiles;
                const uint32_t h = at.head * p.tiling.group + flat - token * p.tiling.group;
                const size_t part_row = static_cast<size_t>(blockIdx.x * 2 + (at.offset == 0 ? 1 : 0)) * Shape::kRows + r;
                uint8_t* const out = p.out + (seg.rows.row0 + token) * p.out_token + h * p.out_head;
                float* const part_o = p.part_o + part_row * D;
                const float inv = whole ? (m == -INFINITY ? 0.0f : 1.0f / l) : 1.0f;
                uint32_t x[32];
#pragma unroll 1
                for (uint32_t c = 0; c < D / 32; ++c) {
                    tc_ld32(o_col(q) + lanes + c * 32, x);
                    tc_ld_wait32(x);
                    if (!live)
                        continue;
                    if (whole) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k)
                                w[k] = pack_bf16x2(__uint_as_float(x[8 * j + 2 * k]) * inv, __uint_as_float(x[8 * j + 2 * k + 1]) * inv);
                            *reinterpret_cast<uint4*>(out + c * 64 + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 8; ++j)
                            *reinterpret_cast<uint4*>(part_o + c * 32 + j * 4) = make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&bar.o_free[q]);
                if (live && whole && p.lse != nullptr)
                    p.lse[(seg.rows.row0 + token) * p.lse_token + h * p.lse_head]
                        = m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
                if (live && !whole)
                    p.part_ml[part_row] = make_float2(m, l);
            }
            left -= n;
            next_item(p, &at, row_tiles(p.tiling, seg.rows.fresh));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Shape::kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <uint32_t D> cudaError_t launch_prefill_as(const AttnParams& p, cudaStream_t stream)
{
    using Shape = PrefillShape<D>;
    const cudaError_t err = cudaFuncSetAttribute(attn_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (err != cudaSuccess)
        return err;
    // Pages that a box fits into a whole number of times are fetched by TMA, others and the ends of sequences row by row.
    const auto box = [&](CUtensorMap* map, const PagedPool& pool, uint32_t most) {
        const uint32_t size = p.view.page_size;
        const uint32_t rows = size < most ? size : most;
        const uint64_t dims[4] = { D, size, p.view.kv_heads, p.view.pages };
        const uint64_t strides[3] = { static_cast<uint64_t>(pool.slot_stride), static_cast<uint64_t>(pool.head_stride),
                                      static_cast<uint64_t>(pool.page_stride) };
        if (rows < 8 || size % rows != 0 || most % rows != 0 || !make_page_map(map, pool.data, dims, strides, rows))
            return 0u;
        return rows;
    };
    CUtensorMap k_map {}, v_map {};
    const uint32_t k_box = box(&k_map, p.view.k, kKeyTile), v_box = box(&v_map, p.view.v, Shape::kPieceKeys);
    return launch_chained(attn_prefill_kernel<D>, dim3(p.blocks), Shape::kThreads, Shape::kSmem, stream, p, k_map, v_map, k_box, v_box);
}

} // namespace

uint32_t attn_prefill_rows(uint32_t head_dim) { return head_dim == 256 ? kRowTile : 2 * kRowTile; }

cudaError_t launch_attn_prefill(const AttnParams& p, cudaStream_t stream)
{
    const uint32_t d = p.view.head_dim;
    return d == 64 ? launch_prefill_as<64>(p, stream) : d == 128 ? launch_prefill_as<128>(p, stream) : launch_prefill_as<256>(p, stream);
}

} // namespace qs3
