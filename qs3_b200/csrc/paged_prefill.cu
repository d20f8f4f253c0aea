// Attention of chunks of new tokens over a paged KV cache, on the tensor cores with accumulators in tensor memory.
//
// A block holds 128 query rows (heads of 256 elements) or two tiles of 128 (smaller heads); a row is a new token and one of the
// query heads that share a KV head, so that a short chunk still fills a tile. Keys arrive by 128 and pass in steps of 128 (one
// query tile) or 64 (two):
//   S = Q K^T           tcgen05.mma 128 x 128 or 128 x 64, both operands in shared memory
//   P = exp2(c S - m)   tensor memory -> registers -> tensor memory, in 16 bits; a thread has 64 keys of a row: half a step with
//                       one query tile, whose row two threads share, else a step of its own row
//   O += P V            tcgen05.mma 128 x head_dim, P from tensor memory, V as it lies in the cache (its rows along k)
// Beside O (256 columns of 512) there is room for one score tile of each query tile and two of its weights. Scores are read into
// registers at once, so that the next ones are on their way while their exponentials are taken: where weights took the place of
// the scores that they came from, with two such tiles in turn, the scores waited for the sums of the step before the last
// (8192 tokens of 16 heads of 256: 559 us, 541; with heads of 128 the mixed batch of 12 sequences lost by it, 118 us, 124). Eight warps take the exponentials, because one alone waits longer for each of its
// instructions than they take. One warp issues the scores and another the sums: every wait, product and commit costs its thread
// 50 to 100 cycles, together twice as much as the products take.
// m follows the row's maximum only when that has grown by 2^8 (the weights stay below 256, the sums take the difference):
// steps that rescale O in tensor memory are then few.
//
// bf16 caches: five warps fetch, three K in panels of 64 elements and two V in groups of keys, in pieces of 32 KB, each warp its
// own slots of K's or V's ring: a slot's barriers then pass their phases in one order for all, which parities need. Pages that a
// box of TMA divides come that way; other page sizes, the ends of sequences and windows row by row with cp.async, 16 bytes being
// the unit in which every page size, stride and swizzled place works. Keys that no row sees are zeros then.
//
// e4m3 caches: K's codes are multiplied as they are. A row of queries is scaled by the power of two that brings its largest element
// to 2^7 or just above and becomes the sum of two e4m3 numbers, the high one rounded to 4 bits and the low one the rest: bf16's 8
// bits exactly, and no element is off by more than 2^-17 of the largest. Two products of twice the rate take the time of one.
// K's scales are a factor on the scores. V's are part of the weights, w = exp2(s + log2(scale) - m), of which the largest is again
// at a known place; a second e4m3 number would keep 8 bits of a weight but only 14 of the range below the largest, which many
// small weights together need. So the weights are f16 and V is converted, by the four warps that fetch it: boxes to a staging
// area, from there to registers, which makes room for the next ones, and to the ring. A fifth warp fetches K and a sixth the
// scales. The row's sum takes V's scale out again.
// 1021 tokens behind 31 111 cached ones take 676 us; with V's loads straight to registers, which fill what the first-level cache
// has left beside so much shared memory, it was 765; with everything converted to f16, K too, 965. Shared memory is the bound: codes
// in and out, V in f16, the products' operands and the scales.
#include "paged_attention.cuh"
#include "tcgen05.cuh"

#include <cmath>
#include <type_traits>

namespace qs3 {

namespace {

using namespace tc;

constexpr uint32_t kRowTile = 128;
constexpr uint32_t kKeyTile = 128;
constexpr uint32_t kMine = 64;     // keys of a step that a thread has
constexpr uint32_t kSoftmaxWarps = 8;
constexpr uint32_t kMostSlots = 6;
constexpr uint32_t kScaleTiles = 4; // key tiles whose scales are held
constexpr uint32_t kTmemCols = 512;
// Growth of a row's maximum, in powers of two, before O is rescaled, and where the largest weight lies at first: f16 weights end at
// 2^16 and lose bits below 2^-14.
template <bool FP8> constexpr float kGrowth = FP8 ? 7.0f : 8.0f;
template <bool FP8> constexpr float kTop = FP8 ? 8.0f : 0.0f;
// e4m3: 1 / scale of V, at most 1e30, times this, so that sums of a long row of zeros stay finite.
template <bool FP8> constexpr float kSumUnit = FP8 ? 20.0f : 0.0f;
template <bool FP8> constexpr float kSumFactor = FP8 ? 1.0f / 1048576.0f : 1.0f;

enum : uint32_t {
    ERR_PF_EMPTY_WAIT = 0x5c000001u,
    ERR_PF_FULL_WAIT = 0x5c000002u,
    ERR_PF_QUERY_WAIT = 0x5c000003u,
    ERR_PF_SCORE_WAIT = 0x5c000004u,
    ERR_PF_WEIGHT_WAIT = 0x5c000005u,
    ERR_PF_SUM_WAIT = 0x5c000006u,
};

struct Barriers {
    uint64_t k_full[kMostSlots], k_empty[kMostSlots], v_full[kMostSlots], v_empty[kMostSlots];
    uint64_t scale_full[kScaleTiles], staged[4];
    uint64_t q_full, q_free;
    uint64_t s_full[2], s_free[2], o_free[2]; // of a query tile
    uint64_t p_full[2][2], pv_done[2][2];     // of its tiles of weights
    uint64_t drain;
    float share[2][kRowTile];       // between the two threads of a row
    uint32_t tmem;
    volatile uint32_t abort;
};

template <uint32_t D, bool FP8> struct PrefillShape {
    static constexpr uint32_t kTiles = D == 256 ? 1 : 2; // query tiles
    static constexpr uint32_t kStep = kTiles == 1 ? 128 : 64; // keys of a score tile
    static constexpr uint32_t kSteps = kKeyTile / kStep;      // of a key tile
    static constexpr uint32_t kRows = kTiles * kRowTile;
    static constexpr uint32_t kWidth = FP8 && D == 64 ? 64 : 128; // bytes of a row in a panel of K, and of Q
    static constexpr uint32_t kPieceK = FP8 ? kKeyTile * kWidth : D == 64 ? 16384 : 32768, kPieceV = D == 64 || FP8 ? 16384 : 32768;
    static constexpr uint32_t kWarpsK = FP8 ? 1 : 3, kWarpsV = FP8 ? 4 : 2, kScaleWarps = FP8 ? 1 : 0;
    static constexpr uint32_t kLoadWarps = kWarpsK + kWarpsV + kScaleWarps;
    static constexpr uint32_t kQueryWarps = FP8 ? kWarpsV : kWarpsK; // load the queries too
    // of the rings
    static constexpr uint32_t kSlotsK = FP8 ? (D == 256 ? 3 : 2) : D == 64 ? 6 : 3, kSlotsV = FP8 || D == 64 ? 4 : 2;
    static constexpr uint32_t kStage = FP8 ? kPieceV / 2 : 0; // codes of a piece of V, for each warp that fetches them
    static constexpr uint32_t kScales = FP8 ? kScaleTiles * kKeyTile * 3 * 4 : 0;
    static constexpr uint32_t kQueryScales = FP8 ? 2 * kRows * 4 : 0;
    static constexpr uint32_t kPanels = kPieceK / (kKeyTile * kWidth); // of a piece of K
    static constexpr uint32_t kPieceKeys = kPieceV / (2 * D);          // of a piece of V
    static constexpr uint32_t kPerTileK = kKeyTile * D * (FP8 ? 1 : 2) / kPieceK, kPerTileV = kKeyTile / kPieceKeys; // pieces of a tile
    static constexpr uint32_t kQ = kRows * D * 2;
    static constexpr uint32_t kLoadWarp = kSoftmaxWarps;            // first of those that fetch
    static constexpr uint32_t kScoreWarp = kSoftmaxWarps + kLoadWarps;
    static constexpr uint32_t kThreads = (kSoftmaxWarps + kLoadWarps + 2) * 32;
    static constexpr uint32_t kRingK = kSlotsK * kPieceK, kRing = kRingK + kSlotsV * kPieceV;
    static constexpr uint32_t kSmem = 1024 + kQ + kRing + kWarpsV * kStage + kScales + kQueryScales + sizeof(Barriers);
    static_assert(kSlotsK % kWarpsK == 0 && kSlotsV % kWarpsV == 0, "a slot is one warp's");
    static_assert(kSmem <= 227 * 1024, "shared memory of a block");
    static_assert(kRing >= kMaxBatch * 8, "the search for the block's range uses the ring");
    static_assert(kSlotsK <= kMostSlots && kSlotsV <= kMostSlots, "barriers of the slots");
    static_assert(kThreads <= 512, "128 registers for each");
};

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
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

// Two codes in the low half, that of a in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x2(float a, float b)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t x)
{
    float2 r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(x));
    return r;
}
__device__ __forceinline__ float load_scale(const float* p, bool there)
{
    float r;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.global.nc.f32 %0, [%1];\n\t}"
                 : "=&f"(r)
                 : "l"(p), "r"(static_cast<uint32_t>(there)));
    return r;
}
__device__ __forceinline__ float log2_approx(float x)
{
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// What the place of a row's unit of 16 bytes is crossed with, rows being 128 or 64 bytes.
template <uint32_t WIDTH> __device__ __forceinline__ uint32_t swizzle_of(uint32_t row) { return WIDTH == 128 ? row & 7 : row >> 1 & 3; }

// Two floats in a register pair, one instruction for both.
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float low2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

template <uint32_t D, bool FP8>
__global__ void __launch_bounds__(PrefillShape<D, FP8>::kThreads, 1)
attn_prefill_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map, const uint32_t k_box, const uint32_t v_box)
{
    using Shape = PrefillShape<D, FP8>;
    constexpr uint32_t kWarpsK = Shape::kWarpsK, kWarpsV = Shape::kWarpsV;
    constexpr uint32_t TILES = Shape::kTiles, STEP = Shape::kStep, STEPS = Shape::kSteps, PANELS = Shape::kPanels, PIECE_KEYS = Shape::kPieceKeys;
    constexpr uint32_t PER_TILE_K = Shape::kPerTileK, PER_TILE_V = Shape::kPerTileV, SLOTS_K = Shape::kSlotsK, SLOTS_V = Shape::kSlotsV;
    constexpr uint32_t kPieceK = Shape::kPieceK, kPieceV = Shape::kPieceV, WIDTH = Shape::kWidth;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const ring = smem + Shape::kQ;
    uint8_t* const staging = ring + Shape::kRing;
    float* const scales = reinterpret_cast<float*>(staging + kWarpsV * Shape::kStage); // of a tile's key pairs: K's, log2 of V's; then 1 / V's
    float* const q_scales = scales + Shape::kScales / 4; // what the rows of queries were divided by, of this segment and the next
    Barriers& bar = *reinterpret_cast<Barriers*>(staging + kWarpsV * Shape::kStage + Shape::kScales + Shape::kQueryScales);
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;

    if (tid == 0) {
        for (uint32_t i = 0; i < kMostSlots; ++i) {
            mbar_init(&bar.k_full[i], 1);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.v_full[i], 1);
            mbar_init(&bar.v_empty[i], 1);
        }
        for (uint32_t i = 0; i < kScaleTiles; ++i)
            mbar_init(&bar.scale_full[i], 1);
        for (uint32_t i = 0; i < 4; ++i)
            mbar_init(&bar.staged[i], 1);
        mbar_init(&bar.q_full, Shape::kQueryWarps);
        mbar_init(&bar.q_free, 1);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.s_free[i], kSoftmaxWarps / TILES);
            mbar_init(&bar.o_free[i], kSoftmaxWarps / TILES);
            for (uint32_t j = 0; j < 2; ++j) {
                mbar_init(&bar.p_full[i][j], kSoftmaxWarps / TILES);
                mbar_init(&bar.pv_done[i][j], 1);
            }
        }
        mbar_init(&bar.drain, 2);
        bar.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == Shape::kScoreWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    const auto o_col = [&](uint32_t q) { return tmem + q * D; };
    const auto s_col = [&](uint32_t q) { return tmem + 256 + q * STEP; };
    const auto p_col = [&](uint32_t q, uint32_t step) { return tmem + 256 + TILES * STEP + (q * 2 + (step & 1)) * (STEP / 2); };
    chain_begin();

    const BlockRange range = find_range<Shape::kThreads>(p, reinterpret_cast<uint64_t*>(ring), blockIdx.x);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // boxes overwrite what the search wrote and read there
    __syncthreads();
    uint64_t left = range.end - range.begin;
    AttnPlace at = range.place;
    Segment seg; // every role follows the range for itself
    if (tid == 0)
        note_split(p, range);

    if (warp >= Shape::kLoadWarp && warp < Shape::kScoreWarp) {
        // ------------------------------------------------------------------------------ fetching --
        const uint32_t role = warp - Shape::kLoadWarp;
        const bool value = role >= kWarpsK && role < kWarpsK + kWarpsV, scaling = role >= kWarpsK + kWarpsV; // fetches V, the scales
        const uint32_t w = value ? role - kWarpsK : scaling ? 0 : role, warps = value ? kWarpsV : kWarpsK;
        const uint32_t slots = value ? SLOTS_V : SLOTS_K, piece_bytes = value ? kPieceV : kPieceK;
        uint64_t* const full_bar = value ? bar.v_full : bar.k_full;
        uint64_t* const empty_bar = value ? bar.v_empty : bar.k_empty;
        const uint32_t ring_at = smem_u32(ring) + (value ? Shape::kRingK : 0);
        Copies copies;
        uint32_t before = 0, segments = 0; // pieces of earlier segments
        uint32_t filled = 0;               // this warp's pieces so far, the n-th of them being number n * warps + w of all
        bool ok = true;
        bool boxed = false;                // e4m3: boxes are under way to this warp's staging area
        uint32_t staged_phase = 0;
        const auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
            if (__all_sync(0xffffffffu, mbar_test_wait(b, parity)))
                return true;
            copies.drain();
            return __all_sync(0xffffffffu, mbar_wait(b, parity, &bar.abort, p.err, code)) != 0;
        };
        while (ok && this_segment<false>(p, at, left, &seg)) {
            uint32_t seen_lo, seen_hi, unused;
            visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, p.tiling.group.div(seg.row0), &seen_lo, &unused);
            visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, p.tiling.group.div(seg.row0 + seg.nrows - 1), &unused, &seen_hi);
            seen_hi = min(seen_hi, seg.pages.room);

            const auto load_query = [&] {
                if (!wait(&bar.q_free, (segments & 1) ^ 1, ERR_PF_QUERY_WAIT))
                    return false;
                static_assert(Shape::kRows % 4 == 0, "four rows of a warp at a time");
#pragma unroll 1
                for (uint32_t r0 = w * 4; r0 < Shape::kRows; r0 += Shape::kQueryWarps * 4) {
                    const uint32_t r = r0 + lane / 8, in_tile = r & (kRowTile - 1);
                    const bool there = r < seg.nrows;
                    const uint32_t flat = seg.row0 + (there ? r : 0), token = p.tiling.group.div(flat);
                    const uint8_t* src = p.q + (seg.rows.row0 + token) * p.q_token
                        + (at.head * p.tiling.group.d + flat - token * p.tiling.group.d) * p.q_head + (lane & 7) * 16;
                    const uint32_t tile_at = (r / kRowTile) * (kRowTile * D * 2);
                    if constexpr (!FP8) {
                        const uint32_t dst = tile_at + in_tile * 128 + (((lane & 7) ^ (r & 7)) * 16);
#pragma unroll
                        for (uint32_t panel = 0; panel < D / 64; ++panel)
                            cp_async16(smem_u32(smem) + dst + panel * (kRowTile * 128), src + panel * 128, there);
                    } else {
                        uint4 v[D / 64];
                        uint32_t most = 0; // of the magnitudes, which are in the order of their bits
#pragma unroll
                        for (uint32_t panel = 0; panel < D / 64; ++panel) {
                            v[panel] = there ? *reinterpret_cast<const uint4*>(src + panel * 128) : make_uint4(0, 0, 0, 0);
                            const uint32_t a[4] = { v[panel].x, v[panel].y, v[panel].z, v[panel].w };
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j)
                                most = max(most, max(a[j] & 0x7fffu, a[j] >> 16 & 0x7fffu));
                        }
#pragma unroll
                        for (uint32_t o = 1; o < 8; o <<= 1)
                            most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                        // the power of two and its reciprocal are both f32's; a row with an infinity or a NaN becomes NaN
                        const int power = most >= 0x7f80u ? 0 : max(-126, min(126, 127 + 7 - static_cast<int>(most >> 7)));
                        const float up = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
                        if ((lane & 7) == 0)
                            q_scales[(segments & 1) * Shape::kRows + r] = __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
#pragma unroll
                        for (uint32_t panel = 0; panel < D / 64; ++panel) {
                            const uint32_t a[4] = { v[panel].x, v[panel].y, v[panel].z, v[panel].w };
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                const float x = bf16_bits_to_f32(a[j] & 0xffffu) * up, y = bf16_bits_to_f32(a[j] >> 16) * up;
                                hi[j] = most >= 0x7f80u ? 0x7f7fu : pack_e4m3x2(x, y);
                                const float2 h = f16x2_to_f32(e4m3x2_to_f16x2(hi[j]));
                                lo[j] = pack_e4m3x2(x - h.x, y - h.y);
                            }
                            const uint32_t at_byte = panel * 64 + (lane & 7) * 8, unit = at_byte % WIDTH / 16;
                            uint8_t* const dst = smem + tile_at + at_byte / WIDTH * (kRowTile * WIDTH) + in_tile * WIDTH
                                + ((unit ^ swizzle_of<WIDTH>(in_tile)) * 16) + at_byte % 16;
                            *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
                            *reinterpret_cast<uint2*>(dst + kRowTile * D) = make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
                        }
                    }
                }
                if constexpr (FP8) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar.q_full);
                } else {
                    __syncwarp();
                    copies.push(&bar.q_full);
                }
                return true;
            };

            const uint32_t pieces = seg.count * (value ? PER_TILE_V : PER_TILE_K);
            uint32_t mine = (w + warps - before % warps) % warps; // the first that goes to one of this warp's slots
            bool query = FP8 || value; // loaded, or not this warp's business
            if (FP8 && value) {
                // ---- V: codes to a staging area, from there to registers, and in f16 to the ring
                constexpr uint32_t UNITS = D / 16, AT_ONCE = 32 / UNITS, SETS = PIECE_KEYS / 32, LOADS = PIECE_KEYS / AT_ONCE;
                struct Places {
                    int32_t page[SETS]; // of keys lane + 32 j, or of the lane's box; not looked at yet
                    uint32_t slot[SETS];
                    bool boxes; // whole boxes of cached tokens
                };
                const auto first_key = [&](uint32_t piece) { return seg.tile0 * kKeyTile + piece * PIECE_KEYS; };
                const auto look = [&](uint32_t piece) {
                    Places l;
                    const uint32_t key0 = first_key(piece);
                    l.boxes = v_box != 0 && key0 >= seen_lo && key0 + PIECE_KEYS <= seg.pages.room;
#pragma unroll
                    for (uint32_t j = 0; j < SETS; ++j) {
                        const uint32_t key = key0 + (l.boxes ? lane * v_box : j * 32 + lane);
                        l.page[j] = -1;
                        l.slot[j] = 0;
                        if (l.boxes ? j == 0 && lane * v_box < PIECE_KEYS : key >= seen_lo && key < seen_hi) {
                            const uint32_t i = p.view.page_div.div(key);
                            l.slot[j] = key - i * p.view.page_size;
                            l.page[j] = __ldg(p.view.indices + seg.pages.first + i);
                        }
                    }
                    return l;
                };
                uint8_t* const stage = staging + w * Shape::kStage;
                const auto fetch = [&](uint32_t piece, Places l) {
                    const uint32_t key0 = first_key(piece), stage_at = smem_u32(stage);
                    if (l.boxes) {
                        const bool mine = lane * v_box < PIECE_KEYS, bad = mine && static_cast<uint32_t>(l.page[0]) >= p.view.pages;
                        boxed = !__any_sync(0xffffffffu, bad);
                        if (boxed) {
                            if (lane == 0)
                                mbar_expect_tx(&bar.staged[w], Shape::kStage);
                            __syncwarp();
                            if (mine)
                                tma_load_page(stage_at + lane * v_box * D, &v_map, &bar.staged[w], 0, static_cast<int>(l.slot[0]),
                                              static_cast<int>(at.head), l.page[0]);
                            return;
                        }
                    }
                    uint32_t row[SETS];
#pragma unroll
                    for (uint32_t j = 0; j < SETS; ++j) {
                        const uint32_t key = key0 + j * 32 + lane;
                        const bool seen = key >= seen_lo && key < seen_hi;
                        if (l.boxes) // one of the boxes' pages is not there
                            l.page[j] = seen ? page_of(p.view, seg.pages, key, &l.slot[j]) : -1;
                        const bool there = static_cast<uint32_t>(l.page[j]) < p.view.pages;
                        if (seen && !there)
                            atomicCAS(p.err, 0u, static_cast<uint32_t>(ERR_PAGE_TABLE));
                        row[j] = row_units(p.view.v, there ? l.page[j] : -1, l.slot[j]);
                    }
                    const uint8_t* const from = p.view.v.data + at.head * p.view.v.head_stride + (lane % UNITS) * 16;
#pragma unroll
                    for (uint32_t j = 0; j < LOADS; ++j) {
                        const uint32_t r = __shfl_sync(0xffffffffu, row[j * AT_ONCE / 32], (j * AT_ONCE + lane / UNITS) & 31);
                        cp_async16(stage_at + (j * 32 + lane) * 16, from + row_bytes(p.view.v, r), r != kNoRow);
                    }
                };
                Places ahead;
                if (mine < pieces) {
                    fetch(mine, look(mine));
                    if (mine + kWarpsV < pieces)
                        ahead = look(mine + kWarpsV);
                }
                ok = load_query();
                for (; ok && mine < pieces; mine += kWarpsV) {
                    if (boxed) {
                        ok = wait(&bar.staged[w], staged_phase, ERR_PF_FULL_WAIT);
                        if (!ok)
                            break;
                        staged_phase ^= 1;
                        boxed = false;
                    } else {
                        asm volatile("cp.async.wait_all;" ::: "memory"); // (a lane reads what it copied)
                    }
                    uint4 codes[LOADS];
#pragma unroll
                    for (uint32_t j = 0; j < LOADS; ++j)
                        codes[j] = *reinterpret_cast<const uint4*>(stage + (j * 32 + lane) * 16);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // before boxes overwrite them
                    __syncwarp();
                    if (mine + kWarpsV < pieces) {
                        fetch(mine + kWarpsV, ahead);
                        if (mine + 2 * kWarpsV < pieces)
                            ahead = look(mine + 2 * kWarpsV);
                    }
                    const uint32_t s = (before + mine) % SLOTS_V;
                    ok = wait(&empty_bar[s], (((before + mine) / SLOTS_V) & 1) ^ 1, ERR_PF_EMPTY_WAIT);
                    if (!ok)
                        break;
                    uint8_t* const to = ring + Shape::kRingK + s * kPieceV + lane % UNITS / 4 * (PIECE_KEYS * 128);
#pragma unroll
                    for (uint32_t j = 0; j < LOADS; ++j) {
                        const uint32_t key = j * AT_ONCE + lane / UNITS, first = lane % 4 * 2;
                        const uint32_t x[4] = { codes[j].x, codes[j].y, codes[j].z, codes[j].w };
                        uint32_t y[8];
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            y[k] = e4m3x2_to_f16x2(x[k / 2] >> (16 * (k & 1)));
                        *reinterpret_cast<uint4*>(to + key * 128 + ((first ^ (key & 7)) * 16)) = make_uint4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<uint4*>(to + key * 128 + (((first + 1) ^ (key & 7)) * 16)) = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the tensor core reads what was written here
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&full_bar[s]);
                }
                before += pieces;
                ++segments;
                next_segment(p, seg, &at, &left);
                continue;
            }
            if (FP8 && scaling) {
                // ---- scales of K and V; pages of a tile are looked up two tiles ahead, its scales one
                struct Tile { // of keys lane + 32 j
                    int32_t page[kKeyTile / 32];
                    uint32_t slot[kKeyTile / 32];
                    float k[kKeyTile / 32], v[kKeyTile / 32];
                };
                const auto seen = [&](uint32_t tile, uint32_t j) {
                    const uint32_t key = (seg.tile0 + tile) * kKeyTile + j * 32 + lane;
                    return key >= seen_lo && key < seen_hi;
                };
                const auto look = [&](uint32_t tile) {
                    Tile t;
#pragma unroll
                    for (uint32_t j = 0; j < kKeyTile / 32; ++j) {
                        const uint32_t key = (seg.tile0 + tile) * kKeyTile + j * 32 + lane;
                        t.page[j] = -1;
                        t.slot[j] = 0;
                        if (seen(tile, j)) {
                            const uint32_t i = p.view.page_div.div(key);
                            t.slot[j] = key - i * p.view.page_size;
                            t.page[j] = __ldg(p.view.indices + seg.pages.first + i);
                        }
                    }
                    return t;
                };
                const uint8_t* const k_scale = reinterpret_cast<const uint8_t*>(p.view.k.scale + at.head * p.view.k.scale_head_stride);
                const uint8_t* const v_scale = reinterpret_cast<const uint8_t*>(p.view.v.scale + at.head * p.view.v.scale_head_stride);
                const auto load_scales = [&](Tile& t) { // (who fetches the rows reports a page that is not there)
#pragma unroll
                    for (uint32_t j = 0; j < kKeyTile / 32; ++j) {
                        const bool there = static_cast<uint32_t>(t.page[j]) < p.view.pages;
                        t.k[j] = load_scale(scale_at(p.view.k, k_scale, t.page[j], t.slot[j]), there);
                        t.v[j] = load_scale(scale_at(p.view.v, v_scale, t.page[j], t.slot[j]), there);
                    }
                };
                Tile next = look(0), after = next;
                if (seg.count > 1)
                    after = look(1);
                load_scales(next);
                for (uint32_t tile = 0; ok && tile < seg.count; ++tile) {
                    const Tile t = next;
                    next = after;
                    if (tile + 2 < seg.count)
                        after = look(tile + 2);
                    if (tile + 1 < seg.count)
                        load_scales(next);
                    // The place is free when the weights of four tiles ago are written. Those of the first query tile two steps
                    // before this tile's first stand for that: the second one's scores of the step before had been asked for by
                    // then, and its scores of the step before that one been read. The weights of this barrier's next phase need
                    // these scales, so the parity stands for the phase that is meant.
                    const uint32_t number = before + tile, place = number % kScaleTiles;
                    if (number * STEPS >= 2) {
                        const uint32_t step = number * STEPS - 2;
                        ok = wait(&bar.p_full[0][step & 1], (step >> 1) & 1, ERR_PF_WEIGHT_WAIT);
                        if (!ok)
                            break;
                    }
                    float* const out = scales + place * (kKeyTile * 3);
#pragma unroll
                    for (uint32_t j = 0; j < kKeyTile / 32; ++j) {
                        const uint32_t key = j * 32 + lane;
                        const float v = t.v[j] < 1.0e-30f ? 1.0e-30f : t.v[j]; // (a NaN stays one)
                        out[key / 2 * 4 + (key & 1)] = t.k[j] * p.scale_log2;
                        out[key / 2 * 4 + 2 + (key & 1)] = log2_approx(v);
                        out[kKeyTile * 2 + key] = __fdividef(kSumFactor<FP8>, v);
                    }
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar.scale_full[place]);
                }
                before += seg.count;
                ++segments;
                next_segment(p, seg, &at, &left);
                continue;
            }
            // A warp looks up the pages of its next piece before it waits for room.
            struct Ahead {
                uint32_t key0, slot; // slot, page: of this lane's box
                int32_t page;
                bool boxes;          // whole boxes of cached tokens
            };
            const auto look = [&](uint32_t piece) { // of the segment
                Ahead a;
                a.key0 = seg.tile0 * kKeyTile + (value ? piece * PIECE_KEYS : piece / PER_TILE_K * kKeyTile);
                const uint32_t keys = value ? PIECE_KEYS : kKeyTile, box = value ? v_box : k_box;
                a.slot = 0;
                a.page = 0;
                a.boxes = box != 0 && a.key0 >= seen_lo && a.key0 + keys <= seg.pages.room;
                if (a.boxes) {
                    const uint32_t per_panel = keys / box, panels = value ? D / 64 : PANELS;
                    if (lane < per_panel * panels)
                        a.page = page_of(p.view, seg.pages, a.key0 + lane % per_panel * box, &a.slot);
                }
                return a;
            };
            // KEYS keys, UNITS units of 16 bytes of each from `skip` bytes on, to panels of 64 elements
            const auto load = [&](uint32_t piece, const Ahead& a, const PagedPool& pool, const CUtensorMap& map, uint32_t box, auto keys, auto units,
                                  uint32_t skip) {
                constexpr uint32_t KEYS = decltype(keys)::value, UNITS = decltype(units)::value, AT_ONCE = 32 / UNITS;
                const uint32_t s = (before + piece) % slots;
                const bool boxes = a.boxes && __all_sync(0xffffffffu, a.page >= 0);
                // otherwise the rows of keys lane + 32 j
                uint32_t row[KEYS / 32];
                if (!boxes) {
#pragma unroll
                    for (uint32_t j = 0; j < KEYS / 32; ++j) {
                        const uint32_t key = a.key0 + j * 32 + lane;
                        uint32_t slot = 0;
                        row[j] = row_units(pool, key >= seen_lo && key < seen_hi ? page_of(p.view, seg.pages, key, &slot) : -1, slot);
                    }
                }
                if (!wait(&empty_bar[s], (((before + piece) / slots) & 1) ^ 1, ERR_PF_EMPTY_WAIT))
                    return false;
                if (boxes) {
                    const uint32_t per_panel = KEYS / box;
                    if (lane == 0)
                        mbar_expect_tx(&full_bar[s], piece_bytes);
                    __syncwarp();
                    if (lane < per_panel * ((UNITS + 7) / 8)) {
                        const uint32_t panel = lane / per_panel, first = (lane - panel * per_panel) * box;
                        tma_load_page(ring_at + s * piece_bytes + panel * (KEYS * 128) + first * WIDTH, &map, &full_bar[s],
                                      static_cast<int>(skip / (FP8 ? 1 : 2) + panel * 64), static_cast<int>(a.slot), static_cast<int>(at.head),
                                      a.page);
                    }
                    ++filled;
                    return true;
                }
                const uint8_t* const from = pool.data + at.head * pool.head_stride + skip + (lane % UNITS) * 16;
                const uint32_t to = ring_at + s * piece_bytes + (lane % UNITS / 8) * (KEYS * 128);
#pragma unroll
                for (uint32_t j = 0; j < KEYS / AT_ONCE; ++j) {
                    const uint32_t key = j * AT_ONCE + lane / UNITS;
                    const uint32_t r = __shfl_sync(0xffffffffu, row[j * AT_ONCE / 32], key & 31);
                    cp_async16(to + key * WIDTH + ((lane % (WIDTH / 16) ^ swizzle_of<WIDTH>(key)) * 16),
                                from + row_bytes(pool, r), r != kNoRow);
                }
                copies.push(&full_bar[s]);
                ++filled;
                return true;
            };
            Ahead ahead;
            if (mine < pieces)
                ahead = look(mine);
            for (; ok && mine < pieces; mine += warps) {
                const Ahead a = ahead;
                if (mine + warps < pieces)
                    ahead = look(mine + warps);
                ok = !FP8 && value ? load(mine, a, p.view.v, v_map, v_box, std::integral_constant<uint32_t, PIECE_KEYS> {},
                                  std::integral_constant<uint32_t, D / 8> {}, 0)
                           : load(mine, a, p.view.k, k_map, k_box, std::integral_constant<uint32_t, kKeyTile> {},
                                  std::integral_constant<uint32_t, WIDTH / 16 * PANELS> {}, mine % PER_TILE_K * (PANELS * WIDTH));
                if (ok && !query) { // behind the first piece, which may find room before the queries do
                    ok = load_query();
                    query = true;
                }
            }
            if (ok && !query)
                ok = load_query();
            before += pieces;
            ++segments;
            next_segment(p, seg, &at, &left);
        }
        copies.drain();
        if (!ok) { // a wait gave up: boxes that are under way still write to this block's memory
            volatile uint32_t never = 0;
            if (boxed)
                mbar_wait(&bar.staged[w], staged_phase, &never, p.err, ERR_PF_FULL_WAIT);
            for (uint32_t n = filled - min(filled, slots / warps); n < filled; ++n)
                mbar_wait(&full_bar[(n * warps + w) % slots], (n * warps + w) / slots & 1, &never, p.err, ERR_PF_FULL_WAIT);
        }
    } else if (warp >= Shape::kScoreWarp) {
        // ------------------------------------------------------------------------------- products --
        // The whole warp goes through the loops and one lane issues.
        constexpr uint32_t kFormat = (1u << 4) | (FP8 ? 0u : (1u << 7) | (1u << 10)) | ((kRowTile >> 4) << 24); // f16 or bf16 -> f32
        constexpr uint32_t kScores = kFormat | ((STEP >> 3) << 17);
        constexpr uint32_t kSums = kFormat | ((D >> 3) << 17) | (1u << 16);
        constexpr uint64_t kOperand = (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
        constexpr uint64_t kNarrow = (static_cast<uint64_t>(512 >> 4) << 32) | (1ull << 46) | (4ull << 61); // rows of 64 bytes
        constexpr uint64_t kRow = WIDTH == 64 ? kNarrow : kOperand;
        // V as the B operand with its n side contiguous: panels of 64 elements, keys 128 bytes apart, groups of eight keys 1024
        constexpr uint64_t kValue = kOperand | (static_cast<uint64_t>(PIECE_KEYS * 128 >> 4) << 16);
        const auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
        const uint32_t ring_lo = uniform(smem_u32(ring) >> 4), query_lo = uniform(smem_u32(smem) >> 4), columns = uniform(tmem);
        uint32_t before = 0, segments = 0;   // key tiles of earlier segments
        uint32_t done[2] = {}, segs[2] = {}; // steps and segments of a query tile
        bool ok = true;
        const auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
            return __all_sync(0xffffffffu, mbar_wait<true>(b, parity, &bar.abort, p.err, code)) != 0;
        };
        // Scores of step u of the segment, once the last ones have been read. The last to use a piece of K lets go of it.
        const auto scores = [&](uint32_t u, uint32_t q, bool last) {
            const uint32_t d = columns + 256 + q * STEP;
            if (!wait(&bar.s_free[q], (done[q] & 1) ^ 1, ERR_PF_SUM_WAIT))
                return false;
            tc_fence_after();
            const uint32_t part = u % STEPS; // of the key tile
#pragma unroll
            for (uint32_t i = 0; i < PER_TILE_K; ++i) {
                const uint32_t piece = (before + u / STEPS) * PER_TILE_K + i, s = piece % SLOTS_K;
                if (part == 0 && q == 0 && !wait(&bar.k_full[s], (piece / SLOTS_K) & 1, ERR_PF_FULL_WAIT))
                    return false;
                const uint32_t a_lo = query_lo + (q * (kRowTile * D * 2) + i * (PANELS * kRowTile * WIDTH)) / 16;
                const uint32_t b_lo = uniform(ring_lo + (s * kPieceK + part * (STEP * WIDTH)) / 16);
                if (elect_one()) {
                    if constexpr (FP8) {
#pragma unroll
                        for (uint32_t j = 0; j < WIDTH / 16; ++j) { // 32 elements each: of the queries' high parts, of the low ones
                            const uint32_t k = j % (WIDTH / 32) * 2, low = j / (WIDTH / 32) * (kRowTile * D / 16);
                            tc_mma_f8(d, kRow | (a_lo + low + k), kRow | (b_lo + k), kScores, i > 0 || j > 0);
                        }
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 4 * PANELS; ++j) {
                            const uint32_t k = j / 4 * (kKeyTile * 128 / 16) + j % 4 * 2; // (query tiles are as high as key tiles)
                            tc_mma_bf16(d, kOperand | (a_lo + k), kOperand | (b_lo + k), kScores, i > 0 || j > 0);
                        }
                    }
                    if (last && part + 1 == STEPS)
                        tc_commit(&bar.k_empty[s]);
                    if (i + 1 == PER_TILE_K)
                        tc_commit(&bar.s_full[q]);
                }
            }
            ++done[q];
            return true;
        };
        // A step's keys are one or more pieces of V, or a part of one.
        constexpr bool WHOLE = PER_TILE_V >= STEPS;
        constexpr uint32_t OF_STEP = WHOLE ? PER_TILE_V / STEPS : 1;
        const auto sums = [&](uint32_t u, uint32_t q, bool last) {
            const uint32_t half = done[q] & 1, part = u % STEPS;
            const uint32_t d = columns + q * D, a = columns + 256 + TILES * STEP + (q * 2 + half) * (STEP / 2);
            if (u == 0 && !wait(&bar.o_free[q], (segs[q] & 1) ^ 1, ERR_PF_SUM_WAIT))
                return false;
#pragma unroll
            for (uint32_t i = 0; i < OF_STEP; ++i) {
                const uint32_t piece = before * PER_TILE_V + (WHOLE ? u * OF_STEP + i : u / STEPS), s = piece % SLOTS_V;
                if ((WHOLE || part == 0) && q == 0 && !wait(&bar.v_full[s], (piece / SLOTS_V) & 1, ERR_PF_FULL_WAIT))
                    return false;
                if (i == 0) {
                    if (!wait(&bar.p_full[q][half], (done[q] >> 1) & 1, ERR_PF_WEIGHT_WAIT))
                        return false;
                    tc_fence_after();
                }
                const uint32_t b_lo = uniform(ring_lo + (Shape::kRingK + s * kPieceV) / 16 + (WHOLE ? 0 : part * (STEP * 128 / 16)));
                constexpr uint32_t COUNT = STEP / OF_STEP / 16; // products of 16 keys: 2048 bytes of V, eight columns of P
                if (elect_one()) {
#pragma unroll
                    for (uint32_t j = 0; j < COUNT; ++j)
                        mma_ts(d, a + (i * COUNT + j) * 8, kValue | (b_lo + j * (2048 >> 4)), kSums, u > 0 || i > 0 || j > 0);
                    if (i + 1 == OF_STEP)
                        tc_commit(&bar.pv_done[q][half]);
                    if (last && (WHOLE || part + 1 == STEPS))
                        tc_commit(&bar.v_empty[s]);
                }
            }
            ++done[q];
            return true;
        };
        while (ok && this_segment<false>(p, at, left, &seg)) {
            const uint32_t n = uniform(seg.count);
            const bool second = TILES == 2 && uniform(seg.nrows) > kRowTile, score = warp == Shape::kScoreWarp;
            if (score)
                ok = wait(&bar.q_full, segments & 1, ERR_PF_QUERY_WAIT);
            for (uint32_t u = 0; ok && u < n * STEPS; ++u)
#pragma unroll
                for (uint32_t q = 0; q < TILES; ++q)
                    if (ok && (q == 0 || second))
                        ok = score ? scores(u, q, q == 1 || !second) : sums(u, q, q == 1 || !second);
            if (score && elect_one())
                tc_commit(&bar.q_free);
            ++segs[0];
            segs[1] += second ? 1 : 0;
            ++segments;
            before += n;
            next_segment(p, seg, &at, &left);
        }
        // whatever was issued is complete before the tensor memory goes back
        volatile uint32_t never = 0;
        if (elect_one())
            tc_commit(&bar.drain);
        mbar_wait<true>(&bar.drain, 0, &never, p.err, ERR_PF_SUM_WAIT);
        __syncwarp();
    } else if (warp < kSoftmaxWarps) {
        // -------------------------------------------------------------------------------- weights --
        const uint32_t q = TILES == 1 ? 0 : warp / 4, half = TILES == 1 ? warp / 4 : 0;
        const uint32_t lanes = (warp & 3) << 21, tile_row = (warp & 3) * 32 + lane; // 32 lanes of tensor memory
        uint32_t done = 0, segments = 0, tiles_before_this = 0;                     // steps; key tiles of earlier segments
        bool ok = true;
        const auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
            const bool r = __all_sync(0xffffffffu, mbar_wait(b, parity, &bar.abort, p.err, code)) != 0;
            tc_fence_after();
            return r;
        };
        // The sums of step `d`. Those of d - 2 are awaited before the weights of d are written, so the parity stands for this step.
        const auto wait_sums = [&](uint32_t d) { return wait(&bar.pv_done[q][d & 1], (d >> 1) & 1, ERR_PF_SUM_WAIT); };
        // True in all threads of the rows that this warp has a part in, where `v` is in any.
        const auto any = [&](bool v) {
            if constexpr (TILES == 2)
                return __any_sync(0xffffffffu, v) != 0;
            return !group_all(1 + (warp & 3), 64, !v);
        };
        while (ok && this_segment<false>(p, at, left, &seg)) {
            const uint32_t steps = seg.count * STEPS;
            if (q * kRowTile < seg.nrows) {
                const uint32_t r = q * kRowTile + tile_row;
                const bool live = r < seg.nrows, idle = !__any_sync(0xffffffffu, live);
                const uint32_t flat = seg.row0 + (live ? r : 0), token = p.tiling.group.div(flat);
                uint32_t lo = 0, hi = 0xffffffffu; // (rows past the last one need no mask)
                if (live) {
                    visible_keys(p.tiling, seg.rows.fresh, seg.pages.length, token, &lo, &hi);
                    hi = min(hi, seg.pages.room);
                }
                float m = -INFINITY, l = 0.0f, q_scale = 1.0f;
                for (uint32_t u = 0; u < steps; ++u, ++done) {
                    ok = wait(&bar.s_full[q], done & 1, ERR_PF_SCORE_WAIT);
                    uint32_t x[kMine];
                    if (!idle) {
                        tc_ld32(s_col(q) + lanes + half * kMine, x);
                        tc_ld32(s_col(q) + lanes + half * kMine + 32, x + 32);
                        tc_ld_wait32(x);
                        tc_ld_wait32(x + 32);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar.s_free[q]);
                    if (done >= 2)
                        ok = wait_sums(done - 2) && ok;
                    const uint32_t in_tile = u % STEPS * STEP + half * kMine; // this thread's first key
                    const float* scale = nullptr;
                    if constexpr (FP8) {
                        const uint32_t tile = tiles_before_this + u / STEPS;
                        ok = wait(&bar.scale_full[tile % kScaleTiles], (tile / kScaleTiles) & 1, ERR_PF_SCORE_WAIT) && ok;
                        scale = scales + tile % kScaleTiles * (kKeyTile * 3);
                        if (u == 0)
                            q_scale = q_scales[(segments & 1) * Shape::kRows + r];
                    }
                    if (idle && !ok)
                        break;
                    if (!idle) {
                        const uint32_t key0 = (seg.tile0 + u / STEPS) * kKeyTile + in_tile;
                        if constexpr (FP8) {
                            const uint64_t q2 = pack2(q_scale, q_scale);
#pragma unroll
                            for (uint32_t j = 0; j < kMine / 2; ++j) {
                                const float4 kv = *reinterpret_cast<const float4*>(scale + (in_tile / 2 + j) * 4);
                                const uint64_t e = fma2(mul2(pack2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), q2),
                                                        pack2(kv.x, kv.y), pack2(kv.z, kv.w));
                                x[2 * j] = static_cast<uint32_t>(e);
                                x[2 * j + 1] = static_cast<uint32_t>(e >> 32);
                            }
                        }
                        const bool part = __any_sync(0xffffffffu, lo > key0 || hi < key0 + kMine);
                        if (part) {
#pragma unroll
                            for (uint32_t j = 0; j < kMine; ++j)
                                x[j] = key0 + j >= lo && key0 + j < hi ? x[j] : 0xff800000u; // -infinity
                        }
                        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
                        for (uint32_t j = 0; j < kMine; j += 4) {
                            top0 = fmaxf(top0, fmaxf(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
                            top1 = fmaxf(top1, fmaxf(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])));
                        }
                        float top = FP8 ? fmaxf(top0, top1) : fmaxf(top0, top1) * p.scale_log2;
                        if (any(!ok || top > m + kGrowth<FP8>)) { // (m = -inf: whenever something is seen)
                            if constexpr (TILES == 1) // the two warps of a row stop together
                                ok = group_all(1 + (warp & 3), 64, ok);
                            if (!ok)
                                break;
                            if constexpr (TILES == 1) {
                                bar.share[half][tile_row] = top;
                                group_all(1 + (warp & 3), 64, true);
                                top = fmaxf(top, bar.share[half ^ 1][tile_row]);
                            }
                            const bool grow = top > m + kGrowth<FP8>;
                            const float next = grow ? top : m;
                            const float keep = grow ? exp2_fast(m - next) : 1.0f;
                            m = next;
                            l *= keep;
                            if (u > 0) { // O holds the sums up to step u - 1 once they are through
                                ok = wait_sums(done - 1);
                                if (ok) {
                                    uint32_t o[32];
#pragma unroll 1
                                    for (uint32_t c = 0; c < D / 32 / (TILES == 1 ? 2 : 1); ++c) {
                                        const uint32_t o_addr = o_col(q) + half * (D / 2) + lanes + c * 32;
                                        tc_ld32(o_addr, o);
                                        tc_ld_wait32(o);
#pragma unroll
                                        for (uint32_t j = 0; j < 32; ++j)
                                            o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                                        tc_st16(o_addr, o);
                                        tc_st16(o_addr + 16, o + 16);
                                    }
                                }
                            }
                        }
                        const float base = m == -INFINITY ? 0.0f : m - kTop<FP8>;
                        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), base2 = pack2(-base, -base);
                        uint64_t sum2 = pack2(0.0f, 0.0f);
#pragma unroll
                        for (uint32_t c = 0; c < kMine / 32; ++c) {
                            uint32_t w[16];
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) {
                                const uint32_t i = c * 32 + 2 * j;
                                const uint64_t x2 = pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                                const uint64_t e = FP8 ? add2(x2, base2) : fma2(x2, scale2, base2);
                                const float a = exp2_fast(low2(e)), b = exp2_fast(high2(e));
                                if constexpr (FP8) {
                                    const float2 inv = *reinterpret_cast<const float2*>(scale + kKeyTile * 2 + in_tile + i);
                                    sum2 = fma2(pack2(a, b), pack2(inv.x, inv.y), sum2);
                                    w[j] = pack_f16x2(a, b);
                                } else {
                                    sum2 = add2(sum2, pack2(a, b));
                                    w[j] = pack_bf16x2(a, b);
                                }
                            }
                            tc_st16(p_col(q, done) + lanes + half * (kMine / 2) + c * 16, w);
                        }
                        l += low2(sum2) + high2(sum2);
                        tc_st_wait();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar.p_full[q][done & 1]);
                }
                ok = ok && wait_sums(done - 1);
                if constexpr (TILES == 1) {
                    ok = group_all(1 + (warp & 3), 64, ok);
                    bar.share[half][tile_row] = l;
                    group_all(1 + (warp & 3), 64, true);
                    l += bar.share[half ^ 1][tile_row];
                }
                if (!ok)
                    break;
                const bool whole = seg.whole;
                if (whole && m == -INFINITY) // as in without_scores
                    l = lo < hi ? __int_as_float(0x7fffffff) : 0.0f;
                // in units of the sums: O counts 2^kSumUnit times too much
                if (m != -INFINITY)
                    m += kSumUnit<FP8> - kTop<FP8>;
                const uint32_t h = at.head * p.tiling.group.d + flat - token * p.tiling.group.d;
                const size_t part_row = static_cast<size_t>(blockIdx.x * 2 + (seg.starts ? 1 : 0)) * Shape::kRows + r;
                uint8_t* const out = p.out + (seg.rows.row0 + token) * p.out_token + h * p.out_head;
                float* const part_o = p.part_o + part_row * D;
                const float inv = whole ? (m == -INFINITY ? l : kSumFactor<FP8> / l) : kSumFactor<FP8>;
                uint32_t x[32];
#pragma unroll 1
                for (uint32_t i = 0; i < D / 32 / (TILES == 1 ? 2 : 1); ++i) {
                    const uint32_t c = half * (D / 64) + i;
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
                            *reinterpret_cast<float4*>(part_o + c * 32 + j * 4)
                                = make_float4(__uint_as_float(x[4 * j]) * inv, __uint_as_float(x[4 * j + 1]) * inv,
                                              __uint_as_float(x[4 * j + 2]) * inv, __uint_as_float(x[4 * j + 3]) * inv);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&bar.o_free[q]);
                if (live && whole && half == 0 && p.lse != nullptr)
                    p.lse[(seg.rows.row0 + token) * p.lse_token + h * p.lse_head]
                        = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
                if (live && !whole && half == 0)
                    p.part_ml[part_row] = make_float2(m, l);
            }
            tiles_before_this += seg.count;
            ++segments;
            next_segment(p, seg, &at, &left);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Shape::kScoreWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <uint32_t D, bool FP8> cudaError_t launch_prefill_as(const AttnParams& p, cudaStream_t stream)
{
    using Shape = PrefillShape<D, FP8>;
    const cudaError_t err = cudaFuncSetAttribute(attn_prefill_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (err != cudaSuccess)
        return err;
    // Pages that a box fits into a whole number of times are fetched by TMA, others and the ends of sequences row by row.
    const auto box = [&](CUtensorMap* map, const PagedPool& pool, uint32_t most, uint32_t bytes, bool swizzle) {
        const uint32_t size = p.view.page_size;
        const uint32_t rows = size < most ? size : most;
        const uint64_t dims[4] = { D, size, p.view.kv_heads, p.view.pages };
        const uint64_t strides[3] = { static_cast<uint64_t>(pool.slot_stride), static_cast<uint64_t>(pool.head_stride),
                                      static_cast<uint64_t>(pool.page_stride) };
        if (rows < 8 || size % rows != 0 || most % rows != 0 || !make_page_map(map, FP8, pool.data, dims, strides, bytes, rows, swizzle))
            return 0u;
        return rows;
    };
    CUtensorMap k_map {}, v_map {};
    const uint32_t k_box = box(&k_map, p.view.k, kKeyTile, Shape::kWidth, true);
    const uint32_t v_box = box(&v_map, p.view.v, Shape::kPieceKeys, FP8 ? D : 128, !FP8);
    return launch_chained(attn_prefill_kernel<D, FP8>, dim3(p.blocks), Shape::kThreads, Shape::kSmem, stream, p, k_map, v_map, k_box, v_box);
}

} // namespace

uint32_t attn_prefill_rows(uint32_t head_dim) { return head_dim == 256 ? kRowTile : 2 * kRowTile; }

cudaError_t launch_attn_prefill(const AttnParams& p, bool fp8, cudaStream_t stream)
{
    const uint32_t d = p.view.head_dim;
    if (fp8)
        return d == 64 ? launch_prefill_as<64, true>(p, stream)
            : d == 128 ? launch_prefill_as<128, true>(p, stream)
                       : launch_prefill_as<256, true>(p, stream);
    return d == 64 ? launch_prefill_as<64, false>(p, stream)
        : d == 128 ? launch_prefill_as<128, false>(p, stream)
                   : launch_prefill_as<256, false>(p, stream);
}

} // namespace qs3
