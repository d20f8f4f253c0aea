// Attention of a few new tokens per sequence over a paged KV cache (decode), and the join of results that were split along the
// context; the entry points choose between this kernel and the tensor-memory one for chunks (paged_prefill.cu).
//
//   s_j = scale q.k_j,  m = max_j s_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum_j exp(s_j - m)
//
// in one pass over the keys with a running maximum and sum. A row does 2 D multiplications per cached byte or less, so the
// cache's stream from HBM is the bound and the point of the layout: every warp is on its own. It streams 16 keys at a time
// through its own ring in shared memory (cp.async, three stages), and the only barriers are those at an item's ends. The
// products run on the tensor cores with the keys on the M side and the rows (at most 16: query heads that share the KV head,
// times new tokens) on the N side of m16n8k16: S^T = K Q^T, then O^T += V^T P^T, so that no row of a tile is padding when eight
// heads share a KV head, and the running maximum of a row sits in the lane that rescales it.
//
// e4m3 caches are multiplied in f16 as in paged_prefill.cu: queries scaled by powers of two, K's scales a factor on the scores, V's
// scales part of the weights. (With codes moved to bf16 by integer instructions, five for two codes instead of one conversion,
// the kernel waited for those: 66 sequences of up to 16 384 tokens 335 us.)
#include "paged_attention.cuh"
#include "tcgen05.cuh"

#include <cmath>

namespace qs3 {

namespace {

constexpr uint32_t kStreamWarps = 4;
constexpr uint32_t kStreamThreads = kStreamWarps * 32;
constexpr uint32_t kWarpKeys = 16;
constexpr uint32_t kStreamKeys = kStreamWarps * kWarpKeys; // of a key tile
constexpr uint32_t kStreamStages = 3;

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <bool F16> __device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async4z(uint32_t dst, const void* src, uint32_t there)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait_group()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// e4m3: where the largest weight lies, in powers of two (f16 ends at 2^16 and loses bits below 2^-14), and a factor on 1 / scale
// of V, at most 1e30, so that sums of a long row of zeros stay finite.
template <bool FP8> constexpr float kTop = FP8 ? 14.0f : 0.0f;
template <bool FP8> constexpr float kSumUnit = FP8 ? 20.0f : 0.0f;
template <bool FP8> constexpr float kSumFactor = FP8 ? 1.0f / 1048576.0f : 1.0f;

template <uint32_t D, uint32_t NT, bool FP8> struct StreamShape {
    static constexpr uint32_t kRows = 8 * NT;
    static constexpr uint32_t kRowBytes = D * (FP8 ? 1 : 2);
    static constexpr uint32_t kHalf = kWarpKeys * kRowBytes;                       // K or V of a stage
    static constexpr uint32_t kStage = 2 * kHalf + (FP8 ? 2 * kWarpKeys * 4 : 0);  // and scales
    static constexpr uint32_t kRing = kStreamWarps * kStreamStages * kStage;
    static constexpr uint32_t kQ = kRows * D * 2;
    // after the last tile of an item the ring holds the warps' sums instead
    static constexpr uint32_t kSums = kStreamWarps * kRows * D * 4;
    // and before its first the costs of the sequences
    static constexpr uint32_t kCosts = kMaxBatch * 8;
    static constexpr uint32_t kLarger = kRing > kSums ? kRing : kSums;
    static constexpr uint32_t kUnion = kLarger > kCosts ? kLarger : kCosts;
    static constexpr uint32_t kSmem = kUnion + kQ + kStreamWarps * kRows * 8 + (FP8 ? kRows * 4 : 0);
    // per SM, by shared memory and by 128 registers a thread where that is more than two
    static constexpr uint32_t kFit = 227 * 1024 / (kSmem + 1024);
    static constexpr uint32_t kBlocks = kFit < 4 ? kFit : 4;
};

// Byte offset of 16-byte unit `c` of row `r`: eight rows that one ldmatrix reads lie in different banks.
template <uint32_t ROW_BYTES> __device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c)
{
    if constexpr (ROW_BYTES >= 128)
        return r * ROW_BYTES + ((c ^ (r & 7)) * 16);
    else
        return r * ROW_BYTES + ((c ^ (r >> 1 & 3)) * 16);
}

template <uint32_t D, uint32_t NT, bool FP8>
__global__ void __launch_bounds__(kStreamThreads, StreamShape<D, NT, FP8>::kBlocks) attn_stream_kernel(AttnParams p)
{
    using Shape = StreamShape<D, NT, FP8>;
    constexpr uint32_t ROWS = Shape::kRows, ROW_BYTES = Shape::kRowBytes;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const s_q = smem + Shape::kUnion;
    float2* const s_ml = reinterpret_cast<float2*>(s_q + Shape::kQ); // [warps][rows]
    float* const s_q_scale = reinterpret_cast<float*>(s_ml + kStreamWarps * ROWS); // e4m3: what a row was divided by
    chain_begin();

    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const BlockRange range = find_range<kStreamThreads>(p, reinterpret_cast<uint64_t*>(smem), blockIdx.x);
    uint64_t left = range.end - range.begin;
    AttnPlace at = range.place;
    uint8_t* const ring = smem + warp * kStreamStages * Shape::kStage;
    const uint32_t ring_u32 = tc::smem_u32(ring);
    if (tid == 0)
        note_split(p, range);

    Segment seg;
    while (this_segment<true>(p, at, left, &seg)) {
        const SeqRows& rows = seg.rows;
        const SeqPages& pages = seg.pages;
        const uint32_t count = seg.count, tile0 = seg.tile0, row0 = seg.row0, nrows = seg.nrows;

        // query rows; a row past the last one is zeros
        __syncthreads();
        for (uint32_t i = tid; i < ROWS * D / 8; i += kStreamThreads) {
            const uint32_t r = i / (D / 8), c = i % (D / 8);
            uint4 w = make_uint4(0, 0, 0, 0);
            if (r < nrows) {
                const uint32_t token = p.tiling.group.div(row0 + r), h = at.head * p.tiling.group.d + row0 + r - token * p.tiling.group.d;
                w = *reinterpret_cast<const uint4*>(p.q + (rows.row0 + token) * p.q_token + h * p.q_head + c * 16);
            }
            if constexpr (FP8) { // to f16, the row's largest element brought to 2^13 or just above; an infinity or NaN stays one
                static_assert(ROWS * D / 8 % 32 == 0, "whole warps");
                uint32_t a[4] = { w.x, w.y, w.z, w.w }, most = 0; // of the magnitudes, which are in the order of their bits
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    most = max(most, max(a[j] & 0x7fffu, a[j] >> 16 & 0x7fffu));
#pragma unroll
                for (uint32_t o = 1; o < D / 8; o <<= 1)
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                const int power = most >= 0x7f80u ? 0 : max(-126, min(126, 127 + 13 - static_cast<int>(most >> 7)));
                const float up = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    a[j] = pack_f16x2(bf16_bits_to_f32(a[j] & 0xffffu) * up, bf16_bits_to_f32(a[j] >> 16) * up);
                w = make_uint4(a[0], a[1], a[2], a[3]);
                if (c == 0)
                    s_q_scale[r] = __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
            }
            *reinterpret_cast<uint4*>(s_q + swizzled<D * 2>(r, c)) = w;
        }
        __syncthreads();

        // keys that any row sees: others are not fetched, and whatever they hold does not count
        uint32_t seen_lo, seen_hi, unused;
        visible_keys(p.tiling, rows.fresh, pages.length, p.tiling.group.div(row0), &seen_lo, &unused);
        visible_keys(p.tiling, rows.fresh, pages.length, p.tiling.group.div(row0 + nrows - 1), &unused, &seen_hi);
        seen_hi = min(seen_hi, pages.room);
        // keys that the rows of this lane's columns see
        uint32_t lo[NT][2], hi[NT][2];
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                const uint32_t r = n * 8 + (lane & 3) * 2 + j;
                lo[n][j] = hi[n][j] = 0;
                if (r < nrows) {
                    visible_keys(p.tiling, rows.fresh, pages.length, p.tiling.group.div(row0 + r), &lo[n][j], &hi[n][j]);
                    hi[n][j] = min(hi[n][j], pages.room);
                }
            }

        float q_scale[NT][2];
        if constexpr (FP8)
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
                    q_scale[n][j] = s_q_scale[n * 8 + (lane & 3) * 2 + j];

        // B fragments of the queries: for 8-bit keys the four consecutive elements that a lane converts from one word
        uint32_t qf[NT == 1 ? D / 16 : 1][2];
        const auto q_frag = [&](uint32_t n, uint32_t ks, uint32_t* b) {
            const uint32_t r = n * 8 + lane / 4, c = lane & 3;
            if constexpr (FP8) {
                const uint2 w = *reinterpret_cast<const uint2*>(s_q + swizzled<D * 2>(r, ks * 2 + c / 2) + (c & 1) * 8);
                b[0] = w.x;
                b[1] = w.y;
            } else {
                b[0] = *reinterpret_cast<const uint32_t*>(s_q + swizzled<D * 2>(r, ks * 2) + c * 4);
                b[1] = *reinterpret_cast<const uint32_t*>(s_q + swizzled<D * 2>(r, ks * 2 + 1) + c * 4);
            }
        };
        if constexpr (NT == 1)
#pragma unroll
            for (uint32_t ks = 0; ks < D / 16; ++ks)
                q_frag(0, ks, qf[ks]);

        float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (uint32_t i = 0; i < D / 16; ++i)
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    o[i][n][j] = 0.0f;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
            m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

        const uint8_t* const k_head = p.view.k.data + at.head * p.view.k.head_stride;
        const uint8_t* const v_head = p.view.v.data + at.head * p.view.v.head_stride;
        const auto issue = [&](uint32_t i) {
            if (i < count) {
                const uint32_t base = ring_u32 + (i % kStreamStages) * Shape::kStage;
                const uint32_t key = (tile0 + i) * kStreamKeys + warp * kWarpKeys + (lane & 15);
                uint32_t slot = 0;
                int32_t page = -1;
                if (key >= seen_lo && key < seen_hi)
                    page = page_of(p.view, pages, key, &slot);
                const uint32_t k_row = row_units(p.view.k, page, slot), v_row = row_units(p.view.v, page, slot);
                constexpr uint32_t UNITS = ROW_BYTES / 16, STEP = 32 / UNITS == 0 ? 1 : 32 / UNITS; // rows per instruction
                const uint32_t r_lane = lane / UNITS, c = lane % UNITS;
                static_assert(UNITS <= 32, "a row is at most 512 bytes");
#pragma unroll
                for (uint32_t r0 = 0; r0 < kWarpKeys; r0 += STEP) {
                    const uint32_t r = r0 + r_lane;
                    const uint32_t k = __shfl_sync(0xffffffffu, k_row, r & 15), v = __shfl_sync(0xffffffffu, v_row, r & 15);
                    const uint32_t dst = base + swizzled<ROW_BYTES>(r, c);
                    cp_async16(dst, k_head + row_bytes(p.view.k, k) + c * 16, k != kNoRow);
                    cp_async16(dst + Shape::kHalf, v_head + row_bytes(p.view.v, v) + c * 16, v != kNoRow);
                }
                if constexpr (FP8) {
                    const PagedPool& pool = lane < 16 ? p.view.k : p.view.v;
                    const int64_t pg0 = page < 0 ? 0 : page;
                    cp_async4z(base + 2 * Shape::kHalf + lane * 4,
                               pool.scale + pg0 * pool.scale_page_stride + at.head * pool.scale_head_stride
                                   + slot * pool.scale_slot_stride,
                               page >= 0);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (uint32_t i = 0; i < kStreamStages - 1; ++i)
            issue(i);

        for (uint32_t i = 0; i < count; ++i) {
            issue(i + kStreamStages - 1);
            cp_async_wait_group<kStreamStages - 1>();
            __syncwarp();
            const uint32_t stage = ring_u32 + (i % kStreamStages) * Shape::kStage;
            const uint32_t key0 = (tile0 + i) * kStreamKeys + warp * kWarpKeys;

            // S^T: two chains of products per column tile
            float s[NT][2][4];
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    s[n][j / 4][j & 3] = 0.0f;
            if constexpr (!FP8) {
#pragma unroll
                for (uint32_t ks = 0; ks < D / 16; ++ks) {
                    uint32_t a[4];
                    ldmatrix4(a, stage + swizzled<ROW_BYTES>(lane & 15, ks * 2 + lane / 16));
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n) {
                        uint32_t b[2];
                        if constexpr (NT == 1)
                            b[0] = qf[ks][0], b[1] = qf[ks][1];
                        else
                            q_frag(n, ks, b);
                        mma16816<FP8>(s[n][ks & 1], a, b[0], b[1]);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t kb = 0; kb < D / 32; ++kb) {
                    uint32_t w[4];
                    ldmatrix4(w, stage + swizzled<ROW_BYTES>(lane & 15, kb * 2 + lane / 16));
#pragma unroll
                    for (uint32_t u = 0; u < 2; ++u) {
                        const uint32_t ks = kb * 2 + u;
                        const uint32_t a[4] = { e4m3x2_to_f16x2(w[2 * u]), e4m3x2_to_f16x2(w[2 * u + 1]),
                                                e4m3x2_to_f16x2(w[2 * u] >> 16), e4m3x2_to_f16x2(w[2 * u + 1] >> 16) };
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) {
                            uint32_t b[2];
                            if constexpr (NT == 1)
                                b[0] = qf[ks][0], b[1] = qf[ks][1];
                            else
                                q_frag(n, ks, b);
                            mma16816<FP8>(s[n][u], a, b[0], b[1]);
                        }
                    }
                }
            }
            // factor on the scores, what is added to them, and the factor on the weights in the row's sum, of a lane's two keys
            float ks0 = p.scale_log2, ks1 = p.scale_log2, lv0 = 0.0f, lv1 = 0.0f, unit0 = 1.0f, unit1 = 1.0f;
            if constexpr (FP8) {
                const float* sc = reinterpret_cast<const float*>(ring + (i % kStreamStages) * Shape::kStage + 2 * Shape::kHalf);
                ks0 *= sc[lane / 4];
                ks1 *= sc[lane / 4 + 8];
                const float v0 = sc[16 + lane / 4], v1 = sc[16 + lane / 4 + 8];
                lv0 = __log2f(v0 < 1.0e-30f ? 1.0e-30f : v0); // (a NaN stays one)
                lv1 = __log2f(v1 < 1.0e-30f ? 1.0e-30f : v1);
                unit0 = kSumFactor<FP8> / (v0 < 1.0e-30f ? 1.0e-30f : v0);
                unit1 = kSumFactor<FP8> / (v1 < 1.0e-30f ? 1.0e-30f : v1);
            }

            // P^T, a lane's keys lane / 4 and lane / 4 + 8 and rows 2 (lane % 4) and the next
            uint32_t pf[NT][2];
            const uint32_t ka = key0 + lane / 4, kb = ka + 8;
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                float v[4] = { s[n][0][0] + s[n][1][0], s[n][0][1] + s[n][1][1], s[n][0][2] + s[n][1][2], s[n][0][3] + s[n][1][3] };
                if constexpr (FP8) {
                    v[0] = fmaf(v[0] * q_scale[n][0], ks0, lv0);
                    v[1] = fmaf(v[1] * q_scale[n][1], ks0, lv0);
                    v[2] = fmaf(v[2] * q_scale[n][0], ks1, lv1);
                    v[3] = fmaf(v[3] * q_scale[n][1], ks1, lv1);
                } else {
                    v[0] *= ks0, v[1] *= ks0, v[2] *= ks1, v[3] *= ks1;
                }
                float w[4];
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    v[j] = ka >= lo[n][j] && ka < hi[n][j] ? v[j] : -INFINITY;
                    v[j + 2] = kb >= lo[n][j] && kb < hi[n][j] ? v[j + 2] : -INFINITY;
                    float top = fmaxf(v[j], v[j + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = fmaxf(top, m[n][j]);
                    const float base = top == -INFINITY ? 0.0f : top; // nothing seen yet: exp2(-inf - 0) = 0
                    const float keep = exp2_fast(m[n][j] - base);
                    m[n][j] = top;
                    w[j] = exp2_fast(v[j] - (base - kTop<FP8>));
                    w[j + 2] = exp2_fast(v[j + 2] - (base - kTop<FP8>));
                    l[n][j] = FP8 ? fmaf(w[j], unit0, fmaf(w[j + 2], unit1, l[n][j] * keep)) : l[n][j] * keep + (w[j] + w[j + 2]);
                    if (__any_sync(0xffffffffu, keep != 1.0f)) {
#pragma unroll
                        for (uint32_t d = 0; d < D / 16; ++d) {
                            o[d][n][j] *= keep;
                            o[d][n][j + 2] *= keep;
                        }
                    }
                }
                pf[n][0] = transpose8(FP8 ? pack_f16x2(w[0], w[1]) : tc::pack_bf16x2(w[0], w[1]));
                pf[n][1] = transpose8(FP8 ? pack_f16x2(w[2], w[3]) : tc::pack_bf16x2(w[2], w[3]));
            }

            // O^T += V^T P^T
            const uint32_t v_base = stage + Shape::kHalf;
            if constexpr (!FP8) {
#pragma unroll
                for (uint32_t d = 0; d < D / 16; ++d) {
                    uint32_t a[4];
                    ldmatrix4_trans(a, v_base + swizzled<ROW_BYTES>((lane & 7) + lane / 16 * 8, d * 2 + (lane >> 3 & 1)));
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n)
                        mma16816<FP8>(o[d][n], a, pf[n][0], pf[n][1]);
                }
            } else {
#pragma unroll
                for (uint32_t db = 0; db < D / 32; ++db) {
                    uint32_t w[4]; // keys 0-7 and 8-15 of 16 elements, then of the next 16
                    ldmatrix4_trans(w, v_base + swizzled<ROW_BYTES>(lane & 15, db * 2 + lane / 16));
#pragma unroll
                    for (uint32_t u = 0; u < 2; ++u) {
                        // a word holds elements 2r, 2r + 1 of two keys: rows r and r + 8 of the product
                        const uint32_t first = __byte_perm(w[2 * u], 0, 0x3120), second = __byte_perm(w[2 * u + 1], 0, 0x3120);
                        const uint32_t a[4] = { e4m3x2_to_f16x2(first), e4m3x2_to_f16x2(first >> 16), e4m3x2_to_f16x2(second),
                                                e4m3x2_to_f16x2(second >> 16) };
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n)
                            mma16816<FP8>(o[db * 2 + u][n], a, pf[n][0], pf[n][1]);
                    }
                }
            }
            __syncwarp(); // the stage is free again
        }
        cp_async_wait_group<0>();

        // join the four warps: sums of the lanes' keys, then one scale for all
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1)
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
                if (lane < 4)
                    s_ml[warp * ROWS + n * 8 + lane * 2 + j] = make_float2(m[n][j], l[n][j]);
            }
        __syncthreads(); // every warp is through with its ring
        float* const sums = reinterpret_cast<float*>(smem); // [warps][rows][D]
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                const uint32_t r = n * 8 + (lane & 3) * 2 + j;
                float top = -INFINITY;
#pragma unroll
                for (uint32_t w = 0; w < kStreamWarps; ++w)
                    top = fmaxf(top, s_ml[w * ROWS + r].x);
                const float factor = exp2_fast(m[n][j] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
                for (uint32_t d = 0; d < D / 16; ++d) {
                    const uint32_t e0 = FP8 ? d * 16 + lane / 4 * 2 : d * 16 + lane / 4, e1 = FP8 ? e0 + 1 : e0 + 8;
                    sums[(warp * ROWS + r) * D + e0] = o[d][n][j] * factor;
                    sums[(warp * ROWS + r) * D + e1] = o[d][n][j + 2] * factor;
                }
            }
        __syncthreads();
        constexpr float kUnits = kSumUnit<FP8> - kTop<FP8>; // from a row's maximum to the unit of its sums
        const bool whole = seg.whole;
        const uint32_t slot = blockIdx.x * 2 + (seg.starts ? 1 : 0);
        for (uint32_t i = tid; i < nrows * (D / 4); i += kStreamThreads) {
            const uint32_t r = i / (D / 4), e = i % (D / 4) * 4;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kStreamWarps; ++w)
                top = fmaxf(top, s_ml[w * ROWS + r].x);
            const float base = top == -INFINITY ? 0.0f : top;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t w = 0; w < kStreamWarps; ++w) {
                const float2 ml = s_ml[w * ROWS + r];
                sum += ml.y * exp2_fast(ml.x - base);
                const float4 x = *reinterpret_cast<const float4*>(sums + (w * ROWS + r) * D + e);
                acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
            }
            if (whole) {
                const uint32_t token = p.tiling.group.div(row0 + r), h = at.head * p.tiling.group.d + row0 + r - token * p.tiling.group.d;
                const bool scored = top != -INFINITY;
                const float inv = scored ? kSumFactor<FP8> / sum : without_scores(p, rows.fresh, pages, row0 + r);
                const uint2 w = make_uint2(tc::pack_bf16x2(acc.x * inv, acc.y * inv), tc::pack_bf16x2(acc.z * inv, acc.w * inv));
                *reinterpret_cast<uint2*>(p.out + (rows.row0 + token) * p.out_token + h * p.out_head + e * 2) = w;
                if (e == 0 && p.lse != nullptr)
                    p.lse[(rows.row0 + token) * p.lse_token + h * p.lse_head]
                        = scored ? (top + kUnits + log2f(sum)) * 0.693147180559945f : inv == 0.0f ? -INFINITY : inv;
            } else {
                constexpr float f = kSumFactor<FP8>;
                *reinterpret_cast<float4*>(p.part_o + (static_cast<size_t>(slot) * ROWS + r) * D + e)
                    = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
                if (e == 0)
                    p.part_ml[static_cast<size_t>(slot) * ROWS + r] = make_float2(top + kUnits, sum);
            }
        }
        next_segment(p, seg, &at, &left);
    }
}

// Joins the parts of items that were split: slot 1 of block c - 1, slots 0 of c and the blocks after it. SHARED: a block per
// row, its warps with a part each in turn (few rows, a long context over many blocks); else a warp per row.
constexpr uint32_t kJoinWarps = 8;

// (Launch bounds: with a few registers more than 32 three quarters as many rows are under way at a time, mixed batch 129.2 us and 127.1.)
template <uint32_t D, bool SHARED>
__global__ void __launch_bounds__(kJoinWarps * 32, D == 256 ? 5 : 8) attn_join_kernel(AttnParams p)
{
    constexpr uint32_t E = D / 32; // elements of a lane
    __shared__ float s_acc[SHARED ? kJoinWarps * D : 1];
    chain_begin();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t r = SHARED ? blockIdx.y : blockIdx.y * kJoinWarps + warp, rows_of_item = 1u << p.tiling.row_shift;
    for (uint32_t c = blockIdx.x + 1; c < p.blocks; c += gridDim.x) {
        const SplitNote n = p.notes[c];
        if (n.parts == 0)
            continue;
        const SeqRows rows = seq_rows(p, n.seq);
        const uint32_t row0 = n.tile << p.tiling.row_shift;
        if (row0 + r >= rows.fresh * p.tiling.group.d)
            continue;
        const auto slot_of = [&](uint32_t i) {
            return static_cast<size_t>(i == 0 ? 2 * c - 1 : 2 * (c + i - 1)) * rows_of_item + r;
        };
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t i = lane; i <= n.parts; i += 32)
            top = fmaxf(top, p.part_ml[slot_of(i)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float base = top == -INFINITY ? 0.0f : top;
        for (uint32_t i = lane; i <= n.parts; i += 32) {
            const float2 ml = p.part_ml[slot_of(i)];
            sum += ml.y * exp2_fast(ml.x - base);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        float acc[E];
#pragma unroll
        for (uint32_t j = 0; j < E; ++j)
            acc[j] = 0.0f;
        constexpr uint32_t STEP = SHARED ? kJoinWarps : 1;
#pragma unroll 4
        for (uint32_t i = SHARED ? warp : 0; i <= n.parts; i += STEP) {
            const size_t s = slot_of(i);
            const float w = exp2_fast(p.part_ml[s].x - base);
            const float* x = p.part_o + s * D + lane * E;
            float v[E];
            if constexpr (E == 2) {
                *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(x);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < E; j += 4)
                    *reinterpret_cast<float4*>(v + j) = *reinterpret_cast<const float4*>(x + j);
            }
#pragma unroll
            for (uint32_t j = 0; j < E; ++j)
                acc[j] += v[j] * w;
        }
        if constexpr (SHARED) {
            __syncthreads(); // (the row before)
#pragma unroll
            for (uint32_t j = 0; j < E; ++j)
                s_acc[warp * D + lane * E + j] = acc[j];
            __syncthreads();
            if (warp != 0)
                continue;
#pragma unroll
            for (uint32_t j = 0; j < E; ++j)
#pragma unroll
                for (uint32_t w = 1; w < kJoinWarps; ++w)
                    acc[j] += s_acc[w * D + lane * E + j];
        }
        const bool scored = top != -INFINITY;
        const float inv = scored ? 1.0f / sum : without_scores(p, rows.fresh, seq_pages(p.view, n.seq), row0 + r);
        const uint32_t token = p.tiling.group.div(row0 + r), h = n.head * p.tiling.group.d + row0 + r - token * p.tiling.group.d;
        uint8_t* out = p.out + (rows.row0 + token) * p.out_token + h * p.out_head + lane * E * 2;
        uint32_t w[E / 2];
#pragma unroll
        for (uint32_t j = 0; j < E / 2; ++j)
            w[j] = tc::pack_bf16x2(acc[2 * j] * inv, acc[2 * j + 1] * inv);
        if constexpr (E == 2)
            *reinterpret_cast<uint32_t*>(out) = w[0];
        else if constexpr (E == 4)
            *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
        if (lane == 0 && p.lse != nullptr)
            p.lse[(rows.row0 + token) * p.lse_token + h * p.lse_head]
                = scored ? (top + log2f(sum)) * 0.693147180559945f : inv == 0.0f ? -INFINITY : inv;
    }
}

template <uint32_t D, uint32_t NT, bool FP8> cudaError_t launch_stream_as(const AttnParams& p, cudaStream_t stream)
{
    using Shape = StreamShape<D, NT, FP8>;
    const auto kernel = attn_stream_kernel<D, NT, FP8>;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (err != cudaSuccess)
        return err;
    return launch_chained(kernel, dim3(p.blocks), kStreamThreads, Shape::kSmem, stream, p);
}

template <uint32_t D> uint32_t stream_blocks_as(uint32_t rows, bool fp8)
{
    return rows == 8 ? (fp8 ? StreamShape<D, 1, true>::kBlocks : StreamShape<D, 1, false>::kBlocks)
                     : (fp8 ? StreamShape<D, 2, true>::kBlocks : StreamShape<D, 2, false>::kBlocks);
}

} // namespace

uint32_t attn_stream_rows(uint32_t rows_per_seq) { return rows_per_seq <= 8 ? 8 : 16; }

uint32_t attn_stream_blocks(uint32_t tile_rows, uint32_t head_dim, bool fp8)
{
    const uint32_t per_sm = head_dim == 64 ? stream_blocks_as<64>(tile_rows, fp8)
        : head_dim == 128                  ? stream_blocks_as<128>(tile_rows, fp8)
                                           : stream_blocks_as<256>(tile_rows, fp8);
    return per_sm * kSmCount;
}

cudaError_t launch_attn_stream(const AttnParams& p, bool fp8, cudaStream_t stream)
{
    const uint32_t d = p.view.head_dim;
    const bool two = p.tiling.row_shift == 4;
#define QS3_STREAM(DIM)                                                                                                      \
    if (d == DIM)                                                                                                            \
        return two ? (fp8 ? launch_stream_as<DIM, 2, true>(p, stream) : launch_stream_as<DIM, 2, false>(p, stream))          \
                   : (fp8 ? launch_stream_as<DIM, 1, true>(p, stream) : launch_stream_as<DIM, 1, false>(p, stream));
    QS3_STREAM(64)
    QS3_STREAM(128)
    QS3_STREAM(256)
#undef QS3_STREAM
    return cudaErrorInvalidValue;
}

cudaError_t launch_attn_join(const AttnParams& p, cudaStream_t stream)
{
    const uint32_t d = p.view.head_dim;
    const uint32_t wide = p.blocks - 1 < kSmCount ? p.blocks - 1 : kSmCount;
    const uint32_t rows = 1u << p.tiling.row_shift;
    if (rows <= 16)
        return launch_chained(d == 64 ? attn_join_kernel<64, true> : d == 128 ? attn_join_kernel<128, true> : attn_join_kernel<256, true>,
                              dim3(wide, rows), kJoinWarps * 32, 0, stream, p);
    return launch_chained(d == 64 ? attn_join_kernel<64, false> : d == 128 ? attn_join_kernel<128, false> : attn_join_kernel<256, false>,
                          dim3(wide, rows / kJoinWarps), kJoinWarps * 32, 0, stream, p);
}

} // namespace qs3

using namespace qs3;

namespace {

struct AttnSizes {
    size_t notes, ml, o; // offsets
    size_t bytes;
};

AttnSizes attn_sizes(uint32_t blocks, uint32_t tile_rows, uint32_t head_dim)
{
    AttnSizes s;
    s.notes = 0;
    s.ml = align_up(blocks * sizeof(SplitNote), kWorkspaceAlign);
    s.o = s.ml + align_up(static_cast<size_t>(blocks) * 2 * tile_rows * sizeof(float2), kWorkspaceAlign);
    s.bytes = s.o + static_cast<size_t>(blocks) * 2 * tile_rows * head_dim * sizeof(float);
    return s;
}

bool head_dim_ok(uint32_t d) { return d == 64 || d == 128 || d == 256; }

// Blocks and bytes of the streaming kernel at most, over both cache types.
size_t stream_bytes(uint32_t tile_rows, uint32_t d)
{
    size_t most = 0;
    for (const bool fp8 : { false, true }) {
        const size_t n = attn_sizes(attn_stream_blocks(tile_rows, d, fp8), tile_rows, d).bytes;
        most = n > most ? n : most;
    }
    return most;
}

} // namespace

extern "C" {

qsfi_status qs3_paged_attention_workspace_size(qsfi_context* ctx, uint32_t rows, uint32_t batch, uint32_t heads,
                                               uint32_t kv_heads, uint32_t head_dim, size_t* bytes)
{
    if (ctx == nullptr)
        return QSFI_STATUS_INVALID_ARGUMENT;
    clear_error(&ctx->last_error);
    if (bytes == nullptr)
        return set_invalid_arg(ctx, "paged_attention bytes must not be null");
    if (rows == 0 || batch == 0 || heads == 0 || kv_heads == 0 || heads % kv_heads != 0)
        return set_invalid_arg(ctx, "paged_attention sizes must be positive and heads a multiple of kv_heads");
    if (!head_dim_ok(head_dim))
        return set_unsupported(ctx, "paged_attention head_dim must be 64, 128 or 256");
    const size_t a = stream_bytes(8, head_dim), b = stream_bytes(16, head_dim);
    const size_t c = attn_sizes(kSmCount, attn_prefill_rows(head_dim), head_dim).bytes;
    *bytes = a > b ? (a > c ? a : c) : b > c ? b : c;
    return QSFI_STATUS_OK;
}

qsfi_status qs3_paged_attention(qsfi_context* ctx, const qs3_paged_attention_desc* d)
{
    if (ctx == nullptr)
        return QSFI_STATUS_INVALID_ARGUMENT;
    clear_error(&ctx->last_error);
    if (d == nullptr)
        return set_invalid_arg(ctx, "paged_attention desc must not be null");
    qsfi_status s = activate_context(ctx);
    if (s != QSFI_STATUS_OK)
        return s;
    AttnParams p {};
    bool fp8 = false;
    s = paged_view(ctx, d->cache, d->table, "paged_attention", &p.view, &fp8);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->q, "paged_attention", "q", QSFI_DTYPE_BF16);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->out, "paged_attention", "out", QSFI_DTYPE_BF16);
    if (s != QSFI_STATUS_OK)
        return s;
    const uint32_t dim = p.view.head_dim;
    if (!head_dim_ok(dim))
        return set_unsupported(ctx, "paged_attention head_dim must be 64, 128 or 256");
    if (d->q.shape[2] != dim)
        return set_invalid_arg(ctx, "paged_attention q must have the cache's head_dim");
    qsfi_tensor3 dst;
    int in_place = 0; // (every item reads its rows before it writes them)
    s = check_out(ctx, d->q, d->out, "paged_attention", "out", &dst, &in_place);
    if (s != QSFI_STATUS_OK)
        return s;
    const int64_t rows = d->q.shape[0], heads = d->q.shape[1];
    if (heads % p.view.kv_heads != 0)
        return set_invalid_arg(ctx, "paged_attention heads must be a multiple of kv_heads");
    const int64_t group = heads / p.view.kv_heads;
    if (rows * heads > (int64_t { 1 } << 30) || rows > (1 << 24) || heads > 4096)
        return set_unsupported(ctx, "paged_attention takes at most 2^24 rows, 4096 heads and 2^30 rows times heads");
    if (d->q_indptr.data != nullptr) {
        s = check_index(ctx, d->q_indptr, "paged_attention", "q_indptr", p.view.batch + 1);
        if (s != QSFI_STATUS_OK)
            return s;
        p.q_indptr = static_cast<const int32_t*>(d->q_indptr.data);
    } else if (rows < static_cast<int64_t>(p.view.batch)) {
        return set_invalid_arg(ctx, "paged_attention without q_indptr needs a row per sequence");
    }
    if (d->lse.data != nullptr) {
        if (d->lse.dtype != QSFI_DTYPE_F32 || d->lse.shape[0] != rows || d->lse.shape[1] != heads || d->lse.stride[0] < 0
            || d->lse.stride[1] < 0 || (reinterpret_cast<uintptr_t>(d->lse.data) & 3u) != 0)
            return set_invalid_arg(ctx, "paged_attention lse must be f32 [rows, heads]");
        p.lse = static_cast<float*>(d->lse.data);
        p.lse_token = d->lse.stride[0];
        p.lse_head = d->lse.stride[1];
    }
    if (!rows_fit(p.view))
        return set_unsupported(ctx, "paged_attention cache has more than 2^32 rows' worth of memory between its first and last, "
                                    "or scales 2^30 apart");
    if (d->window != 0 && d->causal == 0)
        return set_unsupported(ctx, "paged_attention window needs causal");
    if (!std::isfinite(d->sm_scale) || d->sm_scale < 0.0f)
        return set_invalid_arg(ctx, "paged_attention sm_scale must be finite and not negative");
    if (d->workspace.data == nullptr || (d->workspace.dtype != QSFI_DTYPE_U8 && d->workspace.dtype != QSFI_DTYPE_I8)
        || d->workspace.stride[0] != 1 || (reinterpret_cast<uintptr_t>(d->workspace.data) & 255u) != 0)
        return set_invalid_arg(ctx, "paged_attention workspace must be a contiguous, 256-byte aligned u8 tensor");
    size_t need = 0;
    s = qs3_paged_attention_workspace_size(ctx, static_cast<uint32_t>(rows), p.view.batch, static_cast<uint32_t>(heads),
                                           p.view.kv_heads, dim, &need);
    if (s != QSFI_STATUS_OK)
        return s;
    if (static_cast<uint64_t>(d->workspace.shape[0]) < need)
        return set_invalid_arg(ctx, "paged_attention workspace has %lld bytes, needs %llu",
                               static_cast<long long>(d->workspace.shape[0]), static_cast<unsigned long long>(need));
    const RowSet read = row_set(d->q), written = row_set(dst), scratch { d->workspace.data, 1, 1, 0, 0, static_cast<int64_t>(need) };
    const RowSet lse { d->lse.data, rows, heads, p.lse_token * 4, p.lse_head * 4, 4 };
    if (p.lse != nullptr && !rows_apart(lse))
        return set_invalid_arg(ctx, "paged_attention lse rows must not overlap");
    s = check_apart(ctx, "paged_attention", "workspace", scratch, "out", written);
    if (s == QSFI_STATUS_OK)
        s = check_apart(ctx, "paged_attention", "workspace", scratch, "q", read);
    if (s == QSFI_STATUS_OK)
        s = check_apart(ctx, "paged_attention", "workspace", scratch, "lse", lse);
    if (s == QSFI_STATUS_OK)
        s = check_apart(ctx, "paged_attention", "lse", lse, "q", read);
    if (s == QSFI_STATUS_OK)
        s = check_apart(ctx, "paged_attention", "lse", lse, "out", written);
    if (s != QSFI_STATUS_OK)
        return s;

    p.q = static_cast<const uint8_t*>(d->q.data);
    p.q_token = d->q.stride[0] * 2;
    p.q_head = d->q.stride[1] * 2;
    p.out = static_cast<uint8_t*>(d->out.data);
    p.out_token = d->out.stride[0] * 2;
    p.out_head = d->out.stride[1] * 2;
    p.rows = static_cast<uint32_t>(rows);
    p.heads = static_cast<uint32_t>(heads);
    p.scale_log2 = (d->sm_scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(dim)) : d->sm_scale) * 1.4426950408889634f;
    p.err = p.view.err = device_error_word();
    if (p.err == nullptr)
        return set_cuda_error(ctx, cudaErrorUnknown, "device error word");

    // most rows of a sequence, as far as the caller says
    const uint64_t fresh = d->q_indptr.data == nullptr ? 1
        : d->max_q_len != 0                            ? (d->max_q_len < rows ? d->max_q_len : static_cast<uint64_t>(rows))
                                                       : static_cast<uint64_t>(rows);
    const uint64_t room = static_cast<uint64_t>(p.view.num_indices) * p.view.page_size;
    const uint64_t longest = d->max_kv_len != 0 && d->max_kv_len < room ? d->max_kv_len : room;
    p.tiling.group = FastDiv(static_cast<uint32_t>(group));
    p.tiling.kv_heads = p.view.kv_heads;
    p.tiling.window = d->window;
    p.tiling.causal = d->causal;
    // A tile of the streaming kernel has 16 rows. Up to there it is the faster one, or not far behind where the cache's stream
    // bounds both: 8 sequences of 700 tokens 21.5 us (chunk kernel 31.7), 64 of 4096 tokens with 4 new ones, 32 heads over 8,
    // 212 (236), over an e4m3 cache 191 (472), 128 of 4096 with 16 heads over 2 of 256 208 (200), L2 flushed before each call.
    // The border is a bf16 cache's: just beyond it, with 5 new tokens, the 64 sequences take 246 us, and over an e4m3 cache, where
    // the chunk kernel converts V anew for every row tile, 465 (with 4: 202 and 224, calls one after another). There it lies too low.
    const bool chunks = fresh * group > 16;
    uint32_t item_rows;
    if (chunks) {
        item_rows = attn_prefill_rows(dim);
        p.tiling.key_shift = 7;
        p.tiling.item_cost = 4;
        p.blocks = kSmCount;
    } else {
        item_rows = attn_stream_rows(static_cast<uint32_t>(fresh * group));
        p.tiling.key_shift = 6;
        p.tiling.item_cost = 1;
        p.blocks = attn_stream_blocks(item_rows, dim, fp8);
    }
    while ((1u << p.tiling.row_shift) < item_rows)
        ++p.tiling.row_shift;
    p.least = p.tiling.item_cost + 1;
    // no more blocks than there can be work for: those without any would only start and end
    const uint64_t tiles = (longest + (1u << p.tiling.key_shift) - 1) >> p.tiling.key_shift;
    const uint64_t items = (rows * group / item_rows + p.view.batch) * p.view.kv_heads; // ends of sequences begin items of their own
    // Contexts too short to be worth cutting, and the launch that joins them. A call in a graph of them, cut or not: 8 sequences of
    // one new token, 32 heads over 8 of 128, 128 cached ones 11.0 us, 7.6; 384 12.7, 10.6; 700 15.9, 14.5; 16 heads over 2 of 256,
    // 128 12.6, 9.1; 384 13.3, 13.3; 700 13.8, 18.8. Chunks: 4 of 128 new tokens in 128 20.1, 16.5, of 512 in 512 48.1, 40.5.
    if (longest <= (chunks ? 512 : 384)) {
        p.tiling.even = 1;
        p.least = 1;
    }
    const uint64_t most = (items * cost_of(p.tiling, static_cast<uint32_t>(tiles > 0 ? tiles : 1)) + p.least - 1) / p.least;
    p.blocks = most < p.blocks ? static_cast<uint32_t>(most) : p.blocks;
    const AttnSizes at = attn_sizes(p.blocks, item_rows, dim);
    char* ws = static_cast<char*>(d->workspace.data);
    p.notes = reinterpret_cast<SplitNote*>(ws + at.notes);
    p.part_ml = reinterpret_cast<float2*>(ws + at.ml);
    p.part_o = reinterpret_cast<float*>(ws + at.o);
    cudaError_t err = chunks ? launch_attn_prefill(p, fp8, ctx->stream) : launch_attn_stream(p, fp8, ctx->stream);
    if (err == cudaSuccess && p.blocks > 1 && !p.tiling.even) // (otherwise there is nothing to join)
        err = launch_attn_join(p, ctx->stream);
    return set_cuda_error(ctx, err, "paged_attention");
}

} // extern "C"
