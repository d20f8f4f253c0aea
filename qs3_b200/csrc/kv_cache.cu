// Rotary positions, and a paged KV cache as it is written and read back: the passes around attention over that cache
// (paged_attention.cu). All three move rows of one head, at most 256 elements, and are bound by HBM at prefill sizes and by
// their one launch at decode sizes.
//
// A row is held by the lanes of a part of a warp, eight or sixteen elements each: the partner of an element in the half layout is
// then in the lane or one shuffle away, and the row's maximum a few, so that a row is read once and written once, turned and
// quantised in between.
// A block takes all rows of a token or of a few; their sines and cosines are computed once per block, behind the first loads.
#include "fp8.cuh"
#include "paged.cuh"

#include <algorithm>
#include <cmath>
#include <limits>

namespace qs3 {

namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxTokens = 8; // of a block

enum Layout { LAYOUT_NONE = 0, LAYOUT_HALF = 1, LAYOUT_HALF_ODD = 2, LAYOUT_PAIRS = 3 };
enum Target { TARGET_ROWS = 0, TARGET_BF16 = 1, TARGET_FP8 = 2 };

struct Rows { // [tokens, heads, dim], strides in bytes
    const uint8_t* src;
    uint8_t* dst;
    int64_t src_token, src_head, dst_token, dst_head;
    uint32_t heads;
};

struct TurnParams {
    Rows q, k, v;      // v and the dst of k: cache targets only
    uint32_t tokens, dim, half, group_log; // lanes per row = 1 << group_log
    uint32_t rows_per_token, block_tokens;
    FastDiv row_div;   // by rows_per_token
    const void* positions;
    int positions64;
    const double* inv_freq;
    float scale;
    int in_place_q, in_place_k; // the part that is passed through stays where it is
    const int32_t* q_indptr;
    PagedView view;
};

template <typename T> struct Eight; // eight consecutive elements of a lane
template <> struct Eight<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void unpack(float* f) const
    {
        const uint32_t a[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = bf16_bits_to_f32(a[j] & 0xffffu);
            f[2 * j + 1] = bf16_bits_to_f32(a[j] >> 16);
        }
    }
    __device__ __forceinline__ Eight from(int lane) const
    {
        Eight e;
        e.w.x = __shfl_sync(0xffffffffu, w.x, lane);
        e.w.y = __shfl_sync(0xffffffffu, w.y, lane);
        e.w.z = __shfl_sync(0xffffffffu, w.z, lane);
        e.w.w = __shfl_sync(0xffffffffu, w.w, lane);
        return e;
    }
    __device__ __forceinline__ void change_sign(bool yes)
    {
        const uint32_t bits = yes ? 0x80008000u : 0u;
        w.x ^= bits, w.y ^= bits, w.z ^= bits, w.w ^= bits;
    }
    static __device__ __forceinline__ void store(uint8_t* p, const float* f)
    {
        uint32_t a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 r = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
            a[j] = *reinterpret_cast<const uint32_t*>(&r);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(a[0], a[1], a[2], a[3]);
    }
    static __device__ __forceinline__ float one(const uint8_t* p, uint32_t i)
    {
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    }
    static __device__ __forceinline__ void store_one(uint8_t* p, uint32_t i, float f)
    {
        reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(f);
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const uint8_t* p)
    {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void unpack(float* f) const
    {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ Eight from(int lane) const
    {
        Eight e;
        e.a.x = __shfl_sync(0xffffffffu, a.x, lane), e.a.y = __shfl_sync(0xffffffffu, a.y, lane);
        e.a.z = __shfl_sync(0xffffffffu, a.z, lane), e.a.w = __shfl_sync(0xffffffffu, a.w, lane);
        e.b.x = __shfl_sync(0xffffffffu, b.x, lane), e.b.y = __shfl_sync(0xffffffffu, b.y, lane);
        e.b.z = __shfl_sync(0xffffffffu, b.z, lane), e.b.w = __shfl_sync(0xffffffffu, b.w, lane);
        return e;
    }
    __device__ __forceinline__ void change_sign(bool yes)
    {
        const float sign = yes ? -1.0f : 1.0f;
        a.x *= sign, a.y *= sign, a.z *= sign, a.w *= sign;
        b.x *= sign, b.y *= sign, b.z *= sign, b.w *= sign;
    }
    static __device__ __forceinline__ void store(uint8_t* p, const float* f)
    {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    static __device__ __forceinline__ float one(const uint8_t* p, uint32_t i) { return reinterpret_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store_one(uint8_t* p, uint32_t i, float f) { reinterpret_cast<float*>(p)[i] = f; }
};

// A NaN stays one, and becomes its row's scale.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void load4(float* out, const float* from) // 16-byte aligned
{
    const float4 v = *reinterpret_cast<const float4*>(from);
    out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
}

// e4m3 codes of four elements, two of them an instruction.
__device__ __forceinline__ uint32_t four_codes(const float* f, float inv)
{
    uint16_t a, b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(__fmul_rn(f[1], inv)), "f"(__fmul_rn(f[0], inv)));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(__fmul_rn(f[3], inv)), "f"(__fmul_rn(f[2], inv)));
    return static_cast<uint32_t>(a) | static_cast<uint32_t>(b) << 16;
}

// What a block knows of a token.
struct TokenPlace {
    int32_t live; // has a place in the cache (rows targets: always)
    int64_t position;
    int64_t row[2], scale[2]; // of K and V: bytes to its row of the first head, elements to its scale
};

__device__ __forceinline__ int64_t given_position(const TurnParams& p, uint32_t token)
{
    return p.positions64 ? static_cast<const int64_t*>(p.positions)[token] : static_cast<const int32_t*>(p.positions)[token];
}

// Whole warp. The sequence of a row and its place in the cache.
__device__ __forceinline__ TokenPlace place_in_cache(const TurnParams& p, uint32_t token)
{
    TokenPlace r {};
    uint32_t seq = token, fresh = 1, within = 0;
    bool there = token < p.view.batch;
    if (p.q_indptr != nullptr) {
        seq = warp_upper(p.q_indptr, p.view.batch + 1, static_cast<int32_t>(token));
        there = seq < p.view.batch;
        if (there) {
            const int32_t a = p.q_indptr[seq], b = p.q_indptr[seq + 1];
            there = a >= 0 && static_cast<uint32_t>(a) <= token && b > static_cast<int32_t>(token);
            fresh = b - a;
            within = token - a;
        }
    }
    if (!there)
        return r;
    const SeqPages s = seq_pages(p.view, seq);
    const int64_t pos = static_cast<int64_t>(s.length) - fresh + within;
    if (pos < 0 || pos >= s.room)
        return r;
    uint32_t slot;
    const int64_t page = page_of(p.view, s, static_cast<uint32_t>(pos), &slot);
    r.live = page >= 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const PagedPool& pool = i == 0 ? p.view.k : p.view.v;
        r.row[i] = page * pool.page_stride + slot * pool.slot_stride;
        r.scale[i] = page * pool.scale_page_stride + slot * pool.scale_slot_stride;
    }
    r.position = p.positions != nullptr ? given_position(p, token) : pos;
    return r;
}

template <typename T, int TARGET, int LAYOUT, int PARTS> __global__ void __launch_bounds__(kRowThreads) turn_rows_kernel(TurnParams p)
{
    constexpr bool CACHE = TARGET != TARGET_ROWS;
    static_assert(PARTS == 1 || LAYOUT != LAYOUT_HALF_ODD, "eights of a half");
    __shared__ __align__(16) float s_cos[LAYOUT == LAYOUT_NONE ? 1 : kMaxTokens * kMaxHeadDim / 2];
    __shared__ __align__(16) float s_sin[LAYOUT == LAYOUT_NONE ? 1 : kMaxTokens * kMaxHeadDim / 2];
    __shared__ TokenPlace s_place[kMaxTokens];
    chain_begin();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t lanes = 1u << p.group_log, sub = lane & (lanes - 1);
    const uint32_t per_warp = 32 >> p.group_log, per_pass = (kRowThreads / 32) * per_warp;
    const uint32_t token0 = blockIdx.x * p.block_tokens;
    const uint32_t tokens = min(p.block_tokens, p.tokens - token0);
    const uint32_t count = tokens * p.rows_per_token;
    const uint32_t step = p.dim / PARTS; // from one of a lane's eights to the next
    const auto first_of = [&](int part) { return sub * 8 + part * step; };
    const bool in_row = sub * 8 < step;

    struct Row {
        uint32_t token, head, kind; // token of the block; kind 0 q, 1 k, 2 v, 3 none
        const uint8_t* src;
    };
    const auto row_at = [&](uint32_t i) {
        Row r { 0, 0, 3, nullptr };
        if (i < count) {
            r.token = p.row_div.div(i);
            r.head = i - r.token * p.rows_per_token;
            const Rows* rows = &p.q;
            r.kind = 0;
            if (r.head >= p.q.heads) {
                r.head -= p.q.heads;
                rows = &p.k;
                r.kind = 1;
                if (r.head >= p.k.heads) {
                    r.head -= p.k.heads;
                    rows = &p.v;
                    r.kind = 2;
                }
            }
            r.src = rows->src + (token0 + r.token) * rows->src_token + r.head * rows->src_head;
        }
        return r;
    };

    uint32_t i = warp * per_warp + (lane >> p.group_log);
    Row row = row_at(i);
    Eight<T> x[PARTS];
#pragma unroll
    for (int u = 0; u < PARTS; ++u) {
        x[u].zero();
        if (row.kind < 3 && in_row)
            x[u].load(row.src + first_of(u) * sizeof(T));
    }

    if (warp < tokens) {
        TokenPlace place {};
        place.live = 1;
        if constexpr (CACHE)
            place = place_in_cache(p, token0 + warp);
        else
            place.position = given_position(p, token0 + warp);
        if (lane == 0)
            s_place[warp] = place;
    }
    if constexpr (LAYOUT != LAYOUT_NONE) {
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < tokens * p.half; j += kRowThreads) {
            const uint32_t t = j / p.half, f = j - t * p.half;
            // whole turns are taken off in 64 bits; what is left is below half a turn and exact to 2^-25 of one
            double turns = static_cast<double>(s_place[t].position) * p.inv_freq[f] * 0.15915494309189533577;
            turns -= rint(turns);
            float s, c;
            sincospif(2.0f * static_cast<float>(turns), &s, &c);
            s_cos[t * (kMaxHeadDim / 2) + f] = c * p.scale;
            s_sin[t * (kMaxHeadDim / 2) + f] = s * p.scale;
        }
    }
    __syncthreads();

    // every warp makes the same number of passes, for its shuffles
    for (uint32_t base = warp * per_warp; base < count; base += per_pass) {
        const uint32_t next = i + per_pass;
        const Row next_row = row_at(next);
        Eight<T> next_x[PARTS];
        float f[8 * PARTS];
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            next_x[u].zero();
            if (next_row.kind < 3 && in_row)
                next_x[u].load(next_row.src + first_of(u) * sizeof(T));
            x[u].unpack(f + 8 * u);
        }
        const float* cs = s_cos + row.token * (kMaxHeadDim / 2);
        const float* sn = s_sin + row.token * (kMaxHeadDim / 2);
        const uint32_t e0 = sub * 8;
        const bool turned = LAYOUT != LAYOUT_NONE && row.kind < 2 && e0 < 2 * p.half && in_row;
        if constexpr (LAYOUT == LAYOUT_HALF && PARTS == 2) { // half = dim / 2: the partners are the lane's own
            if (turned) {
                float c[8], s[8];
                load4(c, cs + e0), load4(c + 4, cs + e0 + 4);
                load4(s, sn + e0), load4(s + 4, sn + e0 + 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float a = f[j], b = f[8 + j];
                    f[j] = a * c[j] - b * s[j];
                    f[8 + j] = b * c[j] + a * s[j];
                }
            }
        } else if constexpr (LAYOUT == LAYOUT_HALF) { // half % 8 == 0: a lane's elements are all in one half
            const bool second = e0 >= p.half;
            const int32_t away = second ? -static_cast<int32_t>(p.half / 8) : static_cast<int32_t>(p.half / 8);
            Eight<T> other = x[0].from(turned ? static_cast<int32_t>(lane) + away : static_cast<int32_t>(lane));
            if (turned) {
                other.change_sign(!second);
                float o[8], c[8], s[8];
                other.unpack(o);
                const uint32_t j0 = second ? e0 - p.half : e0;
                load4(c, cs + j0), load4(c + 4, cs + j0 + 4);
                load4(s, sn + j0), load4(s + 4, sn + j0 + 4);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    f[j] = f[j] * c[j] + o[j] * s[j];
            }
        } else if constexpr (LAYOUT == LAYOUT_HALF_ODD) {
            if (turned) {
                for (int j = 0; j < 8; ++j) {
                    const uint32_t e = e0 + j;
                    if (e < p.half) {
                        f[j] = f[j] * cs[e] - Eight<T>::one(row.src, e + p.half) * sn[e];
                    } else if (e < 2 * p.half) {
                        f[j] = f[j] * cs[e - p.half] + Eight<T>::one(row.src, e - p.half) * sn[e - p.half];
                    }
                }
            }
            __syncwarp(); // in place: a row's partners are read before any of it is written
        } else if constexpr (LAYOUT == LAYOUT_PAIRS) {
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const uint32_t pair0 = first_of(u) / 2;
                if (turned && pair0 < p.half) {
                    float c[4], s[4]; // (what lies behind the row's angles is not used)
                    load4(c, cs + pair0);
                    load4(s, sn + pair0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (pair0 + j < p.half) {
                            const float a = f[8 * u + 2 * j], b = f[8 * u + 2 * j + 1];
                            f[8 * u + 2 * j] = a * c[j] - b * s[j];
                            f[8 * u + 2 * j + 1] = b * c[j] + a * s[j];
                        }
                    }
                }
            }
        }

        const TokenPlace& place = s_place[row.token];
        const bool live = row.kind < 3 && place.live != 0;
        if (row.kind == 0 || (!CACHE && row.kind == 1)) {
            const Rows& r = row.kind == 0 ? p.q : p.k;
            const bool in_place = row.kind == 0 ? p.in_place_q : p.in_place_k;
            if (live && in_row) {
                uint8_t* dst = r.dst + (token0 + row.token) * r.dst_token + row.head * r.dst_head;
#pragma unroll
                for (int u = 0; u < PARTS; ++u)
                    if (!in_place || (turned && first_of(u) < 2 * p.half)) // what is passed through in place stays there
                        Eight<T>::store(dst + first_of(u) * sizeof(T), f + 8 * u);
            }
        }
        if constexpr (CACHE) {
            const bool to_cache = live && row.kind != 0;
            const PagedPool& pool = row.kind == 1 ? p.view.k : p.view.v;
            uint8_t* const cached = pool.data + (row.kind == 1 ? place.row[0] : place.row[1]) + row.head * pool.head_stride;
            if constexpr (TARGET == TARGET_BF16) {
                if (to_cache && in_row)
#pragma unroll
                    for (int u = 0; u < PARTS; ++u)
                        Eight<T>::store(cached + first_of(u) * 2, f + 8 * u);
            } else {
                float amax = 0.0f;
                if (__any_sync(0xffffffffu, to_cache)) {
#pragma unroll
                    for (int j = 0; j < 8 * PARTS; ++j)
                        amax = max_nan(amax, fabsf(f[j]));
                    for (uint32_t o = lanes / 2; o > 0; o >>= 1)
                        amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                }
                if (to_cache) {
                    const float s = amax != amax ? amax : fp8_scale_of(amax), inv = __frcp_rn(s);
                    if (in_row)
#pragma unroll
                        for (int u = 0; u < PARTS; ++u)
                            *reinterpret_cast<uint2*>(cached + first_of(u))
                                = make_uint2(four_codes(f + 8 * u, inv), four_codes(f + 8 * u + 4, inv));
                    if (sub == 0)
                        pool.scale[(row.kind == 1 ? place.scale[0] : place.scale[1]) + row.head * pool.scale_head_stride] = s;
                }
            }
        }
        i = next;
        row = next_row;
#pragma unroll
        for (int u = 0; u < PARTS; ++u)
            x[u] = next_x[u];
    }
}

// ---- reading back ------------------------------------------------------------------------------

constexpr uint32_t kGatherTokens = 8; // rows of the output per block

struct GatherParams {
    PagedView view;
    const int32_t* start;
    const int32_t* out_indptr;
    uint8_t *k_out, *v_out;
    int64_t k_token, k_head, v_token, v_head; // bytes
    uint32_t rows, group_log, units; // a lane moves 16 bytes of the cache; `units` of them in a row
    FastDiv head_div;                // by kv_heads
};

template <bool FP8>
__device__ __forceinline__ void put_cached(uint8_t* dst, const uint4& w, float scale)
{
    if constexpr (!FP8) {
        *reinterpret_cast<uint4*>(dst) = w;
    } else {
        const uint32_t in[4] = { w.x, w.y, w.z, w.w };
        uint32_t out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = e4m3x2_to_f16x2(in[j / 2] >> (16 * (j & 1)));
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
            const __nv_bfloat162 r = __floats2bfloat162_rn(v.x * scale, v.y * scale);
            out[j] = *reinterpret_cast<const uint32_t*>(&r);
        }
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(out[0], out[1], out[2], out[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
}

template <bool FP8> __global__ void __launch_bounds__(kRowThreads, 6) kv_gather_kernel(GatherParams p)
{
    __shared__ int32_t s_page[kGatherTokens];
    __shared__ uint32_t s_slot[kGatherTokens];
    chain_begin();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row0 = blockIdx.x * kGatherTokens;
    const uint32_t rows = min(kGatherTokens, p.rows - row0);
    for (uint32_t r = warp; r < rows; r += kRowThreads / 32) {
        const int32_t row = static_cast<int32_t>(row0 + r);
        const uint32_t seq = warp_upper(p.out_indptr, p.view.batch + 1, row);
        int32_t page = -1;
        uint32_t slot = 0;
        if (seq < p.view.batch) {
            const int32_t a = p.out_indptr[seq], b = p.out_indptr[seq + 1];
            const int64_t pos = static_cast<int64_t>(row) - a + (p.start != nullptr ? p.start[seq] : 0);
            if (a <= row && b > row && pos >= 0) {
                const SeqPages s = seq_pages(p.view, seq);
                if (pos < s.room)
                    page = page_of(p.view, s, static_cast<uint32_t>(pos), &slot);
            }
        }
        if (lane == 0) {
            s_page[r] = page;
            s_slot[r] = slot;
        }
    }
    __syncthreads();
    const uint32_t sub = lane & ((1u << p.group_log) - 1);
    const uint32_t step = kRowThreads >> p.group_log;
    const uint32_t count = rows * p.view.kv_heads;
    if (sub >= p.units)
        return;
    constexpr uint32_t kWide = FP8 ? 32 : 16; // bytes written per lane
#pragma unroll 4
    for (uint32_t i = threadIdx.x >> p.group_log; i < count; i += step) {
        const uint32_t r = p.head_div.div(i), head = i - r * p.view.kv_heads;
        const int64_t page = s_page[r];
        if (page < 0)
            continue;
        const uint32_t slot = s_slot[r];
        const PagedPool &k = p.view.k, &v = p.view.v;
        const uint4 kw = *reinterpret_cast<const uint4*>(k.data + page * k.page_stride + head * k.head_stride
                                                         + slot * k.slot_stride + sub * 16);
        const uint4 vw = *reinterpret_cast<const uint4*>(v.data + page * v.page_stride + head * v.head_stride
                                                         + slot * v.slot_stride + sub * 16);
        float ks = 1.0f, vs = 1.0f;
        if constexpr (FP8) {
            ks = k.scale[page * k.scale_page_stride + head * k.scale_head_stride + slot * k.scale_slot_stride];
            vs = v.scale[page * v.scale_page_stride + head * v.scale_head_stride + slot * v.scale_slot_stride];
        }
        put_cached<FP8>(p.k_out + (row0 + r) * p.k_token + head * p.k_head + sub * kWide, kw, ks);
        put_cached<FP8>(p.v_out + (row0 + r) * p.v_token + head * p.v_head + sub * kWide, vw, vs);
    }
}

// ---- checks ----------------------------------------------------------------------------------------

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// Elements of tables are read one by one, by their own size.
qsfi_status check_aligned(qsfi_context* ctx, const void* ptr, uint32_t size, const char* op, const char* name)
{
    if (reinterpret_cast<uintptr_t>(ptr) % size != 0)
        return set_invalid_arg(ctx, "%s %s must be aligned to its elements of %u bytes", op, name, size);
    return QSFI_STATUS_OK;
}

qsfi_status check_dim(qsfi_context* ctx, int64_t dim, const char* op)
{
    if (dim % 8 != 0 || dim > static_cast<int64_t>(kMaxHeadDim))
        return set_unsupported(ctx, "%s head_dim must be a multiple of 8 and at most %u", op, kMaxHeadDim);
    return QSFI_STATUS_OK;
}

qsfi_status check_rotary(qsfi_context* ctx, const qsfi_tensor1& inv_freq, float scale, int64_t dim, const char* op)
{
    if (inv_freq.dtype != QS3_DTYPE_F64 || inv_freq.stride[0] != 1)
        return set_invalid_arg(ctx, "%s inv_freq must be contiguous f64", op);
    if (inv_freq.shape[0] <= 0 || 2 * inv_freq.shape[0] > dim)
        return set_invalid_arg(ctx, "%s inv_freq must have between 1 and head_dim / 2 entries", op);
    if (!std::isfinite(scale))
        return set_invalid_arg(ctx, "%s scale must be finite", op);
    return check_aligned(ctx, inv_freq.data, 8, op, "inv_freq");
}

qsfi_status check_positions(qsfi_context* ctx, const qsfi_tensor1& t, int64_t rows, const char* op)
{
    if ((t.dtype != QSFI_DTYPE_I32 && t.dtype != QS3_DTYPE_I64) || t.stride[0] != 1 || t.shape[0] < rows)
        return set_invalid_arg(ctx, "%s positions must be contiguous i32 or i64, one per row", op);
    return check_aligned(ctx, t.data, t.dtype == QS3_DTYPE_I64 ? 8 : 4, op, "positions");
}

void fill_rows(Rows* r, const qsfi_tensor3& src, const qsfi_tensor3& dst, int64_t size)
{
    r->src = static_cast<const uint8_t*>(src.data);
    r->dst = static_cast<uint8_t*>(dst.data);
    r->src_token = src.stride[0] * size;
    r->src_head = src.stride[1] * size;
    r->dst_token = dst.stride[0] * size;
    r->dst_head = dst.stride[1] * size;
    r->heads = static_cast<uint32_t>(src.shape[1]);
}

uint32_t log2_up(uint32_t v)
{
    uint32_t l = 0;
    while ((1u << l) < v)
        ++l;
    return l;
}

void fill_blocks(TurnParams* p, uint32_t parts)
{
    p->group_log = log2_up(p->dim / (8 * parts));
    p->rows_per_token = p->q.heads + p->k.heads + p->v.heads;
    p->row_div = FastDiv(p->rows_per_token);
    // As many tokens as the angles have room for, while every SM gets eight blocks: angles of several tokens keep a block's
    // threads busy where one token's would a quarter of them, and its rows' loads run ahead of its stores. A token of 40 rows a
    // block: 8190 tokens 38.7 us, 36.3 with eight; 10 800 tokens of 48 rows into an e4m3 cache 61.2, 55.7.
    uint32_t n = kMaxTokens;
    while (n > 1 && p->tokens / n < kSmCount * 8)
        --n;
    p->block_tokens = n;
}

// A lane has sixteen elements of a row, eight of either half, where none needs a partner from another lane: what is done once a
// row, addresses, scales and places, is then done by half as many lanes. 8192 tokens of 32 and 8 heads of 128, eight elements a
// lane and sixteen: turned in halves 43.7 us, 32.8, appended as well to an e4m3 cache 52.8, 39.5; 128 tokens 3.1, 2.6 and 4.8, 4.2.
template <typename T, int TARGET, int PARTS> cudaError_t launch_turn_parts(TurnParams* p, bool interleaved, cudaStream_t stream)
{
    fill_blocks(p, PARTS);
    const dim3 grid((p->tokens + p->block_tokens - 1) / p->block_tokens);
    auto kernel = turn_rows_kernel<T, TARGET, LAYOUT_PAIRS, PARTS>;
    if (p->half == 0) {
        if constexpr (TARGET != TARGET_ROWS)
            kernel = turn_rows_kernel<T, TARGET, LAYOUT_NONE, PARTS>;
    } else if (!interleaved) {
        if constexpr (PARTS == 1)
            kernel = p->half % 8 == 0 ? turn_rows_kernel<T, TARGET, LAYOUT_HALF, 1> : turn_rows_kernel<T, TARGET, LAYOUT_HALF_ODD, 1>;
        else
            kernel = turn_rows_kernel<T, TARGET, LAYOUT_HALF, PARTS>;
    }
    return launch_chained(kernel, grid, kRowThreads, 0, stream, *p);
}

template <typename T, int TARGET> cudaError_t launch_turn(TurnParams* p, bool interleaved, cudaStream_t stream)
{
    if constexpr (sizeof(T) == 2) {
        const bool own = p->half == 0 || interleaved || 2 * p->half == p->dim;
        if (p->dim % 16 == 0 && own)
            return launch_turn_parts<T, TARGET, 2>(p, interleaved, stream);
    }
    return launch_turn_parts<T, TARGET, 1>(p, interleaved, stream);
}

// Offsets of slots, heads and pages stay positive and apart.
template <typename Pool> bool pool_strides_ok(const Pool& t, int64_t unit)
{
    return t.stride[3] == 1 && t.stride[0] * unit % 16 == 0 && t.stride[1] * unit % 16 == 0 && t.stride[2] * unit % 16 == 0
        && t.stride[0] >= 0 && t.stride[1] >= 0 && t.stride[2] >= t.shape[3];
}

// Slots of a pool that is written, `width` elements each, share no memory. (Enough, and true of every order of the dimensions.)
bool slots_apart(const int64_t* shape, const int64_t* stride, int64_t width)
{
    int order[3] = { 0, 1, 2 };
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
    for (const int i : order) {
        if (shape[i] == 1)
            continue;
        if (stride[i] < width)
            return false;
        width += (shape[i] - 1) * stride[i];
    }
    return true;
}

qsfi_status check_written_cache(qsfi_context* ctx, const qs3_paged_kv_cache& c, bool fp8, const char* op)
{
    if (c.k.data == c.v.data || (fp8 && c.k_scale.data == c.v_scale.data))
        return set_invalid_arg(ctx, "%s cache k and v must be apart", op);
    bool apart = slots_apart(c.k.shape, c.k.stride, c.k.shape[3]) && slots_apart(c.v.shape, c.v.stride, c.v.shape[3]);
    if (fp8)
        apart = apart && slots_apart(c.k_scale.shape, c.k_scale.stride, 1) && slots_apart(c.v_scale.shape, c.v_scale.stride, 1);
    if (!apart)
        return set_invalid_arg(ctx, "%s slots of the cache must not overlap", op);
    return QSFI_STATUS_OK;
}

} // namespace

// A tensor of rows of one head: positive extents, contiguous and 16-byte aligned rows.
qsfi_status check_rows(qsfi_context* ctx, const qsfi_tensor3& t, const char* op, const char* name, qsfi_dtype dtype)
{
    if (t.data == nullptr)
        return set_invalid_arg(ctx, "%s %s.data must not be null", op, name);
    if (t.dtype != dtype)
        return set_invalid_arg(ctx, "%s %s dtype does not match expected dtype", op, name);
    const int64_t size = dtype == QSFI_DTYPE_F32 ? 4 : 2;
    for (int i = 0; i < 3; ++i)
        if (t.shape[i] <= 0 || t.stride[i] < 0 || t.shape[i] > std::numeric_limits<int32_t>::max())
            return set_invalid_arg(ctx, "%s %s shape entries must be positive and strides not negative", op, name);
    if (t.stride[2] != 1 || !aligned16(t.data) || t.stride[0] * size % 16 != 0 || t.stride[1] * size % 16 != 0)
        return set_invalid_arg(ctx, "%s %s needs a contiguous head dimension and 16-byte aligned rows", op, name);
    return QSFI_STATUS_OK;
}

qsfi_status check_index(qsfi_context* ctx, const qsfi_tensor1& t, const char* op, const char* name, int64_t length)
{
    if (t.data == nullptr)
        return set_invalid_arg(ctx, "%s %s.data must not be null", op, name);
    if (t.dtype != QSFI_DTYPE_I32)
        return set_invalid_arg(ctx, "%s %s must be i32", op, name);
    if (t.stride[0] != 1 || t.shape[0] < length || t.shape[0] > std::numeric_limits<int32_t>::max())
        return set_invalid_arg(ctx, "%s %s must be contiguous and hold at least %lld entries", op, name,
                               static_cast<long long>(length));
    return check_aligned(ctx, t.data, 4, op, name);
}

RowSet row_set(const qsfi_tensor3& t)
{
    const int64_t size = t.dtype == QSFI_DTYPE_F32 ? 4 : 2;
    return RowSet { t.data, t.shape[0], t.shape[1], t.stride[0] * size, t.stride[1] * size, t.shape[2] * size };
}

// What is written may not lie over another operand.
qsfi_status check_apart(qsfi_context* ctx, const char* op, const char* written, const RowSet& a, const char* other, const RowSet& b)
{
    if (a.data != nullptr && b.data != nullptr && rows_meet(a, b))
        return set_invalid_arg(ctx, "%s %s overlaps %s", op, written, other);
    return QSFI_STATUS_OK;
}

// `out`, or where it is absent x itself, becomes `dst`. The two may be the same rows or apart, nothing between.
qsfi_status check_out(qsfi_context* ctx, const qsfi_tensor3& x, const qsfi_tensor3& out, const char* op, const char* name,
                      qsfi_tensor3* dst, int* in_place)
{
    *dst = out.data != nullptr ? out : x;
    if (out.data != nullptr) {
        if (const qsfi_status s = check_rows(ctx, out, op, name, x.dtype); s != QSFI_STATUS_OK)
            return s;
        for (int i = 0; i < 3; ++i)
            if (out.shape[i] != x.shape[i])
                return set_invalid_arg(ctx, "%s %s shape must match its input", op, name);
    }
    const RowSet from = row_set(x), to = row_set(*dst);
    if (!rows_apart(to))
        return set_invalid_arg(ctx, "%s %s rows must not overlap", op, name);
    *in_place = same_rows(from, to);
    if (!*in_place && rows_meet(from, to))
        return set_invalid_arg(ctx, "%s %s overlaps its input without being the same rows", op, name);
    return QSFI_STATUS_OK;
}

bool rows_fit(const PagedView& v)
{
    for (const PagedPool* p : { &v.k, &v.v })
        if (((v.pages - 1) * static_cast<uint64_t>(p->page_stride) + (v.page_size - 1) * static_cast<uint64_t>(p->slot_stride)) >> p->unit_shift
                >= 0xffffffffu
            || (v.pages > 1 && p->scale_page_stride >> 30 != 0) || (v.page_size > 1 && p->scale_slot_stride >> 30 != 0))
            return false;
    return true;
}

qsfi_status paged_view(qsfi_context* ctx, const qs3_paged_kv_cache& cache, const qs3_page_table& table, const char* op,
                       PagedView* out, bool* fp8)
{
    if (cache.k.data == nullptr || cache.v.data == nullptr)
        return set_invalid_arg(ctx, "%s cache k.data and v.data must not be null", op);
    *fp8 = cache.k.dtype == QSFI_DTYPE_FP8_E4M3;
    if (!*fp8 && cache.k.dtype != QSFI_DTYPE_BF16)
        return set_unsupported(ctx, "%s supports only bf16 and e4m3 caches", op);
    if (cache.v.dtype != cache.k.dtype)
        return set_invalid_arg(ctx, "%s cache k and v must have the same dtype", op);
    for (int i = 0; i < 4; ++i) {
        if (cache.k.shape[i] <= 0 || cache.k.shape[i] > std::numeric_limits<int32_t>::max())
            return set_invalid_arg(ctx, "%s cache shape entries must be positive", op);
        if (cache.v.shape[i] != cache.k.shape[i])
            return set_invalid_arg(ctx, "%s cache k and v must have the same shape", op);
    }
    if (const qsfi_status s = check_dim(ctx, cache.k.shape[3], op); s != QSFI_STATUS_OK)
        return s;
    if (*fp8 && cache.k.shape[3] % 16 != 0)
        return set_unsupported(ctx, "%s e4m3 caches need a head_dim that is a multiple of 16", op);
    const int64_t unit = *fp8 ? 1 : 2;
    if (!pool_strides_ok(cache.k, unit) || !pool_strides_ok(cache.v, unit) || !aligned16(cache.k.data)
        || !aligned16(cache.v.data))
        return set_invalid_arg(ctx, "%s cache needs a contiguous head dimension and 16-byte aligned rows", op);
    if (*fp8) {
        for (const qsfi_tensor3* s : { &cache.k_scale, &cache.v_scale }) {
            if (s->data == nullptr || s->dtype != QSFI_DTYPE_F32)
                return set_invalid_arg(ctx, "%s an e4m3 cache needs f32 k_scale and v_scale", op);
            for (int i = 0; i < 3; ++i)
                if (s->shape[i] != cache.k.shape[i] || s->stride[i] < 0)
                    return set_invalid_arg(ctx, "%s k_scale and v_scale must be [pages, kv_heads, page_size]", op);
            if ((reinterpret_cast<uintptr_t>(s->data) & 3u) != 0)
                return set_invalid_arg(ctx, "%s k_scale and v_scale must be 4-byte aligned", op);
        }
    } else if (cache.k_scale.data != nullptr || cache.v_scale.data != nullptr) {
        return set_invalid_arg(ctx, "%s a bf16 cache takes no scales", op);
    }
    const int64_t batch = table.kv_len.shape[0];
    if (batch <= 0)
        return set_invalid_arg(ctx, "%s kv_len must have one entry per sequence", op);
    if (batch > static_cast<int64_t>(kMaxBatch))
        return set_unsupported(ctx, "%s takes at most %u sequences", op, kMaxBatch);
    qsfi_status s = check_index(ctx, table.kv_len, op, "kv_len", batch);
    if (s == QSFI_STATUS_OK)
        s = check_index(ctx, table.kv_indptr, op, "kv_indptr", batch + 1);
    if (s == QSFI_STATUS_OK)
        s = check_index(ctx, table.kv_indices, op, "kv_indices", 1);
    if (s != QSFI_STATUS_OK)
        return s;

    PagedView v {};
    const auto pool = [&](const qsfi_tensor4& t, const qsfi_tensor3& scale) {
        PagedPool p {};
        p.data = static_cast<uint8_t*>(t.data);
        p.page_stride = t.stride[0] * unit;
        p.head_stride = t.stride[1] * unit;
        p.slot_stride = t.stride[2] * unit;
        p.unit_shift = 4; // (16-byte rows)
        while (p.unit_shift < 20 && (p.page_stride | p.slot_stride) % (int64_t { 2 } << p.unit_shift) == 0)
            ++p.unit_shift;
        p.unit = 1u << p.unit_shift;
        p.page_units = static_cast<uint32_t>(p.page_stride >> p.unit_shift);
        p.slot_units = static_cast<uint32_t>(p.slot_stride >> p.unit_shift);
        p.scale = static_cast<float*>(scale.data);
        p.scale_page_stride = scale.stride[0];
        p.scale_head_stride = scale.stride[1];
        p.scale_slot_stride = scale.stride[2];
        p.scale_page = static_cast<uint32_t>(scale.stride[0] * 4);
        p.scale_slot = static_cast<uint32_t>(scale.stride[2] * 4);
        return p;
    };
    v.k = pool(cache.k, cache.k_scale);
    v.v = pool(cache.v, cache.v_scale);
    v.pages = static_cast<uint32_t>(cache.k.shape[0]);
    v.kv_heads = static_cast<uint32_t>(cache.k.shape[1]);
    v.page_size = static_cast<uint32_t>(cache.k.shape[2]);
    v.head_dim = static_cast<uint32_t>(cache.k.shape[3]);
    v.page_div = FastDiv(v.page_size);
    v.indptr = static_cast<const int32_t*>(table.kv_indptr.data);
    v.indices = static_cast<const int32_t*>(table.kv_indices.data);
    v.length = static_cast<const int32_t*>(table.kv_len.data);
    v.batch = static_cast<uint32_t>(batch);
    v.num_indices = static_cast<uint32_t>(table.kv_indices.shape[0]);
    *out = v;
    return QSFI_STATUS_OK;
}

} // namespace qs3

using namespace qs3;

extern "C" {

qsfi_status qs3_rope(qsfi_context* ctx, const qs3_rope_desc* d)
{
    if (ctx == nullptr)
        return QSFI_STATUS_INVALID_ARGUMENT;
    clear_error(&ctx->last_error);
    if (d == nullptr)
        return set_invalid_arg(ctx, "rope desc must not be null");
    qsfi_status s = activate_context(ctx);
    if (s != QSFI_STATUS_OK)
        return s;
    if (d->q.data != nullptr && d->q.dtype != QSFI_DTYPE_BF16 && d->q.dtype != QSFI_DTYPE_F32)
        return set_unsupported(ctx, "rope supports only bf16/f32 tensors");
    TurnParams p {};
    qsfi_tensor3 dst, k_dst {};
    s = check_rows(ctx, d->q, "rope", "q", d->q.dtype);
    if (s == QSFI_STATUS_OK)
        s = check_dim(ctx, d->q.shape[2], "rope");
    if (s == QSFI_STATUS_OK)
        s = check_out(ctx, d->q, d->q_out, "rope", "q_out", &dst, &p.in_place_q);
    if (s != QSFI_STATUS_OK)
        return s;
    const int64_t size = d->q.dtype == QSFI_DTYPE_F32 ? 4 : 2;
    fill_rows(&p.q, d->q, dst, size);
    if (d->k.data != nullptr) {
        s = check_rows(ctx, d->k, "rope", "k", d->q.dtype);
        if (s != QSFI_STATUS_OK)
            return s;
        if (d->k.shape[0] != d->q.shape[0] || d->k.shape[2] != d->q.shape[2])
            return set_invalid_arg(ctx, "rope q and k must have the same tokens and head_dim");
        s = check_out(ctx, d->k, d->k_out, "rope", "k_out", &k_dst, &p.in_place_k);
        if (s != QSFI_STATUS_OK)
            return s;
        fill_rows(&p.k, d->k, k_dst, size);
    } else if (d->k_out.data != nullptr) {
        return set_invalid_arg(ctx, "rope k_out needs k");
    }
    if (d->positions.data == nullptr || d->inv_freq.data == nullptr)
        return set_invalid_arg(ctx, "rope positions.data and inv_freq.data must not be null");
    s = check_positions(ctx, d->positions, d->q.shape[0], "rope");
    if (s == QSFI_STATUS_OK)
        s = check_rotary(ctx, d->inv_freq, d->scale, d->q.shape[2], "rope");
    if (s != QSFI_STATUS_OK)
        return s;
    if (d->q.shape[1] + d->k.shape[1] > 65536)
        return set_unsupported(ctx, "rope takes at most 65536 heads");
    if (d->k.data != nullptr) {
        s = check_apart(ctx, "rope", "q_out", row_set(dst), "k", row_set(d->k));
        if (s == QSFI_STATUS_OK)
            s = check_apart(ctx, "rope", "k_out", row_set(k_dst), "q", row_set(d->q));
        if (s == QSFI_STATUS_OK)
            s = check_apart(ctx, "rope", "q_out", row_set(dst), "k_out", row_set(k_dst));
        if (s != QSFI_STATUS_OK)
            return s;
    }
    p.tokens = static_cast<uint32_t>(d->q.shape[0]);
    p.dim = static_cast<uint32_t>(d->q.shape[2]);
    p.half = static_cast<uint32_t>(d->inv_freq.shape[0]);
    p.positions = d->positions.data;
    p.positions64 = d->positions.dtype == QS3_DTYPE_I64;
    p.inv_freq = static_cast<const double*>(d->inv_freq.data);
    p.scale = d->scale == 0.0f ? 1.0f : d->scale;
    const bool pairs = d->interleaved != 0;
    return set_cuda_error(ctx,
                          size == 2 ? launch_turn<__nv_bfloat16, TARGET_ROWS>(&p, pairs, ctx->stream)
                                    : launch_turn<float, TARGET_ROWS>(&p, pairs, ctx->stream),
                          "rope");
}

qsfi_status qs3_kv_append(qsfi_context* ctx, const qs3_kv_append_desc* d)
{
    if (ctx == nullptr)
        return QSFI_STATUS_INVALID_ARGUMENT;
    clear_error(&ctx->last_error);
    if (d == nullptr)
        return set_invalid_arg(ctx, "kv_append desc must not be null");
    qsfi_status s = activate_context(ctx);
    if (s != QSFI_STATUS_OK)
        return s;
    TurnParams p {};
    bool fp8 = false;
    s = paged_view(ctx, d->cache, d->table, "kv_append", &p.view, &fp8);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->k, "kv_append", "k", QSFI_DTYPE_BF16);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->v, "kv_append", "v", QSFI_DTYPE_BF16);
    if (s != QSFI_STATUS_OK)
        return s;
    const int64_t rows = d->k.shape[0];
    for (const qsfi_tensor3* t : { &d->k, &d->v })
        if (t->shape[0] != rows || t->shape[1] != static_cast<int64_t>(p.view.kv_heads)
            || t->shape[2] != static_cast<int64_t>(p.view.head_dim))
            return set_invalid_arg(ctx, "kv_append k and v must be [rows, kv_heads, head_dim] of the cache");
    if (d->q_indptr.data != nullptr) {
        s = check_index(ctx, d->q_indptr, "kv_append", "q_indptr", p.view.batch + 1);
        if (s != QSFI_STATUS_OK)
            return s;
        p.q_indptr = static_cast<const int32_t*>(d->q_indptr.data);
    } else if (rows < static_cast<int64_t>(p.view.batch)) {
        return set_invalid_arg(ctx, "kv_append without q_indptr needs a row per sequence");
    }
    fill_rows(&p.k, d->k, d->k, 2);
    fill_rows(&p.v, d->v, d->v, 2);
    if (d->inv_freq.data != nullptr) {
        s = check_rotary(ctx, d->inv_freq, d->rope_scale, p.view.head_dim, "kv_append");
        if (s != QSFI_STATUS_OK)
            return s;
        p.inv_freq = static_cast<const double*>(d->inv_freq.data);
        p.half = static_cast<uint32_t>(d->inv_freq.shape[0]);
        if (d->positions.data != nullptr) {
            s = check_positions(ctx, d->positions, rows, "kv_append");
            if (s != QSFI_STATUS_OK)
                return s;
            p.positions = d->positions.data;
            p.positions64 = d->positions.dtype == QS3_DTYPE_I64;
        }
    } else if (d->q.data != nullptr || d->positions.data != nullptr) {
        return set_invalid_arg(ctx, "kv_append q and positions need inv_freq");
    }
    qsfi_tensor3 dst {};
    if (d->q.data != nullptr) {
        s = check_rows(ctx, d->q, "kv_append", "q", QSFI_DTYPE_BF16);
        if (s == QSFI_STATUS_OK)
            s = check_out(ctx, d->q, d->q_out, "kv_append", "q_out", &dst, &p.in_place_q);
        if (s != QSFI_STATUS_OK)
            return s;
        if (d->q.shape[0] != rows || d->q.shape[2] != static_cast<int64_t>(p.view.head_dim))
            return set_invalid_arg(ctx, "kv_append q must have the rows and head_dim of k");
        if (d->q.shape[1] > 65536)
            return set_unsupported(ctx, "kv_append takes at most 65536 heads");
        fill_rows(&p.q, d->q, dst, 2);
    } else if (d->q_out.data != nullptr) {
        return set_invalid_arg(ctx, "kv_append q_out needs q");
    }
    if (p.view.kv_heads > 65536)
        return set_unsupported(ctx, "kv_append takes at most 65536 heads");
    if (d->q.data != nullptr) {
        s = check_apart(ctx, "kv_append", "q_out", row_set(dst), "k", row_set(d->k));
        if (s == QSFI_STATUS_OK)
            s = check_apart(ctx, "kv_append", "q_out", row_set(dst), "v", row_set(d->v));
    }
    if (s == QSFI_STATUS_OK)
        s = check_written_cache(ctx, d->cache, fp8, "kv_append");
    if (s != QSFI_STATUS_OK)
        return s;
    p.view.err = device_error_word();
    if (p.view.err == nullptr)
        return set_cuda_error(ctx, cudaErrorUnknown, "device error word");
    p.tokens = static_cast<uint32_t>(rows);
    p.dim = p.view.head_dim;
    p.scale = d->rope_scale == 0.0f ? 1.0f : d->rope_scale;
    const bool pairs = d->interleaved != 0;
    return set_cuda_error(ctx,
                          fp8 ? launch_turn<__nv_bfloat16, TARGET_FP8>(&p, pairs, ctx->stream)
                              : launch_turn<__nv_bfloat16, TARGET_BF16>(&p, pairs, ctx->stream),
                          "kv_append");
}

qsfi_status qs3_kv_gather(qsfi_context* ctx, const qs3_kv_gather_desc* d)
{
    if (ctx == nullptr)
        return QSFI_STATUS_INVALID_ARGUMENT;
    clear_error(&ctx->last_error);
    if (d == nullptr)
        return set_invalid_arg(ctx, "kv_gather desc must not be null");
    qsfi_status s = activate_context(ctx);
    if (s != QSFI_STATUS_OK)
        return s;
    GatherParams p {};
    bool fp8 = false;
    s = paged_view(ctx, d->cache, d->table, "kv_gather", &p.view, &fp8);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->k_out, "kv_gather", "k_out", QSFI_DTYPE_BF16);
    if (s == QSFI_STATUS_OK)
        s = check_rows(ctx, d->v_out, "kv_gather", "v_out", QSFI_DTYPE_BF16);
    if (s == QSFI_STATUS_OK)
        s = check_index(ctx, d->out_indptr, "kv_gather", "out_indptr", p.view.batch + 1);
    if (s == QSFI_STATUS_OK && d->kv_start.data != nullptr)
        s = check_index(ctx, d->kv_start, "kv_gather", "kv_start", p.view.batch);
    if (s != QSFI_STATUS_OK)
        return s;
    for (const qsfi_tensor3* t : { &d->k_out, &d->v_out })
        if (t->shape[0] != d->k_out.shape[0] || t->shape[1] != static_cast<int64_t>(p.view.kv_heads)
            || t->shape[2] != static_cast<int64_t>(p.view.head_dim) || !rows_apart(row_set(*t)))
            return set_invalid_arg(ctx, "kv_gather k_out and v_out must be [rows, kv_heads, head_dim] of the cache");
    if (p.view.kv_heads > 65536)
        return set_unsupported(ctx, "kv_gather takes at most 65536 heads");
    s = check_apart(ctx, "kv_gather", "k_out", row_set(d->k_out), "v_out", row_set(d->v_out));
    if (s != QSFI_STATUS_OK)
        return s;
    p.view.err = device_error_word();
    if (p.view.err == nullptr)
        return set_cuda_error(ctx, cudaErrorUnknown, "device error word");
    p.start = static_cast<const int32_t*>(d->kv_start.data);
    p.out_indptr = static_cast<const int32_t*>(d->out_indptr.data);
    p.k_out = static_cast<uint8_t*>(d->k_out.data);
    p.v_out = static_cast<uint8_t*>(d->v_out.data);
    p.k_token = d->k_out.stride[0] * 2;
    p.k_head = d->k_out.stride[1] * 2;
    p.v_token = d->v_out.stride[0] * 2;
    p.v_head = d->v_out.stride[1] * 2;
    p.rows = static_cast<uint32_t>(d->k_out.shape[0]);
    p.units = p.view.head_dim / (fp8 ? 16 : 8);
    p.group_log = log2_up(p.units);
    p.head_div = FastDiv(p.view.kv_heads);
    const dim3 grid((p.rows + kGatherTokens - 1) / kGatherTokens);
    return set_cuda_error(
        ctx, launch_chained(fp8 ? kv_gather_kernel<true> : kv_gather_kernel<false>, grid, kRowThreads, 0, ctx->stream, p),
        "kv_gather");
}

} // extern "C"
