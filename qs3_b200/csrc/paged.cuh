// Views of a paged KV cache and its page table, shared by the kernels that write it, read it back and attend over it.
#pragma once

#include "common.cuh"
#include "paged_schedule.h"
#include "row_sets.h"

namespace qs3 {

// Codes in the device error word: a page id outside the pool, or a sequence longer than its pages.
enum : uint32_t { ERR_PAGE_TABLE = 0x5d000001u };

constexpr uint32_t kMaxHeadDim = 256;
constexpr uint32_t kMaxBatch = 4096;

// Pages of [kv_heads, page_size, head_dim] elements; strides in bytes, scales in elements.
struct PagedPool {
    uint8_t* data;
    int64_t page_stride, head_stride, slot_stride;
    uint32_t unit, unit_shift; // power of two that divides page_stride and slot_stride
    uint32_t page_units, slot_units;
    float* scale;
    int64_t scale_page_stride, scale_head_stride, scale_slot_stride;
    uint32_t scale_page, scale_slot; // the same in bytes, for reads (rows_fit)
};

struct PagedView {
    PagedPool k, v;
    uint32_t pages, kv_heads, page_size, head_dim;
    FastDiv page_div;
    const int32_t* indptr;  // [batch + 1]
    const int32_t* indices; // [num_indices]
    const int32_t* length;  // [batch]
    uint32_t batch, num_indices;
    uint32_t* err;
};

#ifdef __CUDACC__

// 16 bytes to shared memory, zeros where `there` is false.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// Two codes in the low half of x.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t x)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(x)));
    return r;
}

// Tokens of a sequence, and where its page ids begin. Positions, masks and angles go by `length`, as the table says it; what may be
// read or written by `room`, the tokens that its pages hold of them: whatever the tables hold, the ids of positions below it lie
// inside `indices`.
struct SeqPages {
    uint32_t first;  // index of the first page id
    uint32_t length; // tokens
    uint32_t room;   // of them with a place, the first ones
};

__device__ __forceinline__ SeqPages seq_pages(const PagedView& p, uint32_t seq)
{
    const int32_t a = p.indptr[seq], b = p.indptr[seq + 1], n = p.length[seq];
    SeqPages s { 0, 0, 0 };
    if (n <= 0)
        return s;
    s.length = static_cast<uint32_t>(n);
    if (a >= 0 && b > a && static_cast<uint32_t>(a) < p.num_indices) {
        const uint32_t end = min(static_cast<uint32_t>(b), p.num_indices);
        const uint64_t room = static_cast<uint64_t>(end - a) * p.page_size;
        s.first = static_cast<uint32_t>(a);
        s.room = static_cast<uint32_t>(min(room, static_cast<uint64_t>(n)));
    }
    if (s.room != s.length)
        atomicCAS(p.err, 0u, ERR_PAGE_TABLE);
    return s;
}

// Page of position `pos` < room, and the slot in it; -1: the table names a page that is not there.
__device__ __forceinline__ int32_t page_of(const PagedView& p, const SeqPages& s, uint32_t pos, uint32_t* slot)
{
    const uint32_t i = p.page_div.div(pos);
    *slot = pos - i * p.page_size;
    const int32_t page = __ldg(p.indices + s.first + i);
    if (static_cast<uint32_t>(page) < p.pages)
        return page;
    atomicCAS(p.err, 0u, ERR_PAGE_TABLE);
    return -1;
}

// Where a token's row of the first head begins, in the pool's units, which 32 bits hold (rows_fit on the host). None: a token
// that is not there, whose row counts as zeros.
constexpr uint32_t kNoRow = 0xffffffffu;
__device__ __forceinline__ uint32_t row_units(const PagedPool& pool, int32_t page, uint32_t slot)
{
    return page < 0 ? kNoRow : page * pool.page_units + slot * pool.slot_units;
}
__device__ __forceinline__ uint64_t row_bytes(const PagedPool& pool, uint32_t row)
{
    return static_cast<uint64_t>(row == kNoRow ? 0 : row) * pool.unit;
}

// Scale of a token, from that of the first page's first one of the head on.
__device__ __forceinline__ const float* scale_at(const PagedPool& pool, const uint8_t* head, int32_t page, uint32_t slot)
{
    return reinterpret_cast<const float*>(head + static_cast<uint64_t>(static_cast<uint32_t>(page)) * pool.scale_page
                                          + static_cast<uint64_t>(slot) * pool.scale_slot);
}

// Largest i in [0, n) with table[i] <= x, for ascending table[0 .. n] with table[0] <= x; the whole warp searches, 32 places
// at a time. Any table gives an i in range.
__device__ __forceinline__ uint32_t warp_upper(const int32_t* table, uint32_t n, int32_t x)
{
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, len = n; // the answer is in [lo, lo + len)
    while (len > 1) {
        const uint32_t step = (len + 31) / 32;
        const uint32_t at = lo + lane * step;
        const bool le = lane * step < len && (lane == 0 || table[at] <= x);
        const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, le));
        lo += last * step;
        len = min(step, len - last * step);
    }
    return lo;
}

#endif

// Host side: checks and views of the descriptors (kv_cache.cu).
RowSet row_set(const qsfi_tensor3& t);
bool rows_fit(const PagedView& v);
qsfi_status check_rows(qsfi_context* ctx, const qsfi_tensor3& t, const char* op, const char* name, qsfi_dtype dtype);
qsfi_status check_out(qsfi_context* ctx, const qsfi_tensor3& x, const qsfi_tensor3& out, const char* op, const char* name,
                      qsfi_tensor3* dst, int* in_place);
qsfi_status check_apart(qsfi_context* ctx, const char* op, const char* written, const RowSet& a, const char* other, const RowSet& b);
qsfi_status check_index(qsfi_context* ctx, const qsfi_tensor1& t, const char* op, const char* name, int64_t length);
qsfi_status paged_view(qsfi_context* ctx, const qs3_paged_kv_cache& cache, const qs3_page_table& table, const char* op,
                       PagedView* out, bool* fp8);

} // namespace qs3
