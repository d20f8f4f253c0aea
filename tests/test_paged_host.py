"""The paged cache's operators without a GPU: the arithmetic that cuts a batch into ranges of key tiles (compiled for the host),
and the refusals, which come before any device addressing (made-up device pointers)."""
import ctypes as C
import os
import subprocess

import pytest

from qs3_b200 import capi

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qs3_b200", "csrc")

PROGRAM = r"""
#include "paged_schedule.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace qs3;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main()
{
    // division by multiplication, at the places where it could round wrongly
    for (uint32_t d = 1; d < 5000; d = d < 70 ? d + 1 : d * 5 / 4 + 1) {
        const FastDiv f(d);
        for (uint64_t k = 0; k * d < (1ull << 31); k = k < 100 ? k + 1 : k + (1ull << 31) / d / 97 + 1)
            for (int64_t n : { int64_t(k * d) - 1, int64_t(k * d), int64_t(k * d) + 1 })
                if (n >= 0 && n < (int64_t(1) << 31))
                    CHECK(f.div(uint32_t(n)) == uint32_t(n) / d);
        CHECK(f.div(0x7fffffffu) == 0x7fffffffu / d);
    }
    // every key that a row sees lies in its item's key tiles, every key tile holds one, an item has one at least
    for (uint32_t group : { 1u, 2u, 5u, 16u })
    for (uint32_t row_shift : { 3u, 4u, 7u, 8u })
    for (uint32_t key_shift : { 6u, 7u })
    for (uint32_t window : { 0u, 1u, 7u, 200u })
    for (uint32_t causal : { 0u, 1u })
    for (uint32_t fresh : { 1u, 2u, 3u, 70u, 257u })
    for (uint32_t length : { 0u, 1u, 2u, 63u, 64u, 65u, 300u, 1000u }) {
        if (window != 0 && causal == 0)
            continue;
        const uint32_t rows = 1u << row_shift, keys = 1u << key_shift;
        const AttnTiling a { FastDiv(group), row_shift, key_shift, 2, window, causal, 0 };
        const uint32_t tiles = row_tiles(a, fresh);
        CHECK(uint64_t(tiles) * rows >= uint64_t(fresh) * group && uint64_t(tiles - 1) * rows < uint64_t(fresh) * group);
        for (uint32_t t = 0; t < tiles; ++t) {
            const KeyTiles k = key_tiles(a, fresh, length, t);
            CHECK(k.end > k.first);
            uint32_t low = ~0u, high = 0;
            for (uint32_t r = t * rows; r < (t + 1) * rows && r < fresh * group; ++r) {
                uint32_t lo, hi;
                visible_keys(a, fresh, length, r / group, &lo, &hi);
                const int64_t pos = int64_t(length) - fresh + r / group;
                for (int64_t j = 0; j < length; ++j) {
                    const bool seen = (!causal || j <= pos) && (!window || j > pos - int64_t(window));
                    CHECK(seen == (j >= lo && j < hi));
                }
                if (hi > lo) {
                    low = lo < low ? lo : low;
                    high = hi > high ? hi : high;
                }
            }
            if (high > 0)
                CHECK(k.first <= low / keys && k.end == (high + keys - 1) / keys);
        }
    }
    // key tiles of an item before a place in it
    for (uint32_t cost : { 0u, 1u, 3u }) {
        const AttnTiling a { FastDiv(1), 3, 6, 1, 0, 1, cost };
        for (uint64_t offset = 0; offset < 20; ++offset)
            CHECK(tiles_before(a, offset, 10) == (offset <= cost ? 0 : offset - cost < 10 ? offset - cost : 10));
    }
    // even items are never cut
    {
        AttnTiling a { FastDiv(1), 3, 6, 1, 0, 1, 3 };
        a.even = 1;
        CHECK(cost_of(a, 1) == 1 && cost_of(a, 9) == 1 && tiles_before(a, 0, 9) == 0 && tiles_before(a, 1, 9) == 9 && tiles_before(a, 7, 9) == 9);
    }
    // ranges follow each other, hold everything and differ by one at most
    for (uint64_t total : { 1ull, 2ull, 147ull, 148ull, 149ull, 12345ull, 1ull << 52 })
        for (uint32_t blocks : { 1u, 148u, 1184u })
            for (uint32_t least : { 1u, 2u, 5u }) {
                const uint32_t n = active_blocks(total, blocks, least);
                CHECK(n >= 1 && n <= blocks && block_begin(total, n, 0) == 0 && block_begin(total, n, n) == total);
                for (uint32_t c = 0; c < n; ++c) {
                    const uint64_t size = block_begin(total, n, c + 1) - block_begin(total, n, c);
                    CHECK(size == total / n || size == total / n + 1);
                    // the last block that begins before some place
                    for (uint64_t end : { block_begin(total, n, c) + 1, block_begin(total, n, c + 1) })
                        CHECK(block_of_end(total, n, end) == c);
                }
            }
    return 0;
}
"""


def test_division_into_ranges(tmp_path):
    src, exe = tmp_path / "schedule.cpp", tmp_path / "schedule"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


BF16, F32, I32, I64, U8, F64, E4M3 = (capi.DTYPE_BF16, capi.DTYPE_F32, capi.DTYPE_I32, capi.DTYPE_I64, capi.DTYPE_U8,
                                      capi.DTYPE_F64, capi.DTYPE_FP8_E4M3)


def t(dtype, *shape, ptr=0x10000, stride=None):
    d = (capi.Tensor1, capi.Tensor2, capi.Tensor3, capi.Tensor4)[len(shape) - 1]()
    d.data, d.dtype = ptr, dtype
    strides = [1] * len(shape)
    for i in range(len(shape) - 2, -1, -1):
        strides[i] = strides[i + 1] * max(1, shape[i + 1])
    for i, n in enumerate(shape):
        d.shape[i] = n
        d.stride[i] = strides[i] if stride is None else stride[i]
    return d


@pytest.fixture(scope="module")
def lib():
    return capi.load()


@pytest.fixture()
def ctx(lib):
    handle = C.c_void_p()
    desc = capi.ContextDesc(-1, None)
    assert lib.qsfi_context_create(C.byref(desc), C.byref(handle)) == capi.STATUS_OK
    yield handle
    lib.qsfi_context_destroy(handle)


def refused(lib, ctx, fn, desc, status, fragment):
    assert getattr(lib, fn)(ctx, C.byref(desc)) == status, fragment
    info = capi.ErrorInfo()
    lib.qsfi_context_get_last_error(ctx, C.byref(info))
    assert info.status == status and fragment in info.message.decode(), (fragment, info.message.decode())


INVALID, UNSUPPORTED = capi.STATUS_INVALID_ARGUMENT, capi.STATUS_UNSUPPORTED


def test_null_arguments(lib, ctx):
    for fn in ("qs3_rope", "qs3_kv_append", "qs3_kv_gather", "qs3_paged_attention"):
        assert getattr(lib, fn)(None, None) == INVALID
        assert getattr(lib, fn)(ctx, None) == INVALID


def rope_desc(**kw):
    d = capi.RopeDesc()
    d.q, d.positions, d.inv_freq, d.scale = t(BF16, 4, 2, 64), t(I32, 4), t(F64, 16), 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,fragment", [
    (dict(q=t(BF16, 4, 2, 64, ptr=0)), INVALID, "q.data must not be null"),
    (dict(q=t(U8, 4, 2, 64)), UNSUPPORTED, "bf16/f32"),
    (dict(q=t(BF16, 4, 2, 60)), INVALID, "16-byte aligned rows"),
    (dict(q=t(F32, 4, 2, 60)), UNSUPPORTED, "multiple of 8"),
    (dict(q=t(BF16, 4, 2, 264)), UNSUPPORTED, "at most 256"),
    (dict(q=t(BF16, 0, 2, 64)), INVALID, "positive"),
    (dict(q=t(BF16, 4, 2, 64, ptr=0x10008)), INVALID, "16-byte aligned rows"),
    (dict(q=t(BF16, 4, 2, 64, stride=(128, 64, 2))), INVALID, "contiguous head dimension"),
    (dict(q=t(BF16, 4, 2, 64, stride=(0, 64, 1))), INVALID, "must not overlap"),
    (dict(q=t(BF16, 4, 2, 64, stride=(64, 64, 1))), INVALID, "must not overlap"),
    (dict(k=t(BF16, 5, 2, 64)), INVALID, "same tokens"),
    (dict(k=t(F32, 4, 2, 64)), INVALID, "k dtype"),
    (dict(k_out=t(BF16, 4, 2, 64)), INVALID, "k_out needs k"),
    (dict(q_out=t(BF16, 4, 3, 64)), INVALID, "shape must match"),
    (dict(q_out=t(F32, 4, 2, 64)), INVALID, "q_out dtype"),
    (dict(q_out=t(BF16, 4, 2, 64, ptr=0x10010)), INVALID, "overlaps its input"),
    (dict(positions=t(I32, 4, ptr=0)), INVALID, "positions.data"),
    (dict(positions=t(F32, 4)), INVALID, "i32 or i64"),
    (dict(positions=t(I64, 3)), INVALID, "one per row"),
    (dict(inv_freq=t(F32, 16)), INVALID, "f64"),
    (dict(inv_freq=t(F64, 33)), INVALID, "between 1 and head_dim / 2"),
    (dict(scale=float("nan")), INVALID, "finite"),
])
def test_rope_refusals(lib, ctx, kw, status, fragment):
    refused(lib, ctx, "qs3_rope", rope_desc(**kw), status, fragment)


def cache(fp8=False, pages=10, heads=2, page=16, dim=64, **kw):
    c = capi.PagedKvCache()
    c.k = c.v = t(E4M3 if fp8 else BF16, pages, heads, page, dim)
    if fp8:
        c.k_scale = c.v_scale = t(F32, pages, heads, page)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def table(batch=3, **kw):
    p = capi.PageTable()
    p.kv_indptr, p.kv_indices, p.kv_len = t(I32, batch + 1), t(I32, 8), t(I32, batch)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


PAGED = [
    (dict(cache=cache(k=t(BF16, 10, 2, 16, 64, ptr=0))), INVALID, "must not be null"),
    (dict(cache=cache(k=t(F32, 10, 2, 16, 64))), UNSUPPORTED, "bf16 and e4m3"),
    (dict(cache=cache(v=t(E4M3, 10, 2, 16, 64))), INVALID, "same dtype"),
    (dict(cache=cache(v=t(BF16, 10, 2, 8, 64))), INVALID, "same shape"),
    (dict(cache=cache(k=t(BF16, 10, 0, 16, 64))), INVALID, "positive"),
    (dict(cache=cache(k=t(BF16, 10, 2, 16, 64, ptr=0x10004))), INVALID, "16-byte aligned rows"),
    (dict(cache=cache(k=t(BF16, 10, 2, 16, 64, stride=(2048, 1024, 60, 1)))), INVALID, "16-byte aligned rows"),
    (dict(cache=cache(fp8=True, k_scale=t(F32, 10, 2, 16, ptr=0))), INVALID, "needs f32 k_scale"),
    (dict(cache=cache(fp8=True, v_scale=t(F32, 10, 2, 8))), INVALID, "k_scale and v_scale must be"),
    (dict(cache=cache(k_scale=t(F32, 10, 2, 16))), INVALID, "takes no scales"),
    (dict(table=table(kv_len=t(I64, 3))), INVALID, "kv_len must be i32"),
    (dict(table=table(kv_indptr=t(I32, 3))), INVALID, "kv_indptr must be contiguous"),
    (dict(table=table(kv_indices=t(I32, 8, ptr=0))), INVALID, "kv_indices.data"),
    (dict(table=table(batch=4097)), UNSUPPORTED, "at most 4096"),
]


def append_desc(**kw):
    d = capi.KvAppendDesc()
    d.cache, d.table, d.k, d.v, d.rope_scale = cache(), table(), t(BF16, 3, 2, 64), t(BF16, 3, 2, 64), 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,fragment", PAGED + [
    (dict(cache=cache(dim=12)), UNSUPPORTED, "multiple of 8"),
    (dict(cache=cache(fp8=True, dim=24)), UNSUPPORTED, "multiple of 16"),
    (dict(k=t(BF16, 3, 1, 64)), INVALID, "of the cache"),
    (dict(v=t(BF16, 4, 2, 64)), INVALID, "of the cache"),
    (dict(k=t(F32, 3, 2, 64)), INVALID, "k dtype"),
    (dict(k=t(BF16, 2, 2, 64), v=t(BF16, 2, 2, 64)), INVALID, "a row per sequence"),
    (dict(q_indptr=t(I32, 3)), INVALID, "q_indptr"),
    (dict(q=t(BF16, 3, 4, 64)), INVALID, "need inv_freq"),
    (dict(positions=t(I32, 3)), INVALID, "need inv_freq"),
    (dict(inv_freq=t(F64, 33)), INVALID, "between 1"),
    (dict(inv_freq=t(F64, 8), q=t(BF16, 2, 4, 64)), INVALID, "rows and head_dim of k"),
    (dict(inv_freq=t(F64, 8), q_out=t(BF16, 3, 4, 64)), INVALID, "q_out needs q"),
    (dict(inv_freq=t(F64, 8), positions=t(I32, 2)), INVALID, "one per row"),
])
def test_append_refusals(lib, ctx, kw, status, fragment):
    refused(lib, ctx, "qs3_kv_append", append_desc(**kw), status, fragment)


def gather_desc(**kw):
    d = capi.KvGatherDesc()
    d.cache, d.table, d.out_indptr, d.k_out, d.v_out = cache(), table(), t(I32, 4), t(BF16, 9, 2, 64), t(BF16, 9, 2, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,fragment", PAGED + [
    (dict(out_indptr=t(I32, 3)), INVALID, "out_indptr"),
    (dict(kv_start=t(I32, 2)), INVALID, "kv_start"),
    (dict(v_out=t(BF16, 8, 2, 64)), INVALID, "of the cache"),
    (dict(k_out=t(BF16, 9, 2, 64, stride=(64, 64, 1))), INVALID, "of the cache"),
    (dict(k_out=t(F32, 9, 2, 64)), INVALID, "k_out dtype"),
])
def test_gather_refusals(lib, ctx, kw, status, fragment):
    refused(lib, ctx, "qs3_kv_gather", gather_desc(**kw), status, fragment)


def attention_desc(**kw):
    d = capi.PagedAttentionDesc()
    d.q, d.out, d.cache, d.table, d.causal = t(BF16, 3, 4, 64), t(BF16, 3, 4, 64), cache(), table(), 1
    d.workspace = t(U8, 1 << 30)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,fragment", PAGED + [
    (dict(cache=cache(dim=96), q=t(BF16, 3, 4, 96), out=t(BF16, 3, 4, 96)), UNSUPPORTED, "64, 128 or 256"),
    (dict(q=t(BF16, 3, 4, 128)), INVALID, "cache's head_dim"),
    (dict(q=t(F32, 3, 4, 64)), INVALID, "q dtype"),
    (dict(out=t(BF16, 3, 2, 64)), INVALID, "out shape"),
    (dict(out=t(BF16, 3, 4, 64, stride=(64, 64, 1))), INVALID, "must not overlap"),
    (dict(out=t(BF16, 3, 4, 64, ptr=0x10000 + 128)), INVALID, "overlaps its input"),
    (dict(q=t(BF16, 3, 3, 64), out=t(BF16, 3, 3, 64)), INVALID, "multiple of kv_heads"),
    (dict(q=t(BF16, 2, 4, 64), out=t(BF16, 2, 4, 64)), INVALID, "a row per sequence"),
    (dict(q=t(BF16, 1 << 25, 4, 64), out=t(BF16, 1 << 25, 4, 64)), UNSUPPORTED, "2^24 rows"),
    (dict(q_indptr=t(I32, 3)), INVALID, "q_indptr"),
    (dict(lse=t(F32, 3, 3)), INVALID, "lse"),
    (dict(window=4, causal=0), UNSUPPORTED, "window needs causal"),
    (dict(cache=cache(k=t(E4M3, 4, 2, 16, 64), v=t(E4M3, 4, 2, 16, 64), k_scale=t(F32, 4, 2, 16, stride=(1 << 30, 16, 1)),
                      v_scale=t(F32, 4, 2, 16))), UNSUPPORTED, "scales 2^30 apart"),
    (dict(cache=cache(k=t(BF16, 1 << 30, 2, 16, 64, stride=(2056, 1024, 64, 1)), v=t(BF16, 1 << 30, 2, 16, 64))), UNSUPPORTED, "2^32 rows"),
    (dict(sm_scale=float("inf")), INVALID, "sm_scale"),
    (dict(sm_scale=-1.0), INVALID, "sm_scale"),
    (dict(workspace=t(U8, 1000)), INVALID, "workspace has"),
    (dict(workspace=t(U8, 1 << 30, ptr=0x10080)), INVALID, "256-byte aligned"),
    (dict(workspace=t(F32, 1 << 30)), INVALID, "u8"),
])
def test_attention_refusals(lib, ctx, kw, status, fragment):
    refused(lib, ctx, "qs3_paged_attention", attention_desc(**kw), status, fragment)


def test_workspace_size(lib, ctx):
    n = C.c_size_t(0)
    assert lib.qs3_paged_attention_workspace_size(ctx, 8, 8, 16, 2, 256, C.byref(n)) == capi.STATUS_OK and n.value > 0
    for args in ((0, 8, 16, 2, 256), (8, 8, 15, 2, 256), (8, 0, 16, 2, 256)):
        assert lib.qs3_paged_attention_workspace_size(ctx, *args, C.byref(n)) == INVALID
    assert lib.qs3_paged_attention_workspace_size(ctx, 8, 8, 16, 2, 80, C.byref(n)) == UNSUPPORTED
    assert lib.qs3_paged_attention_workspace_size(ctx, 8, 8, 16, 2, 64, None) == INVALID


ROOM_PROGRAM = r"""
#include "paged_schedule.h"
#include <cstdio>
#include <initializer_list>
using namespace qs3;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main()
{
    // an item's key tiles hold every key that is there and that a row sees by the stated length, and none that lies behind them
    for (uint32_t key_shift : { 6u, 7u })
    for (uint32_t window : { 0u, 1u, 200u })
    for (uint32_t causal : { 0u, 1u })
    for (uint32_t fresh : { 1u, 3u, 70u, 257u })
    for (uint32_t length : { 1u, 64u, 300u, 1000u, 0x7fffffffu })
    for (uint32_t room : { 0u, 1u, 63u, 64u, 65u, 128u, 290u, 300u }) {
        if ((window != 0 && causal == 0) || room > length)
            continue;
        const AttnTiling a { FastDiv(4), 7, key_shift, 2, window, causal, 0 };
        for (uint32_t t = 0; t < row_tiles(a, fresh); ++t) {
            const KeyTiles k = key_tiles(a, fresh, length, t, room);
            CHECK(k.end > k.first);
            CHECK(k.end == k.first + 1 || (uint64_t(k.end - 1) << key_shift) < room);
            CHECK((uint64_t(k.first) << key_shift) <= room);
            for (uint32_t r = t * 128; r < (t + 1) * 128 && r < fresh * 4; ++r) {
                const int64_t pos = int64_t(length) - fresh + r / 4;
                for (int64_t j = 0; j < room; ++j)
                    if ((!causal || j <= pos) && (!window || j > pos - int64_t(window)))
                        CHECK((uint32_t(j) >> key_shift) >= k.first && (uint32_t(j) >> key_shift) < k.end);
            }
        }
    }
    return 0;
}
"""


def test_key_tiles_stay_inside_the_pages(tmp_path):
    src, exe = tmp_path / "room.cpp", tmp_path / "room"
    src.write_text(ROOM_PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


def paged_call(name, pool_dtype, scales=True):
    """A call of ops.<name> on small CPU tensors, by a context without a device: what is refused is refused before any of them is read."""
    import torch

    from qs3_b200 import ops
    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype)
    i32 = lambda n: new(n, dtype=torch.int32)
    scale = lambda: new(4, 2, 16, dtype=torch.float32) if scales else None
    pool = lambda: new(4, 2, 16, 64, dtype=torch.uint8).view(pool_dtype) if pool_dtype.itemsize == 1 else new(4, 2, 16, 64, dtype=pool_dtype)
    c = ops.PagedKvCache(pool(), pool(), scale(), scale())
    p, ctx = ops.PageTable(i32(4), i32(8), i32(3)), ops.Context(device=-1)
    if name == "kv_append":
        ops.kv_append(ctx, c, p, new(3, 2, 64), new(3, 2, 64))
    elif name == "kv_gather":
        ops.kv_gather(ctx, c, p, i32(4), new(3, 2, 64), new(3, 2, 64))
    else:
        ops.paged_attention(ctx, new(3, 4, 64), c, p, new(3, 4, 64), new(1 << 16, dtype=torch.uint8))


@pytest.mark.parametrize("name", ["kv_append", "kv_gather", "paged_attention"])
@pytest.mark.parametrize("dtype", ["float8_e5m2", "int8", "bool", "float8_e4m3fnuz", "bfloat16"])
def test_codes_of_another_kind_are_refused(name, dtype):
    import torch

    from qs3_b200 import ops
    with pytest.raises(ops.Qs3Error, match="e4m3 codes") as e:
        paged_call(name, getattr(torch, dtype))
    assert e.value.status == INVALID


ROWS_PROGRAM = r"""
#include "row_sets.h"
#include <cstdio>
#include <random>
#include <vector>
using namespace qs3;
int main()
{
    static uint8_t memory[1];
    std::mt19937 rng(1);
    const auto pick = [&](int n) { return static_cast<int64_t>(rng() % n); };
    long met = 0, exact = 0, wrong = 0;
    for (int n = 0; n < 400000; ++n) {
        RowSet s[2];
        for (RowSet& x : s) {
            x = RowSet { memory + pick(80), 1 + pick(5), 1 + pick(5), pick(24), pick(24), 1 + pick(4) };
            if (&x == s + 1 && pick(3) != 0)
                x.s0 = s[0].s0, x.s1 = pick(2) ? s[0].s1 : x.s1;
        }
        std::vector<int> used(800);
        bool apart = true, meet = false;
        for (int64_t i = 0; i < s[0].n0; ++i)
            for (int64_t j = 0; j < s[0].n1; ++j)
                for (int64_t k = 0; k < s[0].width; ++k)
                    apart = used[(const uint8_t*)s[0].data - memory + i * s[0].s0 + j * s[0].s1 + k]++ == 0 && apart;
        for (int64_t i = 0; i < s[1].n0; ++i)
            for (int64_t j = 0; j < s[1].n1; ++j)
                for (int64_t k = 0; k < s[1].width; ++k)
                    meet = used[(const uint8_t*)s[1].data - memory + i * s[1].s0 + j * s[1].s1 + k] != 0 || meet;
        if (rows_apart(s[0]) && !apart) { std::printf("rows share memory\n"); return 1; }
        const bool same = (s[0].n0 == 1 || s[1].n0 == 1 || s[0].s0 == s[1].s0) && (s[0].n1 == 1 || s[1].n1 == 1 || s[0].s1 == s[1].s1);
        const bool said = rows_meet(s[0], s[1]);
        if (said != rows_meet(s[1], s[0])) { std::printf("not symmetric\n"); return 1; }
        if (meet && !said) { std::printf("an overlap was missed\n"); return 1; }
        if (same && said && !meet) { std::printf("rows that are apart were taken to meet\n"); return 1; }
        met += meet, exact += same, wrong += said != meet;
    }
    std::printf("%ld %ld %ld\n", met, exact, wrong);
    return met > 10000 && exact > 10000 ? 0 : 1;
}
"""


def test_rows_that_share_memory(tmp_path):
    """Against every byte of small sets."""
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(ROWS_PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


ROPE_Q = dict(q=t(BF16, 4, 2, 64, ptr=0x100000))
KV_PARTS = dict(k=t(BF16, 3, 2, 64, ptr=0x200000), v=t(BF16, 3, 2, 64, ptr=0x300000), inv_freq=t(F64, 8))


@pytest.mark.parametrize("fn,make,kw,fragment", [
    ("qs3_rope", "rope_desc", dict(ROPE_Q, k=t(BF16, 4, 2, 64, ptr=0x100000)), "q_out overlaps k"),
    ("qs3_rope", "rope_desc", dict(ROPE_Q, k=t(BF16, 4, 2, 64, ptr=0x100080)), "q_out overlaps k"),
    ("qs3_rope", "rope_desc", dict(ROPE_Q, q_out=t(BF16, 4, 2, 64, ptr=0x200000), k=t(BF16, 4, 1, 64, ptr=0x200200)), "q_out overlaps k"),
    ("qs3_rope", "rope_desc", dict(ROPE_Q, k=t(BF16, 4, 2, 64, ptr=0x300000), k_out=t(BF16, 4, 2, 64, ptr=0x100000)), "k_out overlaps q"),
    ("qs3_rope", "rope_desc", dict(ROPE_Q, q_out=t(BF16, 4, 2, 64, ptr=0x200000), k=t(BF16, 4, 2, 64, ptr=0x300000),
                                   k_out=t(BF16, 4, 2, 64, ptr=0x200000)), "q_out overlaps k_out"),
    ("qs3_kv_append", "append_desc", dict(KV_PARTS, q=t(BF16, 3, 2, 64, ptr=0x400000), q_out=t(BF16, 3, 2, 64, ptr=0x200000)), "q_out overlaps k"),
    ("qs3_kv_append", "append_desc", dict(KV_PARTS, q=t(BF16, 3, 2, 64, ptr=0x300080)), "q_out overlaps v"),
    ("qs3_kv_append", "append_desc", dict(k=t(BF16, 3, 2, 64, ptr=0x200000)), "cache k and v"),
    ("qs3_kv_append", "append_desc", dict(cache=cache(v=t(BF16, 10, 2, 16, 64, ptr=0x400000, stride=(1024, 0, 64, 1)))), "slots of the cache"),
    ("qs3_kv_append", "append_desc", dict(cache=cache(k=t(BF16, 10, 2, 16, 64, ptr=0x400000, stride=(1024, 1024, 64, 1)))), "slots of the cache"),
    ("qs3_kv_append", "append_desc", dict(cache=cache(fp8=True, k=t(E4M3, 10, 2, 16, 64, ptr=0x400000))), "cache k and v"),
    ("qs3_kv_append", "append_desc", dict(cache=cache(fp8=True, k=t(E4M3, 10, 2, 16, 64, ptr=0x400000),
                                                      k_scale=t(F32, 10, 2, 16, ptr=0x500000, stride=(0, 0, 0)))), "slots of the cache"),
    ("qs3_kv_gather", "gather_desc", dict(), "k_out overlaps v_out"),
    ("qs3_kv_gather", "gather_desc", dict(v_out=t(BF16, 9, 2, 64, ptr=0x10100)), "k_out overlaps v_out"),
    ("qs3_paged_attention", "attention_desc", dict(), "workspace overlaps out"),
    ("qs3_paged_attention", "attention_desc", dict(out=t(BF16, 3, 4, 64, ptr=0x80000000)), "workspace overlaps q"),
    ("qs3_paged_attention", "attention_desc", dict(workspace=t(U8, 1 << 30, ptr=0x1000000), lse=t(F32, 3, 4)), "lse overlaps q"),
    ("qs3_paged_attention", "attention_desc", dict(workspace=t(U8, 1 << 30, ptr=0x1000000), lse=t(F32, 3, 4, ptr=0x200020),
                                                   out=t(BF16, 3, 4, 64, ptr=0x200000)), "lse overlaps out"),
    ("qs3_paged_attention", "attention_desc", dict(workspace=t(U8, 1 << 30, ptr=0x1000000), lse=t(F32, 3, 4, ptr=0x1000020)), "workspace overlaps lse"),
    ("qs3_paged_attention", "attention_desc", dict(workspace=t(U8, 1 << 30, ptr=0x1000000), lse=t(F32, 3, 4, ptr=0x200000, stride=(0, 1))),
     "lse rows must not overlap"),
])
def test_outputs_over_other_operands_are_refused(lib, ctx, fn, make, kw, fragment):
    refused(lib, ctx, fn, globals()[make](**kw), INVALID, fragment)


@pytest.mark.parametrize("fn,make,kw,name", [
    ("qs3_rope", "rope_desc", dict(positions=t(I32, 4, ptr=0x10002)), "positions"),
    ("qs3_rope", "rope_desc", dict(positions=t(I64, 4, ptr=0x10004)), "positions"),
    ("qs3_rope", "rope_desc", dict(inv_freq=t(F64, 16, ptr=0x10004)), "inv_freq"),
    ("qs3_kv_append", "append_desc", dict(inv_freq=t(F64, 16, ptr=0x10004)), "inv_freq"),
    ("qs3_kv_append", "append_desc", dict(inv_freq=t(F64, 16), positions=t(I64, 3, ptr=0x10004)), "positions"),
    ("qs3_kv_append", "append_desc", dict(q_indptr=t(I32, 4, ptr=0x10001)), "q_indptr"),
    ("qs3_kv_append", "append_desc", dict(table=table(kv_len=t(I32, 3, ptr=0x10002))), "kv_len"),
    ("qs3_kv_gather", "gather_desc", dict(table=table(kv_indptr=t(I32, 4, ptr=0x10002))), "kv_indptr"),
    ("qs3_kv_gather", "gather_desc", dict(out_indptr=t(I32, 4, ptr=0x10002)), "out_indptr"),
    ("qs3_kv_gather", "gather_desc", dict(kv_start=t(I32, 3, ptr=0x10002)), "kv_start"),
    ("qs3_paged_attention", "attention_desc", dict(table=table(kv_indices=t(I32, 8, ptr=0x10002))), "kv_indices"),
    ("qs3_paged_attention", "attention_desc", dict(q_indptr=t(I32, 4, ptr=0x10002)), "q_indptr"),
])
def test_misaligned_tables_are_refused(lib, ctx, fn, make, kw, name):
    refused(lib, ctx, fn, globals()[make](**kw), INVALID, f"{name} must be aligned")


@pytest.mark.parametrize("name", ["rope", "kv_append", "kv_gather", "paged_attention"])
def test_tensors_off_the_device_are_refused(name, monkeypatch):
    """CPU tensors in a call by a context of a device (no call is made)."""
    import torch

    from qs3_b200 import ops
    real = ops.Context

    class OfDevice(real):
        def __init__(self, device):
            super().__init__(device=-1)
            self.device = 0
    monkeypatch.setattr(ops, "Context", OfDevice)
    with pytest.raises(ops.Qs3Error, match="on cuda:0") as e:
        if name == "rope":
            ops.rope(OfDevice(0), torch.zeros(4, dtype=torch.int32), ops.rope_frequencies(16, device="cpu").inv_freq,
                     torch.zeros((4, 2, 64), dtype=torch.bfloat16))
        else:
            paged_call(name, torch.bfloat16, scales=False)
    assert e.value.status == INVALID


@pytest.mark.parametrize("zero", [0.0, -0.0, 1e-60])
@pytest.mark.parametrize("name", ["rope", "kv_append", "paged_attention"])
def test_a_scale_of_zero_is_not_the_default(name, zero):
    """0 stands for the default in the C interface, which takes no other zero; the Python one has None and 1."""
    import torch

    from qs3_b200 import ops
    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype)
    i32 = lambda n: new(n, dtype=torch.int32)
    ctx, freq = ops.Context(device=-1), ops.rope_frequencies(16, device="cpu").inv_freq
    c, p = ops.PagedKvCache(new(4, 2, 16, 64), new(4, 2, 16, 64)), ops.PageTable(i32(4), i32(8), i32(3))
    with pytest.raises(ops.Qs3Error, match="scale must not be 0") as e:
        if name == "rope":
            ops.rope(ctx, i32(4), freq, new(4, 2, 64), scale=zero)
        elif name == "kv_append":
            ops.kv_append(ctx, c, p, new(3, 2, 64), new(3, 2, 64), inv_freq=freq, rope_scale=zero)
        else:
            ops.paged_attention(ctx, new(3, 4, 64), c, p, new(3, 4, 64), new(1 << 26, dtype=torch.uint8), sm_scale=zero)
    assert e.value.status == INVALID
