"""Attention of new tokens over a paged cache against the formula in 64 bits: head sizes, groups, types, page sizes, lengths
from none to several splits, windows, rows that see nothing, stale memory around everything."""
import math

import pytest
import torch

from paged_helpers import attention_reference, check_attention, ints, make_case, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from qs3_b200 import ops as m
    return m


@pytest.fixture(scope="module")
def ctx(ops):
    return ops.Context()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (4, 2), (5, 1), (16, 2), (16, 1), (40, 2)])
def test_single_tokens(ops, ctx, dim, fp8, heads, kv_heads):
    kv = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 200, 1000, 0]
    c = make_case(ops, [1] * len(kv), kv, heads=heads, kv_heads=kv_heads, dim=dim, fp8=fp8, seed=dim + heads, tail=2)
    out, lse = run_attention(ops, ctx, c, decode=True)
    check_attention(out, lse, c)
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 24, 128])
def test_page_sizes(ops, ctx, page, fp8):
    c = make_case(ops, [1, 3, 1, 9], [50, 131, 7, 300], heads=8, kv_heads=2, dim=128, page=page, fp8=fp8, seed=page)
    out, lse = run_attention(ops, ctx, c)
    check_attention(out, lse, c)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (128, 32, 8), (128, 7, 1), (256, 16, 2), (256, 3, 3)])
@pytest.mark.parametrize("q_len,kv_len", [
    ([1, 0, 5, 33, 130], [1, 0, 700, 40, 130]),
    ([300], [300]),
    ([257, 1, 1], [1030, 513, 2]),
    ([0, 0, 64, 0], [10, 0, 65, 0]),
    ([2, 3, 4], [2000, 1, 3]),          # the second sequence has more new tokens than cache: its first rows see nothing
])
def test_chunks(ops, ctx, q_len, kv_len, dim, heads, kv_heads, fp8):
    c = make_case(ops, q_len, kv_len, heads=heads, kv_heads=kv_heads, dim=dim, fp8=fp8, seed=len(q_len) + dim, tail=3)
    out, lse = run_attention(ops, ctx, c)
    check_attention(out, lse, c)
    out2, _ = run_attention(ops, ctx, c, max_q_len=max(q_len), max_kv_len=max(kv_len))
    check_attention(out2, None, c)


@pytest.mark.parametrize("dim,fp8", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 5000])
def test_windows(ops, ctx, window, dim, fp8):
    c = make_case(ops, [1, 90, 7, 200], [500, 300, 3, 200], heads=8, kv_heads=2, dim=dim, fp8=fp8, seed=window)
    out, lse = run_attention(ops, ctx, c, window=window)
    check_attention(out, lse, c, window=window)


@pytest.mark.parametrize("dim,fp8", [(64, True), (128, False), (256, False)])
def test_without_causal_mask(ops, ctx, dim, fp8):
    c = make_case(ops, [1, 90, 7, 40], [500, 300, 3, 0], heads=8, kv_heads=2, dim=dim, fp8=fp8, seed=3)
    out, lse = run_attention(ops, ctx, c, causal=False, sm_scale=0.05)
    check_attention(out, lse, c, causal=False, scale=0.05)


@pytest.mark.parametrize("dim,fp8,heads", [(64, False, 2), (128, False, 8), (128, True, 4), (256, False, 16), (256, True, 8)])
@pytest.mark.parametrize("kv", [[9001], [64, 8192, 3], [4097, 0, 1, 6000]])
def test_contexts_split_over_blocks(ops, ctx, kv, dim, fp8, heads):
    c = make_case(ops, [1] * len(kv), kv, heads=heads, kv_heads=2, dim=dim, fp8=fp8, seed=sum(kv))
    out, lse = run_attention(ops, ctx, c, decode=True)
    check_attention(out, lse, c)


def test_many_short_sequences(ops, ctx):
    kv = [(37 * i) % 90 for i in range(700)]
    c = make_case(ops, [1] * len(kv), kv, heads=4, kv_heads=2, dim=64, seed=1)
    out, lse = run_attention(ops, ctx, c, decode=True)
    check_attention(out, lse, c)


@pytest.mark.parametrize("fp8", [False, True])
def test_layouts_and_strides(ops, ctx, fp8):
    """A pool of [pages, slots, heads, dim], q and out inside wider rows, heads before tokens."""
    c = make_case(ops, [4, 70], [200, 90], heads=8, kv_heads=2, dim=64, fp8=fp8, seed=5, slots_first=True, q_pad=64)
    wide = torch.full((8, 74, 192), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = run_attention(ops, ctx, c, out=wide.transpose(0, 1)[..., 64:128])
    check_attention(out, lse, c)
    assert bool((wide[..., :64] == 7.0).all()) and bool((wide[..., 128:] == 7.0).all())


def test_large_scores_and_minus_infinity(ops, ctx):
    """Scores of several thousand, and keys of -infinity times a positive query: weights of exactly zero."""
    c = make_case(ops, [1, 40], [70, 100], heads=4, kv_heads=2, dim=64, seed=6)
    c.q.mul_(200.0)
    check_attention(*run_attention(ops, ctx, c), c)
    c = make_case(ops, [1, 1], [70, 100], heads=4, kv_heads=2, dim=64, seed=7)
    c.q.abs_()
    page, slot = int(c.table.kv_indices[0]), 3
    c.cache.k[page, :, slot, 0] = -math.inf
    c.keys[0][slot, :, 0] = -math.inf
    out, lse = run_attention(ops, ctx, c, decode=True)
    want, want_lse, bound, _ = attention_reference(c)
    bound = torch.where(torch.isfinite(bound), bound, 2.0 ** -6 * c.values[0].abs().max())   # (the bound sums |k|)
    assert bool(((out.double() - want).abs() <= bound).all()) and bool(torch.isfinite(lse).all())


def test_pages_that_are_not_there(ops, ctx):
    """Ids outside the pool and lengths beyond the pages are reported, touch nothing and leave the others' results alone."""
    c = make_case(ops, [1, 1, 1], [100, 200, 300], heads=4, kv_heads=2, dim=64, seed=8)
    good, _ = run_attention(ops, ctx, c, decode=True)
    c.table.kv_indices[8] = 1 << 20
    c.table.kv_len[2] = 5000
    out, lse = run_attention(ops, ctx, c, decode=True)
    # (the third sequence's result takes in the stale slots of its last page: its length says that they are tokens)
    assert torch.equal(out[0], good[0]) and bool(torch.isfinite(out[1].float()).all())
    assert ctx.read_device_error() == 0x5d000001
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_replayed_graph_follows_the_tables(ops, fp8):
    """A captured call reads lengths and pages anew at each replay; two graphs may share one workspace."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = ops.Context()
        cases = [make_case(ops, [1, 1, 1], kv, heads=16, kv_heads=2, dim=128, fp8=fp8, seed=9 + i)
                 for i, kv in enumerate(([3000, 5, 700], [64, 2000, 1]))]
        ws = torch.empty(ops.paged_attention_workspace_size(ctx, cases[0].q, cases[0].cache, batch=3), dtype=torch.uint8, device="cuda")
        outs, graphs = [], []
        for c in cases:
            out = torch.zeros_like(c.q)
            ops.paged_attention(ctx, c.q, c.cache, c.table, out, ws)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                ops.paged_attention(ctx, c.q, c.cache, c.table, out, ws)
            outs.append(out)
            graphs.append(graph)
        for short in (False, True):
            if short:
                for c in cases:
                    c.kv_len = [max(1, n // 3) for n in c.kv_len]
                    c.table.kv_len.copy_(ints(c.kv_len))
                    c.keys, c.values = ([x[:n] for x, n in zip(v, c.kv_len)] for v in (c.keys, c.values))
            for out, graph in zip(outs, graphs):
                out.fill_(7.0)
                graph.replay()
            stream.synchronize()
            for c, out in zip(cases, outs):
                check_attention(out, None, c)


def test_results_do_not_depend_on_the_run(ops, ctx):
    c = make_case(ops, [1, 300, 20], [9000, 300, 2222], heads=16, kv_heads=2, dim=128, seed=10)
    first = run_attention(ops, ctx, c)
    for _ in range(3):
        again = run_attention(ops, ctx, c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,heads", [(64, 6), (128, 4), (256, 10)])
@pytest.mark.parametrize("page,slots_first", [(8, False), (32, True), (48, False), (64, False), (128, True), (256, False)])
def test_chunks_over_page_sizes_and_windows(ops, ctx, page, slots_first, dim, heads, fp8):
    """Whole boxes of a page, ends of sequences inside one, and windows that begin inside one, in both row tiles of a chunk."""
    c = make_case(ops, [200, 1, 37], [900, 300, 37], heads=heads, kv_heads=2, dim=dim, page=page, fp8=fp8, seed=page + dim,
                  slots_first=slots_first, tail=1)
    check_attention(*run_attention(ops, ctx, c), c)
    check_attention(*run_attention(ops, ctx, c, window=333), c, window=333)
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q_len", [[1, 1], [3, 150]])
def test_in_place_and_on_another_stream(ops, q_len, fp8):
    """`out` may be q; contexts on streams of their own, each with its workspace, may run at the same time."""
    cases = [make_case(ops, q_len, [2000, 700], heads=8, kv_heads=2, dim=128, fp8=fp8, seed=20 + i) for i in range(2)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], []
    kept = []
    for c, stream in zip(cases, streams):
        with torch.cuda.stream(stream):
            ctx = ops.Context()
            ws = torch.empty(ops.paged_attention_workspace_size(ctx, c.q, c.cache, batch=2), dtype=torch.uint8, device="cuda")
            x = c.q.clone()
            for _ in range(5):
                x.copy_(c.q)
                ops.paged_attention(ctx, x, c.cache, c.table, x, ws, q_indptr=c.q_indptr)
            outs.append(x)
            kept += [ctx, ws]
    torch.cuda.synchronize()
    for c, x in zip(cases, outs):
        check_attention(x, None, c)


def test_queries_with_an_outlier_over_an_8_bit_cache(ops, ctx):
    """An element of q is off by 2^-17 of the largest of its row at most."""
    c = make_case(ops, [100], [400], heads=16, kv_heads=2, dim=256, fp8=True, seed=30)
    c.q[..., 7] *= 64.0
    check_attention(*run_attention(ops, ctx, c, sm_scale=0.02), c, scale=0.02, q_off=2.0 ** -17)


def test_a_query_that_is_not_finite(ops, ctx):
    """Its row becomes NaN, the others do not."""
    for fp8 in (False, True):
        for q_len in ([1, 1], [1, 40]):
            c = make_case(ops, q_len, [50, 300], heads=4, kv_heads=2, dim=64, fp8=fp8, seed=31)
            good, _ = run_attention(ops, ctx, c)
            c.q[0, 1, 3] = math.nan
            c.q[1, 2, 5] = math.inf
            out, lse = run_attention(ops, ctx, c)
            assert bool(out[0, 1].isnan().all()) and bool(out[1, 2].isnan().all())
            assert bool(lse[0, 1].isnan()) and bool(lse[1, 2].isnan()) and int(lse[: c.rows].isnan().sum()) == 2
            out[0, 1], out[1, 2] = good[0, 1], good[1, 2]
            assert torch.equal(out, good)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q_len", [[1] * 9, [5, 0, 130, 1, 2, 64, 3, 1, 9]])
@pytest.mark.parametrize("said", [384, 100])
def test_short_contexts_are_not_cut(ops, ctx, said, q_len, fp8):
    """Contexts that the caller calls short, whether they are or not."""
    kv = [0, 1, 384, 383, 65, 64, 3, 200, 385]
    c = make_case(ops, q_len, [max(a, b) for a, b in zip(q_len, kv)] if max(q_len) > 1 else kv, heads=8, kv_heads=2, dim=128,
                  fp8=fp8, seed=40)
    check_attention(*run_attention(ops, ctx, c, max_kv_len=said), c)
    check_attention(*run_attention(ops, ctx, c), c)


def test_many_sequences_in_one_call(ops, ctx):
    """As many sequences as a call takes, several items to a block."""
    kv = [(41 * i) % 70 for i in range(4096)]
    c = make_case(ops, [1] * len(kv), kv, heads=2, kv_heads=1, dim=64, page=64, seed=41)
    check_attention(*run_attention(ops, ctx, c, decode=True, max_kv_len=70), c)
    check_attention(*run_attention(ops, ctx, c, decode=True), c)


@pytest.mark.parametrize("fp8", [False, True])
def test_pages_more_than_32_bits_apart(ops, ctx, fp8):
    """Pages 3 GiB apart, scales 1 GiB: written, attended over by both kernels, and read back."""
    q_len, kv_len, heads, kv_heads, dim, page = [70, 1], [300, 64], 8, 2, 128, 128
    c = make_case(ops, q_len, kv_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8, seed=50)
    pages = c.cache.k.shape[0]
    room = torch.empty(pages * (3 << 30), dtype=torch.uint8, device="cuda")
    room_scales = torch.empty(pages * (1 << 28), dtype=torch.float32, device="cuda") if fp8 else None

    def far(pool, at):
        size = pool.element_size()
        flat = room.view(pool.dtype) if size == 1 else room.view(torch.bfloat16)
        return flat.as_strided(pool.shape, ((3 << 30) // size, page * dim, dim, 1), at * kv_heads * page * dim)

    def far_scales(at):
        return room_scales.as_strided((pages, kv_heads, page), (1 << 28, page, 1), at * kv_heads * page)

    near = c.cache
    c.cache = ops.PagedKvCache(far(near.k, 0), far(near.v, 1), *([far_scales(0), far_scales(1)] if fp8 else ()))
    for a, b in ((c.cache.k, near.k), (c.cache.v, near.v)):
        a.view(torch.uint8).copy_(b.view(torch.uint8)) if fp8 else a.copy_(b)
    if fp8:
        c.cache.k_scale.copy_(near.k_scale), c.cache.v_scale.copy_(near.v_scale)
    check_attention(*run_attention(ops, ctx, c), c)
    rows = sum(kv_len)
    out = [torch.zeros((rows, kv_heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    indptr = ints([0, kv_len[0], rows])
    ops.kv_gather(ctx, c.cache, c.table, indptr, *out)
    for got, want in zip(out, (c.keys, c.values)):
        assert torch.equal(got, torch.cat(want).to(torch.bfloat16))
    c.cache.k.view(torch.uint8).zero_(), c.cache.v.view(torch.uint8).zero_()
    ops.kv_append(ctx, c.cache, c.table, *out, q_indptr=indptr)
    again = [torch.zeros_like(x) for x in out]
    ops.kv_gather(ctx, c.cache, c.table, indptr, *again)
    for got, want in zip(again, out):   # (e4m3: once more rounded, by half a step of 2^-3 and of the bf16 result)
        assert bool(((got.float() - want.float()).abs() <= (want.float().abs() * (2.0 ** -4 + 2.0 ** -8)
                                                             + want.float().abs().amax(-1, keepdim=True) * 2.0 ** -18
                                                             if fp8 else 0)).all())
    small = make_case(ops, [1, 1], kv_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seed=51)
    c.q, c.q_len, c.rows, c.q_indptr = small.q, [1, 1], 2, small.q_indptr
    c.keys, c.values = ([torch.split(x.double(), kv_len) for x in again][i] for i in range(2))
    if not fp8:
        check_attention(*run_attention(ops, ctx, c, decode=True), c)
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,heads", [(64, 8), (256, 4)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("said", [1, 384, 3000])
def test_bounds_that_the_caller_says_too_small(ops, ctx, said, window, dim, heads, fp8):
    """`max_kv_len` and `max_q_len` below the lengths there are: other kernels, the same results up to rounding."""
    for q_len in ([1, 1, 1], [300, 1, 20]):
        c = make_case(ops, q_len, [4000, 200, 20], heads=heads, kv_heads=2, dim=dim, fp8=fp8, seed=80)
        for most in (1, 4, 1000):
            check_attention(*run_attention(ops, ctx, c, max_kv_len=said, max_q_len=most, window=window), c, window=window)


def test_single_tokens_over_far_8_bit_pages(ops, ctx):
    """The streaming kernel over e4m3 pages 3 GiB apart with scales 1 GiB apart, against the codes and scales that lie there."""
    kv_len, heads, kv_heads, dim, page = [300, 64, 1], 8, 2, 128, 128
    c = make_case(ops, [1, 1, 1], kv_len, heads=heads, kv_heads=kv_heads, dim=dim, page=page, fp8=True, seed=52)
    near, pages = c.cache, c.cache.k.shape[0]
    room = torch.empty(pages * (3 << 30), dtype=torch.uint8, device="cuda")
    room_scales = torch.empty(pages * (1 << 28), dtype=torch.float32, device="cuda")
    far = lambda at: room.view(near.k.dtype).as_strided(near.k.shape, (3 << 30, page * dim, dim, 1), at * kv_heads * page * dim)
    far_scales = lambda at: room_scales.as_strided((pages, kv_heads, page), (1 << 28, page, 1), at * kv_heads * page)
    c.cache = ops.PagedKvCache(far(0), far(1), far_scales(0), far_scales(1))
    for a, b in ((c.cache.k, near.k), (c.cache.v, near.v)):
        a.view(torch.uint8).copy_(b.view(torch.uint8))
    c.cache.k_scale.copy_(near.k_scale), c.cache.v_scale.copy_(near.v_scale)
    for attempt in (dict(decode=True), dict()):
        check_attention(*run_attention(ops, ctx, c, max_q_len=1, **attempt), c)
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 8, 2), (256, 4, 1)])
@pytest.mark.parametrize("q_len,rooms,said", [
    ([400, 3, 2], [304, 64, 48], [500, 64, 1000000]),
    ([1, 1, 1], [9008, 64, 48], [9500, 70, (1 << 31) - 1]),
])
@pytest.mark.parametrize("kw", [dict(), dict(window=250), dict(causal=False)])
def test_lengths_beyond_the_pages(ops, ctx, kw, q_len, rooms, said, dim, heads, kv_heads, fp8):
    """Rows stay at the positions that the length gives them, and see of the keys before them those that are there."""
    c = make_case(ops, q_len, rooms, heads=heads, kv_heads=kv_heads, dim=dim, fp8=fp8, seed=60 + dim, tail=1)
    c.table.kv_len.copy_(ints(said))
    check_attention(*run_attention(ops, ctx, c, **kw), c, said=said, **kw)
    if max(q_len) == 1:
        check_attention(*run_attention(ops, ctx, c, decode=True, **kw), c, said=said, **kw)
    assert ctx.read_device_error() == 0x5d000001


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("q_len,kv_len", [([1, 1], [1, 90]), ([40, 1], [40, 2]), ([1, 1], [9000, 3]), ([30, 1], [6000, 3])])
def test_scores_that_are_all_infinite(ops, ctx, q_len, kv_len, sign, dim, fp8):
    """A query element of infinity over keys of one sign there: every score is an infinity of that sign, and no softmax exists."""
    c = make_case(ops, q_len, kv_len, heads=4, kv_heads=2, dim=dim, fp8=fp8, seed=70)
    good, good_lse = run_attention(ops, ctx, c)
    pages = c.table.kv_indices.long()
    if fp8:
        c.cache.k.view(torch.uint8)[pages, ..., 5] = 0xb8 if sign < 0 else 0x38
    else:
        c.cache.k[pages, ..., 5] = sign
    c.q[..., 5] = 0.0
    good, good_lse = run_attention(ops, ctx, c)
    assert bool(torch.isfinite(good).all()) and bool(torch.isfinite(good_lse).all())
    row = q_len[0] - 1
    c.q[row, 1, 5] = math.inf
    out, lse = run_attention(ops, ctx, c)
    assert bool(out[row, 1].isnan().all()) and bool(lse[row, 1].isnan())
    out[row, 1], lse[row, 1] = good[row, 1], good_lse[row, 1]
    assert torch.equal(out, good) and torch.equal(lse, good_lse)


@pytest.mark.parametrize("fp8", [False, True])
def test_keys_of_minus_infinity_alone(ops, ctx, fp8):
    """Rows that see keys but no finite score are NaN, rows that see no key 0 and -infinity, in one call."""
    for q_len, kv_len in (([1, 1, 1], [3, 70, 0]), ([2, 40, 20], [3, 70, 9])):
        c = make_case(ops, q_len, kv_len, heads=4, kv_heads=2, dim=64, fp8=fp8, seed=71)
        c.q.abs_()
        page = int(c.table.kv_indices[0])
        if fp8:
            c.cache.k.view(torch.uint8)[page] = 0xb8
            c.cache.k_scale[page] = math.inf
        else:
            c.cache.k[page] = -math.inf
        out, lse = run_attention(ops, ctx, c)
        row = 0
        for b, n in enumerate(q_len):
            for i in range(n):
                o, l = out[row + i].float(), lse[row + i]
                if b == 0:
                    assert bool(o.isnan().all()) and bool(l.isnan().all())
                elif kv_len[b] - n + i < 0:
                    assert bool((o == 0).all()) and bool((l == -math.inf).all())
                else:
                    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(l).all())
            row += n
