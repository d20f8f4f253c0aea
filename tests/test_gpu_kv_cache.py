"""Rotary positions and the paged cache as it is written and read back, against the formulas in 64 bits."""
import math

import pytest
import torch

from paged_helpers import FP8, check_attention, ints, make_case, run_attention, running

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from qs3_b200 import ops as m
    return m


@pytest.fixture(scope="module")
def ctx(ops):
    return ops.Context()


def turn(x, positions, freq, scale, interleaved):
    """x [tokens, heads, dim] turned, in 64 bits."""
    r = 2 * freq.numel()
    angle = positions.double()[:, None, None] * freq.double()
    c, s = angle.cos() * scale, angle.sin() * scale
    x = x.double().clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2: r])
    a0, b0 = a.clone(), b.clone()
    a.copy_(a0 * c - b0 * s)
    b.copy_(b0 * c + a0 * s)
    return x


def turn_bound(x, want, r, scale, half_step):
    """Sine and cosine are within 4 units of 2^-24, a product and the sum add one each: 2^-21 of |x| + |y| (both of a pair are
    below the row's largest); then the rounding to the tensor's type."""
    most = x.double().abs().amax(-1, keepdim=True)
    return half_step * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -21 * 2 * abs(scale) * most + 1e-38


FORMS = [("q only, in place", False, False), ("q and k, in place", True, False), ("q and k, out of place", True, True)]


@pytest.mark.parametrize("name,with_k,out_of_place", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (128, 128), (128, 6), (256, 64), (96, 96), (8, 2), (80, 24), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(ops, ctx, dtype, dim, rotary, interleaved, name, with_k, out_of_place):
    gen = torch.Generator(device="cuda").manual_seed(dim + rotary)
    tokens, heads, kv_heads = 37, 5, 2
    q, k = (torch.randn((tokens, h, dim), generator=gen, device="cuda").to(dtype) for h in (heads, kv_heads))
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen, device="cuda")
    positions[0], positions[1] = 0, -5
    f = ops.rope_frequencies(rotary, 10000.0)
    outs = [torch.full_like(x, 7.0) for x in (q, k)] if out_of_place else [q.clone(), k.clone()]
    src = [q, k] if out_of_place else outs
    ops.rope(ctx, positions if dim != 128 else positions.int(), f.inv_freq, src[0], src[1] if with_k else None,
             q_out=outs[0] if out_of_place else None, k_out=outs[1] if out_of_place else None, scale=1.25, interleaved=interleaved)
    torch.cuda.synchronize()
    for x, got in list(zip((q, k), outs))[: 2 if with_k else 1]:
        want = turn(x, positions, f.inv_freq, 1.25, interleaved)
        off = (got.double() - want).abs()
        assert bool((off <= turn_bound(x, want, rotary, 1.25, torch.finfo(dtype).eps / 2)).all())
        assert torch.equal(got[..., rotary:], x[..., rotary:])
    if not with_k and not out_of_place:
        assert torch.equal(outs[1], k)


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 64), (1000, 3), (3, 300)])
def test_rope_sizes_and_views(ops, ctx, tokens, heads):
    """q and k as parts of one projection's output, in place and into parts of another buffer."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    qkv = torch.randn((tokens, heads + 4, 64), generator=gen, device="cuda").to(torch.bfloat16)
    before = qkv.clone()
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) * 1000
    f = ops.rope_frequencies(32, 500000.0)
    ops.rope(ctx, positions, f.inv_freq, qkv[:, :heads], qkv[:, heads: heads + 2])
    want = turn(before[:, : heads + 2], positions, f.inv_freq, 1.0, False)
    torch.cuda.synchronize()
    off = (qkv[:, : heads + 2].double() - want).abs()
    assert bool((off <= turn_bound(before[:, : heads + 2], want, 32, 1.0, 2.0 ** -8)).all())
    assert torch.equal(qkv[:, heads + 2:], before[:, heads + 2:])
    # from one part of a buffer into another part of it
    ops.rope(ctx, positions, f.inv_freq, qkv[:, :1], q_out=qkv[:, heads + 3:])
    torch.cuda.synchronize()
    again = turn(want[:, :1].to(torch.bfloat16), positions, f.inv_freq, 1.0, False)
    assert float((qkv[:, heads + 3:].double() - again).abs().max()) < 0.2


def test_scaled_frequencies_follow_their_definitions(ops):
    base = [10000.0 ** (-2 * j / 64) for j in range(32)]
    get = lambda **kw: ops.rope_frequencies(64, 10000.0, **kw)
    assert torch.allclose(get().inv_freq.cpu(), torch.tensor(base, dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(get(scaling="linear", factor=4.0).inv_freq.cpu(), torch.tensor(base, dtype=torch.float64) / 4, rtol=1e-14)
    ntk = get(scaling="ntk", factor=4.0).inv_freq.cpu()
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], base[-1] / 4, rel_tol=1e-12)
    for kind in ("yarn", "llama3"):
        f = get(scaling=kind, factor=8.0, original_length=4096).inv_freq.cpu()
        assert f[0] == base[0] and math.isclose(f[-1], base[-1] / 8, rel_tol=1e-12)
        assert bool((f[1:] < f[:-1]).all())
    assert math.isclose(get(scaling="yarn", factor=8.0).scale, 0.1 * math.log(8.0) + 1)
    for bad in (dict(scaling="other"), dict(factor=0.0)):
        with pytest.raises(ops.Qs3Error):
            get(**bad)


def empty_cache(ops, q_len, kv_len, *, kv_heads, dim, page, fp8, seed, slots_first=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in kv_len]
    pages = sum(need) + 2
    cache = ops.PagedKvCache.empty(pages, *((page, kv_heads) if slots_first else (kv_heads, page)), dim, fp8=fp8)
    if slots_first:
        t = lambda x: None if x is None else x.transpose(1, 2)
        cache = ops.PagedKvCache(t(cache.k), t(cache.v), t(cache.k_scale), t(cache.v_scale))
    for x in (cache.k, cache.v):
        (x.view(torch.uint8) if fp8 else x).fill_(0x33 if fp8 else 7.0)
    for x in (cache.k_scale, cache.v_scale) if fp8 else ():
        x.fill_(7.0)
    ids = torch.randperm(pages, generator=gen, device="cuda")[: max(1, sum(need))].to(torch.int32)
    return cache, ops.PageTable(ints(running(need)), ids, ints(kv_len)), running(need)


def raw(cache):
    return [x.view(torch.uint8) if x.element_size() == 1 else x for x in (cache.k, cache.v)] + (
        [cache.k_scale, cache.v_scale] if cache.fp8 else [])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,page,slots_first", [(64, 16, False), (128, 24, True), (256, 1, False), (96, 16, False), (16, 5, True)])
@pytest.mark.parametrize("rotary,interleaved,own_positions", [(0, False, False), (16, False, False), (12, False, True), (10, True, False)])
@pytest.mark.parametrize("q_len,kv_len", [([1, 1, 1], [5, 1, 40]), ([0, 3, 17, 0, 4], [4, 3, 40, 0, 2]), ([70], [75])])
def test_append(ops, ctx, q_len, kv_len, fp8, dim, page, slots_first, rotary, interleaved, own_positions):
    gen = torch.Generator(device="cuda").manual_seed(dim + page)
    kv_heads, heads = 3, 5
    cache, table, indptr = empty_cache(ops, q_len, kv_len, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8, seed=dim, slots_first=slots_first)
    before = [x.clone() for x in raw(cache)]
    decode = all(n == 1 for n in q_len)
    rows = sum(q_len)
    qkv = torch.randn((rows + 2, heads + 2 * kv_heads, dim), generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    q_out = torch.full((rows + 2, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    kw = {}
    positions = torch.randint(0, 100000, (rows + 2,), generator=gen, device="cuda") if own_positions else None
    if rotary:
        f = ops.rope_frequencies(rotary)
        kw = dict(q=q, q_out=q_out, inv_freq=f.inv_freq, rope_scale=1.5, interleaved=interleaved, positions=positions)
    ops.kv_append(ctx, cache, table, k, v, q_indptr=None if decode else ints(running(q_len)), **kw)
    torch.cuda.synchronize()
    assert ctx.read_device_error() == 0
    after = raw(cache)
    touched = torch.zeros((before[0].shape[0], kv_heads, page), dtype=torch.bool, device="cuda")
    row = 0
    for b, (n, length) in enumerate(zip(q_len, kv_len)):
        for i in range(n):
            pos, r = length - n + i, row + i
            if pos < 0:
                assert bool((q_out[r] == 7.0).all())
                continue
            at = (int(table.kv_indices[indptr[b] + pos // page]), slice(None), pos % page)
            touched[at] = True
            angle = positions[r: r + 1] if own_positions else torch.tensor([pos], device="cuda")
            for x, pool, side in ((k[r: r + 1], cache.k, 0), (v[r: r + 1], cache.v, 1)):
                want = turn(x, angle, f.inv_freq, 1.5, interleaved) if rotary and side == 0 else x.double()
                slack = turn_bound(x, want, rotary, 1.5, 0.0) if rotary and side == 0 else torch.zeros_like(want)
                if fp8:
                    scale = (cache.k_scale, cache.v_scale)[side][at]
                    ideal = want[0].abs().amax(-1) / 448
                    assert bool(((scale.double() - ideal).abs() <= 2.0 ** -22 * ideal + slack[0].amax(-1) / 448).all())
                    got = pool[at].double() * scale.double()[:, None]
                    # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale among the subnormals
                    bound = (2.0 ** -4 * want[0].abs()).clamp(min=2.0 ** -10 * ideal[:, None]) * (1 + 2.0 ** -20) + 2 * slack[0]
                else:
                    got = pool[at].double()
                    bound = 2.0 ** -8 * want[0].abs() + slack[0] * 1.01 + 1e-38
                assert bool(((got - want[0]).abs() <= bound).all())
            if rotary:
                want = turn(q[r: r + 1], angle, f.inv_freq, 1.5, interleaved)
                assert bool(((q_out[r].double() - want[0]).abs() <= turn_bound(q[r: r + 1], want, rotary, 1.5, 2.0 ** -8)[0]).all())
        row += n
    if rotary:
        assert bool((q_out[rows:] == 7.0).all())
    for a, b in zip(before, after):     # nothing else was written
        assert torch.equal(a[~touched], b[~touched])


def test_append_of_what_cannot_be_scaled(ops, ctx):
    """Zeros, the smallest and largest values; a row with an infinity or NaN reads back as NaN, its neighbours do not."""
    cache, table, _ = empty_cache(ops, [6], [6], kv_heads=2, dim=64, page=16, fp8=True, seed=1)
    k = torch.zeros((6, 2, 64), dtype=torch.bfloat16, device="cuda")
    k[1] = 3.0e38
    k[2] = 1.0e-38
    k[3, 0, 5] = math.inf
    k[4, 1, 7] = math.nan
    k[5] = -1.0
    ops.kv_append(ctx, cache, table, k, k, q_indptr=ints([0, 6]))
    out = torch.zeros_like(k)
    v_out = torch.zeros_like(k)
    ops.kv_gather(ctx, cache, table, ints([0, 6]), out, v_out)
    torch.cuda.synchronize()
    assert bool((out[0] == 0).all()) and bool((out[1] == k[1]).all()) and bool((out[5] == -1.0).all())
    assert bool((out[2].abs() <= 2e-38).all())
    assert bool(out[3, 0].isnan().all()) and bool((out[3, 1] == 0).all())
    assert bool(out[4, 1].isnan().all()) and bool((out[4, 0] == 0).all())
    assert torch.equal(out.nan_to_num(9), v_out.nan_to_num(9))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,page,slots_first", [(64, 16, False), (128, 24, True), (256, 3, False), (96, 16, False), (16, 1, True)])
def test_gather(ops, ctx, fp8, dim, page, slots_first):
    kv = [0, 5, 300, 17, 0, 64]
    c = make_case(ops, [0] * len(kv), kv, heads=2, kv_heads=2, dim=dim, page=page, fp8=fp8, seed=dim, slots_first=slots_first, tail=1)
    indptr = ints(running(kv))
    wide = torch.full((sum(kv) + 3, 3, 2, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    k_out, v_out = wide[:, 0], wide[:, 2]
    ops.kv_gather(ctx, c.cache, c.table, indptr, k_out, v_out)
    torch.cuda.synchronize()
    for got, want in ((k_out, c.keys), (v_out, c.values)):
        want = torch.cat(want)
        assert bool(((got[: sum(kv)].double() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -20)).all())
        assert bool((got[sum(kv):] == 7.0).all())
    assert bool((wide[:, 1] == 7.0).all())
    # parts of sequences, some of them beyond the end
    start, take = [0, 2, 290, 20, 0, 1], [2, 3, 20, 4, 0, 5]
    part_k = torch.full((sum(take), 2, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    part_v = torch.full_like(part_k, 7.0)
    ops.kv_gather(ctx, c.cache, c.table, ints(running(take)), part_k, part_v, kv_start=ints(start))
    torch.cuda.synchronize()
    row = 0
    for b in range(len(kv)):
        for i in range(take[b]):
            pos = start[b] + i
            if pos < kv[b]:
                assert torch.equal(part_v[row], v_out[int(indptr[b]) + pos])
            else:
                assert bool((part_k[row] == 7.0).all()) and bool((part_v[row] == 7.0).all())
            row += 1


def test_bad_pages_are_left_alone(ops, ctx):
    cache, table, _ = empty_cache(ops, [1, 1, 1], [20, 40, 40], kv_heads=2, dim=64, page=16, fp8=False, seed=2)
    table.kv_indices[4] = -7           # the second sequence's last page
    table.kv_len[2] = 500              # more than its pages hold: its last token has no place but the last one there is
    k = torch.randn((3, 2, 64), device="cuda").to(torch.bfloat16)
    before = cache.k.clone()
    ops.kv_append(ctx, cache, table, k, k)
    torch.cuda.synchronize()
    assert ctx.read_device_error() == 0x5d000001
    page0 = int(table.kv_indices[1])
    assert torch.equal(cache.k[page0, :, 3], k[0])
    changed = (cache.k != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {page0, int(table.kv_indices[7])}
    out = torch.full((100, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv_gather(ctx, cache, table, ints([0, 20, 60, 100]), out, out.clone())
    torch.cuda.synchronize()
    assert ctx.read_device_error() == 0x5d000001
    assert torch.equal(out[19], k[0]) and bool((out[52:60] == 7.0).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (256, 16, 2)])
def test_steps_of_a_serving_loop(ops, ctx, dim, heads, kv_heads, fp8):
    """Prompts, then single tokens: append with rotation, attention, and the cache read back, step by step, against attention
    over the rows that the cache stands for."""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    page, room = 16, 160
    pages = 3 * room // page
    cache = ops.PagedKvCache.empty(pages, kv_heads, page, dim, fp8=fp8)
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = ops.PageTable(ints([0, 10, 20, 30]), ids, ints([0, 0, 0]))
    f = ops.rope_frequencies(dim // 4, scaling="llama3", factor=8.0)
    lengths = [0, 0, 0]
    for step, q_len in enumerate(([70, 1, 33], [1, 1, 1], [1, 20, 1], [1, 1, 1])):
        lengths = [a + b for a, b in zip(lengths, q_len)]
        table.kv_len.copy_(ints(lengths))
        qkv = torch.randn((sum(q_len), heads + 2 * kv_heads, dim), generator=gen, device="cuda").to(torch.bfloat16)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
        indptr = ints(running(q_len))
        ops.kv_append(ctx, cache, table, k, v, q_indptr=indptr, q=q, inv_freq=f.inv_freq)   # q in place
        out_indptr = running(lengths)
        k_rows, v_rows = (torch.empty((sum(lengths), kv_heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.kv_gather(ctx, cache, table, ints(out_indptr), k_rows, v_rows)
        from paged_helpers import Case
        truth = []
        for pool, scale, rows in ((cache.k, cache.k_scale, k_rows), (cache.v, cache.v_scale, v_rows)):
            seqs = []
            for b, n in enumerate(lengths):
                own = ids.long()[b * 10: b * 10 + -(-n // page)]
                x = pool[own].double() if scale is None else pool[own].double() * scale[own].double()[..., None]
                seqs.append(x.transpose(1, 2).flatten(0, 1)[:n])
            truth.append(seqs)
            whole = torch.cat(seqs)
            assert bool(((rows.double() - whole).abs() <= 2.0 ** -8 * whole.abs() * (1 + 2.0 ** -20)).all())
        c = Case(q_len, lengths, page, heads, kv_heads, dim, table, cache, indptr, truth[0], truth[1], q, sum(q_len))
        check_attention(*run_attention(ops, ctx, c), c)
    assert ctx.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q_len", [[1, 1, 1], [2, 30, 40]])
def test_tokens_beyond_the_pages_have_no_place(ops, ctx, q_len, fp8):
    """New tokens keep their positions where a length says more than the pages hold: those beyond drop out, and nothing else moves."""
    said, rooms, kv_heads, heads, dim, page = [20, 60, 500], [32, 48, 48], 2, 4, 64, 16
    cache, table, indptr = empty_cache(ops, q_len, rooms, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8, seed=3)
    table.kv_len.copy_(ints(said))
    roomy, wide, wide_indptr = empty_cache(ops, q_len, said, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8, seed=4)
    before = [x.clone() for x in raw(cache)]
    rows = sum(q_len)
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn((rows, h, dim), generator=gen, device="cuda").to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    f = ops.rope_frequencies(16)
    outs = [torch.full_like(q, 7.0) for _ in range(2)]
    for c, t, out in ((roomy, wide, outs[0]), (cache, table, outs[1])):
        assert ctx.read_device_error() == 0
        ops.kv_append(ctx, c, t, k, v, q_indptr=None if max(q_len) == 1 else ints(running(q_len)), q=q, q_out=out, inv_freq=f.inv_freq)
    torch.cuda.synchronize()
    assert ctx.read_device_error() == 0x5d000001
    touched = torch.zeros((before[0].shape[0], kv_heads, page), dtype=torch.bool, device="cuda")
    row = 0
    for b, n in enumerate(q_len):
        for i in range(n):
            pos, r = said[b] - n + i, row + i
            if pos >= rooms[b]:
                assert bool((outs[1][r] == 7.0).all())
                continue
            assert torch.equal(outs[1][r], outs[0][r])
            at = (int(table.kv_indices[indptr[b] + pos // page]), slice(None), pos % page)
            there = (int(wide.kv_indices[wide_indptr[b] + pos // page]), slice(None), pos % page)
            touched[at] = True
            for x, y in zip(raw(cache), raw(roomy)):
                assert torch.equal(x[at], y[there])
        row += n
    for a, b in zip(before, raw(cache)):
        assert torch.equal(a[~touched], b[~touched])


@pytest.mark.parametrize("tokens", [1, 7, 300])
def test_parts_between_each_other(ops, ctx, tokens):
    """Outputs that lie between other operands without sharing memory, and one token's rows in place under another token stride."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    wide = torch.randn((tokens, 2, 6, 64), generator=gen, device="cuda").to(torch.bfloat16)
    before, f = wide.clone(), ops.rope_frequencies(64)
    positions = torch.arange(tokens, device="cuda")
    # q, q_out, k and k_out: heads of one buffer in turn
    q, q_out, k, k_out = wide[:, 0, 0::2], wide[:, 0, 1::2], wide[:, 1, 0::2], wide[:, 1, 1::2]
    ops.rope(ctx, positions, f.inv_freq, q, k, q_out=q_out, k_out=k_out)
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :, 0::2], before[:, :, 0::2])
    for x, got in ((before[:, 0, 0::2], q_out), (before[:, 1, 0::2], k_out)):
        want = turn(x, positions, f.inv_freq, 1.0, False)
        assert bool(((got.double() - want).abs() <= turn_bound(x, want, 64, 1.0, 2.0 ** -8)).all())
    # K and V of a token side by side in every head
    c = make_case(ops, [0], [tokens], heads=2, kv_heads=2, dim=64, seed=tokens, tail=1)
    both = torch.zeros((tokens, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    ops.kv_gather(ctx, c.cache, c.table, ints([0, tokens]), both[:, :, 0], both[:, :, 1])
    torch.cuda.synchronize()
    assert torch.equal(both[:, :, 0].double(), c.keys[0]) and torch.equal(both[:, :, 1].double(), c.values[0])
    if tokens == 1:
        x = before[:, 0, :2].clone()
        want = turn(x, positions + 5, f.inv_freq, 1.0, False)
        ops.rope(ctx, positions + 5, f.inv_freq, x, q_out=x.as_strided(x.shape, (1024, 64, 1)))
        torch.cuda.synchronize()
        assert bool(((x.double() - want).abs() <= turn_bound(before[:, 0, :2], want, 64, 1.0, 2.0 ** -8)).all())


def test_positions_in_pinned_memory(ops, ctx):
    """Host memory that the device addresses stands for device memory; other host memory is refused."""
    q = torch.randn((5, 2, 64), device="cuda").to(torch.bfloat16)
    f, positions = ops.rope_frequencies(64), torch.arange(5)
    got, want = torch.empty_like(q), torch.empty_like(q)
    ops.rope(ctx, positions.pin_memory(), f.inv_freq, q, q_out=got)
    ops.rope(ctx, positions.cuda(), f.inv_freq, q, q_out=want)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(ops.Qs3Error, match="on cuda:0"):
        ops.rope(ctx, positions, f.inv_freq, q, q_out=got)
