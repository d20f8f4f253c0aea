"""Small paged caches with everything around them that must not matter (spare pages, stale slots, rows behind the last
sequence), and the operators over them in 64 bits, with the bounds their results are held to."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

FP8 = torch.float8_e4m3fn


@dataclass
class Case:
    q_len: list
    kv_len: list
    page: int
    heads: int
    kv_heads: int
    dim: int
    table: object
    cache: object
    q_indptr: torch.Tensor
    keys: list      # of every sequence, f64 [kv_len, kv_heads, dim], as the cache stands for them
    values: list
    q: torch.Tensor
    rows: int       # of the sequences; q has `tail` more


def running(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def make_case(ops, q_len, kv_len, *, heads, kv_heads, dim, page=16, fp8=False, seed=0, tail=0, slots_first=False, stale=math.nan,
              q_pad=0):
    """`slots_first`: pool laid out [pages, page, kv_heads, dim]. `stale`: what unused slots and pages hold."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda")
    need = [-(-n // page) for n in kv_len]
    pages = sum(need) + 2
    shape = (pages, page, kv_heads, dim) if slots_first else (pages, kv_heads, page, dim)
    view = (lambda t: t.transpose(1, 2)) if slots_first else (lambda t: t)
    ids = torch.randperm(pages, generator=gen, device="cuda")[: max(1, sum(need))].to(torch.int32)
    indptr = running(need)
    pools, scales, truth = [], [], []
    for _ in range(2):
        if fp8:
            pool = view(torch.full(shape, 0x7f, dtype=torch.uint8, device="cuda"))
            scale = view(torch.full(shape[:3], stale, device="cuda"))
        else:
            pool, scale = view(torch.full(shape, stale, dtype=torch.bfloat16, device="cuda")), None
        rows = []
        for b, n in enumerate(kv_len):
            x = normal(n, kv_heads, dim)
            pos = torch.arange(n, device="cuda")
            at = ids.long()[indptr[b] + pos // page], pos % page
            if fp8:
                codes = (x * 100).clamp(-448, 448).to(FP8)
                unit = torch.rand((n, kv_heads), generator=gen, device="cuda") * 0.02 + 0.001
                pool[at[0], :, at[1]] = codes.view(torch.uint8)
                scale[at[0], :, at[1]] = unit
                rows.append(codes.double() * unit.double()[..., None])
            else:
                pool[at[0], :, at[1]] = x.to(torch.bfloat16)
                rows.append(x.to(torch.bfloat16).double())
        pools.append(pool.view(FP8) if fp8 else pool)
        scales.append(scale)
        truth.append(rows)
    total = sum(q_len) + tail
    q = normal(total, heads, dim + q_pad).to(torch.bfloat16)[..., :dim]
    return Case(q_len, kv_len, page, heads, kv_heads, dim, ops.PageTable(ints(indptr), ids, ints(kv_len)),
                ops.PagedKvCache(*pools, *scales), ints(running(q_len)), truth[0], truth[1], q, sum(q_len))


def attention_reference(c: Case, *, causal=True, window=0, scale=None, q_off=0.0, said=None):
    """out, lse in 64 bits, and the most that each may be off. `said`: the lengths that the page table gives, where they are more
    than the pages hold; kv_len counts the tokens there are.

    A kernel computes scores in 32 bits (each product's sum off by at most (D + 8) 2^-24 of the sum of the magnitudes, the
    weights by e to that, and by a few units of 2^-22 for the exponential), rounds the weights to bf16 (2^-8 of each, half a
    step) and the result once more. `q_off`: what an element of q may be off besides, of the largest of its row."""
    scale = c.dim ** -0.5 if scale is None else scale
    group = c.heads // c.kv_heads
    out = torch.zeros((c.rows, c.heads, c.dim), dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    lse = torch.full((c.rows, c.heads), -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    row = 0
    for b, (n, length) in enumerate(zip(c.q_len, c.kv_len)):
        last = length if said is None else said[b]
        pos = torch.arange(last - n, last, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        seen = (j <= pos) if causal else (j >= 0).expand(n, length)
        if window:
            seen = seen & (j > pos - window)
        for h in range(c.heads):
            if n == 0 or length == 0:
                continue
            q, k, v = c.q[row: row + n, h].double(), c.keys[b][:, h // group], c.values[b][:, h // group]
            s = torch.where(seen, q @ k.T * scale, -math.inf)
            off = ((c.dim + 8) * 2.0 ** -24 * scale * (q.abs() @ k.abs().T).masked_fill(~seen, 0)).amax(1, keepdim=True) + 2.0 ** -20
            off = off + q_off * scale * q.abs().amax(1, keepdim=True) * torch.where(seen, k.abs().sum(1)[None], 0.0).amax(1, keepdim=True)
            some = seen.any(1, keepdim=True)
            w = torch.where(some, torch.softmax(torch.where(some, s, 0.0), dim=1), 0.0)
            o = w @ v
            out[row: row + n, h] = o
            bound[row: row + n, h] = 2.0 ** -8 * o.abs() + (2.0 ** -8 * 1.01 + 2.02 * off) * (w @ v.abs()) + 1e-30
            lse[row: row + n, h] = torch.where(some, torch.logsumexp(torch.where(some, s, 0.0), dim=1, keepdim=True), -math.inf)[:, 0]
            lse_bound[row: row + n, h] = off[:, 0] + 2.0 ** -22 * (lse[row: row + n, h].abs().nan_to_num(0, 0, 0) + 1)
        row += n
    return out, lse, bound, lse_bound


def check_attention(got, lse, c: Case, **kw):
    out, want_lse, bound, lse_bound = attention_reference(c, **kw)
    off = (got[: c.rows].double() - out).abs()
    assert bool((off <= bound).all()), f"out is {float((off / bound).max()):.3g} times its bound off"
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(lse[: c.rows] == -math.inf, empty)
        off = torch.where(empty, 0.0, (lse[: c.rows].double() - want_lse).abs())
        assert bool((off <= lse_bound).all()), f"lse is {float((off / lse_bound).nan_to_num().max()):.3g} times its bound off"


def run_attention(ops, ctx, c: Case, *, decode=False, lse=True, ws=None, out=None, **kw):
    """out and lse, with sentinels in the rows behind the last sequence checked."""
    out = torch.full((c.q.shape[0], c.heads, c.dim), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    l = torch.full((c.q.shape[0], c.heads), 7.0, device="cuda") if lse else None
    if ws is None:
        ws = torch.empty(ops.paged_attention_workspace_size(ctx, c.q, c.cache, batch=len(c.kv_len)), dtype=torch.uint8, device="cuda")
    ops.paged_attention(ctx, c.q, c.cache, c.table, out, ws, q_indptr=None if decode else c.q_indptr, lse=l, **kw)
    torch.cuda.synchronize()
    assert bool((out[c.rows:] == 7.0).all()) and (l is None or bool((l[c.rows:] == 7.0).all()))
    return out, l
