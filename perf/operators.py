"""Performance cases of the gated-attention path between its projections and its output: rotary positions, the paged
KV cache as it is written and read back, and attention of new tokens over it.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges. ``prepare`` makes what a serving
loop has in hand before the call (projected q, k and v, page pool, page table, rotary frequencies), ``run`` is one pass,
``work`` the bytes and operations the pass cannot do without, ``exact`` the pass in 64 bits.

Kinds of pass:

* ``attention``  new tokens (one per sequence, or a ragged batch of chunks) over the paged cache, with the log-sum-exp
                 of every row: ``ops.paged_attention``;
* ``rope``       rotary positions on q and k out of place: ``ops.rope``;
* ``append``     k and v of the new tokens into the cache, q and k rotated on the way: ``ops.kv_append``;
* ``gather``     the cache of every sequence read back as contiguous bf16 rows: ``ops.kv_gather``.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

FP8_MAX = 448.0
FP8_TINY = 1e-30


def listed():
    return [
        # the smallest hybrid configuration: eight sequences, one new token each; launches decide
        dict(name="attention_tiny_8", kind="attention", batch=8, old_lo=20, old_hi=25, heads=4, kv_heads=2, dim=64, page=16,
             fp8=False, chunk=False, q_lo=1, q_hi=1, window=0, idle=0, tail=0, lens=1),
        # one long conversation: two KV heads for the whole GPU, the context is split
        dict(name="attention_decode_1_long", kind="attention", batch=1, old_lo=65573, old_hi=65573, heads=16, kv_heads=2,
             dim=256, page=16, fp8=False, chunk=False, q_lo=1, q_hi=1, window=0, idle=0, tail=0, lens=2),
        # the hybrid decode loop's batch in the middle of its 256 generated tokens
        dict(name="attention_decode_128", kind="attention", batch=128, old_lo=4096, old_hi=4351, heads=16, kv_heads=2, dim=256,
             page=16, fp8=False, chunk=False, q_lo=1, q_hi=1, window=0, idle=0, tail=0, lens=3),
        # a serving batch of very different contexts over a quantised cache, with two idle slots
        dict(name="attention_decode_fp8_66", kind="attention", batch=66, old_lo=0, old_hi=16383, heads=32, kv_heads=8, dim=128,
             page=64, fp8=True, chunk=False, q_lo=1, q_hi=1, window=0, idle=2, tail=0, lens=4),
        # a mixed step of continuous batching: chunks of prompts beside sequences that decode, padded at its end
        dict(name="attention_mixed_12", kind="attention", batch=12, old_lo=0, old_hi=5000, heads=32, kv_heads=8, dim=128, page=16,
             fp8=False, chunk=True, q_lo=1, q_hi=509, window=0, idle=1, tail=7, lens=5),
        # a long prompt in one go
        dict(name="attention_prefill_8192", kind="attention", batch=1, old_lo=0, old_hi=0, heads=16, kv_heads=2, dim=256, page=16,
             fp8=False, chunk=True, q_lo=8192, q_hi=8192, window=0, idle=0, tail=0, lens=6),
        # a chunk at the end of a long document in a quantised cache
        dict(name="attention_chunk_fp8_1021", kind="attention", batch=1, old_lo=31111, old_hi=31111, heads=16, kv_heads=2, dim=256,
             page=64, fp8=True, chunk=True, q_lo=1021, q_hi=1021, window=0, idle=0, tail=0, lens=7),
        # rotary positions of a decode batch on a quarter of the head
        dict(name="rope_decode_128", kind="rope", tokens=128, heads=16, kv_heads=2, dim=256, rotary=64, interleaved=False,
             scaling="none", factor=1.0, far=4352, f32=False),
        # a prompt with the interleaved layout, at positions of a context that was extended
        dict(name="rope_prefill_8190", kind="rope", tokens=8190, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=True,
             scaling="yarn", factor=32.0, far=1048576, f32=False),
        # the hybrid decode loop's batch into a quantised cache
        dict(name="append_decode_fp8_128", kind="append", batch=128, old_lo=900, old_hi=1100, q_lo=1, q_hi=1, heads=16,
             kv_heads=2, dim=256, page=16, fp8=True, chunk=False, rotary=64, interleaved=False, idle=0, tail=0, lens=8),
        # chunks of several prompts into a quantised cache
        dict(name="append_prefill_fp8_9", kind="append", batch=9, old_lo=0, old_hi=700, q_lo=500, q_hi=1900, heads=32,
             kv_heads=8, dim=128, page=64, fp8=True, chunk=True, rotary=128, interleaved=False, idle=1, tail=5, lens=9),
        # a quantised cache read back for a path that wants contiguous rows
        dict(name="gather_fp8_32", kind="gather", batch=32, old_lo=1000, old_hi=4500, kv_heads=8, dim=128, page=64, fp8=True,
             idle=1, lens=10),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["rope", "append", "append", "gather"])
    lens = rng.randrange(1 << 20)
    dim, kv_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8])
    page, fp8 = rng.choice([16, 16, 24, 32, 64, 128]), rng.random() < 0.4
    if kind == "rope":
        dim = rng.choice([64, 96, 128, 256])
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), heads=kv_heads * rng.choice([1, 2, 4, 8]), kv_heads=kv_heads,
                    dim=dim, rotary=rng.choice([16, dim // 4, dim // 2, dim]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn", "llama3"]), factor=float(rng.choice([2, 4, 8, 32])),
                    far=_log_int(rng, 1000, 1 << 20), f32=rng.random() < 0.2)
    if kind == "gather":
        batch = _log_int(rng, 1, 64)
        most = min(16384, (1 << 28) // (batch * kv_heads * dim * 2))
        top = _log_int(rng, 1, most)
        return dict(kind=kind, batch=batch, old_lo=rng.randint(1, top), old_hi=top, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8,
                    idle=rng.choice([0, 0, 1]) if batch > 1 else 0, lens=lens)
    group = rng.choice([1, 2, 4, 5, 8, 16])
    chunk = rng.random() < 0.5
    if kind == "append":
        batch = _log_int(rng, 1, 128)
        top = _log_int(rng, 1, 16384 // batch) if chunk else 1
        old = _log_int(rng, 1, max(2, 2048 // batch))
        return dict(kind=kind, batch=batch, old_lo=0, old_hi=old, q_lo=rng.randint(1, top), q_hi=top, heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, page=page, fp8=fp8, chunk=chunk, rotary=rng.choice([0, dim // 4, dim // 2, dim]),
                    interleaved=rng.random() < 0.5, idle=rng.choice([0, 0, 1]) if batch > 1 else 0,
                    tail=rng.choice([0, 3]) if chunk else 0, lens=lens)
    window = _log_int(rng, 16, 4096) if rng.random() < 0.25 else 0
    if chunk:
        batch = _log_int(rng, 1, 16)
        q_hi = _log_int(rng, 2, 8000 // batch)
        # the scores of the padded batch, held at once by the plain form
        most = int(6e8 / (batch * q_hi * kv_heads * group)) - q_hi
        old = _log_int(rng, 1, max(1, min(32768, most, int(5e8 / (batch * kv_heads * dim * 4)))))
        q_lo = rng.randint(1, q_hi)
    else:
        batch = _log_int(rng, 1, 256)
        old = _log_int(rng, 1, min(65536, int(8e8 / (batch * kv_heads * dim * 4))))
        q_lo = q_hi = 1
    return dict(kind=kind, batch=batch, old_lo=rng.randint(0, old), old_hi=old, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                page=page, fp8=fp8, chunk=chunk, q_lo=q_lo, q_hi=q_hi, window=window, idle=rng.choice([0, 0, 1]) if batch > 1 else 0,
                tail=rng.choice([0, 0, 5]) if chunk else 0, lens=lens)


# ---- the shapes of a case ------------------------------------------------------------------


def _lengths(case):
    """New tokens and length of the cache with them, per sequence. The last `idle` ones are empty slots."""
    rng = random.Random(case["lens"])
    lo, hi = case.get("q_lo", 0), case.get("q_hi", 0)
    q, kv = [], []
    for b in range(case["batch"]):
        if b >= case["batch"] - case["idle"]:
            q.append(1 if hi and not case["chunk"] else 0)   # a decode batch has a row for an idle slot too
            kv.append(0)
            continue
        q.append(_log_int(rng, lo, hi) if hi else 0)
        kv.append(rng.randint(case["old_lo"], case["old_hi"]) + q[-1])
    return q, kv


def _visible(case, q, kv):
    """Pairs of a new token and a cached one that it sees, and cached tokens that any new one sees."""
    w, pairs, keys = case["window"], 0, 0
    for n, length in zip(q, kv):
        if length == 0 or n == 0:
            continue
        first = length - n
        if w == 0 or length <= w:
            pairs += n * first + n * (n + 1) // 2
            keys += length
        else:
            full = sum(min(p + 1, w) for p in range(first, length)) if n < 64 else None
            if full is None:   # positions below w - 1 see all before them, the others w
                below = max(0, min(length, w) - first)
                full = below * first + below * (below + 1) // 2 + (n - below) * w
            pairs += full
            keys += length - max(0, first - w + 1)
    return pairs, keys


def _frequencies(case):
    """Rotary frequencies in radians per position (64 bits) and the factor on cosine and sine."""
    r, base, kind, s = case["rotary"], 10000.0, case.get("scaling", "none"), case.get("factor", 1.0)
    freq, scale = [base ** (-2.0 * j / r) for j in range(r // 2)], 1.0
    if kind == "linear":
        freq = [f / s for f in freq]
    elif kind == "yarn":   # wavelengths below 1/32 of the trained context stay, those above it are divided by s
        trained = 4096
        dim_of = lambda turns: r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), r - 1)
        ramp = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(r // 2)]
        freq = [f / s * t + f * (1 - t) for f, t in zip(freq, ramp)]
        scale = 0.1 * math.log(s) + 1.0
    elif kind == "llama3":
        trained, low, high = 8192, 1.0, 4.0
        smooth = [min(1.0, max(0.0, (trained * f / (2 * math.pi) - low) / (high - low))) for f in freq]
        freq = [f / s * (1 - t) + f * t for f, t in zip(freq, smooth)]
    return freq, scale


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        size = 4 if case["f32"] else 2
        return {"bytes": 2 * n * case["dim"] * size + 8 * case["tokens"] + 4 * case["rotary"], "flops": 3 * n * case["rotary"]}
    q, kv = _lengths(case)
    d, hk, unit = case["dim"], case["kv_heads"], 1 if case["fp8"] else 2
    row = 2 * hk * (d * unit + (4 if case["fp8"] else 0))   # one token of the cache
    table = 4 * sum(-(-n // case["page"]) for n in kv) + 12 * case["batch"]
    if kind == "gather":
        return {"bytes": sum(kv) * (row + 4 * hk * d) + table, "flops": 2 * hk * d * sum(kv)}
    tokens, h = sum(q), case["heads"]
    if kind == "append":
        live = sum(n for n, length in zip(q, kv) if length)
        rotated = 4 * live * h * d if case["rotary"] else 0
        return {"bytes": live * (4 * hk * d + row) + rotated + 12 * case["batch"] + 4 * live, "flops": 8 * live * (h + hk) * d}
    pairs, keys = _visible(case, q, kv)
    return {"bytes": 4 * tokens * h * d + 4 * tokens * h + keys * row + table, "flops": 4 * d * h * pairs}


# ---- what a program has before the call ---------------------------------------------------------


def _pool(case, gen, pages):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen)
    if not case["fp8"]:
        return x, None
    scale = (torch.rand(shape[:3], device="cuda", generator=gen) * 0.4 + 0.8) / 100
    return (x * 100).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.bfloat16: torch.randn(shape, dtype=dtype, device="cuda", generator=gen)
    d, hk = case["dim"], case["kv_heads"]
    s = dict(case=case, heads=case.get("heads", 0))
    if case.get("rotary"):
        freq, s["rope_scale"] = _frequencies(case)
        s["inv_freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
    if case["kind"] == "rope":
        dtype = torch.float32 if case["f32"] else torch.bfloat16
        s["q"], s["k"] = normal(case["tokens"], case["heads"], d, dtype=dtype), normal(case["tokens"], hk, d, dtype=dtype)
        s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), dtype=torch.int64, device="cuda", generator=gen)
        return s
    q, kv = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 3
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    running = lambda v: [sum(v[:i]) for i in range(len(v) + 1)] if len(v) < 512 else torch.tensor([0] + v).cumsum(0).tolist()
    s.update(kv_indptr=ints(running(need)), kv_len=ints(kv), longest=max(kv), q_longest=max(q),
             kv_indices=torch.randperm(pages, device="cuda", generator=gen)[: max(1, sum(need))].to(torch.int32))
    (s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"]) = _pool(case, gen, pages), _pool(case, gen, pages)
    if case["kind"] == "gather":
        s["rows"] = sum(kv)
        s["out_indptr"] = ints(running(kv))
        s["k_out"], s["v_out"] = (torch.zeros((max(1, s["rows"]), hk, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        return s
    tokens, h = sum(q) + case["tail"], case["heads"]
    s["tokens"] = sum(q)
    s["q_indptr"] = ints(running(q))
    s["q_arg"] = s["q_indptr"] if case["chunk"] else None
    if case["kind"] == "append":   # one projection's output holds q, k and v of a token side by side
        s["qkv"] = normal(tokens, h + 2 * hk, d)
        s["q"], s["k"], s["v"] = s["qkv"].split([h, hk, hk], dim=1)
        s["q_out"] = torch.zeros((tokens, h, d), dtype=torch.bfloat16, device="cuda")
    else:
        s["q"] = normal(tokens, h, d) * 2
        s["out"] = torch.zeros((tokens, h, d), dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.zeros((tokens, h), dtype=torch.float32, device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------------------------------


def _turn(x, positions, s):
    """x [tokens, heads, dim] in 32 bits, rotated."""
    half = s["inv_freq"].numel()
    angle = positions.double()[:, None] * s["inv_freq"]
    cos, sin = ((f(angle) * s["rope_scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    if s["case"]["interleaved"]:
        a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half: 2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _rows_of_tokens(s):
    """Sequence of every new token, its position, whether it has one, and its page and slot."""
    rows = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["q_indptr"].long(), rows, right=True) - 1
    fresh = s["q_indptr"].long().diff()
    pos = s["kv_len"].long()[seq] - fresh[seq] + rows - s["q_indptr"].long()[seq]
    live = pos >= 0
    page = s["case"]["page"]
    at = (s["kv_indptr"].long()[seq] + pos.clamp(min=0) // page).clamp(max=s["kv_indices"].numel() - 1)
    return seq, pos, live, s["kv_indices"].long()[at], pos.clamp(min=0) % page


def _padded_cache(s, pool, scale):
    """[batch, kv_heads, longest context in whole pages, dim] in 32 bits, zero behind a sequence's end."""
    page = s["case"]["page"]
    count = -(-s["longest"] // page)
    at = s["kv_indptr"].long()[:-1, None] + torch.arange(count, device="cuda")
    pages = s["kv_indices"].long()[at.clamp(max=s["kv_indices"].numel() - 1)]
    x = pool[pages].float()                                      # [batch, pages, heads, page, dim]
    if scale is not None:
        x = x * scale[pages][..., None]
    x = x.transpose(1, 2).flatten(2, 3)
    there = torch.arange(x.shape[2], device="cuda") < s["kv_len"].long()[:, None]
    return x.masked_fill(~there[:, None, :, None], 0.0)


def _plain_attention(s):
    case = s["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out, lse = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    if s["longest"] == 0:
        lse[: s["tokens"]] = -math.inf
        return out, lse
    seq, pos, _, _, _ = _rows_of_tokens(s)
    rows = torch.arange(s["tokens"], device="cuda")
    within = rows - s["q_indptr"].long()[seq]
    most = s["q_longest"]
    q = torch.zeros((case["batch"], most, h, d), device="cuda")
    q[seq, within] = s["q"][: s["tokens"]].float()
    k, v = _padded_cache(s, s["k_pool"], s["k_scale"]), _padded_cache(s, s["v_pool"], s["v_scale"])
    q = q.view(case["batch"], most, hk, h // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [batch, hk, group * most, d]
    p = torch.full((case["batch"], most), -1, dtype=torch.long, device="cuda")
    p[seq, within] = pos
    j = torch.arange(k.shape[2], device="cuda")
    seen = (j <= p[..., None]) & (j < s["kv_len"].long()[:, None, None])
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    scores = (q @ k.transpose(2, 3)) * (d ** -0.5)
    scores = scores.unflatten(2, (h // hk, most)).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.flatten(2, 3) @ v).unflatten(2, (h // hk, most)) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(case["batch"], most, h, d)
    lg = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(case["batch"], most, h)
    out[: s["tokens"]] = o[seq, within].to(out.dtype)
    lse[: s["tokens"]] = lg[seq, within]
    return out, lse


def _quantised(x):
    scale = (x.abs().amax(-1, keepdim=True) / FP8_MAX).clamp(min=FP8_TINY)
    return (x / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale[..., 0]


def _plain_append(s):
    seq, pos, live, page, slot = _rows_of_tokens(s)
    n = s["tokens"]
    q, k, v = (s[x][:n].float() for x in "qkv")
    q_out = s["q_out"]
    if "inv_freq" in s:
        k = _turn(k, pos, s)
        q_out[:n] = torch.where(live[:, None, None], _turn(q, pos, s), q_out[:n].float()).to(q_out.dtype)
    page, slot = page[live], slot[live]
    for pool, scales, x in ((s["k_pool"], s["k_scale"], k[live]), (s["v_pool"], s["v_scale"], v[live])):
        if scales is None:
            pool[page, :, slot] = x.to(pool.dtype)
        else:
            codes, scale = _quantised(x)
            pool.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            scales[page, :, slot] = scale
    return q_out


def _plain_gather(s):
    if s["rows"]:
        there = torch.arange(-(-s["longest"] // s["case"]["page"]) * s["case"]["page"], device="cuda") < s["kv_len"].long()[:, None]
        for name in "kv":
            x = _padded_cache(s, s[name + "_pool"], s[name + "_scale"]).transpose(1, 2)
            s[name + "_out"].copy_(x[there].to(torch.bfloat16))


# ---- one pass --------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _context():
    """The library context a program keeps for its stream."""
    from qs3_b200 import ops
    return ops.Context()


_workspace = {}


def _kept_workspace(nbytes):
    """The workspace a program keeps for its stream; it grows to the largest call."""
    if "ws" not in _workspace or _workspace["ws"].numel() < nbytes:
        _workspace["ws"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return _workspace["ws"]


def run(state):
    s, case = state, state["case"]
    if case["kind"] == "rope":
        if own:
            from qs3_b200 import ops
            ops.rope(_context(), s["positions"], s["inv_freq"], s["q"], s["k"], q_out=s["q_out"], k_out=s["k_out"],
                     scale=s["rope_scale"], interleaved=case["interleaved"])
        else:
            for name in "qk":
                s[name + "_out"].copy_(_turn(s[name].float(), s["positions"], s))
        return [s["q_out"], s["k_out"]]
    if own:
        from qs3_b200 import ops
        cache = ops.PagedKvCache(s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
        table = ops.PageTable(s["kv_indptr"], s["kv_indices"], s["kv_len"])
    if case["kind"] == "gather":
        if own:
            ops.kv_gather(_context(), cache, table, s["out_indptr"], s["k_out"], s["v_out"])
        else:
            _plain_gather(s)
        return [s["k_out"], s["v_out"]]
    if case["kind"] == "append":
        if own:
            turned = dict(q=s["q"], q_out=s["q_out"], inv_freq=s["inv_freq"], rope_scale=s["rope_scale"],
                          interleaved=case["interleaved"]) if case["rotary"] else {}
            ops.kv_append(_context(), cache, table, s["k"], s["v"], q_indptr=s["q_arg"], **turned)
        else:
            _plain_append(s)
        out = [s["q_out"], s["k_pool"], s["v_pool"]]
        return out + [s["k_scale"], s["v_scale"]] if case["fp8"] else out
    if own:
        ws = _kept_workspace(ops.paged_attention_workspace_size(_context(), s["q"], cache, batch=case["batch"]))
        ops.paged_attention(_context(), s["q"], cache, table, s["out"], ws, q_indptr=s["q_arg"], max_q_len=s["q_longest"],
                            max_kv_len=s["longest"], window=case["window"], lse=s["lse"])
        return [s["out"], s["lse"]]
    return list(_plain_attention(s))


# ---- the same in 64 bits -------------------------------------------------------------------------------


def _spin(x, position, freq, scale, interleaved):
    """x [..., dim] in 64 bits times exp(i * position * freq), pairs as complex numbers. position: [tokens]."""
    r = 2 * len(freq)
    z = torch.polar(torch.full_like(position.double()[:, None] * freq, scale), position.double()[:, None] * freq)[:, None]
    body = x[..., :r]
    pairs = body.unflatten(-1, (-1, 2)) if interleaved else body.unflatten(-1, (2, -1)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    turned = turned if interleaved else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), x[..., r:]], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, d = case["kind"], case["dim"]
    if kind == "rope":
        return [_spin(s[n].double(), s["positions"], s["inv_freq"], s["rope_scale"], case["interleaved"]) for n in "qk"]
    q_len, kv_len = _lengths(case)
    indptr, indices, page = s["kv_indptr"].tolist(), s["kv_indices"].long(), case["page"]

    def cached(b, pool, scale):
        """[tokens, kv_heads, dim] of sequence b."""
        ids = indices[indptr[b]: indptr[b + 1]]
        x = pool[ids].double()
        if scale is not None:
            x = x * scale[ids].double()[..., None]
        return x.transpose(1, 2).flatten(0, 1)[: kv_len[b]]

    if kind == "gather":
        return [torch.cat([cached(b, s[n + "_pool"], s[n + "_scale"]) for b in range(case["batch"])]) if s["rows"] else None
                for n in "kv"]
    if kind == "append":
        q_out = s["q_out"].double()
        pools = {n: s[n + "_pool"].double() for n in "kv"}
        scales = {n: s[n + "_scale"].double() if case["fp8"] else None for n in "kv"}
        row = 0
        for b in range(case["batch"]):
            n = q_len[b]
            if kv_len[b] and n:
                pos = torch.arange(kv_len[b] - n, kv_len[b], device="cuda")
                at = (indices[indptr[b] + pos // page], pos % page)
                for name in "kv":
                    x = s[name][row: row + n].double()
                    if name == "k" and case["rotary"]:
                        x = _spin(x, pos, s["inv_freq"], s["rope_scale"], case["interleaved"])
                    if case["fp8"]:
                        unit = (x.abs().amax(-1) / FP8_MAX).clamp(min=FP8_TINY)
                        scales[name][at[0], :, at[1]] = unit
                        x = x / unit[..., None]
                    pools[name][at[0], :, at[1]] = x
                if case["rotary"]:
                    q_out[row: row + n] = _spin(s["q"][row: row + n].double(), pos, s["inv_freq"], s["rope_scale"],
                                                case["interleaved"])
            row += n
        out = [q_out, pools["k"], pools["v"]]
        return out + [scales["k"], scales["v"]] if case["fp8"] else out
    h, hk = case["heads"], case["kv_heads"]
    out, lse = s["out"].double(), s["lse"].double()
    row = 0
    for b in range(case["batch"]):
        n, length = q_len[b], kv_len[b]
        lse[row: row + n] = -math.inf
        if length and n:
            k, v = cached(b, s["k_pool"], s["k_scale"]), cached(b, s["v_pool"], s["v_scale"])
            for first in range(0, n, 2048):
                some = slice(row + first, row + min(n, first + 2048))
                pos = torch.arange(length - n + first, length - n + min(n, first + 2048), device="cuda")[:, None]
                j = torch.arange(length, device="cuda")[None]
                hidden = j > pos
                if case["window"]:
                    hidden = hidden | (j + case["window"] <= pos)
                for g in range(h):
                    x = s["q"][some, g].double() @ k[:, g * hk // h].T / math.sqrt(d)
                    x = torch.where(hidden, -math.inf, x)
                    lse[some, g] = torch.logsumexp(x, dim=1)
                    out[some, g] = torch.softmax(x, dim=1) @ v[:, g * hk // h]
        row += n
    return [out, lse]
