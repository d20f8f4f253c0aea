"""The hybrid decode loop with this library's attention over the paged cache: the layer against its torch stand-in on the
same weights and cache, graph replays against eager steps, and the pages it may write."""
import numpy as np
import pytest
import torch

from helpers import f32, to_np

pytestmark = pytest.mark.gpu


def _pair(cfg, fp8):
    from dataclasses import replace
    from qs3_b200 import ops
    from qs3_b200.hybrid_decode import _Attention, _PagedAttention
    dev = torch.device("cuda", 0)
    max_len = cfg.context + cfg.new_tokens
    new = lambda: torch.Generator(device=dev).manual_seed(3)
    ctx = ops.Context()
    kv_len = torch.full((cfg.batch,), cfg.context + 1, dtype=torch.int32, device=dev)
    return (_Attention(cfg, new(), dev, max_len),
            _PagedAttention(replace(cfg, attention="paged", kv_fp8=fp8), new(), dev, max_len, ctx, kv_len), ctx)


def _inputs(cfg, a):
    dev = a.k_pool.device
    mask = torch.full((1, 1, a.pages_per_seq * a.page), float("-inf"), device=dev)
    mask[..., : cfg.context + 1] = 0.0
    x = (torch.randn((cfg.batch, cfg.hidden), generator=torch.Generator(device=dev).manual_seed(4), device=dev) * 0.5)
    return x.to(torch.bfloat16), torch.full((1,), cfg.context, dtype=torch.long, device=dev), mask


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("sizes", [dict(), dict(q_heads=16, head_dim=256, rotary_dim=64, context=333, page_size=16)])
def test_layer_matches_its_stand_in(sizes, fp8):
    from qs3_b200.hybrid_decode import tiny_config
    cfg = tiny_config(new_tokens=8, **sizes)
    a, b, ctx = _pair(cfg, fp8)
    x, pos, mask = _inputs(cfg, a)
    if fp8:   # the stand-in attends over what the e4m3 cache holds
        from qs3_b200 import ops
        n, cached = cfg.context, b._cache()
        for i in range(cfg.batch):
            rows = torch.tensor([0, n], dtype=torch.int32, device=x.device)
            table = ops.PageTable(a.kv_indptr[i: i + 2].contiguous(), a.kv_indices, rows[1:].contiguous())
            k, v = (torch.empty((n, cfg.kv_heads, cfg.head_dim), dtype=torch.bfloat16, device=x.device) for _ in range(2))
            ops.kv_gather(ctx, cached, table, rows, k, v)
            ops.kv_append(ctx, ops.PagedKvCache(a.k_pool, a.v_pool), table, k, v, q_indptr=rows)
    want, got = f32(to_np(a(x, pos, mask))), f32(to_np(b(x, pos, mask)))
    assert ctx.read_device_error() == 0
    # Both round q, k and the output to bf16 and the weights to 16 bits: each of these by 2^-8 / sqrt(3) of a value at most in
    # the mean square, once in either layer, so scores of unit variance differ by a few times 2^-8 and so do weights and
    # outputs: ten such steps. An e4m3 row that is gathered to bf16 adds another step, and this step's own token, of at least
    # 25, is rounded to e4m3 by 2^-4 on one side.
    bound = 10 * 2.0 ** -8 + (2.0 ** -4 / 5 if fp8 else 0.0)
    assert np.linalg.norm(got - want) <= bound * np.linalg.norm(want)


@pytest.mark.parametrize("fp8", [False, True])
def test_replays_follow_eager_steps(fp8):
    from qs3_b200.hybrid_decode import HybridDecoder, tiny_config
    cfg = tiny_config(new_tokens=8, attention="paged", kv_fp8=fp8)
    model = HybridDecoder(cfg)
    start = model.snapshot()

    def run(n, graph=None):
        model.restore(start)
        toks = []
        with torch.cuda.stream(model.stream):
            model.ctx.use_current_stream()
            for _ in range(n):
                model.replay(graph) if graph is not None else model.step()
                toks.append(model.tokens.clone())
            model.stream.synchronize()
        return torch.stack(toks).cpu().numpy(), to_np(model.logits)

    eager_tokens, eager_logits = run(3)
    model.restore(start)
    graph = model.capture()
    graph_tokens, graph_logits = run(3, graph)
    assert model.ctx.read_device_error() == 0
    assert np.array_equal(eager_tokens, graph_tokens)
    assert np.array_equal(eager_logits, graph_logits)
    assert np.isfinite(f32(graph_logits)).all()
    before = [t.clone() for t, _ in model._state_tensors()]
    assert model.time_steps(2) > 0
    for t, (now, _) in zip(before, model._state_tensors()):
        assert torch.equal(t, now)


def test_only_the_new_tokens_slots_are_written():
    from qs3_b200.hybrid_decode import tiny_config
    cfg = tiny_config(new_tokens=8, page_size=16)
    a, b, ctx = _pair(cfg, False)
    x, pos, mask = _inputs(cfg, a)
    k_before, v_before = b.k_pool.clone(), b.v_pool.clone()
    b(x, pos, mask)
    pages = b.kv_indices.view(cfg.batch, b.pages_per_seq)[:, cfg.context // b.page].long()
    for pool, before in ((b.k_pool, k_before), (b.v_pool, v_before)):
        changed = (pool != before).any(dim=-1)                                # [pages, kv_heads, page]
        assert changed[pages, :, cfg.context % b.page].all()
        assert int(changed.sum()) == cfg.batch * cfg.kv_heads


def test_an_unknown_attention_is_refused():
    from qs3_b200.hybrid_decode import HybridDecoder, tiny_config
    for kw in (dict(attention="flat"), dict(kv_fp8=True)):
        with pytest.raises(ValueError, match="attention"):
            HybridDecoder(tiny_config(**kw))


def test_lengths_are_kept_for_paged_attention_only():
    """The torch stand-in reads no lengths, and its step writes none."""
    from qs3_b200.hybrid_decode import HybridDecoder, tiny_config
    assert HybridDecoder(tiny_config()).kv_len is None
    model = HybridDecoder(tiny_config(attention="paged"))
    with torch.cuda.stream(model.stream):
        model.ctx.use_current_stream()
        model.step()
        model.stream.synchronize()
    assert bool((model.kv_len == model.cfg.context + 1).all())


def test_attention_layers_share_one_workspace():
    from qs3_b200.hybrid_decode import HybridDecoder, _PagedAttention, tiny_config
    model = HybridDecoder(tiny_config(layers=8, attention="paged"))
    layers = [m for m in model.mixers if isinstance(m, _PagedAttention)]
    assert len(layers) == 2 and len({m.workspace.data_ptr() for m in layers}) == 1


@pytest.mark.parametrize("attention", ["torch", "paged"])
def test_library_share_counts_the_attention_calls(attention, monkeypatch):
    """A step without the stand-ins still makes every call of this library that a whole step makes."""
    from qs3_b200 import hybrid_decode as m
    cfg = m.tiny_config(layers=8, new_tokens=12, attention=attention)
    model, calls = m.HybridDecoder(cfg), {}
    for name in ("kv_append", "paged_attention", "moe_layer_execute", "rmsnorm", "fused_add_rmsnorm_nvfp4"):
        def counted(*a, _name=name, _real=getattr(m.ops, name), **kw):
            calls[_name] = calls.get(_name, 0) + 1
            return _real(*a, **kw)
        monkeypatch.setattr(m.ops, name, counted)
    made = []
    with torch.cuda.stream(model.stream):
        model.ctx.use_current_stream()
        for mixers in (True, False):
            calls.clear()
            model.step(mixers)
            made.append(dict(calls))
        model.stream.synchronize()
    assert made[0] == made[1] and made[0].get("paged_attention", 0) == (2 if attention == "paged" else 0)
    record = m.measure(2, cfg)
    assert ("attention" in record["library_calls"]) == (attention == "paged")
    assert record["device_error"] == 0
