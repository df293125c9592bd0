"""B200Transformer.extend over a PagedKVCache: chunks and single tokens give the rows of one whole forward."""

import math

import pytest
import torch

import oracle
from tiktoktechjam2026_b200 import B200Transformer, PagedKVCache, TransformerConfig, copy_mixed_model_weights, ops

DEV = "cuda:0"


class _Baseline(torch.nn.Module):
    def __init__(self, sd):
        super().__init__()
        self._sd = sd

    def state_dict(self, *a, **k):
        return dict(self._sd)


def build(d, heads, ffn, layers, batch=2, seq=160):
    cfg = oracle.Config(batch, seq, d, heads, ffn, layers, True)
    sd = oracle.seeded_state_dict(cfg, 77)
    model = B200Transformer(TransformerConfig(batch, seq, d, heads, ffn, layers, True))
    copy_mixed_model_weights(_Baseline(sd), model)
    model = model.to(DEV).eval()
    model.convert_projections_to_fp16()
    return cfg, sd, model


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def passes(ref, out):
    """The reference's per-element rule: absolute error within 2e-3, or 0.02 of the value."""
    res = oracle.compare(ref, out.cpu())
    assert res.passed, res


MODELS = [(128, 4, 128, 2), (256, 8, 1024, 2), (512, 8, 2048, 1), (128, 16, 128, 2), (32, 2, 128, 3), (64, 1, 96, 2),
          (1024, 8, 1024, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,ffn,layers", MODELS)
def test_chunks_equal_the_oracle(tt_lib, strict_fp32, d, heads, ffn, layers):
    """A prompt in chunks of 1, 37, 64 and 58 tokens: every row within the rule of the strict FP32 model."""
    cfg, sd, model = build(d, heads, ffn, layers)
    x, _ = oracle.generate_case(cfg, 5)
    ref = oracle.forward(sd, cfg, x, None)
    cache = PagedKVCache.for_model(model, slots=5, max_len=160, page=16)
    slots = ints([3, 1])
    got, at = [], 0
    with torch.inference_mode():
        for t in (1, 37, 64, 58):
            got.append(model.extend(x[:, at:at + t].to(DEV), cache, slots=slots))
            at += t
    passes(ref, torch.cat(got, 1))
    assert cache.lens.tolist() == [0, 160, 0, 160, 0]


@pytest.mark.gpu
def test_ragged_tokens_fork_and_compact(tt_lib, strict_fp32):
    """Ragged prompts, a fork that answers differently, a released slot and a compaction in between."""
    cfg, sd, model = build(256, 8, 1024, 2, batch=3, seq=140)
    x, _ = oracle.generate_case(cfg, 9)
    ref = oracle.forward(sd, cfg, x, None)
    xd = x.to(DEV)
    cache = PagedKVCache.for_model(model, slots=6, max_len=256, page=32)
    prompts = [70, 33, 96]
    cu = ints([0, 70, 103, 199])
    with torch.inference_mode():
        out = model.extend(torch.cat([xd[b, :t] for b, t in enumerate(prompts)]), cache, cu)
        for b, t in enumerate(prompts):
            passes(ref[b, :t], out[int(cu[b]):int(cu[b + 1])])
        cache.fork(ints([0, 2]), ints([5, 4]))
        cache.check()
        cache.release(ints([0, 2]))  # the children go on alone
        live = int(cache.compact())
        assert live == 3 + 2 + 3 and int(cache.tables.max()) == live - 1
        for j in range(12):  # token by token, sequences 0, 1, 2 now in slots 5, 1, 4
            step = torch.stack([xd[b, t + j] for b, t in enumerate(prompts)])[:, None]
            out = model.extend(step, cache, slots=ints([5, 1, 4]))
            for b, t in enumerate(prompts):
                passes(ref[b, t + j], out[b, 0])


@pytest.mark.gpu
def test_two_answers_of_one_prompt(tt_lib):
    """Parent and child write into pages of their own after a fork: neither sees the other's tokens."""
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    x, _ = oracle.generate_case(cfg, 3)
    a = torch.randn(1, 20, 128, device=DEV)
    b = torch.randn(1, 20, 128, device=DEV)
    xd = x.to(DEV)[:, :41]
    with torch.inference_mode():
        alone = []
        for tail in (a, b):
            cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
            model.extend(xd, cache, slots=ints([0]))
            alone.append(model.extend(tail, cache, slots=ints([0])))
        cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
        model.extend(xd, cache, slots=ints([0]))
        cache.fork(ints([0]), ints([1]))
        both = model.extend(torch.cat([a, b]), cache)
    assert cache.refs.tolist()[:2] == [2, 2]
    assert torch.equal(both[0], alone[0][0]) and torch.equal(both[1], alone[1][0])


@pytest.mark.gpu
def test_window_with_trimmed_pages(tt_lib):
    """Trimming what the window left behind changes no row, and bounds the pages a sequence holds."""
    cfg, sd, model = build(256, 8, 1024, 2, batch=1, seq=300)
    x, _ = oracle.generate_case(cfg, 4)
    xd = x.to(DEV)
    window, sinks = 48, 4
    with torch.inference_mode():
        whole = PagedKVCache.for_model(model, slots=1, max_len=320, page=16)
        want = model.extend(xd, whole, window=window, sinks=sinks)
        cache = PagedKVCache.for_model(model, slots=1, max_len=320, page=16, pages=8)
        at = 0
        for t in (40, 1, 1, 30, 17, 1) + (30,) * 7:
            got = model.extend(xd[:, at:at + t], cache, window=window, sinks=sinks)
            torch.testing.assert_close(got, want[:, at:at + t], rtol=2e-2, atol=2e-3)
            at += t
            cache.trim(window, sinks)
            assert int((cache.refs > 0).sum()) <= 1 + 48 // 16 + 1
    assert at == 300


@pytest.mark.gpu
def test_no_room_leaves_the_cache_alone(tt_lib):
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    x = torch.randn(1, 64, 128, device=DEV)
    cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16, pages=3)
    cache.k.zero_(), cache.v.zero_()  # fresh pages may hold NaN, which equals nothing
    with torch.inference_mode():
        model.extend(x[:, :40], cache, slots=ints([0]))
        state = [t.clone() for t in (cache.k[:, :3], cache.v[:, :3], cache.tables, cache.lens, cache.refs)]
        with pytest.raises(RuntimeError, match="2 page"):
            model.extend(x[:, :20], cache, slots=ints([1]))
        model.extend(x[:, :20], cache, slots=ints([1]), check=False)
        with pytest.raises(RuntimeError, match="2 page"):
            cache.check()
        with pytest.raises(RuntimeError, match="outgrow"):
            model.extend(x[:, :30], cache, slots=ints([0]))
        with pytest.raises(RuntimeError, match="slot"):
            model.extend(x[:, :3], cache, slots=ints([2]))
        for a, b in zip(state, (cache.k[:, :3], cache.v[:, :3], cache.tables, cache.lens, cache.refs)):
            assert torch.equal(a, b)
        assert model.extend(x[:, :0], cache, slots=ints([0])).shape == (1, 0, 128)


@pytest.mark.gpu
def test_extend_refusals(tt_lib):
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    cache = PagedKVCache.for_model(model, slots=2, max_len=64)
    x = torch.randn(1, 3, 128, device=DEV)
    bad = [(x.half(), cache, None), (x[..., :64], cache, None), (x[0], cache, None), (x, cache, ints([0, 3])),
           (x.cpu(), cache, None),
           (x, PagedKVCache(1, 4, 4, 32, slots=1, max_len=64, device=DEV), None),
           (x, PagedKVCache(2, 4, 8, 16, slots=1, max_len=64, device=DEV), None),
           (x, PagedKVCache(2, 4, 4, 32, slots=1, max_len=64, dtype=torch.bfloat16, device=DEV), None)]
    for a in bad:
        with pytest.raises(ValueError):
            model.extend(*a)
    both_ways = B200Transformer(TransformerConfig(1, 64, 128, 4, 128, 2, False))
    with pytest.raises(ValueError, match="causal"):
        both_ways.extend(x, cache)


def test_cache_refusals_need_no_gpu():
    ok = dict(slots=1, max_len=64)
    for args, kw in [((1, 1, 1, 32), dict(ok, page=24)), ((1, 0, 1, 32), ok), ((1, 1, 1, 48), ok),
                     ((1, 1, 1, 32), dict(ok, dtype=torch.float32)), ((1, 1, 1, 32), dict(ok, device="cpu"))]:
        with pytest.raises(ValueError):
            PagedKVCache(*args, **kw)
    assert ops.stored_head_dim(8) == 16 and math.isclose(8**-0.5, 0.35355, rel_tol=1e-4)
