"""B200Transformer.extend: what it refuses leaves the cache as it was."""

import pytest
import torch

from test_extend_gpu import DEV, _Baseline, build, ints
from tiktoktechjam2026_b200 import (B200Transformer, PagedKVCache, TransformerConfig, _lib, copy_mixed_model_weights,
                                    ops)


def _state(cache):
    return [t.clone() for t in (cache.tables, cache.lens, cache.refs)]


def _refused(model, cache, x, exc, **kw):
    before = _state(cache)
    with pytest.raises(exc):
        model.extend(x, cache, **kw)
    for a, b in zip(before, _state(cache)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refused_window_leaves_the_cache_alone(tt_lib):
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
    x = torch.randn(1, 20, 128, device=DEV)
    with torch.inference_mode():
        model.extend(x, cache)
        _refused(model, cache, x, ValueError, window=-1)
        _refused(model, cache, x, ValueError, window=8, sinks=-1)
        _refused(model, cache, x, TypeError, window=8.5)
        _refused(model, cache, x, TypeError, max_q_len="20")


@pytest.mark.gpu
def test_model_that_is_not_ready_leaves_the_cache_alone(tt_lib):
    """FP32 projections, as before convert_projections_to_fp16; one layer left behind; a shape without kernels."""
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
    x = torch.randn(1, 20, 128, device=DEV)
    fresh = B200Transformer(TransformerConfig(1, 64, 128, 4, 128, 2, True))
    copy_mixed_model_weights(_Baseline(sd), fresh)
    with torch.inference_mode():
        model.extend(x, cache)
        _refused(fresh.to(DEV).eval(), cache, x, RuntimeError)
        model.layers[1].ffn_out.float()
        _refused(model, cache, x, RuntimeError)
    wide = B200Transformer(TransformerConfig(1, 64, 160, 5, 100, 2, True)).to(DEV).eval()  # ffn_dim of 100
    wide.convert_projections_to_fp16()
    with torch.inference_mode():
        _refused(wide, PagedKVCache.for_model(wide, slots=2, max_len=64), torch.randn(1, 3, 160, device=DEV), RuntimeError)


@pytest.mark.gpu
def test_model_on_another_device_is_refused(tt_lib):
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    cache = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
    x = torch.randn(1, 20, 128, device=DEV)
    model.layers[1].norm2.to("cpu")
    _refused(model, cache, x, ValueError)
    model.to("cpu")
    _refused(model, cache, x, ValueError)


@pytest.mark.gpu
def test_tokens_at_any_address(tt_lib):
    """x may begin at any float of a larger buffer; the layer norm operator itself asks for whole 16 bytes."""
    cfg, sd, model = build(128, 4, 128, 2, batch=1, seq=64)
    buf = torch.randn(20 * 128 + 1, device=DEV)
    x = buf[1:].view(1, 20, 128)
    with torch.inference_mode():
        want = model.extend(x.clone(), PagedKVCache.for_model(model, slots=1, max_len=64, page=16))
        got = model.extend(x, PagedKVCache.for_model(model, slots=1, max_len=64, page=16))
    assert torch.equal(got, want)
    with pytest.raises(_lib.TTError, match="aligned"):
        ops.layernorm_rows(x, model.layers[0].norm1.weight, model.layers[0].norm1.bias)


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,ffn", [(128, 4, 128), (512, 8, 2048)])
def test_tokens_from_a_captured_graph(tt_lib, d, heads, ffn):
    """extend(check=False) captured once gives, replayed token by token, the rows of the same calls made one by one."""
    cfg, sd, model = build(d, heads, ffn, 2, batch=2, seq=64)
    prompt, steps = torch.randn(2, 37, d, device=DEV), torch.randn(12, 2, 1, d, device=DEV)
    one, two = (PagedKVCache.for_model(model, slots=2, max_len=64, page=16) for _ in range(2))
    with torch.inference_mode():
        for cache in (one, two):
            model.extend(prompt, cache)
        want = [model.extend(x, one) for x in steps]
        x = steps[0].clone()
        warm = PagedKVCache.for_model(model, slots=2, max_len=64, page=16)
        model.extend(x, warm, check=False)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.extend(x, two, check=False)
        for step, row in zip(steps, want):
            x.copy_(step)
            graph.replay()
            assert torch.equal(out, row)
        two.check()
    assert two.lens.tolist() == one.lens.tolist() == [49, 49]
