"""Paged caches of another dtype than the model: prompts and decode steps run, the
steps in the cache's type.  On the CPU with plain forms for the device kernels,
and on a B200."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import model, ops
from tests import test_ragged_serving
from tests.test_ragged_layers import CONFIG, on_cpu  # noqa: F401
from tests.test_ragged_serving import paged  # noqa: F401

PAIRS = [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float16),
         (torch.float32, torch.float32)]


@torch.no_grad()
def run(device, own, cached, rope_qk):
    """A layer's step over a cache, and the formula on the same rows in the cache's type."""
    torch.manual_seed(5)
    cfg = sd.ModelConfig(**CONFIG)
    layer = sd.B200DenseAttention(cfg, 0).to(device, own)
    pages = sd.PageTable(3, 64, 12, torch.device(device), page_size=16)
    cache = sd.B200PagedKVCache(pages, 1, 64, torch.device(device), cached)
    rope = sd.RotaryEmbedding(64, 64).to(device)
    pages.reserve(20)
    layer(torch.randn(3, 20, 128, device=device).to(own), rope, cache)
    pages.advance(20)
    pages.reserve(1)
    q, k, v = (torch.randn(3, h, 64, device=device).to(own) for h in (2, 1, 1))
    got = layer.core(q, k, v, 3, 1, rope, cache)
    pages.advance(1)
    pos = torch.full((3,), 20, device=device)
    q, k = (y[0] for y in rope_qk(q[None], k[None], rope.cos[pos], rope.sin[pos]))
    for b in range(3):
        assert torch.equal(cache.k_pages[pages.owned[b][1], :, 4], k[b].to(cached))
        assert torch.equal(cache.v_pages[pages.owned[b][1], :, 4], v[b].to(cached))
    want = ops.paged_decode_attention(q.to(cached), cache.k_pages, cache.v_pages, pages.table, pages.lens)
    assert got.dtype == own and torch.equal(got, want.to(own))
    m = model.SparDAB200Model(cfg).to(device, own).eval()
    caches = m.allocate_paged_caches(2, 64, dtype=cached)
    ids = torch.randint(0, 50, (2, 7), device=device)
    m(ids, kv_caches=caches)
    logits = m(ids[:, :1], kv_caches=caches)["logits"]
    assert logits.dtype == own and torch.isfinite(logits).all()
    full = m(torch.cat([ids, ids[:, :1]], 1))["logits"][:, -1:]
    # k, v, q and the result rounded to the narrower type once each, through two layers of O(1) values
    u = max(torch.finfo(t).eps for t in (own, cached))
    assert float((logits.float() - full.float()).abs().max()) < 16 * u * max(1.0, float(full.float().abs().max()))


@pytest.mark.parametrize("types", PAIRS, ids=lambda t: "_in_".join(str(x).split(".")[1] for x in t))
def test_plain(paged, monkeypatch, types):  # noqa: F811
    def same_type(q, k_pages, *rest, **more):
        if q.dtype is not k_pages.dtype:
            raise TypeError(f"q of {q.dtype} does not fit pages of {k_pages.dtype}")
        return test_ragged_serving.plain_decode(q, k_pages, *rest, **more)

    monkeypatch.setattr(ops, "paged_decode_attention", same_type)
    monkeypatch.setattr(ops, "rope_qk", lambda q, k, c, s, offset=0: tuple(
        y.to(q.dtype) for y in test_ragged_serving.plain_rope(q.float(), k.float(), c, s)))
    run("cpu", *types, ops.rope_qk)


@pytest.mark.gpu
@pytest.mark.parametrize("types", PAIRS, ids=lambda t: "_in_".join(str(x).split(".")[1] for x in t))
def test_kernels(dev, types):
    run(dev, *types, ops.rope_qk)
    ops.check_device_errors(dev)
