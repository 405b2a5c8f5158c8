"""The dense backend's layers and model on the CPU, with the device kernels that
they call replaced by plain forms: which path they take, and what reaches whom."""

import itertools

import pytest
import torch
import torch.nn.functional as F

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import attention, model, ops, scoring
from local_research_small_language_model_b200.rope import rotate_half


def plain_rope(xq, xk, cos, sin, offset=0):
    c, s = (torch.cat([x, x], -1)[None, :, None] for x in (cos, sin))
    return tuple(x * c + rotate_half(x) * s for x in (xq, xk))


def plain_attention(q, k, v, cu_seqlens, scale=None):
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    cu = cu_seqlens.tolist()
    parts = [out[:cu[0]]]
    for a, b in zip(cu, cu[1:]):
        kk, vv = (x[a:b].repeat_interleave(group, 1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q[a:b], kk) / 8
        late = torch.ones(b - a, b - a, dtype=torch.bool).triu(1)
        parts.append(torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(late, -torch.inf), -1), vv))
    return torch.cat(parts + [out[cu[-1]:]])


def plain_scores(logits, targets, top_k=0, ignore_index=-100):
    lp = torch.log_softmax(logits.float(), -1)
    kept = targets != ignore_index
    chosen = lp.gather(1, targets.clamp_min(0)[:, None])[:, 0] * kept
    top = lp.topk(top_k, -1)
    return scoring.TokenLogprobs(chosen, -(lp.exp() * lp).sum(-1), top.values, top.indices)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(ops, "rope_qk", plain_rope)
    monkeypatch.setattr(attention, "packed_attention", plain_attention)
    monkeypatch.setattr(model, "token_logprobs", plain_scores)
    monkeypatch.setattr(ops, "silu_mul", lambda x: F.silu(x[:, :x.shape[1] // 2]) * x[:, x.shape[1] // 2:])


CONFIG = dict(vocab_size=50, n_layer=2, n_embd=128, n_head=2, n_kv_head=1, ffn_dim=64, context_length=64,
              attention_backend="b200_dense")


@pytest.mark.parametrize("trained", [c for n in (1, 2, 3) for c in itertools.combinations(("wq", "wk", "wv"), n)],
                         ids="+".join)
def test_frozen_projections_leave_the_others_their_gradients(on_cpu, trained):
    """Whichever of wq, wk and wv are trained get the gradients that they have
    when all are, also where the layer's input has none."""
    torch.manual_seed(0)
    layer = sd.B200DenseAttention(sd.ModelConfig(**CONFIG), 0)
    rope = sd.RotaryEmbedding(64, 64)
    x, weight = torch.randn(2, 9, 128), torch.randn(2, 9, 128)
    names = ("wq", "wk", "wv")
    (layer(x, rope) * weight).sum().backward()
    want = {n: getattr(layer, n).weight.grad.clone() for n in names}
    layer.zero_grad()
    for n in names:
        getattr(layer, n).weight.requires_grad_(n in trained)
    (layer(x, rope) * weight).sum().backward()
    for n in names:
        got = getattr(layer, n).weight.grad
        assert (got is None) == (n not in trained)
        if got is not None:
            assert torch.allclose(got, want[n], rtol=1e-5, atol=1e-6)


def test_training_some_projections_of_a_model_trains_its_first_layer(on_cpu):
    torch.manual_seed(1)
    m = model.SparDAB200Model(sd.ModelConfig(**CONFIG))
    for name, p in m.named_parameters():
        p.requires_grad_("wv" in name or "wo" in name)
    ids = torch.randint(0, 50, (2, 12))
    m(ids, targets=ids)["loss"].backward()
    for name, p in m.named_parameters():
        assert (p.grad is not None and bool(p.grad.any())) == p.requires_grad, name


@pytest.mark.parametrize("grad", [False, True])
def test_forecasts_are_returned_where_they_are_asked_for(on_cpu, grad):
    """The projection of every layer's normed input, as the reference's block
    computes it whatever attends (model/transformer.py:104-107)."""
    torch.manual_seed(2)
    m = model.SparDAB200Model(sd.ModelConfig(**CONFIG))
    ids = torch.randint(0, 50, (2, 6))
    inputs = []
    for layer in m.layers:
        layer.attn_norm.register_forward_hook(lambda mod, args, out: inputs.append(out))
    with torch.set_grad_enabled(grad):
        got = m(ids, return_forecasts=True)
    assert len(got["forecasts"]) == 2
    for f, x, layer in zip(got["forecasts"], inputs, m.layers):
        assert torch.equal(f, layer.forecast(x)) and f.requires_grad == grad
    assert "forecasts" not in m(ids)


def test_lengths_have_to_be_those_of_the_bounds(on_cpu):
    """They bound the tokens' positions: wrong ones would rotate tokens wrongly."""
    m = model.SparDAB200Model(sd.ModelConfig(**CONFIG)).eval()
    ids = torch.randint(0, 50, (1, 12))
    cu = torch.tensor([0, 8, 11], dtype=torch.int32)
    with torch.no_grad():
        want = m(ids, cu_seqlens=cu)["logits"]
        assert torch.equal(m(ids, cu_seqlens=cu, lengths=[8, 3])["logits"], want)
        for wrong in ([3], [8, 3, 1], [9, 4], [-1, 3], []):
            with pytest.raises(ValueError, match="lengths"):
                m(ids, cu_seqlens=cu, lengths=wrong)
        caches = m.allocate_paged_caches(3, 64)
        with pytest.raises(ValueError, match="lengths"):
            m(ids, kv_caches=caches, cu_seqlens=cu, lengths=[8, 4, 0])
        assert not any(caches[0].pages.owned)  # nothing was reserved


def test_a_step_without_a_cache_is_refused(on_cpu):
    layer = sd.B200DenseAttention(sd.ModelConfig(**CONFIG), 0)
    rope = sd.RotaryEmbedding(64, 64)
    step = sd.RaggedBatch.step(torch.tensor([3, 4], dtype=torch.int32), 64, rope)
    with torch.no_grad(), pytest.raises(ValueError, match="paged cache"):
        layer(torch.randn(2, 1, 128), rope, ragged=step)
