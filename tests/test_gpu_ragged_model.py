"""The operators for ragged batches together, as a user runs them: packed
prompts into paged caches, decode steps (eager and as a captured graph),
scores, and a training step over packed documents, through SparDAB200Model's
"b200_dense" backend against a plain restatement of the model in 64 bits.

Tolerances: fp32 end to end through three layers, whose values are O(1); the
sums are at most 2048 long, so a result is off by a few hundred u32 = 2^-24 of
its terms' sum: 2e-4 as for the other model tests, and 1e-3 relative for
gradients (sums over all tokens).  Needs a B200."""

import pytest
import torch
import torch.nn.functional as F

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from local_research_small_language_model_b200.model import SparDAB200Model
from local_research_small_language_model_b200.rope import apply_rotary_emb, precompute_rope_freqs

pytestmark = pytest.mark.gpu

LENGTHS = [70, 3, 129, 1, 64]


def model(dev, dtype=torch.float32, page=64):
    torch.manual_seed(3)
    cfg = sd.ModelConfig(vocab_size=1000, n_layer=3, n_embd=256, n_head=4, n_kv_head=2, ffn_dim=512,
                         context_length=256, attention_backend="b200_dense")
    return SparDAB200Model(cfg).to(dev, dtype)


def plain(m, p, ids):
    """Logits [T,V] of one sequence from the parameters p (64 bits)."""
    cfg = m.config

    def norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.norm_eps) * w

    t = ids.numel()
    cos, sin = (x.double().to(ids.device) for x in precompute_rope_freqs(cfg.head_dim, t, cfg.rope_theta))
    late = torch.ones(t, t, dtype=torch.bool, device=ids.device).triu(1)
    x = p["embeddings.weight"][ids]
    for i in range(cfg.n_layer):
        w = {k.split(f"layers.{i}.")[1]: v for k, v in p.items() if k.startswith(f"layers.{i}.")}
        h = norm(x, w["attn_norm.weight"])
        q, k, v = ((h @ w[f"attention.{n}.weight"].t()).view(1, t, -1, cfg.head_dim) for n in ("wq", "wk", "wv"))
        q, k = (y[0] for y in apply_rotary_emb(q, k, cos, sin))
        g = cfg.num_queries_per_kv
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(g, 1)) / 8
        a = torch.softmax(s.masked_fill(late, -float("inf")), -1)
        o = torch.einsum("hij,jhd->ihd", a, v[0].repeat_interleave(g, 1)).reshape(t, -1)
        x = x + o @ w["attention.wo.weight"].t()
        h = norm(x, w["ffn_norm.weight"])
        x = x + (F.silu(h @ w["ffn.w_gate.weight"].t()) * (h @ w["ffn.w_up.weight"].t())) @ w["ffn.w_down.weight"].t()
    return norm(x, p["final_norm.weight"]) @ p["embeddings.weight"].t()


def params(m):
    return {k: v.detach().double().requires_grad_() for k, v in m.named_parameters()}


def tokens(dev, n, seed=0):
    return torch.randint(0, 1000, (n,), generator=torch.Generator(device=dev).manual_seed(seed), device=dev)


def bounds(dev, lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu, torch.tensor(cu, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("page", [16, 64])
@torch.no_grad()
def test_prompts_then_decode_steps(dev, page):
    m = model(dev).eval()
    p = params(m)
    cu, dcu = bounds(dev, LENGTHS)
    ids = tokens(dev, cu[-1])
    caches = m.allocate_paged_caches(len(LENGTHS), 200, page_size=page)
    pages = caches[0].pages
    logits = m(ids[None], kv_caches=caches, cu_seqlens=dcu, lengths=LENGTHS)["logits"][0]
    seqs = [ids[a:b] for a, b in zip(cu, cu[1:])]
    for s, a in zip(seqs, cu):
        assert float((logits[a:a + len(s)] - plain(m, p, s)).abs().max()) < 2e-4
    assert pages.held == LENGTHS and pages.lens.tolist() == LENGTHS
    for step in range(4):
        new = tokens(dev, len(LENGTHS), 10 + step)
        lg = m(new[:, None], kv_caches=caches)["logits"][:, 0]
        seqs = [torch.cat([s, n[None]]) for s, n in zip(seqs, new)]
        for b, s in enumerate(seqs):
            assert float((lg[b] - plain(m, p, s)[-1]).abs().max()) < 2e-4, (step, b)
    ops.check_device_errors(dev)
    assert pages.held == [n + 4 for n in LENGTHS] == pages.lens.tolist()
    # a captured step: pages reserved ahead, lengths advanced on the device by the graph
    pages.reserve(8)
    feed = tokens(dev, len(LENGTHS), 20)[:, None].clone()
    held = list(pages.held)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(feed, kv_caches=caches)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    pages.lens.sub_(1)
    pages.held = list(held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = m(feed, kv_caches=caches)["logits"]
    pages.held = list(held)
    for step in range(3):
        feed.copy_(tokens(dev, len(LENGTHS), 30 + step)[:, None])
        graph.replay()
        pages.advance(1, device=False)
        seqs = [torch.cat([s, n]) for s, n in zip(seqs, feed)]
        for b, s in enumerate(seqs):
            assert float((kept[b, 0] - plain(m, p, s)[-1]).abs().max()) < 2e-4, (step, b)
    assert pages.held == pages.lens.tolist() == [n + 7 for n in LENGTHS]
    ops.check_device_errors(dev)


@torch.no_grad()
def test_batch_of_one_length_and_scores(dev):
    m = model(dev).eval()
    p = params(m)
    ids = tokens(dev, 2 * 90, 4).view(2, 90)
    targets = torch.cat([ids[:, 1:], torch.full((2, 1), -100, device=dev)], dim=1)
    got = m.score(ids, targets, top_k=3)
    caches = m.allocate_paged_caches(2, 128)
    cached = m(ids, kv_caches=caches)["logits"]
    for b in range(2):
        lp = torch.log_softmax(plain(m, p, ids[b]), -1)
        want = lp[:-1].gather(1, ids[b, 1:, None])[:, 0]
        assert float((got.logprobs.view(2, 90)[b, :-1] - want).abs().max()) < 2e-4
        assert got.logprobs.view(2, 90)[b, -1] == 0
        assert float((got.entropy.view(2, 90)[b] + (lp.exp() * lp).sum(-1)).abs().max()) < 4e-3
        assert float((got.top_logprobs.view(2, 90, 3)[b] - lp.topk(3).values).abs().max()) < 2e-4
        assert float((cached[b] - plain(m, p, ids[b])).abs().max()) < 2e-4
    nxt = m(ids[:, :1], kv_caches=caches)["logits"]
    for b in range(2):
        assert float((nxt[b, 0] - plain(m, p, torch.cat([ids[b], ids[b, :1]]))[-1]).abs().max()) < 2e-4


def test_training_step_over_packed_documents(dev):
    m = model(dev)
    p = params(m)
    cu, dcu = bounds(dev, LENGTHS)
    ids = tokens(dev, cu[-1], 5)
    targets = torch.cat([ids[1:], ids.new_full((1,), -100)])
    targets[[c - 1 for c in cu[1:]]] = -100  # no target across a document's end
    out = m(ids[None], targets=targets[None], cu_seqlens=dcu)
    out["loss"].backward()
    logits = torch.cat([plain(m, p, ids[a:b]) for a, b in zip(cu, cu[1:])])
    loss = F.cross_entropy(logits, targets, ignore_index=-100)
    names = [k for k in p if "forecast" not in k]
    want = dict(zip(names, torch.autograd.grad(loss, [p[k] for k in names])))
    assert abs(float(out["loss"]) - float(loss)) < 2e-5
    for name, w in m.named_parameters():
        if "forecast" in name:
            assert w.grad is None
            continue
        off = float((w.grad - want[name]).norm() / want[name].norm())
        assert off < 1e-3, (name, off)
    ops.check_device_errors(dev)


def test_bf16_training_step_runs_and_caches_refuse_gradients(dev):
    m = model(dev, torch.bfloat16)
    cu, dcu = bounds(dev, LENGTHS)
    ids = tokens(dev, cu[-1], 6)
    loss = m(ids[None], targets=ids[None], cu_seqlens=dcu)["loss"]
    loss.backward()
    assert all(torch.isfinite(w.grad).all() for n, w in m.named_parameters() if "forecast" not in n)
    caches = m.allocate_paged_caches(len(LENGTHS), 200)
    with pytest.raises(NotImplementedError, match="without a cache"):
        m(ids[None], kv_caches=caches, cu_seqlens=dcu, lengths=LENGTHS)
    with torch.no_grad():
        caches = m.allocate_paged_caches(len(LENGTHS), 200)
        with pytest.raises(ValueError, match="lengths"):
            m(ids[None], kv_caches=caches, cu_seqlens=dcu)
        m(ids[None], kv_caches=caches, cu_seqlens=dcu, lengths=LENGTHS)
        with pytest.raises(NotImplementedError, match="non-empty"):
            m(ids[None], kv_caches=caches, cu_seqlens=dcu, lengths=LENGTHS)
