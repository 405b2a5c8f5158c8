"""token_logprobs and its gradient against log_softmax in 64 bits.

Bounds (u32 = 2^-24, u half a step of the logits' type).  With m the maximum
and n = V: each exponential is good to a few 2^-23 and its argument x - m to
u32 |x - m| (at most 104 where it matters: beyond, exp is 0 in fp32), so
s = sum exp(x - m) is off by the factor 1 + eps, eps = 2^-20 + 104 u32 +
(n / 256 + 16) u32 (256 or more running sums, then a tree), and
  logprob = (x - m) - log s: eps + 4 u32 (|x - m| + log n);
  entropy = log s - w / s with w = sum exp(x - m) (x - m): eps + eps (E|x - m|)
    + 4 u32 (log n + 1), E the mean under p;
  gradient: p is off by the factor 1 + 2 eps + u32 (|x - m| + log n) * 4, the
    entropy part also by the error of (log p + H); one rounding to the type.
Needs a B200."""

import math

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U32 = 2.0 ** -24


def make(dev, dtype, rows, vocab, seed=0, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=dev) * spread).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g, device=dev)


def exact(x, targets):
    """(log probabilities of all tokens, the targets', entropy) and the bounds of the last two."""
    vocab = x.shape[1]
    xd = x.double()
    d = (xd - xd.max(-1, keepdim=True).values)
    lp = torch.log_softmax(xd, dim=-1)
    p = lp.exp()
    eps = 2.0 ** -20 + 104 * U32 + (vocab / 256 + 16) * U32
    at = targets.clamp(0, vocab - 1)[:, None]
    away = torch.where(p > 0, d.abs().nan_to_num(posinf=0.0), 0.0)
    chosen = lp.gather(1, at)[:, 0]
    echosen = eps + 4 * U32 * (d.gather(1, at)[:, 0].abs() + math.log(vocab) + 1)
    mean = (p * away).sum(-1)
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    eh = eps * (1 + mean) + 4 * U32 * (math.log(vocab) + 1 + mean)
    return lp, chosen, echosen, h, eh, eps, away


def check(got, val, err, what):
    off = (got.double() - val).abs()
    bad = ~((off <= err) | (got.double() == val))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float(off[bad].max()):.3e}"


def same_order(got, x, k):
    """Best first, ties by lowest index: a stable descending sort."""
    want = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 7), (2, 63), (130, 257), (700, 1031), (64, 32000), (9, 32003), (3, 100001)],
                         ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_scores(dev, dtype, shape):
    x, t = make(dev, dtype, *shape, seed=shape[1])
    lp, chosen, echosen, h, eh, _, away = exact(x, t)
    for k in sorted({0, 1, min(8, shape[1]), min(64, shape[1])}):
        got = sd.token_logprobs(x, t, top_k=k)
        check(got.logprobs, chosen, echosen, "logprobs")
        check(got.entropy, h, eh, "entropy")
        assert got.top_ids.shape == (shape[0], k)
        if k:
            same_order(got.top_ids, x, k)
            check(got.top_logprobs, lp.gather(1, got.top_ids), echosen.max(), "top_logprobs")
    ops.check_device_errors(dev)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_ties_and_signed_zeros(dev, dtype):
    """Equal logits go to the lowest index, -0 equals +0."""
    x = torch.zeros(4, 5000, dtype=dtype, device=dev)
    x[0, ::2] = -0.0
    x[1] = 1.5
    x[2, 4000:] = 2.0
    x[3] = torch.arange(5000, device=dev).remainder(3).to(dtype)
    got = sd.token_logprobs(x, torch.zeros(4, dtype=torch.int64, device=dev), top_k=40)
    assert torch.equal(got.top_ids[0], torch.arange(40, device=dev))
    assert torch.equal(got.top_ids[1], torch.arange(40, device=dev))
    assert torch.equal(got.top_ids[2], torch.arange(4000, 4040, device=dev))
    assert torch.equal(got.top_ids[3], torch.arange(2, 122, 3, device=dev))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_many_candidates(dev, dtype):
    """Rows that leave the quick search too much: thousands of equal values at
    the bound (also all of them: a masked vocabulary), and thousands of large
    values in a few threads' shares."""
    x, t = make(dev, dtype, 6, 32003, seed=12)
    x[0] = 0.25
    x[1, 7:] = -math.inf
    x[2, 100:] = -math.inf
    x[3, ::3] = 9.0
    x[4].clamp_(max=1.0)
    piece = torch.arange(32003, device=dev) // (16 // x.element_size())
    x[5] = x[5] * 0.01 + torch.where(piece % 512 < 200, 5.0, 0.0).to(dtype)
    for k in (1, 8, 63, 64):
        same_order(sd.token_logprobs(x, t, top_k=k).top_ids, x, k)
        same_order(sd.token_logprobs(x[:, 3:], t.clamp(max=100), top_k=k).top_ids, x[:, 3:], k)


def grads(x, t, g, ge):
    leaf = x.detach().requires_grad_()
    got = sd.token_logprobs(leaf, t)
    outs, weights = [], []
    for o, w in ((got.logprobs, g), (got.entropy, ge)):
        if w is not None:
            outs.append(o)
            weights.append(w)
    return torch.autograd.grad(outs, leaf, weights)[0]


def exact_grad(x, t, g, ge):
    u = torch.finfo(x.dtype).eps / 2
    lp, _, _, h, eh, eps, away = exact(x, t)
    p = lp.exp()
    kept = (t >= 0).double()
    rel = 2 * eps + 4 * U32 * (away + math.log(x.shape[1]))
    val = torch.zeros_like(lp)
    err = torch.zeros_like(lp)
    if g is not None:
        w = (g.double() * kept)[:, None]
        val -= w * p
        val.scatter_add_(1, t.clamp_min(0)[:, None], w)
        err += w.abs() * p * rel + U32 * (w.abs() * p + val.abs())
    if ge is not None:
        e = torch.where(p > 0, lp, 0.0) + h[:, None]
        val -= ge.double()[:, None] * p * e
        err += ge.double().abs()[:, None] * p * (rel * e.abs() + eh[:, None] + eps + 4 * U32 * (away + math.log(x.shape[1]) + 1))
    least = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -126
    return val, err * (1 + u) + u * val.abs() + 4 * U32 * val.abs() + least


@pytest.mark.parametrize("which", ["logprobs", "entropy", "both"])
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (130, 257), (700, 1031), (33, 32000), (9, 32003)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_gradient(dev, dtype, shape, which):
    x, t = make(dev, dtype, *shape, seed=shape[0])
    t[::4] = -100
    gen = torch.Generator(device=dev).manual_seed(9)
    g = torch.randn(shape[0], generator=gen, device=dev) if which != "entropy" else None
    ge = torch.randn(shape[0], generator=gen, device=dev) if which != "logprobs" else None
    d = grads(x, t, g, ge)
    assert d.dtype == dtype
    val, err = exact_grad(x, t, g, ge)
    check(d, val, err, "dlogits")
    assert torch.equal(d, grads(x, t, g, ge))


def test_gradient_against_differences(dev):
    x, t = make(dev, torch.float32, 6, 50, seed=3)
    t[2] = -100
    g = torch.linspace(-1, 2, 6, device=dev)
    ge = torch.linspace(0.5, -0.3, 6, device=dev)
    d = grads(x, t, g, ge)

    def loss(z):
        lp, chosen, _, h, _, _, _ = exact(z, t)
        return float((chosen * (t >= 0) * g.double()).sum() + (h * ge.double()).sum())

    step = torch.randn(6, 50, generator=torch.Generator(device=dev).manual_seed(1), device=dev,
                       dtype=torch.float64) * 1e-4
    slope = (loss(x.double() + step) - loss(x.double() - step)) / 2
    _, err = exact_grad(x, t, g, ge)
    assert abs(float((d.double() * step).sum()) - slope) <= float((err * step.abs()).sum()) + 1e-9


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_masked_infinite_and_nan_logits(dev, dtype):
    """-inf logits have probability 0 and zero gradient; a NaN, a +inf or a row
    of nothing but -inf makes its own row NaN, as log_softmax, and no other."""
    x, t = make(dev, dtype, 8, 700, seed=5)
    x[0, 10:690] = -math.inf
    t[0] = 5
    t[1] = 400
    x[1, 400] = -math.inf
    x[2] = -math.inf
    x[3, 77] = math.nan
    x[4, 78] = math.inf
    x[5, :699] = -math.inf
    t[5] = 699
    x[6] = torch.finfo(dtype).min
    ref = torch.log_softmax(x.double(), -1).gather(1, t[:, None])[:, 0]
    got = sd.token_logprobs(x, t, top_k=3)
    lp, chosen, echosen, h, eh, _, _ = exact(x, t)
    for r in (0, 5, 6, 7):
        check(got.logprobs[r:r + 1], chosen[r:r + 1], echosen[r:r + 1], "logprobs")
        check(got.entropy[r:r + 1], h[r:r + 1], eh[r:r + 1], "entropy")
    assert got.logprobs[1] == -math.inf and torch.isfinite(got.entropy[1])
    assert got.logprobs[2:5].isnan().all() and got.entropy[2:5].isnan().all() and ref[2:5].isnan().all()
    assert got.logprobs[5] == 0.0 and got.entropy[5] == 0.0
    assert torch.equal(got.top_ids[2], torch.arange(3, device=dev)) and got.top_ids[3, 0] == 77
    assert got.top_ids[4, 0] == 78 and got.top_ids[5].tolist() == [699, 0, 1]
    assert got.top_logprobs[5].tolist() == [0.0, -math.inf, -math.inf]
    ones = torch.ones(8, device=dev)
    d = grads(x, t, ones, ones)
    for r in (0, 1, 5, 6, 7):
        assert torch.isfinite(d[r]).all()
        assert not d[r][(x[r] == -math.inf) & (torch.arange(700, device=dev) != t[r])].any()
    assert d[2].isnan().any() and d[3].isnan().any() and d[4].isnan().any()


def test_ignored_and_bad_targets(dev):
    x, t = make(dev, torch.bfloat16, 6, 300, seed=6)
    t[1], t[3] = -100, 7
    got = sd.token_logprobs(x, t)
    assert got.logprobs[1] == 0.0
    ops.check_device_errors(dev)
    other = sd.token_logprobs(x, t, ignore_index=7)
    with pytest.raises(sd.SparDAError, match="error code 2"):
        ops.check_device_errors(dev)
    assert other.logprobs[3] == 0.0 and other.logprobs[1].isnan()
    for wrong in (300, -1, 2 ** 40):
        t[0] = wrong
        got = sd.token_logprobs(x, t)
        with pytest.raises(sd.SparDAError, match="error code 2"):
            ops.check_device_errors(dev)
        assert got.logprobs[0].isnan() and torch.isfinite(got.entropy).all()
        g = torch.ones(6, device=dev)
        d = grads(x, t, g, None)
        ops._err_bufs[dev.index or 0].zero_()
        assert not d[:2].any() and torch.isfinite(d).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_strides_shifts_and_streams(dev, dtype):
    """Row views of a wider tensor, odd offsets and transposes give the same
    values; large common offsets change nothing much; a graph replays."""
    x, t = make(dev, dtype, 20, 1001, seed=7)
    want = sd.token_logprobs(x, t, top_k=5)
    wide = torch.full((20, 1205), math.nan, dtype=dtype, device=dev)
    wide[:, 101:1102] = x
    wide_t = torch.zeros(20, 2, dtype=torch.int64, device=dev)
    wide_t[:, 1] = t
    for view in (wide[:, 101:1102], x.t().contiguous().t()):
        got = sd.token_logprobs(view, wide_t[:, 1], top_k=5)
        lp, chosen, echosen, h, eh, _, _ = exact(x, t)
        check(got.logprobs, chosen, echosen, "logprobs")
        check(got.entropy, h, eh, "entropy")
        assert torch.equal(got.top_ids, want.top_ids)
        d = grads(view, t, torch.ones(20, device=dev), None)
        check(d, *exact_grad(x, t, torch.ones(20, device=dev), None), "dlogits")
    far = (x.float() + 3000.0).to(dtype)
    got = sd.token_logprobs(far, t)
    lp, chosen, echosen, h, eh, _, _ = exact(far, t)
    check(got.logprobs, chosen, echosen, "logprobs")
    check(got.entropy, h, eh, "entropy")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = sd.token_logprobs(x, t, top_k=5)
    y, s = make(dev, dtype, 20, 1001, seed=8)
    x.copy_(y)
    t.copy_(s)
    graph.replay()
    for a, b in zip(kept, sd.token_logprobs(x, t, top_k=5)):
        assert torch.equal(a, b)


def test_rows_past_32_bits(dev):
    """More than 2^31 logits: the last rows are found, forward and backward."""
    rows, vocab = 67200, 32000
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=dev)
    tail, t_tail = make(dev, torch.bfloat16, 3, vocab, seed=10)
    x[-3:] = tail
    t = torch.zeros(rows, dtype=torch.int64, device=dev)
    t[-3:] = t_tail
    *found, stats = ops.token_logprobs(x, t, 4, return_stats=True)
    want = sd.token_logprobs(tail, t_tail, 4)
    for a, b in zip(found, want):
        assert torch.equal(a[-3:], b)
    d = ops.token_logprobs_backward(x, t, stats, torch.ones(rows, device=dev), None)
    assert torch.equal(d[-3:], grads(tail, t_tail, torch.ones(3, device=dev), None))
