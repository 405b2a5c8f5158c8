"""Causal attention over packed sequences (sd_packed_attention and its
backward) against the formulas in 64 bits.

Bounds, per element, from the arithmetic.  u is half a step of the type (the
largest relative error of one rounding), u32 = 2^-24.
  scores: 64 fp32 additions of products, a scaling and the subtraction of the
    reference maximum, then an exponential good to 2^-21: a weight p is off by
    at most the factor 1 + eps, eps = 2 (68 u32 max sum|q k| scale + 2^-21 +
    n u32), the last term for the n-fold sum in the denominator and the first
    factor for numerator and denominator.
  out: weights are rounded to the type once (fp16 also to a multiple of 2^-24),
    sums are fp32, the result is rounded once:
    (u + eps) sum p|v| + 2^-24 sum|v| [fp16] + u |out|.
  delta = dout.out takes out as stored: off by sum |dout| (error of out) +
    64 u32 sum |dout out|.
  dS = p (dout.v - delta): eps |dS| + p (65 u32 sum|dout v| + error of delta),
    and one rounding u |dS|; fp16 holds dS scaled by a power of two that takes
    the largest |dout| below 1, so its smallest step adds 2^-24 max|dout|.
  Weights below 2^-126, fp32's smallest normal number, may be taken as zero:
    an absolute 2^-126 on every weight (times |dout.v| + |delta| on dS), and
    the same least step on a result.
  dv, dq, dk: the sums of those errors with |dout|, |k|, |q|, n u32 for their
    own sums, and one rounding.
Needs a B200."""

import math

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
U32 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HEADS = [(12, 4), (4, 4), (8, 1)]
LENGTHS = {
    "one": [1],
    "two": [2, 1, 0, 3],
    "tile": [64, 128],
    "off_tile": [63, 65, 127, 129],
    "ragged": [300, 1, 0, 77, 513, 2],
    "long": [1100],
    "many": [5] * 70 + [0] * 7 + [40],
    "crowd": [3, 0, 130] * 60,
}


def bounds(lengths, lead=0):
    cu = [lead]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def inputs(dev, dtype, total, hq, hkv, seed=0, scale_out=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = torch.randn(total, (hq + 2 * hkv), 64, generator=g, device=dev).to(dtype)
    dout = (torch.randn(total, hq, 64, generator=g, device=dev) * scale_out).to(dtype)
    return rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], dout


def exact(q, k, v, dout, cu, scale):
    """Values and error bounds of out, dq, dk, dv; rows outside every sequence 0."""
    dtype, u = q.dtype, U[q.dtype]
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    group = q.shape[1] // k.shape[1]
    names = ("out", "dq", "dk", "dv")
    val = {x: torch.zeros_like(k if x in ("dk", "dv") else q) for x in names}
    err = {x: torch.zeros_like(val[x]) for x in names}
    top = float(dout.abs().max()) if dout.numel() else 0.0
    for a, b in zip(cu, cu[1:]):
        n = b - a
        if n == 0:
            continue
        late = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(q.shape[1]):
            j = h // group
            qh, kh, vh, g = q[a:b, h], k[a:b, j], v[a:b, j], dout[a:b, h]
            s = (qh @ kh.t() * scale).masked_fill(late, -math.inf)
            p = torch.softmax(s, dim=-1)
            big = float((qh.abs() @ kh.abs().t()).max()) * scale
            eps = 2 * (68 * U32 * big + 2.0 ** -21 + n * U32)
            o = p @ vh
            eo = (u + eps) * (p @ vh.abs()) + (tiny + 2.0 ** -126) * vh.abs().sum(0) + u * o.abs()
            val["out"][a:b, h], err["out"][a:b, h] = o, eo
            delta = (g * o).sum(-1, keepdim=True)
            edelta = (g.abs() * eo).sum(-1, keepdim=True) + 64 * U32 * (g * o).abs().sum(-1, keepdim=True)
            ds = p * (g @ vh.t() - delta)
            eds = (u + eps) * ds.abs() + p * (65 * U32 * (g.abs() @ vh.abs().t()) + edelta)
            none = 2.0 ** -126 * ((g.abs() @ vh.abs().t()) + delta.abs() + edelta)
            eds = eds + (tiny * top + none) * ~late
            ep = (u + eps) * p + (tiny + 2.0 ** -126) * ~late
            val["dq"][a:b, h] = ds @ kh * scale
            err["dq"][a:b, h] = scale * ((eds + n * U32 * ds.abs()) @ kh.abs())
            val["dk"][a:b, j] += ds.t() @ qh * scale
            err["dk"][a:b, j] += scale * ((eds + group * n * U32 * ds.abs()).t() @ qh.abs())
            val["dv"][a:b, j] += p.t() @ g
            err["dv"][a:b, j] += (ep + group * n * U32 * p).t() @ g.abs()
    # one rounding of the gradients (fp16: at least its smallest step)
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    for x in names:
        if x != "out":
            err[x] += u * (val[x].abs() + err[x]) + least
        else:
            err[x] = err[x] * (1 + u) + least
    return val, err


def check(got, val, err, what):
    off = (got.double() - val).abs()
    bad = ~(off <= err)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(off.max()):.3e}, "
                           f"first at {bad.nonzero()[0].tolist()}: off {float(off[bad][0]):.3e} bound "
                           f"{float(err[bad][0]):.3e}")


def run(q, k, v, dout, cu, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = sd.packed_attention(*leaves, cu, scale)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}to{h[1]}")
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_packed_attention_and_gradients(dev, dtype, heads, name):
    cu = bounds(LENGTHS[name])
    q, k, v, dout = inputs(dev, dtype, cu[-1], *heads, seed=len(name))
    dcu = torch.tensor(cu, dtype=torch.int32, device=dev)
    got = run(q, k, v, dout, dcu)
    ops.check_device_errors(dev)
    val, err = exact(q, k, v, dout, cu, 0.125)
    for x, y in zip(("out", "dq", "dk", "dv"), got):
        check(y, val[x], err[x], x)
    # the output's low bits: out and rest together are nearer (the weights' rounding remains); without them the
    # gradients hold the same bounds
    rest = torch.empty(q.shape, dtype=dtype, device=dev) if dtype != torch.float32 else None
    out, lse = ops.packed_attention(q, k, v, dcu, return_lse=True, rest=rest)
    assert torch.equal(out, got[0])
    if rest is not None:
        check(out.double() + rest.double(), val["out"], err["out"] - U[dtype] * val["out"].abs() * 0.9, "out + rest")
        for x, y in zip(("dq", "dk", "dv"), ops.packed_attention_backward(q, k, v, out, dout, lse, dcu)):
            check(y, val[x], err[x], x + " without rest")
    # without autograd, and again: the same bits
    assert torch.equal(sd.packed_attention(q, k, v, dcu), got[0])
    for x, y in zip(got, run(q, k, v, dout, dcu)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_rows_outside_every_sequence(dev, dtype):
    """Rows before the first and behind the last sequence: zero in new outputs
    and gradients, left as they were in a caller's out; NaN there reaches no
    sequence, nor does one sequence's NaN reach another."""
    cu = bounds([70, 0, 131], lead=9)
    total = cu[-1] + 85
    q, k, v, dout = inputs(dev, dtype, total, 4, 2, seed=3)
    rest = torch.ones(total, dtype=torch.bool, device=dev)
    rest[cu[0]:cu[-1]] = False
    clean = run(q, k, v, dout, torch.tensor(cu, device=dev, dtype=torch.int32))
    val, err = exact(q, k, v, dout, cu, 0.125)
    for x, y in zip(("out", "dq", "dk", "dv"), clean):
        check(y, val[x], err[x], x)
        assert not y[rest].any()
    bad = [x.clone() for x in (q, k, v, dout)]
    for i, x in enumerate(bad):
        x[rest] = math.nan if i % 2 else math.inf
    for x, y in zip(run(*bad, torch.tensor(cu, device=dev, dtype=torch.int32)), clean):
        assert torch.equal(x, y)
    for x in bad:
        x[cu[1]:cu[2]] = math.nan
        x[:cu[0] + 70] = math.inf
    for x, y in zip(run(*bad, torch.tensor(cu, device=dev, dtype=torch.int32)), clean):
        assert torch.equal(x[cu[2]:], y[cu[2]:])
    out = torch.full((total, 4, 64), 7.0, dtype=dtype, device=dev)
    ops.packed_attention(q, k, v, torch.tensor(cu, device=dev, dtype=torch.int32), out=out)
    assert torch.equal(out[~rest], clean[0][~rest]) and (out[rest] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_later_tokens_do_not_show(dev, dtype, bad):
    """A NaN or an infinity in k or v of a later token of the same sequence, in
    the same tile or another, changes no bound of the rows before it; the rows
    from it on are what the formula makes of it."""
    cu = bounds([70, 300])
    dcu = torch.tensor(cu, dtype=torch.int32, device=dev)
    for token in (71, 70 + 130, 70 + 299):
        q, k, v, dout = inputs(dev, dtype, 370, 4, 2, seed=21)
        val, err = exact(q, k, v, dout, cu, 0.125)
        for kind in ("k", "v"):
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            (k2 if kind == "k" else v2)[token, 1, 5] = bad
            got = ops.packed_attention(q2, k2, v2, dcu)
            check(got[:token], val["out"][:token], err["out"][:token], f"{kind} {token}")
            assert torch.isfinite(got[:, :2]).all()  # the other kv head's rows
            if kind == "v":
                seen = got[token:, 2:, 5].double()
                assert (seen.isnan() if math.isnan(bad) else (seen == bad) | seen.isnan()).all()
                keep = [c for c in range(64) if c != 5]
                check(got[token:, 2:][..., keep], val["out"][token:, 2:][..., keep], err["out"][token:, 2:][..., keep], "v")


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_rows_whose_first_scores_are_infinite(dev, dtype):
    """Keys with a score of -inf weigh nothing, also where a whole first block
    has no other; a row that sees nothing else is NaN, as softmax of -inf is."""
    q, k, v, dout = inputs(dev, dtype, 260, 2, 2, seed=22)
    q = (q.abs() + 0.5).to(dtype)
    k = k.clone()
    k[:150] = -math.inf
    got, lse = ops.packed_attention(q, k, v, torch.tensor([0, 260], dtype=torch.int32, device=dev), return_lse=True)
    val, err = exact(q[150:], k[150:], v[150:], dout[150:], [0, 110], 0.125)
    check(got[150:], val["out"], err["out"], "out")
    assert got[:150].isnan().all() and torch.isfinite(lse[:, 150:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_strides_views_and_broadcast(dev, dtype):
    """Head-major storage, an unaligned base, an int64 cu, and k and v shared by
    expanding one head: the gradient of the one head is the heads' sum."""
    cu = bounds([40, 100])
    dcu = torch.tensor(cu, device=dev)  # int64
    q, k, v, dout = inputs(dev, dtype, 140, 4, 4, seed=5)
    want = run(q, k, v, dout, dcu)
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, dout)]
    for x, y in zip(run(*hm, dcu), want):
        assert torch.equal(x, y)
    odd = []
    for x in (q, k, v, dout):
        flat = torch.empty(x.numel() + 1, dtype=dtype, device=dev)[1:]
        odd.append(flat.view(x.shape).copy_(x))
    for x, y in zip(run(*odd, dcu), want):
        assert torch.equal(x, y)
    one_k, one_v = k[:, :1].clone().requires_grad_(), v[:, :1].clone().requires_grad_()
    out = sd.packed_attention(q, one_k.expand(-1, 4, -1), one_v.expand(-1, 4, -1), dcu)
    gk, gv = torch.autograd.grad(out, (one_k, one_v), dout)
    val, err = exact(q, one_k.detach(), one_v.detach(), dout, cu, 0.125)
    check(out.detach(), val["out"], err["out"], "out")
    # each head's gradient is rounded before autograd's sum rounds again
    per = run(q, k[:, :1].expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1), dout, dcu)
    for got, x, y in ((gk, "dk", per[2]), (gv, "dv", per[3])):
        check(got, val[x], err[x] + 4 * U[dtype] * y.double().abs().sum(1, keepdim=True), x)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("scale_out", [1e-5, 300.0])
def test_gradients_of_small_and_large_losses(dev, dtype, scale_out):
    """A loss averaged over many tokens has output gradients near fp16's
    smallest values: the gradients keep their digits."""
    cu = bounds([200, 90])
    q, k, v, dout = inputs(dev, dtype, 290, 6, 2, seed=8, scale_out=scale_out)
    got = run(q, k, v, dout, torch.tensor(cu, device=dev, dtype=torch.int32), 0.2)
    val, err = exact(q, k, v, dout, cu, 0.2)
    for x, y in zip(("out", "dq", "dk", "dv"), got):
        check(y, val[x], err[x], x)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_large_scores(dev, dtype):
    """Scores of several hundred, rising along the keys (the running maximum
    moves at every tile) and falling."""
    for sign in (1.0, -1.0):
        q, k, v, dout = inputs(dev, dtype, 400, 4, 4, seed=9)
        ramp = torch.linspace(0.5, 12.0, 400, device=dev)[:, None, None]
        k = (k.abs() * ramp * sign).to(dtype)
        q = (q.abs() + 1).to(dtype)
        got = run(q, k, v, dout, torch.tensor([0, 400], device=dev, dtype=torch.int32))
        val, err = exact(q, k, v, dout, [0, 400], 0.125)
        for x, y in zip(("out", "dq", "dk", "dv"), got):
            check(y, val[x], err[x], x)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_gradients_against_differences(dev, dtype):
    """The gradients against central differences of the formula in 64 bits along
    random directions, which shares nothing with the backward's formulas."""
    cu = bounds([33, 50])
    q, k, v, dout = inputs(dev, dtype, 83, 4, 2, seed=11)
    _, dq, dk, dv = run(q, k, v, dout, torch.tensor(cu, device=dev, dtype=torch.int32))
    val, err = exact(q, k, v, dout, cu, 0.125)

    def loss(*x):
        return float((exact_out(*x, cu) * dout.double()).sum())

    g = torch.Generator(device=dev).manual_seed(1)
    for i, (got, name) in enumerate(((dq, "dq"), (dk, "dk"), (dv, "dv"))):
        x = [y.double() for y in (q, k, v)]
        step = torch.randn(x[i].shape, generator=g, device=dev, dtype=torch.float64) * 1e-4
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + step, x[i] - step
        slope = (loss(*up) - loss(*down)) / 2
        # the directional derivative: the gradient's bound along the step, and the third-order term
        room = float((err[name] * step.abs()).sum()) + 1e-6 * float(step.abs().sum())
        assert abs(float((got.double() * step).sum()) - slope) <= room, name


def exact_out(q, k, v, cu):
    group = q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    for a, b in zip(cu, cu[1:]):
        late = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1)
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(group, 1)) * 0.125
        p = torch.softmax(s.masked_fill(late, -math.inf), dim=-1)
        out[a:b] = torch.einsum("hij,jhd->ihd", p, v[a:b].repeat_interleave(group, 1))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
def test_streams_and_graph_replay(dev, dtype):
    """Forward and backward captured into a CUDA graph follow new inputs and new
    bounds on replay; two streams at once give the eager bits."""
    q, k, v, dout = (x.clone() for x in inputs(dev, dtype, 300, 4, 2, seed=12))
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=dev)

    def both():
        out, lse = ops.packed_attention(q, k, v, cu, return_lse=True)
        return (out, *ops.packed_attention_backward(q, k, v, out, dout, lse, cu))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    graph.replay()
    for x, y in zip(kept, first):
        assert torch.equal(x, y)
    q2, k2, v2, g2 = inputs(dev, dtype, 300, 4, 2, seed=13)
    for x, y in ((q, q2), (k, k2), (v, v2), (dout, g2), (cu, torch.tensor([0, 257, 300], device=dev))):
        x.copy_(y)
    graph.replay()
    want = both()
    for x, y in zip(kept, want):
        assert torch.equal(x, y)
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([both() for _ in range(3)])
    torch.cuda.synchronize()
    for runs in outs:
        for r in runs:
            for x, y in zip(r, want):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("lengths", [[1], [700, 5, 40], [2500], [90] * 12], ids=["one", "mixed", "long", "equal"])
def test_what_follows_the_backward_waits_for_all_of_it(dev, dtype, lengths):
    """Inputs overwritten and gradients read right behind the call on its stream,
    and calls one behind the other, give the bits of calls that stand alone."""
    total = sum(lengths)
    cu = torch.tensor(bounds(lengths), dtype=torch.int32, device=dev)
    sets = [inputs(dev, dtype, total, 12, 4, seed=20 + i) for i in range(3)]
    want = []
    for q, k, v, dout in sets:
        out, lse = ops.packed_attention(q, k, v, cu, return_lse=True)
        torch.cuda.synchronize()
        want.append(ops.packed_attention_backward(q, k, v, out, dout, lse, cu))
        torch.cuda.synchronize()
    got = []
    for q, k, v, dout in sets:
        q, k, v, dout = (x.clone() for x in (q, k, v, dout))
        out, lse = ops.packed_attention(q, k, v, cu, return_lse=True)
        grads = ops.packed_attention_backward(q, k, v, out, dout, lse, cu)
        for x in (q, k, v, dout, out, lse):
            x.fill_(7.0)
        copies = [x.clone() for x in grads]
        for x in grads:
            x.fill_(7.0)
        got.append(copies)
    for g, w in zip(got, want):
        for x, y in zip(g, w):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t)[6:])
def test_gradients_outside_the_sequences_do_not_count(dev, dtype):
    """dout's rows outside every sequence change no bit of a gradient, be they
    large (they take no part in fp16's common scale), infinite or NaN."""
    total, cu = 200, torch.tensor([40, 130, 170], dtype=torch.int32, device=dev)
    q, k, v, dout = inputs(dev, dtype, total, 4, 2, seed=31)
    out, lse = ops.packed_attention(q, k, v, cu, return_lse=True)
    want = ops.packed_attention_backward(q, k, v, out, dout, lse, cu)
    for bad in (3.0e4, math.inf, math.nan):
        other = dout.clone()
        other[:40] = bad
        other[170:] = bad
        got = ops.packed_attention_backward(q, k, v, out, other, lse, cu)
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_malformed_bounds_stay_inside(dev):
    """Bounds that descend or leave the rows give wrong rows, not faults: the
    memory around the output is untouched."""
    for dtype in DTYPES:
        q, k, v, dout = inputs(dev, dtype, 200, 4, 2, seed=14)
        pool = torch.full((600, 4, 64), 3.0, dtype=dtype, device=dev)
        for cu in ([0, 500], [-70, 90, 200], [0, 150, 60, 200], [190, 10, 300]):
            dcu = torch.tensor(cu, dtype=torch.int32, device=dev)
            ops.packed_attention(q, k, v, dcu, out=pool[200:400])
            out, lse = ops.packed_attention(q, k, v, dcu, return_lse=True)
            ops.packed_attention_backward(q, k, v, out, dout, torch.zeros_like(lse), dcu)
            torch.cuda.synchronize()
            assert (pool[:200] == 3.0).all() and (pool[400:] == 3.0).all()
