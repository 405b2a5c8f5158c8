"""The range of fp16 in the gradients of packed attention: a sequence's gradients
do not depend on how large the output gradients of others are, and values of v
up to the type's own range leave dS = P (dO V^T - delta) inside it.

Bounds as in tests/test_gpu_packed.py, but for the step of dS.  fp16 holds dS
scaled by a power of two per row (of queries in dQ, of keys in dK) that takes
64 max|dout| max|v| + max|delta| over the pairs of that row's own into
(2^14, 2^15], so a rounding is off by half a step relative, or by 2^-25 at the
least, which is 2^-25 2^-14 of that sum, absolute.  |delta| is at most
64 max|dout| max|v| (1 + 2^-9: out as rounded), so 2^-32 (1 + 2^-8) times
max|dout| max|v|.  The other types have fp32's exponents: nothing to scale.
Needs a B200."""

import math

import pytest
import torch

from local_research_small_language_model_b200 import ops
from tests.test_gpu_packed import DTYPES, U, U32, bounds, check, inputs, run

pytestmark = pytest.mark.gpu


def exact(q, k, v, dout, scale=0.125, causal_step=False, tiny_p=None):
    """(out, dq, dk, dv) of one sequence and their bounds.  causal_step: the
    sum above over the pairs that a row sees, not over the whole sequence.
    tiny_p: fp16's least step of P in dV (2^-24 unless given)."""
    dtype, u = q.dtype, U[q.dtype]
    half = dtype == torch.float16
    tiny = 2.0 ** -24 if half else 0.0
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    n, group = q.shape[0], q.shape[1] // k.shape[1]
    val = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(k)}
    err = {x: torch.zeros_like(y) for x, y in val.items()}
    late = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
    step = 2.0 ** -32 * (1 + 2.0 ** -8) if half else 0.0
    heads = dout.abs().amax(2).view(n, -1, group).amax(2)  # [n, Hkv]: the group's largest |dout| a row
    for h in range(q.shape[1]):
        j = h // group
        qh, kh, vh, g = q[:, h], k[:, j], v[:, j], dout[:, h]
        s = (qh @ kh.t() * scale).masked_fill(late, -math.inf)
        p = torch.softmax(s, dim=-1)
        eps = 2 * (68 * U32 * float((qh.abs() @ kh.abs().t()).max()) * scale + 2.0 ** -21 + n * U32)
        o = p @ vh
        eo = (u + eps) * (p @ vh.abs()) + (tiny + 2.0 ** -126) * vh.abs().sum(0) + u * o.abs()
        val["out"][:, h], err["out"][:, h] = o, eo * (1 + u) + (2.0 ** -25 if half else 2.0 ** -126)
        delta = (g * o).sum(-1, keepdim=True)
        edelta = (g.abs() * eo).sum(-1, keepdim=True) + 64 * U32 * (g * o).abs().sum(-1, keepdim=True)
        ds = p * (g @ vh.t() - delta)
        none = 2.0 ** -126 * ((g.abs() @ vh.abs().t()) + delta.abs() + edelta)
        eds = (u + eps) * ds.abs() + p * (65 * U32 * (g.abs() @ vh.abs().t()) + edelta) + none * ~late
        big_g, big_v = g.abs().amax(1), vh.abs().amax(1)
        if causal_step:  # dQ: the row's own |dout|, the v it sees; dK: its own |v| and delta of the rows that see it
            seen_v = big_v.cummax(0).values
            mq = (big_g * seen_v)[:, None]
            seen_g = heads[:, j].flip(0).cummax(0).values.flip(0)
            seen_gv = (heads[:, j] * seen_v).flip(0).cummax(0).values.flip(0)
            mk = ((seen_g * big_v + seen_gv) / 2)[None, :]
        else:
            mq = mk = (heads[:, j].max() * big_v.max()).expand(1, 1)
        ep = (u + eps) * p + ((tiny if tiny_p is None else tiny_p) + 2.0 ** -126) * ~late
        val["dq"][:, h] = ds @ kh * scale
        err["dq"][:, h] = scale * ((eds + step * mq * ~late + n * U32 * ds.abs()) @ kh.abs())
        val["dk"][:, j] += ds.t() @ qh * scale
        err["dk"][:, j] += scale * ((eds + step * mk * ~late + group * n * U32 * ds.abs()).t() @ qh.abs())
        val["dv"][:, j] += p.t() @ g
        err["dv"][:, j] += (ep + group * n * U32 * p).t() @ g.abs()
    least = 2.0 ** -25 if half else 2.0 ** -126
    for x in ("dq", "dk", "dv"):
        err[x] += u * (val[x].abs() + err[x]) + least
    return val, err


def check_all(got, val, err, what):
    for x, y in zip(("out", "dq", "dk", "dv"), got):
        check(y, val[x], err[x], f"{what} {x}")


@pytest.mark.parametrize("heads", [(12, 4), (2, 2)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_a_sequence_does_not_depend_on_its_neighbours_loss(dev, dtype, heads):
    """Output gradients 2^14 apart in two packed sequences: each has the bounds
    of its own, and in 16 bits the bits it has alone (in fp32 the number of
    tiles decides how many CTAs share one, and so the order of its sums)."""
    cu = bounds([300, 500])
    q, k, v, dout = inputs(dev, dtype, 800, *heads, seed=41)
    dout = dout.clone()
    dout[:300] *= 64.0
    dout[300:] *= 2.0 ** -8
    got = run(q, k, v, dout, torch.tensor(cu, dtype=torch.int32, device=dev))
    ops.check_device_errors(dev)
    for a, b in zip(cu, cu[1:]):
        part = [x[a:b] for x in (q, k, v, dout)]
        val, err = exact(*part)
        check_all([x[a:b] for x in got], val, err, f"rows {a}")
        if dtype != torch.float32:
            alone = run(*part, torch.tensor([0, b - a], dtype=torch.int32, device=dev))
            for x, y in zip(got, alone):
                assert torch.equal(x[a:b], y)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_a_key_depends_on_what_sees_it(dev, dtype):
    """One sequence whose first tokens have output gradients (or values of v)
    thousands of times the rest's: keys and queries that are in no pair with
    them keep the bounds of the pairs that they are in."""
    cu = torch.tensor([0, 450], dtype=torch.int32, device=dev)
    for what in ("dout", "v"):
        q, k, v, dout = (x.clone() for x in inputs(dev, dtype, 450, 6, 2, seed=42))
        if what == "dout":
            dout *= 2.0 ** -8
            dout[:5] *= 2.0 ** 13
        else:
            v *= 2.0 ** -4
            v[440:] *= 2.0 ** 12
        got = run(q, k, v, dout, cu)
        val, err = exact(q, k, v, dout, causal_step=True)
        check_all(got, val, err, what)


@pytest.mark.parametrize("size", [4000.0, 30000.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_large_values(dev, dtype, size):
    """Values of v in the thousands, in one head of one size with a sign a token
    (so that dout.v adds up over the columns and differs between the tokens):
    dS passes 65504 unless its scale takes v into account."""
    lengths = [200, 330]
    cu = bounds(lengths)
    q, k, v, dout = inputs(dev, dtype, 530, 6, 2, seed=43)
    v = (v.float().clamp(-2, 2) * size).to(dtype)
    v[:, 1] = torch.where(v[:, 1, :1] > 0, size, -size).to(dtype)
    dout = (dout.float().clamp(-3, 3) / 4).to(dtype)
    dout[:, 3:] = 0.75
    # queries and keys so small that the gradients stay in fp16's range
    k = (k.float() / 64).to(dtype)
    q = (q.float() / 64).to(dtype)
    got = run(q, k, v, dout, torch.tensor(cu, dtype=torch.int32, device=dev))
    for a, b in zip(cu, cu[1:]):
        val, err = exact(*(x[a:b] for x in (q, k, v, dout)))
        assert max(float(x.abs().max()) for x in val.values()) <= 60000.0
        check_all([x[a:b] for x in got], val, err, f"rows {a}")


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_keys_that_get_little_weight(dev, dtype):
    """Keys whose every weight is far below fp16's smallest normal number, 2^-14:
    their dV keeps its digits.  fp16 holds P scaled by 2^15, so a rounding is off
    by half a step relative, or by 2^-40 at the least."""
    n = 400
    q, k, v, dout = inputs(dev, dtype, n, 4, 2, seed=44, scale_out=512.0)
    q, k = q.clone(), k.clone()
    q[..., 0], k[..., 0] = 8.0, 0.0
    few = torch.arange(n, device=dev) % 3 == 1
    k[few, :, 0] = -12.0  # scores lower by 12: e^-12 / n
    got = run(q, k, v, dout, torch.tensor([0, n], dtype=torch.int32, device=dev))
    val, err = exact(q, k, v, dout, tiny_p=2.0 ** -40 if dtype == torch.float16 else 0.0)
    check_all(got, val, err, "little weight")
    assert float(val["dv"][few].abs().max()) < 0.1 < float(val["dv"].abs().max())  # the case is what it says
