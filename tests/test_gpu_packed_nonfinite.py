"""Packed attention over values that are not finite: rows before them keep their
bounds, and no such value makes a call many times slower.  Needs a B200."""

import math

import pytest
import torch

from local_research_small_language_model_b200 import ops
from tests.test_gpu_packed import DTYPES, bounds, check, exact, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("shift", [0, 40])
def test_values_that_are_not_finite_in_many_columns(dev, dtype, shift):
    """NaN and infinities of v in many tokens and columns, some columns with one
    early and one late: a result is finite, and within its bound, exactly where
    no token up to the row's own has such a value in that column."""
    cu = bounds([150 + shift, 700])
    total = cu[-1]
    q, k, v, dout = inputs(dev, dtype, total, 4, 2, seed=51)
    val, err = exact(q, k, v, dout, cu, 0.125)
    v = v.clone()
    g = torch.Generator(device=dev).manual_seed(shift)
    for i, bad in enumerate((math.nan, math.inf, -math.inf, math.nan) * 10):
        token = int(torch.randint(0, total, (1,), generator=g, device=dev))
        first = int(torch.randint(0, 60, (1,), generator=g, device=dev))
        v[token, i % 2, first:first + 1 + i % 5] = bad
    for token in (cu[1] + 127, cu[1] + 128, cu[1] + 255, cu[1] + 699, cu[1] - 1):
        v[token, 0, 61] = math.inf
    reached = torch.zeros_like(v, dtype=torch.bool)
    for a, b in zip(cu, cu[1:]):
        reached[a:b] = (~torch.isfinite(v[a:b])).cumsum(0) > 0
    got, lse = ops.packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), return_lse=True)
    reached = reached.repeat_interleave(2, 1)
    assert not torch.isfinite(got[reached]).any()
    assert torch.isfinite(lse).all()
    err["out"][reached] = math.inf
    check(torch.where(reached, torch.zeros_like(got), got), val["out"], err["out"], "out")


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("where", ["first_token", "everywhere", "queries", "every_tile"])
def test_values_that_are_not_finite_take_no_longer(dev, dtype, where):
    """8192 tokens: an overflow somewhere costs at most a few times the call, not
    the hundreds of a row-by-row evaluation."""
    q, k, v, _ = (x.clone() for x in inputs(dev, dtype, 8192, 4, 2, seed=52))
    cu = torch.tensor([0, 8192], dtype=torch.int32, device=dev)

    def call():
        ops.packed_attention(q, k, v, cu)

    def best():
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            call()
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    call()
    clean = best()
    if where == "first_token":
        v[0] = math.nan
    elif where == "everywhere":
        v.fill_(math.nan)
    elif where == "queries":
        q.fill_(math.nan)
    else:
        v[7] = math.inf
        v[127::128] = math.inf
    assert best() < 6 * clean + 0.1
    assert not torch.isfinite(ops.packed_attention(q, k, v, cu)[8:]).any()
