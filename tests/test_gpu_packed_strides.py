"""Calls of one row, one head or one page whose stride in that direction means
nothing: any value of it is the same call.  Needs a B200."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from tests.test_gpu_packed import DTYPES, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride", [0, 3, 1021])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_strides_of_single_rows_heads_and_pages(dev, dtype, stride):
    q, k, v, dout = (x.contiguous() for x in inputs(dev, dtype, 1, 4, 2, seed=61))
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)

    def odd(x, dim):
        st = list(x.stride())
        st[dim] = stride
        return x.as_strided(x.shape, st)

    for x, y in zip(run(*(odd(x, 0) for x in (q, k, v, dout)), cu), run(q, k, v, dout, cu)):
        assert torch.equal(x, y)
    out = torch.zeros_like(q)
    assert ops.packed_attention(q, k, v, cu, out=odd(out, 0)).data_ptr() == out.data_ptr()
    assert torch.equal(out, ops.packed_attention(q, k, v, cu))
    # one kv head over many rows
    q, k, v, dout = (x.contiguous() for x in inputs(dev, dtype, 90, 1, 1, seed=62))
    cu = torch.tensor([0, 50, 90], dtype=torch.int32, device=dev)
    for x, y in zip(run(*(odd(x, 1) for x in (q, k, v, dout)), cu), run(q, k, v, dout, cu)):
        assert torch.equal(x, y)
    # one page, one kv head, one sequence
    pk, pv = (torch.randn(1, 1, 16, 64, device=dev).to(dtype) for _ in range(2))
    row = torch.randn(1, 1, 64, device=dev).to(dtype)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.full((1,), 9, dtype=torch.int32, device=dev)
    want_k, want_v = pk.clone(), pv.clone()
    want_k[0, :, 9], want_v[0, :, 9] = row[0], row[0]
    for dim in (0, 1):
        a, b = pk.clone(), pv.clone()
        sd.paged_append(odd(row, 0), odd(row, 1), odd(a, dim), odd(b, dim), table, lens)
        assert torch.equal(a, want_k) and torch.equal(b, want_v)
        got = sd.paged_decode_attention(odd(row, dim), odd(a, dim), odd(b, dim), odd(table, 0), lens + 1)
        assert torch.equal(got, sd.paged_decode_attention(row, a, b, table, lens + 1))
        out = torch.zeros_like(row)
        sd.paged_decode_attention(row, a, b, table, lens + 1, out=odd(out, dim))
        assert torch.equal(out, got)
    ops.check_device_errors(dev)
