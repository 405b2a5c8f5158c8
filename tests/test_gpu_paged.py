"""Paged key-value cache: the append moves rows bit for bit, and the attention
of one new token per sequence against the formula in 64 bits.

Bounds of the attention as in tests/test_gpu_packed.py: a weight is off by the
factor 1 + eps, eps = 2 (68 u32 max sum|q k| scale + 2^-21 + n u32), weights of
16-bit caches are rounded to the type once (u, half a step; fp16 also to a
multiple of 2^-24), the parts of a split cache are joined in fp32, and the
result is rounded once: (u + eps) sum p|v| + u |out|.  Needs a B200."""

import math

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U32 = 2.0 ** -24


def pool(dev, dtype, lens, hkv, page, seed=0, spare=3, width=None):
    """Scattered pages for sequences of the given lengths: (k_pages, v_pages, table)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(counts))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    k = torch.randn(pages, hkv, page, 64, generator=g, device=dev).to(dtype)
    v = torch.randn(pages, hkv, page, 64, generator=g, device=dev).to(dtype)
    return k, v, table


def exact(q, k_pages, v_pages, table, lens, scale=0.125):
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 0.0
    hkv, page = k_pages.shape[1:3]
    val = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(val)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = table[b, :-(-n // page)].long()
        k = k_pages[ids].double().transpose(0, 1).reshape(hkv, -1, 64)[:, :n]
        v = v_pages[ids].double().transpose(0, 1).reshape(hkv, -1, 64)[:, :n]
        qb = q[b].double().view(hkv, -1, 64)
        p = torch.softmax(qb @ k.transpose(1, 2) * scale, dim=-1)
        big = float((qb.abs() @ k.abs().transpose(1, 2)).max()) * scale
        eps = 2 * (68 * U32 * big + 2.0 ** -21 + n * U32)
        o = p @ v
        e = (u + eps) * (p @ v.abs()) + tiny * v.abs().sum(1, keepdim=True) + u * o.abs()
        val[b], err[b] = o.reshape(-1, 64), e.reshape(-1, 64) * (1 + u) + tiny
    return val, err


def check(got, val, err):
    off = (got.double() - val).abs()
    bad = ~(off <= err)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float(off.max()):.3e}, first at "
                           f"{bad.nonzero()[0].tolist()}")


def query(dev, dtype, b, hq, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(b, hq, 64, generator=g, device=dev).to(dtype)


BATCHES = {
    "one_token": [1],
    "empty_and_short": [0, 1, 2, 0, 63, 64, 65],
    "one_long": [5000],
    "ragged": [3000, 17, 0, 129, 1024, 700, 64, 1],
    "wide": [90 + 7 * i for i in range(70)],
}


@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("page", [1, 8, 24, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_decode_attention(dev, dtype, page, name):
    lens = BATCHES[name]
    k, v, table = pool(dev, dtype, lens, 4, page, seed=page)
    q = query(dev, dtype, len(lens), 12)
    dl = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = sd.paged_decode_attention(q, k, v, table, dl)
    ops.check_device_errors(dev)
    check(got, *exact(q, k, v, table, lens))
    assert torch.equal(got, sd.paged_decode_attention(q, k, v, table, dl))


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 1), (16, 1), (40, 2), (66, 2)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_head_groups(dev, dtype, heads):
    lens = [200, 0, 1500, 31]
    k, v, table = pool(dev, dtype, lens, heads[1], 32, seed=heads[0])
    q = query(dev, dtype, 4, heads[0])
    got = sd.paged_decode_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev), scale=0.3)
    check(got, *exact(q, k, v, table, lens, 0.3))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_layouts_and_hidden_places(dev, dtype):
    """Token-major pools, strided q, out and tables give the same bits; NaN and
    infinities behind a sequence's end and in unused pages do not show."""
    lens = [130, 0, 77, 900]
    k, v, table = pool(dev, dtype, lens, 4, 24, seed=2, width=60)
    q = query(dev, dtype, 4, 12)
    dl = torch.tensor(lens, dtype=torch.int64, device=dev)
    want = sd.paged_decode_attention(q, k, v, table, dl)
    tok = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    wide_q = torch.zeros(4, 30, 64, dtype=dtype, device=dev)
    wide_q[:, 3:15] = q
    room = torch.full((4, 20, 64), 5.0, dtype=dtype, device=dev)
    wide_t = torch.full((4, 99), -7, dtype=torch.int32, device=dev)
    wide_t[:, 9:69] = table
    got = sd.paged_decode_attention(wide_q[:, 3:15], *tok, wide_t[:, 9:69], dl, out=room[:, 4:16])
    assert torch.equal(got, want) and torch.equal(room[:, 4:16], want)
    assert (room[:, :4] == 5.0).all() and (room[:, 16:] == 5.0).all()
    used = torch.zeros(k.shape[0], 24, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for t in range(n):
            used[table[b, t // 24].long(), t % 24] = True
    for x, fill in ((k, math.nan), (v, math.inf)):
        x.masked_fill_(~used[:, None, :, None], fill)
    assert torch.equal(sd.paged_decode_attention(q, k, v, table, dl), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_bad_pages_and_lengths_are_reported(dev, dtype):
    """A page id outside the pool counts as absent, a length past the table is
    cut, and both are reported."""
    k, v, table = pool(dev, dtype, [100, 100], 4, 16, seed=3)
    q = query(dev, dtype, 2, 4)
    want = sd.paged_decode_attention(q, k, v, table, torch.tensor([100, 112], dtype=torch.int32, device=dev))
    ops.check_device_errors(dev)
    lens = torch.tensor([100, 5000], dtype=torch.int32, device=dev)
    assert torch.equal(sd.paged_decode_attention(q, k, v, table, lens), want)
    with pytest.raises(sd.SparDAError, match="error code 2"):
        ops.check_device_errors(dev)
    for wrong in (-1, k.shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[0, 2] = wrong
        got = sd.paged_decode_attention(q, k, v, bad, torch.tensor([100, 112], dtype=torch.int32, device=dev))
        with pytest.raises(sd.SparDAError, match="error code 2"):
            ops.check_device_errors(dev)
        assert torch.equal(got[1], want[1])
        keep = [t for t in range(100) if t // 16 != 2]
        pages = table[0].long()[torch.tensor(keep, device=dev) // 16]
        rows = torch.tensor(keep, device=dev) % 16
        one_k = k[pages, :, rows].transpose(0, 1)[None].contiguous()  # one page of the kept tokens
        one_v = v[pages, :, rows].transpose(0, 1)[None].contiguous()
        val, err = exact(q[:1], one_k, one_v, torch.zeros(1, 1, dtype=torch.int32, device=dev), [len(keep)])
        check(got[:1], val, err)
    negative = sd.paged_decode_attention(q, k, v, table, torch.tensor([-5, 112], dtype=torch.int32, device=dev))
    with pytest.raises(sd.SparDAError):
        ops.check_device_errors(dev)
    assert not negative[0].any()


@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_append(dev, dtype, page):
    """Packed prompts behind cached tokens, then one token each: every row at
    its place, everything else as it was."""
    before, new = [5, 0, 131, 64, 0], [70, 1, 0, 129, 3]
    held = [a + n + 1 for a, n in zip(before, new)]
    k, v, table = pool(dev, dtype, held, 4, page, seed=page + 1)
    wk, wv = k.clone(), v.clone()
    g = torch.Generator(device=dev).manual_seed(4)
    rows = torch.randn(sum(new) + 6, 8, 64, generator=g, device=dev).to(dtype)
    cu = [2]
    for n in new:
        cu.append(cu[-1] + n)
    lens = torch.tensor(before, dtype=torch.int32, device=dev)
    sd.paged_append(rows[:, :4], rows[:, 4:], k, v, table, lens, torch.tensor(cu, dtype=torch.int32, device=dev))
    for b, n in enumerate(new):
        for i in range(n):
            t = before[b] + i
            wk[table[b, t // page].long(), :, t % page] = rows[cu[b] + i, :4]
            wv[table[b, t // page].long(), :, t % page] = rows[cu[b] + i, 4:]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    now = [a + n for a, n in zip(before, new)]
    sd.paged_append(rows[:5, :4], rows[:5, 4:], k, v, table, torch.tensor(now, dtype=torch.int32, device=dev))
    for b, t in enumerate(now):
        wk[table[b, t // page].long(), :, t % page] = rows[b, :4]
        wv[table[b, t // page].long(), :, t % page] = rows[b, 4:]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    ops.check_device_errors(dev)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_append_of_many_rows(dev, dtype):
    """Thousands of rows (the larger CTAs), token-major pages, strided rows."""
    new = [4000, 0, 1500, 1, 700]
    k, v, table = pool(dev, dtype, [n + 9 for n in new], 2, 16, seed=8)
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    wk, wv = k.clone(), v.clone()
    g = torch.Generator(device=dev).manual_seed(5)
    rows = torch.randn(sum(new), 7, 64, generator=g, device=dev).to(dtype)
    ends = torch.tensor([0, *new], device=dev).cumsum(0)
    lens = torch.full((5,), 9, dtype=torch.int32, device=dev)
    sd.paged_append(rows[:, 1:3], rows[:, 4:6], k, v, table, lens, ends.to(torch.int32))
    for b, n in enumerate(new):
        t = torch.arange(9, 9 + n, device=dev)
        wk[table[b].long()[t // 16], :, t % 16] = rows[ends[b]:ends[b] + n, 1:3]
        wv[table[b].long()[t // 16], :, t % 16] = rows[ends[b]:ends[b] + n, 4:6]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    ops.check_device_errors(dev)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_more_sequences_than_one_launch_plans(dev, dtype):
    lens = [(7 * b) % 90 for b in range(2100)]
    k, v, table = pool(dev, dtype, lens, 2, 16, seed=9)
    q = query(dev, dtype, 2100, 4)
    got = sd.paged_decode_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev))
    check(got, *exact(q, k, v, table, lens))
    ops.check_device_errors(dev)


def test_append_out_of_range_is_dropped_and_reported(dev):
    k, v, table = pool(dev, torch.bfloat16, [40, 40], 2, 16, seed=6)
    wk, wv = k.clone(), v.clone()
    x = torch.randn(2, 2, 64, device=dev, dtype=torch.bfloat16)
    for lens, tab in (([48, 2 ** 31 - 1], table), ([-1, 48], table), ([0, 20], table * 0 - 1),
                      ([0, 20], table * 0 + k.shape[0])):
        sd.paged_append(x, x, k, v, tab, torch.tensor(lens, dtype=torch.int32, device=dev))
        with pytest.raises(sd.SparDAError, match="error code 2"):
            ops.check_device_errors(dev)
        assert torch.equal(k, wk) and torch.equal(v, wv)


def test_offsets_past_32_bits(dev):
    """A pool of more than 2^31 elements: pages at its end are found."""
    pages = (2 ** 31 + 2 ** 27) // (4 * 64 * 64)
    k = torch.zeros(pages, 4, 64, 64, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    table = torch.tensor([[pages - 1, pages - 3, 5], [pages - 2, 7, -1]], dtype=torch.int32, device=dev)
    lens = [180, 100]
    cu = torch.tensor([0, 180, 280], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(280, 8, 64, generator=g, device=dev).bfloat16()
    sd.paged_append(x[:, :4], x[:, 4:], k, v, table, torch.zeros(2, dtype=torch.int32, device=dev), cu)
    assert torch.equal(k[pages - 3, :, 10], x[74, :4]) and torch.equal(v[pages - 2, :, 63], x[243, 4:])
    q = query(dev, torch.bfloat16, 2, 12)
    got = sd.paged_decode_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev))
    ops.check_device_errors(dev)
    check(got, *exact(q, k, v, table, lens))


def test_graphs_and_streams(dev):
    """Two captured decode graphs, replayed in turn and at once on two streams
    with lengths that grow, give the eager bits."""
    lens = [700, 3, 0, 2000]
    cases = []
    for seed in (1, 2):
        k, v, table = pool(dev, torch.bfloat16, [3000] * 4, 4, 64, seed=seed)
        cases.append((query(dev, torch.bfloat16, 4, 12, seed), k, v, table,
                      torch.tensor(lens, dtype=torch.int32, device=dev)))
    for c in cases:
        sd.paged_decode_attention(*c)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(sd.paged_decode_attention(*c))
        graphs.append(graph)
    for more in (0, 1, 900):
        for c in cases:
            c[4].copy_(torch.tensor(lens, dtype=torch.int32, device=dev) + more)
        want = [sd.paged_decode_attention(*c) for c in cases]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in cases]
        for _ in range(5):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)
