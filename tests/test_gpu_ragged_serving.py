"""Serving with sequences that end and begin while others go on: released
sequences take no part in steps, eager or captured, and prompts take their
places.  Tolerance as in tests/test_gpu_ragged_model.py.  Needs a B200."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from tests.test_gpu_paged import DTYPES, pool
from tests.test_gpu_ragged_model import LENGTHS, bounds, model, params, plain, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("packed", [False, True])
def test_rows_of_absent_sequences_are_dropped_without_a_report(dev, dtype, packed):
    lens = [17, 0, 40, 5]
    k, v, table = pool(dev, dtype, [n + 2 for n in lens], 4, 16, seed=71)
    wk, wv = k.clone(), v.clone()
    x = torch.randn(4, 8, 64, device=dev).to(dtype)
    dl = torch.tensor([lens[0], ops.LEN_ABSENT, lens[2], ops.LEN_ABSENT], dtype=torch.int32, device=dev)
    table[1] = -1
    cu = torch.arange(5, dtype=torch.int32, device=dev) if packed else None
    sd.paged_append(x[:, :4], x[:, 4:], k, v, table, dl, cu)
    ops.check_device_errors(dev)
    for b in (0, 2):
        wk[table[b, lens[b] // 16].long(), :, lens[b] % 16] = x[b, :4]
        wv[table[b, lens[b] // 16].long(), :, lens[b] % 16] = x[b, 4:]
    assert torch.equal(k, wk) and torch.equal(v, wv)


@torch.no_grad()
def test_release_and_admission_between_eager_and_captured_steps(dev):
    m = model(dev).eval()
    p = params(m)
    cu, dcu = bounds(dev, LENGTHS)
    ids = tokens(dev, cu[-1])
    caches = m.allocate_paged_caches(len(LENGTHS), 200, page_size=16, num_pages=34)
    pages = caches[0].pages
    m(ids[None], kv_caches=caches, cu_seqlens=dcu, lengths=LENGTHS)
    seqs = [ids[a:b] for a, b in zip(cu, cu[1:])]
    feed = torch.zeros(len(LENGTHS), 1, dtype=torch.int64, device=dev)
    seed = [100]

    def check(logits):
        for b, s in enumerate(seqs):
            if s is not None:
                assert float((logits[b, 0] - plain(m, p, s)[-1]).abs().max()) < 2e-4, b
        ops.check_device_errors(dev)
        assert pages.held == pages.lens.tolist() == [0 if s is None else len(s) for s in seqs]

    def new_tokens():
        seed[0] += 1
        feed.copy_(tokens(dev, len(LENGTHS), seed[0])[:, None])
        for b, s in enumerate(seqs):
            if s is not None:
                seqs[b] = torch.cat([s, feed[b]])

    def step():
        new_tokens()
        check(m(feed, kv_caches=caches)["logits"])

    def release(b):
        pages.release(b)
        seqs[b] = None

    def admit(b, n):
        seed[0] += 1
        s = tokens(dev, n, seed[0])
        lengths = [n if i == b else 0 for i in range(len(LENGTHS))]
        got = m(s[None], kv_caches=caches, cu_seqlens=bounds(dev, lengths)[1], lengths=lengths)["logits"][0]
        assert float((got - plain(m, p, s)).abs().max()) < 2e-4
        seqs[b] = s

    release(1)
    release(2)
    free = len(pages.free)
    for _ in range(3):
        step()
    assert len(pages.free) >= free - 3 and pages.owned[1] == pages.owned[2] == []
    # a captured step: what is released or admitted between replays counts in the next
    pages.reserve(8)
    held = list(pages.held)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(feed, kv_caches=caches)
    torch.cuda.current_stream().wait_stream(side)
    pages.lens.sub_(pages.active)
    pages.held = list(held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = m(feed, kv_caches=caches)["logits"]
    pages.held = list(held)

    def replay():
        new_tokens()
        graph.replay()
        pages.advance(1, device=False)
        check(kept)

    replay()
    release(0)
    replay()
    admit(1, 33)
    pages.reserve(8)
    replay()
    replay()
    step()
