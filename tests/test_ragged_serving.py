"""Sequences of a paged cache that end and begin while others go on, on the CPU
with the device kernels replaced by plain forms: a released sequence takes no
part in the steps that follow, and a prompt may take its place."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import model, ops
from tests.test_ragged_layers import CONFIG, on_cpu, plain_rope  # noqa: F401


def plain_append(xk, xv, k_pages, v_pages, page_table, lens, cu_seqlens=None):
    page = k_pages.shape[2]
    cu = cu_seqlens.tolist() if cu_seqlens is not None else range(lens.numel() + 1)
    for b, n in enumerate(lens.tolist()):
        if n == ops.LEN_ABSENT:
            continue
        for i, r in enumerate(range(cu[b], cu[b + 1])):
            p = int(page_table[b, (n + i) // page])
            assert p >= 0 and n >= 0, "a row without a place"
            k_pages[p, :, (n + i) % page], v_pages[p, :, (n + i) % page] = xk[r], xv[r]


def plain_decode(q, k_pages, v_pages, page_table, lens, scale=None, out=None):
    out = torch.zeros_like(q)
    hkv = k_pages.shape[1]
    for b, n in enumerate(lens.tolist()):
        assert n >= 0
        if n == 0:
            continue
        ids = page_table[b, :-(-n // k_pages.shape[2])].long()
        assert (ids >= 0).all(), "a page that is not held"
        k, v = (x[ids].transpose(0, 1).reshape(hkv, -1, 64)[:, :n] for x in (k_pages, v_pages))
        p = torch.softmax(q[b].view(hkv, -1, 64) @ k.transpose(1, 2) / 8, -1)
        out[b] = (p @ v).reshape(-1, 64)
    return out


@pytest.fixture
def paged(on_cpu, monkeypatch):  # noqa: F811
    monkeypatch.setattr(ops, "paged_append", plain_append)
    monkeypatch.setattr(ops, "paged_decode_attention", plain_decode)


def test_page_table_keeps_released_sequences_out():
    t = sd.PageTable(3, 64, 6, torch.device("cpu"), page_size=16)
    t.reserve([16, 16, 5])
    t.advance([16, 16, 5])
    t.release(1)
    for _ in range(3):
        t.reserve(1)
        t.advance(1)
    assert t.held == [19, 0, 8] == t.lens.tolist() and t.owned[1] == [] and len(t.free) == 3
    assert t.active.tolist() == [1, 0, 1] and t.absent.tolist() == [0, ops.LEN_ABSENT, 0]
    assert (t.table[1] == -1).all()
    t.reserve([0, 0, 0])
    assert t.released == [False, True, False]
    assert t.fills([1, 0, 0]) and not t.fills([0, 4, 0]) and t.fills(None)
    t.reserve([0, 30, 0])  # a prompt takes the place
    t.advance([0, 30, 0])
    t.reserve(1)
    t.advance(1)
    assert t.held == [20, 31, 9] == t.lens.tolist()
    assert t.active.tolist() == [1, 1, 1] and t.absent.tolist() == [0, 0, 0]
    t.release(0)
    t.reset()
    assert t.active.tolist() == [1, 1, 1] and t.absent.tolist() == [0, 0, 0] and t.released == [False] * 3
    with pytest.raises(ValueError):
        t.reserve(-1)


@torch.no_grad()
def test_steps_after_a_release_and_a_prompt_in_its_place(paged):
    torch.manual_seed(2)
    m = model.SparDAB200Model(sd.ModelConfig(**CONFIG)).eval()
    caches = m.allocate_paged_caches(3, 64, num_pages=6, page_size=16)
    pages = caches[0].pages

    def check(logits, seqs):
        for b, s in enumerate(seqs):
            if s is not None:
                assert torch.allclose(logits[b], m(s[None])["logits"][0, -1], atol=1e-5), b

    seqs = [torch.randint(0, 50, (n,)) for n in (16, 16, 5)]
    cu = torch.tensor([0, 16, 32, 37], dtype=torch.int32)
    m(torch.cat(seqs)[None], kv_caches=caches, cu_seqlens=cu, lengths=[16, 16, 5])
    pages.release(1)
    seqs[1] = None
    assert len(pages.free) == 4

    def step():
        new = torch.randint(0, 50, (3, 1))
        logits = m(new, kv_caches=caches)["logits"][:, 0]
        for b in range(3):
            if seqs[b] is not None:
                seqs[b] = torch.cat([seqs[b], new[b]])
        check(logits, seqs)

    for _ in range(3):
        step()
    assert len(pages.free) == 3 and pages.held == [19, 0, 8]
    prompt = torch.randint(0, 50, (20,))
    with pytest.raises(NotImplementedError, match="non-empty"):
        m(prompt[None], kv_caches=caches, cu_seqlens=torch.tensor([0, 2, 20, 20], dtype=torch.int32),
          lengths=[2, 18, 0])
    got = m(prompt[None], kv_caches=caches, cu_seqlens=torch.tensor([0, 0, 20, 20], dtype=torch.int32),
            lengths=[0, 20, 0])["logits"]
    assert torch.allclose(got, m(prompt[None])["logits"], atol=1e-5)
    seqs[1] = prompt
    for _ in range(2):
        step()
    assert pages.held == [21, 22, 10] == pages.lens.tolist()


def test_append_leaves_released_sequences_out(paged):
    """A step's rows written by hand, without the model."""
    t = sd.PageTable(3, 64, 6, torch.device("cpu"), page_size=16)
    cache = sd.B200PagedKVCache(t, 1, 64, torch.device("cpu"), torch.float32)
    t.reserve([3, 4, 5])
    t.advance([3, 4, 5])
    t.release(1)
    t.reserve(1)
    x = torch.randn(3, 1, 64)
    cache.append(x, x)
    t.advance(1)
    assert t.lens.tolist() == [4, 0, 6]
    want = torch.zeros_like(cache.k_pages)
    want[t.owned[0][0], :, 3], want[t.owned[2][0], :, 5] = x[0], x[2]
    assert torch.equal(cache.k_pages, want)
