"""Ragged batches without a GPU: the C entry points and their wrappers refuse
bad arguments before any launch, and the page table's bookkeeping."""

import ctypes

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from local_research_small_language_model_b200.model import SparDAB200Model

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4098)
INVALID, UNSUPPORTED, ALIGN = -1, -2, -4


def packed(lib, **kw):
    a = dict(q=P, k=P, v=P, dtype=1, total=10, hq=4, hkv=2, d=64, q_st=256, q_sh=64, k_st=128, k_sh=64, v_st=128,
             v_sh=64, cu=P, nseq=1, scale=0.125, out=P, o_st=256, o_sh=64, lse=P, rest=P, zero=1)
    a.update(kw)
    return lib.sd_packed_attention(*a.values(), None, None)


def backward(lib, **kw):
    a = dict(q=P, k=P, v=P, out=P, dout=P, dtype=1, total=10, hq=4, hkv=2, d=64, q_st=256, q_sh=64, k_st=128,
             k_sh=64, v_st=128, v_sh=64, o_st=256, o_sh=64, g_st=256, g_sh=64, cu=P, nseq=1, scale=0.125, lse=P,
             rest=P, delta=P, dq=P, dk=P, dv=P)
    a.update(kw)
    return lib.sd_packed_attention_backward(*a.values(), None, None)


def append(lib, **kw):
    a = dict(xk=P, xv=P, dtype=1, n=4, hkv=2, d=64, k_sn=128, k_sh=64, v_sn=128, v_sh=64, kp=P, vp=P, pages=9,
             page=16, p_sp=2048, p_sh=1024, p_st=64, table=P, t_sb=3, width=3, lens=P, b=4, cu=None)
    a.update(kw)
    return lib.sd_paged_append(*a.values(), None, None)


def decode(lib, **kw):
    a = dict(q=P, dtype=1, b=4, hq=4, hkv=2, d=64, q_sb=256, q_sh=64, kp=P, vp=P, pages=9, page=16, p_sp=2048,
             p_sh=1024, p_st=64, table=P, t_sb=3, width=3, lens=P, scale=0.125, out=P, o_sb=256, o_sh=64, ws=P,
             ws_bytes=1 << 30)
    a.update(kw)
    return lib.sd_paged_decode_attention(*a.values(), None, None)


def scores(lib, **kw):
    a = dict(x=P, dtype=1, rows=3, v=100, ld=100, t=P, ignore=-100, lp=P, h=P, stats=P, k=4, tlp=P, ids=P)
    a.update(kw)
    return lib.sd_token_logprobs(*a.values(), None, None)


def scores_backward(lib, **kw):
    a = dict(x=P, dtype=1, rows=3, v=100, ld=100, t=P, ignore=-100, stats=P, g=P, ge=None, d=P, d_ld=100)
    a.update(kw)
    return lib.sd_token_logprobs_backward(*a.values(), None)


REFUSED = [
    (packed, dict(q=None), INVALID), (packed, dict(cu=None), INVALID), (packed, dict(out=None), INVALID),
    (packed, dict(total=0), INVALID), (packed, dict(hq=5), INVALID), (packed, dict(hkv=0), INVALID),
    (packed, dict(dtype=9), INVALID), (packed, dict(scale=0.0), INVALID), (packed, dict(scale=-1.0), INVALID),
    (packed, dict(scale=float("nan")), INVALID), (packed, dict(scale=float("inf")), INVALID),
    (packed, dict(nseq=-1), INVALID), (packed, dict(d=128), UNSUPPORTED), (packed, dict(hq=131072), UNSUPPORTED),
    (packed, dict(total=2 ** 31), UNSUPPORTED), (packed, dict(k=ODD), ALIGN), (packed, dict(v_st=129), ALIGN),
    (packed, dict(o_sh=60), ALIGN), (packed, dict(rest=ODD), ALIGN), (backward, dict(rest=ODD), ALIGN),
    (backward, dict(dout=None), INVALID), (backward, dict(lse=None), INVALID), (backward, dict(delta=None), INVALID),
    (backward, dict(dk=None), INVALID), (backward, dict(dv=ODD), ALIGN), (backward, dict(g_st=4), ALIGN),
    (backward, dict(d=32), UNSUPPORTED),
    (append, dict(xv=None), INVALID), (append, dict(n=0), INVALID), (append, dict(n=3), INVALID),
    (append, dict(page=0), INVALID), (append, dict(width=0), INVALID), (append, dict(pages=0), INVALID),
    (append, dict(lens=None), INVALID), (append, dict(d=96), UNSUPPORTED), (append, dict(p_st=65), ALIGN),
    (append, dict(xk=ODD), ALIGN), (append, dict(width=2 ** 30, page=8), UNSUPPORTED),
    (decode, dict(q=None), INVALID), (decode, dict(b=0), INVALID), (decode, dict(hq=3), INVALID),
    (decode, dict(scale=0.0), INVALID), (decode, dict(table=None), INVALID), (decode, dict(d=128), UNSUPPORTED),
    (decode, dict(out=ODD), ALIGN), (decode, dict(kp=ODD), ALIGN), (decode, dict(q_sb=100), ALIGN),
    (scores, dict(x=None), INVALID), (scores, dict(t=None), INVALID), (scores, dict(lp=None), INVALID),
    (scores, dict(rows=0), INVALID), (scores, dict(v=0), INVALID), (scores, dict(k=-1), INVALID),
    (scores, dict(v=3), INVALID), (scores, dict(k=65), UNSUPPORTED), (scores, dict(ids=None), INVALID),
    (scores, dict(dtype=3), INVALID),
    (scores_backward, dict(stats=None), INVALID), (scores_backward, dict(d=None), INVALID),
    (scores_backward, dict(d_ld=99), INVALID), (scores_backward, dict(v=0), INVALID),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_entry_points_refuse(case):
    call, wrong, code = REFUSED[case]
    assert call(sd.load_library(), **wrong) == code


def test_argument_blocks_reach_the_same_entry_points():
    """sd_invoke with the declared number of words gives the entry point's own
    status; another number of words, or call, is refused."""
    from local_research_small_language_model_b200 import _lib
    lib = sd.load_library()
    for call, wrong, code in REFUSED:
        name = {packed: "sd_packed_attention", backward: "sd_packed_attention_backward", append: "sd_paged_append",
                decode: "sd_paged_decode_attention", scores: "sd_token_logprobs",
                scores_backward: "sd_token_logprobs_backward"}[call]

        class Spy:
            def __getattr__(self, entry):
                def run(*args):
                    assert entry == name and len(args) == len(_lib._SIGS[name])
                    plain = [a.value if isinstance(a, ctypes.c_void_p) else a for a in args]
                    return _lib.block_call(name)(*[0 if a is None else a for a in plain])
                return run

        assert call(Spy(), **wrong) == code, (name, wrong)
    words = (ctypes.c_int64 * 40)()
    block = ctypes.cast(words, ctypes.c_char_p)
    for number in range(6):
        assert lib.sd_invoke(number, block, 3) == INVALID
    assert lib.sd_invoke(6, block, 13) == INVALID and lib.sd_invoke(0, None, 24) == INVALID


def test_workspace_sizes():
    lib = sd.load_library()
    n = ctypes.c_int64(-1)
    assert lib.sd_paged_decode_workspace(4, 12, 4, ctypes.byref(n)) == 0 and n.value >= 0
    assert lib.sd_paged_decode_workspace(0, 12, 4, ctypes.byref(n)) == INVALID
    assert lib.sd_paged_decode_workspace(4, 12, 4, None) == INVALID


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


CU = torch.tensor([0, 10], dtype=torch.int32)
WRAPPERS = [
    (lambda: sd.packed_attention(z(10, 4, 64), z(10, 2, 64), z(10, 2, 64), CU), ValueError, "CUDA"),
    (lambda: sd.packed_attention(z(10, 4, 64), z(9, 2, 64), z(9, 2, 64), CU), ValueError, "total"),
    (lambda: sd.packed_attention(z(10, 4, 64), z(10, 3, 64), z(10, 3, 64), CU), ValueError, "multiple"),
    (lambda: sd.packed_attention(z(10, 4, 32), z(10, 2, 32), z(10, 2, 32), CU), ValueError, "head size"),
    (lambda: sd.packed_attention(z(10, 4, 64), z(10, 2, 64), z(10, 2, 64).half(), CU), TypeError, "dtype"),
    (lambda: sd.packed_attention(z(10, 4, 64), z(10, 2, 64), z(10, 2, 64), CU[:1]), ValueError, "cu_seqlens"),
    (lambda: ops.packed_attention(z(10, 4, 64), z(10, 2, 64), z(10, 2, 64), CU, out=z(10, 2, 64)), ValueError, "out"),
    (lambda: ops.packed_attention_backward(z(10, 4, 64), z(10, 2, 64), z(10, 2, 64), z(10, 4, 64), z(10, 3, 64),
                                           z(4, 10), CU), ValueError, "dout"),
    (lambda: sd.paged_append(z(4, 2, 64), z(4, 2, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(1, 2), CU), ValueError,
     "page_table"),
    (lambda: sd.paged_append(z(4, 2, 64), z(4, 2, 64), z(9, 3, 16, 64), z(9, 3, 16, 64), CU.view(2, 1), CU), ValueError,
     "kv heads"),
    (lambda: sd.paged_append(z(4, 2, 64), z(4, 2, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(2, 1), CU), ValueError,
     "one row"),
    (lambda: sd.paged_append(z(2, 2, 64), z(2, 2, 64), z(9, 2, 16, 64).half(), z(9, 2, 16, 64).half(), CU.view(2, 1),
                             CU), TypeError, "fit"),
    (lambda: sd.paged_append(z(2, 2, 64), z(2, 2, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(2, 1), CU),
     ValueError, "CUDA"),
    (lambda: sd.paged_decode_attention(z(2, 4, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(2, 1), CU), ValueError,
     "CUDA"),
    (lambda: sd.paged_decode_attention(z(2, 3, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(2, 1), CU), ValueError,
     "multiple"),
    (lambda: sd.paged_decode_attention(z(3, 4, 64), z(9, 2, 16, 64), z(9, 2, 16, 64), CU.view(2, 1), CU), ValueError,
     "lens"),
    (lambda: sd.paged_decode_attention(z(2, 4, 64), z(9, 2, 64, 16).transpose(2, 3), z(9, 2, 64, 16).transpose(2, 3),
                                       CU.view(2, 1), CU), ValueError, "stride"),
    (lambda: sd.token_logprobs(z(3, 10), torch.zeros(3, dtype=torch.int64)), ValueError, "CUDA"),
    (lambda: sd.token_logprobs(z(3, 10), torch.zeros(3, dtype=torch.int32)), ValueError, "targets"),
    (lambda: sd.token_logprobs(z(3, 10), torch.zeros(2, dtype=torch.int64)), ValueError, "targets"),
    (lambda: sd.token_logprobs(z(3, 10), torch.zeros(3, dtype=torch.int64), top_k=11), ValueError, "top_k"),
    (lambda: sd.token_logprobs(z(3, 0), torch.zeros(3, dtype=torch.int64)), ValueError, "logits"),
]


@pytest.mark.parametrize("case", range(len(WRAPPERS)))
def test_wrappers_refuse(case):
    call, kind, text = WRAPPERS[case]
    with pytest.raises(kind, match=text):
        call()


def test_scale_must_be_positive():
    for bad in (0.0, -0.1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            ops._scale(bad, 64)


def test_page_table_bookkeeping():
    t = sd.PageTable(3, 100, 8, torch.device("cpu"), page_size=16)
    assert (t.width, t.capacity) == (7, 112)
    t.reserve([20, 0, 33])
    assert [len(o) for o in t.owned] == [2, 0, 3] and len(t.free) == 3
    t.advance([20, 0, 33])
    assert t.held == [20, 0, 33] and t.lens.tolist() == [20, 0, 33]
    held = {p for o in t.owned for p in o}
    assert len(held) == 5 and held.isdisjoint(t.free)
    for b in range(3):
        n = len(t.owned[b])
        assert t.table[b, :n].tolist() == t.owned[b] and (t.table[b, n:] == -1).all()
    t.reserve(1)  # sequence 1 opens its first page, the others have room
    assert [len(o) for o in t.owned] == [2, 1, 3]
    t.advance(1)
    assert t.lens.tolist() == [21, 1, 34]
    before = [list(o) for o in t.owned]
    with pytest.raises(ValueError, match="out of pages"):
        t.reserve([60, 0, 0])
    with pytest.raises(ValueError, match="overflow"):
        t.reserve([0, 112, 0])
    with pytest.raises(ValueError, match="reserve"):
        t.advance([60, 0, 0])
    with pytest.raises(ValueError):
        t.reserve([1, 2])
    with pytest.raises(ValueError):
        t.reserve(-1)
    assert t.owned == before and t.held == [21, 1, 34]
    t.release(0)
    assert t.held[0] == 0 and len(t.free) == 4 and (t.table[0] == -1).all() and t.lens[0] == 0
    t.reserve([0, 60, 0])
    t.reset()
    assert len(t.free) == 8 and t.lens.sum() == 0 and (t.table == -1).all()
    with pytest.raises(ValueError):
        sd.PageTable(0, 1, 1, torch.device("cpu"))


def test_dense_backend_is_selected_and_keeps_the_state_dict():
    kw = dict(n_layer=2, block_size=64, top_k_blocks=8)
    dense = SparDAB200Model(sd.ModelConfig(attention_backend="b200_dense", **kw))
    sparse = SparDAB200Model(sd.ModelConfig(**kw))
    assert all(isinstance(x.attention, sd.B200DenseAttention) for x in dense.layers)
    assert all(isinstance(x.attention, sd.B200SparseAttention) for x in sparse.layers)
    dense.load_state_dict(sparse.state_dict())
    assert {k: v.shape for k, v in dense.state_dict().items()} == {k: v.shape for k, v in sparse.state_dict().items()}
    with pytest.raises(NotImplementedError, match="b200_dense"):
        sparse(torch.zeros(1, 4, dtype=torch.int64), cu_seqlens=CU)
    with pytest.raises(NotImplementedError, match="Paged"):
        dense(torch.zeros(1, 4, dtype=torch.int64), kv_caches=[object()])


def test_ragged_positions_restart_with_every_sequence():
    rope = sd.RotaryEmbedding(64, 32)
    cu = torch.tensor([0, 3, 3, 8], dtype=torch.int32)
    batch = sd.RaggedBatch.prompts(cu, 10, rope)
    pos = torch.tensor([0, 1, 2, 0, 1, 2, 3, 4])
    assert torch.equal(batch.cos[:8], rope.cos[pos]) and torch.equal(batch.sin[:8], rope.sin[pos])
    step = sd.RaggedBatch.step(torch.tensor([0, 7, 31], dtype=torch.int32), 32, rope)
    assert torch.equal(step.cos, rope.cos[torch.tensor([0, 7, 31])]) and step.lens_after.tolist() == [1, 8, 32]
