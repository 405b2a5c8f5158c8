"""Cases, plain forms and exact values of the operators for ragged batches:

* causal attention over packed prompts of different lengths, and its gradients;
* a paged key-value cache: the append, and the attention of one new token over it;
* log probabilities of given tokens with the distribution's entropy, its
  likeliest alternatives, and the gradient of the logits.

``run`` computes a case in its plain form (elementary torch operations in fp32,
rounded once at the end), or through the package's entry points where ``own``
is set.  Head counts, the head size of 64, the vocabulary of 32000, the 64-token
block and the contexts of 1K to 32K are the model configuration's and the
benchmark's own."""

import math

import torch

own = False


DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HEAD_DIM = 64


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a few short chat turns prefilled together: launch and pipeline latency
        dict(name="prompt_short", op="prompt", dtype="bf16", heads=12, kv_heads=4, tokens=203, seqs=4, train=False),
        # a serving step's prompts of mixed lengths, f16, views of one projection
        dict(name="prompt_mixed", op="prompt", dtype="f16", heads=12, kv_heads=4, tokens=16384, seqs=11, train=False),
        # one prompt of the longest context
        dict(name="prompt_32k", op="prompt", dtype="bf16", heads=12, kv_heads=4, tokens=32768, seqs=1, train=False),
        # a training step over documents packed into one row of tokens
        dict(name="train_packed", op="prompt", dtype="bf16", heads=12, kv_heads=4, tokens=16000, seqs=9, train=True),
        # fp32 training (the reference's default parameter type), odd sizes
        dict(name="train_f32", op="prompt", dtype="f32", heads=12, kv_heads=4, tokens=1023, seqs=3, train=True),
        # prompts of a serving step written into a fragmented page pool
        dict(name="append_prompts", op="append", dtype="bf16", kv_heads=4, page=64, tokens=32768, seqs=13, step=False),
        # one new token of every sequence written
        dict(name="append_step", op="append", dtype="f16", kv_heads=4, page=16, tokens=64, seqs=64, step=True),
        # one sequence at the longest context: the split over its length
        dict(name="decode_one", op="decode", dtype="bf16", heads=12, kv_heads=4, page=64, seqs=1, longest=32768),
        # a few sequences in fp32, some of them just begun, pages of odd size
        dict(name="decode_few", op="decode", dtype="f32", heads=12, kv_heads=4, page=24, seqs=5, longest=1100),
        # a full decode batch at 16K
        dict(name="decode_batch", op="decode", dtype="bf16", heads=12, kv_heads=4, page=64, seqs=64, longest=16384),
        # the next tokens of a decode batch, with alternatives and entropy
        dict(name="score_step", op="score", dtype="bf16", rows=64, vocab=32000, top_k=8, train=False, bonus=False),
        # the loss of a training step over packed documents
        dict(name="score_train", op="score", dtype="bf16", rows=8192, vocab=32000, top_k=0, train=True, bonus=False),
    ]


def _between(rng, low, high):
    """Log-uniform whole number."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "append", "decode", "decode", "score", "score"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    heads, kv_heads = rng.choice([(12, 4), (12, 4), (12, 12), (8, 2), (16, 2), (6, 1)])
    if op == "prompt":
        train = rng.random() < 0.5
        tokens = _between(rng, 16 if train else 1, 2000 if dtype == "f32" else 12000 if train else 24000)
        # a training row holds documents: sequences of one token have no gradients of q and k
        seqs = _between(rng, 1, max(1, min(40, tokens // 16)) if train else 40)
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, tokens=tokens, seqs=seqs, train=train)
    page = rng.choice([8, 16, 24, 32, 64, 100, 128])
    if op == "append":
        step = rng.random() < 0.5
        seqs = _between(rng, 1, 200)
        return dict(op=op, dtype=dtype, kv_heads=kv_heads, page=page, seqs=seqs, step=step,
                    tokens=seqs if step else _between(rng, 1, 30000))
    if op == "decode":
        seqs = _between(rng, 1, 128)
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, page=page, seqs=seqs,
                    longest=_between(rng, 1, min(32768, 400000 // seqs)))
    train = rng.random() < 0.5
    vocab = _between(rng, 300, 130000)
    return dict(op=op, dtype=dtype, rows=_between(rng, 1, max(1, min(8192, 80000000 // vocab))), vocab=vocab,
                top_k=0 if train else rng.choice([0, 1, 5, 8, 20]), train=train,
                bonus=train and rng.random() < 0.5)


# ------------------------------------------------------------------ their inputs
def _lengths(total, seqs, gen):
    """Lengths of ``seqs`` sequences with the given sum, spread over a factor of
    about twenty; with more sequences than tokens some of them are empty."""
    share = torch.exp(3.0 * torch.rand(seqs, generator=gen, dtype=torch.float64))
    ends = torch.round(torch.cumsum(share, 0) / share.sum() * total).to(torch.int64)
    ends[-1] = total
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.int64)).tolist()


def _kept(case, seed):
    """Sequence lengths of a case (host), from the seed alone."""
    gen = torch.Generator().manual_seed(seed)
    if case["op"] == "decode":
        # most of a batch is near its longest, some have just begun
        u = torch.rand(case["seqs"], generator=gen, dtype=torch.float64)
        lens = torch.ceil(case["longest"] * (1.0 - 0.5 * u)).to(torch.int64)
        lens[::5] = torch.ceil(lens[::5] * u[::5]).to(torch.int64)
        lens[0] = case["longest"]
        return lens.tolist()
    if case["op"] == "append" and case["step"]:
        return [1] * case["seqs"]
    return _lengths(case["tokens"], case["seqs"], gen)


def _normal(shape, dtype, gen, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return (x * scale if scale != 1.0 else x).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bounds(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


def _page_table(need, page, pages, gen):
    """A table of scattered pages of a pool for sequences of ``need`` tokens:
    [S, most pages] int32, -1 where a sequence has no page."""
    counts = [-(-n // page) for n in need]
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    width = table.shape[1]
    held = torch.arange(width, device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table[held] = order[:sum(counts)]
    return table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal((rows, vocab), dtype, gen, 3.0)
        state["logits"] = logits.requires_grad_() if case["train"] else logits
        state["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        if case["train"]:
            state["targets"][rows // 2::7] = -100  # padding and prompt tokens carry no loss
            state["weight"] = torch.full((rows,), -1.0 / rows, device="cuda")
            state["bonus_weight"] = torch.full((rows,), 0.01 / rows, device="cuda")
        return state
    lengths = _kept(case, seed)
    hkv = case["kv_heads"]
    if case["op"] == "prompt":
        hq, total = case["heads"], case["tokens"]
        # q, k and v are views of one projection's rows
        rows = _normal((total, (hq + 2 * hkv) * HEAD_DIM), dtype, gen)
        heads = rows.view(total, hq + 2 * hkv, HEAD_DIM)
        state["q"], state["k"], state["v"] = heads[:, :hq], heads[:, hq:hq + hkv], heads[:, hq + hkv:]
        state["lengths"] = lengths
        state["cu_seqlens"] = _int32(_bounds(lengths))
        if case["train"]:
            state["dout"] = _normal((total, hq, HEAD_DIM), dtype, gen)
            for name in ("q", "k", "v"):
                state[name] = state[name].detach().requires_grad_()
        return state
    page = case["page"]
    if case["op"] == "append":
        total = case["tokens"]
        before = torch.randint(0, 300, (case["seqs"],), generator=gen, device="cuda")
        held = before.tolist()
        pages = total // page + case["seqs"] * (300 // page + 2)  # enough for any lengths of this sum
        table = _page_table([a + n for a, n in zip(held, lengths)], page, pages, gen)
        rows = _normal((total, 2 * hkv, HEAD_DIM), dtype, gen)
        state.update(xk=rows[:, :hkv], xv=rows[:, hkv:], table=table, before=before.to(torch.int32),
                     k_pages=_normal((pages, hkv, page, HEAD_DIM), dtype, gen),
                     v_pages=_normal((pages, hkv, page, HEAD_DIM), dtype, gen))
        state["cu_seqlens"] = None if case["step"] else _int32(_bounds(lengths))
        return state
    pages = sum(-(-n // page) for n in lengths) + 2
    table = _page_table(lengths, page, pages, gen)
    state.update(q=_normal((case["seqs"], case["heads"], HEAD_DIM), dtype, gen), table=table,
                 lens=_int32(lengths),
                 k_pages=_normal((pages, hkv, page, HEAD_DIM), dtype, gen),
                 v_pages=_normal((pages, hkv, page, HEAD_DIM), dtype, gen))
    return state


# ------------------------------------------------------------------ the plain forms
def _plain_prompt(state):
    """softmax(q k^T / 8 + causal mask) v per sequence, in fp32; with ``train``
    also the gradients of q, k and v for the output gradient.  One sequence and
    key-value head at a time, so that the score matrices fit the card."""
    q, k, v = state["q"], state["k"], state["v"]
    hkv = k.shape[1]
    group = q.shape[1] // hkv
    train = state["train"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)) if train else (None,) * 3
    scale = 1.0 / math.sqrt(HEAD_DIM)
    start = 0
    with torch.no_grad():
        for n in state["lengths"]:
            here = slice(start, start + n)
            start += n
            if n == 0:
                continue
            hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
            for h in range(hkv):
                of = slice(h * group, (h + 1) * group)
                qh = q[here, of].float().transpose(0, 1)  # [group, n, 64]
                kh, vh = k[here, h].float(), v[here, h].float()
                s = torch.matmul(qh, kh.t()).mul_(scale).masked_fill_(hidden, -math.inf)
                s -= s.amax(-1, keepdim=True)
                p = s.exp_()
                p /= p.sum(-1, keepdim=True)
                out[here, of] = torch.matmul(p, vh).transpose(0, 1).to(out.dtype)
                if train:
                    g = state["dout"][here, of].float().transpose(0, 1)
                    dv[here, h] = torch.matmul(p.transpose(1, 2), g).sum(0).to(dv.dtype)
                    dp = torch.matmul(g, vh.t())
                    ds = (dp - (p * dp).sum(-1, keepdim=True)).mul_(p)
                    dq[here, of] = (torch.matmul(ds, kh) * scale).transpose(0, 1).to(dq.dtype)
                    dk[here, h] = (torch.matmul(ds.transpose(1, 2), qh).sum(0) * scale).to(dk.dtype)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else {"out": out}


def _plain_append(state):
    """Row i of sequence s goes to position before[s] + i, i.e. to row
    (position mod page) of page table[s, position div page]."""
    xk, xv, page = state["xk"], state["xv"], state["page"]
    rows = torch.arange(xk.shape[0], device=xk.device)
    if state["cu_seqlens"] is None:
        seq, place = rows, state["before"].long()
    else:
        ends = state["cu_seqlens"].long()
        seq = torch.searchsorted(ends[1:], rows, right=True)
        place = rows - ends[seq] + state["before"].long()[seq]
    pages = state["table"][seq, place // page].long()
    state["k_pages"][pages, :, place % page] = xk
    state["v_pages"][pages, :, place % page] = xv
    return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _plain_decode(state):
    """softmax(q k^T / 8) v over the first lens[s] tokens of each sequence's pages."""
    q, table, lens = state["q"], state["table"].long().clamp_min(0), state["lens"].long()
    seqs, hq = q.shape[0], q.shape[1]
    hkv = state["k_pages"].shape[1]
    k = state["k_pages"][table].transpose(1, 2).reshape(seqs, hkv, -1, HEAD_DIM).float()
    v = state["v_pages"][table].transpose(1, 2).reshape(seqs, hkv, -1, HEAD_DIM).float()
    qh = q.float().view(seqs, hkv, hq // hkv, HEAD_DIM)
    s = torch.matmul(qh, k.transpose(2, 3)) * (1.0 / math.sqrt(HEAD_DIM))
    past = torch.arange(k.shape[2], device=q.device)[None, :] >= lens[:, None]
    s = s.masked_fill_(past[:, None, None, :], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = v.masked_fill_(past[:, None, :, None], 0.0)
    return {"out": torch.matmul(p, v).view(seqs, hq, HEAD_DIM).to(q.dtype)}


def _plain_score(state):
    """log softmax at the targets (0 where the target is -100), the entropy, the
    top_k likeliest tokens (ties: lowest index); with ``train`` the gradient of
    sum(weight * log probability [+ bonus_weight * entropy])."""
    logits, targets = state["logits"].detach(), state["targets"]
    x = logits.float()
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    logp = x - torch.log(total)
    p = e / total
    entropy = -(p * logp).sum(-1)
    kept = targets != -100
    at = targets.clamp_min(0)[:, None]
    chosen = torch.where(kept, logp.gather(1, at)[:, 0], torch.zeros_like(entropy))
    found = {"logprobs": chosen, "entropy": entropy}
    if state["top_k"]:
        ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :state["top_k"]]
        found.update(top_logprobs=logp.gather(1, ids), top_ids=ids)
    if state["train"]:
        w = torch.where(kept, state["weight"], torch.zeros_like(state["weight"]))[:, None]
        d = p * -w
        d.scatter_add_(1, at, w)
        if state["bonus"]:
            d -= state["bonus_weight"][:, None] * p * (logp + entropy[:, None])
        found["dlogits"] = d.to(logits.dtype)
    return found


def run(state):
    op = state["op"]
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "decode": _plain_decode,
                "score": _plain_score}[op](state)
    import local_research_small_language_model_b200 as sd
    if op == "prompt":
        q, k, v = state["q"], state["k"], state["v"]
        out = sd.packed_attention(q, k, v, state["cu_seqlens"])
        if not state["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if op == "append":
        sd.paged_append(state["xk"], state["xv"], state["k_pages"], state["v_pages"], state["table"],
                        state["before"], state["cu_seqlens"])
        return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    if op == "decode":
        return {"out": sd.paged_decode_attention(state["q"], state["k_pages"], state["v_pages"], state["table"],
                                                 state["lens"])}
    got = sd.token_logprobs(state["logits"], state["targets"], top_k=state["top_k"])
    found = {"logprobs": got.logprobs.detach(), "entropy": got.entropy.detach()}
    if state["top_k"]:
        found.update(top_logprobs=got.top_logprobs, top_ids=got.top_ids)
    if state["train"]:
        outputs, weights = [got.logprobs], [state["weight"]]
        if state["bonus"]:
            outputs.append(got.entropy)
            weights.append(state["bonus_weight"])
        found["dlogits"], = torch.autograd.grad(outputs, (state["logits"],), weights)
    return found


# ------------------------------------------------------------------ the least work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        moved = n * size * (2 if case["train"] else 1) + case["rows"] * (16 + 12 * case["top_k"])
        return {"bytes": moved, "flops": n * (8 if case["train"] else 4)}
    row = HEAD_DIM * size
    hkv = case["kv_heads"]
    if case["op"] == "append":
        return {"bytes": 4 * case["tokens"] * hkv * row, "flops": 0}
    hq = case["heads"]
    lengths = _kept(case, 0)
    if case["op"] == "decode":
        held = sum(lengths)
        return {"bytes": 2 * held * hkv * row + 2 * case["seqs"] * hq * row, "flops": 4 * held * hq * HEAD_DIM}
    pairs = sum(n * (n + 1) // 2 for n in lengths)
    total = case["tokens"]
    if not case["train"]:
        return {"bytes": total * row * (2 * hq + 2 * hkv), "flops": 4 * HEAD_DIM * hq * pairs}
    return {"bytes": total * row * (4 * hq + 4 * hkv), "flops": 14 * HEAD_DIM * hq * pairs}


# ------------------------------------------------------------------ in 64 bits
def _exact_prompt(state):
    q, k, v = (state[x].detach().double() for x in ("q", "k", "v"))
    hq, group = q.shape[1], q.shape[1] // k.shape[1]
    names = ("out", "dq", "dk", "dv") if state["train"] else ("out",)
    found = {x: torch.zeros_like(k if x in ("dk", "dv") else q) for x in names}
    ends = state["cu_seqlens"].tolist()
    for a, b in zip(ends, ends[1:]):
        for h in range(hq):
            kh, vh = k[a:b, h // group], v[a:b, h // group]
            for r in range(a, b, 2048):  # rows r .. e see keys a .. e
                e = min(b, r + 2048)
                s = q[r:e, h] @ kh[:e - a].t() / math.sqrt(HEAD_DIM)
                late = torch.arange(a, e, device=q.device)[None, :] > torch.arange(r, e, device=q.device)[:, None]
                p = torch.softmax(s.masked_fill(late, -math.inf), dim=-1)
                o = p @ vh[:e - a]
                found["out"][r:e, h] = o
                if state["train"]:
                    g = state["dout"][r:e, h].double()
                    ds = p * (g @ vh[:e - a].t() - (g * o).sum(-1, keepdim=True)) / math.sqrt(HEAD_DIM)
                    found["dq"][r:e, h] = ds @ kh[:e - a]
                    found["dk"][a:e, h // group] += ds.t() @ q[r:e, h]
                    found["dv"][a:e, h // group] += p.t() @ g
    return found


def _exact_decode(state):
    q = state["q"].double()
    out = torch.zeros_like(q)
    hkv = state["k_pages"].shape[1]
    for s, n in enumerate(state["lens"].tolist()):
        if n == 0:
            continue
        pages = state["table"][s, :-(-n // state["page"])].long()
        k = state["k_pages"][pages].double().transpose(0, 1).reshape(hkv, -1, HEAD_DIM)[:, :n]
        v = state["v_pages"][pages].double().transpose(0, 1).reshape(hkv, -1, HEAD_DIM)[:, :n]
        heads = q[s].view(hkv, -1, HEAD_DIM)
        weight = torch.softmax(torch.einsum("hgd,hnd->hgn", heads, k) / math.sqrt(HEAD_DIM), dim=-1)
        out[s] = torch.einsum("hgn,hnd->hgd", weight, v).reshape(-1, HEAD_DIM)
    return {"out": out}


def _exact_score(state):
    logits, targets = state["logits"].detach(), state["targets"]
    rows, vocab = logits.shape
    found = {"logprobs": torch.zeros(rows, dtype=torch.float64, device=logits.device)}
    found["entropy"] = torch.zeros_like(found["logprobs"])
    top = state["top_k"]
    if top:
        found["top_logprobs"] = torch.zeros(rows, top, dtype=torch.float64, device=logits.device)
        found["top_ids"] = None
    if state["train"]:
        found["dlogits"] = torch.empty(rows, vocab, dtype=torch.float64, device=logits.device)
    every = max(1, 60_000_000 // vocab)
    for r in range(0, rows, every):
        e = min(rows, r + every)
        lp = torch.log_softmax(logits[r:e].double(), dim=-1)
        kept = targets[r:e] != -100
        at = targets[r:e].clamp_min(0)[:, None]
        found["logprobs"][r:e] = lp.gather(1, at)[:, 0] * kept
        p = lp.exp()
        h = -(p * lp).sum(-1)
        found["entropy"][r:e] = h
        if top:
            found["top_logprobs"][r:e] = torch.topk(lp, top, dim=-1).values
        if state["train"]:
            w = (state["weight"][r:e].double() * kept)[:, None]
            d = -w * p
            d.scatter_add_(1, at, w)
            if state["bonus"]:
                d -= state["bonus_weight"][r:e, None].double() * p * (lp + h[:, None])
            found["dlogits"][r:e] = d
    return found


def exact(case, seed):
    if case["op"] == "append":
        return None  # rows are moved, nothing is computed
    state = prepare(case, seed)
    return {"prompt": _exact_prompt, "decode": _exact_decode, "score": _exact_score}[case["op"]](state)
