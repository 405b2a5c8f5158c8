"""token_logprobs over rows that mask tokens with the type's lowest finite value
(constrained decoding, a masked vocabulary) beside ordinary logits: finite, as
log_softmax, whatever a thread meets first.  Bounds as in
tests/test_gpu_scoring.py: a masked token's exponential is 0 and adds nothing.
Needs a B200."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from tests.test_gpu_scoring import DTYPES, check, exact, exact_grad, grads, make

pytestmark = pytest.mark.gpu


def masked(dev, dtype, rows, vocab, seed):
    """Rows of six kinds in turn: a masked prefix, all but three tokens masked,
    one aligned run of eight masked, a masked suffix, every second token masked,
    and a masked target."""
    x, t = make(dev, dtype, rows, vocab, seed=seed)
    low = torch.finfo(dtype).min
    kind = torch.arange(rows, device=dev) % 6
    at = torch.arange(vocab, device=dev)[None, :]
    cut = (vocab * 9 // 10 + torch.arange(rows, device=dev) % 7)[:, None]
    x = torch.where((kind == 0)[:, None] & (at < cut), low, x)
    few = (at == 11) | (at == vocab // 2) | (at == vocab - 1)
    x = torch.where((kind == 1)[:, None] & ~few, low, x)
    x = torch.where((kind == 2)[:, None] & (at >= 16) & (at < 24), low, x)
    x = torch.where((kind == 3)[:, None] & (at >= vocab // 5), low, x)
    x = torch.where((kind == 4)[:, None] & (at % 2 == 0), low, x)
    x = torch.where((kind == 5)[:, None] & (at == t[:, None]), low, x)
    t = torch.where(kind == 0, vocab - 1, torch.where(kind == 1, vocab // 2, t))
    return x.to(dtype), t


@pytest.mark.parametrize("shape", [(6, 40), (12, 700), (600, 700), (12, 32000), (600, 32003)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
def test_tokens_masked_with_the_lowest_value(dev, dtype, shape):
    x, t = masked(dev, dtype, *shape, seed=shape[1])
    lp, chosen, echosen, h, eh, _, _ = exact(x, t)
    for k in (0, 3):
        got = sd.token_logprobs(x, t, top_k=k)
        check(got.logprobs, chosen, echosen, "logprobs")
        check(got.entropy, h, eh, "entropy")
    ops.check_device_errors(dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    g, ge = (torch.randn(shape[0], generator=gen, device=dev) for _ in range(2))
    for a, b in ((g, None), (None, ge), (g, ge)):
        d = grads(x, t, a, b)
        check(d, *exact_grad(x, t, a, b), "dlogits")


def test_values_across_the_whole_range_of_fp32(dev):
    """Differences that pass the largest fp32 number: their exponential is 0."""
    x, t = make(dev, torch.float32, 4, 600, seed=2)
    low = torch.finfo(torch.float32).min
    x[0, :300] = low
    x[0, 300:] = x[0, 300:] + 1e32
    x[1, ::2] = low
    x[1, 1::2] = 3e38
    x[2, 5] = -low
    x[3, :590] = low
    t[:] = 599
    lp, chosen, echosen, h, eh, _, _ = exact(x, t)
    got = sd.token_logprobs(x, t)
    check(got.logprobs, chosen, echosen, "logprobs")
    check(got.entropy, h, eh, "entropy")
    one = torch.ones(4, device=dev)
    check(grads(x, t, one, one), *exact_grad(x, t, one, one), "dlogits")
