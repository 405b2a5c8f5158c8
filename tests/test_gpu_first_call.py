"""The first call of a process made inside a graph capture: the word in which
kernels report errors belongs to the library, not to the graph.  Needs a B200."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
dev = torch.device("cuda:0")
x = torch.randn(4, 300, device=dev)
good, bad = (torch.full((4,), t, dtype=torch.int64, device=dev) for t in (5, 900))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    kept = sd.token_logprobs(x, good)
ops.check_device_errors(dev)  # clear before any replay
graph.replay()
ops.check_device_errors(dev)
sd.token_logprobs(x, bad)
graph.replay()  # wipes no report of another call
try:
    ops.check_device_errors(dev)
except sd.SparDAError as e:
    assert "error code 2" in str(e)
else:
    raise AssertionError("the report is lost")
assert torch.equal(kept.logprobs, sd.token_logprobs(x, good).logprobs)
del graph
torch.cuda.empty_cache()
sd.token_logprobs(x, good)
ops.check_device_errors(dev)
print("fine")
"""


def test_first_call_in_a_capture(dev):
    done = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


def test_reports_say_what_happened(dev):
    import torch

    import local_research_small_language_model_b200 as sd
    from local_research_small_language_model_b200 import ops

    sd.token_logprobs(torch.zeros(2, 9, device=dev), torch.full((2,), 9, dtype=torch.int64, device=dev))
    with pytest.raises(sd.SparDAError, match="out of range .device error code 2"):
        ops.check_device_errors(dev)
