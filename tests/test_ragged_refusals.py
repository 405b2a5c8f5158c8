"""Calls that the ragged-batch operators refuse before any launch (no GPU)."""

import pytest
import torch

import local_research_small_language_model_b200 as sd
from local_research_small_language_model_b200 import ops
from tests.test_ragged_host import CU, INVALID, backward, packed, z


@pytest.mark.parametrize("call", [packed, backward])
def test_rest_belongs_to_16_bit_types(call):
    """fp32 has no rounding to keep: a rest would be left unwritten."""
    assert call(sd.load_library(), dtype=0) == INVALID
    f = [z(10, h, 64, dtype=torch.float32) for h in (4, 2, 2)]
    rest = z(10, 4, 64, dtype=torch.float32)
    with pytest.raises(TypeError, match="rest"):
        if call is packed:
            ops.packed_attention(*f, CU, rest=rest)
        else:
            ops.packed_attention_backward(*f, rest, rest, z(4, 10, dtype=torch.float32), CU, rest=rest)
