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


@pytest.mark.parametrize("shape,dim", [((1, 4, 64), 0), ((9, 1, 64), 1), ((1, 1, 16, 64), 0), ((1, 1, 16, 64), 1),
                                       ((3, 1, 1, 64), 2)], ids=str)
@pytest.mark.parametrize("stride", [0, 3, 1021])
def test_the_stride_of_a_single_row_does_not_matter(shape, dim, stride):
    """Kernels get the tensor's own memory, with a stride that they accept."""
    for dtype in (torch.bfloat16, torch.float32):
        t = z(*shape, dtype=dtype)
        strides = list(t.stride())
        strides[dim] = stride
        t = t.as_strided(shape, strides)
        rows = ops._rows16(t)
        assert rows.data_ptr() == t.data_ptr() and rows.shape == t.shape
        assert all(s > 0 and s * t.element_size() % 16 == 0 for s in rows.stride()[:-1]) and rows.stride(-1) == 1
        assert ops._rows16_of("out", t).data_ptr() == t.data_ptr()
