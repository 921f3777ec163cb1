"""How the paged cache's calls describe a tensor of rows to the kernels: on host tensors, without a device call."""
import pytest
import torch

from next_step_ai_amd.kv_cache import _rows

CPU = torch.device("cpu")


@pytest.mark.parametrize("shape,stride,offset", [
    ((1, 2, 64), (1003, 64, 1), 0),   # one token of a projection whose rows are of odd length
    ((1, 2, 64), (1003, 77, 1), 0),
    ((1, 1, 64), (5, 7, 1), 0),
    ((3, 1, 64), (72, 77, 1), 0),     # one head of rows that may be read where they lie
    ((3, 1, 64), (131, 3, 1), 0),
    ((0, 2, 64), (5, 3, 1), 0),
    ((3, 2, 64), (131, 64, 1), 0),
    ((3, 2, 64), (256, 128, 2), 0),
    ((3, 2, 64), (0, 0, 1), 0),       # the same row for all
    ((1, 2, 64), (1003, 64, 1), 4),   # an address that is not a multiple of 16 bytes
    ((3, 2, 64), (192, 64, 1), 0),
    ((1, 2, 64), (128, 64, 1), 0),
])
def test_strides_that_the_kernels_take(shape, stride, offset):
    """Whatever a tensor's strides are, those that go to the kernels are multiples of 8 elements, its address one of 16
    bytes, and its rows are found there; no copy where the tensor itself can be read."""
    t = torch.arange(4096, dtype=torch.float16).as_strided(shape, stride, offset)
    kept, address, row, head = _rows(t, "q", shape[1], shape[2], CPU)
    assert row % 8 == 0 and head % 8 == 0 and address == kept.data_ptr() and (address % 16 == 0 or shape[0] == 0)
    seen = torch.as_strided(kept, shape, (row, head, 1), kept.storage_offset())
    assert torch.equal(seen, t)
    readable = offset % 8 == 0 and stride[2] == 1 and (shape[0] <= 1 or stride[0] % 8 == 0) and (shape[1] == 1 or stride[1] % 8 == 0)
    assert (kept is t) == readable or shape[0] == 0
