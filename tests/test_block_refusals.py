"""Sizes that the block operators refuse before anything is allocated or launched: counts that a 32-bit argument of the C
calls would cut to another, valid one. The tensors are of the meta device and claim to be on the GPU."""
import pytest
import torch

from amdsplat import dropout, gated_scan


class Claimed(torch.Tensor):
    is_cuda = True


def claimed(*shape, dtype=torch.float32):
    return torch.empty(shape, device="meta", dtype=dtype).as_subclass(Claimed)


@pytest.mark.parametrize("width", [1 << 31, (1 << 31) + 5, 1 << 32, (1 << 32) + 5])
@pytest.mark.parametrize("grad", [False, True])
def test_dropout_over_a_long_dimension(width, grad):
    """2^32 + 5 columns would be taken as 5, and the rest of the result never be written."""
    for shape in ((width,), (1, width), (3, 2, width)):
        with pytest.raises(ValueError, match="last dimension"):
            dropout(claimed(*shape, dtype=torch.bfloat16).requires_grad_(grad), 0.5, 1)


@pytest.mark.parametrize("docs", [1 << 30, 1 << 32, (1 << 32) + 2])
def test_a_recurrence_over_many_documents(docs):
    """2^32 + 2 documents would be taken as 2, and the other documents' states never be written."""
    x, offsets = claimed(10, 8), claimed(docs + 1, dtype=torch.int32)
    for initial in (None, claimed(docs, 8)):
        with pytest.raises(ValueError, match="documents"):
            gated_scan(x, x, offsets=offsets, initial=initial, return_state=True)
