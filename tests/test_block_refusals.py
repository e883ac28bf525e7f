"""Sizes that the block operators refuse before anything is allocated or launched: counts that a 32-bit argument of the C
calls would cut to another, valid one. The tensors are of the meta device and claim to be on the GPU."""
import ctypes as C

import pytest
import torch

from amdsplat import _lib, dropout, gated_scan
from test_block_errors import ARG, WORKSPACE, expect, linear_args


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


@pytest.mark.parametrize("kw", [dict(x_stride=32), dict(weight_stride=0), dict(x_stride=0), dict(rows=16, x_stride=60)])
def test_a_projections_gradient_of_rows_that_overlap(kw):
    """(In Python they are copied first.) A single row has any stride."""
    L = _lib.lib()
    a = linear_args(**kw)
    expect(L.gs_linear_bwd(C.byref(a), 256, 256, 256, 256, 256, 1 << 62, None), ARG, "overlap")
    one = linear_args(rows=1, outputs=1, x_stride=0, weight_stride=0)
    expect(L.gs_linear_bwd(C.byref(one), 256, 256, 256, 256, None, 0, None), WORKSPACE, "workspace")
