"""trs_view structs made in Python (tensorrs_b200/abi.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

BASE = 1 << 24


@pytest.mark.parametrize("shape,strides", [
    ([2, 3], None), ((2.0, 3.0), None), ([np.int64(2), np.float64(3)], [np.int32(3), 1.0]), (torch.Size([2, 3]), (3, 1)),
    (torch.tensor([2, 3]), torch.tensor([3, 1]))], ids=str)
def test_make_view_takes_what_int_takes(trs, shape, strides):
    v = trs.make_view(BASE, trs.F32, shape, strides, 4)
    assert (v.data, v.dtype, v.ndim, v.offset, v.storage_len) == (BASE, trs.F32, 2, 4, 10)
    assert list(v.shape) == [2, 3] + [0] * (trs.MAX_DIMS - 2) and list(v.strides) == [3, 1] + [0] * (trs.MAX_DIMS - 2)


def test_make_view_refuses_more_dimensions_than_it_holds(trs):
    assert trs.make_view(BASE, trs.F32, [1] * trs.MAX_DIMS).ndim == trs.MAX_DIMS
    with pytest.raises(IndexError):
        trs.make_view(BASE, trs.F32, [1] * (trs.MAX_DIMS + 1))
