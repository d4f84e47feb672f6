"""What the binding of the row operators makes of its arguments, and what the C entries refuse, without a GPU."""
import pytest
import torch

import paramecia_b200 as pm
from paramecia_b200 import rows


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_ids_are_dense(dtype):
    table = torch.arange(12, dtype=dtype).reshape(3, 4)
    for t in (table, table.t(), table[:, ::2], table.t()[1:]):
        got = rows._ids("ids", t)
        assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == t.tolist()
