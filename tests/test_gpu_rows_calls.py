"""Calls of the row operators beside the plain ones: transposed ids, several threads at once, orders of another slice, outputs over
inputs.  Places and copies are exact."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"


def plain_places(idx, E):
    """The place of each pair of idx [n, k] (a numpy array, ids in [0, E)) in stable expert order."""
    order = np.argsort(idx.reshape(-1), kind="stable")
    place = np.empty(idx.size, np.int64)
    place[order] = np.arange(idx.size)
    return place.reshape(idx.shape)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n, k, E", [(7, 4, 5), (1, 10, 512), (333, 2, 60), (900, 10, 512)])
def test_transposed_ids(n, k, E, dtype):
    idx = np.random.default_rng(n).integers(0, E, (n, k))
    slots_first = torch.from_numpy(idx.T.copy()).to(DEV, dtype)      # [k, n]
    o = pm.sort_by_expert(slots_first.t(), E)
    assert np.array_equal(o.place.cpu().numpy(), plain_places(idx, E))
    every_other = torch.full((n, 2 * k), -1, dtype=dtype, device=DEV)
    every_other[:, ::2] = slots_first.t()
    o = pm.sort_by_expert(every_other[:, ::2], E)
    assert np.array_equal(o.place.cpu().numpy(), plain_places(idx, E))
