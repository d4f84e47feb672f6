"""Low-rank adapters at values where the bits of h and the special values matter.  Everything is chosen so that f32 sums are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"
f32, bf16 = torch.float32, torch.bfloat16
TYPES = [(f32, f32), (bf16, bf16), (f32, bf16), (bf16, f32)]
ROWS = [1, 40, 300]      # a tile of sixteen rows; more than one; tiles of 128 rows where x is bf16


@pytest.mark.parametrize("xt, bt", TYPES)
@pytest.mark.parametrize("r", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("n", ROWS)
def test_h_keeps_the_bits_of_f32(n, r, xt, bt):
    """h = (1 + 2^-9 + 2^-18, 1 + 2^-9, 0, ...) and B's rows (1, -1, 0, ...): the difference of the two is 2^-18."""
    K, N = 64, 72
    x = torch.zeros((n, K), device=DEV)
    x[:, 3], x[:, 20], x[:, 50] = 1.0, 2.0 ** -9, 2.0 ** -18
    a = torch.zeros((1, r, K), dtype=bf16, device=DEV)
    a[0, 0, 3] = a[0, 0, 20] = a[0, 0, 50] = 1.0
    a[0, 1, 3] = a[0, 1, 20] = 1.0
    b = torch.zeros((1, N, r), dtype=bf16, device=DEV)
    b[0, :, 0], b[0, :, 1] = 1.0, -1.0
    got = pm.adapters_add(torch.zeros((n, N), dtype=bt, device=DEV), x.to(xt), a, b, torch.zeros(n, dtype=torch.int32, device=DEV))
    assert torch.equal(got, torch.full_like(got, 2.0 ** -18))
