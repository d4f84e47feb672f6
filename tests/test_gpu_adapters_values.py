"""Low-rank adapters at values where the bits of h and the special values matter.  Values are chosen so that f32 sums are exact, but for
one sum whose bound stands beside it."""
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


@pytest.mark.parametrize("xt, bt", TYPES)
@pytest.mark.parametrize("r", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("n", ROWS)
def test_infinities_stay_infinities(n, r, xt, bt):
    """With A and B positive an infinity of x, or of a sum that overflows, is one of the same sign in its row, whatever lies behind
    the rank and behind K; the largest numbers stay numbers, and a NaN is one, be it in the lowest bits."""
    K, N, inf = 72, 40, float("inf")
    most = torch.finfo(xt).max
    a = torch.full((1, r, K), 2.0 ** -8, dtype=bf16, device=DEV)
    b = torch.full((1, N, r), 2.0 ** -9, dtype=bf16, device=DEV)
    x = torch.zeros((n, K), dtype=xt, device=DEV)
    at = [0, n // 3, n // 2, n - 1]
    for first, value, want in ((0, inf, inf), (1, -inf, -inf), (2, most, None), (3, float("nan"), float("nan"))):
        x.zero_()
        x[at[first], 5] = value
        if value != value and xt == f32:
            x.view(torch.int32)[at[first], 5] = 0x7f800001
        got = pm.adapters_add(torch.zeros((n, N), dtype=bt, device=DEV), x, a, b, torch.zeros(n, dtype=torch.int32, device=DEV))
        row = got[at[first]].clone()
        got[at[first]] = 0
        assert (got == 0).all()
        if want is None:
            # h is exact; the second product adds r equal terms in three pieces.  Three such terms of 24 bits need 26, so partial sums
            # are not exact: the matrix unit aligns the seventeen addends of a step of sixteen ranks and cuts each at 2^-23 of the sum
            # at most, in 3 * ceil(r / 16) steps.  Then one rounding to the result's type.
            exact = most * 2.0 ** -17 * r
            assert ((row.double() - exact).abs() <= (3 * -(-r // 16) * 17 * 2.0 ** -23 + torch.finfo(bt).eps / 2) * exact).all()
        else:
            assert torch.equal(row.float().nan_to_num(7.0, 8.0, 9.0), torch.full_like(row.float(), want).nan_to_num(7.0, 8.0, 9.0))
    x.zero_()
    x[0, :2] = most     # both h and the result overflow
    got = pm.adapters_add(torch.zeros((n, N), dtype=bt, device=DEV), x, a * 2.0 ** 9, b * 2.0 ** 9, torch.zeros(n, dtype=torch.int32, device=DEV))
    assert (got[0] == inf).all() and (got[1:] == 0).all()
