"""The bytes of the residual add + RMS norm in 8-bit floats, next to the ties of the type and in groups without a scale.

No tolerance: r * weight and the group's maximum are whole numbers here, and the nearest e4m3 value of their quotient is found in
rational arithmetic."""
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"
E4M3 = [m * Fraction(2) ** -9 for m in range(8)] + [(8 + m) * Fraction(2) ** (e - 10) for e in range(1, 16) for m in range(8) if e * 8 + m < 127]


def nearest(x):
    """The e4m3 value next to x >= 0, ties to the even one."""
    i = min(range(len(E4M3)), key=lambda i: (abs(E4M3[i] - x), i % 2))
    return float(E4M3[i])


def rows_beside_ties(n, H, seed):
    """Whole numbers below 2^24: a row's maximum top, and numbers d whose quotient 448 d / top is less than half an f32 step
    from a tie of e4m3, on either side of it."""
    rng = np.random.default_rng(seed)
    rows = np.zeros((n, H), np.int64)
    ties = np.array([(2 * m + 1) * 2 ** e for e in range(0, 6) for m in range(8, 16) if (2 * m + 1) * 2 ** e < 448 * 2], np.int64)   # twice the tie
    for row in rows:
        top = int(rng.integers(2 ** 23, 2 ** 24)) | 1
        d = (ties * top + 448) // (2 * 448)
        near = d[(np.abs(2 * 448 * d - ties * top) * 2 ** 26 <= ties * top) & (2 * 448 * d != ties * top)]
        if near.size:
            row[:] = rng.choice(near, H) * rng.choice([-1, 1], H)
        row[::32] = top           # every group has the same maximum
    return rows


@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("H", [64, 61, 1024, 9000])
def test_quotients_beside_a_tie(H, group):
    rows = rows_beside_ties(30, H, H)
    rows[0, :3] = 16576079, 629003, -629003         # 281793344 / 16576079, just above the tie of 16 and 18
    rows[0, 3:] = 16576079
    assert (rows != 0).sum() > rows.size // 2
    _, q, _, _ = pm.add_rms_norm_q8(torch.from_numpy(rows).float().to(DEV), None, None, 1e-6, group=group, q_dtype=torch.float8_e4m3fn)
    got = q.float().cpu().numpy()
    assert got[0, 1] == 18 and got[0, 2] == -18
    for row, out in zip(rows, got):
        top = int(np.abs(row).max())
        want = {int(d): nearest(Fraction(448 * abs(int(d)), top)) for d in set(row.tolist())}
        assert [np.sign(d) * want[int(d)] for d in row] == out.tolist()


@pytest.mark.parametrize("q_dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("H, group", [(512, 32), (505, 64), (9000, 128)])
def test_a_nan_weight_stays_in_its_group(H, group, q_dtype):
    """The other groups' quotients are full of ties, which the 64-bit part rounds once more; the group without a scale is zeros."""
    resid = (torch.arange(2 * H, device=DEV) % 33 - 16).float().view(2, H)        # 28 |d| of 448: 84, 168 and 336 are ties
    resid[:, ::32] = 16.0
    weight = torch.ones(H, device=DEV)
    _, q, scales, values = pm.add_rms_norm_q8(resid, None, weight, 1e-6, group=group, q_dtype=q_dtype, values_dtype=torch.float32)
    weight[group + 3] = float("nan")
    _, q2, scales2, values2 = pm.add_rms_norm_q8(resid, None, weight, 1e-6, group=group, q_dtype=q_dtype, values_dtype=torch.float32)
    inside = torch.zeros(H, dtype=torch.bool, device=DEV)
    inside[group:2 * group] = True
    assert torch.isnan(scales2[:, 1]).all() and torch.isnan(values2[:, inside]).all() and (q2[:, inside].float() == 0).all()
    scales2[:, 1] = scales[:, 1]
    assert torch.equal(scales, scales2) and torch.equal(q.float()[:, ~inside], q2.float()[:, ~inside]) and torch.equal(values[:, ~inside], values2[:, ~inside])
