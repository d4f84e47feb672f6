"""The residual add + RMS norm with an 8-bit output against its 64-bit form.

Tolerances, u = 2^-24: the sum of squares passes at most H / 64 + 16 roundings (a thread's share, then a tree), the root halves
that, and mean, root, quotient, weight and scale add five more; a quotient q is then off by half a step of its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"
U = 2.0 ** -24
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
f32, bf16 = torch.float32, torch.bfloat16


def exact(resid, delta, weight, eps, group, q_dtype):
    r = resid.double() if delta is None else (resid.double() + delta.double())
    r = r.to(torch.float32).to(resid.dtype).double() if delta is not None else r
    v = r / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    v = v if weight is None else v * weight.double()
    n, H = v.shape
    g = group or H
    G = -(-H // g)
    pad = torch.nn.functional.pad(v, (0, G * g - H)).view(n, G, g)
    return r, v, pad.abs().amax(2) / MOST[q_dtype]


def check(resid, delta, weight, group, q_dtype, values_dtype, eps=1e-6):
    n, H = resid.shape
    before = resid.clone()
    new, q, scales, values = pm.add_rms_norm_q8(resid, delta, weight, eps, group=group, q_dtype=q_dtype, values_dtype=values_dtype)
    assert torch.equal(resid, before)
    r, v, want = exact(resid, delta, weight, eps, group, q_dtype)
    assert new.dtype == resid.dtype and q.dtype == q_dtype and tuple(q.shape) == (n, H) and scales.dtype == f32
    assert torch.equal(new.double(), r)
    rel = ((H / 64 + 16) / 2 + 5) * U
    assert ((scales.double() - want).abs() <= rel * want).all()
    per = scales.double().repeat_interleave(group or H, 1)[:, :H]
    qv = q.float().double()
    assert (qv.abs() <= MOST[q_dtype]).all()
    if q_dtype == torch.int8:
        step = 0.5 * per
    else:   # e4m3: 2^-4 of the value, or half of the smallest step 2^-9
        step = torch.maximum(v.abs() * 2.0 ** -4, per * 2.0 ** -10)
    assert ((qv * per - v).abs() <= step + 2 * rel * v.abs() + 127 * U * per).all()
    if values_dtype is None:
        assert values is None
    else:
        assert torch.equal(values, (q.float() * per.float()).to(values_dtype))


@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("n, H, rt", [(400, 2048, f32), (300, 1003, bf16), (50, 9000, f32), (64, 12288, bf16), (333, 520, bf16)])
def test_8_bit_floats_are_the_rounding_of_the_exact_quotient(n, H, rt, group):
    """Products of two f32 numbers are exact in 64 bits, and one more product and quotient are off by 2^-52: no value of
    these rows lies as near to a border of e4m3, so every byte has to be equal."""
    resid, delta, weight = make(n, H, rt, bf16, H)
    weight[:7] = 1.0
    resid[1] = torch.arange(H, device=DEV).to(rt) % 31 - 15          # with delta 0: exact ties among the quotients
    delta[1] = 0
    for w in (weight, None):
        new, q, scales, _ = pm.add_rms_norm_q8(resid, delta, w, 1e-6, group=group, q_dtype=torch.float8_e4m3fn)
        d = new.double() * (1.0 if w is None else w.double())
        g = group or H
        pad = torch.nn.functional.pad(d, (0, -H % g)).view(n, -1, g)
        want = (pad * 448 / pad.abs().amax(2, keepdim=True).clamp(min=1e-300)).view(n, -1)[:, :H]
        assert torch.equal(q.float(), want.float().to(torch.float8_e4m3fn).float())


def make(n, H, rt, dt, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    resid = (torch.randn((n, H), generator=g, device=DEV) * torch.exp(torch.randn((H,), generator=g, device=DEV))).to(rt)
    delta = None if dt is None else torch.randn((n, H), generator=g, device=DEV).to(dt)
    weight = 1 + 0.3 * torch.randn((H,), generator=g, device=DEV)
    return resid, delta, weight


@pytest.mark.parametrize("q_dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("n, H", [(1, 2048), (3, 1), (2, 31), (5, 1000), (7, 2047), (33, 512), (2, 12288), (150, 4096), (4, 8200), (3, 16384), (2, 16383), (300, 264)])
def test_against_64_bits(n, H, group, q_dtype):
    check(*make(n, H, f32, f32, n + H), group, q_dtype, f32)
    check(*make(n, H, bf16, bf16, n + H + 1), group, q_dtype, bf16)


@pytest.mark.parametrize("rt, dt, vt", [(a, b, c) for a in (f32, bf16) for b in (f32, bf16, None) for c in (f32, bf16, None)])
@pytest.mark.parametrize("H", [2048, 250])
def test_types(rt, dt, vt, H):
    resid, delta, weight = make(19, H, rt, dt, 5)
    check(resid, delta, weight, 64, torch.int8, vt)
    check(resid, delta, None, 0, torch.float8_e4m3fn, vt)


def test_views_and_a_weight_of_another_type():
    resid, delta, weight = make(9, 520, f32, f32, 6)
    big = torch.zeros((9, 1041), device=DEV)
    for at in (0, 1):
        view = big[:, at:at + 520]
        view.copy_(resid)
        a = pm.add_rms_norm_q8(view, delta, weight.bfloat16(), 1e-5, group=32)
        b = pm.add_rms_norm_q8(resid, delta, weight.bfloat16().float(), 1e-5, group=32)
        assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))
    flat = torch.zeros(9 * 520 + 1, device=DEV)
    flat[1:] = resid.reshape(-1)                     # rows that begin on a 4-byte boundary only
    a = pm.add_rms_norm_q8(flat[1:].view(9, 520), delta, weight, 1e-5, group=32)
    b = pm.add_rms_norm_q8(resid, delta, weight, 1e-5, group=32)
    # another path may sum in another order: scales within the bound of two such sums
    assert torch.equal(a[0], b[0]) and ((a[2] - b[2]).abs() <= 2 * ((520 / 64 + 16) / 2 + 5) * U * b[2]).all()


@pytest.mark.parametrize("H, group", [(2048, 32), (100, 64), (2048, 0)])
@pytest.mark.parametrize("q_dtype", [torch.int8, torch.float8_e4m3fn])
def test_zeros_infinities_and_nan(H, group, q_dtype):
    resid = torch.ones((4, H), device=DEV)
    resid[0] = 0                                     # an empty row: scale 0, zeros, no NaN
    resid[2, H // 2] = float("nan")
    resid[3, H - 1] = float("inf")
    new, q, scales, values = pm.add_rms_norm_q8(resid, None, None, 1e-6, group=group, q_dtype=q_dtype, values_dtype=f32)
    assert (scales[0] == 0).all() and (q[0].float() == 0).all() and (values[0] == 0).all()
    want = MOST[q_dtype]
    assert (q[1].float() == want).all() and torch.isfinite(scales[1]).all()
    assert torch.isnan(scales[2]).all() and (q[2].float() == 0).all() and torch.isnan(values[2]).all()
    g = (H - 1) // (group or H)
    assert not torch.isfinite(scales[3, g]) and (scales[3, :g] == 0).all()     # 1 / inf = 0, inf / inf = NaN
    assert (q[3].float() == 0).all()
    assert torch.equal(new.nan_to_num(9.0), resid.nan_to_num(9.0))


def test_tiny_and_huge_rows():
    resid = torch.full((3, 256), 1e-30, device=DEV)
    resid[1] = 1e18
    resid[2] = 1e-44
    new, q, scales, values = pm.add_rms_norm_q8(resid, None, None, 0.0, group=32, values_dtype=f32)
    # 1e18^2 * 256 is finite; 1e-30^2 and 1e-44^2 are 0 in f32, so those rows are x / 0 = inf
    assert ((values[1] - 1).abs() <= 2.0 ** -20).all()
    assert not torch.isfinite(scales[0]).any() and (q[0] == 0).all()
    new, q, scales, values = pm.add_rms_norm_q8(resid, None, None, 1e-6, group=32, values_dtype=f32)
    assert torch.isfinite(values).all()


def test_no_rows_and_in_place_through_the_c_entry():
    new, q, scales, values = pm.add_rms_norm_q8(torch.zeros((0, 64), device=DEV), None, None, 1e-6, group=32, values_dtype=bf16)
    assert tuple(q.shape) == (0, 64) and tuple(scales.shape) == (0, 2)
    resid, delta, weight = make(6, 1024, bf16, bf16, 8)
    want = pm.add_rms_norm_q8(resid, delta, weight, 1e-6, group=128)
    q, scales = torch.empty_like(want[1]), torch.empty_like(want[2])
    rc = pm.lib().pmoe_add_rms_norm_q8(0, resid.data_ptr(), pm.BF16, delta.data_ptr(), pm.BF16, weight.data_ptr(), 6, 1024, 1e-6, 128,
                                       resid.data_ptr(), 24, q.data_ptr(), scales.data_ptr(), None, 0,
                                       torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(resid, want[0]) and torch.equal(q, want[1]) and torch.equal(scales, want[2])


def test_captured():
    resid, delta, weight = make(40, 2048, f32, bf16, 9)
    pm.add_rms_norm_q8(resid, delta, weight, 1e-6, group=32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pm.add_rms_norm_q8(resid, delta, weight, 1e-6, group=32)
    resid.mul_(-1.5)
    graph.replay()
    want = pm.add_rms_norm_q8(resid, delta, weight, 1e-6, group=32)
    assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))


def test_refusals():
    x = torch.zeros((4, 64), device=DEV)
    for f in (lambda: pm.add_rms_norm_q8(x[0], None, None, 1e-6), lambda: pm.add_rms_norm_q8(x, x[:3], None, 1e-6),
              lambda: pm.add_rms_norm_q8(x, x.cpu(), None, 1e-6), lambda: pm.add_rms_norm_q8(x, None, x[0, :5], 1e-6)):
        with pytest.raises(ValueError):
            f()
    for f, code in ((lambda: pm.add_rms_norm_q8(x.half(), None, None, 1e-6), -2), (lambda: pm.add_rms_norm_q8(x, x.half(), None, 1e-6), -2),
                    (lambda: pm.add_rms_norm_q8(x, None, None, 1e-6, q_dtype=torch.uint8), -2),
                    (lambda: pm.add_rms_norm_q8(x, None, None, 1e-6, values_dtype=torch.float16), -2),
                    (lambda: pm.add_rms_norm_q8(x, None, None, 1e-6, group=16), -3), (lambda: pm.add_rms_norm_q8(x, None, None, -1.0), -1),
                    (lambda: pm.add_rms_norm_q8(torch.zeros((1, 16385), device=DEV), None, None, 1e-6), -1)):
        with pytest.raises(pm.PmoeError) as e:
            f()
        assert e.value.code == code
