"""Low-rank adapters of many requests against a 64-bit form, and a run of all row operators together.

Tolerances: bf16 products are exact in f32.  Sums on the matrix units keep 24 bits but may cut instead of round: 2^-23 a
step.  A first product sees at most K / 16 + 32 steps, the second r / 16 + 8; between the two an f32 result keeps h in three
bf16 parts (nothing lost), a bf16 result in two (2^-17)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"
CUT = 2.0 ** -23
f32, bf16 = torch.float32, torch.bfloat16


def make(n, K, N, r, L, xt, bt, seed, kind="mixed"):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn((n, K), generator=g, device=DEV).to(xt)
    base = torch.randn((n, N), generator=g, device=DEV).to(bt)
    a = (torch.randn((L, r, K), generator=g, device=DEV) / K ** 0.5).to(bf16)
    b = torch.randn((L, N, r), generator=g, device=DEV).to(bf16)
    scales = 0.5 + torch.rand((L,), generator=g, device=DEV)
    if kind == "mixed":
        ids = torch.randint(-1, L + 1, (n,), generator=g, device=DEV)
    elif kind == "one":
        ids = torch.full((n,), L - 1, device=DEV)
    elif kind == "none":
        ids = torch.randint(0, 2, (n,), generator=g, device=DEV) * (L + 1) - 1
    else:   # runs
        ids = (torch.arange(n, device=DEV) * L) // max(n, 1)
    return base, x, a, b, ids.int(), scales


def check(base, x, a, b, ids, scales, got):
    (L, r, K), N = a.shape, b.shape[1]
    want = base.double()
    size = torch.zeros_like(want)
    first = torch.zeros_like(want)
    for i in range(L):
        t = torch.nonzero(ids == i)[:, 0]
        s = 1.0 if scales is None else float(scales[i])
        A, B, X = a[i].double(), b[i].double(), x[t].double()
        h = X @ A.t()
        want[t] += s * (h @ B.t())
        size[t] = s * (h.abs() @ B.abs().t())                       # of the second product
        first[t] = s * ((X.abs() @ A.abs().t()) @ B.abs().t())      # what errors of the first become
    tol = (K / 16 + 32) * CUT * first + (r / 16 + 8) * CUT * size + 2.0 ** -24 * (want.abs() + 4 * size)
    if base.dtype == bf16:
        tol = tol + 2.0 ** -17 * size + 2.0 ** -8 * (want.abs() + tol)
    assert got.dtype == base.dtype
    assert ((got.double() - want).abs() <= tol).all()
    bare = (ids < 0) | (ids >= L)
    assert torch.equal(got[bare], base[bare])


SHAPES = [(1, 2048, 2048, 16, 8, "one"), (1, 64, 64, 8, 1, "none"), (2, 2048, 512, 64, 3, "mixed"), (17, 1000, 504, 24, 5, "mixed"),
          (64, 2048, 4096, 32, 48, "mixed"), (100, 512, 2048, 128, 2, "one"), (333, 264, 520, 40, 300, "mixed"), (5, 8, 8, 8, 2, "mixed"),
          (1024, 512, 512, 16, 7, "runs"), (1025, 512, 520, 16, 7, "mixed"), (3001, 512, 1024, 64, 4, "runs"), (2000, 256, 256, 8, 4000, "mixed"),
          (5000, 128, 264, 112, 3, "one"), (2000, 264, 136, 32, 5, "mixed"), (700, 8, 8, 8, 1, "one"), (1030, 72, 1000, 16, 8, "runs"), (130, 1024, 1024, 64, 1, "mixed"), (1500, 520, 64, 56, 9, "none"), (129, 4096, 72, 120, 1, "one")]


@pytest.mark.parametrize("xt, bt", [(f32, f32), (bf16, bf16), (f32, bf16), (bf16, f32)])
@pytest.mark.parametrize("n, K, N, r, L, kind", SHAPES)
def test_against_64_bits(n, K, N, r, L, kind, xt, bt):
    base, x, a, b, ids, scales = make(n, K, N, r, L, xt, bt, n + K, kind)
    before = base.clone()
    got = pm.adapters_add(base, x, a, b, ids, scales=scales)
    assert torch.equal(base, before)
    check(base, x, a, b, ids, scales, got)


def test_order_in_place_views_and_no_scales():
    base, x, a, b, ids, _ = make(70, 512, 256, 16, 6, f32, f32, 3)
    want = pm.adapters_add(base, x, a, b, ids)
    check(base, x, a, b, ids, None, want)
    order = pm.sort_by_expert(ids, 6)
    got = pm.adapters_add(base, x, a, b, ids.long(), order=order)
    check(base, x, a, b, ids, None, got)
    wide = torch.zeros((70, 515), device=DEV)
    wide[:, 3:] = x                                        # rows that begin anywhere
    assert torch.equal(pm.adapters_add(base, wide[:, 3:], a, b, ids), want)
    flat = torch.zeros(70 * 512 + 1, device=DEV)
    flat[1:] = x.reshape(-1)
    assert torch.equal(pm.adapters_add(base, flat[1:].view(70, 512), a, b, ids), want)
    assert pm.adapters_add(base, x, a, b, ids, out=base) is base and torch.equal(base, want)


def test_other_rows_are_not_touched_by_a_bad_one():
    base, x, a, b, ids, scales = make(40, 256, 256, 16, 4, bf16, bf16, 4)
    want = pm.adapters_add(base, x, a, b, ids, scales=scales)
    x[7] = float("nan")
    x[9] = float("inf")
    ids[7], ids[9] = 2, 2
    a[3] = float("nan")
    got = pm.adapters_add(base, x, a, b, ids, scales=scales)
    same = (ids != 3) & (torch.arange(40, device=DEV) != 7) & (torch.arange(40, device=DEV) != 9)
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[7]).all() and torch.isnan(got[ids == 3]).all() and not torch.isfinite(got[9]).any()


@pytest.mark.parametrize("n, L, xt", [(90, 5, f32), (500, 3, bf16), (500, 200, bf16), (1024, 2, f32), (3000, 4, bf16)])
def test_with_and_without_the_order_and_twice(n, L, xt):
    """Grouped by the sort, by the kernel itself, and once more on another stream: the same rows meet in the same tiles, so the
    bits are equal wherever the tiles are."""
    base, x, a, b, ids, scales = make(n, 512, 264, 48, L, xt, f32, n + L)
    order = pm.sort_by_expert(ids, L)
    first = pm.adapters_add(base, x, a, b, ids, scales=scales, order=order)
    again = pm.adapters_add(base, x, a, b, ids, scales=scales, order=order)
    assert torch.equal(first, again)
    check(base, x, a, b, ids, scales, first)
    check(base, x, a, b, ids, scales, pm.adapters_add(base, x, a, b, ids, scales=scales))
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        other = pm.adapters_add(base, x, a, b, ids, scales=scales, order=order)
    side.synchronize()
    assert torch.equal(first, other)
    pm.rows_status(DEV)


def test_no_rows_and_long_rows():
    base, x, a, b, ids, scales = make(0, 64, 64, 8, 2, f32, f32, 5)
    assert tuple(pm.adapters_add(base, x, a, b, ids, scales=scales).shape) == (0, 64)
    base, x, a, b, ids, scales = make(3, 20000, 16, 16, 2, bf16, f32, 6)
    check(base, x, a, b, ids, scales, pm.adapters_add(base, x, a, b, ids, scales=scales))
    base, x, a, b, ids, scales = make(3, 16, 20000, 16, 2, f32, bf16, 7)
    check(base, x, a, b, ids, scales, pm.adapters_add(base, x, a, b, ids, scales=scales))


@pytest.mark.parametrize("n", [48, 1500])
def test_captured_with_new_ids(n):
    base, x, a, b, ids, scales = make(n, 512, 512, 32, 10, bf16, bf16, 8)
    pm.adapters_add(base, x, a, b, ids, scales=scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pm.adapters_add(base, x, a, b, ids, scales=scales)
    for seed in (9, 10):
        _, x2, _, _, ids2, _ = make(n, 512, 512, 32, 10, bf16, bf16, seed, "mixed" if seed == 9 else "none")
        x.copy_(x2)
        ids.copy_(ids2)
        graph.replay()
        assert torch.equal(got, pm.adapters_add(base, x, a, b, ids, scales=scales))


def test_refusals():
    base, x, a, b, ids, scales = make(4, 64, 64, 16, 3, f32, f32, 11)
    order = pm.sort_by_expert(ids, 4)
    for f in (lambda: pm.adapters_add(base, x[:3], a, b, ids), lambda: pm.adapters_add(base[:, :8], x, a, b, ids),
              lambda: pm.adapters_add(base, x, a, b[:2], ids), lambda: pm.adapters_add(base, x, a[0], b, ids),
              lambda: pm.adapters_add(base, x, a, b, ids[:2]), lambda: pm.adapters_add(base, x, a, b, ids.cpu()),
              lambda: pm.adapters_add(base, x, a, b, ids, scales=scales[:2]), lambda: pm.adapters_add(base, x, a, b, ids, order=order),
              lambda: pm.adapters_add(base, x, a, b, ids, out=x), lambda: pm.adapters_add(base[:3], x[:3], a, b, ids[:3], out=base[1:]),
              lambda: pm.adapters_add(base, x, a, b, ids, out=base.bfloat16()), lambda: pm.adapters_add(base, x, a, b, ids, out=x[:2])):
        with pytest.raises(ValueError):
            f()
    for f, code in ((lambda: pm.adapters_add(base, x, a.float(), b, ids), -2), (lambda: pm.adapters_add(base, x.half(), a, b, ids), -2),
                    (lambda: pm.adapters_add(base, x, a, b, ids.float()), -2),
                    (lambda: pm.adapters_add(base, x, a[:, :12].contiguous(), b[:, :, :12].contiguous(), ids), -3),
                    (lambda: pm.adapters_add(base[:, :60].contiguous(), x, a, b[:, :60].contiguous(), ids), -3)):
        with pytest.raises(pm.PmoeError) as e:
            f()
        assert e.value.code == code


@pytest.mark.parametrize("n", [1, 37])
def test_the_operators_together_around_the_experts(n):
    """A host's own mixture-of-experts step: norm to 8 bits, route, rows and scales to the experts in 8 bits, the experts'
    products (here the library's own quantised blocks, dequantised) with one adapter per expert beside the down projection,
    and back with the weights and the shared row -- against the same in 64 bits from the 8-bit rows on."""
    from paramecia_b200 import synth

    t = synth.make_layer(E=16, k=4, preset="q4k_m", seed=3)
    blk = synth.make_block(t, DEV, max_tokens=64)
    E, k, H, F = 16, 4, 2048, 512
    g = torch.Generator(device=DEV)
    g.manual_seed(12)
    resid = torch.randn((n, H), generator=g, device=DEV)
    delta = torch.randn((n, H), generator=g, device=DEV)
    new, q, s, y = pm.add_rms_norm_q8(resid, delta, None, 1e-6, group=32, values_dtype=f32)
    logits, w, idx = blk.route(y)
    o = pm.sort_by_expert(idx, E)
    xs = pm.dispatch_rows(q, o).float() * pm.dispatch_rows(s, o).repeat_interleave(32, 1)
    assert torch.equal(xs, pm.dispatch_rows(y, o))
    deq = {nm: pm.QTensor(t[nm].to(DEV), t[f"{nm}_dtype"], shp).dequantize() for nm, shp in
           (("gate", (E, F, H)), ("up", (E, F, H)), ("down", (E, H, F)))}
    off = o.offsets.tolist()
    act = torch.empty((n * k, F), device=DEV)
    rows = torch.empty((n * k, H), device=DEV)
    for e in range(E):
        m = slice(off[e], off[e + 1])
        act[m] = torch.nn.functional.silu(xs[m] @ deq["gate"][e].t()) * (xs[m] @ deq["up"][e].t())
        rows[m] = act[m] @ deq["down"][e].t()
    a = (torch.randn((E, 16, F), generator=g, device=DEV) / F ** 0.5).bfloat16()
    b = torch.randn((E, H, 16), generator=g, device=DEV).bfloat16()
    ids = idx.reshape(-1)[o.order.long()]
    pm.adapters_add(rows, act, a, b, ids, out=rows)
    shared = blk.shared_forward(y)
    out = pm.combine_rows(rows, o, w, extra=shared)
    blk.status()

    y64 = q.double() * s.double().repeat_interleave(32, 1)
    want = shared.double()
    for tok in range(n):
        for j in range(k):
            e = int(idx[tok, j])
            h = torch.nn.functional.silu(deq["gate"][e].double() @ y64[tok]) * (deq["up"][e].double() @ y64[tok])
            want[tok] += float(w[tok, j]) * (deq["down"][e].double() @ h + b[e].double() @ (a[e].double() @ h))
    # f32 throughout: the longest sums have 2048 + 512 terms, an error below (2048 + 512) * 2^-24 of sums of magnitudes that
    # exceed the result by about sqrt(2048): 7e-3 at the very worst, 2^-24 * sqrt(2560) * a few in earnest
    assert float((out.double() - want).norm() / want.norm()) <= 1e-5
