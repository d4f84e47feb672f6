"""Sort by expert, dispatch, combine and their gradients against plain numpy / 64-bit forms.

Tolerances: a copy, a place and a zero are exact.  With u = 2^-24 an f32 sum of m products differs from the exact one by
at most m roundings of partial sums that are no larger than sum |terms| (m * u * sum |terms|); a result rounded to a type is
off by half a step more, finfo(type).eps / 2 of its value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import paramecia_b200 as pm

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def plain_sort(idx, E, base=0):
    key = idx.astype(np.int64).reshape(-1) - base
    kept = (key >= 0) & (key < E)
    pairs = np.nonzero(kept)[0]
    pairs = pairs[np.argsort(key[pairs], kind="stable")]
    order = np.full(key.size, -1, np.int64)
    order[:pairs.size] = pairs
    place = np.full(key.size, -1, np.int64)
    place[pairs] = np.arange(pairs.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key[kept], minlength=E))])
    return order, place.reshape(idx.shape), offsets


def make_idx(n, k, E, kind, seed):
    rng = np.random.default_rng(seed)
    if kind == "uniform":
        return rng.integers(0, E, (n, k)).astype(np.int32)
    if kind == "one":          # every pair to one expert
        return np.full((n, k), E - 1, np.int32)
    if kind == "none":         # nobody's expert
        return np.full((n, k), E, np.int32)
    if kind == "mixed":        # out-of-range and negative ids among them, the extremes too
        idx = rng.integers(-2, E + 2, (n, k)).astype(np.int32)
        idx.reshape(-1)[::7] = np.int32(-2 ** 31)
        idx.reshape(-1)[3::11] = np.int32(2 ** 31 - 1)
        return idx
    z = np.minimum(rng.zipf(1.3, (n, k)) - 1, E - 1)   # "skewed"
    return z.astype(np.int32)


SORTS = [(1, 1, 1, "uniform"), (1, 10, 512, "uniform"), (1, 3, 4096, "one"), (3, 1, 2, "none"), (31, 1, 8, "mixed"), (64, 10, 512, "skewed"),
         (33, 31, 60, "mixed"), (1000, 8, 60, "one"), (4096, 10, 512, "uniform"), (4099, 10, 512, "mixed"), (5000, 3, 4096, "skewed"),
         (2500, 4, 1025, "uniform"), (40000, 10, 512, "skewed"), (200001, 2, 1, "mixed"), (70000, 8, 1024, "uniform")]


@pytest.mark.parametrize("n, k, E, kind", SORTS)
def test_sort(n, k, E, kind):
    idx = make_idx(n, k, E, kind, n + k)
    o = pm.sort_by_expert(torch.from_numpy(idx).to(DEV), E)
    order, place, offsets = plain_sort(idx, E)
    assert np.array_equal(o.offsets.cpu().numpy(), offsets)
    assert np.array_equal(o.order.cpu().numpy(), order)
    assert np.array_equal(o.place.cpu().numpy(), place)


@pytest.mark.parametrize("n, k, E, base", [(1, 10, 128, 384), (777, 10, 128, 256), (20000, 4, 64, 1)])
def test_sort_of_a_slice_and_wide_ids(n, k, E, base):
    idx = make_idx(n, k, 512, "uniform", 5)
    want = plain_sort(idx, E, base)
    wide = torch.from_numpy(idx.astype(np.int64)).to(DEV)
    got = pm.sort_by_expert(wide, E, expert_base=base)
    for a, b in zip((got.order, got.place, got.offsets), want):
        assert np.array_equal(a.cpu().numpy(), b)
    wide[0, 0] = 2 ** 32 + base      # not expert `base`
    idx[0, 0] = -1
    got = pm.sort_by_expert(wide, E, expert_base=base)
    assert np.array_equal(got.place.cpu().numpy(), plain_sort(idx, E, base)[1])


def test_sort_of_nothing():
    o = pm.sort_by_expert(torch.zeros((0, 4), dtype=torch.int32, device=DEV), 9)
    assert o.offsets.tolist() == [0] * 10 and o.order.numel() == 0 and tuple(o.place.shape) == (0, 4)
    x = torch.zeros((0, 16), device=DEV)
    assert tuple(pm.dispatch_rows(x, o).shape) == (0, 16)
    assert tuple(pm.combine_rows(x, o).shape) == (0, 16)
    gr, gw = pm.combine_rows_grad(x, x, o)
    assert tuple(gr.shape) == (0, 16) and tuple(gw.shape) == (0, 4)


def rows_case(n, k, E, kind, seed=0):
    idx = torch.from_numpy(make_idx(n, k, E, kind, seed)).to(DEV)
    return pm.sort_by_expert(idx, E)


CASES = [(1, 10, 512, "uniform", 2048), (5, 2, 3, "mixed", 7), (61, 10, 512, "skewed", 2048), (130, 3, 60, "mixed", 1407),
         (17, 1, 4, "none", 64), (300, 8, 64, "uniform", 520), (9, 32, 16, "mixed", 4096), (2, 2, 8, "uniform", 1), (700, 4, 16, "mixed", 1000),
         (4, 3, 5, "mixed", 20000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8, torch.float64])
@pytest.mark.parametrize("n, k, E, kind, H", CASES)
def test_dispatch(n, k, E, kind, H, dtype):
    o = rows_case(n, k, E, kind)
    x = torch.randint(-100, 100, (n, H), generator=gen(1), device=DEV).to(dtype)
    out = torch.full((n * k, H), 77, dtype=dtype, device=DEV)
    assert pm.dispatch_rows(x, o, out=out) is out
    pair = o.order.long()
    want = torch.where((pair >= 0)[:, None], x[pair.clamp(min=0) // k], torch.zeros((), dtype=dtype, device=DEV))
    assert torch.equal(out, want)
    assert torch.equal(pm.dispatch_rows(x, o), want)


def test_dispatch_of_views():
    o = rows_case(40, 4, 8, "mixed")
    pool = torch.randn((41 * 64 + 1,), generator=gen(2), device=DEV)
    for x in (pool[1:1 + 40 * 64].view(40, 64), pool[:40 * 64].view(64, 40).t(), pool[:41 * 64].view(41, 64)[1:], pool[:40 * 64].view(40, 64)[:, 3:60]):
        pair = o.order.long()
        want = torch.where((pair >= 0)[:, None], x[pair.clamp(min=0) // 4], torch.zeros((), device=DEV))
        assert torch.equal(pm.dispatch_rows(x, o), want)
    out = torch.full((160 * 64 + 1,), 5.0, device=DEV)
    pm.dispatch_rows(pool[:40 * 64].view(40, 64), o, out=out[1:].view(160, 64))     # 4-byte aligned only
    assert out[0] == 5.0 and torch.equal(out[1:].view(160, 64), pm.dispatch_rows(pool[:40 * 64].view(40, 64), o))


def exact_combine(rows, place, w, extra):
    picked = rows.double()[place.long().clamp(min=0)]
    terms = picked * (1.0 if w is None else w.double()[:, :, None])
    terms = torch.where((place >= 0)[:, :, None], terms, 0.0)
    out, size = terms.sum(1), terms.abs().sum(1)
    return (out, size) if extra is None else (out + extra.double(), size + extra.double().abs())


@pytest.mark.parametrize("rt, et, ot", [(a, b, c) for a in TYPES for b in TYPES + [None] for c in TYPES])
@pytest.mark.parametrize("n, k, E, kind, H", CASES)
def test_combine(n, k, E, kind, H, rt, et, ot):
    o = rows_case(n, k, E, kind, 3)
    g = gen(4)
    rows = torch.randn((n * k, H), generator=g, device=DEV).to(rt)
    rows[int(o.offsets[-1]):] = float("nan")        # rows that belong to no pair are not read
    w = torch.rand((n, k), generator=g, device=DEV) if et is not None or n % 2 else None
    extra = None if et is None else torch.randn((n, H), generator=g, device=DEV).to(et)
    out = pm.combine_rows(rows, o, w, extra=extra, out_dtype=ot)
    assert out.dtype == ot
    want, size = exact_combine(torch.nan_to_num(rows), o.place, w, extra)
    tol = (k + 2) * U * size + half_step(ot) * (want.abs() + (k + 2) * U * size) * (ot != torch.float32)
    assert ((out.double() - want).abs() <= tol).all()


def test_combine_into_extra():
    o = rows_case(50, 4, 8, "mixed", 6)
    rows = torch.randn((200, 96), generator=gen(7), device=DEV)
    extra = torch.randn((50, 96), generator=gen(8), device=DEV)
    want = pm.combine_rows(rows, o, extra=extra)
    assert pm.combine_rows(rows, o, extra=extra, out=extra) is extra and torch.equal(extra, want)


@pytest.mark.parametrize("gt", TYPES)
@pytest.mark.parametrize("rt", TYPES)
@pytest.mark.parametrize("n, k, E, kind, H", CASES)
def test_combine_grad(n, k, E, kind, H, rt, gt):
    o = rows_case(n, k, E, kind, 9)
    g = gen(10)
    rows = torch.randn((n * k, H), generator=g, device=DEV).to(rt)
    total = int(o.offsets[-1])
    rows[total:] = float("nan")
    dout = torch.randn((n, H), generator=g, device=DEV).to(gt)
    w = torch.rand((n, k), generator=g, device=DEV) if n != 300 else None
    drows, dw = pm.combine_rows_grad(dout, rows, o, w)
    assert drows.dtype == rt and dw.dtype == torch.float32
    pair = o.order.long().clamp(min=0)
    kept = o.order >= 0
    spread = dout.double()[pair // k]
    want = torch.where(kept[:, None], spread * (1.0 if w is None else w.double().reshape(-1)[pair][:, None]), 0.0)
    # one f32 product, rounded once more to the rows' type
    assert ((drows.double() - want).abs() <= (U + half_step(rt) * (rt != torch.float32) * (1 + U)) * want.abs()).all()
    terms = torch.where(kept[:, None], spread * torch.nan_to_num(rows).double(), 0.0)
    dots, size = terms.sum(1), terms.abs().sum(1)
    place = o.place.long()
    want = torch.where(place >= 0, dots[place.clamp(min=0)], 0.0)
    # a partial sum sees at most H / 32 + 16 roundings: a lane's share of the row, then the tree
    tol = torch.where(place >= 0, (H / 32 + 16) * U * size[place.clamp(min=0)], 0.0)
    assert ((dw.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n, k, H", [(13, 3, 40), (6, 2, 33)])
def test_gradients_against_differences(n, k, H):
    """combine is linear in the rows and in the weights, dispatch in x: a central difference over a step of one is exact
    but for roundings, here of a few units in 2^-24 of sums below 4 * k * sqrt(H)."""
    o = rows_case(n, k, 5, "mixed", 11)
    g = gen(12)
    rows, dout, x, dxs = (torch.randn(s, generator=g, device=DEV) for s in ((n * k, H), (n, H), (n, H), (n * k, H)))
    w = torch.rand((n, k), generator=g, device=DEV)

    def loss(rows, w):
        return (pm.combine_rows(rows, o, w).double() * dout.double()).sum()

    def loss_x(x):
        return (pm.dispatch_rows(x, o).double() * dxs.double()).sum()

    drows, dw = pm.combine_rows_grad(dout, rows, o, w)
    dx = pm.dispatch_rows_grad(dxs, o)
    rng = np.random.default_rng(1)
    for v, d, f in ((rows, drows, lambda v: loss(v, w)), (w, dw, lambda v: loss(rows, v)), (x, dx, loss_x)):
        for at in rng.integers(0, v.numel(), 12):
            step = torch.zeros(v.numel(), device=DEV)
            step[at] = 1.0
            step = step.view_as(v)
            diff = (f(v + step) - f(v - step)) / 2
            assert abs(float(diff) - float(d.reshape(-1)[at])) <= 64 * U * 4 * k * H
    gone = o.order < 0
    assert (drows[gone] == 0).all() and (dw[o.place < 0] == 0).all()


def test_repeated_calls_give_the_same_bits():
    o = [rows_case(500, 10, 64, "skewed", 13) for _ in range(2)]
    rows = torch.randn((5000, 1001), generator=gen(14), device=DEV)
    dout = torch.randn((500, 1001), generator=gen(15), device=DEV)
    w = torch.rand((500, 10), generator=gen(16), device=DEV)
    assert torch.equal(o[0].order, o[1].order)
    assert torch.equal(pm.combine_rows(rows, o[0], w), pm.combine_rows(rows, o[1], w))
    for a, b in zip(pm.combine_rows_grad(dout, rows, o[0], w), pm.combine_rows_grad(dout, rows, o[1], w)):
        assert torch.equal(a, b)


def test_captured_with_new_ids_and_on_another_stream():
    """A step recorded into a graph on a side stream, replayed with other ids and rows, while eager calls go on."""
    n, k, E, H = 200, 4, 32, 264
    idx = torch.from_numpy(make_idx(n, k, E, "mixed", 17)).to(DEV)
    x = torch.randn((n, H), generator=gen(18), device=DEV)
    w = torch.rand((n, k), generator=gen(19), device=DEV)

    def step(idx, x):
        o = pm.sort_by_expert(idx, E)
        xs = pm.dispatch_rows(x, o)
        out = pm.combine_rows(xs, o, w)
        drows, dw = pm.combine_rows_grad(x, xs, o, w)
        return out, drows, dw, pm.dispatch_rows_grad(drows, o)

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(idx, x)
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(idx, x)
    for seed in (20, 21):
        idx.copy_(torch.from_numpy(make_idx(n, k, E, "mixed" if seed == 20 else "none", seed)))
        x.copy_(torch.randn((n, H), generator=gen(seed), device=DEV))
        graph.replay()
        for a, b in zip(got, step(idx, x)):
            assert torch.equal(a, b)


def test_refusals():
    o = rows_case(4, 2, 8, "uniform")
    x = torch.zeros((4, 16), device=DEV)
    rows = torch.zeros((8, 16), device=DEV)
    w = torch.zeros((4, 2), device=DEV)
    bad = [lambda: pm.dispatch_rows(x[:3], o), lambda: pm.dispatch_rows(x[0], o), lambda: pm.dispatch_rows(x, "order"),
           lambda: pm.dispatch_rows(x, o, out=rows[:7]), lambda: pm.dispatch_rows(x, o, out=rows.bfloat16()),
           lambda: pm.combine_rows(x, o), lambda: pm.combine_rows(rows, o, w[:3]), lambda: pm.combine_rows(rows, o, w.t()), lambda: pm.combine_rows_grad(x, rows, o, w.reshape(-1)), lambda: pm.combine_rows(rows, o, w.cpu()),
           lambda: pm.combine_rows(rows, o, extra=rows), lambda: pm.combine_rows(rows, o, out=rows),
           lambda: pm.dispatch_rows(rows[:4], o, out=rows), lambda: pm.combine_rows(rows, o, out=rows[2:6]),
           lambda: pm.combine_rows(torch.ones_like(rows), o, extra=rows[:4], out=rows[1:5]),
           lambda: pm.combine_rows_grad(rows, rows, o), lambda: pm.combine_rows_grad(x, x, o),
           lambda: pm.sort_by_expert(w.int().view(2, 2, 2), 4), lambda: pm.sort_by_expert(w.int(), 4, expert_base=-1),
           lambda: pm.sort_by_expert(torch.zeros((4, 0), dtype=torch.int32, device=DEV), 4)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: pm.combine_rows(rows.half(), o), lambda: pm.combine_rows(rows, o, out_dtype=torch.float16),
              lambda: pm.combine_rows_grad(x.half(), rows, o), lambda: pm.sort_by_expert(w, 4)):
        with pytest.raises(pm.PmoeError) as e:
            f()
        assert e.value.code == -2
    with pytest.raises(pm.PmoeError) as e:
        pm.sort_by_expert(w.int(), 4097)
    assert e.value.code == -3
