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


def test_sorts_of_several_threads():
    """Calls that need different amounts of shared memory, from threads that launch at the same time: none is refused, and
    every one has its own result."""
    shapes = [(4096, 512), (4096, 4096), (4096, 256), (20000, 512), (20000, 4096)]      # pairs, experts
    rc, calls = {}, 4000
    start = threading.Barrier(len(shapes))

    def run(i):
        P, E = shapes[i]
        ids = torch.from_numpy(np.random.default_rng(i).integers(0, E, P).astype(np.int32)).to(DEV)
        places, offsets = torch.empty(P, dtype=torch.int32, device=DEV), torch.empty(E + 1, dtype=torch.int32, device=DEV)
        stream = torch.cuda.Stream(DEV)
        torch.cuda.synchronize()
        sort = pm.lib().pmoe_sort_pairs
        start.wait()
        bad = sum(sort(0, ids.data_ptr(), P, 1, 0, E, None, places.data_ptr(), offsets.data_ptr(), stream.cuda_stream) != 0 for _ in range(calls))
        stream.synchronize()
        rc[i] = bad, np.array_equal(places.cpu().numpy(), plain_places(ids.cpu().numpy(), E))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert rc == {i: (0, True) for i in range(len(shapes))}


@pytest.mark.parametrize("base", [1, 3, 8])
def test_an_order_of_another_slice_is_refused(base):
    """Rows below the slice's first id are in no tile of such an order and would be left unwritten."""
    ids = torch.arange(20, dtype=torch.int32, device=DEV) % 8
    x, rows = torch.ones((20, 16), device=DEV), torch.ones((20, 24), device=DEV)
    a = torch.ones((8, 8, 16), dtype=torch.bfloat16, device=DEV)
    b = torch.ones((8, 24, 8), dtype=torch.bfloat16, device=DEV)
    o = pm.sort_by_expert(ids, 8, expert_base=base)
    assert o.expert_base == base and pm.sort_by_expert(ids, 8).expert_base == 0
    with pytest.raises(ValueError, match="order must be"):
        pm.adapters_add(rows, x, a, b, ids, order=o)
    got = pm.adapters_add(rows, x, a, b, ids, order=pm.sort_by_expert(ids, 8))
    assert torch.equal(got, torch.full_like(got, 129.0))


def test_an_out_over_ids_weights_or_the_order_is_refused():
    n, k, N = 64, 2, 64
    pool = torch.zeros(4096, dtype=torch.int32, device=DEV)              # what the outputs lie in
    out = pool.view(torch.float32).view(n, N)
    ids = pool[:n * k].view(n, k)
    o = pm.sort_by_expert(torch.zeros_like(ids), 4)
    rows, x = torch.ones((n * k, N), device=DEV), torch.ones((n, N), device=DEV)
    a, b = torch.zeros((4, 8, N), dtype=torch.bfloat16, device=DEV), torch.zeros((4, N, 8), dtype=torch.bfloat16, device=DEV)
    first = pool[:n]
    over_order = o._data[:(n * k) // 4 * 4].view(torch.float32).view(n * k, 1)
    for f in (lambda: pm.combine_rows(rows, o, ids.view(torch.float32), out=out), lambda: pm.dispatch_rows(x[:, :1].contiguous(), o, out=over_order),
              lambda: pm.adapters_add(x, x.clone(), a, b, first, out=out), lambda: pm.adapters_add(x, x.clone(), a, b, o.place[:, 0].contiguous(), scales=pool[:4].view(torch.float32), out=out),
              lambda: pm.adapters_add(x, x.clone(), pool.view(torch.bfloat16)[:4 * 8 * N].view(4, 8, N), b, torch.zeros_like(first), out=out)):
        with pytest.raises(ValueError, match="must not overlap"):
            f()
    assert not pool.any()


def test_sizes_that_no_int_holds_are_refused():
    """Views of one element with such shapes: a size that wraps must not reach the C entries as another one."""
    one, ids = torch.ones(1, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    half = one.bfloat16()
    o = pm.sort_by_expert(ids, 4)
    big = 2 ** 32 + 8
    for f in (lambda: pm.combine_rows(one.expand(1, big), o), lambda: pm.combine_rows_grad(one.expand(1, big), one.expand(1, big), o),
              lambda: pm.sort_by_expert(ids.expand(big), 4), lambda: pm.sort_by_expert(ids.expand(2 ** 28, 5), 4),
              lambda: pm.add_rms_norm_q8(one.expand(1, big), None, None, 1e-6), lambda: pm.add_rms_norm_q8(one.expand(big, 8), None, None, 1e-6),
              lambda: pm.adapters_add(one.expand(1, 8), one.expand(1, big), half.expand(1, 8, big), half.expand(1, 8, 8), ids),
              lambda: pm.adapters_add(one.expand(big, 8), one.expand(big, 8), half.expand(1, 8, 8), half.expand(1, 8, 8), ids.expand(big))):
        with pytest.raises(pm.PmoeError) as e:
            f()
        assert e.value.code == -1
    for base in (2 ** 32, 2 ** 31 - 4):
        with pytest.raises(ValueError):
            pm.sort_by_expert(ids, 4, expert_base=base)
    assert pm.sort_by_expert(ids - 2 ** 31, 4, expert_base=2 ** 31 - 5).place.tolist() == [[-1]]
    assert pm.sort_by_expert(ids.long() + 2 ** 40, 4, expert_base=2 ** 31 - 5).place.tolist() == [[-1]]


def test_views_that_negate_or_conjugate():
    """torch keeps a conjugate, and the imaginary part of one, as a view with a mark: the memory holds the other sign."""
    z = torch.complex(*torch.randn((2, 30, 64), device=DEV).unbind(0))
    ids = torch.arange(60, dtype=torch.int32, device=DEV).view(30, 2) % 7
    o = pm.sort_by_expert(ids, 7)
    pair = o.order.long()
    assert z.conj().is_conj() and z.conj().imag.is_neg()
    assert torch.equal(pm.dispatch_rows(z.conj(), o), z.conj().resolve_conj()[pair // 2])
    neg = z.conj().imag                       # strided, negative
    flat = torch._neg_view(neg.contiguous())  # dense, negative
    for v in (neg, flat):
        plain = v.clone().resolve_neg()
        assert v.is_neg() and not plain.is_neg()
        assert torch.equal(pm.dispatch_rows(v, o), plain[pair // 2])
        rows, want = pm.dispatch_rows(plain, o), pm.dispatch_rows(plain, o)
        neg_rows = torch._neg_view(-rows)
        w = torch._neg_view(-torch.rand((30, 2), device=DEV))
        assert torch.equal(pm.combine_rows(neg_rows, o, w, extra=v), pm.combine_rows(want, o, w.clone().resolve_neg(), extra=plain))
        for a, b in zip(pm.combine_rows_grad(v, neg_rows, o, w), pm.combine_rows_grad(plain, want, o, w.clone().resolve_neg())):
            assert torch.equal(a, b)
        for a, b in zip(pm.add_rms_norm_q8(v, v, v[0], 1e-6)[:3], pm.add_rms_norm_q8(plain, plain, plain[0], 1e-6)[:3]):
            assert torch.equal(a, b)
        a, b = (torch.randn(s, device=DEV).bfloat16() for s in ((7, 8, 64), (7, 64, 8)))
        first = ids[:, 0].contiguous()
        assert torch.equal(pm.adapters_add(v, v, a, b, first), pm.adapters_add(plain, plain, a, b, first))
    with pytest.raises(ValueError):
        pm.combine_rows(want, o, out=torch._neg_view(torch.zeros((30, 64), device=DEV)))


def test_an_out_of_another_type_than_out_dtype_is_refused():
    o = pm.sort_by_expert(torch.zeros((4, 2), dtype=torch.int32, device=DEV), 3)
    rows, out = torch.ones((8, 16), device=DEV), torch.zeros((4, 16), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="out_dtype"):
        pm.combine_rows(rows, o, out_dtype=torch.float32, out=out)
    with pytest.raises(pm.PmoeError):
        pm.combine_rows(rows, o, out_dtype=torch.float16, out=out)
    assert pm.combine_rows(rows, o, out_dtype=torch.bfloat16, out=out) is out and (out == 2).all()
