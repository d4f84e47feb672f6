"""Argument checks of the row operators (sort, dispatch, combine, 8-bit norm, adapters): what the binding and the C ABI
refuse before anything is launched.  No GPU is needed: the C entries check their arguments before they select a device."""
import ctypes as C

import pytest
import torch

import paramecia_b200 as pm
from paramecia_b200 import _lib

P = 0x1000   # a non-null, 16-byte aligned address that is never read
NULL = None


def _sort(**k):
    a = dict(device=0, idx=P, n=4, top_k=2, base=0, E=8, order=P, place=P, offsets=P)
    a.update(k)
    return pm.lib().pmoe_sort_pairs(*a.values(), None)


def _dispatch(**k):
    a = dict(device=0, x=P, row_bytes=64, n=4, top_k=2, place=P, offsets=P, E=8, out=P)
    a.update(k)
    return pm.lib().pmoe_dispatch_rows(*a.values(), None)


def _combine(**k):
    a = dict(device=0, rows=P, rd=pm.F32, n_rows=8, n=4, top_k=2, H=64, place=P, w=P, extra=P, ed=pm.F32, out=P, od=pm.F32)
    a.update(k)
    return pm.lib().pmoe_combine_rows(*a.values(), None)


def _grad(**k):
    a = dict(device=0, g=P, gd=pm.F32, rows=P, rd=pm.F32, n=4, top_k=2, H=64, place=P, offsets=P, E=8, w=P, gr=P, gw=P)
    a.update(k)
    return pm.lib().pmoe_combine_rows_grad(*a.values(), None)


def _norm(**k):
    a = dict(device=0, resid=P, rd=pm.F32, delta=P, dd=pm.F32, weight=P, n=4, H=64, eps=1e-6, group=32, out=P, qd=_lib.I8, q=P,
             scales=P, values=P, vd=pm.F32)
    a.update(k)
    return pm.lib().pmoe_add_rms_norm_q8(*a.values(), None)


def _adapters(**k):
    a = dict(device=0, base=P, x=P, xd=pm.F32, n=4, K=64, N=64, rank=16, L=4, a=P, b=P, scales=P, ids=P, order=P, offsets=P, out=P,
             od=pm.F32)
    a.update(k)
    return pm.lib().pmoe_adapters_add(*a.values(), None)


INVALID, DTYPE, SHAPE, TOO_MANY = -1, -2, -3, -5


@pytest.mark.parametrize("call, bad, code", [
    (_sort, dict(n=-1), INVALID), (_sort, dict(top_k=0), INVALID), (_sort, dict(n=1 << 29, top_k=4), INVALID),
    (_sort, dict(E=0), SHAPE), (_sort, dict(E=4097), SHAPE), (_sort, dict(base=-1), INVALID),
    (_sort, dict(idx=NULL), INVALID), (_sort, dict(offsets=NULL), INVALID),
    (_dispatch, dict(row_bytes=0), INVALID), (_dispatch, dict(row_bytes=1 << 31), INVALID), (_dispatch, dict(x=NULL), INVALID),
    (_dispatch, dict(place=NULL), INVALID), (_dispatch, dict(offsets=NULL), INVALID), (_dispatch, dict(out=NULL), INVALID),
    (_dispatch, dict(n=-1), INVALID), (_dispatch, dict(E=0), SHAPE),
    (_combine, dict(H=0), INVALID), (_combine, dict(n_rows=-1), INVALID), (_combine, dict(rd=pm.F16), DTYPE),
    (_combine, dict(ed=pm.Q8_0), DTYPE), (_combine, dict(od=pm.F16), DTYPE), (_combine, dict(rows=NULL), INVALID),
    (_combine, dict(place=NULL), INVALID), (_combine, dict(out=NULL), INVALID), (_combine, dict(top_k=-3), INVALID),
    (_grad, dict(gr=NULL, gw=NULL), INVALID), (_grad, dict(rows=NULL), INVALID), (_grad, dict(g=NULL), INVALID),
    (_grad, dict(gd=pm.F16), DTYPE), (_grad, dict(rd=99), DTYPE), (_grad, dict(H=-1), INVALID), (_grad, dict(offsets=NULL), INVALID),
    (_norm, dict(n=-1), INVALID), (_norm, dict(H=0), INVALID), (_norm, dict(H=16385), INVALID), (_norm, dict(group=48), SHAPE),
    (_norm, dict(group=-32), SHAPE), (_norm, dict(rd=pm.F16), DTYPE), (_norm, dict(dd=pm.F16), DTYPE), (_norm, dict(vd=pm.F16), DTYPE),
    (_norm, dict(qd=pm.Q8_0), DTYPE), (_norm, dict(eps=float("nan")), INVALID), (_norm, dict(eps=-1.0), INVALID),
    (_norm, dict(resid=NULL), INVALID), (_norm, dict(q=NULL), INVALID), (_norm, dict(scales=NULL), INVALID),
    (_adapters, dict(n=-1), INVALID), (_adapters, dict(L=0), INVALID), (_adapters, dict(L=4097), INVALID), (_adapters, dict(K=68), SHAPE),
    (_adapters, dict(N=60), SHAPE), (_adapters, dict(rank=12), SHAPE), (_adapters, dict(rank=136), SHAPE), (_adapters, dict(rank=0), SHAPE),
    (_adapters, dict(xd=pm.F16), DTYPE), (_adapters, dict(od=pm.F16), DTYPE), (_adapters, dict(ids=NULL), INVALID),
    (_adapters, dict(order=NULL), INVALID), (_adapters, dict(offsets=NULL), INVALID), (_adapters, dict(x=P + 2), INVALID),
    (_adapters, dict(b=P + 8), INVALID), (_adapters, dict(out=P + 4), INVALID),
    (_adapters, dict(order=NULL, offsets=NULL, n=1025), TOO_MANY),
])
def test_c_entries_refuse(call, bad, code):
    assert call(**bad) == code
    assert pm.lib().pmoe_last_error()


def test_empty_batches_need_no_device():
    assert _dispatch(n=0, x=NULL, place=NULL, offsets=NULL, out=NULL) == 0
    assert _combine(n=0, rows=NULL, n_rows=0, place=NULL, out=NULL) == 0
    assert _grad(n=0, g=NULL, rows=NULL, place=NULL, offsets=NULL) == 0
    assert _norm(n=0, resid=NULL, q=NULL, scales=NULL) == 0
    assert _adapters(n=0, base=NULL, x=NULL, a=NULL, b=NULL, ids=NULL, out=NULL) == 0


def test_host_tensors_are_refused():
    idx = torch.zeros((2, 2), dtype=torch.int32)
    x = torch.zeros((2, 8))
    for f in (lambda: pm.sort_by_expert(idx, 4), lambda: pm.dispatch_rows(x, None), lambda: pm.combine_rows(x, None),
              lambda: pm.combine_rows_grad(x, x, None), lambda: pm.add_rms_norm_q8(x, None, None, 1e-6),
              lambda: pm.adapters_add(x, x, x, x, idx)):
        with pytest.raises(pm.PmoeError) as e:
            f()
        assert e.value.code == -9
    with pytest.raises(pm.PmoeError):
        pm.rows_status("cpu")
    with pytest.raises(ValueError):
        pm.sort_by_expert([1, 2], 4)
