"""What the binding of the row operators makes of its arguments, and what the C entries refuse, without a GPU."""
import pytest
import torch

import paramecia_b200 as pm
from paramecia_b200 import _lib, rows

A = 1 << 20      # addresses a megabyte apart, never read: every call below is refused before a device is selected
IDX, PLACE, OFFSETS, ORDER, W, X, ROWS, EXTRA, OUT, OUT2, OUT3, OUT4 = range(A, 13 * A, A)
INVALID = -1


def _sort(idx=IDX, order=ORDER, place=PLACE, offsets=OFFSETS):
    return pm.lib().pmoe_sort_pairs(0, idx, 100, 2, 0, 16, order, place, offsets, None)


def _dispatch(x=X, place=PLACE, offsets=OFFSETS, out=OUT):
    return pm.lib().pmoe_dispatch_rows(0, x, 64, 100, 2, place, offsets, 16, out, None)


def _combine(rows=ROWS, place=PLACE, w=W, extra=EXTRA, out=OUT, od=pm.F32):
    return pm.lib().pmoe_combine_rows(0, rows, pm.F32, 200, 100, 2, 32, place, w, extra, pm.F32, out, od, None)


def _grad(g=X, rows=ROWS, place=PLACE, offsets=OFFSETS, w=W, gr=OUT, gw=OUT2):
    return pm.lib().pmoe_combine_rows_grad(0, g, pm.F32, rows, pm.F32, 100, 2, 32, place, offsets, 16, w, gr, gw, None)


def _norm(resid=X, delta=ROWS, weight=W, out=OUT, q=OUT2, scales=OUT3, values=OUT4):
    return pm.lib().pmoe_add_rms_norm_q8(0, resid, pm.F32, delta, pm.F32, weight, 100, 64, 1e-6, 32, out, _lib.I8, q, scales, values, pm.F32, None)


def _adapters(base=ROWS, x=X, a=EXTRA, b=W, scales=OUT3, ids=IDX, order=ORDER, offsets=OFFSETS, out=OUT):
    return pm.lib().pmoe_adapters_add(0, base, x, pm.F32, 100, 64, 64, 8, 4, a, b, scales, ids, order, offsets, out, pm.F32, None)


@pytest.mark.parametrize("call, over", [
    (_sort, dict(order=IDX)), (_sort, dict(place=IDX + 796)), (_sort, dict(offsets=IDX - 64)), (_sort, dict(offsets=ORDER)), (_sort, dict(place=ORDER + 4)),
    (_dispatch, dict(out=X)), (_dispatch, dict(out=X - 12784)), (_dispatch, dict(out=PLACE)), (_dispatch, dict(out=OFFSETS + 64)),
    (_combine, dict(out=ROWS + 16)), (_combine, dict(out=PLACE)), (_combine, dict(out=W)), (_combine, dict(out=EXTRA + 128)), (_combine, dict(out=EXTRA, od=pm.BF16)),
    (_grad, dict(gr=ROWS)), (_grad, dict(gr=X)), (_grad, dict(gr=PLACE - 16)), (_grad, dict(gr=OFFSETS)), (_grad, dict(gr=W)), (_grad, dict(gw=OUT + 4)),
    (_grad, dict(gw=W)), (_grad, dict(gw=PLACE)), (_grad, dict(gw=OFFSETS)), (_grad, dict(gw=ROWS)), (_grad, dict(gw=X)),
    (_norm, dict(q=X)), (_norm, dict(values=ROWS)), (_norm, dict(scales=W)), (_norm, dict(out=X + 256)), (_norm, dict(values=OUT)), (_norm, dict(scales=OUT2 + 4)),
    (_adapters, dict(out=X)), (_adapters, dict(out=ROWS + 256)), (_adapters, dict(out=EXTRA)), (_adapters, dict(out=W)), (_adapters, dict(out=OUT3)),
    (_adapters, dict(out=IDX)), (_adapters, dict(out=ORDER)), (_adapters, dict(out=OFFSETS + 16)),
])
def test_outputs_over_inputs_are_refused(call, over):
    """Some of it another thread still reads: a list of ids that changes under the adapters' clusters would lead their CTAs apart."""
    assert call(**over) == INVALID and b"overlap" in pm.lib().pmoe_last_error()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_ids_are_dense(dtype):
    table = torch.arange(12, dtype=dtype).reshape(3, 4)
    for t in (table, table.t(), table[:, ::2], table.t()[1:]):
        got = rows._ids("ids", t)
        assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == t.tolist()


def test_sizes_beyond_the_kernels_numbers_are_refused():
    """Columns are counted in 32 bits, a stride of the grid beyond them; ids behind the last 32-bit number are none."""
    for H in ((1 << 31) - 1, (1 << 30) + 1):
        assert pm.lib().pmoe_combine_rows(0, ROWS, pm.BF16, 1, 1, 1, H, PLACE, None, None, 0, OUT, pm.BF16, None) == INVALID
        assert pm.lib().pmoe_combine_rows_grad(0, X, pm.BF16, ROWS, pm.BF16, 1, 1, H, PLACE, OFFSETS, 4, None, OUT, OUT2, None) == INVALID
    for base in ((1 << 31) - 1, (1 << 31) - 16):
        assert pm.lib().pmoe_sort_pairs(0, IDX, 1, 1, base, 16, ORDER, PLACE, OFFSETS, None) == INVALID
