"""Row operators around the experts: the stable sort by expert, dispatch and combine with their gradients, the residual
add + RMS norm with an 8-bit output, and low-rank adapters of many requests.

They are for hosts that run something of their own between the router and the experts' outputs (other expert types,
per-expert adapters, a training step); ``MoeBlock`` does all of it inside its kernels.  A training step reads::

    logits, w, idx = block.route(x)
    order = sort_by_expert(idx, E)
    xs = dispatch_rows(x, order)                    # rows of expert e: xs[order.offsets[e]:order.offsets[e + 1]]
    ...                                             # the experts: xs -> rows
    out = combine_rows(rows, order, w, extra=shared)
    grad_rows, grad_w = combine_rows_grad(grad_out, rows, order, w)
    ...                                             # back through the experts: grad_rows -> grad_xs
    grad_x = dispatch_rows_grad(grad_xs, order)

Nothing here waits for the GPU or reads a count back: sizes depend on the shapes alone.  These are plain functions on device
memory, as everything in this package is: autograd does not record them, and the gradients are the ones above.  Inputs that
require a gradient are taken (experts of torch's between the two ends give such rows); the results are detached.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import BF16, F32, F8_E4M3, I8, PmoeError, check, lib
from .moe import _check_buffer

_TYPES = {torch.float32: F32, torch.bfloat16: BF16}
_Q_TYPES = {torch.int8: I8, torch.float8_e4m3fn: F8_E4M3}
_MAX_EXPERTS = 4096
_MAX_PAIRS = _MAX_ROW = 2 ** 30
_MAX_INT = 2 ** 31 - 1


# The current stream's handle by device index: what torch.cuda.current_stream(device).cuda_stream gives, without making the
# stream object (2 us a call, as long as a small operator's launch).
_stream = torch._C._cuda_getCurrentRawStream


def _dense(t: torch.Tensor, dtype: int = F32) -> torch.Tensor:
    """The tensor contiguous, and its values in memory as they are: torch may mark a view as negative instead, one of f32 (half of a
    complex number) but not of bf16."""
    t = t.contiguous()
    return t.resolve_neg() if dtype == F32 and t.is_neg() else t


def _f32(t: torch.Tensor) -> torch.Tensor:
    return _dense(t if t.dtype is torch.float32 else t.to(torch.float32))


def _check_out(out: torch.Tensor, shape, dtype, device) -> None:
    _check_buffer("out", out, shape, dtype, device)
    if out.is_neg() or out.is_conj():
        raise ValueError("out must not be a conjugate or negated view")


def _too_large(limit: int, *sizes: int) -> PmoeError:
    """Sizes go to the C entries as 32-bit numbers, which must not wrap on the way."""
    return PmoeError(-1, f"sizes up to {limit} are served here, got {max(sizes)}")


def _on_gpu(what: str, t: torch.Tensor) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a torch tensor")
    if not t.is_cuda:
        raise PmoeError(-9, f"{what} must be a CUDA tensor; libpmoe has no CPU path")
    return t.device


def _typed(what: str, t: torch.Tensor, device) -> int:
    """The dtype id of an f32 / bf16 tensor on `device`."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{what} must be a tensor on {device}")
    if t.dtype not in _TYPES:
        raise PmoeError(-2, f"{what} must be float32 or bfloat16, got {t.dtype}")
    return _TYPES[t.dtype]


def _out_type(what: str, dtype: torch.dtype) -> int:
    if dtype not in _TYPES:
        raise PmoeError(-2, f"{what} must be float32 or bfloat16, got {dtype}")
    return _TYPES[dtype]


def _ids(what: str, t: torch.Tensor) -> torch.Tensor:
    """int32 ids, contiguous; wider ids outside int32 become ids that no expert has."""
    if t.dtype == torch.int32:
        return t.contiguous()
    if t.dtype == torch.int64:
        return t.clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous()   # both keep the strides of a transposed table
    raise PmoeError(-2, f"{what} must be int32 or int64, got {t.dtype}")


def _apart(what: str, out: torch.Tensor, t: Optional[torch.Tensor], same: bool = False) -> None:
    """Refuses an `out` that lies over an input whose elements other rows still need; `same`: it may be the input itself."""
    if t is None:
        return
    a, b = out.data_ptr(), t.data_ptr()
    if a < b + t.numel() * t.element_size() and b < a + out.numel() * out.element_size():
        if not (same and a == b and out.dtype == t.dtype):
            raise ValueError(f"out must not overlap {what}")


class ExpertOrder:
    """The (token, slot) pairs of a routing table in expert order (pmoe_sort_pairs).

    ``order`` int32 [n * top_k]: the pair at each row, -1 behind the last kept pair; ``place`` int32 [n, top_k]: the row of
    each pair, -1 for a pair that is not kept; ``offsets`` int32 [num_experts + 1]: the rows of expert e are
    offsets[e] to offsets[e + 1].  Expert e is the one whose id is expert_base + e."""

    __slots__ = ("n", "top_k", "num_experts", "expert_base", "device", "_data", "_order", "_place", "_offsets")

    def __init__(self, n: int, top_k: int, num_experts: int, device, expert_base: int = 0):
        self.n, self.top_k, self.num_experts, self.device, self.expert_base = n, top_k, num_experts, device, expert_base
        pairs = n * top_k
        # one allocation for the three arrays; each begins on a 16-byte boundary
        step = (pairs + 3) // 4 * 4
        self._data = torch.empty(2 * step + num_experts + 1, dtype=torch.int32, device=device)
        self._order = self._data.data_ptr()
        self._place, self._offsets = self._order + 4 * step, self._order + 8 * step

    @property
    def order(self) -> torch.Tensor:
        return self._data.as_strided((self.n * self.top_k,), (1,))

    @property
    def place(self) -> torch.Tensor:
        return self._data.as_strided((self.n, self.top_k), (self.top_k, 1), (self.n * self.top_k + 3) // 4 * 4)

    @property
    def offsets(self) -> torch.Tensor:
        return self._data.as_strided((self.num_experts + 1,), (1,), (self.n * self.top_k + 3) // 4 * 8)


def sort_by_expert(indices: torch.Tensor, num_experts: int, expert_base: int = 0) -> ExpertOrder:
    """The stable order of the pairs of ``indices`` [n, top_k] (or [n]: one slot) by expert.  Kept are the ids
    expert_base <= id < expert_base + num_experts (an expert-parallel rank's slice); all others, negative ones among
    them, are skipped.  The result depends on the ids alone, not on timing."""
    device = _on_gpu("indices", indices)
    shape = indices.shape
    if len(shape) not in (1, 2):
        raise ValueError("indices must be [n, top_k] or [n]")
    if not 1 <= int(num_experts) <= _MAX_EXPERTS:
        raise PmoeError(-3, f"1 to {_MAX_EXPERTS} experts are served, got {num_experts}")
    if not 0 <= expert_base < 2 ** 31 - num_experts:
        raise ValueError(f"expert_base must be 0 to 2^31 - 1 - num_experts, got {expert_base}")
    n, top_k = shape[0], shape[1] if len(shape) == 2 else 1
    if top_k == 0:
        raise ValueError("indices must have at least one slot")
    if n * top_k > _MAX_PAIRS:
        raise _too_large(_MAX_PAIRS, n * top_k)
    idx = _ids("indices", indices)
    o = ExpertOrder(n, top_k, int(num_experts), device, int(expert_base))
    i = device.index
    check(lib().pmoe_sort_pairs(i, idx.data_ptr(), n, top_k, o.expert_base, o.num_experts, o._order, o._place, o._offsets, _stream(i)))
    return o


def _ordered(order: ExpertOrder, device) -> None:
    if not isinstance(order, ExpertOrder):
        raise ValueError("order must come from sort_by_expert")
    if order.device != device:
        raise ValueError(f"order lives on {order.device}, the rows on {device}")


def dispatch_rows(x: torch.Tensor, order: ExpertOrder, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every token's row at its places in expert order: [n, H] -> [n * top_k, H], of any element type (f32 / bf16 rows,
    8-bit rows, their scales).  The rows behind the last kept pair are zero.  ``out``: the tensor to fill."""
    device = _on_gpu("x", x)
    _ordered(order, device)
    shape, n, top_k = x.shape, order.n, order.top_k
    if len(shape) != 2 or shape[0] != n:
        raise ValueError(f"x must be [{n}, H], got {tuple(shape)}")
    if x.is_conj():
        x = x.resolve_conj()
    x, H = _dense(x), shape[1]
    if out is None:
        out = torch.empty(n * top_k, H, dtype=x.dtype, device=device)
    else:
        _check_out(out, (n * top_k, H), x.dtype, device)
        _apart("x", out, x)
        _apart("order", out, order._data)
    if H == 0:
        return out
    i = device.index
    check(lib().pmoe_dispatch_rows(i, x.data_ptr(), H * x.element_size(), n, top_k, order._place, order._offsets, order.num_experts,
                                   out.data_ptr(), _stream(i)))
    return out


def _pair_weights(weights: torch.Tensor, order: ExpertOrder, device) -> torch.Tensor:
    if not isinstance(weights, torch.Tensor) or weights.device != device or weights.shape != (order.n, order.top_k):
        raise ValueError(f"weights must be [{order.n}, {order.top_k}] on {device}")
    return _f32(weights)


def _pair_rows(what: str, rows: torch.Tensor, dtype: int, order: ExpertOrder) -> Tuple[torch.Tensor, int, int]:
    """The rows contiguous, their number and their length."""
    shape = rows.shape
    if len(shape) != 2 or shape[0] != order.n * order.top_k or shape[1] == 0:
        raise ValueError(f"{what} must be [{order.n * order.top_k}, H], got {tuple(shape)}")
    if shape[1] > _MAX_ROW:
        raise _too_large(_MAX_ROW, shape[1])
    return _dense(rows, dtype), shape[0], shape[1]


def combine_rows(rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor] = None,
                 extra: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * rows[place[t, j]] (+ extra[t]), summed in f32 in slot order; rows [n * top_k, H] in
    expert order, weights [n, top_k] (None: ones), extra [n, H] (the shared expert's rows).  Pairs that are not kept add
    nothing.  The result has ``out_dtype`` (the rows' own by default); ``out``: the tensor to fill, which may be extra."""
    device = _on_gpu("rows", rows)
    _ordered(order, device)
    rd = _typed("rows", rows, device)
    rows, pairs, H = _pair_rows("rows", rows, rd, order)
    n = order.n
    w = None if weights is None else _pair_weights(weights, order, device)
    e, ed = None, 0
    if extra is not None:
        ed = _typed("extra", extra, device)
        if extra.shape != (n, H):
            raise ValueError(f"extra must be {(n, H)}, got {tuple(extra.shape)}")
        e = _dense(extra, ed)
    if out is None:
        od = rd if out_dtype is None else _out_type("out_dtype", out_dtype)
        out = torch.empty(n, H, dtype=out_dtype or rows.dtype, device=device)
    else:
        _check_out(out, (n, H), tuple(_TYPES), device)
        if out_dtype is not None and _out_type("out_dtype", out_dtype) != _TYPES[out.dtype]:
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        _apart("rows", out, rows)
        _apart("extra", out, e, same=True)
        _apart("weights", out, w)
        _apart("order", out, order._data)
        od = _TYPES[out.dtype]
    i = device.index
    check(lib().pmoe_combine_rows(i, rows.data_ptr(), rd, pairs, n, order.top_k, H, order._place, None if w is None else w.data_ptr(),
                                  None if e is None else e.data_ptr(), ed, out.data_ptr(), od, _stream(i)))
    return out


def dispatch_rows_grad(grad_rows: torch.Tensor, order: ExpertOrder, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Gradient of ``dispatch_rows``: the sum of a token's rows, [n * top_k, H] -> [n, H]."""
    return combine_rows(grad_rows, order, out_dtype=out_dtype)


def combine_rows_grad(grad_out: torch.Tensor, rows: torch.Tensor, order: ExpertOrder,
                      weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradient of ``combine_rows``: ``(grad_rows, grad_weights)``; grad_rows [n * top_k, H] in the rows' type with zeros
    behind the last kept pair, grad_weights [n, top_k] f32 with zeros for pairs that are not kept.  The gradient of
    ``extra`` is grad_out itself."""
    device = _on_gpu("grad_out", grad_out)
    _ordered(order, device)
    gd, rd = _typed("grad_out", grad_out, device), _typed("rows", rows, device)
    rows, pairs, H = _pair_rows("rows", rows, rd, order)
    n, top_k = order.n, order.top_k
    if grad_out.shape != (n, H):
        raise ValueError(f"grad_out must be {(n, H)}, got {tuple(grad_out.shape)}")
    g = _dense(grad_out, gd)
    w = None if weights is None else _pair_weights(weights, order, device)
    grad_rows = torch.empty_like(rows)
    grad_w = torch.empty(n, top_k, dtype=torch.float32, device=device)
    i = device.index
    check(lib().pmoe_combine_rows_grad(i, g.data_ptr(), gd, rows.data_ptr(), rd, n, top_k, H, order._place, order._offsets, order.num_experts,
                                       None if w is None else w.data_ptr(), grad_rows.data_ptr(), grad_w.data_ptr(), _stream(i)))
    return grad_rows, grad_w


def add_rms_norm_q8(resid: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor], eps: float, group: int = 0,
                    q_dtype: torch.dtype = torch.int8, values_dtype: Optional[torch.dtype] = None):
    """``add_rms_norm`` with the normalised row in 8 bits: ``(new_resid, q, scales, values)``.

    new_resid = resid + delta in resid's type (f32 / bf16); q [n, H] int8 or float8_e4m3fn and scales [n, ceil(H / group)]
    f32 (group 0: one per row; else 32, 64, 128 or 256 values), so that q * scale is the row RmsNorm(new_resid) * weight;
    values = q * scale in ``values_dtype`` for consumers that take plain rows but should see what the 8 bits hold (None
    when not asked for).  q and scales go to the experts through ``dispatch_rows``.  Rounding has no gradient: this is an
    operator for inference."""
    device = _on_gpu("resid", resid)
    shape = resid.shape
    if len(shape) != 2:
        raise ValueError("resid must be [n, H]")
    n, H = shape
    if n > _MAX_INT or H > _MAX_INT:
        raise _too_large(_MAX_INT, n, H)
    rd = _typed("resid", resid, device)
    r = _dense(resid, rd)
    d = dd = None
    if delta is not None:
        dd = _typed("delta", delta, device)
        if delta.shape != shape:
            raise ValueError(f"delta must be {(n, H)}, got {tuple(delta.shape)}")
        d = _dense(delta, dd)
    w = None
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.device != device or weight.shape != (H,):
            raise ValueError(f"weight must be [{H}] on {device}")
        w = _f32(weight)
    if q_dtype not in _Q_TYPES:
        raise PmoeError(-2, f"q_dtype must be int8 or float8_e4m3fn, got {q_dtype}")
    if group not in (0, 32, 64, 128, 256):
        raise PmoeError(-3, f"group must be 32, 64, 128, 256 or 0 for the whole row, got {group}")
    if H == 0:
        raise ValueError("resid must have columns")
    vd = 0 if values_dtype is None else _out_type("values_dtype", values_dtype)
    new_resid = torch.empty_like(r)
    q = torch.empty_like(r, dtype=q_dtype)
    scales = torch.empty(n, (H + group - 1) // group if group else 1, dtype=torch.float32, device=device)
    values = None if values_dtype is None else torch.empty_like(r, dtype=values_dtype)
    i = device.index
    check(lib().pmoe_add_rms_norm_q8(i, r.data_ptr(), rd, None if d is None else d.data_ptr(), dd or 0, None if w is None else w.data_ptr(), n, H,
                                     float(eps), group, new_resid.data_ptr(), _Q_TYPES[q_dtype], q.data_ptr(), scales.data_ptr(),
                                     None if values is None else values.data_ptr(), vd, _stream(i)))
    return new_resid, q, scales, values


# rows up to which pmoe_adapters_add groups the ids itself
_ADAPTER_ROWS_UNSORTED = 1024


def adapters_add(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                 scales: Optional[torch.Tensor] = None, order: Optional[ExpertOrder] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = base[t] + scales[i] * B_i (A_i x[t]) with i = ids[t]: the low-rank adapters of many requests (or of the
    experts that sorted rows belong to) beside one projection, whose output is ``base`` (``qmatmul``'s, say).

    base [n, N] and x [n, K] f32 or bf16; a [L, r, K] and b [L, N, r] bf16, r a multiple of 8 up to 128 (pad a smaller one with
    zeros), K and N multiples of 8; ids [n] int32, a row whose id is outside [0, L) keeps base; scales [L] f32 (None: ones).
    ``order`` = sort_by_expert(ids, L), worth keeping when several projections share the ids; made here from 1025
    rows on when it is not given.  ``out``: the tensor to fill (base itself for in place).  An operator for inference."""
    device = _on_gpu("x", x)
    xd, od = _typed("x", x, device), _typed("base", base, device)
    for name, t in (("a", a), ("b", b)):
        if not isinstance(t, torch.Tensor) or t.device != device or t.dim() != 3:
            raise ValueError(f"{name} must be a tensor of three dimensions on {device}")
        if t.dtype != torch.bfloat16:
            raise PmoeError(-2, f"{name} must be bfloat16, got {t.dtype}")
    L, r, K = a.shape
    Lb, N, rb = b.shape
    if L == 0 or Lb != L or rb != r:
        raise ValueError(f"a must be [L, r, K] and b [L, N, r], got {tuple(a.shape)} and {tuple(b.shape)}")
    n = x.shape[0] if x.dim() == 2 else -1
    if n < 0 or x.shape[1] != K or base.shape != (n, N):
        raise ValueError(f"x must be [n, {K}] and base [n, {N}], got {tuple(x.shape)} and {tuple(base.shape)}")
    if n > _MAX_INT or K > _MAX_INT or N > _MAX_INT or r > _MAX_INT:
        raise _too_large(_MAX_INT, n, K, N, r)
    if not isinstance(ids, torch.Tensor) or ids.device != device or ids.numel() != n:
        raise ValueError(f"ids must be [{n}] on {device}")
    if L > _MAX_EXPERTS:
        raise PmoeError(-3, f"at most {_MAX_EXPERTS} adapters are served, got {L}")
    s = None
    if scales is not None:
        if not isinstance(scales, torch.Tensor) or scales.device != device or scales.numel() != L:
            raise ValueError(f"scales must be [{L}] on {device}")
        s = _f32(scales)
    (x, xp), (a, ap), (b, bp), (base, basep) = _aligned(x, xd), _aligned(a, BF16), _aligned(b, BF16), _aligned(base, od)
    ids = _ids("ids", ids if ids.dim() == 1 else ids.reshape(-1))
    if order is not None:
        _ordered(order, device)
        if (order.n, order.top_k, order.num_experts, order.expert_base) != (n, 1, L, 0):   # of a slice: other adapters, and rows in no tile
            raise ValueError(f"order must be sort_by_expert(ids, {L}) of these {n} ids")
    elif n > _ADAPTER_ROWS_UNSORTED:
        order = sort_by_expert(ids, L)
    if out is None:
        out = torch.empty_like(base)
    else:
        _check_out(out, (n, N), base.dtype, device)
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        _apart("base", out, base, same=True)
        for name, t in (("x", x), ("a", a), ("b", b), ("ids", ids), ("scales", s), ("order", None if order is None else order._data)):
            _apart(name, out, t)
    i = device.index
    check(lib().pmoe_adapters_add(i, basep, xp, xd, n, K, N, r, L, ap, bp, None if s is None else s.data_ptr(), ids.data_ptr(),
                                  None if order is None else order._order, None if order is None else order._offsets, out.data_ptr(), od,
                                  _stream(i)))
    return out


def _aligned(t: torch.Tensor, dtype: int) -> Tuple[torch.Tensor, int]:
    """The tensor contiguous and from a 16-byte boundary on (a view may begin anywhere), and its address."""
    t = _dense(t, dtype)
    p = t.data_ptr()
    if p % 16:
        t = t.clone()
        p = t.data_ptr()
    return t, p


def rows_status(device="cuda") -> None:
    """Synchronises the current stream of `device` and raises PmoeError if a bounded wait inside ``adapters_add`` ran out on it, on
    any stream, since this stream's last call (since the library was loaded, if it has made none): outputs from then on are not to
    be used.  Every stream that asks hears of it once.  ``MoeBlock.status`` for the operators that have no handle."""
    d = torch.device(device)
    if d.type != "cuda":
        raise PmoeError(-9, "rows_status needs a CUDA device; libpmoe has no CPU path")
    index = torch.cuda.current_device() if d.index is None else d.index
    check(lib().pmoe_rows_status(index, _stream(index)))
