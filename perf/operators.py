"""Timed cases of the row operators around the experts: the sort by expert with its dispatch and combine (and their
gradient), the residual add + RMS norm with an 8-bit output, and low-rank adapters beside a projection.

`run` computes an operator in plain torch arithmetic (f32, rounded once at the end) while `own` is false, and through the
package's entry points while it is true; `exact` computes the same from the definitions in 64 bits."""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1, "i8": 1}
EPS = 1e-6


def listed():
    # hidden 2048, 512 experts, 10 choices, batches of 1 to 256 and prompts of 4096 are the block's own sizes
    return [
        # one decoding token to its ten experts: launch latency
        dict(name="dispatch 1 token", op="dispatch", n=1, k=10, E=512, H=2048, type="bf16", ranks=1),
        # what a rank of four keeps of a prompt of 4096 tokens (a quarter of the pairs; the rest of the rows is zero)
        dict(name="dispatch 4096 rank of 4", op="dispatch", n=4096, k=10, E=512, H=2048, type="bf16", ranks=4),
        # a decode batch back from the experts, f32 rows, with the shared expert's row added
        dict(name="combine 61 tokens", op="combine", n=61, k=10, E=512, H=2048, type="f32", extra=True, ranks=1),
        # a prompt back from the experts
        dict(name="combine 8192", op="combine", n=8192, k=10, E=512, H=2048, type="bf16", extra=True, ranks=1),
        # a small training step in f32 with an odd row length (no vector loads fit it)
        dict(name="step 500 odd f32", op="step", n=500, k=4, E=60, H=1407, type="f32", ranks=1),
        # a training step: rows to the experts and back, and both gradients
        dict(name="step 4096", op="step", n=4096, k=10, E=512, H=2048, type="bf16", ranks=1),
        # one decoding token's norm, f32 residual as the stack has it, one scale per 32 values
        dict(name="norm 1 row", op="norm", n=1, H=2048, type="f32", delta="f32", q="i8", group=32, values=True),
        # a mixed batch, one scale per row, f32 residual with a bf16 block output
        dict(name="norm 777 rows", op="norm", n=777, H=5120, type="f32", delta="bf16", q="i8", group=0, values=True),
        # a prompt, 8-bit floats with a scale per 128
        dict(name="norm 16384 e4m3", op="norm", n=16384, H=2048, type="bf16", delta="bf16", q="e4m3", group=128, values=False),
        # one decoding request with its adapter
        dict(name="adapters 1 row", op="adapters", n=1, K=2048, N=2048, r=16, L=8, x="f32", base="f32"),
        # a decode batch of many requests, most with an adapter of their own
        dict(name="adapters 64 rows", op="adapters", n=64, K=2048, N=4096, r=32, L=48, x="bf16", base="bf16"),
        # prompts of several requests in one batch
        dict(name="adapters 8192 rows", op="adapters", n=8192, K=2048, N=2048, r=64, L=12, x="bf16", base="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "step", "norm", "norm", "adapters", "adapters"])
    if op == "norm":
        H = rng.choice([512, 1000, 1536, 2048, 2880, 4096, 5120, 7168, 2047])
        kind = rng.choice(["f32", "bf16"])
        q = rng.choice(["i8", "e4m3"])
        return dict(op=op, n=_log(rng, 1, 16384 * 2048 // max(H, 2048) // 2), H=H, type=kind, delta=rng.choice([kind, "bf16"]), q=q,
                    group=rng.choice([0, 32, 64, 128, 256]), values=q == "i8" or rng.random() < 0.5)
    if op == "adapters":
        L, r = _log(rng, 1, 64), rng.choice([8, 16, 24, 32, 64])
        return dict(op=op, n=_log(rng, 1, min(8192, 8192 * 12 * 64 // (L * r))), K=rng.choice([512, 1000, 2048, 4096]),
                    N=rng.choice([504, 512, 1024, 2048, 4096]), r=r, L=L, x=rng.choice(["f32", "bf16"]), base=rng.choice(["f32", "bf16"]))
    E = rng.choice([8, 60, 128, 256, 512])
    k = rng.choice([1, 2, 4, 6, 8, 10]) if E > 8 else rng.choice([1, 2])
    H = rng.choice([256, 500, 1024, 1407, 2048, 4096])
    kind = rng.choice(["f32", "bf16"])
    top = 4096 * 11 * 2048 * 2 // ((k + 1) * H * SIZE[kind])
    case = dict(op=op, n=_log(rng, 1, max(2, min(16384, top))), k=k, E=E, H=H, type=kind, ranks=1 if E % 4 else rng.choice([1, 1, 2, 4]))
    if op == "combine":
        case["extra"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = dict(case)
    n = case["n"]
    if case["op"] == "norm":
        H = case["H"]
        # a residual stream: a few channels are much larger than the rest
        channel = 1.0 + 20.0 * (torch.rand((H,), generator=g, device=DEVICE) > 0.997)
        s["resid"] = (3.0 * rand(n, H) * channel).to(TYPES[case["type"]])
        s["delta"] = rand(n, H).to(TYPES[case["delta"]])
        s["weight"] = 1.0 + 0.2 * rand(H)
        return s
    if case["op"] == "adapters":
        K, N, r, L = case["K"], case["N"], case["r"], case["L"]
        s["x_rows"] = rand(n, K).to(TYPES[case["x"]])
        s["base_rows"] = rand(n, N).to(TYPES[case["base"]])
        s["a"] = (rand(L, r, K) / math.sqrt(K)).bfloat16()
        s["b"] = (rand(L, N, r) / math.sqrt(r)).bfloat16()
        s["scales"] = 0.5 + torch.rand((L,), generator=g, device=DEVICE)
        if n > 512:  # prompts: runs of rows of one request
            ids = (torch.rand((n // 256 + 1,), generator=g, device=DEVICE) * (L + 1)).int().repeat_interleave(256)[:n] - 1
        else:        # single tokens; -1: a request without an adapter
            ids = (torch.rand((n,), generator=g, device=DEVICE) * (L + 1)).int() - 1
        s["ids"] = ids if n > 1 else ids.clamp(min=0)
        return s
    k, E, H, ranks = case["k"], case["E"], case["H"], case["ranks"]
    # a router with favourites
    logits = rand(n, E) + 0.7 * rand(E)
    top, idx = torch.topk(logits, k, dim=1)
    s["idx"] = idx.int()
    s["w"] = torch.softmax(top, dim=1)
    s["E_local"], s["first"] = E // ranks, (E // ranks) * (seed % ranks)  # the experts of one rank
    t = TYPES[case["type"]]
    if case["op"] in ("dispatch", "step"):
        s["x"] = rand(n, H).to(t)
    if case["op"] in ("combine", "step"):
        s["rows"] = rand(n * k, H).to(t)
    if case["op"] == "combine":
        s["extra_rows"] = rand(n, H).to(t) if case["extra"] else None
    if case["op"] == "step":
        s["dout"] = rand(n, H).to(t)
        s["dxs"] = rand(n * k, H).to(t)  # what comes back through the experts
    return s


# ---------------------------------------------------------------- plain forms
def _plain_sort(s):
    key = s["idx"].long() - s["first"]
    kept = (key >= 0) & (key < s["E_local"])
    flat = torch.where(kept, key, s["E_local"]).reshape(-1)
    P = flat.numel()
    sequence = torch.arange(P, device=flat.device)
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(flat)
    place[order] = sequence
    counts = torch.zeros(s["E_local"] + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:-1], 0)])
    order = torch.where(sequence < offsets[-1], order, -1)
    place = torch.where(kept, place.view_as(key), -1)
    return order.int(), place.int(), offsets.int()


def _plain_dispatch(x, order, k):
    pair = order.long().clamp(min=0)
    return torch.where((order >= 0)[:, None], x[pair // k], torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_combine(rows, place, w, extra, dtype):
    picked = rows[place.long().clamp(min=0)].float()
    if w is not None:
        picked = picked * w[:, :, None]
    out = torch.where((place >= 0)[:, :, None], picked, 0.0).sum(1)
    return (out if extra is None else out + extra.float()).to(dtype)


def _plain_combine_grad(dout, rows, order, place, w):
    k = place.shape[1]
    pair = order.long().clamp(min=0)
    kept = order >= 0
    spread = dout[pair // k].float()
    drows = torch.where(kept[:, None], spread * w.reshape(-1)[pair][:, None], 0.0).to(rows.dtype)
    dot = (spread * rows.float()).sum(1)
    dw = torch.where(place >= 0, dot[place.long().clamp(min=0)], 0.0)
    return drows, dw


def _plain_norm(s):
    resid = (s["resid"].float() + s["delta"].float()).to(s["resid"].dtype)
    r = resid.float()
    v = r / torch.sqrt((r.double().square().mean(1, keepdim=True) + EPS).float()) * s["weight"]
    n, H = v.shape
    group = s["group"] or H
    G = -(-H // group)
    pad = torch.nn.functional.pad(v, (0, G * group - H)).view(n, G, group)
    most = 127.0 if s["q"] == "i8" else 448.0
    scales = (pad.abs().amax(2).double() / most).float()
    ratio = torch.where(scales[:, :, None] > 0, pad / scales[:, :, None], 0.0).clamp(-most, most)
    if s["q"] == "i8":
        q = torch.round(ratio)
    else:
        q = ratio.to(torch.float8_e4m3fn)
    out = {"resid": resid, "scales": scales}
    if s["values"]:  # what the 8 bits stand for
        out["values"] = (q.float() * scales[:, :, None]).view(n, G * group)[:, :H].bfloat16()
    else:
        out["q"] = q.view(n, G * group)[:, :H].contiguous()
    return out


def _plain_adapters(s):
    a, b, ids = s["a"].float(), s["b"].float(), s["ids"]
    L, r, K = a.shape
    every = (s["x_rows"].float() @ a.view(L * r, K).t()).view(-1, L, r)
    mine = ids[:, None] == torch.arange(L, device=ids.device)
    h = torch.where(mine[:, :, None], every * s["scales"][None, :, None], 0.0).view(-1, L * r)
    more = h @ b.permute(0, 2, 1).reshape(L * r, -1)
    return (s["base_rows"].float() + more).to(s["base_rows"].dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        import paramecia_b200 as pm

        if op == "norm":
            resid, q, scales, values = pm.add_rms_norm_q8(
                s["resid"], s["delta"], s["weight"], EPS, group=s["group"],
                q_dtype=torch.int8 if s["q"] == "i8" else torch.float8_e4m3fn,
                values_dtype=torch.bfloat16 if s["values"] else None)
            return {"resid": resid, "scales": scales, **({"values": values} if s["values"] else {"q": q})}
        if op == "adapters":
            return {"out": pm.adapters_add(s["base_rows"], s["x_rows"], s["a"], s["b"], s["ids"], scales=s["scales"])}
        plan = pm.sort_by_expert(s["idx"], s["E_local"], expert_base=s["first"])
        if op == "dispatch":
            return {"xs": pm.dispatch_rows(s["x"], plan), "order": plan.order, "place": plan.place, "offsets": plan.offsets}
        if op == "combine":
            return {"out": pm.combine_rows(s["rows"], plan, s["w"], extra=s["extra_rows"])}
        xs = pm.dispatch_rows(s["x"], plan)
        out = pm.combine_rows(s["rows"], plan, s["w"])
        drows, dw = pm.combine_rows_grad(s["dout"], s["rows"], plan, s["w"])
        dx = pm.dispatch_rows_grad(s["dxs"], plan)
        return {"xs": xs, "out": out, "drows": drows, "dw": dw, "dx": dx}
    if op == "norm":
        return _plain_norm(s)
    if op == "adapters":
        return {"out": _plain_adapters(s)}
    order, place, offsets = _plain_sort(s)
    if op == "dispatch":
        return {"xs": _plain_dispatch(s["x"], order, s["k"]), "order": order, "place": place, "offsets": offsets}
    t = s["rows"].dtype
    if op == "combine":
        return {"out": _plain_combine(s["rows"], place, s["w"], s["extra_rows"], t)}
    drows, dw = _plain_combine_grad(s["dout"], s["rows"], order, place, s["w"])
    return {"xs": _plain_dispatch(s["x"], order, s["k"]), "out": _plain_combine(s["rows"], place, s["w"], None, t),
            "drows": drows, "dw": dw, "dx": _plain_combine(s["dxs"], place, None, None, t)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n = case["n"]
    if case["op"] == "norm":
        H = case["H"]
        G = -(-H // (case["group"] or H))
        per = SIZE[case["type"]] * 2 + SIZE[case["delta"]] + 1 + (2 if case["values"] else 0)
        return {"bytes": n * H * per + 4 * n * G + 4 * H, "flops": 8.0 * n * H}
    if case["op"] == "adapters":
        K, N, r = case["K"], case["N"], case["r"]
        hit = min(case["L"], n)
        return {"bytes": n * (K * SIZE[case["x"]] + 2 * N * SIZE[case["base"]]) + 2 * hit * r * (K + N) + 4 * n,
                "flops": 2.0 * n * r * (K + N)}
    P, H, z = n * case["k"], case["H"], SIZE[case["type"]]
    part = 1.0 / case["ranks"]  # of the pairs, about: those that this rank's experts take
    sort = 4 * P + 4 * (case["E"] // case["ranks"] + 1)
    if case["op"] == "dispatch":
        return {"bytes": sort + 8 * P + n * H * z + P * H * z, "flops": 4.0 * P}
    if case["op"] == "combine":
        return {"bytes": sort + 4 * P + part * P * H * z + (2 if case["extra"] else 1) * n * H * z, "flops": 2.0 * P * H}
    # step: x, dout, xs, rows, drows, dxs, out, dx, weights and their gradient
    return {"bytes": sort + 8 * P + (2 * P + 2 * n) * H * z + (2 * part * P + 2 * n) * H * z, "flops": 6.0 * P * H}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    n = case["n"]
    if case["op"] == "norm":
        H = case["H"]
        z = s["resid"].double() + s["delta"].double()
        z = z.to(s["resid"].dtype).double()  # the residual is stored, and the norm is of what is stored
        v = z * torch.rsqrt((z * z).sum(1, keepdim=True) / H + EPS) * s["weight"].double()
        most = 127.0 if case["q"] == "i8" else 448.0
        scales, held = [], []
        for at in range(0, H, case["group"] or H):
            part = v[:, at:at + (case["group"] or H)]
            scale = part.abs().max(1, keepdim=True).values / most
            q = part / torch.where(scale > 0, scale, 1.0)
            q = q.round() if case["q"] == "i8" else q.float().to(torch.float8_e4m3fn).double()
            scales.append(scale)
            held.append(q * scale if case["values"] else q)
        return {"resid": z, "scales": torch.cat(scales, 1), "values" if case["values"] else "q": torch.cat(held, 1)}
    if case["op"] == "adapters":
        out = s["base_rows"].double()
        for i in range(case["L"]):
            t = torch.nonzero(s["ids"] == i)[:, 0]
            out[t] += float(s["scales"][i]) * ((s["x_rows"][t].double() @ s["a"][i].double().t()) @ s["b"][i].double().t())
        return {"out": out}
    k, H = case["k"], case["H"]
    idx = s["idx"].long().reshape(-1) - s["first"]
    lists = torch.where((idx >= 0) & (idx < s["E_local"]), idx, case["E"]) * idx.numel() + torch.arange(idx.numel(), device=DEVICE)
    pairs = torch.sort(lists).values
    pairs = pairs[pairs < case["E"] * idx.numel()] % idx.numel()  # the kept pairs, expert by expert
    m = pairs.numel()
    if case["op"] == "dispatch":
        xs = torch.zeros((n * k, H), dtype=torch.float64, device=DEVICE)
        xs[:m] = s["x"].double()[pairs // k]
        return {"xs": xs, "order": None, "place": None, "offsets": None}
    w = s["w"].double().reshape(-1)[pairs]
    out = torch.zeros((n, H), dtype=torch.float64, device=DEVICE)
    rows = s["rows"][:m].double()
    out.index_add_(0, pairs // k, rows * w[:, None])
    if case["op"] == "combine":
        return {"out": out if s["extra_rows"] is None else out + s["extra_rows"].double()}
    dout = s["dout"].double()[pairs // k]
    dw = torch.zeros(n * k, dtype=torch.float64, device=DEVICE)
    dw[pairs] = (dout * rows).sum(1)
    del rows
    drows = torch.zeros((n * k, H), dtype=torch.float64, device=DEVICE)
    drows[:m] = dout * w[:, None]
    del dout
    dx = torch.zeros((n, H), dtype=torch.float64, device=DEVICE)
    dx.index_add_(0, pairs // k, s["dxs"][:m].double())
    xs = torch.zeros((n * k, H), dtype=torch.float64, device=DEVICE)
    xs[:m] = s["x"].double()[pairs // k]
    return {"xs": xs, "out": out, "drows": drows, "dw": dw.view(n, k), "dx": dx}
