"""Operators a training or serving step needs around routed experts: token rows sorted by expert and back with their
gradients, layer norm with its gradients, and the clipping of gradients by their global norm.

A case is a dict of plain values with "op":

  sort   T tokens with k picks of E experts, rows of width d. mode "forward": plan, rows to the experts, weighted rows back;
         mode "step": the same and both backward passes. x: element type of the token rows; rows: that of the sorted rows;
         align: every expert's rows start on a multiple of it; zipf: skewed load; drop: share of picks without a row (an
         expert's capacity); pad: share of tokens at the batch's end without any pick
  norm   layer norm of T rows of width d. mode "forward" (no statistics kept) or "step" (forward and backward). x: element type
         of the rows and their gradient; y: that of the normalised rows and of their gradient
  clip   gradients of `layers` layers in the layout of the mixture-of-experts layer (router, gate, up, down) with two norm
         weights and `odd` ragged tensors each, clipped to `max_norm` times their norm; dtype: "f32", "bf16" or "mixed"
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
EPS = 1e-5


def _sort(name, mode, T, d, E, k, x="bf16", rows=None, align=1, zipf=False, drop=0.0, pad=0.0):
    c = dict(op="sort", mode=mode, T=T, d=d, E=E, k=k, x=x, rows=rows or x, align=align, zipf=zipf, drop=drop, pad=pad)
    return dict(c, name=name) if name else c


def _norm(name, mode, T, d, x="bf16", y=None):
    c = dict(op="norm", mode=mode, T=T, d=d, x=x, y=y or x)
    return dict(c, name=name) if name else c


def _clip(name, layers, d, dff, E, dtype="f32", max_norm=0.1, odd=0):
    c = dict(op="clip", layers=layers, d=d, dff=dff, E=E, dtype=dtype, max_norm=max_norm, odd=odd)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode step of eight sequences on many small experts: launches and latency
        _sort("sort_decode_8", "forward", 8, 2048, 64, 6, zipf=True),
        # a training step of the mid-size layer, segments of whole 128-row tensor-core tiles
        _sort("sort_step_4096", "step", 4096, 1024, 8, 2, align=128),
        # the engine's fp32 rows, sizes off every tile, a padded batch and picks dropped at the experts' capacity
        _sort("sort_ragged_1531", "step", 1531, 1544, 12, 3, x="f32", align=16, zipf=True, drop=0.04, pad=0.2),
        # a training step on many small experts with a skewed load, fp32 rows in and out, bf16 at the experts
        _sort("sort_step_8192", "step", 8192, 2048, 64, 6, x="f32", rows="bf16", align=128, zipf=True),
        # one token generated
        _norm("norm_decode_1", "forward", 1, 4096),
        # a training step of the mid-size block
        _norm("norm_step_4096", "step", 4096, 1024),
        # rows of an odd width, as a padded vocabulary or a pruned model has them
        _norm("norm_odd_1531", "step", 1531, 1001, x="f32", y="bf16"),
        # a training step of the large block
        _norm("norm_step_16384", "step", 16384, 4096),
        # the small fp32 layer
        _clip("clip_small", 1, 128, 256, 8),
        # a model of many ragged tensors of both types
        _clip("clip_many", 24, 264, 360, 4, dtype="mixed", odd=9),
        # a norm below the limit: nothing is scaled
        _clip("clip_none_mid", 1, 1024, 2816, 8, dtype="bf16", max_norm=2.0),
        # an expert-parallel rank's share of the large layer
        _clip("clip_large", 1, 4096, 14336, 2),
    ]


# What a drawn case may hold: sorted row elements, normalised elements, gradient elements.
_SORT_MAX, _NORM_MAX, _CLIP_MAX = 8192 * 6 * 2048, 16384 * 4096, 2 * 3 * 4096 * 14336


def _log(rng, lo, hi, step=1):
    """Uniform over the logarithm of [lo, hi], a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, step * round(v / step)))


def draw(rng):
    op = rng.choice(["sort", "norm", "clip"])
    if op == "sort":
        E = rng.choice([4, 8, 12, 16, 60, 64, 128])
        k = rng.randint(1, 8 if E >= 60 else 4)
        d = _log(rng, 128, 4096, 1 if rng.random() < 0.15 else 8)
        T = _log(rng, 1, max(2, min(16384, _SORT_MAX // (k * d))))
        x = rng.choice(["bf16", "bf16", "f32"])
        return _sort(None, rng.choice(["forward", "step", "step"]), T, d, E, k, x=x, rows=rng.choice([x, "bf16"]),
                     align=rng.choice([1, 16, 128]), zipf=rng.random() < 0.5, drop=rng.choice([0.0, 0.0, 0.05]),
                     pad=rng.choice([0.0, 0.0, 0.3]))
    if op == "norm":
        d = _log(rng, 64, 16384, 1 if rng.random() < 0.2 else 8)
        T = _log(rng, 1, max(2, min(65536, _NORM_MAX // d)))
        x = rng.choice(["bf16", "bf16", "f32"])
        return _norm(None, rng.choice(["forward", "step", "step"]), T, d, x=x, y=rng.choice([x, "bf16"]))
    while True:
        layers, d, dff, E = _log(rng, 1, 40), _log(rng, 64, 2048, 8), _log(rng, 64, 4096, 8), rng.choice([1, 2, 4, 8])
        odd = rng.randint(0, 8)
        if layers * (3 * E * d * dff + E * d + 2 * d + odd * 5000) <= _CLIP_MAX:
            break
    return _clip(None, layers, d, dff, E, dtype=rng.choice(["f32", "bf16", "mixed"]), max_norm=rng.choice([0.1, 0.5, 2.0]), odd=odd)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _rows_cap(c):
    """Rows that hold every pick and the padding of the experts that can have one."""
    n = c["T"] * c["k"]
    return -(-(n + min(c["E"], n) * (c["align"] - 1)) // c["align"]) * c["align"]


def _sort_inputs(c, seed):
    T, d, E, k = c["T"], c["d"], c["E"], c["k"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    logits = rn(T, E)
    if c["zipf"]:
        logits += 2.0 * (torch.randperm(E, generator=g, device="cuda") + 1.0) ** -1.1
    top, idx = logits.topk(k, dim=1)
    idx = idx.to(torch.int32)
    if c["drop"]:
        idx[torch.rand(T, k, generator=g, device="cuda") < c["drop"]] = -1
    if c["pad"]:
        idx[T - int(c["pad"] * T):] = -1
    cap, x, rows = _rows_cap(c), DTYPE[c["x"]], DTYPE[c["rows"]]
    s = {"idx": idx, "w": top.softmax(1).contiguous(), "x": rn(T, d).to(x), "ys": rn(cap, d).to(rows)}
    if c["mode"] == "step":
        s.update(dy=rn(T, d).to(x), dxs=rn(cap, d).to(rows))
    return s


def _norm_inputs(c, seed):
    T, d = c["T"], c["d"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    # a residual stream: columns with an offset of their own, rows of different size
    x = ((rn(T, d) + 0.5 * rn(d)) * (0.5 + torch.rand(T, 1, generator=g, device="cuda") * 2)).to(DTYPE[c["x"]])
    s = {"x": x, "gamma": 1 + 0.1 * rn(d), "beta": 0.1 * rn(d)}
    if c["mode"] == "step":
        s["dy"] = rn(T, d).to(DTYPE[c["y"]])
    return s


def _clip_shapes(c):
    """(element type, elements) of every gradient."""
    d, dff, E = c["d"], c["dff"], c["E"]
    shapes = []
    for i in range(c["layers"]):
        one = [E * d, E * dff * d, E * dff * d, E * d * dff, d, d] + [(i * 997 + j * 389) % 5000 + 1 for j in range(c["odd"])]
        shapes += [(c["dtype"] if c["dtype"] != "mixed" else "bf16" if j % 2 else "f32", n) for j, n in enumerate(one)]
    return shapes


def _carve(c):
    """One flat buffer per type and each gradient's view of it; views start on multiples of 16 bytes."""
    spans, total = [], {"f32": 0, "bf16": 0}
    for t, n in _clip_shapes(c):
        spans.append((t, total[t], n))
        total[t] += -(-n // 8) * 8
    flat = {t: torch.zeros(n, dtype=DTYPE[t], device="cuda") for t, n in total.items() if n}
    return flat, [flat[t][at:at + n] for t, at, n in spans]


def _clip_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat, grads = _carve(c)
    for i, v in enumerate(grads):
        v.copy_(torch.randn(len(v), generator=g, device="cuda").mul_(10.0 ** -(i % 4)))
    norm = torch.stack([v.double().square().sum() for v in grads]).sum().sqrt()
    return grads, c["max_norm"] * float(norm)


def prepare(case, seed):
    """Inputs, the buffers a program keeps for the sorted rows and the clipped gradients, and its handles."""
    if case["op"] == "sort":
        s = _sort_inputs(case, seed)
        for n in ("xs", "dys") if case["mode"] == "step" else ("xs",):  # rows behind the last expert's stay as they are
            s[n] = torch.zeros(_rows_cap(case), case["d"], dtype=DTYPE[case["rows"]], device="cuda")
        if own:
            from omega_ai_b200 import ops
            s["sort"] = ops.TokenSort(case["T"], case["k"], case["E"], row_align=case["align"])
    elif case["op"] == "norm":
        s = _norm_inputs(case, seed)
    else:
        grads, limit = _clip_inputs(case, seed)
        flat, out = _carve(case)
        s = {"grads": grads, "limit": limit, "flat": flat, "out": out}
        if own:
            from omega_ai_b200 import ops
            s["list"] = ops.GradList(grads, out=out)
    s["case"] = case
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        if c["op"] == "sort":
            return _sort_own(s, c)
        if c["op"] == "norm":
            return _norm_own(s, c)
        norm = s["list"].clip(s["limit"])
        return {"norm": norm, "out": s["flat"]}
    if c["op"] == "sort":
        return _sort_plain(s, c)
    if c["op"] == "norm":
        return _norm_plain(s, c)
    return _clip_plain(s)


def _sort_own(s, c):
    sort = s["sort"]
    sort.plan(s["idx"])
    sort.sort(s["x"], out=s["xs"])
    y = sort.unsort(s["ys"], s["w"], dtype=s["x"].dtype)
    r = {"pos": sort.pos, "perm": sort.perm, "counts": sort.counts, "offsets": sort.offsets, "xs": s["xs"], "y": y}
    if c["mode"] == "step":
        r["dys"], r["dw"] = sort.unsort_backward(s["dy"], s["ys"], s["w"], out=s["dys"])
        r["dx"] = sort.sort_backward(s["dxs"], dtype=s["x"].dtype)
    return r


def _norm_own(s, c):
    from omega_ai_b200 import ops

    if c["mode"] == "forward":
        return {"y": ops.layer_norm(s["x"], s["gamma"], s["beta"], EPS, dtype=DTYPE[c["y"]])}
    y, mean, rstd = ops.layer_norm(s["x"], s["gamma"], s["beta"], EPS, dtype=DTYPE[c["y"]], stats=True)
    dx, dgamma, dbeta = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], mean, rstd)
    return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _sort_plain(s, c):
    T, d, E, k, align = (c[n] for n in ("T", "d", "E", "k", "align"))
    idx, x, ys, w = s["idx"].reshape(-1).long(), s["x"], s["ys"], s["w"]
    key = torch.where((idx >= 0) & (idx < E), idx, E)
    counts = (key.unsqueeze(1) == torch.arange(E, device="cuda")).sum(0)
    ends = ((counts + align - 1) // align * align).cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    by_key = torch.sort(key, stable=True).indices
    first = torch.cat([counts.new_zeros(1), counts.cumsum(0)])  # of every key in by_key
    sorted_key = key[by_key]
    row = torch.arange(T * k, device="cuda") - first[sorted_key] + offsets[sorted_key]
    row = torch.where(sorted_key < E, row, -1)
    pos = torch.empty_like(row)
    pos[by_key] = row
    cap = len(ys)
    wide = torch.full((cap + 1,), -1, dtype=torch.int64, device="cuda")  # picks without a row land behind the last one
    wide[torch.where(pos < 0, cap, pos)] = torch.arange(T * k, device="cuda")
    perm = wide[:cap]
    there = pos.reshape(T, k) >= 0
    at = pos.reshape(T, k).clamp(min=0)
    used = (torch.arange(cap, device="cuda") < offsets[E]).unsqueeze(1)
    full = (perm >= 0).unsqueeze(1)
    token = (perm.clamp(min=0) // k)
    xs = torch.where(used, torch.where(full, x[token], 0).to(s["xs"].dtype), s["xs"])
    terms = torch.where(there.unsqueeze(2), ys[at].float(), 0.0)
    y = (w.unsqueeze(2) * terms).sum(1).to(x.dtype)
    r = {"pos": pos.reshape(T, k).to(torch.int32), "perm": perm.to(torch.int32), "counts": counts.to(torch.int32),
         "offsets": offsets.to(torch.int32), "xs": xs, "y": y}
    if c["mode"] == "step":
        dy = s["dy"].float()
        r["dw"] = (dy.unsqueeze(1) * terms).sum(2)
        scaled = dy[token] * w.reshape(-1)[perm.clamp(min=0)].unsqueeze(1)
        r["dys"] = torch.where(used, torch.where(full, scaled, 0.0).to(ys.dtype), s["dys"])
        r["dx"] = torch.where(there.unsqueeze(2), s["dxs"][at].float(), 0.0).sum(1).to(x.dtype)
    return r


def _norm_plain(s, c):
    x, gamma = s["x"].float(), s["gamma"]
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS)
    hat = (x - mean) * rstd
    r = {"y": (hat * gamma + s["beta"]).to(DTYPE[c["y"]])}
    if c["mode"] == "step":
        dy = s["dy"].float()
        g = dy * gamma
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        r.update(dx=dx.to(s["x"].dtype), dgamma=(dy * hat).sum(0), dbeta=dy.sum(0))
    return r


def _clip_plain(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    scale = torch.where(norm.isfinite(), (s["limit"] / (norm + 1e-6)).clamp(max=1.0), 1.0)
    [o.copy_(g.float() * scale) for g, o in zip(s["grads"], s["out"])]
    return {"norm": norm, "out": s["flat"]}


# ---- what a pass has to move --------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "sort":
        T, d, k = c["T"], c["d"], c["k"]
        live = T * k * (1 - c["drop"]) * (1 - c["pad"])
        pads = min(c["E"], live) * (c["align"] - 1) / 2.0  # rows of zeros, about
        rx, rr = d * SIZE[c["x"]], d * SIZE[c["rows"]]
        some = T * (1 - c["pad"])  # tokens with a pick
        nbytes = 4.0 * (3 * T * k + _rows_cap(c) + 2 * c["E"]) + some * rx + (2 * live + pads) * rr + T * rx
        flops = 2.0 * live * d
        if c["mode"] == "step":
            nbytes += 8.0 * T * k + some * rx + (3 * live + pads) * rr + T * rx  # w again and dw; dy, ys, dys, dxs, dx
            flops += 4.0 * live * d
        return {"bytes": nbytes, "flops": flops}
    if c["op"] == "norm":
        T, d = c["T"], c["d"]
        sx, sy = SIZE[c["x"]], SIZE[c["y"]]
        step = c["mode"] == "step"
        return {"bytes": T * d * (sx + sy) + 8.0 * d + (T * d * (2.0 * sx + sy) + 12.0 * d + 16.0 * T if step else 0.0),
                "flops": T * d * (19.0 if step else 7.0)}
    n = sum(SIZE[t] * m for t, m in _clip_shapes(c))
    return {"bytes": 2.0 * n + 4, "flops": 3.0 * sum(m for _, m in _clip_shapes(c))}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    """The same outputs from the definitions: experts one after the other, gradients as derivatives of the formulas."""
    if case["op"] == "sort":
        return _sort_exact(case, seed)
    if case["op"] == "norm":
        s = _norm_inputs(case, seed)
        x, gamma, beta = (s[n].double().requires_grad_(case["mode"] == "step") for n in ("x", "gamma", "beta"))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) * (var + EPS).rsqrt() * gamma + beta
        r = {"y": y.detach()}
        if case["mode"] == "step":
            r["dx"], r["dgamma"], r["dbeta"] = torch.autograd.grad(y, [x, gamma, beta], s["dy"].double())
        return r
    grads, limit = _clip_inputs(case, seed)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in grads))
    flat, out = _carve(case)
    flat64 = {t: v.double() for t, v in flat.items()}
    scale = min(1.0, limit / (norm + 1e-6))
    for g, o in zip(grads, out):
        f = flat[("bf16" if o.dtype == torch.bfloat16 else "f32")]
        at = o.storage_offset()
        flat64["bf16" if f.dtype == torch.bfloat16 else "f32"][at:at + len(o)] = g.double() * scale
    return {"norm": torch.tensor(norm, dtype=torch.float64), "out": flat64}


def _sort_exact(case, seed):
    s = _sort_inputs(case, seed)
    T, d, E, k, align = (case[n] for n in ("T", "d", "E", "k", "align"))
    cap, step = _rows_cap(case), case["mode"] == "step"
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")
    xs, y = new(cap, d), new(T, d)
    dys, dw, dx = (new(cap, d), new(T, k), new(T, d)) if step else (None, None, None)
    start = 0
    for e in range(E):
        t, j = (s["idx"] == e).nonzero(as_tuple=True)  # in the order of the flat pick index
        n = len(t)
        ys, w = s["ys"][start:start + n].double(), s["w"][t, j].double().unsqueeze(1)
        xs[start:start + n] = s["x"][t].double()
        y.index_add_(0, t, w * ys)
        if step:
            dy = s["dy"][t].double()
            dys[start:start + n] = w * dy
            dw[t, j] = torch.linalg.vecdot(dy, ys)
            dx.index_add_(0, t, s["dxs"][start:start + n].double())
        start += -(-n // align) * align
    r = {"pos": None, "perm": None, "counts": None, "offsets": None, "xs": xs, "y": y}
    if step:
        r.update(dys=dys, dw=dw, dx=dx)
    return r
