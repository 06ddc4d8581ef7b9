"""Cases of the layer norm and mixture-of-experts operators, with plain forms to measure them against.

Three operators: ``layer_norm`` (forward and backward), the expert routing ``expert_route`` /
``expert_dispatch`` / ``expert_combine`` (tokens sorted by expert and back, and the gradients), and
``expert_linear`` (the experts' products on the sorted rows, forward and backward).  ``own`` False: the
operators in elementary torch operations, in 32 bits, rounded once.  ``own`` True: the calls a user makes
of ``flash_eq``.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5


def _package():
    path = os.path.join(os.getcwd(), "flash-eq_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_eq

    return flash_eq


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the scalars of one small molecule (50 nodes, 64 channels) at inference: latency only
        dict(name="norm_molecule", op="norm", rows=50, width=64, dtype="f32", grad=False),
        # a half-precision inference batch with an odd width
        dict(name="norm_odd_f16", op="norm", rows=20011, width=1001, dtype="f16", grad=False),
        # token features of a wide model, training step in bf16
        dict(name="norm_wide_bf16", op="norm", rows=16384, width=2048, dtype="bf16", grad=True),
        # the scalars of a million-node graph (128 channels), training step
        dict(name="norm_million_f32", op="norm", rows=1000000, width=128, dtype="f32", grad=True),
        # one token served: 64 experts, two choices, a row of 64 channels x 9 components
        dict(name="route_token", op="route", tokens=1, experts=64, top_k=2, width=576, dtype="f32", normalize=True,
             masked=0.0, grad=False),
        # the nodes of the 20 000-node graph, 64 channels x 9 components, 16 experts, training step, some nodes padding
        dict(name="route_nodes_f32", op="route", tokens=20000, experts=16, top_k=2, width=576, dtype="f32",
             normalize=True, masked=0.03, grad=True),
        # a large training batch in bf16 with many experts and softmax weights that are not renormalised
        dict(name="route_large_bf16", op="route", tokens=131072, experts=64, top_k=4, width=1024, dtype="bf16",
             normalize=False, masked=0.0, grad=True),
        # the two chosen experts of one token served: the weights' bytes count
        dict(name="linear_token_bf16", op="linear", rows=2, experts=64, lvals="0", c_in=1024, c_out=2048, dtype="bf16",
             bias=True, dropped=0.0, grad=False),
        # a small served batch with odd sizes, four rows an expert
        dict(name="linear_batch_f16", op="linear", rows=131, experts=32, lvals="0", c_in=577, c_out=1001, dtype="f16",
             bias=True, dropped=0.02, grad=False),
        # the equivariant experts of a 20 000-node graph, two choices: lvals 0, 1, 2, 64 -> 128 channels, training step
        dict(name="linear_nodes_f32", op="linear", rows=40000, experts=16, lvals="0,1,2", c_in=64, c_out=128,
             dtype="f32", bias=True, dropped=0.03, grad=True),
        # scalar experts in float32, inference
        dict(name="linear_mid_f32", op="linear", rows=16384, experts=8, lvals="0", c_in=576, c_out=1152, dtype="f32",
             bias=True, dropped=0.0, grad=False),
        # a large training batch in bf16
        dict(name="linear_large_bf16", op="linear", rows=65536, experts=32, lvals="0", c_in=1024, c_out=2048,
             dtype="bf16", bias=True, dropped=0.0, grad=True),
    ]


def _log(rng, lo, hi):
    size = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return size + 1 if size == 3 * 1024 else size


def draw(rng):
    """One more case of the same ranges: sizes log-uniform, every type, both directions."""
    op = rng.choice(("norm", "route", "linear"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    grad = rng.random() < 0.5
    if op == "norm":
        width = _log(rng, 1, 8192)
        return dict(op=op, rows=_log(rng, 1, max(1, min(1000000, 100000000 // width))), width=width, dtype=dtype, grad=grad)
    if op == "route":
        experts = _log(rng, 2, 256)
        top_k, width = rng.randint(1, min(8, experts)), _log(rng, 1, 2048)
        return dict(op=op, tokens=_log(rng, 1, max(1, min(131072, 250000000 // (width * top_k)))), experts=experts,
                    top_k=top_k, width=width, dtype=dtype, normalize=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.05, 0.3)), grad=grad)
    lvals = rng.choice(("0", "0", "0,1", "0,1,2", "1,2", "0,0,1"))
    dim = sum(2 * int(v) + 1 for v in lvals.split(","))
    c_in, c_out, experts = _log(rng, 16, 2048), _log(rng, 16, 2048), _log(rng, 2, 64)
    experts = max(2, min(experts, 100000000 // (c_in * c_out * len(lvals.split(",")))))
    most = min(65536, 100000000000 // (c_in * c_out * dim), 60000000 // (dim * max(c_in, c_out)))
    return dict(op=op, rows=_log(rng, 1, max(1, most)), experts=experts, lvals=lvals, c_in=c_in, c_out=c_out, dtype=dtype,
                bias=rng.random() < 0.7, dropped=rng.choice((0.0, 0.05)), grad=grad)


def _lvals(case):
    return [int(v) for v in str(case["lvals"]).split(",")]


def work(case):
    s = _BYTES[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": float((5 if case["grad"] else 2) * n * s + (4 if case["grad"] else 2) * case["width"] * s),
                "flops": float((20 if case["grad"] else 8) * n)}
    if case["op"] == "route":
        row, tokens, picked = case["width"] * s, case["tokens"], case["tokens"] * case["top_k"]
        scores = tokens * case["experts"] * 4
        moved = 2 * tokens * row + 2 * picked * row + scores + picked * 12
        if case["grad"]:      # read both outputs' gradients and the expert rows, write all three gradients
            moved += 2 * tokens * row + 3 * picked * row + scores
        return {"bytes": float(moved), "flops": float((7 if case["grad"] else 2) * picked * case["width"])}
    lvals = _lvals(case)
    dim, rows = sum(2 * v + 1 for v in lvals), case["rows"]
    touched = min(case["experts"], rows)
    weights = touched * len(lvals) * case["c_in"] * case["c_out"] * s
    a, b = rows * dim * case["c_in"] * s, rows * dim * case["c_out"] * s
    flops = 2.0 * rows * dim * case["c_in"] * case["c_out"]
    if not case["grad"]:
        return {"bytes": float(a + b + weights), "flops": flops}
    # the weights' gradient is written for every expert, the ones without rows too
    return {"bytes": float(3 * a + 2 * b + 2 * weights + case["experts"] * len(lvals) * case["c_in"] * case["c_out"] * s),
            "flops": 3 * flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    st = {"case": dict(case)}
    if case["op"] == "norm":
        m, d = case["rows"], case["width"]
        # features with a mean and a spread of their own in every row
        x = torch.randn(m, d, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))
        st["x"] = (x + torch.randn(m, 1, generator=g, device="cuda")).to(dt)
        st["weight"], st["bias"] = normal(d, scale=0.2, shift=1.0), normal(d, scale=0.2)
        st["diff"] = [st["x"], st["weight"], st["bias"]]
        if case["grad"]:
            st["grad_out"] = normal(m, d)
    elif case["op"] == "route":
        n, e, k, d = case["tokens"], case["experts"], case["top_k"], case["width"]
        # router logits: some experts liked more than others; a masked token has no expert, and one expert in ten
        # is switched off for a masked share of the tokens
        logits = torch.randn(n, e, generator=g, device="cuda") + 0.5 * torch.randn(1, e, generator=g, device="cuda")
        if case["masked"] > 0:
            off = torch.rand(n, 1, generator=g, device="cuda") < case["masked"]
            some = (torch.rand(n, e, generator=g, device="cuda") < 0.1) & (
                torch.rand(n, 1, generator=g, device="cuda") < case["masked"])
            logits = logits.masked_fill(off | some, -math.inf)
        st["logits"] = logits
        st["x"], st["y"] = normal(n, d), normal(n * k, d)
        st["diff"] = [st["logits"], st["x"], st["y"]]
        if case["grad"]:
            st["grad_sorted"], st["grad_out"] = normal(n * k, d), normal(n, d)
    else:
        lvals, r, e = _lvals(case), case["rows"], case["experts"]
        dim, reps, ci, co = sum(2 * v + 1 for v in lvals), len(lvals), case["c_in"], case["c_out"]
        host = np.random.RandomState(int(seed) % (1 << 32))
        kept = r - int(round(r * case["dropped"]))
        liking = np.exp(0.25 * host.randn(e))
        sizes = host.multinomial(kept, liking / liking.sum())
        st["capacity"] = max(1, int(sizes.max()))      # the plan: rows of the fullest expert
        st["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda()
        st["lvals"] = tuple(lvals)
        flat = lvals == [0]
        st["x"] = normal(r, ci) if flat else normal(r, dim, ci)
        st["weight"] = normal(*((e,) if flat else (e, reps)), co, ci, scale=ci ** -0.5)
        scalars = sum(v == 0 for v in lvals)
        st["bias"] = None
        if case["bias"] and scalars:
            st["bias"] = normal(*((e,) if flat else (e, scalars)), co, scale=0.2)
        st["diff"] = [t for t in (st["x"], st["weight"], st["bias"]) if t is not None]
        if case["grad"]:
            st["grad_out"] = normal(r, co) if flat else normal(r, dim, co)
    if case["grad"]:
        for t in st["diff"]:
            t.requires_grad_()
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    one = {"norm": (_norm_plain, _norm_own), "route": (_route_plain, _route_own), "linear": (_linear_plain, _linear_own)}
    if own:
        if case["grad"]:
            return one[case["op"]][1](st)
        with torch.no_grad():
            return one[case["op"]][1](st)
    with torch.no_grad():
        return one[case["op"]][0](st)


def _norm_own(st):
    fe = _package()
    y = fe.layer_norm(st["x"], st["weight"], st["bias"], eps=_EPS)
    if not st["case"]["grad"]:
        return {"y": y}
    gx, gw, gb = torch.autograd.grad([y], st["diff"], [st["grad_out"]])
    return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}


def _norm_plain(st):
    dt = st["x"].dtype
    x, w, b = st["x"].float(), st["weight"].float(), st["bias"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = ((centred * centred).mean(-1, keepdim=True) + _EPS).rsqrt()
    unit = centred * rstd
    y = (unit * w + b).to(dt)
    if not st["case"]["grad"]:
        return {"y": y}
    g = st["grad_out"].float()
    gw = g * w
    gx = rstd * (gw - gw.mean(-1, keepdim=True) - unit * (gw * unit).mean(-1, keepdim=True))
    return {"y": y, "grad_x": gx.to(dt), "grad_weight": (g * unit).sum(0).to(dt), "grad_bias": g.sum(0).to(dt)}


def _route_own(st):
    fe = _package()
    case = st["case"]
    route = fe.expert_route(st["logits"], case["top_k"], normalize=case["normalize"])
    xs = fe.expert_dispatch(st["x"], route)
    out = fe.expert_combine(st["y"], route)
    got = {"experts": route.experts, "slots": route.slots, "offsets": route.offsets, "weights": route.weights,
           "sorted": xs, "out": out}
    if not case["grad"]:
        return got
    gl, gx, gy = torch.autograd.grad([xs, out], st["diff"], [st["grad_sorted"], st["grad_out"]])
    return {**got, "grad_logits": gl, "grad_x": gx, "grad_y": gy}


def _route_plain(st):
    case = st["case"]
    n, e, k = case["tokens"], case["experts"], case["top_k"]
    dt = st["x"].dtype
    logits, x, y = st["logits"], st["x"].float(), st["y"].float()
    top, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    live = top > -math.inf
    biggest = logits.amax(-1, keepdim=True)
    biggest = torch.where(biggest > -math.inf, biggest, torch.zeros_like(biggest))
    chosen, every = (top - biggest).exp(), (logits - biggest).exp()
    total = (chosen if case["normalize"] else every).sum(-1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    weights = chosen / total
    flat = torch.where(live, ids, torch.full_like(ids, e)).reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k, device=order.device)
    offsets = (flat[:, None] < torch.arange(e + 1, device=flat.device)).sum(0)
    keep = live.reshape(-1, 1)
    xs = torch.where(keep[order], x[order // k], torch.zeros((), device=x.device))
    rows = torch.where(keep, y[slots], torch.zeros((), device=x.device)).view(n, k, -1)
    out = (rows * weights[..., None]).sum(1)
    got = {"experts": torch.where(live, ids, torch.full_like(ids, -1)).to(torch.int32),
           "slots": slots.view(n, k).to(torch.int32), "offsets": offsets.to(torch.int32), "weights": weights,
           "sorted": xs.to(dt), "out": out.to(dt)}
    if not case["grad"]:
        return got
    gs, go = st["grad_sorted"].float(), st["grad_out"].float()
    gx = torch.where(keep, gs[slots.view(-1)], torch.zeros((), device=x.device)).view(n, k, -1).sum(1)
    gy = torch.empty_like(y)
    gy[slots.view(-1)] = torch.where(keep.view(n, k, 1), go[:, None] * weights[..., None],
                                     torch.zeros((), device=x.device)).view(n * k, -1)
    gweights = (rows * go[:, None]).sum(-1)
    share = (weights * gweights).sum(-1, keepdim=True)
    picked = torch.zeros_like(logits).scatter(1, ids, weights * gweights * live)
    spread = torch.zeros_like(logits).scatter(1, ids, weights) if case["normalize"] else every / total
    return {**got, "grad_logits": picked - spread * share, "grad_x": gx.to(dt), "grad_y": gy.to(dt)}


def _linear_own(st):
    fe = _package()
    y = fe.expert_linear(st["x"], st["weight"], st["bias"], st["offsets"], lvals=st["lvals"])
    if not st["case"]["grad"]:
        return {"y": y}
    return {"y": y, "grads": list(torch.autograd.grad([y], st["diff"], [st["grad_out"]]))}


def _irreps(lvals):
    return [i for i, v in enumerate(lvals) for _ in range(2 * v + 1)]


def _linear_plain(st):
    """Every expert's rows in a block of the fullest expert's size, and one batched product over the blocks."""
    case, lvals = st["case"], st["lvals"]
    e, r, cap, co, ci = case["experts"], case["rows"], st["capacity"], case["c_out"], case["c_in"]
    dt, dev = st["x"].dtype, st["x"].device
    part = torch.tensor(_irreps(lvals), device=dev)
    scalar = torch.tensor([i for i, v in enumerate(lvals) if v == 0], dtype=torch.long, device=dev)
    dim, reps = part.numel(), len(lvals)
    x, w = st["x"].float().view(r, dim, ci), st["weight"].float().view(e, reps, co, ci)[:, part]
    row = torch.arange(r, device=dev)
    expert = torch.searchsorted(st["offsets"][1:].long(), row, right=True)
    kept = expert < e
    at = torch.where(kept, expert * cap + row - st["offsets"].long()[expert.clamp(max=e - 1)], torch.full_like(row, e * cap))

    def blocks(t):                        # (R, dim, C) -> (E, dim, cap, C)
        buf = torch.zeros(e * cap + 1, dim, t.shape[-1], device=dev)
        buf[at] = torch.where(kept[:, None, None], t, torch.zeros((), device=dev))
        return buf[:-1].view(e, cap, dim, -1).transpose(1, 2)

    def back(t):                          # (E, dim, cap, C) -> (R, dim, C)
        flat = t.transpose(1, 2).reshape(e * cap, dim, -1)
        return torch.where(kept[:, None, None], flat[at.clamp(max=e * cap - 1)], torch.zeros((), device=dev))

    spots = torch.isin(part, scalar)      # the l = 0 components, in the order of the bias
    xb = blocks(x)
    yb = xb @ w.transpose(-1, -2)
    if st["bias"] is not None:
        yb[:, spots] += st["bias"].float().view(e, -1, 1, co)
    y = back(yb).to(dt).view(*st["x"].shape[:-1], co)
    if not case["grad"]:
        return {"y": y}
    gb = blocks(st["grad_out"].float().view(r, dim, co))
    gx = back(gb @ w).to(dt).view_as(st["x"])
    gw = torch.zeros(e, reps, co, ci, device=dev).index_add(1, part, gb.transpose(-1, -2) @ xb).to(dt).view_as(st["weight"])
    grads = [gx, gw]
    if st["bias"] is not None:
        grads.append(gb[:, spots].sum(2).to(dt).view_as(st["bias"]))
    return {"y": y, "grads": grads}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _norm_exact, "route": _route_exact, "linear": _linear_exact}[case["op"]](st)


def _norm_exact(st):
    x, w, b = st["x"].double(), st["weight"].double(), st["bias"].double()
    d = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / d
    sd = torch.sqrt(torch.sum((x - mean) ** 2, -1, keepdim=True) / d + _EPS)
    y = (x - mean) / sd * w + b
    if not st["case"]["grad"]:
        return {"y": y}
    # the Jacobian of one row: (I - 1 1^T / D - u u^T / D) / sd with u the normalised row
    g, u = st["grad_out"].double(), (x - mean) / sd
    v = g * w
    gx = (v - v.sum(-1, keepdim=True) / d - u * (torch.einsum("md,md->m", v, u) / d)[:, None]) / sd
    return {"y": y, "grad_x": gx, "grad_weight": torch.einsum("md,md->d", g, u), "grad_bias": torch.einsum("md->d", g)}


def _route_exact(st):
    case = st["case"]
    n, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = st["logits"].cpu().numpy().astype(np.float64)
    # the k largest by (logit downwards, index upwards); -inf is never chosen
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k]
    val = np.take_along_axis(logits, ids, 1)
    live = val > -np.inf
    with np.errstate(invalid="ignore", divide="ignore"):
        p = np.exp(logits - np.where(live[:, :1], val[:, :1], 0.0))
        mass = (np.take_along_axis(p, ids, 1) * live).sum(1) if case["normalize"] else p.sum(1)
        w = np.where(live, np.take_along_axis(p, ids, 1) / mass[:, None], 0.0)
    key = np.where(live, ids, e).reshape(-1)
    order = np.argsort(key, kind="stable")
    slots = np.empty(n * k, dtype=np.int64)
    slots[order] = np.arange(n * k)
    dev = st["x"].device
    x, y = st["x"].double(), st["y"].double()
    w_, live_ = torch.from_numpy(w).to(dev), torch.from_numpy(live).to(dev)
    slot_, order_ = torch.from_numpy(slots).to(dev).view(n, k), torch.from_numpy(order).to(dev)
    xs = x[order_ // k] * live_.view(-1, 1)[order_]
    out = torch.zeros_like(x)
    for j in range(k):
        out += y[slot_[:, j]] * (w_[:, j] * live_[:, j])[:, None]
    got = {"experts": None, "slots": None, "offsets": None, "weights": w_, "sorted": xs, "out": out}
    if not case["grad"]:
        return got
    gs, go = st["grad_sorted"].double(), st["grad_out"].double()
    gx, gy, gw = torch.zeros_like(x), torch.zeros_like(y), torch.zeros_like(w_)
    for j in range(k):
        gx += gs[slot_[:, j]] * live_[:, j, None]
        gy[slot_[:, j]] = go * (w_[:, j] * live_[:, j])[:, None]
        gw[:, j] = torch.einsum("nd,nd->n", go, y[slot_[:, j]]) * live_[:, j]
    # d w_j / d logit_e = w_j (delta_je - q_e), q the softmax that w was taken from
    q = torch.zeros(n, e, dtype=torch.float64, device=dev)
    at = torch.from_numpy(ids.copy()).to(dev)
    if case["normalize"]:
        q.scatter_(1, at, w_)
    else:
        q = torch.from_numpy(np.where(live[:, :1], p / np.where(mass > 0, mass, 1.0)[:, None], 0.0)).to(dev)
    gl = -q * (w_ * gw).sum(1, keepdim=True)
    gl.scatter_add_(1, at, w_ * gw)
    return {**got, "grad_logits": gl, "grad_x": gx, "grad_y": gy}


def _linear_exact(st):
    case, lvals = st["case"], list(st["lvals"])
    e, r, co, ci = case["experts"], case["rows"], case["c_out"], case["c_in"]
    dim, reps, ends = sum(2 * v + 1 for v in lvals), len(lvals), st["offsets"].tolist()
    x, w = st["x"].double().view(r, dim, ci), st["weight"].double().view(e, reps, co, ci)
    bias = None if st["bias"] is None else st["bias"].double().view(e, -1, co)
    y = torch.zeros(r, dim, co, dtype=torch.float64, device=x.device)
    grad = case["grad"]
    if grad:
        g = st["grad_out"].double().view(r, dim, co)
        gx, gw = torch.zeros_like(x), torch.zeros_like(w)
        gb = None if bias is None else torch.zeros_like(bias)
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        at = scalars = 0
        for rep, v in enumerate(lvals):
            part = slice(at, at + 2 * v + 1)
            at += 2 * v + 1
            y[a:b, part] = torch.einsum("rpc,oc->rpo", x[a:b, part], w[i, rep])
            if grad:
                gx[a:b, part] = torch.einsum("rpo,oc->rpc", g[a:b, part], w[i, rep])
                gw[i, rep] = torch.einsum("rpo,rpc->oc", g[a:b, part], x[a:b, part])
            if v == 0 and bias is not None:
                y[a:b, part] += bias[i, scalars]
                if grad:
                    gb[i, scalars] = g[a:b, part].sum((0, 1))
                scalars += 1
    y = y.view(*st["x"].shape[:-1], co)
    if not grad:
        return {"y": y}
    grads = [gx.view(st["x"].shape), gw.view(st["weight"].shape)]
    return {"y": y, "grads": grads if gb is None else grads + [gb.view(st["bias"].shape)]}
