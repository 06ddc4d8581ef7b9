"""Expert routing, dispatch, combine and expert linear (csrc/feq_experts.cu, csrc/feq_expertlin.cu) and
the layer that runs them together, against plain definitions in float64.

Tolerances, relative L2 over an output.  float32: products and sums of K terms in float32 with
partial sums of a few hundred terms: below 2e-6.  16-bit types: the inputs are exact, the result is
rounded once, at most 2^-9 (bfloat16) or 2^-12 (float16) of each value, doubled.  Experts, slots and
offsets are whole numbers and have to be equal.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

import flash_eq as fe
from conftest import check_equivariance, rel_l2
from flash_eq.cuda import _lib, token_ops

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------
def _route_reference(logits, k, normalize):
    """experts, weights (differentiable, float64), slots, offsets by sorting on the CPU."""
    z = logits.double().cpu()
    n, e = z.shape
    ids = torch.empty(n, k, dtype=torch.long)
    for t in range(n):
        order = sorted(range(e), key=lambda i: (not math.isnan(z[t, i]), -z[t, i].item() if not math.isnan(z[t, i]) else 0, i))
        order = [i for i in order if z[t, i] != -math.inf][:k]
        ids[t] = torch.tensor(order + [-1] * (k - len(order)))
    live = ids >= 0
    zr = z.clone().requires_grad_()
    pick = zr.gather(1, ids.clamp(min=0)).masked_fill(~live, -math.inf)
    dead = ~live.any(1, keepdim=True)
    if normalize:
        w = torch.softmax(pick.masked_fill(dead, 0.0), -1)
    else:
        w = torch.softmax(zr.masked_fill(dead, 0.0), -1).gather(1, ids.clamp(min=0))
    w = torch.where(live, w, torch.zeros_like(w))
    flat = torch.where(live, ids, torch.full_like(ids, e)).reshape(-1)
    perm = torch.sort(flat, stable=True)[1]
    slots = torch.empty_like(perm)
    slots[perm] = torch.arange(n * k)
    offsets = torch.tensor([int((flat < i).sum()) for i in range(e + 1)])
    return ids, w, slots.view(n, k), offsets, zr


ROUTES = [(1, 1, 1), (1, 64, 2), (3, 5, 5), (50, 16, 2), (257, 33, 4), (1000, 512, 3), (700, 40, 32), (4097, 8, 1),
          (9000, 130, 2), (2048, 2, 2)]


def _logits(n, e, seed, dtype=torch.float32, masked=True):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, e, generator=g)
    if masked and n > 2:
        z[torch.rand(n, e, generator=g) < 0.2] = -math.inf
        z[torch.rand(n, generator=g) < 0.1] = -math.inf         # tokens without any expert
    return z.to(dtype)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n,e,k", ROUTES, ids=[f"{n}-{e}-{k}" for n, e, k in ROUTES])
def test_route(cuda_device, n, e, k, normalize):
    z = _logits(n, e, 1)
    ids, w, slots, offsets, zr = _route_reference(z, k, normalize)
    zg = z.to(cuda_device).requires_grad_()
    r = fe.expert_route(zg, k, normalize)
    assert torch.equal(r.experts.cpu().long(), ids)
    assert torch.equal(r.slots.cpu().long(), slots)
    assert torch.equal(r.offsets.cpu().long(), offsets)
    assert (r.num_tokens, r.num_experts, r.top_k) == (n, e, k)
    assert rel_l2(r.weights.detach(), w.detach()) < 2e-6
    go = torch.randn(n, k, generator=torch.Generator().manual_seed(2))
    got = torch.autograd.grad(r.weights, zg, go.to(cuda_device))[0]
    want = torch.autograd.grad(w, zr, go.double())[0]
    # with every choice weighted 1 (one expert) the gradient is exactly zero
    assert rel_l2(got, want) < 2e-6 or (got.cpu().double() - want).abs().max() < 1e-6


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_route_ties_and_types(cuda_device, dtype):
    """Few distinct values: equal logits go to the lower expert; -0 equals +0."""
    g = torch.Generator().manual_seed(3)
    z = torch.randint(-2, 3, (3000, 24), generator=g).to(dtype)
    z[0, :4] = torch.tensor([-0.0, 0.0, -0.0, 0.0], dtype=dtype)
    z[0, 4:] = -5
    ids, w, slots, offsets, _ = _route_reference(z, 3, True)
    r = fe.expert_route(z.to(cuda_device), 3)
    assert torch.equal(r.experts.cpu().long(), ids) and torch.equal(r.slots.cpu().long(), slots)
    assert torch.equal(r.offsets.cpu().long(), offsets) and rel_l2(r.weights, w.detach()) < 2e-6
    assert r.experts[0].tolist() == [0, 1, 2]


def test_route_extremes(cuda_device):
    low = torch.finfo(torch.float32).min
    inf, nan = math.inf, math.nan
    z = torch.tensor([[low, low, low, low], [-inf, -inf, -inf, -inf], [1.0, -inf, low, -inf], [3e38, -3e38, 0.0, 1.0],
                      [nan, 1.0, 2.0, nan], [0.0, inf, 1.0, -inf]], device=cuda_device)
    r = fe.expert_route(z, 2)
    assert r.experts.tolist() == [[0, 1], [-1, -1], [0, 2], [0, 3], [0, 3], [1, 2]]
    assert r.weights[:4].tolist() == [[0.5, 0.5], [0.0, 0.0], [1.0, 0.0], [1.0, 0.0]]
    assert r.weights[4].isnan().all() and r.weights[5].isnan().any()
    assert r.offsets.tolist()[-1] == 10 and sorted(r.slots.flatten().tolist()) == list(range(12))
    # the lowest finite value is an ordinary logit: the softmax over all of them, too
    assert torch.equal(fe.expert_route(z[:1], 4, normalize=False).weights, torch.full((1, 4), 0.25, device=cuda_device))


def test_route_strided_empty_and_one_sided(cuda_device):
    z = _logits(300, 40, 5).to(cuda_device)
    for view in (z[:, 3:20], z[::3], z.t()[:17].t()):
        a, b = fe.expert_route(view, 2), fe.expert_route(view.contiguous(), 2)
        assert all(torch.equal(getattr(a, f), getattr(b, f)) for f in ("experts", "weights", "slots", "offsets"))
    r = fe.expert_route(z[:0], 2)
    assert r.slots.shape == (0, 2) and r.offsets.tolist() == [0] * 41
    z = torch.zeros(6000, 8, device=cuda_device)
    z[:, 5] = 1.0                                           # every token likes one expert
    r = fe.expert_route(z, 1)
    assert r.offsets.tolist() == [0] * 6 + [6000] * 3
    assert torch.equal(r.slots.flatten(), torch.arange(6000, device=cuda_device, dtype=torch.int32))


# ---------------------------------------------------------------------------
# dispatch and combine
# ---------------------------------------------------------------------------
WIDTHS = [1, 3, 8, 31, 64, 129, 576, 1001]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width", WIDTHS)
def test_dispatch_and_combine(cuda_device, width, dtype):
    n, e, k = 203, 12, 3
    z = _logits(n, e, 7).to(cuda_device).requires_grad_()
    g = torch.Generator().manual_seed(width)
    x, y = torch.randn(n, width, generator=g), torch.randn(n * k, width, generator=g)
    gs, go = torch.randn(n * k, width, generator=g), torch.randn(n, width, generator=g)
    x, y, gs, go = (t.to(cuda_device, dtype) for t in (x, y, gs, go))
    x.requires_grad_(), y.requires_grad_()
    r = fe.expert_route(z, k)
    xs, out = fe.expert_dispatch(x, r), fe.expert_combine(y, r)
    gz, gx, gy = torch.autograd.grad([xs, out], [z, x, y], [gs, go])

    slots, live = r.slots.long(), r.experts >= 0
    w = r.weights.detach().double()
    xr = torch.zeros(n * k, width, dtype=torch.float64, device=cuda_device)
    xr[slots[live]] = x.detach().double().unsqueeze(1).expand(n, k, width)[live]
    assert torch.equal(xs.detach().double(), xr)
    rows = y.detach().double()[slots] * live.unsqueeze(-1)
    assert rel_l2(out.detach(), (rows * w.unsqueeze(-1)).sum(1)) < TOL[dtype]
    assert rel_l2(gx, (gs.double()[slots] * live.unsqueeze(-1)).sum(1)) < TOL[dtype]
    gyr = torch.zeros_like(xr)
    gyr[slots.flatten()] = (go.double().unsqueeze(1) * w.unsqueeze(-1)).reshape(n * k, width)
    assert rel_l2(gy, gyr) < TOL[dtype]
    gw = (rows * go.double().unsqueeze(1)).sum(-1)
    zr = z.detach().double().requires_grad_()
    pick = zr.gather(1, r.experts.clamp(min=0).long()).masked_fill(~live, -math.inf)
    dead = ~live.any(1, keepdim=True)
    wr = torch.softmax(pick.masked_fill(dead, 0.0), -1) * live
    # float32 products summed in float32: the logits' gradient is float32 whatever the rows' type
    assert rel_l2(gz, torch.autograd.grad(wr, zr, gw)[0]) < 4e-6


def test_rows_without_an_expert_hide_what_they_hold(cuda_device):
    """NaN and infinity in the rows of pairs without an expert reach nothing."""
    z = _logits(100, 6, 8)
    z[::4] = -math.inf
    z = z.to(cuda_device).requires_grad_()
    r = fe.expert_route(z, 2)
    gone = (r.experts < 0).flatten()
    y = torch.randn(200, 40, device=cuda_device)
    y[r.slots.flatten().long()[gone]] = math.nan
    x = torch.randn(100, 40, device=cuda_device)
    x[::4] = math.inf
    x.requires_grad_(), y.requires_grad_()
    out, xs = fe.expert_combine(y, r), fe.expert_dispatch(x, r)
    assert torch.isfinite(out).all() and torch.equal(out[::4], torch.zeros_like(out[::4]))
    assert torch.isfinite(xs).all()
    gs = torch.randn(200, 40, device=cuda_device)
    gs[r.slots.flatten().long()[gone]] = math.nan
    grads = torch.autograd.grad([xs, out], [z, x, y], [gs, torch.randn_like(out)])
    assert all(torch.isfinite(t).all() for t in grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dispatch_and_combine_strided(cuda_device, dtype):
    r = fe.expert_route(_logits(90, 7, 9).to(cuda_device), 2)
    base = torch.randn(180, 150, device=cuda_device).to(dtype)
    for cols in (slice(0, 64), slice(3, 67), slice(16, 80), slice(0, 75)):
        x, y = base[:90, cols], base[:, cols]
        assert torch.equal(fe.expert_dispatch(x, r), fe.expert_dispatch(x.contiguous(), r))
        assert torch.equal(fe.expert_combine(y, r), fe.expert_combine(y.contiguous(), r))
    x = base[:90].view(90, 5, 30)
    assert torch.equal(fe.expert_dispatch(x, r).view(180, 150), fe.expert_dispatch(base[:90], r))
    assert fe.expert_combine(base.view(180, 5, 30), r).shape == (90, 5, 30)
    assert torch.equal(fe.expert_dispatch(base[:1].expand(90, 150), r)[: int(r.offsets[-1])],
                       base[:1].expand(int(r.offsets[-1]), 150))


def test_a_plan_that_does_not_fit_touches_nothing_else(cuda_device):
    """Slots outside the sorted rows are skipped by the kernels' own check."""
    r = fe.expert_route(torch.randn(8, 4, device=cuda_device), 2)
    slots = r.slots.clone()
    slots[0, 0], slots[1, 1] = 1 << 30, -5
    bad = fe.ExpertRoute(r.experts, r.weights, slots, r.offsets)
    y = torch.randn(16, 24, device=cuda_device)
    out = fe.expert_combine(y, bad)
    assert rel_l2(out[0], y[slots[0, 1].long()] * r.weights[0, 1]) < 2e-6
    guard = token_ops.expert_dispatch(torch.ones(8, 24, device=cuda_device), slots, r.offsets)
    assert guard.shape == (16, 24)


# ---------------------------------------------------------------------------
# expert linear
# ---------------------------------------------------------------------------
def _linear_reference(x, w, b, offsets, lvals, go):
    x, w, go = x.double(), w.double(), go.double()
    y, gx, gw = torch.zeros_like(go), torch.zeros_like(x), torch.zeros_like(w)
    gb = None if b is None else torch.zeros_like(b.double())
    for e in range(w.shape[0]):
        rows, at, s = slice(int(offsets[e]), int(offsets[e + 1])), 0, 0
        for i, l in enumerate(lvals):
            p = slice(at, at + 2 * l + 1)
            at += 2 * l + 1
            y[rows, p] = x[rows, p] @ w[e, i].t()
            gx[rows, p] = go[rows, p] @ w[e, i]
            gw[e, i] = torch.einsum("rpo,rpc->oc", go[rows, p], x[rows, p])
            if l == 0 and b is not None:
                y[rows, p] += b[e, s].double()
                gb[e, s] = go[rows, p].sum((0, 1))
                s += 1
    return y, gx, gw, gb


def _linear_inputs(sizes, dropped, lvals, ci, co, dtype, device, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    e, dim, scalars = len(sizes), sum(2 * v + 1 for v in lvals), sum(v == 0 for v in lvals)
    rows = sum(sizes) + dropped
    r = lambda *s: torch.randn(*s, generator=g).to(device, dtype)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32, device=device)
    x, go = r(rows, dim, ci), r(rows, dim, co)
    w = (torch.randn(e, len(lvals), co, ci, generator=g) * ci ** -0.5).to(device, dtype)
    b = r(e, scalars, co) if bias and scalars else None
    return x, w, b, offsets, go


def _linear_check(x, w, b, offsets, lvals, go, tol=None):
    leaves = [t.detach().requires_grad_() for t in (x, w) + (() if b is None else (b,))]
    y = fe.expert_linear(leaves[0], leaves[1], leaves[2] if b is not None else None, offsets, lvals)
    grads = torch.autograd.grad(y, leaves, go)
    want = _linear_reference(x, w, b, offsets, lvals, go)
    tol = tol or TOL[x.dtype]
    assert y.dtype == x.dtype
    last = int(offsets[-1])
    assert torch.equal(y[last:], torch.zeros_like(y[last:])) and torch.equal(grads[0][last:], torch.zeros_like(grads[0][last:]))
    for name, got, ref in zip(("y", "grad_x", "grad_weight", "grad_bias"), (y.detach(), *grads), want):
        assert got.shape == ref.shape
        assert torch.isfinite(got).all(), name
        assert rel_l2(got, ref) < tol, name


LINEAR = [
    # sizes per expert, rows without one, lvals, c_in, c_out
    ([1], 0, (0,), 16, 16),
    ([1, 0, 2], 1, (0,), 33, 17),
    ([5, 0, 130, 64, 1], 3, (0,), 64, 128),
    ([127, 128, 129, 0], 0, (0,), 65, 200),
    ([300, 20], 140, (0,), 256, 264),
    ([0, 0, 0], 5, (0,), 40, 24),
    ([17, 40, 3], 2, (0, 1, 2), 64, 128),
    ([9, 0, 150], 0, (1,), 24, 40),
    ([33, 70], 1, (0, 0, 1), 8, 72),
    ([4] * 40, 0, (0,), 96, 320),
    ([700, 1, 513], 9, (0, 1), 130, 62),
    ([2500, 3], 0, (0,), 128, 136),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", range(len(LINEAR)))
def test_expert_linear(cuda_device, case, dtype):
    sizes, dropped, lvals, ci, co = LINEAR[case]
    x, w, b, offsets, go = _linear_inputs(sizes, dropped, lvals, ci, co, dtype, cuda_device, seed=case)
    _linear_check(x, w, b, offsets, lvals, go)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_expert_linear_plain_rows_without_bias(cuda_device, dtype):
    x, w, _, offsets, go = _linear_inputs([70, 0, 61], 4, (0,), 72, 48, dtype, cuda_device, bias=False)
    _linear_check(x, w, None, offsets, (0,), go)
    y = fe.expert_linear(x[:, 0], w[:, 0], None, offsets)
    assert y.shape == (135, 48) and torch.equal(y, fe.expert_linear(x, w, None, offsets)[:, 0])
    assert torch.equal(y, fe.expert_linear(x[:, 0], w[:, 0], None, offsets.long()))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_expert_linear_strided(cuda_device, dtype):
    """Rows and components with strides and offsets of their own, aligned and not."""
    lvals = (0, 1)
    x, w, b, offsets, go = _linear_inputs([40, 90, 7], 3, lvals, 48, 64, dtype, cuda_device)
    big = torch.randn(140, 6, 200, device=cuda_device).to(dtype)
    for view in (big[:, 1:5, 8:56], big[:, :4, 3:51], big.transpose(0, 1).contiguous().transpose(0, 1)[:, 2:6, :48]):
        _linear_check(view, w, b, offsets, lvals, go)
    g = torch.randn(140, 9, 100, device=cuda_device).to(dtype)[:, 2:6, 1:65]
    _linear_check(x, w, b, offsets, lvals, g)
    _linear_check(x[:1].expand(140, 4, 48), w, b, offsets, lvals, go)
    _linear_check(x, w.transpose(2, 3).contiguous().transpose(2, 3), b, offsets, lvals, go)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_expert_linear_keeps_other_rows_out(cuda_device, dtype):
    """NaN and infinity of one expert's rows, or of rows without an expert, stay where they are."""
    sizes = [70, 3, 0, 129]
    x, w, b, offsets, go = _linear_inputs(sizes, 6, (0,), 64, 80, dtype, cuda_device)
    clean = fe.expert_linear(x, w, b, offsets)
    x[70:73], go[70:73] = math.nan, math.inf
    x[202:], go[202:] = math.inf, math.nan
    leaves = [x.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    y = fe.expert_linear(*leaves, offsets)
    grads = torch.autograd.grad(y, leaves, go)
    keep = torch.tensor([*range(70), *range(73, 202)], device=cuda_device)
    assert torch.equal(y[keep], clean[keep]) and torch.equal(y[202:], torch.zeros_like(y[202:]))
    assert torch.isfinite(grads[0][keep]).all() and torch.equal(grads[0][202:], torch.zeros_like(grads[0][202:]))
    for t in grads[1:]:
        assert torch.isfinite(t[[0, 2, 3]]).all() and not torch.isfinite(t[1]).any()
        assert torch.equal(t[2], torch.zeros_like(t[2]))


def test_expert_linear_offsets_out_of_range_are_clamped(cuda_device):
    x, w, b, offsets, _ = _linear_inputs([30, 30], 4, (0,), 32, 32, torch.float32, cuda_device)
    bad = torch.tensor([-7, 30, 1 << 30], dtype=torch.int32, device=cuda_device)
    want = fe.expert_linear(x, w, b, torch.tensor([0, 30, 64], dtype=torch.int32, device=cuda_device))
    assert torch.equal(fe.expert_linear(x, w, b, bad), want)


def test_expert_linear_gradient_against_differences(cuda_device):
    """The map is linear in each argument, so a central difference with step 1 is exact up to
    rounding: 1e-7 of the sums' size, bounded by 1e-4 of the slope's scale."""
    x, w, b, offsets, go = _linear_inputs([20, 0, 45], 2, (0, 1), 24, 32, torch.float32, cuda_device, seed=4)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fe.expert_linear(*leaves, offsets, (0, 1)), leaves, go)
    f = lambda p: (fe.expert_linear(*p, offsets, (0, 1)).double() * go.double()).sum().item()
    with torch.no_grad():
        for i, g in enumerate(grads):
            v = torch.randn_like(g)
            up, down = list(leaves), list(leaves)
            up[i], down[i] = leaves[i] + v, leaves[i] - v
            slope = (g.double() * v.double()).sum().item()
            scale = (g.double().norm() * v.double().norm()).item() / g.numel() ** 0.5
            assert abs((f(up) - f(down)) / 2 - slope) < 1e-4 * max(scale, abs(slope))


def test_combine_gradient_against_differences(cuda_device):
    """Through the router's softmax: step 1e-2, truncation O(h^2) about 1e-4, rounding 1e-5: 2e-3."""
    z = torch.randn(30, 6, device=cuda_device).requires_grad_()
    r = fe.expert_route(z, 3)
    y, go = torch.randn(90, 20, device=cuda_device), torch.randn(30, 20, device=cuda_device)
    g = torch.autograd.grad(fe.expert_combine(y, r), z, go)[0].double()
    picked = torch.zeros_like(z).scatter(1, r.experts.long(), 1.0)

    def f(zz):                                              # the choices held fixed
        w = torch.softmax(zz.gather(1, r.experts.long()), -1)
        return (fe.expert_combine(y, fe.ExpertRoute(r.experts, w, r.slots, r.offsets)).double() * go.double()).sum().item()

    with torch.no_grad():
        v = torch.randn_like(z) * picked
        slope = (g * v.double()).sum().item()
        scale = (g.norm() * v.double().norm()).item() / 90 ** 0.5
        assert abs((f(z + 1e-2 * v) - f(z - 1e-2 * v)) / 2e-2 - slope) < 2e-3 * max(scale, abs(slope))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_repeatable_and_on_another_stream(cuda_device, dtype):
    x, w, b, offsets, go = _linear_inputs([900, 33, 1700], 5, (0,), 128, 192, dtype, cuda_device)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = fe.expert_linear(*leaves, offsets)
        return [y.detach(), *torch.autograd.grad(y, leaves, go)]

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (1, 2)])
def test_expert_linear_some_gradients_only(cuda_device, which, dtype):
    x, w, b, offsets, go = _linear_inputs([30, 0, 77], 2, (0, 1), 40, 48, dtype, cuda_device, seed=11)
    want = _linear_reference(x, w, b, offsets, (0, 1), go)[1:]
    leaves = [t.requires_grad_(i in which) for i, t in enumerate((x, w, b))]
    got = torch.autograd.grad(fe.expert_linear(*leaves, offsets, (0, 1)), [leaves[i] for i in which], go)
    for g, i in zip(got, which):
        assert rel_l2(g, want[i]) < TOL[dtype]


def test_gradients_are_differentiable_once(cuda_device):
    x, w, b, offsets, go = _linear_inputs([3, 4], 0, (0,), 8, 16, torch.float32, cuda_device)
    g = torch.autograd.grad(fe.expert_linear(x.requires_grad_(), w, b, offsets), x, go, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    z = torch.randn(6, 4, device=cuda_device, requires_grad=True)
    r = fe.expert_route(z, 2)
    g = torch.autograd.grad(r.weights[:, 0].sum(), z, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    assert torch.autograd.grad(fe.expert_dispatch(torch.randn(6, 3, device=cuda_device, requires_grad=True), r).sum(),
                               z, allow_unused=True) == (None,)


@pytest.mark.parametrize("dtype,sizes,ci,co", [
    (torch.bfloat16, [5000, 3000, 1, 4000], 512, 1024),     # tiles on pairs of CTAs
    (torch.float16, [300, 77, 0, 500], 256, 320),           # tiles on one CTA
    (torch.float32, [2000, 77, 0, 3000], 192, 256)], ids=["pairs", "single", "planes"])
def test_expert_linear_short_wait_limit(cuda_device, dtype, sizes, ci, co):
    """A wait past its limit ends the kernel with status 2, copies and products drained, and the next call is
    right again.  (On single CTAs the waits are shorter than the polls before the first look at the timer.)"""
    x, w, b, offsets, go = _linear_inputs(sizes, 3, (0,), ci, co, dtype, cuda_device)
    want = _linear_reference(x, w, b, offsets, (0,), go)
    lib = _lib.load()

    def both(status):
        y = token_ops.expert_linear_fwd(x, w, b, offsets, (0,), status=status)
        return [y, *token_ops.expert_linear_bwd(go, x, w, offsets, (0,), status=status)]

    for short in (True, False):
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        old = lib.feq_set_wait_limit_ns(1 if short else 0)
        try:
            got = both(status)
            torch.cuda.synchronize()
        finally:
            lib.feq_set_wait_limit_ns(old)
        if short and dtype != torch.float16:
            assert int(status) == 2, "a 1 ns wait limit should have timed out at least one wait"
        assert int(status) in ((0, 2) if short else (0,))
        if int(status) == 0:
            for g, r in zip(got, want):
                assert rel_l2(g, r) < TOL[dtype]


def test_expert_linear_empty(cuda_device):
    x, w, b, offsets, go = _linear_inputs([0, 0], 0, (0,), 16, 24, torch.float32, cuda_device)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = fe.expert_linear(*leaves, offsets)
    grads = torch.autograd.grad(y, leaves, go)
    assert y.shape == (0, 1, 24)
    assert torch.equal(grads[1], torch.zeros_like(w)) and torch.equal(grads[2], torch.zeros_like(b))


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------
def _experts_reference(m, x, mask, plan):
    """The layer in float64 on the CPU, with the plan's choices."""
    d = copy.deepcopy(m).double().cpu()
    x = x.double().cpu()
    lv, at = list(d.lvals), []
    for i, l in enumerate(lv):
        at += [i] * (2 * l + 1)
    sq = torch.stack([(x[..., [j for j, a in enumerate(at) if a == i]] ** 2).sum(-1) for i in range(len(lv))], -1)
    inv = (sq + 1e-8).sqrt().flatten(-2)
    logits = torch.nn.functional.layer_norm(inv, inv.shape[-1:], d.router_norm.weight, d.router_norm.bias, 1e-5) @ d.router.weight.t()
    out = torch.zeros_like(x)
    ids = plan.experts.cpu().long()
    for n in range(x.shape[0]):
        live = [int(e) for e in ids[n] if e >= 0]
        if not live:
            continue
        w = torch.softmax(logits[n, live], 0)
        for wj, e in zip(w, live):
            h = torch.stack([d.weight_up[e, i] @ x[n, :, p] for p, i in enumerate(at)], -1)
            scalars = [p for p, i in enumerate(at) if lv[i] == 0]
            h = torch.stack([h[:, p] + d.bias_up[e, scalars.index(p)] if p in scalars else h[:, p] for p in range(len(at))], -1)
            h = h * torch.sigmoid(h[:, d._gate_at:d._gate_at + 1])
            y = torch.stack([d.weight_down[e, i] @ h[:, p] for p, i in enumerate(at)], -1)
            y = torch.stack([y[:, p] + d.bias_down[e, scalars.index(p)] if p in scalars else y[:, p] for p in range(len(at))], -1)
            out[n] = out[n] + wj * y
    return out, d


@pytest.mark.parametrize("lvals,mult", [((0, 1, 2), 8), ((0,), 20), ((1, 0, 0), 5)])
def test_equivariant_experts_layer(cuda_device, lvals, mult):
    torch.manual_seed(0)
    m = fe.EquivariantExperts(fe.Repr(list(lvals), mult), num_experts=5, top_k=2).to(cuda_device)
    with torch.no_grad():
        for p in (m.bias_up, m.bias_down):
            p.normal_()
    x = torch.randn(40, mult, m.repr.dim(), device=cuda_device).requires_grad_()
    mask = torch.rand(40, device=cuda_device) > 0.2
    y = m(x, mask)
    ref, d = _experts_reference(m, x.detach(), mask, m.route(x.detach(), mask))
    assert rel_l2(y.detach(), ref.detach()) < 1e-5
    assert torch.equal(y[~mask], torch.zeros_like(y[~mask]))
    go = torch.randn_like(y)
    y.backward(go)
    ref.backward(go.double().cpu())
    for (name, p), q in zip(m.named_parameters(), d.parameters()):
        assert rel_l2(p.grad, q.grad) < 2e-5, name
    with torch.no_grad():
        assert rel_l2(m(x, mask), y) < 1e-5                  # the inference path (native norms)


def test_transformer_with_experts_trains(cuda_device):
    torch.manual_seed(1)
    r = fe.Repr([0, 1], 16)
    model = fe.EquivariantTransformer(r, r, r, num_layers=2, num_heads=4, num_experts=4, layer_scale_init=0.5).to(cuda_device)
    n = 60
    xyz, f = torch.randn(n, 3, device=cuda_device) * 2, torch.randn(n, 16, 4, device=cuda_device)
    graph = fe.Graph.random(n, 500, device=cuda_device)
    y = model(xyz, f, graph)
    y.square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert model.layers[0].experts.weight_up.grad.abs().sum() > 0
    with pytest.raises(ValueError):
        fe.EquivariantTransformerBlock(r, r, num_experts=4, use_gating=False)


def test_layer_commutes_with_rotations(cuda_device):
    torch.manual_seed(2)
    r = fe.Repr([0, 1], 12)
    m = fe.EquivariantExperts(r, num_experts=6, top_k=2).to(cuda_device)
    q, _ = torch.linalg.qr(torch.randn(3, 3, dtype=torch.float64))
    q = q * torch.sign(torch.linalg.det(q))
    rot = torch.eye(4, dtype=torch.float64)
    rot[1:, 1:] = q                                          # any orthogonal map of an irrep's components
    rot = rot.to(cuda_device, torch.float32)
    x = torch.randn(80, 12, 4, device=cuda_device)
    with torch.no_grad():
        check_equivariance(m(x @ rot), m(x) @ rot, rtol=1e-4)


def test_layer_replays_in_a_graph(cuda_device):
    """No step synchronises the host: the inference pass is captured and replayed on new inputs."""
    m = fe.EquivariantExperts(fe.Repr([0, 1], 16), num_experts=4).to(cuda_device).eval()
    x = torch.randn(64, 16, 4, device=cuda_device)
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            m(x)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        new = torch.randn_like(x)
        x.copy_(new)
        graph.replay()
        assert torch.equal(y, m(new))


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(cuda_device):
    z = torch.randn(6, 4, device=cuda_device)
    for k in (0, 5, -1):
        with pytest.raises(ValueError):
            fe.expert_route(z, k)
    with pytest.raises(TypeError):
        fe.expert_route(z.double(), 2)
    with pytest.raises(ValueError):
        fe.expert_route(z[0], 2)
    with pytest.raises(ValueError):
        fe.expert_route(torch.randn(2, 513, device=cuda_device), 2)
    r = fe.expert_route(z, 2)
    for bad in (torch.randn(5, 8, device=cuda_device), torch.randn(6, 0, device=cuda_device)):
        with pytest.raises(ValueError):
            fe.expert_dispatch(bad, r)
    with pytest.raises(ValueError):
        fe.expert_combine(torch.randn(11, 8, device=cuda_device), r)
    with pytest.raises(ValueError):
        fe.expert_combine(torch.randn(12, device=cuda_device), r)
    with pytest.raises(RuntimeError):
        fe.expert_dispatch(torch.randn(6, 8), r)
    with pytest.raises(TypeError):
        token_ops.expert_dispatch(torch.randn(6, 8, device=cuda_device), r.slots.long(), r.offsets)
    x, w, b, offsets, _ = _linear_inputs([3, 3], 0, (0, 1), 8, 16, torch.float32, cuda_device)
    ok = dict(x=x, weight=w, bias=b, offsets=offsets, lvals=(0, 1))
    fe.expert_linear(**ok)
    for change in (dict(lvals=(0,)), dict(lvals=()), dict(lvals=(0, -1)), dict(weight=w[..., :7]), dict(weight=w[:1]),
                   dict(bias=b[..., :7]), dict(offsets=offsets[:2]), dict(offsets=offsets.float()), dict(x=x[:, 0])):
        with pytest.raises(ValueError):
            fe.expert_linear(**{**ok, **change})
    for change in (dict(weight=w.half()), dict(bias=b.half()), dict(x=x.double(), weight=w.double(), bias=b.double())):
        with pytest.raises(TypeError):
            fe.expert_linear(**{**ok, **change})
    with pytest.raises(RuntimeError):
        fe.expert_linear(**{**ok, "offsets": offsets.cpu()})
    with pytest.raises(ValueError):
        fe.EquivariantExperts(fe.Repr([1, 2], 8), 4)
    with pytest.raises(ValueError):
        fe.EquivariantExperts(fe.Repr([0, 1], 8), 4, top_k=5)
    with pytest.raises(ValueError):
        fe.EquivariantExperts(fe.Repr([0, 1], 8), 4).to(cuda_device)(torch.randn(3, 8, 3, device=cuda_device))
