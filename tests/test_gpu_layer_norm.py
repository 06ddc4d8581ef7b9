"""Layer norm (csrc/feq_layernorm.cu) against the formula in float64.

Tolerances, relative L2 over an output.  float32: every sum is a tree of at most a few dozen
sequential additions per level, each off by 2^-24 of a partial sum, and the centred values carry
the mean's rounding times |mean| / std (at most 30 in these inputs): 2e-6 bounds y and grad_x; the
parameters' gradients add up to 3000 rows, of which a thread adds at most some hundred in sequence:
1e-5.  16-bit types: one rounding of the result, at most 2^-9 (bfloat16) or 2^-12 (float16) of each
value, doubled.  grad_x is measured against the larger of itself and its terms r g w: at width 2 the
terms cancel down to eps / var of their size.
"""
from __future__ import annotations

import pytest
import torch

import flash_eq as fe
from conftest import rel_l2

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TOL_PARAM = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, width, dtype, device, seed=0, param_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * 2 + torch.randn(rows, 1, generator=g)
    w, b = 1 + 0.3 * torch.randn(width, generator=g), 0.3 * torch.randn(width, generator=g)
    go = torch.randn(rows, width, generator=g)
    pd = param_dtype or dtype
    return x.to(device, dtype), w.to(device, pd), b.to(device, pd), go.to(device, dtype)


def _reference(x, w, b, go, eps):
    x, go = x.double(), go.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    mean = x.mean(-1, keepdim=True)
    rstd = (x.var(-1, unbiased=False, keepdim=True) + eps) ** -0.5
    u = (x - mean) * rstd
    y = u * w + (0 if b is None else b.double())
    gw = go * w
    gx = rstd * (gw - gw.mean(-1, keepdim=True) - u * (gw * u).mean(-1, keepdim=True))
    dims = tuple(range(x.dim() - 1))
    return y, gx, (go * u).sum(dims), go.sum(dims)


def _check(x, w, b, go, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]       # views stay views
    it = iter(leaves)
    xx = next(it)
    ww = next(it) if w is not None else None
    bb = next(it) if b is not None else None
    y = fe.layer_norm(xx, ww, bb, eps)
    grads = torch.autograd.grad(y, leaves, go)
    ry, rgx, rgw, rgb = _reference(x, w, b, go, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    assert rel_l2(y.detach(), ry) < TOL[x.dtype]
    want = [rgx] + ([rgw] if w is not None else []) + ([rgb] if b is not None else [])
    for i, (g, r, leaf) in enumerate(zip(grads, want, leaves)):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if i == 0:
            terms = ((x.double().var(-1, unbiased=False, keepdim=True) + eps) ** -0.5 * go.double()
                     * (1 if w is None else w.double()))
            assert (g.double() - r).norm() < TOL[x.dtype] * torch.maximum(r.norm(), terms.norm())
        else:
            assert rel_l2(g, r) < TOL_PARAM[leaf.dtype], i
    with torch.no_grad():
        assert torch.equal(fe.layer_norm(x, w, b, eps), y)        # the inference path: the same values


SIZES = [(1, 2), (3, 7), (50, 64), (2, 255), (33, 256), (17, 257), (5, 511), (3000, 31), (1001, 128), (40, 1001),
         (9, 2048), (7, 4097), (3, 8192), (2, 8193), (65, 20000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width", SIZES, ids=[f"{r}x{w}" for r, w in SIZES])
def test_against_formula(cuda_device, rows, width, dtype):
    _check(*_inputs(rows, width, dtype, cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_float32_parameters(cuda_device, dtype):
    _check(*_inputs(40, 96, dtype, cuda_device, param_dtype=torch.float32))


@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
def test_missing_parameters(cuda_device, with_w, with_b):
    x, w, b, go = _inputs(37, 90, torch.float32, cuda_device)
    _check(x, w if with_w else None, b if with_b else None, go)


def test_many_rows_use_every_block(cuda_device):
    _check(*_inputs(200000, 40, torch.float32, cuda_device, seed=3))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_strided_and_misaligned_rows(cuda_device, dtype):
    base = _inputs(64, 200, dtype, cuda_device)[0]
    _, w, b, _ = _inputs(64, 96, dtype, cuda_device)
    go_wide = _inputs(64, 131, dtype, cuda_device, seed=2)[3]
    for x, go in ((base[:, 8:104], go_wide[:, :96]), (base[:, 3:99], go_wide[:, 5:101]), (base[::2, :96], go_wide[1::2, :96]),
                  (base.t()[:96, :96].t()[:50], go_wide[:50, 35:131])):
        _check(x, w, b, go)
    y = fe.layer_norm(base.view(4, 16, 200)[..., :96], w, b)          # more than two dimensions
    assert torch.equal(y.view(64, 96), fe.layer_norm(base[:, :96], w, b))
    x = base[:1, :96].expand(30, 96)                                   # one row seen thirty times
    _check(x, w, b, go_wide[:30, :96])


def test_expanded_gradient(cuda_device):
    x, w, b, _ = _inputs(30, 48, torch.float32, cuda_device)
    x.requires_grad_()
    g1 = torch.autograd.grad(fe.layer_norm(x, w, b).sum(), x)[0]
    ref = _reference(x.detach(), w, b, torch.ones(30, 48, device=cuda_device), 1e-5)[1]
    assert (g1.double() - ref).abs().max() < 1e-5          # the exact gradient nearly cancels


def test_constant_rows_width_one_and_extremes(cuda_device):
    """Rows without spread: (x - mean) is zero, so y = b and grad_x is finite; width 1 likewise."""
    w, b = torch.full((64,), 2.0, device=cuda_device), torch.full((64,), -1.0, device=cuda_device)
    x = torch.full((5, 64), 7.0, device=cuda_device, requires_grad=True)
    y = fe.layer_norm(x, w, b)
    assert torch.equal(y, b.expand(5, 64))
    assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()
    one = torch.randn(9, 1, device=cuda_device)
    assert torch.equal(fe.layer_norm(one), torch.zeros_like(one))
    big = torch.tensor([[1e18, -1e18, 1e18, -1e18]], device=cuda_device)      # squares reach 1e36, below the limit
    assert torch.allclose(fe.layer_norm(big), big.sign())
    # a large common offset: the centred sum of squares is exact, no cancellation
    x = 4096.0 + torch.arange(64.0, device=cuda_device).expand(3, 64)
    assert rel_l2(fe.layer_norm(x), _reference(x, None, None, x, 1e-5)[0]) < 2e-6
    # not-finite values stay in their own row
    x = torch.randn(6, 33, device=cuda_device)
    clean = fe.layer_norm(x)
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    y = fe.layer_norm(x)
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and y[2].isnan().all() and y[4].isnan().all()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_some_gradients_only(cuda_device, which):
    x, w, b, go = _inputs(33, 40, torch.float32, cuda_device, seed=9)
    want = _reference(x, w, b, go, 1e-5)[1:]
    leaves = [t.requires_grad_(i in which) for i, t in enumerate((x, w, b))]
    y = fe.layer_norm(*leaves)
    got = torch.autograd.grad(y, [leaves[i] for i in which], go)
    for g, i in zip(got, which):
        assert rel_l2(g, want[i]) < 1e-5
    if 2 in which:                                          # no weight: the bias moves up
        y = fe.layer_norm(x, None, b)
        assert rel_l2(torch.autograd.grad(y, b, go)[0], go.double().sum(0)) < 1e-5


def test_gradients_are_differentiable_once(cuda_device):
    x, w, b, go = _inputs(5, 12, torch.float32, cuda_device)
    x.requires_grad_()
    g = torch.autograd.grad(fe.layer_norm(x, w, b), x, go, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_empty(cuda_device):
    x = torch.empty(0, 16, device=cuda_device, requires_grad=True)
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    y = fe.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty(0, 16, device=cuda_device))
    assert y.shape == gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))


def test_gradient_against_differences(cuda_device):
    """Central differences of the kernel's own forward along random directions.  With step h = 1e-2 the
    truncation is O(h^2) of the third derivative (about 1e-4 of the slope here) and rounding 1e-7 / h = 1e-5:
    2e-3 leaves room for both."""
    x, w, b, go = _inputs(20, 37, torch.float32, cuda_device, seed=5)
    for t in (x, w, b):
        t.requires_grad_()
    grads = torch.autograd.grad(fe.layer_norm(x, w, b), [x, w, b], go)
    f = lambda *p: (fe.layer_norm(*p).double() * go.double()).sum().item()
    with torch.no_grad():
        for i, g in enumerate(grads):
            v = torch.randn_like(g)
            h, at = 1e-2, [x, w, b]
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + h * v, at[i] - h * v
            slope = (g.double() * v.double()).sum().item()
            scale = (g.double().norm() * v.double().norm()).item() / g.numel() ** 0.5
            assert abs((f(*up) - f(*down)) / (2 * h) - slope) < 2e-3 * max(scale, abs(slope))


def test_repeatable_and_on_another_stream(cuda_device):
    x, w, b, go = _inputs(5000, 72, torch.float32, cuda_device, seed=6)
    for t in (x, w, b):
        t.requires_grad_()
    first = torch.autograd.grad(fe.layer_norm(x, w, b), [x, w, b], go)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = torch.autograd.grad(fe.layer_norm(x, w, b), [x, w, b], go)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_module_and_refusals(cuda_device):
    m = fe.InvariantLayerNorm(24)
    x = torch.randn(11, 24)
    want = m(x)                                             # PyTorch on the CPU
    got = m.to(cuda_device)(x.to(cuda_device))
    assert rel_l2(got.detach(), want.detach()) < 2e-6
    assert set(m.state_dict()) == set(torch.nn.LayerNorm(24).state_dict())
    c = x.to(cuda_device)
    with pytest.raises(ValueError):
        m(c[:, :23])
    with pytest.raises(TypeError):
        fe.layer_norm(c.double())
    with pytest.raises(ValueError):
        fe.layer_norm(c, torch.ones(23, device=cuda_device))
    with pytest.raises(TypeError):
        fe.layer_norm(c, torch.ones(24, device=cuda_device, dtype=torch.float16))
    with pytest.raises(ValueError):
        fe.layer_norm(c, eps=-1.0)
    with pytest.raises(ValueError):
        fe.layer_norm(c, eps=float("nan"))
    with pytest.raises(ValueError):
        fe.layer_norm(c[:, :0])
    with pytest.raises(RuntimeError):
        fe.layer_norm(c, torch.ones(24))
