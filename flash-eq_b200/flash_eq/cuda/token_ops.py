"""Torch-facing wrappers of the layer norm and mixture-of-experts kernels (csrc/feq_layernorm.cu,
csrc/feq_experts.cu, csrc/feq_expertlin.cu).

Like ``ops``: inputs are checked, outputs and workspace come from torch's caching allocator and the
kernels are enqueued on the current stream of the inputs' device; no host synchronisation.
Element types: float32, bfloat16, float16.  The last dimension is read contiguous, rows may
be strided; anything else is copied first.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .ops import _p, _require_cuda, _stream, _workspace

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_EXPERTS, MAX_TOP_K = 512, 32


def _dtype(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16; got {t.dtype}")
    return code


def _same_device(first: torch.Tensor, *others) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"flash-eq ops need all tensors on one device; got {first.device} and {t.device}")


def _on(device):
    """Context that makes ``device`` current for the launches (a no-op when it already is)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, width) with a contiguous last dimension."""
    t = t.detach()
    return t if t.stride(1) == 1 else t.contiguous()


def _param(p, like: torch.Tensor, width: int, name: str):
    if p is None:
        return None
    if p.shape != (width,):
        raise ValueError(f"{name} must have shape ({width},); got {tuple(p.shape)}")
    if p.dtype not in (like.dtype, torch.float32):
        raise TypeError(f"{name} must be {like.dtype} or float32; got {p.dtype}")
    return p.detach().contiguous()


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def layer_norm_fwd(x: torch.Tensor, weight, bias, eps: float, keep_stats: bool):
    """(y, mean, rstd) of x (..., D); mean / rstd None unless ``keep_stats``."""
    lib = _require_cuda(x, weight, bias)
    _same_device(x, weight, bias)
    code = _dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last dimension of at least 1; got {tuple(x.shape)}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0; got {eps}")
    width = x.shape[-1]
    weight, bias = _param(weight, x, width, "weight"), _param(bias, x, width, "bias")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type; got {weight.dtype} and {bias.dtype}")
    rows = _rows(x.reshape(-1, width))
    n = rows.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if keep_stats:
        mean, rstd = torch.empty(2, n, dtype=torch.float32, device=x.device)
    p = weight if weight is not None else bias
    with _on(x.device):
        rc = lib.feq_layer_norm_fwd(_p(rows), n, rows.stride(0), width, code, _p(weight), _p(bias),
                                    int(p is not None and p.dtype == torch.float32), eps, _p(y), _p(mean), _p(rstd),
                                    _stream(x.device))
    _lib.check(rc, "feq_layer_norm_fwd")
    return y, mean, rstd


def layer_norm_bwd(grad_out, x, weight, mean, rstd, need_x=True, need_weight=True, need_bias=True, param_dtype=None):
    """(grad_x, grad_weight, grad_bias) of ``layer_norm_fwd``; None where not needed."""
    lib = _require_cuda(grad_out, x, weight)
    code = _dtype(x, "x")
    width = x.shape[-1]
    weight = _param(weight, x, width, "weight")
    rows, g = _rows(x.reshape(-1, width)), _rows(grad_out.reshape(-1, width))
    n, dev = rows.shape[0], x.device
    pd = param_dtype or (weight.dtype if weight is not None else x.dtype)
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = torch.empty(width, dtype=pd, device=dev) if need_weight else None
    gb = torch.empty(width, dtype=pd, device=dev) if need_bias else None
    ws = _workspace(lib.feq_layer_norm_bwd_workspace_bytes(n, width), dev) if need_weight or need_bias else None
    with _on(dev):
        rc = lib.feq_layer_norm_bwd(_p(g), g.stride(0), _p(rows), n, rows.stride(0), width, code, _p(weight),
                                    int(pd == torch.float32), _p(mean), _p(rstd), _p(gx), _p(gw), _p(gb), _p(ws),
                                    0 if ws is None else ws.numel(), _stream(dev))
    _lib.check(rc, "feq_layer_norm_bwd")
    return gx, gw, gb


# ---------------------------------------------------------------------------
# expert routing
# ---------------------------------------------------------------------------
def expert_route(logits: torch.Tensor, top_k: int, normalize: bool = True):
    """(experts, weights, slots, offsets) of logits (tokens, num_experts)."""
    lib = _require_cuda(logits)
    code = _dtype(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be (tokens, num_experts); got {tuple(logits.shape)}")
    n, e = logits.shape
    k = int(top_k)
    if not 1 <= k <= e:
        raise ValueError(f"top_k must be in [1, num_experts = {e}]; got {top_k}")
    if e > MAX_EXPERTS or k > MAX_TOP_K:
        raise ValueError(f"at most {MAX_EXPERTS} experts and top_k {MAX_TOP_K}; got {e} and {k}")
    rows, dev = _rows(logits), logits.device
    ids, slots = torch.empty(2, n, k, dtype=torch.int32, device=dev)
    weights = torch.empty(n, k, dtype=torch.float32, device=dev)
    offsets = torch.empty(e + 1, dtype=torch.int32, device=dev)
    ws = _workspace(lib.feq_expert_route_workspace_bytes(n, k, e), dev)
    with _on(dev):
        rc = lib.feq_expert_route(_p(rows), n, rows.stride(0), e, k, code, int(bool(normalize)), _p(ids), _p(weights),
                                  _p(slots), _p(offsets), _p(ws), ws.numel(), _stream(dev))
    _lib.check(rc, "feq_expert_route")
    return ids, weights, slots, offsets


def expert_route_bwd(logits, ids, weights, grad_weights, normalize):
    lib = _require_cuda(logits, grad_weights)
    n, e = logits.shape
    rows, dev = _rows(logits), logits.device
    grad_weights = grad_weights.detach().to(torch.float32).contiguous()
    out = torch.empty(n, e, dtype=logits.dtype, device=dev)
    with _on(dev):
        rc = lib.feq_expert_route_bwd(_p(rows), n, rows.stride(0), e, ids.shape[1], _dtype(logits, "logits"),
                                      int(bool(normalize)), _p(ids), _p(weights), _p(grad_weights), _p(out),
                                      _stream(dev))
    _lib.check(rc, "feq_expert_route_bwd")
    return out


def _plan(slots: torch.Tensor, offsets: torch.Tensor):
    if slots.dtype != torch.int32 or slots.dim() != 2 or not slots.is_contiguous():
        raise TypeError("slots must be a contiguous int32 (tokens, top_k) tensor")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2 or not offsets.is_contiguous():
        raise TypeError("offsets must be a contiguous int32 (num_experts + 1,) tensor")
    return slots.shape[0], slots.shape[1], offsets.shape[0] - 1


def expert_dispatch(x: torch.Tensor, slots, offsets) -> torch.Tensor:
    """x (tokens, width) -> (tokens * top_k, width) sorted by expert."""
    lib = _require_cuda(x, slots, offsets)
    _same_device(x, slots, offsets)
    n, k, e = _plan(slots, offsets)
    if x.dim() != 2 or x.shape[0] != n or x.shape[1] < 1:
        raise ValueError(f"x must be ({n}, width); got {tuple(x.shape)}")
    code, rows = _dtype(x, "x"), _rows(x)
    out = torch.empty(n * k, x.shape[1], dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = lib.feq_expert_dispatch(_p(rows), n, rows.stride(0), x.shape[1], code, k, e, _p(slots), _p(offsets),
                                     _p(out), _stream(x.device))
    _lib.check(rc, "feq_expert_dispatch")
    return out


def _sorted_rows(y, n, k, name):
    if y.dim() != 2 or y.shape[0] != n * k or y.shape[1] < 1:
        raise ValueError(f"{name} must be ({n * k}, width); got {tuple(y.shape)}")
    return _rows(y)


def expert_combine(y: torch.Tensor, slots, offsets, weights=None) -> torch.Tensor:
    """Sorted rows (tokens * top_k, width) -> (tokens, width), weighted by ``weights`` (tokens, top_k)."""
    lib = _require_cuda(y, slots, offsets, weights)
    _same_device(y, slots, offsets, weights)
    n, k, e = _plan(slots, offsets)
    code, rows = _dtype(y, "y"), _sorted_rows(y, n, k, "y")
    if weights is not None:
        if weights.shape != (n, k) or weights.dtype != torch.float32:
            raise ValueError(f"weights must be a float32 ({n}, {k}) tensor; got {weights.dtype} {tuple(weights.shape)}")
        weights = weights.detach().contiguous()
    out = torch.empty(n, y.shape[1], dtype=y.dtype, device=y.device)
    with _on(y.device):
        rc = lib.feq_expert_combine(_p(rows), rows.stride(0), n, y.shape[1], code, k, e, _p(slots), _p(offsets),
                                    _p(weights), _p(out), _stream(y.device))
    _lib.check(rc, "feq_expert_combine")
    return out


def expert_combine_bwd(grad_out, y, slots, offsets, weights):
    """(grad_y, grad_weights) of ``expert_combine`` with weights."""
    lib = _require_cuda(grad_out, y, slots, offsets, weights)
    n, k, e = _plan(slots, offsets)
    code, rows, g = _dtype(y, "y"), _sorted_rows(y, n, k, "y"), _rows(grad_out)
    gy = torch.empty(n * k, y.shape[1], dtype=y.dtype, device=y.device)
    gw = torch.empty(n, k, dtype=torch.float32, device=y.device)
    weights = weights.detach().contiguous()
    with _on(y.device):
        rc = lib.feq_expert_combine_bwd(_p(g), g.stride(0), _p(rows), rows.stride(0), n, y.shape[1], code, k, e,
                                        _p(slots), _p(offsets), _p(weights), _p(gy), _p(gw), _stream(y.device))
    _lib.check(rc, "feq_expert_combine_bwd")
    return gy, gw


# ---------------------------------------------------------------------------
# expert linear
# ---------------------------------------------------------------------------
def _dim(lvals) -> int:
    return sum(2 * v + 1 for v in lvals)


def _strided(t: torch.Tensor) -> torch.Tensor:
    t = t.detach()
    return t if t.stride(2) == 1 else t.contiguous()


def check_expert_linear(x, weight, bias, offsets, lvals):
    """Shapes of ``expert_linear``: x (rows, dim, c_in), weight (E, reps, c_out, c_in), bias (E, scalars, c_out)."""
    _dtype(x, "x")
    if not lvals or any(v < 0 for v in lvals):
        raise ValueError(f"lvals must be a non-empty list of degrees >= 0; got {list(lvals)}")
    dim, scalars = _dim(lvals), sum(v == 0 for v in lvals)
    if x.dim() != 3 or x.shape[1] != dim or x.shape[2] < 1:
        raise ValueError(f"x must be (rows, {dim}, c_in) for lvals {list(lvals)}; got {tuple(x.shape)}")
    if weight.dim() != 4 or weight.shape[1] != len(lvals) or weight.shape[3] != x.shape[2] or weight.shape[2] < 1 \
            or weight.shape[0] < 1:
        raise ValueError(f"weight must be (num_experts, {len(lvals)}, c_out, {x.shape[2]}); got {tuple(weight.shape)}")
    e, co = weight.shape[0], weight.shape[2]
    if e > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts; got {e}")
    if weight.dtype != x.dtype:
        raise TypeError(f"weight must have x's type {x.dtype}; got {weight.dtype}")
    if bias is not None:
        if scalars == 0:
            raise ValueError(f"a bias needs an l = 0 component; lvals are {list(lvals)}")
        if bias.shape != (e, scalars, co):
            raise ValueError(f"bias must be ({e}, {scalars}, {co}); got {tuple(bias.shape)}")
        if bias.dtype != x.dtype:
            raise TypeError(f"bias must have x's type {x.dtype}; got {bias.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] != e + 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"offsets must be an int32 or int64 ({e + 1},) tensor; got {offsets.dtype} {tuple(offsets.shape)}")
    _same_device(x, weight, bias, offsets)


def _linear_args(x, weight, offsets, lvals, status):
    a = _lib.FeqExpertLinearArgs()
    arr, a.n_lvals = _lib.i32_array(lvals)
    a.lvals = ctypes.cast(arr, _lib.c_i32p)
    a.weight, a.offsets = weight.data_ptr(), offsets.data_ptr()
    a.num_experts, _, a.c_out, a.c_in = weight.shape
    a.dtype = DTYPES[weight.dtype]
    if x is not None:
        a.x, a.rows, a.x_row_stride, a.x_comp_stride = x.data_ptr(), x.shape[0], x.stride(0), x.stride(1)
    if status is not None:
        a.status = status.data_ptr()
    return a, arr


def _linear_workspace(lib, a, backward, device):
    nbytes = lib.feq_expert_linear_workspace_bytes(ctypes.byref(a), backward)
    if nbytes == 0:
        raise RuntimeError("expert_linear: unsupported shape (l <= 16, <= 64 irreps, dim <= 512, < 2^31 rows)")
    return _workspace(nbytes, device)


def expert_linear_fwd(x, weight, bias, offsets, lvals, status=None) -> torch.Tensor:
    lib = _require_cuda(x, weight, bias, offsets)
    check_expert_linear(x, weight, bias, offsets, lvals)
    x, weight = _strided(x), weight.detach().contiguous()
    bias = None if bias is None else bias.detach().contiguous()
    offsets = offsets.to(torch.int32).contiguous()
    out = torch.empty(x.shape[0], x.shape[1], weight.shape[2], dtype=x.dtype, device=x.device)
    a, keep = _linear_args(x, weight, offsets, lvals, status)
    a.out = out.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()
    with _on(x.device):
        ws = _linear_workspace(lib, a, 0, x.device)
        rc = lib.feq_expert_linear_fwd(ctypes.byref(a), _p(ws), ws.numel(), _stream(x.device))
    _lib.check(rc, "feq_expert_linear_fwd")
    return out


def expert_linear_bwd(grad_out, x, weight, offsets, lvals, need_x=True, need_weight=True, need_bias=True, status=None):
    """(grad_x, grad_weight, grad_bias) of ``expert_linear_fwd``; None where not needed."""
    lib = _require_cuda(grad_out, x, weight, offsets)
    x, weight, g = _strided(x), weight.detach().contiguous(), _strided(grad_out)
    offsets = offsets.to(torch.int32).contiguous()
    dev, (e, reps, co, ci) = x.device, weight.shape
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if need_weight else None
    gb = torch.empty(e, sum(v == 0 for v in lvals), co, dtype=x.dtype, device=dev) if need_bias else None
    a, keep = _linear_args(x, weight, offsets, lvals, status)
    a.grad_out, a.grad_row_stride, a.grad_comp_stride = g.data_ptr(), g.stride(0), g.stride(1)
    a.grad_x, a.grad_weight, a.grad_bias = (None if t is None else t.data_ptr() for t in (gx, gw, gb))
    with _on(dev):
        ws = _linear_workspace(lib, a, 1, dev)
        rc = lib.feq_expert_linear_bwd(ctypes.byref(a), _p(ws), ws.numel(), _stream(dev))
    _lib.check(rc, "feq_expert_linear_bwd")
    return gx, gw, gb
