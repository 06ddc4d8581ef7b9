"""Torch-facing wrappers of the layer norm and mixture-of-experts kernels (csrc/feq_layernorm.cu,
csrc/feq_experts.cu, csrc/feq_expertlin.cu).

As in ``ops``: inputs are checked, outputs and workspace come from torch's caching allocator and the
kernels are enqueued on the current stream of the inputs' device; no host synchronisation.
Element types: float32, bfloat16, float16.  The last dimension is read contiguous, rows may
be strided; anything else is copied first.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .ops import _require_cuda

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_EXPERTS, MAX_TOP_K = 512, 32

# These wrappers run in front of kernels of a few microseconds, so they pass plain integers to ctypes and
# ask torch for a stream handle without building a Stream object.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # absent in builds without CUDA
_current_device = torch.cuda.current_device
_empty, _f32, _i32 = torch.empty, torch.float32, torch.int32
_load = _lib.load


def _ready(first: torch.Tensor, *others):
    """The library, after checking that every tensor lies on one CUDA device."""
    dev = first.get_device()
    good = dev >= 0
    for t in others:
        if t is not None and t.get_device() != dev:
            good = False
    if not good:
        _require_cuda(first, *others)
        raise RuntimeError("flash-eq ops need all tensors on one device; got "
                           + ", ".join(str(t.device) for t in (first, *others) if t is not None))
    return _load()


def _call(fn, what: str, dev: int, *args) -> None:
    """fn(*args, stream) with ``dev`` current, on its current stream."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _lib.check(rc, what)


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _dtype(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16; got {t.dtype}")
    return code


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, width) with a contiguous last dimension."""
    return t if t.stride(1) == 1 else t.contiguous()


def _param(p, like: torch.Tensor, width: int, name: str):
    if p is None:
        return None
    if p.shape != (width,):
        raise ValueError(f"{name} must have shape ({width},); got {tuple(p.shape)}")
    if p.dtype is not like.dtype and p.dtype is not torch.float32:
        raise TypeError(f"{name} must be {like.dtype} or float32; got {p.dtype}")
    return p.contiguous()


def _workspace(nbytes: int, device):
    return _empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def layer_norm_fwd(x: torch.Tensor, weight, bias, eps: float, keep_stats: bool):
    """(y, stats) of x (..., D); stats (2, rows) = mean and 1 / std, None unless ``keep_stats``."""
    lib = _ready(x, weight, bias)
    code = _dtype(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError(f"x must have a last dimension of at least 1; got {tuple(x.shape)}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0; got {eps}")
    weight, bias = _param(weight, x, width, "weight"), _param(bias, x, width, "bias")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise TypeError(f"weight and bias must have one type; got {weight.dtype} and {bias.dtype}")
    rows = _rows(x if x.dim() == 2 else x.reshape(-1, width))
    n, dev = rows.shape[0], x.device
    y = _empty(x.shape, dtype=x.dtype, device=dev)
    stats = mean = rstd = None
    if keep_stats:
        stats = _empty(2, n, dtype=_f32, device=dev)
        mean = stats.data_ptr()
        rstd = mean + 4 * n
    p = bias if weight is None else weight
    _call(lib.feq_layer_norm_fwd, "feq_layer_norm_fwd", dev.index, rows.data_ptr(), n, rows.stride(0), width, code,
          None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
          p is not None and p.dtype is _f32, eps, y.data_ptr(), mean, rstd)
    return y, stats


def layer_norm_bwd(grad_out, x, weight, stats, need_x=True, need_weight=True, need_bias=True, param_dtype=None):
    """(grad_x, grad_weight, grad_bias) of ``layer_norm_fwd``; None where not needed."""
    lib = _ready(grad_out, x, weight)
    code, width = _dtype(x, "x"), x.shape[-1]
    weight = _param(weight, x, width, "weight")
    rows, g = _rows(x.reshape(-1, width)), _rows(grad_out.reshape(-1, width))
    n, dev = rows.shape[0], x.device
    pd = param_dtype or (weight.dtype if weight is not None else x.dtype)
    gx = _empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = _empty(width, dtype=pd, device=dev) if need_weight else None
    gb = _empty(width, dtype=pd, device=dev) if need_bias else None
    mean = stats.data_ptr()
    nbytes = lib.feq_layer_norm_bwd_workspace_bytes(n, width) if need_weight or need_bias else 0
    ws = _workspace(nbytes, dev)
    _call(lib.feq_layer_norm_bwd, "feq_layer_norm_bwd", dev.index, g.data_ptr(), g.stride(0), rows.data_ptr(), n,
          rows.stride(0), width, code, _ptr(weight), pd is _f32, mean, mean + 4 * n, _ptr(gx), _ptr(gw),
          _ptr(gb), _ptr(ws), nbytes)
    return gx, gw, gb


# ---------------------------------------------------------------------------
# expert routing
# ---------------------------------------------------------------------------
def expert_route(logits: torch.Tensor, top_k: int, normalize: bool = True):
    """(experts, weights, slots, offsets) of logits (tokens, num_experts)."""
    lib = _ready(logits)
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
    ids = _empty(n, k, dtype=_i32, device=dev)
    slots = torch.empty_like(ids)
    weights = _empty(n, k, dtype=_f32, device=dev)
    offsets = _empty(e + 1, dtype=_i32, device=dev)
    nbytes = lib.feq_expert_route_workspace_bytes(n, k, e)
    ws = _workspace(nbytes, dev)
    _call(lib.feq_expert_route, "feq_expert_route", dev.index, rows.data_ptr(), n, rows.stride(0), e, k, code,
          bool(normalize), ids.data_ptr(), weights.data_ptr(), slots.data_ptr(), offsets.data_ptr(), _ptr(ws),
          nbytes)
    return ids, weights, slots, offsets


def expert_route_bwd(logits, ids, weights, grad_weights, normalize):
    lib = _ready(logits, grad_weights)
    n, e = logits.shape
    rows, dev = _rows(logits), logits.device
    grad_weights = grad_weights.to(torch.float32).contiguous()
    out = _empty(n, e, dtype=logits.dtype, device=dev)
    _call(lib.feq_expert_route_bwd, "feq_expert_route_bwd", dev.index, rows.data_ptr(), n, rows.stride(0), e,
          ids.shape[1], _dtype(logits, "logits"), bool(normalize), ids.data_ptr(), weights.data_ptr(),
          grad_weights.data_ptr(), out.data_ptr())
    return out


def _plan(slots: torch.Tensor, offsets: torch.Tensor):
    if slots.dtype is not torch.int32 or slots.dim() != 2 or not slots.is_contiguous():
        raise TypeError("slots must be a contiguous int32 (tokens, top_k) tensor")
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2 or not offsets.is_contiguous():
        raise TypeError("offsets must be a contiguous int32 (num_experts + 1,) tensor")
    return (*slots.shape, offsets.shape[0] - 1)


def expert_dispatch(x: torch.Tensor, slots, offsets) -> torch.Tensor:
    """x (tokens, width) -> (tokens * top_k, width) sorted by expert."""
    lib = _ready(x, slots, offsets)
    n, k, e = _plan(slots, offsets)
    if x.dim() != 2 or x.shape[0] != n or x.shape[1] < 1:
        raise ValueError(f"x must be ({n}, width); got {tuple(x.shape)}")
    code, rows, width = _dtype(x, "x"), _rows(x), x.shape[1]
    out = _empty(n * k, width, dtype=x.dtype, device=x.device)
    _call(lib.feq_expert_dispatch, "feq_expert_dispatch", x.device.index, rows.data_ptr(), n, rows.stride(0), width,
          code, k, e, slots.data_ptr(), offsets.data_ptr(), out.data_ptr())
    return out


def _sorted_rows(y, n, k):
    if y.dim() != 2 or y.shape[0] != n * k or y.shape[1] < 1:
        raise ValueError(f"y must be ({n * k}, width); got {tuple(y.shape)}")
    return _rows(y)


def expert_combine(y: torch.Tensor, slots, offsets, weights=None) -> torch.Tensor:
    """Sorted rows (tokens * top_k, width) -> (tokens, width), weighted by ``weights`` (tokens, top_k)."""
    lib = _ready(y, slots, offsets, weights)
    n, k, e = _plan(slots, offsets)
    code, rows, width = _dtype(y, "y"), _sorted_rows(y, n, k), y.shape[1]
    if weights is not None:
        if weights.shape != slots.shape or weights.dtype is not torch.float32:
            raise ValueError(f"weights must be a float32 ({n}, {k}) tensor; got {weights.dtype} {tuple(weights.shape)}")
        weights = weights.contiguous()
    out = _empty(n, width, dtype=y.dtype, device=y.device)
    _call(lib.feq_expert_combine, "feq_expert_combine", y.device.index, rows.data_ptr(), rows.stride(0), n, width,
          code, k, e, slots.data_ptr(), offsets.data_ptr(), _ptr(weights), out.data_ptr())
    return out


def expert_combine_bwd(grad_out, y, slots, offsets, weights):
    """(grad_y, grad_weights) of ``expert_combine`` with weights."""
    lib = _ready(grad_out, y, slots, offsets, weights)
    n, k, e = _plan(slots, offsets)
    code, rows, g, width = _dtype(y, "y"), _sorted_rows(y, n, k), _rows(grad_out), y.shape[1]
    gy = _empty(n * k, width, dtype=y.dtype, device=y.device)
    gw = _empty(n, k, dtype=_f32, device=y.device)
    weights = weights.contiguous()
    _call(lib.feq_expert_combine_bwd, "feq_expert_combine_bwd", y.device.index, g.data_ptr(), g.stride(0),
          rows.data_ptr(), rows.stride(0), n, width, code, k, e, slots.data_ptr(), offsets.data_ptr(),
          weights.data_ptr(), gy.data_ptr(), gw.data_ptr())
    return gy, gw


# ---------------------------------------------------------------------------
# expert linear
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=64)
def _degrees(lvals):
    """(dim, number of l = 0 irreps, ctypes array) of a tuple of degrees."""
    if not lvals or any(v < 0 for v in lvals):
        raise ValueError(f"lvals must be a non-empty list of degrees >= 0; got {list(lvals)}")
    return sum(2 * v + 1 for v in lvals), sum(v == 0 for v in lvals), _lib.i32_array(lvals)[0]


def _strided(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _linear_args(x, weight, offsets, lvals):
    """Shapes of ``expert_linear``, and the arguments that both directions share.

    x (rows, dim, c_in) with weight (E, reps, c_out, c_in), or plain x (rows, c_in) with (E, c_out, c_in)."""
    code = _dtype(x, "x")
    dim, scalars, arr = _degrees(lvals)
    plain = x.dim() == 2
    if plain:
        if lvals != (0,):
            raise ValueError(f"plain rows (rows, c_in) need lvals (0,); got {list(lvals)}")
    elif x.dim() != 3 or x.shape[1] != dim:
        raise ValueError(f"x must be (rows, {dim}, c_in) for lvals {list(lvals)}; got {tuple(x.shape)}")
    ci = x.shape[-1]
    shape = weight.shape
    if len(shape) != (3 if plain else 4) or shape[-1] != ci or ci < 1 or shape[-2] < 1 or shape[0] < 1 or not (
            plain or shape[1] == len(lvals)):
        want = "(num_experts, c_out, " if plain else f"(num_experts, {len(lvals)}, c_out, "
        raise ValueError(f"weight must be {want}{ci}); got {tuple(shape)}")
    e, co = shape[0], shape[-2]
    if e > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts; got {e}")
    if weight.dtype is not x.dtype:
        raise TypeError(f"weight must have x's type {x.dtype}; got {weight.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] != e + 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"offsets must be an int32 or int64 ({e + 1},) tensor; got {offsets.dtype} {tuple(offsets.shape)}")
    # kept alive by the caller until the call has returned
    x, weight = _strided(x), weight.contiguous()
    offsets = (offsets if offsets.dtype is torch.int32 else offsets.to(torch.int32)).contiguous()
    a = _lib.FeqExpertLinearArgs(x.data_ptr(), x.stride(0), 0 if plain else x.stride(1), weight.data_ptr(), None,
                                 offsets.data_ptr(), x.shape[0], arr, len(lvals), e, ci, co, code)
    return a, (x, weight, offsets), scalars


def _run_linear(lib, fn, what, a, backward, device, status):
    if status is not None:
        a.status = status.data_ptr()
    ref, dev = ctypes.byref(a), device.index
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _run_linear(lib, fn, what, a, backward, device, None)
    rc = fn(ref, None, 0, _raw_stream(dev))
    if rc == _lib.FEQ_ERR_WORKSPACE:          # an operand has to be packed, or sums joined
        nbytes = lib.feq_expert_linear_workspace_bytes(ref, backward)
        ws = _workspace(nbytes, device)
        rc = fn(ref, ws.data_ptr(), nbytes, _raw_stream(dev))
    if rc:
        _lib.check(rc, what)


def expert_linear_fwd(x, weight, bias, offsets, lvals, status=None) -> torch.Tensor:
    lib = _ready(x, weight, bias, offsets)
    a, kept, scalars = _linear_args(x, weight, offsets, lvals)
    plain = x.dim() == 2
    if bias is not None:
        if scalars == 0:
            raise ValueError(f"a bias needs an l = 0 component; lvals are {list(lvals)}")
        want = (a.num_experts, a.c_out) if plain else (a.num_experts, scalars, a.c_out)
        if bias.shape != want:
            raise ValueError(f"bias must be {want}; got {tuple(bias.shape)}")
        if bias.dtype is not x.dtype:
            raise TypeError(f"bias must have x's type {x.dtype}; got {bias.dtype}")
        bias = bias.contiguous()
        a.bias = bias.data_ptr()
    out = _empty((x.shape[0], a.c_out) if plain else (x.shape[0], x.shape[1], a.c_out), dtype=x.dtype,
                      device=x.device)
    a.out = out.data_ptr()
    _run_linear(lib, lib.feq_expert_linear_fwd, "feq_expert_linear_fwd", a, 0, x.device, status)
    return out


def expert_linear_bwd(grad_out, x, weight, offsets, lvals, need_x=True, need_weight=True, need_bias=True, status=None):
    """(grad_x, grad_weight, grad_bias) of ``expert_linear_fwd``; None where not needed."""
    lib = _ready(grad_out, x, weight, offsets)
    a, kept, scalars = _linear_args(x, weight, offsets, lvals)
    g, dev, plain = _strided(grad_out), x.device, x.dim() == 2
    gx = _empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = _empty(weight.shape, dtype=x.dtype, device=dev) if need_weight else None
    gb = None
    if need_bias:
        gb = _empty((a.num_experts, a.c_out) if plain else (a.num_experts, scalars, a.c_out), dtype=x.dtype,
                         device=dev)
    a.grad_out, a.grad_row_stride, a.grad_comp_stride = g.data_ptr(), g.stride(0), 0 if plain else g.stride(1)
    a.grad_x, a.grad_weight, a.grad_bias = _ptr(gx), _ptr(gw), _ptr(gb)
    _run_linear(lib, lib.feq_expert_linear_bwd, "feq_expert_linear_bwd", a, 1, dev, status)
    return gx, gw, gb
