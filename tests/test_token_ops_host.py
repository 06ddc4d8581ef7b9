"""Host checks of the layer norm and expert entry points (no kernel is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import flash_eq as fe
from flash_eq.cuda import _lib


def test_argument_checks_without_gpu():
    """The C entry points return codes for what they can refuse on the host; they never abort."""
    lib = _lib.load()
    ok, invalid, unsupported, workspace = 0, 1, 2, 3
    fake = ctypes.c_void_p(256)           # never dereferenced: every call below ends before a launch
    ln = lib.feq_layer_norm_fwd
    assert ln(None, 0, 4, 4, 0, None, None, 0, 1e-5, None, None, None, None) == ok           # no rows
    assert ln(None, 3, 4, 4, 0, None, None, 0, 1e-5, None, None, None, None) == invalid      # no tensors
    assert ln(fake, 3, 4, 0, 0, None, None, 0, 1e-5, fake, None, None, None) == invalid      # no width
    assert ln(fake, 3, 4, 4, 9, None, None, 0, 1e-5, fake, None, None, None) == invalid      # no such type
    assert ln(fake, 3, 4, 4, 0, None, None, 0, -1.0, fake, None, None, None) == invalid
    assert ln(fake, 3, 4, (1 << 29) + 1, 0, None, None, 0, 1e-5, fake, None, None, None) == unsupported
    assert lib.feq_layer_norm_bwd(fake, 4, fake, 3, 4, 4, 0, None, 0, fake, fake, fake, fake, None, None, 0,
                                  None) == workspace
    assert lib.feq_layer_norm_bwd_workspace_bytes(0, 8) == 0
    route = lambda n, e, k: lib.feq_expert_route(fake, n, e, e, k, 0, 1, fake, fake, fake, fake, None, 0, None)
    assert route(4, 8, 9) == invalid and route(4, 8, 0) == invalid and route(-1, 8, 2) == invalid
    assert route(4, 513, 2) == unsupported and route(1 << 30, 8, 2) == unsupported
    assert route(100000, 8, 2) == workspace
    rows = lambda n, w: lib.feq_expert_dispatch(fake, n, w, w, 0, 2, 8, fake, fake, None, None)
    assert rows(0, 8) == ok and rows(3, 0) == invalid and rows(3, 8) == invalid
    args = _lib.FeqExpertLinearArgs()
    lv, n = _lib.i32_array([0, 1])
    args.lvals, args.n_lvals = ctypes.cast(lv, _lib.c_i32p), n
    args.num_experts, args.c_in, args.c_out, args.rows = 4, 8, 8, 0
    assert lib.feq_expert_linear_fwd(ctypes.byref(args), None, 0, None) == ok
    assert lib.feq_expert_linear_workspace_bytes(ctypes.byref(args), 0) > 0
    args.rows = 5
    assert lib.feq_expert_linear_fwd(ctypes.byref(args), None, 0, None) == invalid           # no tensors
    args.rows = 1 << 31
    assert lib.feq_expert_linear_fwd(ctypes.byref(args), None, 0, None) == unsupported
    args.rows, args.num_experts = 5, 513
    assert lib.feq_expert_linear_workspace_bytes(ctypes.byref(args), 0) == 0
    args.num_experts, lv[1] = 4, 17
    assert lib.feq_expert_linear_fwd(ctypes.byref(args), None, 0, None) == unsupported
    lv[1] = -1
    assert lib.feq_expert_linear_bwd(ctypes.byref(args), None, 0, None) == invalid
    assert lib.feq_expert_linear_fwd(None, None, 0, None) == invalid


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_no_gpu_fails_loudly():
    for call in (lambda: fe.layer_norm(torch.randn(3, 4)), lambda: fe.expert_route(torch.randn(3, 4), 2),
                 lambda: fe.expert_linear(torch.randn(3, 4), torch.randn(2, 5, 4), None, torch.tensor([0, 1, 3]))):
        with pytest.raises(fe.CUDANotAvailableError):
            call()


def test_native_module_reports_errors():
    """Its C++ exceptions arrive as Python ones."""
    from flash_eq.cuda import token_ops

    m = token_ops.load()
    assert m.abi_version() == _lib.FEQ_ABI_VERSION
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        m.expert_route(torch.randn(3, 4), 2, True)
    with pytest.raises(ValueError, match="degrees"):
        m.check_degrees([0, -1])
    with pytest.raises(TypeError):
        m.check_degrees("x")


def test_layer_bookkeeping():
    m = fe.EquivariantExperts(fe.Repr([0, 1, 2], 8), num_experts=3, top_k=2, mlp_ratio=2)
    assert m.weight_up.shape == (3, 3, 16, 8) and m.weight_down.shape == (3, 3, 8, 16)
    assert m.bias_up.shape == (3, 1, 16) and m.router.weight.shape == (3, 24)
    plain = fe.EquivariantTransformerBlock(fe.Repr([0, 1], 8), fe.Repr([0, 1], 8))
    assert not any("experts" in k for k in plain.state_dict())
    mixed = fe.EquivariantTransformerBlock(fe.Repr([0, 1], 8), fe.Repr([0, 1], 8), num_experts=2, expert_top_k=1)
    assert not any(k.startswith("mlp") for k in mixed.state_dict())
    assert fe.InvariantLayerNorm(6)(torch.randn(2, 6)).shape == (2, 6)
