"""The state-space block without a GPU: refusals of the C entry points before any device work,
workspace sizes, the Python layer's own checks, and the modules' parameters."""

import ctypes

import pytest
import torch

from dudyconv_b200 import capi

F = ctypes.c_void_p(256)  # an address that is never reached


def _conv(B=1, D=4, L=8, S=4, dt=1, x=F):
    return capi.lib().dudy_short_conv_forward(x, F, None, None, None, F, None, B, D, L, S, 1, dt, None)


def _scan(B=1, D=4, L=8, N=3, G=1, dt=1, u=F):
    return capi.lib().dudy_selective_scan_forward(u, F, F, F, F, None, None, None, None, F, None, None, None, 0, B, D, L, N, G,
                                                  1, dt, None)


def _norm(B=1, D=4, L=8, dt=1, rdt=1, x=F):
    return capi.lib().dudy_block_norm_forward(x, None, F, F, None, None, F, None, F, F, None, B, D, L, 0, 1e-5, dt, rdt, None)


@pytest.mark.parametrize("call,kw,msg", [
    (_conv, {"B": 0}, "B, D and L must be positive."), (_conv, {"L": -1}, "B, D and L must be positive."),
    (_conv, {"S": 1}, "S must be between 2 and 8, got 1."), (_conv, {"S": 9}, "S must be between 2 and 8, got 9."),
    (_conv, {"dt": 7}, "Unsupported dtype."), (_conv, {"L": 1 << 40}, "tensor too large."),
    (_conv, {"B": 1 << 30, "D": 1 << 30}, "tensor too large."), (_conv, {"x": None}, "null tensor pointer"),
    (_scan, {"L": 0}, "B, D and L must be positive."), (_scan, {"N": 0}, "N must be between 1 and 64, got 0."),
    (_scan, {"N": 65}, "N must be between 1 and 64, got 65."),
    (_scan, {"G": 3}, "D must be a multiple of the number of groups, got D=4, G=3."),
    (_scan, {"G": 0}, "D must be a multiple of the number of groups, got D=4, G=0."),
    (_scan, {"dt": -1}, "Unsupported dtype."), (_scan, {"L": 1 << 31}, "tensor too large."),
    (_scan, {"u": None}, "null tensor pointer"),
    (_norm, {"D": 0}, "B, D and L must be positive."), (_norm, {"rdt": 2}, "residual dtype must equal x dtype or be float32."),
    (_norm, {"dt": 3}, "Unsupported dtype."), (_norm, {"B": 1 << 20, "L": 1 << 20}, "tensor too large."),
    (_norm, {"x": None}, "null tensor pointer"),
])
def test_refusals(call, kw, msg):
    assert call(**kw) == capi.ERR_INVALID
    assert capi.last_error() == msg


def test_workspace_is_checked_before_the_device():
    lib = capi.lib()
    need = lib.dudy_short_conv_backward_workspace_size(2, 8, 2000, 4, 1)
    assert need >= 5 * 8 * 2 * 2 * 4
    rc = lib.dudy_short_conv_backward(F, None, F, F, None, None, None, F, F, None, None, F, need - 1, 2, 8, 2000, 4, 1, 1, None)
    assert rc == capi.ERR_WORKSPACE and "workspace too small" in capi.last_error()
    need = lib.dudy_selective_scan_backward_workspace_size(2, 8, 100, 16, 1, 1)
    assert need > 0 and need % 256 == 0
    args = [F, None] + [F] * 5 + [None, None, F, None] + [F] * 5 + [None] * 3
    rc = lib.dudy_selective_scan_backward(*args, None, need, 2, 8, 100, 16, 1, 1, 1, None)
    assert rc == capi.ERR_WORKSPACE
    need = lib.dudy_block_norm_backward_workspace_size(2, 8, 100, 1, 1)
    rc = lib.dudy_block_norm_backward(F, None, F, None, F, F, None, None, F, F, F, None, F, None, None, None, None, None, F,
                                      need - 1, 2, 8, 100, 0, 1, 1, None)
    assert need > 0 and rc == capi.ERR_WORKSPACE
    # sizes that the operators refuse have no workspace
    assert lib.dudy_short_conv_backward_workspace_size(0, 8, 10, 4, 1) == 0
    assert lib.dudy_selective_scan_backward_workspace_size(1, 8, 10, 65, 1, 1) == 0
    assert lib.dudy_block_norm_backward_workspace_size(1, 8, 10, 1, 2) == 0
    # a saved state [B,D,N] for each four positions, fp32
    assert lib.dudy_selective_scan_checkpoint_bytes(2, 8, 33, 16, 1, 1) == 2 * 8 * 9 * 16 * 4


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the answer of a machine without a GPU")
def test_no_device():
    assert _conv() == _scan() == _norm() == capi.ERR_DEVICE


def test_python_checks():
    from dudyconv_b200.block_norm import FusedGatedResidualNorm1d, fused_gated_residual_norm
    from dudyconv_b200.state_space import (FusedSelectiveScan1d, FusedShortConv1d, fused_selective_scan, fused_short_conv,
                                           fused_short_conv_step)

    x, w = torch.zeros(1, 2, 3), torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="x must be CUDA tensor."):
        fused_short_conv(x, w)
    with pytest.raises(RuntimeError, match="activation must be 'silu' or None"):
        fused_short_conv(x, w, activation="relu")
    with pytest.raises(RuntimeError, match="no backward"):
        fused_short_conv_step(x[..., 0], torch.zeros(1, 2, 3), w.requires_grad_(True))
    with pytest.raises(RuntimeError, match="u must be CUDA tensor."):
        fused_selective_scan(x, x, w, torch.zeros(1, 4, 3), torch.zeros(1, 4, 3))
    with pytest.raises(RuntimeError, match="norm must be 'rms' or 'layer'"):
        fused_gated_residual_norm(x, x, x[0, :, 0], x[0, :, 0], norm="none")
    for make in (lambda: FusedShortConv1d(0), lambda: FusedShortConv1d(4, 9), lambda: FusedSelectiveScan1d(4, 65),
                 lambda: FusedSelectiveScan1d(4, 16, dt_min=0.0), lambda: FusedGatedResidualNorm1d(-1),
                 lambda: FusedGatedResidualNorm1d(8, use_bias=True)):
        with pytest.raises(ValueError):
            make()
    torch.manual_seed(0)
    s = FusedSelectiveScan1d(8, 4)
    assert torch.allclose(-s.A_log.exp(), -torch.arange(1.0, 5.0).repeat(8, 1))
    dt = torch.nn.functional.softplus(s.delta_bias)
    assert ((dt > 0.99e-3) & (dt < 1.01e-1)).all()
    assert FusedShortConv1d(8, use_bias=False).bias is None
    m = FusedGatedResidualNorm1d(8, "layer", use_bias=True, init_scale=0.1)
    assert sorted(n for n, _ in m.named_parameters()) == ["post_bias", "post_weight", "pre_bias", "pre_weight", "scale"]
