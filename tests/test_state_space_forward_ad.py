"""Forward-mode differentiation of the state-space block's calls is refused: an output without a
tangent would count them as constants. The refusal comes before any check of the device, so it is
seen without a GPU; with one, the same calls run where no tangent is asked for."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device):
    """name -> (the input that carries the tangent, the call on it)"""
    from dudyconv_b200 import state_space as sp
    from dudyconv_b200.block_norm import fused_gated_residual_norm as norm

    x = torch.linspace(-1, 1, 2 * 4 * 6, device=device).view(2, 4, 6)
    w, p = torch.ones(4, 4, device=device), torch.ones(4, device=device)
    A = -torch.ones(4, 3, device=device)
    bc = torch.ones(2, 1, 3, 6, device=device)
    st, cs = torch.ones(2, 4, 3, device=device), torch.ones(2, 4, 3, device=device)
    x0, bc0 = x[..., 0].contiguous(), bc[..., 0].contiguous()
    return {
        "conv x": (x, lambda v: sp.fused_short_conv(v, w)),
        "conv weight": (w, lambda v: sp.fused_short_conv(x, v)),
        "conv bias": (p, lambda v: sp.fused_short_conv(x, w, v)),
        "conv state": (cs, lambda v: sp.fused_short_conv(x, w, initial_state=v)),
        "conv step x": (x0, lambda v: sp.fused_short_conv_step(v, cs.clone(), w)),
        "conv step state": (cs, lambda v: sp.fused_short_conv_step(x0, v, w)),
        "scan u": (x, lambda v: sp.fused_selective_scan(v, x, A, bc, bc)),
        "scan A": (A, lambda v: sp.fused_selective_scan(x, x, v, bc, bc)),
        "scan B": (bc, lambda v: sp.fused_selective_scan(x, x, A, v, bc)),
        "scan delta_bias": (p, lambda v: sp.fused_selective_scan(x, x, A, bc, bc, delta_bias=v)),
        "scan state": (st, lambda v: sp.fused_selective_scan(x, x, A, bc, bc, initial_state=v)),
        "scan step u": (x0, lambda v: sp.fused_selective_scan_step(v, x0, A, bc0, bc0, st.clone())),
        "scan step state": (st, lambda v: sp.fused_selective_scan_step(x0, x0, A, bc0, bc0, v)),
        "norm x": (x, lambda v: norm(v, x, p, p)),
        "norm residual": (x, lambda v: norm(x, v, p, p)),
        "norm scale": (p, lambda v: norm(x, x, p, p, scale=v)),
    }


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_tangents_are_refused(name, grad, device):
    value, call = _calls(device)[name]
    with torch.set_grad_enabled(grad), fwad.dual_level():
        dual = fwad.make_dual(value, torch.ones_like(value))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_without_a_tangent_the_call_runs(name):
    """Inside a dual level plain tensors pass, and so do dual ones where forward mode is off."""
    value, call = _calls("cuda")[name]
    with torch.no_grad(), fwad.dual_level():
        call(value.clone())
        with fwad._set_fwd_grad_enabled(False):
            call(fwad.make_dual(value.clone(), torch.ones_like(value)))
