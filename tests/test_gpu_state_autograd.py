"""What autograd sees of the state-space block's calls: gradients of states that are not
contiguous, and the steps' writes in place."""

import numpy as np
import pytest
import torch

from bounds import dev

pytestmark = pytest.mark.gpu


def _rand(rng, dt, *shape):
    return dev(rng.standard_normal(shape), dt)[0]


# (the leaf's shape, how the leaf becomes a state) of a state [B,D,K]
STATES = {
    "expanded": (lambda B, D, K: (1, D, K), lambda t, B: t.expand(B, -1, -1)),
    "transposed": (lambda B, D, K: (B, K, D), lambda t, B: t.transpose(1, 2)),
    "sliced": (lambda B, D, K: (B, D + 2, 2 * K), lambda t, B: t[:, 1:-1, ::2]),
}


def _state_gradients(call, leaf, view, B, go, gf):
    """The leaf's gradient through the strided state, by grad and by backward, and through its
    contiguous copy; the losses use both outputs."""
    grads = []
    for prep in (lambda s: s, lambda s: s.contiguous()):
        t = leaf.clone().requires_grad_(True)
        state = prep(view(t, B))
        grads.append(torch.autograd.grad(call(state), t, (go, gf), allow_unused=True)[0])
    t = leaf.clone().requires_grad_(True)
    torch.autograd.backward(call(view(t, B)), (go, gf))
    return (*grads, t.grad)


@pytest.mark.parametrize("kind", STATES)
@pytest.mark.parametrize("others", [False, True])
def test_short_conv_state_gradient_of_any_layout(kind, others):
    from dudyconv_b200.state_space import fused_short_conv

    rng = np.random.default_rng(11)
    B, D, L, S = 3, 10, 37, 4
    shape, view = STATES[kind]
    x, w = _rand(rng, "fp16", B, D, L), _rand(rng, "fp16", D, S)
    if others:  # other inputs are differentiated too
        x.requires_grad_(True)
        w.requires_grad_(True)
    leaf = _rand(rng, "fp16", *shape(B, D, S - 1))
    go, gf = _rand(rng, "fp16", B, D, L), _rand(rng, "fp16", B, D, S - 1)
    strided, copied, accumulated = _state_gradients(
        lambda s: fused_short_conv(x, w, initial_state=s, return_final_state=True), leaf, view, B, go, gf)
    assert strided is not None and accumulated is not None, "the state has no gradient"
    assert copied.abs().max() > 0
    assert torch.equal(strided, copied) and torch.equal(accumulated, copied)


@pytest.mark.parametrize("kind", STATES)
@pytest.mark.parametrize("others", [False, True])
def test_selective_scan_state_gradient_of_any_layout(kind, others):
    from dudyconv_b200.state_space import fused_selective_scan

    rng = np.random.default_rng(12)
    B, D, L, N = 3, 20, 45, 6
    shape, view = STATES[kind]
    u, delta = _rand(rng, "bf16", B, D, L), _rand(rng, "bf16", B, D, L)
    Bm, Cm = _rand(rng, "bf16", B, 1, N, L), _rand(rng, "bf16", B, 1, N, L)
    A = -_rand(rng, "fp32", D, N).exp()
    if others:
        u.requires_grad_(True)
        A.requires_grad_(True)
    leaf = _rand(rng, "fp32", *shape(B, D, N))
    go, gf = _rand(rng, "bf16", B, D, L), _rand(rng, "fp32", B, D, N)
    strided, copied, accumulated = _state_gradients(
        lambda s: fused_selective_scan(u, delta, A, Bm, Cm, initial_state=s, return_final_state=True), leaf, view, B,
        go, gf)
    assert strided is not None and accumulated is not None, "the state has no gradient"
    assert copied.abs().max() > 0
    assert torch.equal(strided, copied) and torch.equal(accumulated, copied)


def test_a_step_on_a_saved_state_is_seen():
    """A step writes its state in place: a backward that kept that state is refused, as after
    any in-place operation."""
    from dudyconv_b200.state_space import (fused_selective_scan_step, fused_short_conv, fused_short_conv_step)

    rng = np.random.default_rng(13)
    B, D, L, S, N = 2, 6, 20, 4, 5
    x, w = _rand(rng, "fp32", B, D, L), _rand(rng, "fp32", D, S).requires_grad_(True)
    state = _rand(rng, "fp32", B, D, S - 1)
    out = fused_short_conv(x, w, initial_state=state)
    before = state._version
    with torch.no_grad():
        fused_short_conv_step(x[..., 0], state, w)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), w)

    A, bc = -torch.ones(D, N, device="cuda"), _rand(rng, "fp32", B, 1, N)
    leaf = torch.ones(B, D, N, device="cuda", requires_grad=True)
    h = _rand(rng, "fp32", B, D, N)
    kept = leaf * h  # the product's backward keeps h
    before = h._version
    with torch.no_grad():
        fused_selective_scan_step(x[..., 0], x[..., 0], A, bc, bc, h)
    assert h._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


def test_steps_take_inference_states():
    """States made in inference mode have no version; steps on them run in and outside of it."""
    from dudyconv_b200.state_space import fused_selective_scan_step, fused_short_conv_step

    x = torch.ones(2, 6, device="cuda")
    w, A, bc = torch.ones(6, 4, device="cuda"), -torch.ones(6, 5, device="cuda"), torch.ones(2, 1, 5, device="cuda")
    with torch.inference_mode():
        cs, h = torch.zeros(2, 6, 3, device="cuda"), torch.zeros(2, 6, 5, device="cuda")
        fused_short_conv_step(x, cs, w)
        fused_selective_scan_step(x, x, A, bc, bc, h)
    with torch.no_grad():
        fused_short_conv_step(x, cs, w)
        fused_selective_scan_step(x, x, A, bc, bc, h)
    assert torch.equal(cs, torch.tensor([0.0, 1.0, 1.0], device="cuda").expand(2, 6, 3)) and h.min() > 0
