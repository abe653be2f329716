"""What autograd sees of the state-space block's calls: gradients of states that are not
contiguous."""

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
