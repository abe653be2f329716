"""States that grow: decays above 1 whose product over a long sequence leaves fp32, where the states
themselves stay in range."""

import numpy as np
import pytest
import torch

from bounds import check, dev
from oracle import state_space as ss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("L", [4096, 4001])
def test_growth_over_empty_chunks(L, dt):
    """Inputs (gradients) at the last (first) four positions alone: each state is zero before and at
    most e^4 of its input there, while the decays' product over a chunk of 128 positions is e^128."""
    from dudyconv_b200.state_space import fused_selective_scan

    rng = np.random.default_rng(21)
    B, D, N = 2, 12, 7
    u, go = np.zeros((2, B, D, L))
    u[..., -4:] = rng.standard_normal((B, D, 4))
    go[..., :4] = rng.standard_normal((B, D, 4))
    (u, ur), (go, gr) = dev(u, dt), dev(go, dt)
    (Bm, Br), (Cm, Cr) = (dev(rng.standard_normal((B, 1, N, L)), dt) for _ in range(2))
    (delta, dr), (A, Ar) = dev(np.ones((B, D, L)), dt), dev(np.ones((D, N)), "fp32")
    leaves = [t.requires_grad_(True) for t in (u, delta, A, Bm, Cm)]
    y, h = fused_selective_scan(u, delta, A, Bm, Cm, delta_softplus=False, return_final_state=True)
    ref, mag = (ss.selective_scan(ur, dr, Ar, Br, Cr, softplus=False, go=gr, mag=m) for m in (False, True))
    check(y, ref[0], mag[0], 68, "y")
    check(h, ref[1], mag[1], 68, "final_state", dt)
    for i, (k, g) in enumerate(zip(("u", "delta", "A", "B", "C"), torch.autograd.grad(y, leaves, go))):
        check(g, ref[2 + i], mag[2 + i], 68 + B, f"grad_{k}", dt)
