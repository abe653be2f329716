"""The state-space block at sizes that keep a block busy: scans of many stretches that are not cut
into chunks, and norms of several tiles to a block, against their float64 formulas."""

import numpy as np
import pytest
import torch

from bounds import check, dev
from oracle import state_space as ss

pytestmark = pytest.mark.gpu

# A block of the scan takes 32 / lanes * channels of a thread; from 75 blocks on (a GPU of 148 SMs, two
# of them on each) the forward is not cut, nor the backward from 75 (four channels to a thread, one
# block an SM) or 149. Seven stretches of 64 positions come round the three stretch buffers
# twice, so their barriers' parity returns.
SCAN = [  # B, D, L, N, G, dtype, lengths, state
    (16, 256, 520, 16, 1, "fp16", False, False),  # four channels to a thread in the backward
    (16, 256, 521, 16, 1, "bf16", True, True),
    (16, 250, 456, 13, 1, "fp32", True, True),
    (20, 256, 463, 7, 2, "fp16", True, False),
    (40, 256, 456, 4, 1, "bf16", False, True),
    (5, 256, 470, 32, 1, "fp32", False, True),
    (3, 256, 449, 50, 1, "bf16", True, True),
]


@pytest.mark.parametrize("B,D,L,N,G,dt,padded,has_state", SCAN)
def test_scan_of_many_stretches(B, D, L, N, G, dt, padded, has_state):
    from dudyconv_b200.state_space import fused_selective_scan

    rng = np.random.default_rng(B * 3 + D * 5 + L * 7 + N)
    seq = lambda: dev(rng.standard_normal((B, D, L)), dt)  # noqa: E731
    bc = lambda: dev(rng.standard_normal((B, G, N, L)), dt)  # noqa: E731
    v = {"u": seq(), "delta": seq(), "A": dev(-np.exp(rng.standard_normal((D, N))), "fp32"), "B": bc(), "C": bc(),
         "skip": dev(rng.standard_normal(D), "fp32"), "delta_bias": dev(rng.uniform(-4, 0, D), "fp32"),
         "state": dev(rng.standard_normal((B, D, N)), "fp32") if has_state else (None, None)}
    t, r = {k: a for k, (a, _) in v.items()}, {k: a for k, (_, a) in v.items()}
    (go, gr), (gf, fr) = seq(), dev(rng.standard_normal((B, D, N)), "fp32")
    lengths = [L, 0, 1, 64, 65, 193, 384, L - 1][:B] if padded else None
    if padded:
        lengths += [int(n) for n in rng.integers(200, L + 1, B - len(lengths))]
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    ref, mag = (ss.selective_scan(r["u"], r["delta"], r["A"], r["B"], r["C"], r["skip"], r["delta_bias"], True, r["state"],
                                  lengths, gr, fr, mag=m) for m in (False, True))
    names = [k for k in t if t[k] is not None]
    leaves = [t[k].requires_grad_(True) for k in names]
    y, h = fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"], True, t["state"],
                                n, True)
    check(y, ref[0], mag[0], L + 64, "y")
    check(h, ref[1], mag[1], L + 64, "final_state", dt)
    for k, g in zip(names, torch.autograd.grad((y, h), leaves, (go, gf))):
        i = 2 + list(t).index(k)
        check(g, ref[i], mag[i], L + B + 64, f"grad_{k}", dt)


# Tiles of 32 tokens up to D = 256, 16 up to 512, 8 up to 1024; 296 (forward) and 148 blocks take them
# in turn. 16-bit tensors have two tiles in flight in the backward, fp32 ones and an fp32 residual one.
NORM = [  # B, D, L, dtype, residual dtype, norm, gate
    (8, 256, 2048, "fp16", "fp16", "rms", True),
    (5, 256, 2051, "bf16", "bf16", "layer", True),
    (5, 200, 2048, "bf16", "fp32", "layer", True),
    (4, 256, 2601, "fp16", "fp32", "rms", True),
    (4, 256, 2600, "fp32", "fp32", "rms", True),
    (3, 100, 3301, "fp32", "fp32", "layer", False),
    (4, 64, 2500, "bf16", "bf16", "rms", False),
    (2, 512, 2500, "fp16", "fp16", "layer", True),
    (2, 700, 1203, "fp16", "fp16", "rms", True),
    (3, 1024, 1000, "bf16", "fp32", "layer", True),
    (2, 1024, 8, "bf16", "bf16", "rms", True),
    (1, 1024, 136, "fp32", "fp32", "layer", True),
    (2, 1000, 1201, "fp32", "fp32", "rms", True),
]


@pytest.mark.parametrize("B,D,L,dt,rdt,norm,has_gate", NORM)
def test_norm_of_many_tiles(B, D, L, dt, rdt, norm, has_gate):
    from dudyconv_b200.block_norm import fused_gated_residual_norm

    rng = np.random.default_rng(B * 7 + D * 13 + L)
    layer = norm == "layer"
    seq = lambda t, s=1.0: dev(rng.standard_normal((B, D, L)) * s, t)  # noqa: E731
    par = lambda m, have=True: dev(m + 0.2 * rng.standard_normal(D), dt) if have else (None, None)  # noqa: E731
    v = {"x": seq(dt), "residual": seq(rdt, 2.0), "gate": seq(dt) if has_gate else (None, None), "post_weight": par(1.0),
         "post_bias": par(0.0, layer), "scale": par(0.5), "pre_weight": par(1.0), "pre_bias": par(0.0, layer)}
    t, r = {k: a for k, (a, _) in v.items()}, {k: a for k, (_, a) in v.items()}
    (gy, gyr), (gr, grr) = seq(dt), seq(rdt)
    ref, mag = (ss.block_norm(r["x"], r["residual"], r["post_weight"], r["pre_weight"], r["gate"], r["scale"], r["post_bias"],
                              r["pre_bias"], layer, 1e-5, gyr, grr, mag=m) for m in (False, True))
    names = [k for k in t if t[k] is not None]
    leaves = [t[k].requires_grad_(True) for k in names]
    out = fused_gated_residual_norm(norm=norm, **t)
    big = lambda a: np.abs(a).max()  # noqa: E731
    check(out[0], ref[0], big(ref[0]), 128, "y", dt)
    check(out[1], ref[1], big(ref[1]), 128, "residual_out", dt)
    order = ["x", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias"]
    # a parameter's sum: each term is 128 operations long; a thread adds four of a tile's tokens to each of
    # two sums, at most four tiles in a row, the lanes and 148 blocks' parts follow in 64 more
    for k, g in zip(names, torch.autograd.grad(out, leaves, (gy, gr))):
        i = 2 + order.index(k)
        terms = big(mag[i]) if i >= 5 else max(big(ref[i]), 4.0)
        check(g, ref[i], terms, 128 + (80 if i >= 5 else 0), f"grad_{k}", dt)
