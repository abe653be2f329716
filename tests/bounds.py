"""Error bounds of the state-space block's tests, from arithmetic.

A result of type t is rounded once, by at most half a step of |ref|: eps(t) / 2. Before that it
is an fp32 sum whose error is at most (operations on the longest path) * 2^-24 * (the sum of the
magnitudes of its terms); the oracle gives that sum (``mag``), the test the length of the path.
The 16-bit kernels use the fast exponential, logarithm and division, whose relative errors are up
to 2^-21 (eight times 2^-24) an operation; the accurate functions of the fp32 kernels are within
2 units. fp16 results below 2^-14 are rounded to steps of 2^-24.
"""

import numpy as np
import torch

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def check(got: torch.Tensor, ref, mag, path: float, name: str, math: str | None = None):
    """|got - ref| within the bound; ``math``: the type whose kernels computed an fp32 result."""
    ref, mag = np.asarray(ref, np.float64), np.asarray(mag, np.float64)
    a = got.detach().double().cpu().numpy()
    assert a.shape == ref.shape, (name, a.shape, ref.shape)
    t = {v: k for k, v in TYPES.items()}[got.dtype]
    half = torch.finfo(got.dtype).eps / 2
    fast = 4 if (math or t) == "fp32" else 8
    bound = half * np.abs(ref) + (1 + half) * path * fast * 2.0 ** -24 * mag
    bound += 2.0 ** -25 if t == "fp16" else 1e-30
    bad = ~(np.abs(a - ref) <= bound)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(np.isnan(a), np.inf, np.abs(a - ref) - bound)), a.shape)
        raise AssertionError(f"{name} [{t}]: {int(bad.sum())}/{bad.size} values outside the bound; worst at "
                             f"{i}: got {a[i]!r}, want {ref[i]!r}, bound {np.broadcast_to(bound, a.shape)[i]:.3e}")


def dev(x, dt: str, off: int = 0):
    """A CUDA tensor of type dt, its storage ``off`` elements behind an aligned one, and its
    values in float64."""
    t = torch.from_numpy(np.ascontiguousarray(x)).to("cuda", TYPES[dt])
    if off:
        base = torch.empty(t.numel() + off, device="cuda", dtype=t.dtype)
        base[off:].copy_(t.flatten())
        t = base[off:].view(t.shape)
    return t, t.double().cpu().numpy()
