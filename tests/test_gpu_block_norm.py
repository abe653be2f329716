"""GPU parity of the norms, gate and residual between blocks with their float64 formulas, and the
three operators of the state-space block run together, forwards and backwards."""

import numpy as np
import pytest
import torch

from bounds import check, dev
from oracle import state_space as ss

pytestmark = pytest.mark.gpu

CASES = [  # B, D, L, dtype, residual dtype, norm, gate, scale, biases, offset
    (1, 1, 1, "fp32", "fp32", "rms", True, True, False, 0),
    (3, 5, 1, "fp16", "fp16", "layer", True, True, True, 0),
    (64, 256, 1, "bf16", "bf16", "rms", True, True, False, 0),
    (2, 300, 7, "bf16", "fp32", "layer", True, False, True, 0),
    (2, 64, 8, "fp16", "fp32", "rms", False, True, False, 0),
    (1, 33, 31, "fp32", "fp32", "layer", False, False, True, 0),
    (2, 256, 64, "fp16", "fp16", "rms", True, True, False, 0),
    (1, 256, 136, "bf16", "fp32", "rms", True, True, False, 0),
    (1, 200, 72, "fp32", "fp32", "layer", True, True, True, 0),
    (2, 128, 65, "bf16", "bf16", "layer", True, True, True, 0),
    (1, 512, 128, "fp16", "fp16", "layer", False, True, True, 0),
    (1, 1030, 40, "fp16", "fp16", "rms", True, True, False, 0),
    (1, 256, 128, "bf16", "bf16", "rms", True, True, False, 1),
    (2, 2500, 1, "bf16", "fp32", "rms", True, True, False, 0),
]


@pytest.mark.parametrize("B,D,L,dt,rdt,norm,has_gate,has_scale,has_bias,off", CASES)
def test_block_norm(B, D, L, dt, rdt, norm, has_gate, has_scale, has_bias, off):
    from dudyconv_b200.block_norm import fused_gated_residual_norm

    rng = np.random.default_rng(B * 7 + D * 13 + L)
    seq = lambda t, s=1.0: dev(rng.standard_normal((B, D, L)) * s, t, off)  # noqa: E731
    par = lambda m, have=True: dev(m + 0.2 * rng.standard_normal(D), dt) if have else (None, None)  # noqa: E731
    v = {"x": seq(dt), "residual": seq(rdt, 2.0), "gate": seq(dt) if has_gate else (None, None), "post_weight": par(1.0),
         "post_bias": par(0.0, has_bias), "scale": par(0.5, has_scale), "pre_weight": par(1.0), "pre_bias": par(0.0, has_bias)}
    t, r = {k: a for k, (a, _) in v.items()}, {k: a for k, (_, a) in v.items()}
    (gy, gyr), (gr, grr) = seq(dt), seq(rdt)
    layer = norm == "layer"
    ref, mag = (ss.block_norm(r["x"], r["residual"], r["post_weight"], r["pre_weight"], r["gate"], r["scale"], r["post_bias"],
                              r["pre_bias"], layer, 1e-5, gyr, grr, mag=m) for m in (False, True))

    def call():
        return fused_gated_residual_norm(norm=norm, **t)

    with torch.no_grad():
        y, rout = call()
    # sums over D run in a tree; every value is at most 128 operations of the largest's size away
    big = lambda a: np.abs(a).max()  # noqa: E731
    check(y, ref[0], big(ref[0]), 128, "y", dt)
    check(rout, ref[1], big(ref[1]), 128, "residual_out", dt)
    names = [k for k in t if t[k] is not None]
    leaves = [t[k].requires_grad_(True) for k in names]
    out = call()
    assert torch.equal(out[0], y) and torch.equal(out[1], rout)
    grads = torch.autograd.grad(out, leaves, (gy, gr))
    again = torch.autograd.grad(call(), leaves, (gy, gr))
    order = ["x", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias"]
    for k, g, g2 in zip(names, grads, again):
        assert torch.equal(g, g2), f"grad_{k} is not the same twice"
        i = 2 + order.index(k)
        # a factor 1 / sqrt(var) of small variances multiplies errors as it does the values: one channel
        # alone has hat = +-1 and gradients that cancel, so the bound goes by the terms: |d| inv
        terms = big(mag[i]) if i >= 5 else max(big(ref[i]), 4.0 if D > 1 else 1e3)
        check(g, ref[i], terms, 128 + (B * L if i >= 5 else 0), f"grad_{k}", dt)


def test_one_output_alone_and_refusals():
    from dudyconv_b200.block_norm import fused_gated_residual_norm as f

    rng = np.random.default_rng(5)
    (x, xr), (r, rr), (g, gr) = (dev(rng.standard_normal((2, 8, 9)), "fp32") for _ in range(3))
    w, wr = dev(1 + 0.1 * rng.standard_normal(8), "fp32")
    x.requires_grad_(True)
    for k in (0, 1):
        got = torch.autograd.grad(f(x, r, w, w)[k], x, g)[0]
        zero = np.zeros_like(gr)
        ref = ss.block_norm(xr, rr, wr, wr, gy=gr if k == 0 else zero, gr=gr if k == 1 else zero)
        check(got, ref[2], 4.0, 128, "grad_x")
    x.requires_grad_(False)
    h = x.half()
    for call, msg in [
        (lambda: f(x, r[:, :, :5], w, w), "residual must be"),
        (lambda: f(x, h, w, w), "residual must be of x's type or float32"),
        (lambda: f(h, r, w, w), "post_weight must be Half"),
        (lambda: f(x, r, w[:4], w), "post_weight must be"),
        (lambda: f(x, r, w, w, gate=h), "gate must be Float"),
        (lambda: f(x, r, w, w, norm="batch"), "norm must be"),
        (lambda: f(x, r, w, w, eps=0.0), "eps must be positive"),
        (lambda: f(x, r, w, w, pre_bias=w), "an rms norm has no bias"),
        (lambda: f(x[0], r[0], w, w), r"x must be \[B,D,L\]"),
        (lambda: f(x[..., :0], r[..., :0], w, w), "must be positive"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()


def _block(x, gate, residual, p, lib):
    """conv -> scan -> gate, norm, residual, norm: one block's token mixing."""
    B, D, L = x.shape
    c = lib["conv"](x, p["w"], p["b"])
    y = lib["scan"](c, p["delta"], p["A"], p["B"], p["C"], p["skip"], p["bias"])
    return lib["norm"](y, residual, p["w1"], p["w2"], gate, p["sc"])


def _float64():
    def conv(x, w, b):
        S, L = w.shape[1], x.shape[2]
        xe = torch.nn.functional.pad(x, (S - 1, 0))
        return torch.nn.functional.silu(sum(w[:, j, None] * xe[..., j:j + L] for j in range(S)) + b[:, None])

    def scan(u, de, A, Bm, Cm, skip, bias):
        dt = torch.nn.functional.softplus(de + bias[:, None])
        h, ys = 0.0, []
        for t in range(u.shape[2]):
            h = torch.exp(dt[..., t, None] * A) * h + (dt[..., t] * u[..., t])[..., None] * Bm[:, None, :, t]
            ys.append((h * Cm[:, None, :, t]).sum(2))
        return torch.stack(ys, 2) + skip[:, None] * u

    def norm(x, r, w1, w2, gate, sc):
        rms = lambda v: v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5)  # noqa: E731
        r = r + sc[:, None] * rms(x * torch.nn.functional.silu(gate)) * w1[:, None]
        return rms(r) * w2[:, None], r

    return {"conv": conv, "scan": scan, "norm": norm}


def test_block_forward_and_backward():
    """Two blocks of the three operators in fp32 against torch autograd in float64: the outputs and
    every gradient. Each operator is within (L + 64) * 4 * 2^-24 of its terms (tests above); six of
    them in a row, with amplifications of a few, stay within 2^-11 of the largest value."""
    from dudyconv_b200.block_norm import fused_gated_residual_norm
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv

    ours = {"conv": fused_short_conv, "scan": fused_selective_scan, "norm": fused_gated_residual_norm}
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    B, D, L, N = 2, 40, 52, 16
    shapes = {"w": (D, 4), "b": (D,), "delta": (B, D, L), "A": (D, N), "B": (B, N, L), "C": (B, N, L), "skip": (D,),
              "bias": (D,), "w1": (D,), "w2": (D,), "sc": (D,)}
    sets = []
    for _ in range(2):
        p = {k: rand(*s) * 0.5 for k, s in shapes.items()}
        p["A"] = -p["A"].exp()
        sets.append(p)
    x, gate, res, go, gr = (rand(B, D, L) for _ in range(5))

    def run(cast, lib):
        ps = [{k: cast(v).requires_grad_(True) for k, v in p.items()} for p in sets]
        xs = [cast(v).requires_grad_(True) for v in (x, gate, res)]
        y, r = xs[0], xs[2]
        for p in ps:
            y, r = _block(y, xs[1], r, p, lib)
        leaves = xs + [v for p in ps for v in p.values()]
        return [y, r, *torch.autograd.grad((y, r), leaves, (cast(go), cast(gr)))]

    for i, (a, b) in enumerate(zip(run(lambda v: v.clone(), ours), run(lambda v: v.double(), _float64()))):
        assert (a.double() - b).abs().max() <= 2 ** -11 * b.abs().max(), i


def test_offsets_beyond_32_bits():
    """Tokens behind the 2^31st element of the tensors, against the same tokens alone."""
    from dudyconv_b200.block_norm import fused_gated_residual_norm as f

    B, D, L = 3, 1024, (1 << 20) + 8
    assert (B - 1) * D * L > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(B, D, L, device="cuda", generator=g, dtype=torch.bfloat16)
    w = torch.randn(D, device="cuda", generator=g, dtype=torch.bfloat16)
    y, r = f(x, x, w, w)
    tail = x[2:, :, -520:].contiguous()
    y1, r1 = f(tail, tail, w, w)
    assert torch.equal(y[2:, :, -520:], y1) and torch.equal(r[2:, :, -520:], r1)


def test_module_and_capture():
    from dudyconv_b200.block_norm import FusedGatedResidualNorm1d

    torch.manual_seed(0)
    m = FusedGatedResidualNorm1d(96, "layer", use_bias=True, init_scale=0.5, device="cuda")
    x, z = (torch.randn(2, 96, 40, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    r = torch.randn(2, 96, 40, device="cuda")
    params = list(m.parameters())

    def step():
        y, o = m(x, r, z)
        grads = torch.autograd.grad(y.float().sum() + o.square().sum(), params)
        # no eager graph of the leaves may live while a backward is captured (torch's own rule)
        return [v.detach() for v in (y, o, *grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(0.5)
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
