"""GPU parity of the short causal conv and the selective scan with their float64 formulas:
sequences forward and backward, padded batches, carried states, single tokens, the types,
alignments and streams that a user's calls have, and the refusals."""

import numpy as np
import pytest
import torch

from bounds import TYPES, check, dev
from oracle import state_space as ss

pytestmark = pytest.mark.gpu


def _rng(*key):
    return np.random.default_rng(sum((i + 1) * ord(c) for i, c in enumerate(repr(key))))


# ---------------------------------------------------------------------------------------
# short causal conv
# ---------------------------------------------------------------------------------------
CONV = [  # B, D, L, S, dtype, lengths, state, bias, silu, offset in elements
    (1, 1, 1, 4, "fp32", None, False, True, True, 0),
    (2, 3, 2, 8, "fp16", None, True, True, True, 0),
    (2, 5, 7, 4, "bf16", [7, 0], True, True, True, 0),
    (1, 4, 8, 2, "fp16", None, False, False, True, 0),
    (3, 2, 255, 3, "fp32", [255, 1, 200], True, True, True, 0),
    (1, 3, 256, 4, "fp16", None, False, True, True, 0),
    (2, 2, 257, 5, "bf16", None, True, True, False, 0),
    (1, 2, 1023, 4, "fp16", None, False, True, True, 0),
    (2, 3, 1024, 4, "bf16", [1024, 1023], True, True, True, 0),
    (1, 2, 1025, 6, "fp32", None, True, True, True, 0),
    (2, 2, 2056, 4, "fp16", [2056, 1025], True, True, True, 0),
    (1, 2, 1032, 7, "bf16", None, False, True, True, 1),
    (2, 3, 264, 8, "fp32", [2, 3], True, False, True, 1),
    (5, 200, 64, 4, "fp16", None, False, True, True, 0),
]


@pytest.mark.parametrize("B,D,L,S,dt,lengths,has_state,has_bias,silu,off", CONV)
def test_short_conv(B, D, L, S, dt, lengths, has_state, has_bias, silu, off):
    from dudyconv_b200.state_space import fused_short_conv

    rng = _rng(B, D, L, S, dt)
    x, xr = dev(rng.standard_normal((B, D, L)), dt, off)
    w, wr = dev(rng.standard_normal((D, S)) * S ** -0.5, dt)
    b, br = dev(rng.standard_normal(D), dt) if has_bias else (None, None)
    st, sr = dev(rng.standard_normal((B, D, S - 1)), dt) if has_state else (None, None)
    go, gr = dev(rng.standard_normal((B, D, L)), dt, off)
    gf, fr = dev(rng.standard_normal((B, D, S - 1)), dt)
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    act = "silu" if silu else None
    ref, mag = (ss.short_conv(xr, wr, br, sr, lengths, silu, gr, fr, mag=m) for m in (False, True))
    with torch.no_grad():
        out, fin = fused_short_conv(x, w, b, st, n, act, True)
        plain = fused_short_conv(x, w, b, st, n, act)
    assert torch.equal(plain, out)
    check(out, ref[0], mag[0], S + 16, "out")
    assert np.array_equal(fin.double().cpu().numpy(), ref[1])  # copied values

    leaves = [t.requires_grad_(True) for t in (x, w, b, st) if t is not None]
    out, fin = fused_short_conv(x, w, b, st, n, act, True)
    grads = torch.autograd.grad((out, fin), leaves, (go, gf))
    again = torch.autograd.grad(fused_short_conv(x, w, b, st, n, act, True), leaves, (go, gf))
    names = [k for k, t in zip(("x", "w", "bias", "state"), (x, w, b, st)) if t is not None]
    which = dict(zip(("x", "w", "bias", "state"), range(2, 6)))
    for k, g, h in zip(names, grads, again):
        assert torch.equal(g, h), f"grad_{k} is not the same twice"
        check(g, ref[which[k]], mag[which[k]], S + 80, f"grad_{k}")


def test_short_conv_only_the_state_is_used():
    """A loss of the final state alone, and of the output alone."""
    from dudyconv_b200.state_space import fused_short_conv

    rng = _rng("only")
    x, xr = dev(rng.standard_normal((2, 3, 20)), "fp32")
    w, wr = dev(rng.standard_normal((3, 4)), "fp32")
    gf, fr = dev(rng.standard_normal((2, 3, 3)), "fp32")
    x.requires_grad_(True)
    w.requires_grad_(True)
    _, fin = fused_short_conv(x, w, return_final_state=True)
    gx, gw = torch.autograd.grad(fin, [x, w], gf)
    want = np.zeros((2, 3, 20))
    want[:, :, -3:] = fr
    assert np.array_equal(gx.double().cpu().numpy(), want) and not gw.any()


@pytest.mark.parametrize("B,D,S,dt,bias", [(1, 1, 2, "fp32", True), (3, 130, 4, "fp16", True),
                                           (2, 7, 8, "bf16", False), (64, 256, 4, "bf16", True)])
def test_short_conv_step(B, D, S, dt, bias):
    from dudyconv_b200.state_space import fused_short_conv_step

    rng = _rng("step", B, D, S)
    st, sr = dev(rng.standard_normal((B, D, S - 1)), dt)
    w, wr = dev(rng.standard_normal((D, S)), dt)
    b, br = dev(rng.standard_normal(D), dt) if bias else (None, None)
    for _ in range(3):
        x, xr = dev(rng.standard_normal((B, D)), dt)
        out = fused_short_conv_step(x, st, w, b)
        ref, mag = (ss.short_conv(xr[..., None], wr, br, sr, mag=m) for m in (False, True))
        check(out, ref[0][..., 0], mag[0][..., 0], S + 16, "out")
        assert np.array_equal(st.double().cpu().numpy(), ref[1])
        sr = ref[1]


# ---------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------
SCAN = [  # B, D, L, N, G, dtype, lengths, state, skip, delta_bias, softplus, offset
    (1, 1, 1, 1, 1, "fp32", None, False, True, True, True, 0),
    (2, 3, 2, 3, 1, "fp16", None, True, True, True, True, 0),
    (2, 8, 31, 4, 2, "bf16", [31, 0], True, True, True, True, 0),
    (1, 33, 32, 5, 1, "fp32", None, True, False, True, True, 0),
    (2, 16, 33, 8, 4, "fp16", [1, 33], True, True, False, True, 0),
    (1, 40, 127, 16, 1, "fp16", None, False, True, True, True, 0),
    (3, 32, 128, 16, 1, "bf16", [128, 127, 32], True, True, True, True, 0),
    (2, 12, 129, 17, 3, "fp32", None, True, True, True, True, 0),
    (1, 20, 200, 32, 1, "bf16", None, False, False, False, True, 0),
    (2, 18, 264, 64, 2, "fp16", [264, 100], True, True, True, True, 0),
    (1, 9, 264, 33, 1, "fp32", [161], True, True, True, True, 1),
    (2, 64, 160, 16, 1, "fp32", None, True, True, True, False, 0),
    (1, 256, 300, 16, 1, "fp16", None, True, True, True, True, 0),
    (1, 5, 296, 16, 1, "bf16", None, True, True, True, True, 1),
    (1, 130, 72, 2, 1, "fp16", None, True, True, True, True, 0),
    (1, 70, 96, 7, 2, "bf16", None, True, True, True, True, 0),
    (2, 97, 75, 3, 1, "fp16", [75, 40], True, True, True, True, 0),
    (1, 24, 1000, 16, 1, "bf16", None, True, True, True, True, 0),
    (3, 24, 520, 24, 2, "fp32", [520, 33, 300], True, True, True, True, 0),
    (2, 6, 70, 16, 6, "fp16", None, True, True, True, True, 0),  # a group for each channel
    (16, 256, 40, 16, 1, "fp16", None, True, True, True, True, 0),  # channels enough for four to a thread
    (7, 520, 33, 12, 1, "bf16", [33, 0, 1, 32, 31, 20, 7], True, True, True, True, 0),
    (4, 1000, 37, 16, 1, "fp32", None, True, True, True, True, 1),
]


def _scan_inputs(B, D, L, N, G, dt, rng, softplus=True, off=0, state=True, skip=True, bias=True):
    de = rng.standard_normal((B, D, L))
    if not softplus:
        de = 0.02 + 0.1 * np.abs(de)
    v = {"u": dev(rng.standard_normal((B, D, L)), dt, off), "delta": dev(de, dt, off),
         "A": dev(-np.exp(rng.standard_normal((D, N))), "fp32"),
         "B": dev(rng.standard_normal((B, G, N, L)), dt, off),
         "C": dev(rng.standard_normal((B, G, N, L)), dt, off),
         "skip": dev(rng.standard_normal(D), "fp32") if skip else (None, None),
         "delta_bias": dev(rng.uniform(-4, 0, D) if softplus else rng.uniform(0, 0.1, D), "fp32") if bias else (None, None),
         "state": dev(rng.standard_normal((B, D, N)), "fp32") if state else (None, None)}
    return {k: t for k, (t, _) in v.items()}, {k: r for k, (_, r) in v.items()}


@pytest.mark.parametrize("B,D,L,N,G,dt,lengths,has_state,has_skip,has_bias,softplus,off", SCAN)
def test_selective_scan(B, D, L, N, G, dt, lengths, has_state, has_skip, has_bias, softplus, off):
    from dudyconv_b200.state_space import fused_selective_scan

    rng = _rng(B, D, L, N, G, dt)
    t, r = _scan_inputs(B, D, L, N, G, dt, rng, softplus, off, has_state, has_skip, has_bias)
    go, gr = dev(rng.standard_normal((B, D, L)), dt, off)
    gf, fr = dev(rng.standard_normal((B, D, N)), "fp32")
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    ref, mag = (ss.selective_scan(r["u"], r["delta"], r["A"], r["B"], r["C"], r["skip"], r["delta_bias"], softplus,
                                  r["state"], lengths, gr, fr, mag=m) for m in (False, True))

    def call():
        return fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"], softplus,
                                    t["state"], n, True)

    with torch.no_grad():
        y, h = call()
        y1 = fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"], softplus,
                                  t["state"], n)
    assert torch.equal(y, y1)
    check(y, ref[0], mag[0], L + 64, "y")
    check(h, ref[1], mag[1], L + 64, "final_state", dt)
    names = [k for k in t if t[k] is not None]
    leaves = [t[k].requires_grad_(True) for k in names]
    out = call()
    assert torch.equal(out[0], y) and torch.equal(out[1], h)
    grads = torch.autograd.grad(out, leaves, (go, gf))
    again = torch.autograd.grad(call(), leaves, (go, gf))
    for k, g, g2 in zip(names, grads, again):
        assert torch.equal(g, g2), f"grad_{k} is not the same twice"
        i = 2 + list(t).index(k)
        check(g, ref[i], mag[i], L + B + 64, f"grad_{k}", dt)


@pytest.mark.parametrize("B,D,N,G,dt", [(1, 1, 1, 1, "fp32"), (3, 130, 16, 1, "fp16"), (2, 24, 5, 3, "bf16"),
                                        (5, 16, 64, 2, "fp32"), (64, 256, 16, 1, "bf16"), (2, 9, 33, 1, "fp16")])
def test_selective_scan_step(B, D, N, G, dt):
    from dudyconv_b200.state_space import fused_selective_scan_step

    rng = _rng("step", B, D, N)
    t, r = _scan_inputs(B, D, 3, N, G, dt, rng)
    h, hr = t["state"], r["state"]
    for k in range(3):
        y = fused_selective_scan_step(*(t[n][..., k] if n in ("u", "delta", "B", "C") else t[n]
                                        for n in ("u", "delta", "A", "B", "C")), h, t["skip"], t["delta_bias"])
        ref, mag = (ss.selective_scan(r["u"][..., k:k + 1], r["delta"][..., k:k + 1], r["A"], r["B"][..., k:k + 1],
                                      r["C"][..., k:k + 1], r["skip"], r["delta_bias"], state=hr, mag=m)
                    for m in (False, True))
        check(y, ref[0][..., 0], mag[0][..., 0], 64, "y")
        check(h, ref[1], mag[1], 64, "state", dt)
        hr = h.double().cpu().numpy()


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_prompt_then_tokens_is_the_whole_sequence(dt):
    """A padded batch of prompts, each continued token by token from its own length, gives what
    each sequence gives alone: conv -> scan as a block runs them."""
    from dudyconv_b200.state_space import (fused_selective_scan, fused_selective_scan_step, fused_short_conv,
                                           fused_short_conv_step)

    rng = _rng("chain", dt)
    B, D, L, N, S, more = 3, 24, 70, 16, 4, 3
    lengths = [70, 1, 33]
    x, _ = dev(rng.standard_normal((B, D, L + more)), dt)
    w, _ = dev(rng.standard_normal((D, S)), dt)
    t, _ = _scan_inputs(B, D, L + more, N, 1, dt, rng, state=False)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    pad = lambda v: v[..., :L].masked_fill(torch.arange(L, device="cuda") >= n.view(-1, *[1] * (v.dim() - 1)),  # noqa: E731
                                           float("nan"))
    par = {"skip": t["skip"], "delta_bias": t["delta_bias"]}
    c, cs = fused_short_conv(pad(x), w, lengths=n, return_final_state=True)
    y, h = fused_selective_scan(c, pad(t["delta"]), t["A"], pad(t["B"]), pad(t["C"]), **par, lengths=n,
                                return_final_state=True)
    assert not y.isnan().any() and not h.isnan().any()
    at = lambda v, k: torch.stack([v[b, ..., lengths[b] + k] for b in range(B)])  # noqa: E731
    steps = []
    for k in range(more):
        ck = fused_short_conv_step(at(x, k), cs, w)
        steps.append(fused_selective_scan_step(ck, at(t["delta"], k), t["A"], at(t["B"], k), at(t["C"], k), h, **par))
    eps = torch.finfo(TYPES[dt]).eps
    for b in range(B):
        e = lengths[b] + more
        one = lambda v: v[b:b + 1, ..., :e]  # noqa: E731
        cw = fused_short_conv(one(x), w)
        yw, hw = fused_selective_scan(cw, one(t["delta"]), t["A"], one(t["B"]), one(t["C"]), **par,
                                      return_final_state=True)
        got = torch.cat([y[b, :, :lengths[b]], *(s[b][:, None] for s in steps)], 1).double()
        assert not y[b, :, lengths[b]:].any()
        # the conv's outputs may differ by a rounding (another order of its sum), the scan's by
        # that input's change and a rounding: 4 eps of the largest value
        assert (got - yw[0].double()).abs().max() <= 4 * eps * yw.abs().max()
        assert (h[b] - hw[0]).abs().max() <= 4 * eps * hw.abs().max()


@pytest.mark.parametrize("L", [63, 64, 65, 129, 191, 777])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_rows_that_start_inside_a_word(L, dt):
    """Odd lengths and tensors that start on any element: the elements around a tensor and behind a
    sequence's length (NaN here) are not used, and the bits are those of the same rows in a tensor
    that starts on 16 bytes and has a length of whole words."""
    from dudyconv_b200.state_space import fused_selective_scan

    B, D, N, G = 2, 20, 6, 2
    t, _ = _scan_inputs(B, D, L, N, G, dt, _rng("inside", L, dt))
    lengths = torch.tensor([L, L // 2], device="cuda", dtype=torch.int32)
    wide = (L + 7) // 8 * 8

    def placed(v, off):
        box = torch.full((v.numel() + off + 9,), float("nan"), device="cuda", dtype=v.dtype)
        w = box[off:off + v.numel()].view(v.shape)
        w.copy_(v)
        for b, n in enumerate(lengths.tolist()):
            w[b, ..., n:] = float("nan")
        return w

    def padded(v):
        w = torch.zeros((*v.shape[:-1], wide), device="cuda", dtype=v.dtype)
        w[..., :L] = v
        return w

    rows = ("u", "delta", "B", "C")
    with torch.no_grad():
        def call(u, delta, Bm, Cm):
            return fused_selective_scan(u, delta, t["A"], Bm, Cm, t["skip"], t["delta_bias"], True, t["state"],
                                        lengths, True)

        y, h = call(*(padded(t[k]) for k in rows))
        for offs in ((0, 0, 0, 0), (1, 0, 1, 0), (0, 1, 0, 1), (3, 2, 1, 5)):
            y2, h2 = call(*(placed(t[k], o) for k, o in zip(rows, offs)))
            assert torch.equal(y2, y[..., :L]), offs
            assert torch.equal(h2, h), offs


def test_padding_holds_anything():
    """Infinities and NaN at padded positions change nothing, forwards or backwards."""
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv

    rng = _rng("pad")
    B, D, L, N = 2, 16, 150, 16
    n = torch.tensor([150, 61], device="cuda", dtype=torch.int32)
    res = []
    for fill in (0.0, float("nan"), float("inf"), float("-inf")):
        rng = _rng("pad")
        t, _ = _scan_inputs(B, D, L, N, 1, "bf16", rng)
        go, _ = dev(rng.standard_normal((B, D, L)), "bf16")
        w, _ = dev(rng.standard_normal((D, 4)), "bf16")
        for v in (t["u"], t["delta"], t["B"], t["C"], go):
            v[1, ..., 61:] = fill
        leaves = [v.requires_grad_(True) for v in (*t.values(), w)]
        y = fused_selective_scan(fused_short_conv(t["u"], w, lengths=n), t["delta"], t["A"], t["B"], t["C"], t["skip"],
                                 t["delta_bias"], initial_state=t["state"], lengths=n)
        res.append([y, *torch.autograd.grad(y, leaves, go)])
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["fp32", "fp16", "bf16"])
def test_steps_of_minus_infinity_pass_the_state(dt):
    """delta at -infinity or at the type's lowest value is a step of zero: the state passes, the
    gradients there are zero, and NaN is not made; a NaN in delta stays in its row."""
    from dudyconv_b200.state_space import fused_selective_scan, fused_selective_scan_step

    rng = _rng("low", dt)
    B, D, L, N = 1, 8, 40, 16
    t, r = _scan_inputs(B, D, L, N, 1, dt, rng)
    go, gr = dev(rng.standard_normal((B, D, L)), dt)
    de = t["delta"]
    de[..., 10:14] = float("-inf")
    de[..., 20:22] = torch.finfo(de.dtype).min
    r["delta"] = de.double().cpu().numpy().clip(-1e4)  # exp(-1e4) is zero in float64 too
    leaves = [t[k].requires_grad_(True) for k in t]
    y = fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"], initial_state=t["state"])
    grads = torch.autograd.grad(y, leaves, go)
    ref, mag = (ss.selective_scan(r["u"], r["delta"], r["A"], r["B"], r["C"], r["skip"], r["delta_bias"], True, r["state"],
                                  None, gr, None, mag=m) for m in (False, True))
    check(y, ref[0], mag[0], L + 64, "y")
    for k, g in zip(t, grads):
        i = 2 + list(t).index(k)
        check(g, ref[i], mag[i], L + 65, f"grad_{k}", dt)
    with torch.no_grad():
        h = t["state"].clone()
        fused_selective_scan_step(t["u"][..., 0], de[..., 10], t["A"], t["B"][..., 0], t["C"][..., 0], h, t["skip"], t["delta_bias"])
        assert torch.equal(h, t["state"])
        de[0, 3, 5] = float("nan")
        y = fused_selective_scan(t["u"], de, t["A"], t["B"], t["C"])
        bad = y.isnan()[0]
        assert bad[3, 5:].all() and not bad[3, :5].any() and not bad[:3].any() and not bad[4:].any()


def test_strides_and_orders():
    """Slices of a projection, a transposed tensor and an expanded gradient are taken as they are."""
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv

    rng = _rng("strides")
    B, D, L, N = 2, 16, 40, 8
    both, _ = dev(rng.standard_normal((B, 2 * D, L)), "fp16")
    last, _ = dev(rng.standard_normal((B, L, D)), "fp16")
    bc, _ = dev(rng.standard_normal((B, 3 + 2 * N, L)), "fp16")
    t, _ = _scan_inputs(B, D, L, N, 1, "fp16", rng)
    w, _ = dev(rng.standard_normal((D, 4)), "fp16")
    u, de, Bm, Cm = both[:, D:], last.transpose(1, 2), bc[:, 3:3 + N], bc[:, 3 + N:]

    def run(u, de, Bm, Cm):
        u, de = u.detach().requires_grad_(True), de.detach().requires_grad_(True)
        y = fused_selective_scan(fused_short_conv(u, w), de, t["A"], Bm, Cm)
        return (y, *torch.autograd.grad(y.sum(), [u, de]))

    for a, b in zip(run(u, de, Bm, Cm), run(*(v.contiguous() for v in (u, de, Bm, Cm)))):
        assert torch.equal(a, b)


def test_other_stream_and_graph():
    """Calls on a side stream, and a captured forward, backward and token step replayed on new inputs."""
    from dudyconv_b200.state_space import (fused_selective_scan, fused_selective_scan_step, fused_short_conv,
                                           fused_short_conv_step)

    rng = _rng("graph")
    B, D, L, N = 2, 48, 136, 16
    t, _ = _scan_inputs(B, D, L, N, 1, "bf16", rng)
    go, _ = dev(rng.standard_normal((B, D, L)), "bf16")
    w, _ = dev(rng.standard_normal((D, 4)), "bf16")
    cs, _ = dev(rng.standard_normal((B, D, 3)), "bf16")
    h = t.pop("state")
    leaves = [v.requires_grad_(True) for v in (*t.values(), w)]

    def step():
        y = fused_selective_scan(fused_short_conv(t["u"], w), t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"])
        grads = torch.autograd.grad(y, leaves, go)
        with torch.no_grad():
            c = fused_short_conv_step(t["u"][..., 0], cs, w)
            s = fused_selective_scan_step(c, t["delta"][..., 0], t["A"], t["B"][..., 0], t["C"][..., 0], h)
        # no eager graph of the leaves may live while a backward is captured (torch's own rule)
        return [v.detach() for v in (y, *grads, s)]

    cs0, h0 = cs.clone(), h.clone()
    want = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cs.copy_(cs0), h.copy_(h0)
        for a, b in zip(step(), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    cs.copy_(cs0), h.copy_(h0)
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        t["u"].mul_(-0.5)
        go.mul_(2)
    cs.copy_(cs0), h.copy_(h0)
    graph.replay()
    got = [v.clone() for v in got]
    cs.copy_(cs0), h.copy_(h0)
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_lengths_beyond_the_batch_are_clamped():
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv

    rng = _rng("clamp")
    t, _ = _scan_inputs(3, 16, 50, 8, 1, "fp16", rng)
    w, _ = dev(rng.standard_normal((16, 4)), "fp16")
    res = []
    for lengths in ([-5, 1 << 30, 20], [0, 50, 20]):
        n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        res.append([*fused_short_conv(t["u"], w, lengths=n, return_final_state=True),
                    *fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], initial_state=t["state"], lengths=n,
                                          return_final_state=True)])
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_the_same_tensor_twice():
    """u as delta and B as C: each gradient is the sum of its two."""
    from dudyconv_b200.state_space import fused_selective_scan

    rng = _rng("twice")
    t, _ = _scan_inputs(2, 16, 33, 8, 1, "fp32", rng)
    go, _ = dev(rng.standard_normal((2, 16, 33)), "fp32")
    u, b = t["u"].requires_grad_(True), t["B"].requires_grad_(True)
    gu, gb = torch.autograd.grad(fused_selective_scan(u, u, t["A"], b, b), [u, b], go)
    four = [v.detach().clone().requires_grad_(True) for v in (u, u, b, b)]
    g = torch.autograd.grad(fused_selective_scan(four[0], four[1], t["A"], four[2], four[3]), four, go)
    assert torch.equal(gu, g[0] + g[1]) and torch.equal(gb, g[2] + g[3])


def test_two_streams_at_once():
    """Calls that overlap on two streams give what they give alone."""
    from dudyconv_b200.state_space import fused_selective_scan

    rng = _rng("two")
    sets = [_scan_inputs(2, 64, 700, 16, 1, "fp16", rng)[0] for _ in range(2)]

    def run(t):
        u = t["u"].detach().requires_grad_(True)
        y = fused_selective_scan(u, t["delta"], t["A"], t["B"], t["C"], t["skip"], t["delta_bias"])
        return y.detach(), *torch.autograd.grad(y, u, t["delta"])

    want = [run(t) for t in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_c_abi():
    """The C entries with a caller's buffers: results of the torch binding, nothing written beside
    them, and the state of a step in place."""
    from dudyconv_b200 import capi
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv, fused_short_conv_step

    rng = _rng("capi")
    B, D, L, N = 2, 40, 70, 16
    t, _ = _scan_inputs(B, D, L, N, 1, "bf16", rng)
    w, _ = dev(rng.standard_normal((D, 4)), "bf16")

    def guarded(like, *shape):
        buf = torch.full((like.numel() + 128,), 7.0, device="cuda", dtype=like.dtype)
        return buf, buf[64:64 + like.numel()].view(shape or like.shape)

    want, fin = fused_short_conv(t["u"], w, return_final_state=True)
    buf, out = guarded(t["u"])
    fbuf, f = guarded(fin)
    capi.short_conv_forward(t["u"], w, None, None, None, out, f)
    assert torch.equal(out, want) and torch.equal(f, fin)
    assert (buf[:64] == 7).all() and (buf[-64:] == 7).all() and (fbuf[:64] == 7).all() and (fbuf[-64:] == 7).all()
    st = fin.clone()
    o = torch.empty(B, D, device="cuda", dtype=torch.bfloat16)
    capi.short_conv_step(t["u"][..., 0].contiguous(), st, w, None, o)
    st2 = fin.clone()
    assert torch.equal(o, fused_short_conv_step(t["u"][..., 0], st2, w)) and torch.equal(st, st2)
    y, h = fused_selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], return_final_state=True)
    need = capi.selective_scan_forward_workspace_size(t["u"], t["A"], t["B"])
    ws = torch.full((need + 64,), 9, device="cuda", dtype=torch.uint8)
    ybuf, yo = guarded(t["u"])
    ck = torch.full((capi.selective_scan_checkpoint_bytes(t["u"], t["A"], t["B"]) + 64,), 9, device="cuda", dtype=torch.uint8)
    capi.selective_scan_forward(t["u"], t["delta"], t["A"], t["B"], t["C"], None, None, None, None, yo, None, ck, ws)
    assert torch.equal(yo, y) and (ybuf[:64] == 7).all() and (ybuf[-64:] == 7).all()
    assert (ws[need:] == 9).all() and (ck[-64:] == 9).all()
    if need:
        with pytest.raises(capi.DudyError, match="workspace too small"):
            capi.selective_scan_forward(t["u"], t["delta"], t["A"], t["B"], t["C"], None, None, None, None, yo, None, None,
                                        ws[:need - 1])
    assert capi.device_error() == 0


def test_offsets_beyond_32_bits():
    """Rows behind the 2^31st element: the last channels of a large batch against the same rows alone."""
    from dudyconv_b200.state_space import fused_selective_scan, fused_short_conv

    B, D, L, N = 2, 1028, (1 << 20) + 8, 2
    assert B * D * L > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.randn(B, D, L, device="cuda", generator=g, dtype=torch.bfloat16)
    w = torch.randn(D, 4, device="cuda", generator=g, dtype=torch.bfloat16)
    A = -torch.rand(D, N, device="cuda", generator=g)
    bc = torch.randn(B, 1, N, L, device="cuda", generator=g, dtype=torch.bfloat16)
    tail = slice(D - 4, D)
    c = fused_short_conv(u, w)
    assert torch.equal(c[1:, tail], fused_short_conv(u[1:, tail], w[tail]))
    y, h = fused_selective_scan(c, u, A, bc, bc, return_final_state=True)
    y1, h1 = fused_selective_scan(c[1:, tail], u[1:, tail], A[tail], bc[1:], bc[1:], return_final_state=True)
    # another split of the sequence may round the states differently: the bound of 16-bit outputs
    assert (y[1:, tail].float() - y1.float()).abs().max() <= 2 ** -7 * y1.float().abs().max()
    assert (h[1:, tail] - h1).abs().max() <= 2 ** -12 * h1.abs().max()


def test_refusals():
    from dudyconv_b200 import state_space as sp

    x = torch.zeros(2, 4, 8, device="cuda", dtype=torch.float16)
    w = torch.zeros(4, 4, device="cuda", dtype=torch.float16)
    A = torch.zeros(4, 3, device="cuda")
    bc = torch.zeros(2, 1, 3, 8, device="cuda", dtype=torch.float16)
    st = torch.zeros(2, 4, 3, device="cuda")
    i32 = torch.zeros(2, device="cuda", dtype=torch.int32)
    cases = [
        (lambda: sp.fused_short_conv(x[0], w), r"x must be \[B,D,L\]"),
        (lambda: sp.fused_short_conv(x[..., :0], w), "must be positive"),
        (lambda: sp.fused_short_conv(x, w[:, :1]), "S must be between 2 and 8"),
        (lambda: sp.fused_short_conv(x, w.repeat(1, 3)), "S must be between 2 and 8"),
        (lambda: sp.fused_short_conv(x, w.float()), "weight must be Half"),
        (lambda: sp.fused_short_conv(x, w[:3]), "weight must be"),
        (lambda: sp.fused_short_conv(x, w, lengths=i32.long()), "lengths must be Int"),
        (lambda: sp.fused_short_conv(x, w, lengths=i32[:1]), "lengths must be"),
        (lambda: sp.fused_short_conv(x, w, initial_state=x[..., :2]), "initial_state must be"),
        (lambda: sp.fused_short_conv(x, w.cpu()), "weight must be CUDA tensor"),
        (lambda: sp.fused_short_conv(x, w, activation="gelu"), "activation must be"),
        (lambda: sp.fused_short_conv(x.int(), w.int()), "Unsupported dtype"),
        (lambda: sp.fused_short_conv_step(x[..., 0], x[..., ::3], w), "conv_state must be contiguous"),
        (lambda: sp.fused_short_conv_step(x[..., 0], x[..., :3].float(), w), "conv_state must be Half"),
        (lambda: sp.fused_short_conv_step(x[..., 0].requires_grad_(True), x[..., :3].contiguous(), w), "no backward"),
        (lambda: sp.fused_selective_scan(x, x, A, bc, bc[:, :, :2]), "C must be"),
        (lambda: sp.fused_selective_scan(x, x, A.half(), bc, bc), "A must be Float"),
        (lambda: sp.fused_selective_scan(x, x, torch.zeros(4, 65, device="cuda"), bc, bc), "N must be between 1 and 64"),
        (lambda: sp.fused_selective_scan(x, x, A, bc.repeat(1, 3, 1, 1), bc.repeat(1, 3, 1, 1)), "multiple of the number of groups"),
        (lambda: sp.fused_selective_scan(x, x, A, bc, bc, skip=w[0]), "skip must be Float"),
        (lambda: sp.fused_selective_scan(x, x, A, bc, bc, initial_state=st.half()), "initial_state must be Float"),
        (lambda: sp.fused_selective_scan_step(x[..., 0], x[..., 0], A, bc[..., 0], bc[..., 0], st.half()), "state must be Float"),
        (lambda: sp.fused_selective_scan_step(x[..., 0], x[..., 0], A, bc[..., 0], bc[..., 0], st.transpose(0, 1).contiguous().transpose(0, 1)), "state must be contiguous"),
    ]
    for call, msg in cases:
        with pytest.raises(RuntimeError, match=msg):
            call()
    u = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        torch.autograd.grad(sp.fused_short_conv(u, w).sum(), u, create_graph=True)


def test_modules():
    from dudyconv_b200.state_space import FusedSelectiveScan1d, FusedShortConv1d

    torch.manual_seed(0)
    conv = FusedShortConv1d(16, device="cuda")
    scan = FusedSelectiveScan1d(16, 8, device="cuda")
    x = torch.randn(2, 16, 12, device="cuda", dtype=torch.bfloat16)
    bc = torch.randn(2, 8, 12, device="cuda", dtype=torch.bfloat16)
    c, cs = conv(x, return_final_state=True)
    y, h = scan(c, x, bc, bc, return_final_state=True)
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == p.dtype for m in (conv, scan) for p in m.parameters())
    s = scan.step(conv.step(x[..., 0], cs.detach()), x[..., 0], bc[..., 0], bc[..., 0], h.detach())
    assert s.shape == (2, 16) and not s.requires_grad
