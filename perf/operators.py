"""The state-space block's operators as a user's program calls them, each beside its plain form.

Three operators of the `[B, D, L]` layout (batch, channels, positions) that the dynamic conv uses:

* the short causal depthwise conv with SiLU (`fused_short_conv`, one token: `fused_short_conv_step`),
* the selective state space scan (`fused_selective_scan`, one token: `fused_selective_scan_step`),
* the norms after and before a block with its gate, residual and residual scale
  (`fused_gated_residual_norm`).

`own` chooses between the plain form (elementary torch operations in 32 bits, rounded once) and
the package's kernels. Modes of a case: "train" is forward and backward, "prompt" a forward from
a carried state over a padded batch (the norm: forward alone), "step" one new token per sequence
with the state updated in place.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # decoding: eight sequences, one new token each
        {"name": "conv_step", "op": "conv", "mode": "step", "B": 8, "D": 256, "S": 4, "dtype": "fp16"},
        # five prompts of different lengths in one padded batch of odd length
        {"name": "conv_prompt", "op": "conv", "mode": "prompt", "B": 5, "D": 256, "L": 1001, "S": 4, "dtype": "bf16"},
        # a training step at the benchmark's batch and sequence length
        {"name": "conv_train", "op": "conv", "mode": "train", "B": 16, "D": 256, "L": 4096, "S": 4, "dtype": "fp16"},
        # decoding, as above
        {"name": "scan_step", "op": "scan", "mode": "step", "B": 8, "D": 256, "N": 16, "G": 1, "dtype": "fp16"},
        # one long prompt alone: few rows, a long axis
        {"name": "scan_prompt_one", "op": "scan", "mode": "prompt", "B": 1, "D": 256, "L": 4096, "N": 16, "G": 1, "dtype": "bf16"},
        # a padded batch of prompts in 32 bits
        {"name": "scan_prompt_ragged", "op": "scan", "mode": "prompt", "B": 5, "D": 256, "L": 1001, "N": 16, "G": 1, "dtype": "fp32"},
        # a training step at the benchmark's batch and sequence length
        {"name": "scan_train", "op": "scan", "mode": "train", "B": 16, "D": 256, "L": 4096, "N": 16, "G": 1, "dtype": "fp16"},
        # a small model with two groups of channels, an odd length and a small state
        {"name": "scan_train_odd", "op": "scan", "mode": "train", "B": 3, "D": 192, "L": 777, "N": 8, "G": 2, "dtype": "bf16"},
        # one 256-token chunk of training in 32 bits with a wide state
        {"name": "scan_train_chunk", "op": "scan", "mode": "train", "B": 4, "D": 128, "L": 256, "N": 32, "G": 1, "dtype": "fp32"},
        # decoding: one token of 64 sequences
        {"name": "norm_step", "op": "norm", "mode": "prompt", "B": 64, "D": 256, "L": 1, "norm": "rms", "wide": False, "dtype": "bf16"},
        # a training step at the benchmark's batch and sequence length
        {"name": "norm_train", "op": "norm", "mode": "train", "B": 16, "D": 256, "L": 4096, "norm": "rms", "wide": False, "dtype": "fp16"},
        # layer norms, a 32-bit residual stream, odd channels and length
        {"name": "norm_train_odd", "op": "norm", "mode": "train", "B": 3, "D": 300, "L": 777, "norm": "layer", "wide": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    mode = rng.choice(["train", "prompt", "step"] if op != "norm" else ["train", "prompt"])
    case = {"op": op, "mode": mode, "dtype": rng.choice(["fp32", "fp16", "bf16"])}
    if mode == "step":
        case |= {"B": _log_int(rng, 1, 256), "D": _log_int(rng, 64, 1024)}
    else:
        case |= {"B": _log_int(rng, 1, 16), "D": _log_int(rng, 64, 512), "L": _log_int(rng, 1, 4096)}
        if op == "norm" and mode == "prompt" and rng.random() < 0.3:
            case["L"] = 1
    if op == "conv":
        case["S"] = rng.choice([2, 3, 4, 4, 4, 5, 8])
    if op == "scan":
        case["G"] = rng.choice([1, 1, 1, 2, 4])
        case["D"] = -(-case["D"] // case["G"]) * case["G"]
        case["N"] = _log_int(rng, 4, 64)
    if op == "norm":
        case |= {"norm": rng.choice(["rms", "rms", "layer"]), "wide": case["dtype"] != "fp32" and rng.random() < 0.3}
    if mode != "step":  # no more work than the largest listed case of the operator
        most = 16 * 256 * 4096 * (16 if op == "scan" else 1)
        row = case["B"] * case["D"] * case.get("N", 1) * (2 if case["dtype"] == "fp32" else 1) * (2 if case.get("wide") else 1)
        case["L"] = max(1, min(case["L"], most // row))
    return case


# ---- inputs --------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, device="cuda", generator=g) * (hi - lo) + lo

    B, D = case["B"], case["D"]
    mode, s = case["mode"], {"case": dict(case)}
    L = case.get("L", 1)
    seq = (B, D) if mode == "step" else (B, D, L)
    if mode == "prompt" and case["op"] != "norm":  # one prompt fills the batch's length, the others are padded to it
        s["lengths"] = torch.maximum((uniform(0.3, 1.0, B) * L).to(torch.int32), torch.tensor(1, device="cuda", dtype=torch.int32))
        s["lengths"][-1:] = L
    if case["op"] == "conv":
        S = case["S"]
        s |= {"x": normal(*seq), "weight": normal(D, S, scale=S ** -0.5), "bias": normal(D, scale=0.1)}
        if mode != "train":
            s["state"] = normal(B, D, S - 1)
        leaves = ["x", "weight", "bias"]
    elif case["op"] == "scan":
        N, G = case["N"], case["G"]
        bc = (B, G, N) if mode == "step" else (B, G, N, L)
        # steps of 1e-3 to 1e-1 behind the softplus, decay rates of 1 to N
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))
        rate = torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(D, 1)
        s |= {"u": normal(*seq), "delta": normal(*seq, scale=0.5), "A": -rate * torch.exp(normal(D, N, scale=0.1, dtype=torch.float32)),
              "Bm": normal(*bc), "Cm": normal(*bc), "skip": 1 + normal(D, scale=0.1, dtype=torch.float32),
              "delta_bias": step + torch.log(-torch.expm1(-step))}
        if mode != "train":
            s["state"] = normal(B, D, N, dtype=torch.float32, scale=0.3)
        leaves = ["u", "delta", "A", "Bm", "Cm", "skip", "delta_bias"]
    else:
        wide = torch.float32 if case["wide"] else dt
        s |= {"x": normal(*seq), "gate": normal(*seq), "residual": normal(*seq, scale=2.0, dtype=wide),
              "post_weight": 1 + normal(D, scale=0.1), "pre_weight": 1 + normal(D, scale=0.1), "scale": normal(D, scale=0.3)}
        leaves = ["x", "gate", "residual", "post_weight", "pre_weight", "scale"]
        if case["norm"] == "layer":
            s |= {"post_bias": normal(D, scale=0.1), "pre_bias": normal(D, scale=0.1)}
            leaves += ["post_bias", "pre_bias"]
    if mode == "train":
        s["leaves"] = leaves
        s["grad"] = normal(*seq)
        if case["op"] == "norm":
            s["grad_residual"] = normal(*seq, dtype=s["residual"].dtype)
        for name in leaves:
            s[name].requires_grad_(True)
    return s


# ---- the package's calls -------------------------------------------------------------------


def run(s):
    case = s["case"]
    op, mode = case["op"], case["mode"]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "norm": _own_norm}[op](s, mode, case)
    with torch.no_grad():
        return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[op](s, mode, case)


def _own_conv(s, mode, case):
    from dudyconv_b200.state_space import fused_short_conv, fused_short_conv_step

    if mode == "step":
        return fused_short_conv_step(s["x"], s["state"], s["weight"], s["bias"]), s["state"]
    if mode == "prompt":
        return fused_short_conv(s["x"], s["weight"], s["bias"], initial_state=s["state"], lengths=s["lengths"], return_final_state=True)
    out = fused_short_conv(s["x"], s["weight"], s["bias"])
    return (out, *torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["grad"]))


def _own_scan(s, mode, case):
    from dudyconv_b200.state_space import fused_selective_scan, fused_selective_scan_step

    if mode == "step":
        y = fused_selective_scan_step(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["state"], skip=s["skip"], delta_bias=s["delta_bias"])
        return y, s["state"]
    if mode == "prompt":
        return fused_selective_scan(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], skip=s["skip"], delta_bias=s["delta_bias"],
                                    initial_state=s["state"], lengths=s["lengths"], return_final_state=True)
    y = fused_selective_scan(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], skip=s["skip"], delta_bias=s["delta_bias"])
    return (y, *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["grad"]))


def _own_norm(s, mode, case):
    from dudyconv_b200.block_norm import fused_gated_residual_norm

    y, r = fused_gated_residual_norm(s["x"], s["residual"], s["post_weight"], s["pre_weight"], gate=s["gate"], scale=s["scale"],
                                     post_bias=s.get("post_bias"), pre_bias=s.get("pre_bias"), norm=case["norm"], eps=EPS)
    if mode == "prompt":
        return y, r
    return (y, r, *torch.autograd.grad((y, r), [s[k] for k in s["leaves"]], (s["grad"], s["grad_residual"])))


# ---- plain forms ---------------------------------------------------------------------------


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _inside(s, L):
    """Positions before each sequence's length, [B, 1, L]; None where all are."""
    if "lengths" not in s:
        return None
    return (torch.arange(L, device="cuda")[None] < s["lengths"][:, None])[:, None]


def _plain_conv(s, mode, case):
    x, dt = s["x"], s["x"].dtype
    w, bias, S = s["weight"].float(), s["bias"].float(), case["S"]
    if mode == "step":
        ext = torch.cat([s["state"].float(), x.float()[:, :, None]], 2)
        v = (ext * w).sum(2) + bias
        s["state"].copy_(ext[:, :, 1:])
        return (v * _sigmoid(v)).to(dt), s["state"]
    B, D, L = x.shape
    inside = _inside(s, L)
    xf = x.float() if inside is None else torch.where(inside, x.float(), 0.0)
    before = s["state"].float() if "state" in s else xf.new_zeros(B, D, S - 1)
    ext = torch.cat([before, xf], 2)
    v = bias[:, None] + sum(w[:, j, None] * ext[:, :, j:j + L] for j in range(S))
    sig = _sigmoid(v)
    out = v * sig
    if mode == "prompt":
        at = s["lengths"].long()[:, None, None] + torch.arange(S - 1, device="cuda")
        return torch.where(inside, out, 0.0).to(dt), ext.gather(2, at.expand(B, D, S - 1)).to(dt)
    dv = s["grad"].float() * sig * (1 + v * (1 - sig))
    dext = sum(torch.nn.functional.pad(w[:, j, None] * dv, (j, S - 1 - j)) for j in range(S))
    dw = torch.stack([(dv * ext[:, :, j:j + L]).sum((0, 2)) for j in range(S)], 1)
    return out.to(dt), dext[:, :, S - 1:].to(dt), dw.to(dt), dv.sum((0, 2)).to(dt)


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the last axis from h = 0: pairs of steps joined, then fours, and so on."""
    span, L = 1, a.shape[-1]
    while span < L:
        b = torch.cat([b[..., :span], b[..., span:] + a[..., span:] * b[..., :-span]], -1)
        a = torch.cat([a[..., :span], a[..., span:] * a[..., :-span]], -1)
        span *= 2
    return b


def _plain_scan(s, mode, case):
    dtype = s["u"].dtype
    B, D, N, G = case["B"], case["D"], case["N"], case["G"]
    L, R = case.get("L", 1), D // G
    A = s["A"].reshape(G, R, N, 1)
    skip = s["skip"][:, None]
    u, raw = s["u"].float().reshape(B, D, L), s["delta"].float().reshape(B, D, L) + s["delta_bias"][:, None]
    Bm, Cm = (s[k].float().reshape(B, G, 1, N, L) for k in ("Bm", "Cm"))
    dt = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    inside = _inside(s, L)
    if inside is not None:
        u, dt, Bm, Cm = (torch.where(m, v, 0.0) for m, v in ((inside, u), (inside, dt), (inside[:, None, None], Bm), (inside[:, None, None], Cm)))

    def heads(v):
        return v.reshape(B, G, R, 1, L)

    a = torch.exp(heads(dt) * A)
    b = heads(dt * u) * Bm
    h0 = s["state"].reshape(B, G, R, N) if "state" in s else None
    if h0 is not None:
        b[..., 0] += a[..., 0] * h0
    h = _recurrence(a, b)
    del b
    y = (h * Cm).sum(3).reshape(B, D, L) + skip * u
    if mode == "step":
        s["state"].copy_(h[..., -1].reshape(B, D, N))
        return y.reshape(B, D).to(dtype), s["state"]
    if mode == "prompt":
        return y.to(dtype), h[..., -1].reshape(B, D, N)
    dy = s["grad"].float()
    dC = (h * heads(dy)).sum(2)
    down = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1)  # the decay between a step and the next
    g = _recurrence(down.flip(-1), (heads(dy) * Cm).flip(-1)).flip(-1)
    del down
    dB = (g * heads(dt * u)).sum(2)
    through = (g * Bm).sum(3).reshape(B, D, L)
    g *= a
    g[..., 1:] *= h[..., :-1]
    g[..., 0] = 0
    dA = (g * heads(dt)).sum((0, 4)).reshape(D, N)
    ddt = u * through + (g * A).sum(3).reshape(B, D, L)
    dlogit = ddt * _sigmoid(raw)
    du = dt * through + skip * dy
    return (y.to(dtype), du.to(dtype), dlogit.to(dtype), dA, dB.to(dtype), dC.to(dtype), (dy * u).sum((0, 2)), dlogit.sum((0, 2)))


def _plain_norm(s, mode, case):
    layer, dt = case["norm"] == "layer", s["x"].dtype
    p = {k: s[k].float()[:, None] for k in ("post_weight", "pre_weight", "scale", "post_bias", "pre_bias") if k in s}
    x, z, r = s["x"].float(), s["gate"].float(), s["residual"].float()

    def normed(v):
        c = v - v.mean(1, keepdim=True) if layer else v
        inv = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
        return c * inv, inv

    def back(d, hat, inv):
        out = d - hat * (d * hat).mean(1, keepdim=True)
        return inv * (out - d.mean(1, keepdim=True) if layer else out)

    sig = _sigmoid(z)
    hat1, inv1 = normed(x * z * sig)
    post = hat1 * p["post_weight"] + p.get("post_bias", 0.0)
    rout = r + p["scale"] * post
    hat2, inv2 = normed(rout)
    y = hat2 * p["pre_weight"] + p.get("pre_bias", 0.0)
    if mode == "prompt":
        return y.to(dt), rout.to(s["residual"].dtype)
    dy = s["grad"].float()
    dr = s["grad_residual"].float() + back(dy * p["pre_weight"], hat2, inv2)
    dpost = dr * p["scale"]
    dg = back(dpost * p["post_weight"], hat1, inv1)
    grads = [(dg * z * sig).to(dt), (dg * x * sig * (1 + z * (1 - sig))).to(dt), dr.to(s["residual"].dtype),
             (dpost * hat1).sum((0, 2)).to(dt), (dy * hat2).sum((0, 2)).to(dt), (dr * post).sum((0, 2)).to(dt)]
    if layer:
        grads += [dpost.sum((0, 2)).to(dt), dy.sum((0, 2)).to(dt)]
    return (y.to(dt), rout.to(s["residual"].dtype), *grads)


# ---- what has to move and be computed ------------------------------------------------------


def work(case):
    B, D, L, mode = case["B"], case["D"], case.get("L", 1), case["mode"]
    es = 4 if case["dtype"] == "fp32" else 2
    rows = B * D * L
    if case["op"] == "conv":
        S = case["S"]
        if mode == "train":  # x and the gradient in, the output and x's gradient out
            return {"bytes": es * (4 * rows + 2 * D * (S + 1)), "flops": rows * (6 * S + 12)}
        return {"bytes": es * (2 * rows + 2 * B * D * (S - 1) + D * (S + 1)), "flops": rows * (2 * S + 5)}
    if case["op"] == "scan":
        N, G = case["N"], case["G"]
        bc, par = 2 * B * G * N * L, D * (N + 2)
        if mode == "train":  # u, delta, the gradient and B, C in; y and the gradients out
            return {"bytes": es * (6 * rows + 2 * bc) + 8 * par, "flops": rows * (N * 27 + 20)}
        return {"bytes": es * (3 * rows + bc) + 4 * (2 * B * D * N + par), "flops": rows * (N * 7 + 8)}
    rs = 4 if case["wide"] else es
    if mode == "train":  # x, gate, residual and both gradients in; two outputs and three gradients out
        return {"bytes": rows * (6 * es + 4 * rs) + 8 * D * es, "flops": rows * 60}
    return {"bytes": rows * (3 * es + 2 * rs) + 3 * D * es, "flops": rows * 20}


# ---- 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](s, case)


def _leaf(t):
    return t.detach().double().requires_grad_(True)


def _exact_conv(s, case):
    S, D, mode = case["S"], case["D"], case["mode"]
    x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
    seq = x[:, :, None] if mode == "step" else x
    B, _, L = seq.shape
    first = s["state"].double() if "state" in s else seq.new_zeros(B, D, S - 1)
    ext = torch.cat([first, seq], 2)
    v = (ext.unfold(2, S, 1) * w[:, None]).sum(3) + b[:, None]
    out = torch.nn.functional.silu(v)
    if mode == "step":
        return out[:, :, 0].detach(), ext[:, :, 1:].detach()
    if mode == "prompt":
        ends = s["lengths"].tolist()
        return (torch.stack([torch.cat([o[:, :n], torch.zeros_like(o[:, n:])], 1) for o, n in zip(out.detach(), ends)]),
                torch.stack([e[:, n:n + S - 1] for e, n in zip(ext.detach(), ends)]))
    return (out.detach(), *torch.autograd.grad(out, [x, w, b], s["grad"].double()))


def _exact_scan(s, case):
    B, D, N, G, mode = case["B"], case["D"], case["N"], case["G"], case["mode"]
    L = case.get("L", 1)
    u, raw = (s[k].detach().double().reshape(B, D, L) for k in ("u", "delta"))
    A, skip = s["A"].detach().double(), s["skip"].detach().double()
    raw = raw + s["delta_bias"].detach().double()[:, None]
    Bm, Cm = (s[k].detach().double().reshape(B, G, N, L) for k in ("Bm", "Cm"))
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    h = s["state"].double() if "state" in s else u.new_zeros(B, D, N)
    ends = s["lengths"].long()[:, None, None] if "lengths" in s else None
    wide = lambda m, t: m[..., t].repeat_interleave(D // G, 1)  # noqa: E731
    states, ys = [h], []
    for t in range(L):
        new = torch.exp(dt[:, :, t, None] * A) * h + (dt[:, :, t] * u[:, :, t])[:, :, None] * wide(Bm, t)
        y = (new * wide(Cm, t)).sum(2) + skip * u[:, :, t]
        if ends is not None:
            new, y = torch.where(t < ends, new, h), torch.where(t < ends[:, 0], y, 0.0)
        h = new
        ys.append(y)
        if mode == "train":
            states.append(h)
    y = torch.stack(ys, 2)
    if mode == "step":
        return y.reshape(B, D), h
    if mode == "prompt":
        return y, h
    dy = s["grad"].double()
    du, ddt, dA = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(A)
    dB, dC = torch.zeros_like(Bm), torch.zeros_like(Cm)
    later = torch.zeros_like(h)
    for t in reversed(range(L)):
        decay, x, go = torch.exp(dt[:, :, t, None] * A), u[:, :, t, None], dy[:, :, t, None]
        g = wide(Cm, t) * go + later
        dC[..., t] = (states[t + 1] * go).reshape(B, G, D // G, N).sum(2)
        dB[..., t] = (g * dt[:, :, t, None] * x).reshape(B, G, D // G, N).sum(2)
        later = decay * g
        moved = later * states[t]
        dA += (moved * dt[:, :, t, None]).sum(0)
        into = (g * wide(Bm, t)).sum(2)
        ddt[:, :, t] = into * u[:, :, t] + (moved * A).sum(2)
        du[:, :, t] = into * dt[:, :, t] + skip * dy[:, :, t]
    ddelta = ddt * torch.sigmoid(raw)
    return y, du, ddelta, dA, dB, dC, (dy * u).sum((0, 2)), ddelta.sum((0, 2))


def _exact_norm(s, case):
    names = ["x", "gate", "residual", "post_weight", "pre_weight", "scale"] + (["post_bias", "pre_bias"] if case["norm"] == "layer" else [])
    v = {k: _leaf(s[k]) for k in names}
    last = lambda t: t.transpose(1, 2)  # noqa: E731

    def norm(t, w, b):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(t, (case["D"],), w, b, EPS)
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w

    post = norm(last(v["x"] * torch.nn.functional.silu(v["gate"])), v["post_weight"], v.get("post_bias"))
    rout = last(v["residual"]) + v["scale"] * post
    y, rout = last(norm(rout, v["pre_weight"], v.get("pre_bias"))), last(rout)
    if case["mode"] == "prompt":
        return y.detach(), rout.detach()
    return (y.detach(), rout.detach(), *torch.autograd.grad((y, rout), [v[k] for k in names], (s["grad"].double(), s["grad_residual"].double())))
