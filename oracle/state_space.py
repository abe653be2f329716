"""float64 formulas of the state-space block: short causal conv, selective scan, and the norms,
gate and residual between blocks, with their gradients. Test infrastructure only.

Each function takes float64 arrays in the operators' layouts. ``mag=True`` gives, in the place of
a result, the sum of the magnitudes of the terms that make it up (every input and every term
taken positive): what the rounding errors of its evaluation are proportional to.
"""

from __future__ import annotations

import numpy as np


def sigmoid(v):
    return 0.5 * (1.0 + np.tanh(0.5 * v))


def _ends(lengths, B, L):
    n = np.full(B, L) if lengths is None else np.clip(np.asarray(lengths), 0, L)
    return n, np.arange(L)[None, :] < n[:, None]


def short_conv(x, w, bias=None, state=None, lengths=None, silu=True, go=None, gfinal=None,
               mag=False):
    """out, final_state and, with ``go``, grad_x, grad_w, grad_bias, grad_state."""
    B, D, L = x.shape
    S = w.shape[1]
    n, inside = _ends(lengths, B, L)
    x = np.where(inside[:, None], x, 0.0)
    state = np.zeros((B, D, S - 1)) if state is None else state
    bias = np.zeros(D) if bias is None else bias
    # the activation's slope is taken at the true v, also where magnitudes are asked for
    v = bias[None, :, None] + _taps(np.concatenate([state, x], 2), w, L)
    if mag:
        x, w, bias, state = np.abs(x), np.abs(w), np.abs(bias), np.abs(state)
        go = None if go is None else np.abs(go)
        gfinal = None if gfinal is None else np.abs(gfinal)
    xe = np.concatenate([state, x], 2)
    if mag:
        vm = bias[None, :, None] + _taps(xe, w, L)
        out = vm * 1.1 if silu else vm
    else:
        out = v * sigmoid(v) if silu else v
    out = np.where(inside[:, None], out, 0.0)
    final = np.stack([xe[b, :, n[b]:n[b] + S - 1] for b in range(B)])
    if go is None:
        return out, final
    s = sigmoid(v)
    slope = s * (1 + v * (1 - s)) if silu else np.ones_like(v)
    if mag:  # |slope| <= 1.1 and |slope'| <= 0.5 times the error of v
        slope = 1.1 + 0.5 * vm if silu else slope
    dv = np.where(inside[:, None], go * slope, 0.0)
    dxe = np.zeros_like(xe)
    gw = np.zeros_like(w)
    for j in range(S):
        dxe[:, :, j:j + L] += w[None, :, j, None] * dv
        gw[:, j] = (dv * xe[:, :, j:j + L]).sum((0, 2))
    if gfinal is not None:
        for b in range(B):
            dxe[b, :, n[b]:n[b] + S - 1] += gfinal[b]
    return out, final, dxe[:, :, S - 1:], gw, dv.sum((0, 2)), dxe[:, :, :S - 1]


def _taps(xe, w, L):
    return sum(w[None, :, j, None] * xe[:, :, j:j + L] for j in range(w.shape[1]))


def selective_scan(u, delta, A, Bm, Cm, skip=None, delta_bias=None, softplus=True, state=None,
                   lengths=None, go=None, gfinal=None, mag=False):
    """y, final_state and, with ``go``, the gradients of u, delta, A, B, C, skip, delta_bias and
    state."""
    B, D, L = u.shape
    N, G = A.shape[1], Bm.shape[1]
    n, inside = _ends(lengths, B, L)
    raw = delta + (0.0 if delta_bias is None else delta_bias[None, :, None])
    raw = np.where(inside[:, None], raw, 0.0)
    dt = np.logaddexp(raw, 0.0) if softplus else raw
    dt = np.where(inside[:, None], dt, 0.0)
    slope = np.where(inside[:, None], sigmoid(raw) if softplus else 1.0, 0.0)
    u = np.where(inside[:, None], u, 0.0)
    wide = lambda m: np.repeat(np.where(inside[:, None, None], m, 0.0), D // G, axis=1)  # noqa: E731
    Bw, Cw = wide(Bm), wide(Cm)
    skip = np.zeros(D) if skip is None else skip
    h = np.zeros((B, D, N)) if state is None else state
    As, step = A, dt
    if mag:
        u, Bw, Cw, skip, h, As, step = (np.abs(t) for t in (u, Bw, Cw, skip, h, A, dt))
        go = None if go is None else np.abs(go)
        gfinal = None if gfinal is None else np.abs(gfinal)
    dec = lambda t: np.exp(dt[:, :, t, None] * A)  # noqa: E731
    hs, y = [h], np.zeros((B, D, L))
    for t in range(L):
        h = dec(t) * h + (step[:, :, t] * u[:, :, t])[..., None] * Bw[..., t]
        hs.append(h)
        y[:, :, t] = (h * Cw[..., t]).sum(2) + skip * u[:, :, t]
    y = np.where(inside[:, None], y, 0.0)
    if go is None:
        return y, h
    go = np.where(inside[:, None], go, 0.0)
    r = np.zeros((B, D, N)) if gfinal is None else gfinal.copy()
    gu, gdt, gA = np.zeros_like(u), np.zeros_like(u), np.zeros_like(A)
    gB, gC = np.zeros((B, G, N, L)), np.zeros((B, G, N, L))
    heads = lambda v: v.reshape(B, G, D // G, N).sum(2)  # noqa: E731
    for t in reversed(range(L)):
        g = Cw[..., t] * go[:, :, t, None] + r
        gC[..., t] = heads(hs[t + 1] * go[:, :, t, None])
        gB[..., t] = heads(g * (step[:, :, t] * u[:, :, t])[..., None])
        r = dec(t) * g
        moved = r * hs[t]
        gA += (moved * step[:, :, t, None]).sum(0)
        through = (g * Bw[..., t]).sum(2)
        gdt[:, :, t] = through * u[:, :, t] + (moved * As).sum(2)
        gu[:, :, t] = through * step[:, :, t] + skip * go[:, :, t]
    gdelta = gdt * slope
    keep = inside[:, None]
    gu, gdelta = np.where(keep, gu, 0.0), np.where(keep, gdelta, 0.0)
    gB, gC = (np.where(inside[:, None, None], v, 0.0) for v in (gB, gC))
    return (y, h, gu, gdelta, gA, gB, gC, (go * u).sum((0, 2)), gdelta.sum((0, 2)), r)


def block_norm(x, residual, w1, w2, gate=None, scale=None, b1=None, b2=None, layer=False,
               eps=1e-5, gy=None, gr=None, mag=False):
    """y, residual_out and, with ``gy``, the gradients of x, residual, gate, post_weight,
    post_bias, scale, pre_weight and pre_bias. ``mag``: the sums' magnitudes (parameters only)."""
    D = x.shape[1]
    col = lambda p, other: np.full((D, 1), other) if p is None else p[:, None]  # noqa: E731
    w1, w2, b1, b2, sc = col(w1, 1.0), col(w2, 1.0), col(b1, 0.0), col(b2, 0.0), col(scale, 1.0)
    s = None if gate is None else sigmoid(gate)
    g = x if gate is None else x * gate * s

    def normed(v):
        c = v - v.mean(1, keepdims=True) if layer else v
        inv = 1.0 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
        return c * inv, inv

    def back(d, hat, inv):
        out = d - hat * (d * hat).mean(1, keepdims=True)
        return inv * (out - d.mean(1, keepdims=True) if layer else out)

    hat1, inv1 = normed(g)
    p = hat1 * w1 + b1
    rout = residual + sc * p
    hat2, inv2 = normed(rout)
    y = hat2 * w2 + b2
    if gy is None:
        return y, rout
    dr = back(gy * w2, hat2, inv2) + (0.0 if gr is None else gr)
    dp = dr * sc
    dg = back(dp * w1, hat1, inv1)
    gx = dg if gate is None else dg * gate * s
    ggate = None if gate is None else dg * x * s * (1 + gate * (1 - s))
    total = (lambda v: np.abs(v).sum((0, 2))) if mag else (lambda v: v.sum((0, 2)))
    return (y, rout, gx, dr, ggate, total(dp * hat1), total(dp), total(dr * p), total(gy * hat2),
            total(gy))
