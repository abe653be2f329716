"""The float64 formulas of the state-space block against themselves: their gradients against
central differences, a sequence against its chunks, and a padded batch against its sequences."""

import numpy as np
import pytest

from oracle import state_space as ss


def _diff(f, arrays, k, eps=1e-6):
    g = np.zeros_like(arrays[k])
    it = np.nditer(arrays[k], flags=["multi_index"])
    for _ in it:
        i = it.multi_index
        up, down = [a.copy() for a in arrays], [a.copy() for a in arrays]
        up[k][i] += eps
        down[k][i] -= eps
        g[i] = (f(*up) - f(*down)) / (2 * eps)
    return g


@pytest.mark.parametrize("lengths", [None, [3, 0]])
@pytest.mark.parametrize("S,silu", [(2, True), (4, True), (3, False)])
def test_short_conv_gradients(S, silu, lengths):
    rng = np.random.default_rng(1)
    B, D, L = 2, 2, 5
    x, w, b, st = (rng.standard_normal(s) for s in ((B, D, L), (D, S), (D,), (B, D, S - 1)))
    go, gf = rng.standard_normal((B, D, L)), rng.standard_normal((B, D, S - 1))

    def loss(x, w, b, st):
        o, f = ss.short_conv(x, w, b, st, lengths, silu)
        return (o * go).sum() + (f * gf).sum()

    got = ss.short_conv(x, w, b, st, lengths, silu, go, gf)[2:]
    for k in range(4):
        np.testing.assert_allclose(got[k], _diff(loss, [x, w, b, st], k), atol=1e-7)


@pytest.mark.parametrize("lengths", [None, [2, 4]])
@pytest.mark.parametrize("G,softplus", [(1, True), (2, True), (2, False)])
def test_selective_scan_gradients(G, softplus, lengths):
    rng = np.random.default_rng(2)
    B, D, L, N = 2, 4, 4, 3
    u, de = rng.standard_normal((2, B, D, L))
    A = -np.exp(rng.standard_normal((D, N)))
    Bm, Cm = rng.standard_normal((2, B, G, N, L))
    sk, db = rng.standard_normal((2, D))
    if not softplus:
        de, db = 0.1 + np.abs(de), np.abs(db)
    st, gf = rng.standard_normal((2, B, D, N))
    go = rng.standard_normal((B, D, L))
    args = [u, de, A, Bm, Cm, sk, db, st]

    def loss(u, de, A, Bm, Cm, sk, db, st):
        y, h = ss.selective_scan(u, de, A, Bm, Cm, sk, db, softplus, st, lengths)
        return (y * go).sum() + (h * gf).sum()

    got = ss.selective_scan(*args[:7], softplus, st, lengths, go, gf)[2:]
    for k in range(8):
        np.testing.assert_allclose(got[k], _diff(loss, args, k), atol=2e-7, rtol=1e-5)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("full", [False, True])
def test_block_norm_gradients(layer, full):
    rng = np.random.default_rng(3)
    B, D, L = 2, 3, 2
    x, r, z, gy, gr = rng.standard_normal((5, B, D, L))
    p = rng.standard_normal((5, D))
    args = [x, r, z, *p] if full else [x, r, p[0], p[1]]

    def call(args, **kw):
        if full:
            x, r, z, w1, b1, sc, w2, b2 = args
            return ss.block_norm(x, r, w1, w2, z, sc, b1, b2, layer, 1e-2, **kw)
        return ss.block_norm(args[0], args[1], args[2], args[3], layer=layer, eps=1e-2, **kw)

    def loss(*args):
        y, o = call(args)
        return (y * gy).sum() + (o * gr).sum()

    got = call(args, gy=gy, gr=gr)[2:]
    want = list(range(8)) if full else [0, 1, 3, 6]
    for k, i in enumerate(want):
        np.testing.assert_allclose(got[i], _diff(loss, args, k), atol=1e-6)


def test_chunks_and_padding():
    rng = np.random.default_rng(4)
    B, D, L, N, S = 2, 2, 9, 3, 4
    x, de = rng.standard_normal((2, B, D, L))
    w = rng.standard_normal((D, S))
    A = -np.exp(rng.standard_normal((D, N)))
    Bm, Cm = rng.standard_normal((2, B, 1, N, L))
    o, f = ss.short_conv(x, w)
    y, h = ss.selective_scan(x, de, A, Bm, Cm)
    o1, f1 = ss.short_conv(x[..., :2], w)
    o2, f2 = ss.short_conv(x[..., 2:], w, state=f1)
    y1, h1 = ss.selective_scan(x[..., :2], de[..., :2], A, Bm[..., :2], Cm[..., :2])
    y2, h2 = ss.selective_scan(x[..., 2:], de[..., 2:], A, Bm[..., 2:], Cm[..., 2:], state=h1)
    np.testing.assert_allclose(np.concatenate([o1, o2], 2), o)
    np.testing.assert_allclose(f2, f)
    np.testing.assert_allclose(np.concatenate([y1, y2], 2), y)
    np.testing.assert_allclose(h2, h)
    n = [9, 4]
    bad = x.copy()
    bad[1, :, 4:] = np.nan
    op, fp = ss.short_conv(bad, w, lengths=n)
    yp, hp = ss.selective_scan(bad, de, A, Bm, Cm, lengths=n)
    o4, f4 = ss.short_conv(x[1:, :, :4], w)
    y4, h4 = ss.selective_scan(x[1:, :, :4], de[1:, :, :4], A, Bm[1:, ..., :4], Cm[1:, ..., :4])
    for got, want, state, wstate in ((op, o4, fp, f4), (yp, y4, hp, h4)):
        np.testing.assert_allclose(got[1, :, :4], want[0])
        assert not got[1, :, 4:].any()
        np.testing.assert_allclose(state[1], wstate[0])
