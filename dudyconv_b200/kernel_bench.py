"""Per-kernel timing of the fused dynamic conv through the C ABI.

    python -m dudyconv_b200.kernel_bench [--batch 16 --seq 4096 --basis 128 --dilation 1]
           [--stage all|forward|grad_h|grad_kc_mix] [--plan tc|simt] [--iters 50]
           [--profile]
    python -m dudyconv_b200.kernel_bench --op fscm [--channels 16 --taps 3 --dilation 1]
    python -m dudyconv_b200.kernel_bench --op short_conv|selective_scan|block_norm
           [--dim 256 --taps 4 --state 16 --groups 1 --dtype fp16|bf16|fp32]


Times each stage (forward, grad_h, grad_kc + grad_mix) with CUDA events, rotating two
input sets so every launch streams from HBM, and prints one JSON line. ``--profile``
runs three warm-up launches of the chosen stage and then exactly one more, for an
``ncu -k <kernel> -s 3 -c 1`` capture of that launch.
"""

from __future__ import annotations

import argparse
import json

import torch

from . import capi

STAGES = ("forward", "grad_h", "grad_kc_mix")


def algorithmic_bytes(stage, B, T, D, N, K, es=2):
    bt = B * T
    if stage in ("forward", "grad_h"):
        return (2 * bt * D + bt * K * N + D * N) * es
    return (2 * bt * D + 2 * bt * K * N + 2 * D * N) * es


def fscm_main(a):
    """Source conv (fused_source_conv_mixed) forward and backward through the C ABI.
    Algorithmic bytes: forward x + out, backward go + x + grad_x (parameters are KB)."""
    dev = torch.device("cuda")
    dt = torch.float16 if a.dtype == "fp16" else torch.bfloat16
    B, T, D, C, S, dil = a.batch, a.seq, a.dim, a.channels, a.taps, a.dilation
    L = T
    gen = torch.Generator(device=dev).manual_seed(0)

    def make():
        return (torch.randn(B, D, L, device=dev, generator=gen).to(dt),
                (torch.randn(D, C, S, device=dev, generator=gen) * 3 ** -0.5).to(dt),
                (torch.randn(D, C, device=dev, generator=gen) * C ** -0.5).to(dt),
                (torch.randn(D, C, device=dev, generator=gen) * C ** -0.5).to(dt),
                torch.zeros(D, device=dev, dtype=dt),
                torch.randn(B, D, T, device=dev, generator=gen).to(dt))

    sets = [make() for _ in range(2)]
    out = torch.empty(B, D, T, device=dev, dtype=dt)
    x0, w0 = sets[0][0], sets[0][1]
    gx = torch.empty_like(x0)
    gw = torch.empty_like(w0)
    gb = torch.empty(D, C, device=dev, dtype=dt)
    gmw = torch.empty(D, C, device=dev, dtype=dt)
    gmb = torch.empty(D, device=dev, dtype=dt)
    ws = torch.empty(max(256, capi.fscm_backward_workspace_size(x0, w0, 0, T, dil)),
                     dtype=torch.uint8, device=dev)

    def launch(stage, i):
        x, w, bias, mw, mb, go = sets[i % 2]
        if stage == "forward":
            capi.fscm_forward(x, w, bias, mw, mb, out, 0, T, dil)
        else:
            capi.fscm_backward(go, x, w, bias, mw, mb, gx, gw, gb, gmw, gmb, ws, 0, T, dil)

    if a.profile:  # 4 launches of each pass, nothing timed (for ncu -k ... -s 3 -c 1)
        for st in ("forward", "backward"):
            for i in range(4):
                launch(st, i)
        torch.cuda.synchronize()
        print(json.dumps({"profile_launches": 4, "device_error": capi.device_error_info()}))
        return
    bt = B * T
    alg = {"forward": 2 * bt * D * 2, "backward": 3 * bt * D * 2}
    res = {"op": "fscm", "batch": B, "seq": T, "D": D, "C": C, "S": S, "dilation": dil,
           "dtype": a.dtype, "gelu_per_forward": bt * D * C}
    for st in ("forward", "backward"):
        for i in range(3):
            launch(st, i)
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for i in range(a.iters):
            launch(st, i)
        e1.record()
        torch.cuda.synchronize()
        us = e0.elapsed_time(e1) / a.iters * 1e3
        res[st] = {"us": us, "GB/s": alg[st] / us / 1e3}
    res["device_error"] = capi.device_error_info()
    print(json.dumps(res))


def state_space_main(a):
    """Forward and backward of one operator of the state-space block (short_conv,
    selective_scan, block_norm) through the C ABI. Algorithmic bytes: each row tensor once. Launches
    rotate through sets of rows (and of B and C), so many that even a launch of two row tensors comes
    back to its own after twice the L2's bytes: rows come from HBM. Saved states, statistics and partial
    sums are one set, left where the launch before put them."""
    dev = torch.device("cuda")
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}[a.dtype]
    B, L, D, N, G, S = a.batch, a.seq, a.dim, a.state, a.groups, a.taps
    gen = torch.Generator(device=dev).manual_seed(0)

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=gen) * scale).to(dtype)

    def scratch(nbytes):
        return torch.empty(max(256, nbytes), dtype=torch.uint8, device=dev)

    l2 = torch.cuda.get_device_properties(dev).L2_cache_size
    sets = min(512, max(2, -(-l2 // (B * D * L * dt.itemsize))))
    rows = [[randn(B, D, L) for _ in range(5)] for _ in range(sets)]
    outs = [[torch.empty(B, D, L, device=dev, dtype=dt) for _ in range(3)] for _ in range(sets)]
    x0 = rows[0][0]
    if a.op == "short_conv":
        w, bias = randn(D, S, scale=S ** -0.5), randn(D)
        gw, gb = torch.empty_like(w), torch.empty_like(bias)
        ws = scratch(capi.short_conv_backward_workspace_size(x0, w))
        moved = {"forward": 2, "backward": 3}

        def launch(stage, i):
            (x, go), o = rows[i % sets][:2], outs[i % sets]
            if stage == "forward":
                capi.short_conv_forward(x, w, bias, None, None, o[0])
            else:
                capi.short_conv_backward(go, None, x, w, bias, None, None, o[1], gw, gb, None, ws)
    elif a.op == "selective_scan":
        A = -torch.arange(1, N + 1, device=dev, dtype=torch.float32).repeat(D, 1)
        skip, dbias = torch.ones(D, device=dev), torch.full((D,), -4.0, device=dev)
        bc = [[randn(B, G, N, L) for _ in range(2)] for _ in range(sets)]
        gA, gskip, gbias = torch.empty_like(A), torch.empty_like(skip), torch.empty_like(skip)
        gB, gC = torch.empty_like(bc[0][0]), torch.empty_like(bc[0][0])
        ck = scratch(capi.selective_scan_checkpoint_bytes(x0, A, bc[0][0]))
        wf = scratch(capi.selective_scan_forward_workspace_size(x0, A, bc[0][0]))
        ws = scratch(capi.selective_scan_backward_workspace_size(x0, A, bc[0][0]))
        moved = {"forward": 3, "forward_saving": 3, "backward": 5}

        def launch(stage, i):
            (u, de, go), o = rows[i % sets][:3], outs[i % sets]
            Bm, Cm = bc[i % sets]
            if stage != "backward":
                capi.selective_scan_forward(u, de, A, Bm, Cm, skip, dbias, None, None, o[0], None,
                                            ck if stage == "forward_saving" else None, wf)
            else:
                capi.selective_scan_backward(go, None, u, de, A, Bm, Cm, skip, dbias, ck, None,
                                             o[1], o[2], gA, gB, gC, gskip, gbias, None, ws)
    else:
        par = [randn(D) for _ in range(3)]
        gp = [torch.empty_like(p) for p in par]
        stats = torch.empty(4, B, L, device=dev)
        ws = scratch(capi.block_norm_backward_workspace_size(x0, x0))
        moved = {"forward": 5, "backward": 8}

        def launch(stage, i):
            (x, z, r, gy, gr), o = rows[i % sets], outs[i % sets]
            if stage == "forward":
                capi.block_norm_forward(x, z, r, par[0], None, par[1], par[2], None, o[0], o[1], stats)
            else:
                capi.block_norm_backward(gy, gr, x, z, r, par[0], None, par[1], par[2], stats,
                                         o[0], o[1], o[2], gp[0], None, gp[1], gp[2], None, ws)

    if a.profile:  # 4 launches of each pass, nothing timed
        for st in moved:
            for i in range(4):
                launch(st, i)
        torch.cuda.synchronize()
        print(json.dumps({"profile_launches": 4, "device_error": capi.device_error_info()}))
        return
    res = {"op": a.op, "batch": B, "seq": L, "D": D, "N": N, "G": G, "S": S, "dtype": a.dtype, "sets": sets}
    for st, n in moved.items():
        for i in range(3):
            launch(st, i)
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for i in range(a.iters):
            launch(st, i)
        e1.record()
        torch.cuda.synchronize()
        us = e0.elapsed_time(e1) / a.iters * 1e3
        res[st] = {"us": round(us, 2), "GB/s": round(n * x0.numel() * x0.element_size() / us / 1e3, 1)}
    res["device_error"] = capi.device_error_info()
    print(json.dumps(res))


STATE_SPACE = ("short_conv", "selective_scan", "block_norm")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--op", default="fdc", choices=("fdc", "fscm") + STATE_SPACE)
    ap.add_argument("--state", type=int, default=16, help="selective_scan: states N")
    ap.add_argument("--groups", type=int, default=1, help="selective_scan: groups G of B and C")
    ap.add_argument("--channels", type=int, default=16, help="fscm: source channels C")
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--seq", type=int, default=4096)
    ap.add_argument("--basis", type=int, default=128)
    ap.add_argument("--taps", type=int, default=3)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--dilation", type=int, default=1)
    ap.add_argument("--offset", type=int, default=0)
    ap.add_argument("--dtype", default="fp16", choices=["fp16", "bf16", "fp32"],
                    help="fp32: the state-space operators only")
    ap.add_argument("--stage", default="all", choices=("all",) + STAGES)
    ap.add_argument("--plan", default="tc", choices=["tc", "simt"])
    ap.add_argument("--iters", type=int, default=50)
    ap.add_argument("--profile", action="store_true")
    a = ap.parse_args()
    if a.op == "fscm":
        return fscm_main(a)
    if a.op in STATE_SPACE:
        return state_space_main(a)

    dev = torch.device("cuda")
    dt = torch.float16 if a.dtype == "fp16" else torch.bfloat16
    B, T, D, N, K, dil, off = a.batch, a.seq, a.dim, a.basis, a.taps, a.dilation, a.offset
    L = off + T
    plan = capi.PLAN_TC if a.plan == "tc" else capi.PLAN_SIMT
    gen = torch.Generator(device=dev).manual_seed(0)
    nsets = 1 if a.profile else 2

    def make():
        return (torch.randn(B, D, L, device=dev, generator=gen).to(dt),
                (torch.randn(B, K, N, T, device=dev, generator=gen) * N ** -0.5).to(dt),
                (torch.randn(D, N, device=dev, generator=gen) * 3 ** -0.5).to(dt),
                torch.randn(B, D, T, device=dev, generator=gen).to(dt))

    sets = [make() for _ in range(nsets)]
    out = torch.empty(B, D, T, device=dev, dtype=dt)
    gh = torch.empty(B, D, L, device=dev, dtype=dt)
    gk = torch.empty(B, K, N, T, device=dev, dtype=dt)
    gm = torch.empty(D, N, device=dev, dtype=dt)
    h0, k0 = sets[0][0], sets[0][1]
    ws = torch.empty(max(256, capi.fdc_backward_workspace_size(h0, k0, off, dil, plan)),
                     dtype=torch.uint8, device=dev)

    def launch(stage, i):
        h, kc, mix, go = sets[i % nsets]
        if stage == "forward":
            capi.fdc_forward(h, kc, mix, out, off, dil, plan)
        elif stage == "grad_h":
            capi.fdc_backward_grad_h(go, kc, mix, gh, off, dil, plan)
        else:
            capi.fdc_backward_grad_kc_mix(go, h, kc, mix, gk, gm, ws, off, dil, plan)

    stages = STAGES if a.stage == "all" else (a.stage,)
    if a.profile:
        for i in range(4):
            launch(stages[0], i)
        torch.cuda.synchronize()
        print(json.dumps({"profile_launches": 4, "stage": stages[0],
                          "device_error": capi.device_error_info()}))
        return
    res = {"batch": B, "seq": T, "D": D, "N": N, "K": K, "dilation": dil, "offset": off,
           "dtype": a.dtype, "plan": a.plan}
    for st in stages:
        for i in range(5):
            launch(st, i)
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for i in range(a.iters):
            launch(st, i)
        e1.record()
        torch.cuda.synchronize()
        us = e0.elapsed_time(e1) / a.iters * 1e3
        res[st] = {"us": us, "GB/s": algorithmic_bytes(st, B, T, D, N, K) / us / 1e3}
    res["device_error"] = capi.device_error_info()
    print(json.dumps(res))


if __name__ == "__main__":
    main()
