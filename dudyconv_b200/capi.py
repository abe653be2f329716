"""ctypes binding of the C ABI in ``include/dudyconv_b200.h`` (libdudyconv_b200.so).

This is the reference-facing boundary with plain pointers and sizes; the parity tests
call it directly, and it is the binding a non-torch host (or a ctypes-based caller)
would use. Tensor arguments may be torch tensors (their ``data_ptr()`` is passed) or
raw integer device addresses.
"""

from __future__ import annotations

import ctypes
import os

from . import PKG_DIR

LIB_PATH = os.path.join(PKG_DIR, "libdudyconv_b200.so")
HEADER_PATH = os.path.join(os.path.dirname(PKG_DIR), "include", "dudyconv_b200.h")

DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_CUDA, ERR_WORKSPACE, ERR_DEVICE = 0, 1, 2, 3, 4, 5
PLAN_AUTO, PLAN_SIMT, PLAN_TC = -1, 100, 200

_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_int = ctypes.c_int
_sz = ctypes.c_size_t

MAX_PEERS = 8


class PeerExchange(ctypes.Structure):
    """DudyPeerExchange of the C ABI (the data-parallel backward's peer buffers)."""
    _fields_ = [("bufs", ctypes.c_void_p * MAX_PEERS), ("rank", ctypes.c_int),
                ("world", ctypes.c_int), ("epoch", ctypes.c_uint32)]


# name -> (restype, argtypes)
SIGNATURES = {
    "dudy_version": (ctypes.c_char_p, []),
    "dudy_last_error": (ctypes.c_char_p, []),
    "dudy_device_error": (_int, [_int]),
    "dudy_device_error_info": (_int, [ctypes.POINTER(ctypes.c_int), _int]),
    "dudy_fdc_plan_name": (ctypes.c_char_p, [_int]),
    "dudy_fdc_default_plan": (_int, [_vp, _vp, _vp] + [_i64] * 8 + [_int]),
    "dudy_fdc_plan_available": (_int, [_int, _vp, _vp, _vp] + [_i64] * 8 + [_int]),
    "dudy_fdc_forward": (_int, [_vp] * 4 + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fdc_backward_workspace_size": (_sz, [_i64] * 8 + [_int, _int]),
    "dudy_fdc_backward": (_int, [_vp] * 8 + [_sz] + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fdc_backward_grad_h": (_int, [_vp] * 4 + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fdc_backward_grad_kc_mix": (_int, [_vp] * 7 + [_sz] + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fdc_backward_noalloc": (_int, [_vp] * 7 + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fscm_forward_plan_legal": (_int, [_int] + [_i64] * 5),
    "dudy_fscm_forward_default_plan": (_int, [_i64] * 8),
    "dudy_fscm_forward": (_int, [_vp] * 6 + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fscm_backward_plan_legal": (_int, [_int, _i64, _i64, _i64]),
    "dudy_fscm_backward_default_plan": (_int, [_i64] * 8),
    "dudy_fscm_backward_workspace_size": (_sz, [_i64] * 8 + [_int, _int, _i64]),
    "dudy_fscm_backward": (_int, [_vp] * 12 + [_sz] + [_i64] * 8 + [_int, _int, _i64, _vp]),
    "dudy_check_phi_approx": (_int, [_vp]),
    "dudy_selftest_wait_timeout": (_int, [_int, ctypes.POINTER(ctypes.c_int)]),
    "dudy_logits_to_kernel": (_int, [_vp, _vp] + [_i64] * 4 + [_int, _vp]),
    "dudy_fdc_exchange_bytes": (_sz, [_i64, _i64]),
    "dudy_fdc_backward_dp": (_int, [_vp] * 8 + [_sz, ctypes.POINTER(PeerExchange)] + [_i64] * 8
                             + [_int, _int, _vp]),
    "dudy_fdc_backward_dp_deferred": (_int, [_vp] * 9 + [_sz, ctypes.POINTER(PeerExchange)]
                                      + [_i64] * 8 + [_int, _int, _vp]),
    "dudy_fdc_exchange_finish": (_int, [ctypes.POINTER(PeerExchange), _vp, _i64, _i64, _int, _vp]),
    "dudy_logits_to_kernel_backward": (_int, [_vp] * 3 + [_i64] * 4 + [_int, _vp]),
    "dudy_short_conv_forward": (_int, [_vp] * 7 + [_i64] * 4 + [_int, _int, _vp]),
    "dudy_short_conv_backward_workspace_size": (_sz, [_i64] * 4 + [_int]),
    "dudy_short_conv_backward": (_int, [_vp] * 12 + [_sz] + [_i64] * 4 + [_int, _int, _vp]),
    "dudy_short_conv_step": (_int, [_vp] * 5 + [_i64] * 3 + [_int, _int, _vp]),
    "dudy_selective_scan_checkpoint_bytes": (_sz, [_i64] * 5 + [_int]),
    "dudy_selective_scan_forward_workspace_size": (_sz, [_i64] * 5 + [_int]),
    "dudy_selective_scan_forward": (_int, [_vp] * 13 + [_sz] + [_i64] * 5 + [_int, _int, _vp]),
    "dudy_selective_scan_backward_workspace_size": (_sz, [_i64] * 5 + [_int]),
    "dudy_selective_scan_backward": (_int, [_vp] * 20 + [_sz] + [_i64] * 5 + [_int, _int, _vp]),
    "dudy_selective_scan_step": (_int, [_vp] * 9 + [_i64] * 4 + [_int, _int, _vp]),
    "dudy_block_norm_forward": (_int, [_vp] * 11 + [_i64] * 3 + [_int, ctypes.c_float, _int, _int,
                                                                 _vp]),
    "dudy_block_norm_backward_workspace_size": (_sz, [_i64] * 3 + [_int, _int]),
    "dudy_block_norm_backward": (_int, [_vp] * 19 + [_sz] + [_i64] * 3 + [_int, _int, _int, _vp]),
}

_LIB = None


class DudyError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"{msg} (status {status})")
        self.status = status


def lib() -> ctypes.CDLL:
    """Load libdudyconv_b200.so and declare every exported entry point."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is not built; run `python -m dudyconv_b200.build`")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = L
    return _LIB


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


_DTYPE_CODES = None


def dtype_code(t) -> int:
    global _DTYPE_CODES
    if _DTYPE_CODES is None:
        import torch
        _DTYPE_CODES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16,
                        torch.bfloat16: DTYPE_BF16}
    return _DTYPE_CODES[t.dtype]


def last_error() -> str:
    return lib().dudy_last_error().decode()


def _check(rc: int):
    if rc != OK:
        raise DudyError(rc, last_error())


def fdc_forward(h, kc, mix, out, off: int, dilation: int, plan: int = PLAN_AUTO, stream=None):
    B, D, L = h.shape
    _, K, N, T = kc.shape
    _check(lib().dudy_fdc_forward(_ptr(h), _ptr(kc), _ptr(mix), _ptr(out), B, D, L, T, N, K,
                                  off, dilation, dtype_code(h), plan, _stream(stream)))


def fdc_backward_workspace_size(h, kc, off: int, dilation: int, plan: int = PLAN_AUTO) -> int:
    B, D, L = h.shape
    _, K, N, T = kc.shape
    return int(lib().dudy_fdc_backward_workspace_size(B, D, L, T, N, K, off, dilation,
                                                      dtype_code(h), plan))


def fdc_backward(go, h, kc, mix, grad_h, grad_kc, grad_mix, workspace, off: int, dilation: int,
                 plan: int = PLAN_AUTO, stream=None):
    B, D, L = h.shape
    _, K, N, T = kc.shape
    ws_bytes = workspace.numel() * workspace.element_size()
    _check(lib().dudy_fdc_backward(_ptr(go), _ptr(h), _ptr(kc), _ptr(mix), _ptr(grad_h),
                                   _ptr(grad_kc), _ptr(grad_mix), _ptr(workspace), ws_bytes,
                                   B, D, L, T, N, K, off, dilation, dtype_code(h), plan,
                                   _stream(stream)))


def fdc_backward_grad_h(go, kc, mix, grad_h, off: int, dilation: int, plan: int = PLAN_AUTO,
                        stream=None):
    B, D, L = grad_h.shape
    _, K, N, T = kc.shape
    _check(lib().dudy_fdc_backward_grad_h(_ptr(go), _ptr(kc), _ptr(mix), _ptr(grad_h), B, D, L,
                                          T, N, K, off, dilation, dtype_code(go), plan,
                                          _stream(stream)))


def fdc_backward_grad_kc_mix(go, h, kc, mix, grad_kc, grad_mix, workspace, off: int,
                             dilation: int, plan: int = PLAN_AUTO, stream=None):
    B, D, L = h.shape
    _, K, N, T = kc.shape
    ws_bytes = workspace.numel() * workspace.element_size()
    _check(lib().dudy_fdc_backward_grad_kc_mix(_ptr(go), _ptr(h), _ptr(kc), _ptr(mix),
                                               _ptr(grad_kc), _ptr(grad_mix), _ptr(workspace),
                                               ws_bytes, B, D, L, T, N, K, off, dilation,
                                               dtype_code(h), plan, _stream(stream)))


def fdc_backward_noalloc(go, h, kc, mix, grad_h, grad_kc, grad_mix, off: int, dilation: int,
                         plan: int = PLAN_AUTO, stream=None):
    """Backward with the library's fixed scratch array instead of a caller workspace."""
    B, D, L = h.shape
    _, K, N, T = kc.shape
    _check(lib().dudy_fdc_backward_noalloc(_ptr(go), _ptr(h), _ptr(kc), _ptr(mix), _ptr(grad_h),
                                           _ptr(grad_kc), _ptr(grad_mix), B, D, L, T, N, K, off,
                                           dilation, dtype_code(h), plan, _stream(stream)))


def fdc_default_plan(h, kc, mix, off: int, dilation: int) -> int:
    B, D, L = h.shape
    _, K, N, T = kc.shape
    return int(lib().dudy_fdc_default_plan(_ptr(h), _ptr(kc), _ptr(mix), B, D, L, T, N, K, off,
                                           dilation, dtype_code(h)))


def fscm_forward(x, weight, bias, mix_w, mix_b, out, off: int, T: int, dilation: int,
                 plan: int = PLAN_AUTO, stream=None):
    B, D, L = x.shape
    _, C, S = weight.shape
    _check(lib().dudy_fscm_forward(_ptr(x), _ptr(weight), _ptr(bias), _ptr(mix_w), _ptr(mix_b),
                                   _ptr(out), B, D, L, C, S, off, T, dilation, dtype_code(x),
                                   plan, _stream(stream)))


def fscm_backward_workspace_size(x, weight, off: int, T: int, dilation: int,
                                 plan: int = PLAN_AUTO, tile_t: int = 0) -> int:
    B, D, L = x.shape
    _, C, S = weight.shape
    return int(lib().dudy_fscm_backward_workspace_size(B, D, L, C, S, off, T, dilation,
                                                       dtype_code(x), plan, tile_t))


def fscm_backward(go, x, weight, bias, mix_w, mix_b, grad_x, grad_w, grad_bias, grad_mix_w,
                  grad_mix_b, workspace, off: int, T: int, dilation: int, plan: int = PLAN_AUTO,
                  tile_t: int = 0, stream=None):
    B, D, L = x.shape
    _, C, S = weight.shape
    ws_bytes = workspace.numel() * workspace.element_size()
    _check(lib().dudy_fscm_backward(_ptr(go), _ptr(x), _ptr(weight), _ptr(bias), _ptr(mix_w),
                                    _ptr(mix_b), _ptr(grad_x), _ptr(grad_w), _ptr(grad_bias),
                                    _ptr(grad_mix_w), _ptr(grad_mix_b), _ptr(workspace),
                                    ws_bytes, B, D, L, C, S, off, T, dilation, dtype_code(x),
                                    plan, tile_t, _stream(stream)))


def device_error(reset: bool = False) -> int:
    return int(lib().dudy_device_error(1 if reset else 0))


def device_error_info(reset: bool = False):
    """(site, block, thread, counter) of the first timed-out device wait; site 0 = none."""
    buf = (ctypes.c_int * 4)()
    lib().dudy_device_error_info(buf, 1 if reset else 0)
    return tuple(int(v) for v in buf)


def selftest_wait_timeout(limit_us: int = 2000):
    """Run the bounded-wait self-test kernel; returns (warp0 completed, warp1 completed)."""
    buf = (ctypes.c_int * 2)()
    _check(lib().dudy_selftest_wait_timeout(int(limit_us), buf))
    return int(buf[0]), int(buf[1])


def logits_to_kernel(logits, kc, stream=None):
    """kc [B,K,N,T] <- softmax over K of logits [B,N*K,T], flipped (kk = 0 current token)."""
    B, K, N, T = kc.shape
    _check(lib().dudy_logits_to_kernel(_ptr(logits), _ptr(kc), B, N, K, T, dtype_code(kc),
                                       _stream(stream)))


def logits_to_kernel_backward(kc, grad_kc, grad_logits, stream=None):
    B, K, N, T = kc.shape
    _check(lib().dudy_logits_to_kernel_backward(_ptr(kc), _ptr(grad_kc), _ptr(grad_logits), B, N,
                                                K, T, dtype_code(kc), _stream(stream)))


def fdc_exchange_bytes(D: int, N: int) -> int:
    return int(lib().dudy_fdc_exchange_bytes(D, N))


def fdc_backward_dp(go, h, kc, mix, grad_h, grad_kc, grad_mix, workspace, xchg: PeerExchange,
                    off: int, dilation: int, plan: int = PLAN_AUTO, stream=None):
    """dudy_fdc_backward_dp: the backward with grad_mix summed over the ranks of `xchg`."""
    B, D, L = h.shape
    _, K, N, T = kc.shape
    ws_bytes = workspace.numel() * workspace.element_size()
    _check(lib().dudy_fdc_backward_dp(_ptr(go), _ptr(h), _ptr(kc), _ptr(mix), _ptr(grad_h),
                                      _ptr(grad_kc), _ptr(grad_mix), _ptr(workspace), ws_bytes,
                                      ctypes.byref(xchg), B, D, L, T, N, K, off, dilation,
                                      dtype_code(h), plan, _stream(stream)))


def fdc_backward_dp_deferred(go, h, kc, mix, grad_h, grad_kc, grad_mix, grad_mix_prev, workspace,
                             xchg: PeerExchange, off: int, dilation: int, plan: int = PLAN_AUTO,
                             stream=None):
    """dudy_fdc_backward_dp_deferred: this rank's backward; grad_mix gets this rank's own sum,
    grad_mix_prev the sum over ranks of the previous call."""
    B, D, L = h.shape
    _, K, N, T = kc.shape
    ws_bytes = workspace.numel() * workspace.element_size()
    _check(lib().dudy_fdc_backward_dp_deferred(
        _ptr(go), _ptr(h), _ptr(kc), _ptr(mix), _ptr(grad_h), _ptr(grad_kc), _ptr(grad_mix),
        _ptr(grad_mix_prev), _ptr(workspace), ws_bytes, ctypes.byref(xchg), B, D, L, T, N, K,
        off, dilation, dtype_code(h), plan, _stream(stream)))


def fdc_exchange_finish(xchg: PeerExchange, grad_mix, stream=None):
    """dudy_fdc_exchange_finish: the sum over ranks of call xchg.epoch into grad_mix."""
    D, N = grad_mix.shape
    _check(lib().dudy_fdc_exchange_finish(ctypes.byref(xchg), _ptr(grad_mix), D, N,
                                          dtype_code(grad_mix), _stream(stream)))


def _ws_bytes(workspace) -> int:
    return 0 if workspace is None else workspace.numel() * workspace.element_size()


def short_conv_forward(x, weight, bias, state, lengths, out, final_state=None, silu: bool = True,
                       stream=None):
    """Short causal depthwise conv; bias, state, lengths and final_state may be None."""
    B, D, L = x.shape
    _check(lib().dudy_short_conv_forward(_ptr(x), _ptr(weight), _ptr(bias), _ptr(state),
                                         _ptr(lengths), _ptr(out), _ptr(final_state), B, D, L,
                                         weight.shape[1], int(silu), dtype_code(x),
                                         _stream(stream)))


def short_conv_backward_workspace_size(x, weight) -> int:
    B, D, L = x.shape
    return int(lib().dudy_short_conv_backward_workspace_size(B, D, L, weight.shape[1],
                                                             dtype_code(x)))


def short_conv_backward(go, grad_final, x, weight, bias, state, lengths, grad_x, grad_weight,
                        grad_bias, grad_state, workspace, silu: bool = True, stream=None):
    B, D, L = x.shape
    _check(lib().dudy_short_conv_backward(
        _ptr(go), _ptr(grad_final), _ptr(x), _ptr(weight), _ptr(bias), _ptr(state),
        _ptr(lengths), _ptr(grad_x), _ptr(grad_weight), _ptr(grad_bias), _ptr(grad_state),
        _ptr(workspace), _ws_bytes(workspace), B, D, L, weight.shape[1], int(silu),
        dtype_code(x), _stream(stream)))


def short_conv_step(x, state, weight, bias, out, silu: bool = True, stream=None):
    """One token per sequence; state [B,D,S-1] is updated in place."""
    B, D = x.shape
    _check(lib().dudy_short_conv_step(_ptr(x), _ptr(state), _ptr(weight), _ptr(bias), _ptr(out),
                                      B, D, weight.shape[1], int(silu), dtype_code(x),
                                      _stream(stream)))


def _scan_dims(u, A, Bm):
    B, D, L = u.shape
    return B, D, L, A.shape[1], Bm.shape[1]


def selective_scan_checkpoint_bytes(u, A, Bm) -> int:
    return int(lib().dudy_selective_scan_checkpoint_bytes(*_scan_dims(u, A, Bm), dtype_code(u)))


def selective_scan_forward_workspace_size(u, A, Bm) -> int:
    return int(lib().dudy_selective_scan_forward_workspace_size(*_scan_dims(u, A, Bm),
                                                                dtype_code(u)))


def selective_scan_forward(u, delta, A, Bm, Cm, skip, delta_bias, state, lengths, y,
                           final_state=None, checkpoints=None, workspace=None,
                           softplus: bool = True, stream=None):
    """Selective scan; skip, delta_bias, state, lengths, final_state, checkpoints may be None."""
    _check(lib().dudy_selective_scan_forward(
        _ptr(u), _ptr(delta), _ptr(A), _ptr(Bm), _ptr(Cm), _ptr(skip), _ptr(delta_bias),
        _ptr(state), _ptr(lengths), _ptr(y), _ptr(final_state), _ptr(checkpoints),
        _ptr(workspace), _ws_bytes(workspace), *_scan_dims(u, A, Bm), int(softplus),
        dtype_code(u), _stream(stream)))


def selective_scan_backward_workspace_size(u, A, Bm) -> int:
    return int(lib().dudy_selective_scan_backward_workspace_size(*_scan_dims(u, A, Bm),
                                                                 dtype_code(u)))


def selective_scan_backward(go, grad_final, u, delta, A, Bm, Cm, skip, delta_bias, checkpoints,
                            lengths, grad_u, grad_delta, grad_A, grad_B, grad_C, grad_skip,
                            grad_delta_bias, grad_state, workspace, softplus: bool = True,
                            stream=None):
    _check(lib().dudy_selective_scan_backward(
        _ptr(go), _ptr(grad_final), _ptr(u), _ptr(delta), _ptr(A), _ptr(Bm), _ptr(Cm),
        _ptr(skip), _ptr(delta_bias), _ptr(checkpoints), _ptr(lengths), _ptr(grad_u),
        _ptr(grad_delta), _ptr(grad_A), _ptr(grad_B), _ptr(grad_C), _ptr(grad_skip),
        _ptr(grad_delta_bias), _ptr(grad_state), _ptr(workspace), _ws_bytes(workspace),
        *_scan_dims(u, A, Bm), int(softplus), dtype_code(u), _stream(stream)))


def selective_scan_step(u, delta, A, Bm, Cm, skip, delta_bias, state, y, softplus: bool = True,
                        stream=None):
    """One token per sequence; state [B,D,N] (fp32) is updated in place."""
    B, D = u.shape
    _check(lib().dudy_selective_scan_step(
        _ptr(u), _ptr(delta), _ptr(A), _ptr(Bm), _ptr(Cm), _ptr(skip), _ptr(delta_bias),
        _ptr(state), _ptr(y), B, D, A.shape[1], Bm.shape[1], int(softplus), dtype_code(u),
        _stream(stream)))


def block_norm_forward(x, gate, residual, post_weight, post_bias, scale, pre_weight, pre_bias, y,
                       residual_out, stats=None, layer: bool = False, eps: float = 1e-5,
                       stream=None):
    """Norms after and before a block with gate and scaled residual; optional inputs None."""
    B, D, L = x.shape
    _check(lib().dudy_block_norm_forward(
        _ptr(x), _ptr(gate), _ptr(residual), _ptr(post_weight), _ptr(post_bias), _ptr(scale),
        _ptr(pre_weight), _ptr(pre_bias), _ptr(y), _ptr(residual_out), _ptr(stats), B, D, L,
        int(layer), eps, dtype_code(x), dtype_code(residual), _stream(stream)))


def block_norm_backward_workspace_size(x, residual) -> int:
    B, D, L = x.shape
    return int(lib().dudy_block_norm_backward_workspace_size(B, D, L, dtype_code(x),
                                                             dtype_code(residual)))


def block_norm_backward(grad_y, grad_residual_out, x, gate, residual, post_weight, post_bias,
                        scale, pre_weight, stats, grad_x, grad_gate, grad_residual,
                        grad_post_weight, grad_post_bias, grad_scale, grad_pre_weight,
                        grad_pre_bias, workspace, layer: bool = False, stream=None):
    B, D, L = x.shape
    _check(lib().dudy_block_norm_backward(
        _ptr(grad_y), _ptr(grad_residual_out), _ptr(x), _ptr(gate), _ptr(residual),
        _ptr(post_weight), _ptr(post_bias), _ptr(scale), _ptr(pre_weight), _ptr(stats),
        _ptr(grad_x), _ptr(grad_gate), _ptr(grad_residual), _ptr(grad_post_weight),
        _ptr(grad_post_bias), _ptr(grad_scale), _ptr(grad_pre_weight), _ptr(grad_pre_bias),
        _ptr(workspace), _ws_bytes(workspace), B, D, L, int(layer), dtype_code(x),
        dtype_code(residual), _stream(stream)))
