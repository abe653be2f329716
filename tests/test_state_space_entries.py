"""What the state-space block's C entries refuse before any device work: buffers that start
where their kernels cannot read or write them."""

import ctypes

import pytest

from dudyconv_b200 import capi

F = ctypes.c_void_p(256)  # an address that is never reached


def _at(offset):
    return ctypes.c_void_p(256 + offset)


def _scan_forward(checkpoints=F):
    return capi.lib().dudy_selective_scan_forward(F, F, F, F, F, None, None, None, None, F, None, checkpoints, F, 1 << 30,
                                                  1, 8, 100, 16, 1, 1, 1, None)


def _scan_backward(checkpoints=F, workspace=F):
    return capi.lib().dudy_selective_scan_backward(F, None, F, F, F, F, F, None, None, checkpoints, None, F, F, F, F, F, None,
                                                   None, None, workspace, 1 << 30, 1, 8, 100, 16, 1, 1, 1, None)


@pytest.mark.parametrize("offset", [4, 8, 12])
@pytest.mark.parametrize("call,name", [(_scan_forward, "checkpoints"), (_scan_backward, "checkpoints"),
                                       (_scan_backward, "workspace")])
def test_buffers_start_on_16_bytes(call, name, offset):
    """The scan writes and reads saved states and partial sums 16 bytes at a time."""
    assert call(**{name: _at(offset)}) == capi.ERR_INVALID
    assert capi.last_error() == f"{name} must be 16-byte aligned."


def test_a_final_state_is_not_the_initial_one():
    """Blocks of a sequence's chunks read the initial state at times of their own, so the final state
    cannot take its place."""
    lib = capi.lib()
    rc = lib.dudy_selective_scan_forward(F, F, F, F, F, None, None, _at(64), None, F, _at(64), None, F, 1 << 30, 1, 8, 4096, 16,
                                         1, 1, 1, None)
    assert rc == capi.ERR_INVALID and capi.last_error() == "final_state must not be the initial state's memory."
    rc = lib.dudy_short_conv_forward(F, F, None, _at(64), None, F, _at(64), 1, 8, 4096, 4, 1, 1, None)
    assert rc == capi.ERR_INVALID and capi.last_error() == "final_state must not be the initial state's memory."
