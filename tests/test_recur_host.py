"""Refusals of the gated recurrence that need no GPU: sizes, pointers, workspaces, tensors."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from twotower import _lib

    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def fwd(L, x=1 << 20, g=1 << 20, dt=0, B=1, S=4, D=8, last=1 << 20, ws=None, nws=0):
    return L.tt_gated_scan_fwd(x, g, dt, B, S, D, S * D, D, S * D, D, None, 0, None, None, last,
                               None, ws, nws, None)


def test_sizes_and_pointers(L):
    assert fwd(L, dt=2) == -1 and fwd(L, B=-1) == -1 and fwd(L, S=-1) == -1 and fwd(L, D=0) == -1
    assert fwd(L, x=None) == -1 and fwd(L, g=None) == -1 and fwd(L, last=None) == -1
    assert fwd(L, B=0, x=None, g=None, last=None) == 0
    assert L.tt_gated_scan_bwd(1 << 20, 1 << 20, 0, 1, 4, 8, 32, 8, 32, 8, None, 0, None, None,
                               None, 1 << 20, 1 << 20, None, None, 0, None) == -1  # no states
    assert b"null pointer" in L.tt_last_error()


def test_workspace(L):
    n = ctypes.c_int64(-1)
    assert L.tt_gated_scan_workspace_bytes(512, 100, 768, ctypes.byref(n)) == 0 and n.value == 0
    assert L.tt_gated_scan_workspace_bytes(1, 20000, 384, ctypes.byref(n)) == 0 and n.value > 0
    assert fwd(L, S=20000, D=384) == -4
    assert fwd(L, S=20000, D=384, ws=1 << 20, nws=n.value // 4) == -4
    assert L.tt_gated_scan_workspace_bytes(1, 1, 0, ctypes.byref(n)) == -1


def test_host_tensors_are_refused():
    from twotower import BuyerTower
    from twotower._lib import HipUnavailable
    from twotower.recurrence import gated_scan

    x = torch.zeros(2, 3, 4)
    with pytest.raises(HipUnavailable):
        gated_scan(x, x)
    with pytest.raises(ValueError, match="multiple of 32"):
        BuyerTower(100, "recurrent")
    with pytest.raises(ValueError, match="recurrent_state needs"):
        BuyerTower(64, "weighted_avg").recurrent_state(x, x[..., 0])


@pytest.mark.gpu
def test_refusals_on_the_device():
    from twotower.recurrence import gated_scan

    x = torch.zeros(2, 3, 4, device="cuda")
    for bad, exc in ((dict(gate=x.half()), TypeError), (dict(gate=x[:, :2]), ValueError),
                     (dict(gate=x, weights=x[0]), ValueError), (dict(gate=x, h0=x[0]), ValueError),
                     (dict(gate=x, weights=torch.zeros(2, 3)), ValueError),
                     (dict(gate=x.bfloat16()), TypeError)):
        with pytest.raises(exc):
            gated_scan(x, **bad)
    w = torch.ones(2, 3, device="cuda", requires_grad=True)
    _, last = gated_scan(x, x, w)
    with pytest.raises(NotImplementedError):
        last.sum().backward()


def test_when_histories_are_split(L):
    """Histories that fill the card are not split (no workspace), few long ones are."""
    n = ctypes.c_int64(-1)

    def need(B, S, D):
        assert L.tt_gated_scan_workspace_bytes(B, S, D, ctypes.byref(n)) == 0
        return n.value

    assert need(639, 1000, 128) > 0 and need(1, 128, 64) > 0
    assert need(1024, 1000, 64) == 0  # (with one channel a lane as well)
    assert need(700, 1000, 64) == 0 and need(700, 100000, 64) == 0 and need(3, 127, 64) == 0
