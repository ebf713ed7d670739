"""Refusals of the catalog log-probabilities that need no GPU."""
import ctypes
import os

import pytest
import torch

P = 1 << 20  # a 16-byte aligned address that no refused call may touch


@pytest.fixture(scope="module")
def L():
    from twotower import _lib

    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def fwd(L, x=P, w=P, ldx=64, ldw=64, dt=0, N=4, V=40, E=64, ids=P, temp=0.1, lp=P, lse=P, top=0, ti=None,
        ws=P, nws=1 << 30):
    return L.tt_catalog_logprobs(x, ldx, w, ldw, dt, N, V, E, ids, None, temp, lp, None, lse, top, ti, ti, ws,
                                 nws, None)


def test_forward_arguments(L):
    for kw in (dict(dt=2), dict(N=-1), dict(V=0), dict(E=0), dict(E=96), dict(E=32), dict(N=1 << 24),
               dict(V=1 << 30), dict(temp=0.0), dict(temp=-1.0), dict(temp=float("nan")),
               dict(x=None), dict(w=None), dict(lse=None), dict(ids=None), dict(x=P + 4),
               dict(w=P + 8), dict(ldx=66), dict(ldw=32), dict(ldx=60), dict(top=33), dict(top=-1),
               dict(top=3, ti=None), dict(V=2, top=3, ti=P)):
        assert fwd(L, **kw) == -1, kw
    assert fwd(L, N=0, x=None, w=None) == 0
    assert fwd(L, ws=None) == -4 and fwd(L, nws=8) == -4


def test_workspace_sizes(L):
    n = ctypes.c_int64(-1)
    assert L.tt_catalog_logprobs_workspace_bytes(0, 40, 64, 0, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert L.tt_catalog_logprobs_workspace_bytes(1, 1000000, 384, 1, 10, ctypes.byref(n)) == 0
    assert 4 * 62500 < n.value < 4 << 20  # a float per 16 items, and the candidates
    assert fwd(L, N=1, V=1000000, top=10, ti=P, nws=n.value - 1) == -4
    assert L.tt_catalog_logprobs_workspace_bytes(1, 10, 64, 0, 11, ctypes.byref(n)) == -1
    assert L.tt_catalog_logprobs_workspace_bytes(1, 10, 63, 0, 0, ctypes.byref(n)) == -1
    for dt, sz in ((0, 4), (1, 2)):  # the coefficients of a large problem: one 256 MB chunk
        assert L.tt_catalog_logprobs_bwd_workspace_bytes(4096, 10 ** 6, 64, dt, 0, 1, 1,
                                                         ctypes.byref(n)) == 0
        assert n.value < 1 << 30


def test_backward_arguments(L):
    def bwd(N=4, lse=P, g=P, ge=None, ent=None, ids=P, dx=P, dw=P, ws=P, nws=1 << 30):
        return L.tt_catalog_logprobs_bwd(P, 64, P, 64, 0, N, 40, 64, ids, None, 0.1, lse, ent, g, ge, dx, dw,
                                         ws, nws, None)

    assert bwd(lse=None) == -1 and bwd(ids=None) == -1 and bwd(ge=P) == -1
    assert bwd(dx=P + 2) == -1 and bwd(dw=P + 8) == -1
    assert bwd(ws=None) == -4 and bwd(nws=100) == -4
    assert bwd(N=0, dw=None) == 0 and bwd(N=0) == -1


def test_host_tensors_are_refused():
    from twotower._lib import HipUnavailable
    from twotower.losses import catalog_log_probs

    with pytest.raises(HipUnavailable):
        catalog_log_probs(torch.zeros(2, 64), torch.zeros(3, 64))


def test_a_trainable_temperature_is_refused():
    """Its gradient is not computed: refused, not lost."""
    from twotower.losses import CatalogSoftmaxLoss, catalog_log_probs

    x, w, ids = torch.zeros(2, 64), torch.zeros(3, 64), torch.zeros(2, dtype=torch.int64)
    t = torch.tensor(0.07, requires_grad=True)
    with pytest.raises(NotImplementedError, match="temperature"):
        catalog_log_probs(x, w, ids, temperature=t)
    with pytest.raises(NotImplementedError, match="temperature"):
        CatalogSoftmaxLoss(t)(x, w, ids)
    from twotower._lib import HipUnavailable

    with torch.no_grad(), pytest.raises(HipUnavailable):  # (a value without a gradient is one)
        catalog_log_probs(x, w, ids, temperature=t)
    with pytest.raises(HipUnavailable):
        catalog_log_probs(x, w, ids, temperature=torch.tensor(0.07))
