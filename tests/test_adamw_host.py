"""Refusals of the many-tensor AdamW that need no GPU."""
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


def step(L, tab=1 << 20, items=1 << 20, n=1, ng=1, chunk=1024, bits=32, b1=0.9, grads=True):
    g = (ctypes.c_void_p * 512)()
    return L.tt_adamw_step(tab, items, n, 0, g if grads else None, ng, chunk, bits, 1e-3, b1, 0.999,
                           1e-8, 0.0, None)


def test_arguments(L):
    assert step(L, bits=16) == -1 and step(L, n=-1) == -1 and step(L, n=1 << 23) == -1
    assert step(L, ng=417) == -1 and step(L, chunk=1000) == -1 and step(L, chunk=0) == -1
    assert step(L, b1=1.0) == -1 and step(L, b1=-0.1) == -1
    assert step(L, tab=None) == -1 and step(L, items=None) == -1 and step(L, grads=False) == -1
    assert step(L, n=0, tab=None, items=None) == 0
    for fn in (L.tt_adamw_decode, L.tt_adamw_encode):
        assert fn(None, 1 << 20, 1, 1024, 1 << 20, 1 << 20, 1 << 20, None) == -1
        assert fn(1 << 20, 1 << 20, 1, 1000, 1 << 20, 1 << 20, 1 << 20, None) == -1
        assert fn(None, None, 0, 1024, None, None, None, None) == 0


def test_table_layout_matches_the_header():
    from twotower.optim import _TENSOR

    assert _TENSOR.itemsize == 72
    assert [_TENSOR.fields[k][1] for k in ("p", "step", "n", "dtype", "blocks")] == \
        [0, 40, 56, 64, 68]


def test_hyperparameters():
    from twotower.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
               dict(weight_decay=-0.1), dict(state_bits=16), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(TypeError):
        AdamW([p], lr=torch.tensor(1e-3))


def test_host_parameters_are_refused():
    from twotower._lib import HipUnavailable
    from twotower.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(HipUnavailable):
        AdamW([p]).step()
