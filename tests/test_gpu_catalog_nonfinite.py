"""Gradients of catalog log-probabilities that are not numbers: a row whose log_prob is NaN has NaN
gradients (a check for non-finite gradients has to see it), the others keep theirs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# (64-, 128- and 256-wide tiles, rows in registers, two-part coefficients)
SHAPES = [(torch.float32, 10, 300, 64), (torch.float32, 300, 9000, 64), (torch.bfloat16, 10, 300, 64),
          (torch.bfloat16, 130, 17000, 64), (torch.bfloat16, 300, 33000, 64),
          (torch.bfloat16, 384, 90000, 384)]


def grads(x, w, ids, b=None, entropy=False):
    from twotower.losses import catalog_log_probs

    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=entropy)
    outs = [r.log_prob, r.entropy] if entropy else [r.log_prob]
    torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    return r.log_prob.detach(), xl.grad, wl.grad


def make(dt, N, V, E):
    gen = torch.Generator().manual_seed(N + V)
    x = torch.nn.functional.normalize(torch.randn(N, E, generator=gen), dim=1).to(dt).cuda()
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1).to(dt).cuda()
    return x, w, torch.randint(0, V, (N,), generator=gen).cuda()


@pytest.mark.parametrize("dt,N,V,E", SHAPES)
@pytest.mark.parametrize("entropy", [False, True])
def test_a_nan_query(dt, N, V, E, entropy):
    x, w, ids = make(dt, N, V, E)
    _, dx0, _ = grads(x, w, ids, entropy=entropy)
    x[3, 5] = float("nan")
    lp, dx, dw = grads(x, w, ids, entropy=entropy)
    other = torch.arange(N) != 3
    assert torch.isnan(lp[3]) and torch.isfinite(lp[other]).all()
    assert torch.isnan(dx[3]).all() and torch.equal(dx[other], dx0[other])
    assert torch.isnan(dw[:, 5]).all()


@pytest.mark.parametrize("dt,N,V,E", SHAPES)
def test_a_nan_item_and_one_that_is_taken_out(dt, N, V, E):
    x, w, ids = make(dt, N, V, E)
    ids[ids == 7] = 8
    b = torch.zeros(V).cuda()
    b[7] = float("-inf")
    _, dx0, dw0 = grads(x, w, ids, b)
    w[7] = float("nan")
    lp, dx, dw = grads(x, w, ids, b)
    assert torch.isfinite(lp).all() and torch.equal(dx, dx0) and torch.equal(dw, dw0)
    lp, dx, dw = grads(x, w, ids)
    assert torch.isnan(lp).all() and torch.isnan(dx).all() and torch.isnan(dw).all()


@pytest.mark.parametrize("dt,N,V,E", SHAPES)
def test_a_logit_past_the_range(dt, N, V, E):
    """Finite vectors whose product is not: log_prob is no number, and neither are the gradients."""
    x, w, ids = make(dt, N, V, E)
    x[4] = 0.0
    x[4, 0] = 1e25
    w[11, 0] = 1e25
    lp, dx, dw = grads(x, w, ids)
    other = torch.arange(N) != 4
    assert not torch.isfinite(lp[4]) and not torch.isfinite(dx[4]).any()
    assert not torch.isfinite(dw[:, 0]).any()
    assert other.sum() == N - 1
