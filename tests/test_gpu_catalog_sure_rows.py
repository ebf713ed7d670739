"""Gradients of f32 catalog log-probabilities where one item has nearly all of the probability: the
coefficient g (1 - p) is the difference of two nearly equal values, and the log-sum must not be rounded on
the way (in 32 bits it is off by 2^-25 of some 100, and p by as much)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("N,V", [(5, 30), (300, 30), (200, 100), (1100, 78)])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_nearly_certain_rows(N, V, entropy, bias):
    """Elements are small multiples of 1/8, temperature 1: the products are exact.  z = l log2 e is off by 2^-25
    of itself (the factor's rounding; all items alike) and by the rounding of its difference with the
    log-sum, together u (|z| + |lse|) of p_v; the sum of exponentials by at most V / 8 + 8 roundings (a lane's
    adds and the joins), the exponential 2, the products and differences 10.  So p_v is off by
    (V / 8 + 20 + |z| + |lse|) u of itself, but the item with nearly all of it by (V / 8 + 20) u and the
    others' errors.  The gradients' sums: 34 + K / 32 roundings."""
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(N + V)
    w = torch.randint(-8, 9, (V, 64), generator=gen) / 8.0
    ids = torch.randint(0, V, (N,), generator=gen)
    x = w[ids] + torch.randint(-2, 3, (N, 64), generator=gen) / 8.0
    x = torch.round(x * 8 * 0.5) / 8.0
    b = torch.randint(-4, 5, (V,), generator=gen) / 4.0 if bias else None
    g = torch.randn(N, generator=gen)
    ge = 0.01 * torch.randn(N, generator=gen) if entropy else torch.zeros(N)
    xl, wl = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = catalog_log_probs(xl, wl, ids.cuda(), 1.0, b.cuda() if bias else None, entropy=True)
    torch.autograd.backward([r.log_prob, r.entropy], [g.cuda(), ge.cuda()])
    xd, wd, gd, ed = x.double().cuda(), w.double().cuda(), g.double().cuda(), ge.double().cuda()
    l = xd @ wd.t() + (b.double().cuda() if bias else 0.0)
    lse = torch.logsumexp(l, 1, keepdim=True)
    lp = l - lse
    p = torch.exp(lp)
    assert (p.max(1).values > 0.9).double().mean() > 0.3
    ent = -(p * lp).sum(1, keepdim=True)
    rows = torch.arange(N)
    f = gd[:, None] + ed[:, None] * (lp + ent)
    c = -p * f
    c[rows, ids] += gd
    size = gd.abs()[:, None] + ed.abs()[:, None] * (lp.abs() + ent + 1)
    rel = (V / 8 + 20) * U + 1.45 * U * (l.abs() + lse.abs()) * (1 - p)  # (the sure one's: with 1 - p)
    off = size * p * rel + 2 * U * c.abs()
    # entropy's own error (see test_gpu_catalog: 2 T (1 + range), here T the few roundings above)
    off = off + p * ed.abs()[:, None] * 2 * (V / 8 + 20) * U * (1 + lp.abs())
    for got, want, other, cc, oo, k in ((xl.grad, c @ wd, wd, c, off, V),
                                        (wl.grad, c.t() @ xd, xd, c.t(), off.t(), N)):
        tol = oo @ other.abs() + (34 + -(-k // 32)) * U * (cc.abs() @ other.abs()) + 1e-30
        err = (got.double() - want).abs()
        assert (err <= tol).all(), (err / tol).max().item()
