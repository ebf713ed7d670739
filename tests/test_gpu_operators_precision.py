"""Bounds of a few last places, where the inputs leave nothing else: what 32-bit arithmetic gives, and
fewer bits anywhere would not."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("N,V", [(5, 70), (200, 1000), (130, 9000), (700, 2500), (33, 20000)])
@pytest.mark.parametrize("entropy", [False, True])
def test_catalog_gradients_f32(N, V, entropy):
    """Logits that 32 bits hold exactly: x and w are multiples of 1/8 in 32 channels, temperature 1, so a
    product is a multiple of 1/64 below 1, z = l log2 e off by 3 u |z| < 5 u; lse (below 11) and its
    product with log2 e are rounded once each, 11 + 16 u; exp2 2 u.  p is off by 40 u of itself, with the
    entropy's factor (logit and entropy below 12, off by 40 u of that) by 40 u of 24 p.  The sums run in
    stages of 32, then over the stages: 34 + K / 32 roundings.
    32 more channels carry full 24-bit values on one side (and 0 on the other, so that no logit moves):
    their gradients are sums of c w and c x with all of their bits."""
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(N + V)
    g = torch.randn(N, generator=gen)
    ge = 0.1 * torch.randn(N, generator=gen) if entropy else torch.zeros(N)
    ids = torch.randint(0, V, (N,), generator=gen)
    for side in (0, 1):
        x = torch.randint(-1, 2, (N, 64), generator=gen) / 8.0
        w = torch.randint(-1, 2, (V, 64), generator=gen) / 8.0
        x[:, 32:], w[:, 32:] = 0.0, 0.0
        (w if side == 0 else x)[:, 32:] = torch.randn((V, N)[side], 32, generator=gen)
        xl, wl = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        r = catalog_log_probs(xl, wl, ids.cuda(), 1.0, entropy=True)
        torch.autograd.backward([r.log_prob, r.entropy], [g.cuda(), ge.cuda()])
        xd, wd = x.double().cuda(), w.double().cuda()
        lp = torch.log_softmax(xd @ wd.t(), 1)
        p, gd, ed = torch.exp(lp), g.double().cuda(), ge.double().cuda()
        ent = -(p * lp).sum(1)
        c = -p * (gd[:, None] + ed[:, None] * (lp + ent[:, None]))
        c[torch.arange(N), ids] += gd
        off = 40 * U * p * (gd.abs() + 24 * ed.abs())[:, None] + 2 * U * c.abs()
        for got, want, other, k in ((xl.grad, c @ wd, wd, V), (wl.grad, c.t() @ xd, xd, N)):
            cc, oo = (c, off) if k == V else (c.t(), off.t())
            tol = oo @ other.abs() + (34 + -(-k // 32)) * U * (cc.abs() @ other.abs()) + 1e-30
            err = (got.double() - want).abs()
            assert (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("B,S,D", [(300, 33, 48), (1, 1000, 384), (2, 4099, 66), (1024, 40, 130)])
@pytest.mark.parametrize("weighted", [False, True])
def test_recurrence_f32(B, S, D, weighted):
    """Gates at or below 0: a memory of at most 2 events.  A gate is off by 6 roundings, a state's update
    by 2 more of the largest state: 2 x 8 u; the gradients' products add 4 and run over states and
    gradients that are themselves off so: 2 x (8 + 8 + 4 + 8) u."""
    from test_gpu_recur import reference
    from twotower.recurrence import gated_scan

    gen = torch.Generator().manual_seed(B + S)
    x = torch.randn(B, S, D, generator=gen)
    g = -3 * torch.rand(B, S, D, generator=gen)
    w = (torch.rand(B, S, generator=gen) < 0.7).float() if weighted else None
    dh, dl = torch.randn(B, S, D, generator=gen), torch.randn(B, D, generator=gen)
    ref = reference(x, g, w, None, dh, dl)
    leaves = [x.cuda().requires_grad_(), g.cuda().requires_grad_()]
    h, last = gated_scan(*leaves, w.cuda() if weighted else None)
    dx, dg = torch.autograd.grad([h, last], leaves, [dh.cuda(), dl.cuda()])
    for got, key, k in ((h, "h", 16), (last, "last", 16), (dx, "dx", 56), (dg, "dgate", 56)):
        err = (got.detach().cpu().double() - ref[key]).abs().max()
        assert err <= k * U * ref[key].abs().max(), (key, (err / ref[key].abs().max() / U).item())
