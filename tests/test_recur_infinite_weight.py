"""An event of infinite weight: the state becomes x whatever it was.  Its gradients are the limits: dx = G,
dgate = 0, nothing passes to the events before."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 6, 400])  # (400: the history split along its events)
@pytest.mark.parametrize("weight", [float("inf"), 3.4e38])
def test_gradients_of_an_infinite_weight(dt, S, weight):
    from twotower.recurrence import gated_scan

    gen = torch.Generator().manual_seed(S)
    x = torch.randn(2, S, 66, generator=gen).to(dt).cuda()
    g = (3 * torch.randn(2, S, 66, generator=gen)).to(dt).cuda()
    g[1, S // 2, :4] = torch.tensor([float("-inf"), -100.0, 80.0, 0.0]).to(dt).cuda()
    w = torch.ones(2, S).cuda()
    w[1, S // 2] = weight
    s0 = torch.randn(2, 66, generator=gen).cuda()
    dh = torch.randn(2, S, 66, generator=gen).to(dt).cuda()
    leaves = [t.requires_grad_() for t in (x, g, s0)]
    h, last = gated_scan(x, g, w, s0)
    dx, dg, d0 = torch.autograd.grad([h, last], leaves, [dh, torch.ones_like(last)])
    for t in (h, last, dx, dg, d0):
        assert torch.isfinite(t).all()
    t = S // 2
    assert torch.equal(h[1, t].detach(), x[1, t].detach())
    assert not dg[1, t].any()
    tol = 2.0 ** -16 if dt == torch.float32 else 2.0 ** -7  # (either side rounded: half a step each)
    # the events before it are a history of their own: nothing reaches them from here
    cut = [v[1:2, :t].detach().clone().requires_grad_() for v in (x, g)]
    st = s0[1:2].detach().clone().requires_grad_()
    h1, _ = gated_scan(*cut, w[1:2, :t], st)
    if t:
        e = torch.autograd.grad([h1], cut + [st], [dh[1:2, :t]])
        for a, b in ((dx[1, :t], e[0][0]), (dg[1, :t], e[1][0]), (d0[1], e[2][0])):
            assert ((a - b).abs() <= tol * b.abs().max()).all()
    else:
        assert not d0[1].any()
    # the events from it on are a history of their own that starts with this event as its state
    if t + 1 < S:
        cut = [v[1:2, t + 1:].detach().clone().requires_grad_() for v in (x, g)]
        st = x[1:2, t].detach().float().requires_grad_()
        h2, l2 = gated_scan(*cut, w[1:2, t + 1:], st)
        e = torch.autograd.grad([h2, l2], cut + [st], [dh[1:2, t + 1:], torch.ones_like(l2)])
        for a, b in ((dx[1, t + 1:], e[0][0]), (dg[1, t + 1:], e[1][0])):
            assert ((a - b).abs() <= tol * b.abs().max()).all()
        want = e[2][0] + dh[1, t].float()
        assert ((dx[1, t].float() - want).abs() <= tol * want.abs().max()).all()
