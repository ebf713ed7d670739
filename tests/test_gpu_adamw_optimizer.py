"""AdamW as a torch.optim.Optimizer: what autograd, schedulers and checkpoints rely on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(sizes=((50,), (7, 9)), **kw):
    from twotower.optim import AdamW

    gen = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).cuda()) for s in sizes]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen).cuda()
    return ps, AdamW(ps, **kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_backward_pass_over_changed_weights_is_refused(bits):
    """The step writes the parameters behind torch's back; their versions say so, as after any in-place
    operation."""
    ps, opt = make(state_bits=bits)
    ps[1].grad = None
    x = torch.randn(9, 3, device="cuda", requires_grad=True)
    y = ps[1] @ x  # (saves ps[1] for x's gradient)
    z = ps[0] * x.sum()
    before = [p._version for p in ps]
    opt.step()
    assert ps[0]._version > before[0] and ps[1]._version == before[1]  # (no gradient: not moved)
    torch.autograd.grad(y.sum(), [x])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_versions_do_not_disturb_a_captured_step():
    ps, opt = make()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    old = ps[0].detach().clone()
    graph.replay()
    torch.cuda.synchronize()
    assert (ps[0] != old).any()
