"""AdamW as a torch.optim.Optimizer: what autograd, schedulers and checkpoints rely on."""
import copy

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


def test_load_state_dict_restores_whole_groups():
    """Schedulers keep initial_lr (and others their own keys) in the groups."""
    ps, opt = make(lr=1e-2)
    sch = torch.optim.lr_scheduler.LambdaLR(opt, lambda e: 0.5 ** e)
    opt.param_groups[0]["name"] = "towers"
    for _ in range(3):
        opt.step()
        sch.step()
    sd = copy.deepcopy(opt.state_dict())
    qs, other = make(lr=1.0)
    other.load_state_dict(sd)
    g = other.param_groups[0]
    assert g["initial_lr"] == 1e-2 and g["name"] == "towers" and g["lr"] == 1e-2 * 0.125
    assert all(p is q for p, q in zip(g["params"], qs))
    # a scheduler that resumes reads initial_lr
    s2 = torch.optim.lr_scheduler.LambdaLR(other, lambda e: 0.5 ** e, last_epoch=sch.last_epoch)
    assert s2.base_lrs == sch.base_lrs
    sd["param_groups"][0]["name"] = "changed"  # the groups are copies
    assert g["name"] == "towers"


def test_load_hooks_run():
    ps, opt = make()
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    qs, other = make()
    seen = []

    def pre(o, d):
        seen.append(("pre", o is other))
        d = dict(d)
        d["param_groups"] = [dict(g, lr=0.25) for g in d["param_groups"]]
        return d

    other.register_load_state_dict_pre_hook(pre)
    other.register_load_state_dict_post_hook(lambda o: seen.append(("post", o.param_groups[0]["lr"])))
    other.load_state_dict(sd)
    assert seen == [("pre", True), ("post", 0.25)]


@pytest.mark.parametrize("key", ["amsgrad", "maximize"])
def test_other_optimizers_options_are_refused(key):
    ps, _ = make()
    t = torch.optim.AdamW(ps, **{key: True})
    t.step()
    qs, opt = make()
    with pytest.raises(ValueError, match=key):
        opt.load_state_dict(t.state_dict())


@pytest.mark.parametrize("bits,bad", [(b, k) for b in (32, 8) for k in ("size", "missing", "lr")]
                         + [(8, "scale")])
def test_a_refused_state_changes_nothing(bits, bad):
    ps, opt = make(state_bits=bits, lr=1e-2)
    opt.step()
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    want = {k: v.clone() for k, v in opt.state[ps[0]].items()}
    if bad == "size":
        sd["state"][1]["exp_avg_sq"] = sd["state"][1]["exp_avg_sq"][:3]
    elif bad == "scale":
        sd["state"][1]["exp_avg_scale"] = torch.zeros(2)
    elif bad == "missing":
        del sd["state"][1]["exp_avg"]
    else:
        sd["param_groups"][0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 1e-2
    assert all(torch.equal(opt.state[ps[0]][k], v) for k, v in want.items())
