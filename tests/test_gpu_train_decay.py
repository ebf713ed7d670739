"""Checkpoints of TwoTowerTrainStep's AdamW form describe the optimizer that wrote them: loaded into a
step built with the defaults, or into torch's optimizers, training goes on with the same update."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
E, B, S, N = 64, 8, 5, 2


def _towers():
    from test_gpu_train import _setup

    it, bt = _setup(E)
    it.eval()
    return it, bt


def _args(it):
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    ids = lambda *s: torch.randint(0, 3, s, generator=gen, dtype=torch.int32).cuda()  # noqa: E731
    Ht = it.text_encoder.get_sentence_embedding_dimension()
    return (rn(B, S, E), torch.ones(B, S).cuda(), rn(B, Ht), rn(B, N, Ht), ids(B), ids(B), ids(B, N),
            ids(B, N))


def _trained(**kw):
    from twotower.train import TwoTowerTrainStep

    it, bt = _towers()
    step = TwoTowerTrainStep(it, bt, lr=1e-2, **kw)
    args = _args(it)
    for _ in range(3):
        step.step(*args)
    return step, torch.nn.ModuleList([it, bt]), args


def _resumed(sd, model, **kw):
    from twotower.train import TwoTowerTrainStep

    it, bt = _towers()
    twin = torch.nn.ModuleList([it, bt])
    twin.load_state_dict(model.state_dict())
    step = TwoTowerTrainStep(it, bt, **kw)
    step.load_optimizer_state_dict(twin, sd)
    return step, twin


@pytest.mark.parametrize("graph", [False, True])
def test_a_default_step_goes_on_with_the_saved_decay(graph):
    step, model, args = _trained(weight_decay=0.1)
    sd = copy.deepcopy(step.optimizer_state_dict(model))
    assert sd["param_groups"][0]["decoupled_weight_decay"] is True
    other, twin = _resumed(sd, model, graph=graph)
    assert other.weight_decay == 0.1 and other.t == 3 and other.lr == 1e-2
    for _ in range(3):
        step.step(*args)
        other.adam({k: g.clone() for k, g in step.g.items()})  # (embedding rows' gradients are summed in
        for p, q in zip(model.parameters(), twin.parameters()):  # no fixed order: one set for both)
            assert torch.equal(p, q)
    for _ in range(3):
        assert torch.isfinite(other.step(*args))


def test_a_step_with_decay_takes_over_a_checkpoint_without():
    step, model, args = _trained()
    sd = copy.deepcopy(step.optimizer_state_dict(model))
    assert sd["param_groups"][0]["decoupled_weight_decay"] is False
    other, twin = _resumed(sd, model, weight_decay=0.1)
    assert other.weight_decay == 0
    step.step(*args)
    other.adam({k: g.clone() for k, g in step.g.items()})
    for k, p in step.params.items():
        # Adam's and AdamW's kernels round differently, a few last places; and Adam's has 1 - b2^t in f32:
        # 0.999 is off by 2^-25, its 4th power by 4 of that and two roundings, 6 2^-25 of 0.004 = 4.5e-5, its
        # root half; an update is at most 3 lr
        assert ((p - other.params[k]).abs() <= 16 * U * (p.abs() + step.lr) + 3 * 2.3e-5 * step.lr).all()


@pytest.mark.parametrize("cls", [torch.optim.Adam, torch.optim.AdamW])
def test_torch_optimizers_go_on_alike(cls):
    """f32 steps of torch from the same state: 16 roundings of |p| + the update (at most lr / (1 - b1))."""
    step, model, args = _trained(weight_decay=0.1)
    params = [torch.nn.Parameter(p.detach().clone()) for p in model.parameters()]
    opt = cls(params)
    opt.load_state_dict(copy.deepcopy(step.optimizer_state_dict(model)))
    pos = {p.data_ptr(): i for i, p in enumerate(model.parameters())}
    at = {k: pos[p.data_ptr()] for k, p in step.params.items()}
    step.step(*args)
    for k in step.params:
        params[at[k]].grad = step.g[k].clone()
    opt.step()
    for k, p in step.params.items():
        assert ((p - params[at[k]]).abs() <= 16 * U * (p.abs() + 10 * step.lr)).all(), k


def test_decay_of_another_kind_is_refused():
    step, model, args = _trained()
    sd = copy.deepcopy(step.optimizer_state_dict(model))
    sd["param_groups"][0]["weight_decay"] = 0.1  # torch.optim.Adam(weight_decay=0.1): added to the gradient
    with pytest.raises(ValueError, match="decoupled"):
        _resumed(sd, model)
    with pytest.raises(ValueError, match="decoupled"):
        _resumed(sd, model, weight_decay=0.2)
    other, _ = _resumed(sd, model, weight_decay=0.1)  # asked for by its caller: what earlier files hold
    assert other.weight_decay == 0.1
    for key in ("amsgrad", "maximize"):
        sd = copy.deepcopy(step.optimizer_state_dict(model))
        sd["param_groups"][0][key] = True
        with pytest.raises(ValueError, match=key):
            _resumed(sd, model)


def test_eight_bit_moments_go_on_with_the_saved_decay():
    """The width of the moments is the constructor's, the decay the checkpoint's."""
    step, model, args = _trained(weight_decay=0.1, state_bits=8)
    sd = copy.deepcopy(step.optimizer_state_dict(model))
    other, twin = _resumed(sd, model, state_bits=8)
    assert other.weight_decay == 0.1 and other.adamw.bits == 8
    step.step(*args)
    other.adam({k: g.clone() for k, g in step.g.items()})
    # (moments decoded and coded again: the codes stay, a scale may move by a rounding)
    for p, q in zip(model.parameters(), twin.parameters()):
        assert ((p - q).abs() <= 64 * U * (p.abs() + 10 * step.lr)).all()


def test_a_refused_state_changes_nothing():
    step, model, args = _trained(weight_decay=0.1)
    sd = copy.deepcopy(step.optimizer_state_dict(model))
    e = sd["state"][max(sd["state"])]
    e["exp_avg"] = torch.zeros(3)
    plain, _, _ = _trained()
    before = {k: m.clone() for k, m in plain.m.items()}
    owner = torch.nn.ModuleList([plain.it, plain.bt])
    with pytest.raises(ValueError):
        plain.load_optimizer_state_dict(owner, sd)
    assert plain.weight_decay == 0 and plain.adamw is None and plain.t == 3
    assert all(torch.equal(plain.m[k], m) for k, m in before.items())
