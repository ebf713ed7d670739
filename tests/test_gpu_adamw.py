"""AdamW over many tensors (csrc/tt_adamw.hip, twotower.optim) against the formulas in 64 bits.

Tolerances (one step from a known state, f32, u = 2^-24 = half a step): m = b1 m + c1 g is three
roundings and two rounded constants, at most 4 u of |b1 m| + |c1 g|; v likewise 5 u; the update
m / (sqrt(v) rs + eps) adds the roundings of sqrt, rs, two operations, the quotient, the factor and
the product: 16 u of its size with the moments' own; p two more roundings of |p| + |update|.  A bf16
parameter is rounded once more, half a step (2^-8 of the value).  8 bits: a scale is the block's
largest 64-bit moment rounded to f32, so within half a step of it (either neighbour where the 64-bit
values, equal to 2^-50, lie at the middle: 0.9 s + 0.1 g of two floats often does); given the
scale, the codes are the nearest ones, equal to the reference's."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2
SIZES = [(1,), (3,), (255,), (256,), (257,), (1000,), (3, 5, 7), (4097,), (0,), (130, 33), (1, 1),
         (70001,)]
HP = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def blocks(t):
    f = t.reshape(-1)
    return torch.nn.functional.pad(f, (0, (-f.numel()) % 256)).view(-1, 256)


def dec(q, s, top, power):
    v = torch.sign(q.double()) * (q.double().abs() / top) ** power
    return (blocks(v) * s.double()[:, None]).reshape(-1)[:q.numel()].view(q.shape)


def enc(t, s, top, power, lowest):
    """Codes of t for the scales s, which are checked first."""
    b = blocks(t)
    top64 = b.abs().amax(1)
    assert ((s.double() - top64).abs() <= U * (1 + 2.0 ** -20) * top64 + 1e-45).all()
    r = (b.abs() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, None]) ** (1.0 / power)
    q = torch.round(r * top).clamp(max=top)
    q = torch.where(b != 0, q.clamp(min=lowest), q) * torch.sign(b)
    return q.reshape(-1)[:t.numel()].view(t.shape)


def entries(opt, p):
    s = opt.state[p]
    return {k: v.detach().cpu().clone() for k, v in s.items()}


def expect(p, g, s, bits, lr, betas, eps, weight_decay):
    """One step in f64 from the state s: (p, |update|, m, v)."""
    b1, b2 = betas
    t = int(s["step"]) + 1
    if bits == 8:
        m = dec(s["exp_avg"], s["exp_avg_scale"], 127.0, 2)
        v = dec(s["exp_avg_sq"], s["exp_avg_sq_scale"], 255.0, 4)
    else:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    g = g.double()
    sz = (b1 * m).abs() + ((1 - b1) * g).abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    den = torch.sqrt(v / (1 - b2 ** t)) + eps
    up = lr / (1 - b1 ** t) * m / den
    upsz = lr / (1 - b1 ** t) * sz / den
    return p.double() * (1 - lr * weight_decay) - up, upsz, m, v, sz


def check_step(opt, params, before, bits, hp=HP, grads=None):
    for i, p in enumerate(params):
        p0, s = before[i]
        g = (p.grad if grads is None else grads[i])
        if g is None:
            assert torch.equal(p.detach().cpu(), p0)
            assert int(opt.state[p]["step"]) == int(s["step"])
            continue
        want, upsz, m, v, sz = expect(p0, g.detach().cpu(), s, bits, **hp)
        got = p.detach().cpu().double()
        tol = 4 * U * (p0.double().abs() + upsz) + 24 * U * upsz
        if p.dtype == torch.bfloat16:
            tol = tol + BF16_HALF * want.abs()
        assert ((got - want).abs() <= tol).all(), (i, tuple(p.shape))
        st = opt.state[p]
        if p.numel():
            assert int(st["step"]) == int(s["step"]) + 1
        if bits == 32:
            assert ((st["exp_avg"].cpu().double() - m).abs() <= 4 * U * sz).all()
            assert ((st["exp_avg_sq"].cpu().double() - v).abs() <= 6 * U * v).all()
        else:
            for k, val, top, power, low in (("exp_avg", m, 127.0, 2, 0.0),
                                            ("exp_avg_sq", v, 255.0, 4, 1.0)):
                if p.numel() == 0:
                    continue
                q = enc(val, st[k + "_scale"].cpu(), top, power, low)
                assert torch.equal(st[k].cpu().double(), q.double()), (i, k)


def snapshot(opt, params):
    if not opt._tables:
        opt._build()
    return [(p.detach().cpu().clone(), entries(opt, p)) for p in params]


def make(dtype, sizes=SIZES, seed=0, odd=False):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for sh in sizes:
        n = int(np.prod(sh))
        if odd:  # views one element into a buffer: no vector access possible
            buf = torch.zeros(n + 1, dtype=dtype, device="cuda")
            t = buf[1:].view(sh)
        else:
            t = torch.zeros(sh, dtype=dtype, device="cuda")
        t.copy_(torch.randn(sh, generator=gen) * 0.05)
        out.append(torch.nn.Parameter(t))
    return out


def set_grads(params, seed, skip=()):
    gen = torch.Generator().manual_seed(seed)
    for i, p in enumerate(params):
        g = torch.randn(p.shape, generator=gen) * torch.exp(2 * torch.randn(p.shape, generator=gen))
        p.grad = None if i in skip else (g * 1e-2).to(p.dtype).cuda()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("odd", [False, True])
def test_steps_vs_f64(bits, dtype, odd):
    from twotower.optim import AdamW

    params = make(dtype, odd=odd)
    opt = AdamW(params, state_bits=bits, **HP)
    for k in range(5):
        set_grads(params, 100 + k, skip=(3,) if k in (1, 2) else ())
        before = snapshot(opt, params)
        opt.step()
        check_step(opt, params, before, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_against_torch_adamw(bits):
    """20 steps beside torch.optim.AdamW in f64.  32 bits: 20 steps of the bound above, and the
    update is at most about lr, so 20 (24 + 4) 2^-24 lr + 40 2^-24 |p|.  8 bits: a level is at most
    1.6% of m's block maximum off (half of 2 / 127) and 0.8% of v; a step can be off by a few
    percent of lr, more where m lies far below its block's maximum: held to lr a step."""
    from twotower.optim import AdamW

    params = make(torch.float32)
    ref = [torch.nn.Parameter(p.detach().cpu().double()) for p in params]
    a, b = AdamW(params, state_bits=bits, **HP), torch.optim.AdamW(ref, **HP)
    for k in range(20):
        set_grads(params, k)
        for p, r in zip(params, ref):
            r.grad = p.grad.cpu().double()
        a.step()
        b.step()
    lr = HP["lr"]
    for p, r in zip(params, ref):
        d = (p.detach().cpu().double() - r.detach()).abs()
        if bits == 32:
            # (a quotient of two rounded moments: its 24 u counts the sizes before cancellation,
            # |m| sums up to 10 terms; 2^4 more covers it)
            assert (d <= 16 * 20 * 28 * U * lr + 40 * U * (r.detach().abs() + 20 * lr)).all()
        else:
            assert (d <= 20 * lr).all() and (d.numel() == 0 or d.mean() <= 0.1 * 20 * lr)


def test_gradients_not_contiguous_and_expanded():
    from twotower.optim import AdamW

    params = make(torch.float32, [(33, 65), (40, 20)])
    opt = AdamW(params, **HP)
    params[0].grad = torch.full((1, 1), 0.3, device="cuda").expand(33, 65)
    params[1].grad = torch.randn(20, 40, device="cuda").t()
    before = snapshot(opt, params)
    opt.step()
    check_step(opt, params, before, 32)


def test_groups_scheduler_and_added_group():
    from twotower.optim import AdamW

    params = make(torch.float32, [(100,), (300, 3), (7,)])
    opt = AdamW([{"params": params[:1], "lr": 1e-2}, {"params": params[1:2], "weight_decay": 0.0}],
                **HP)
    sch = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    hps = [dict(HP, lr=1e-2), dict(HP, weight_decay=0.0)]
    for k in range(2):
        set_grads(params, k)
        before = snapshot(opt, params[:2])
        opt.step()
        for i in range(2):
            check_step(opt, params[i:i + 1], before[i:i + 1], 32, hps[i])
        sch.step()
        for h in hps:
            h["lr"] *= 0.5
    moments = [opt.state[p]["exp_avg"].clone() for p in params[:2]]
    opt.add_param_group({"params": params[2:], "lr": 1e-3})
    assert all(torch.equal(opt.state[p]["exp_avg"], m) for p, m in zip(params, moments))
    set_grads(params, 9)
    before = snapshot(opt, params)
    opt.step()
    for i, h in enumerate(hps + [dict(HP, lr=1e-3)]):
        check_step(opt, params[i:i + 1], before[i:i + 1], 32, h)


def test_step_hooks_and_closure():
    from twotower.optim import AdamW

    params = make(torch.float32, [(50,)])
    opt = AdamW(params, **HP)
    seen = []
    opt.register_step_pre_hook(lambda o, a, k: seen.append(("pre", o is opt)))
    opt.register_step_post_hook(lambda o, a, k: seen.append(("post", int(o.state[params[0]]["step"]))))
    set_grads(params, 0)
    assert opt.step(lambda: 7.0) == 7.0
    assert seen == [("pre", True), ("post", 1)]


def test_more_tensors_than_one_launch_takes():
    from twotower.optim import AdamW

    params = make(torch.float32, [(1 + i % 300,) for i in range(1000)])
    opt = AdamW(params, **HP)
    set_grads(params, 1, skip=(0, 415, 416, 999))
    before = snapshot(opt, params)
    opt.step()
    check_step(opt, params, before, 32)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trips(bits):
    from twotower.optim import AdamW

    params = make(torch.float32)
    opt = AdamW(params, state_bits=bits, **HP)
    for k in range(3):
        set_grads(params, k)
        opt.step()
    sd = copy.deepcopy(opt.state_dict())
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(twin, lr=1.0, state_bits=bits)
    other.load_state_dict(sd)
    assert other.param_groups[0]["lr"] == HP["lr"]
    dc = copy.deepcopy(opt)  # a copied optimizer holds its own parameters and moments
    set_grads(params, 7)
    for p, t, c in zip(params, twin, dc.param_groups[0]["params"]):
        t.grad, c.grad = p.grad.clone(), p.grad.clone()
    for o in (opt, other, dc):
        o.step()
    for p, t, c in zip(params, twin, dc.param_groups[0]["params"]):
        assert torch.equal(p, t) and torch.equal(p, c)
        for k, v in opt.state[p].items():
            assert torch.equal(v, other.state[t][k]) and torch.equal(v, dc.state[c][k])
    # the other width takes the values: 8 -> 32 exactly what the codes stand for
    wide = AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=40 - bits,
                 **HP)
    wide.load_state_dict(opt.state_dict())
    for p, q in zip(params, wide.param_groups[0]["params"]):
        m, v = opt.moments_of(p)
        mw, vw = wide.moments_of(q)
        if bits == 8:
            assert ((m - mw).abs() <= 2 * U * m.abs()).all()
            assert ((v - vw).abs() <= 2 * U * v.abs()).all()
        elif p.numel():
            # half a level: r = sqrt(|m| / s) is off by 1 / 254, so m by at most s / 127 (1 + 1 / 508)
            top = blocks(m).abs().amax(1, keepdim=True)
            assert (blocks(m - mw).abs() <= top / 126.0).all()
            assert (blocks(v - vw).abs() <= blocks(v).amax(1, keepdim=True) * 4 / 505.0).all()
            assert ((vw > 0) == (v > 0)).all()


def test_loads_torch_adamw_state():
    from twotower.optim import AdamW

    params = make(torch.float32)
    t = torch.optim.AdamW(params, **HP)
    set_grads(params, 0)
    t.step()
    opt = AdamW(params, **HP)
    opt.load_state_dict(t.state_dict())
    for p in params:
        assert torch.equal(opt.state[p]["exp_avg"], t.state[p]["exp_avg"])
        assert int(opt.state[p]["step"]) == 1
    set_grads(params, 1)
    before = snapshot(opt, params)
    opt.step()
    check_step(opt, params, before, 32)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_advances_on_replay(bits):
    from twotower.optim import AdamW

    params, twin = make(torch.float32), make(torch.float32)
    a, b = AdamW(params, state_bits=bits, **HP), AdamW(twin, state_bits=bits, **HP)
    set_grads(params, 0)
    for p, q in zip(params, twin):
        q.grad = p.grad.clone()
    a.step()
    b.step()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        a.step()
    for k in range(4):
        set_grads(twin, 50 + k)
        for p, q in zip(params, twin):
            p.grad.copy_(q.grad)
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        if k == 1:  # a state loaded between replays is what the next replay goes on from
            a.load_state_dict(copy.deepcopy(a.state_dict()))
        for p, q in zip(params, twin):
            assert torch.equal(p, q)
            for key, v in a.state[p].items():
                assert torch.equal(v, b.state[q][key])


def test_what_a_captured_step_forbids():
    """A replay would go on with the tables and gradients of the capture."""
    from twotower.optim import AdamW

    p, q = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], **HP)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with pytest.raises(RuntimeError, match="captured"):
        opt.add_param_group({"params": [q]})
    assert len(opt.param_groups) == 1
    old = p.data
    p.grad = None
    p.data = p.data.bfloat16()
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    p.data = old
    before = p.detach().clone()
    graph.replay()
    torch.cuda.synchronize()
    assert (p != before).all()


def test_replaced_storage_is_followed():
    from twotower.optim import AdamW

    params = make(torch.float32, [(100,), (50,)])
    opt = AdamW(params, **HP)
    set_grads(params, 0)
    opt.step()
    old = params[0].data
    kept = old.clone()
    params[0].data = old.clone()
    set_grads(params, 1)
    before = snapshot(opt, params)
    opt.step()
    check_step(opt, params, before, 32)
    assert torch.equal(old, kept)


def test_non_finite_gradients_stay_where_they_are():
    """A NaN gradient: its own parameter, and with 8 bits the moments of its block of 256 from the
    next step on; no other."""
    from twotower.optim import AdamW

    for bits in (32, 8):
        params = make(torch.float32, [(1000,)])
        opt = AdamW(params, state_bits=bits, **HP)
        set_grads(params, 0)
        params[0].grad[300] = float("nan")
        params[0].grad[900] = float("inf")
        opt.step()
        bad = ~torch.isfinite(params[0].detach())
        assert bad[300] and bad.sum() <= 2
        set_grads(params, 1)
        opt.step()
        bad = ~torch.isfinite(params[0].detach())
        assert not bad[:256].any() and not bad[512:768].any()
        if bits == 32:
            assert bad.sum() <= 2


def test_zero_gradients_and_extremes():
    """All-zero blocks (scale 0), tiny gradients whose squares leave f32's range, large ones."""
    from twotower.optim import AdamW

    for bits in (32, 8):
        params = make(torch.float32, [(1024,)])
        opt = AdamW(params, state_bits=bits, **HP)
        g = torch.zeros(1024)
        g[256:512] = 1e-25 * torch.arange(256)
        g[512:768] = 1e15 * torch.arange(256)
        params[0].grad = g.cuda()
        for _ in range(3):
            opt.step()
        assert torch.isfinite(params[0]).all()
        m, v = opt.moments_of(params[0])
        assert torch.isfinite(m).all() and torch.isfinite(v).all()
        assert not m[:256].any() and not v[:256].any()


def test_past_32_bit_offsets():
    """One bf16 tensor of 2^31 + 700 elements, 8-bit moments: its last block moves as a small
    tensor's does."""
    from twotower.optim import AdamW

    n = 2 ** 31 + 700
    big = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    gen = torch.Generator().manual_seed(0)
    tail = torch.randn(700, generator=gen).bfloat16()
    gt = torch.randn(700, generator=gen).bfloat16()
    with torch.no_grad():
        big[-700:] = tail.cuda()
    big.grad = torch.zeros_like(big)
    big.grad[-700:] = gt.cuda()
    small = torch.nn.Parameter(tail.clone().cuda())
    small.grad = gt.cuda()
    a, b = AdamW([big], state_bits=8, **HP), AdamW([small], state_bits=8, **HP)
    for _ in range(2):
        a.step()
        b.step()
    assert torch.equal(big[-700:], small)
    assert not big[:1 << 20].any()
    assert torch.equal(a.state[big]["exp_avg"][-700:], b.state[small]["exp_avg"])


def test_refusals_on_the_device():
    from twotower.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    buf = torch.zeros(100, device="cuda")
    a, b = torch.nn.Parameter(buf[:60]), torch.nn.Parameter(buf[50:])
    a.grad, b.grad = torch.zeros_like(a), torch.zeros_like(b)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([a, b]).step()
    q = torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([q]).step()
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        AdamW([torch.nn.Parameter(torch.zeros(3, device="cuda").half())]).moments()
    p.grad = torch.sparse_coo_tensor(torch.zeros(1, 1, dtype=torch.int64, device="cuda"),
                                     torch.ones(1, device="cuda"), (10,))
    with pytest.raises(ValueError, match="dense"):
        AdamW([p]).step()
    p.grad = torch.zeros(10, device="cuda")
    fresh = AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            fresh.step()
    fresh.step()
    sd = fresh.state_dict()
    with pytest.raises(ValueError, match="do not match"):
        AdamW([p, torch.nn.Parameter(torch.zeros(3, device="cuda"))]).load_state_dict(sd)
    with pytest.raises(ValueError, match="elements"):
        AdamW([torch.nn.Parameter(torch.zeros(11, device="cuda"))]).load_state_dict(sd)


@pytest.mark.parametrize("bits", [32, 8])
def test_train_step_takes_adamw(bits):
    """TwoTowerTrainStep(weight_decay, state_bits): its update is AdamW's on its own gradients, and
    its checkpoint carries the moments."""
    from test_gpu_train import _setup
    from twotower.optim import AdamW
    from twotower.train import TwoTowerTrainStep

    E, B, S, N = 64, 8, 5, 2
    it, bt = _setup(E)
    it.eval()
    step = TwoTowerTrainStep(it, bt, lr=1e-2, weight_decay=0.1, state_bits=bits)
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    Ht = it.text_encoder.get_sentence_embedding_dimension()
    ids = lambda *s: torch.randint(0, 3, s, generator=gen, dtype=torch.int32).cuda()  # noqa: E731
    args = (rn(B, S, E), torch.ones(B, S).cuda(), rn(B, Ht), rn(B, N, Ht), ids(B), ids(B),
            ids(B, N), ids(B, N))
    twin = [torch.nn.Parameter(p.detach().clone()) for p in step.params.values()]
    ref = AdamW(twin, lr=1e-2, weight_decay=0.1, state_bits=bits)
    for _ in range(3):
        step.step(*args)
        for t, k in zip(twin, step.params):
            t.grad = step.g[k].clone()
        ref.step()
        assert all(torch.equal(p, t) for p, t in zip(step.params.values(), twin))
    model = torch.nn.ModuleList([it, bt])
    sd = step.optimizer_state_dict(model)
    assert sd["param_groups"][0]["weight_decay"] == 0.1
    want = [m.clone() for m in step.adamw.moments()]
    step.load_optimizer_state_dict(model, sd)
    assert step.t == 3 and int(step.adamw.steps[0]) == 3
    for a, b in zip(step.adamw.moments(), want):
        # decoded, coded again: the same codes, the scale within a rounding
        assert ((a - b).abs() <= (0 if bits == 32 else 4 * U) * b.abs()).all()
    with pytest.raises(ValueError):
        TwoTowerTrainStep(it, bt, state_bits=16)
