"""The gated linear recurrence (csrc/tt_recur.hip) against its definition in 64 bits.

Tolerances.  f32: a gate is off by at most ~6 roundings (2^-24 each, relative, of A or of 1 - A,
whichever is smaller), a state update by 2 more of the state's size; errors of earlier events decay
with the state, so after M = 1 / (1 - A) events of memory the roundings add up to at most M 2^-23
of the largest state.  The gates drawn here keep M below 2^7 except where a test says otherwise:
2^7 2^-23 = 2^-16 of the largest state, and the same for the gradients (64 more for products).
Outputs in bf16 add half a step, 2^-8 of the value (torch.finfo(bf16).eps / 2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32_TOL = 2.0 ** -16
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


def reference(x, g, w, h0, dh=None, dlast=None):
    """Event by event in f64 on the CPU, gradients from the formulas."""
    x, g = x.double().cpu(), g.double().cpu()
    B, S, D = x.shape
    w = torch.ones(B, S, dtype=torch.float64) if w is None else w.double().cpu()
    live = (w > 0)
    ww = torch.where(live, w, torch.zeros_like(w)).unsqueeze(2)
    lv = live.unsqueeze(2)
    g = torch.where(lv, g, torch.zeros_like(g))
    x = torch.where(lv, x, torch.zeros_like(x))
    la = torch.where(lv, ww * torch.nn.functional.logsigmoid(g), torch.zeros_like(g))
    A, nA = torch.exp(la), -torch.expm1(la)
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double().cpu()
    hs = [h]
    for t in range(S):
        h = A[:, t] * h + nA[:, t] * x[:, t]
        hs.append(h)
    H = torch.stack(hs, dim=1)
    out = {"h": H[:, 1:], "last": h}
    if dh is None and dlast is None:
        return out
    R = torch.zeros(B, D, dtype=torch.float64) if dlast is None else dlast.double().cpu()
    G = torch.zeros_like(x)
    for t in range(S - 1, -1, -1):
        G[:, t] = R if dh is None else R + dh[:, t].double().cpu()
        R = A[:, t] * G[:, t]
    out["dx"] = nA * G * lv
    out["dgate"] = G * (H[:, :-1] - x) * ww * A * torch.sigmoid(-g)
    out["dh0"] = R
    return out


def make(B, S, D, dt, weighted, h0, seed=0, scale=1.0, shift=1.5):
    gen = torch.Generator().manual_seed(seed + 7 * B + 31 * S + D)
    x = torch.randn(B, S, D, generator=gen).to(dt)
    g = (torch.randn(B, S, D, generator=gen).clamp(-3, 3) * scale + shift).to(dt)
    w = None
    if weighted:
        w = torch.tensor([0.0, 1.0, 1.0, 5.0, 10.0, 0.25, -1.0])[
            torch.randint(0, 7, (B, S), generator=gen)]
    s0 = torch.randn(B, D, generator=gen) if h0 else None
    return x, g, w, s0


def cu(*ts):
    return [t.cuda() if t is not None else None for t in ts]


def close(got, want, dt, tol=F32_TOL):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    if want.numel() == 0:
        return
    bound = tol * max(want.abs().max().item(), 1e-30)
    if dt == torch.bfloat16:
        bound = bound + BF16_HALF * want.abs() + 1e-38
    bad = (got - want).abs() > bound
    assert not bad.any(), f"max error {(got - want).abs().max().item()}, bound {bound}"


SHAPES = [(1, 1, 1), (1, 1, 384), (3, 0, 32), (2, 7, 37), (5, 16, 64), (2, 17, 130), (300, 33, 48),
          (1, 127, 96), (1, 128, 96), (1, 1000, 384), (2, 4099, 66), (7, 300, 257)]


@pytest.mark.parametrize("B,S,D", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("weighted,h0", [(False, False), (True, True)])
def test_forward_and_gradients_vs_f64(B, S, D, dt, weighted, h0):
    from twotower.recurrence import gated_scan

    x, g, w, s0 = make(B, S, D, dt, weighted, h0)
    gen = torch.Generator().manual_seed(3)
    dh = torch.randn(B, S, D, generator=gen).to(dt)
    dl = torch.randn(B, D, generator=gen)
    ref = reference(x, g, w, s0, dh, dl)
    xc, gc, wc, sc = cu(x, g, w, s0)
    leaves = [xc.requires_grad_(), gc.requires_grad_()] + ([sc.requires_grad_()] if h0 else [])
    h, last = gated_scan(xc, gc, wc, sc)
    assert h.dtype == dt and last.dtype == torch.float32
    close(h.detach(), ref["h"], dt)
    close(last.detach(), ref["last"], torch.float32)
    grads = torch.autograd.grad([h, last], leaves, [dh.cuda(), dl.cuda()])
    close(grads[0], ref["dx"], dt)
    close(grads[1], ref["dgate"], dt)
    if h0:
        close(grads[2], ref["dh0"], torch.float32)
    # last state only: its gradient alone
    ref = reference(x, g, w, s0, None, dl)
    _, last = gated_scan(xc, gc, wc, sc, states=False)
    grads = torch.autograd.grad([last], leaves, [dl.cuda()])
    close(grads[0], ref["dx"], dt)
    close(grads[1], ref["dgate"], dt)


def test_gradient_vs_differences():
    """Central differences of the kernel's own forward (f32): step 2^-6, truncation ~ step^2 =
    2^-12 of the third derivative, rounding 2^-20 / 2^-6."""
    from twotower.recurrence import gated_scan

    x, g, w, s0 = make(2, 40, 8, torch.float32, True, True, seed=5)
    xc, gc, wc, sc = cu(x, g, w, s0)
    up = torch.randn(2, 40, 8, generator=torch.Generator().manual_seed(1)).cuda()

    def f(a, b, c):
        h, last = gated_scan(a, b, wc, c)
        return ((h * up).double().sum() + last.double().sum())

    leaves = [t.clone().requires_grad_() for t in (xc, gc, sc)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    eps = 2.0 ** -6
    with torch.no_grad():
        for i in range(3):
            gen = torch.Generator().manual_seed(i)
            v = torch.randn(leaves[i].shape, generator=gen).cuda()
            a, b = [list(leaves) for _ in range(2)]
            a[i], b[i] = leaves[i] + eps * v, leaves[i] - eps * v
            num = ((f(*a) - f(*b)) / (2 * eps)).item()
            ana = (grads[i] * v).double().sum().item()
            assert abs(num - ana) <= 2.0 ** -8 * max(1.0, abs(ana))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_long_memory_keeps_its_precision(dt):
    """Gates of 9 to 14 (memories to 1e6 events) over 20000 events: A rounds next to 1, and the
    state must not drift.  Rounding of the state itself: 2^-24 an event, at most 20000 2^-24 =
    2^-9.7 of its size if all fell one way (bound used); a rounded A would be off by
    2^-25 / (1 - A) = 3% of it."""
    from twotower.recurrence import gated_scan

    gen = torch.Generator().manual_seed(2)
    x = (torch.rand(1, 20000, 64, generator=gen) + 0.5).to(dt)
    g = (9 + 5 * torch.rand(1, 1, 64, generator=gen)).expand(1, 20000, 64).contiguous().to(dt)
    ref = reference(x, g, None, None)
    _, last = gated_scan(x.cuda(), g.cuda(), states=False)
    assert ((last.cpu().double() - ref["last"]).abs() <= 2.0 ** -9.7 * ref["last"].abs()).all()
    assert ((last.cpu().double() - ref["last"]).abs().mean() <= 2.0 ** -16)


@pytest.mark.parametrize("weight", [2, 5, 10])
def test_weight_counts_events(weight):
    """An event of weight w = w equal events (the same formula in exact arithmetic)."""
    from twotower.recurrence import gated_scan

    x, g, _, s0 = make(2, 6, 64, torch.float32, False, True)
    xc, gc, sc = cu(x, g, s0)
    w = torch.full((2, 6), float(weight)).cuda()
    _, a = gated_scan(xc, gc, w, sc, states=False)
    _, b = gated_scan(xc.repeat_interleave(weight, 1), gc.repeat_interleave(weight, 1), None, sc,
                      states=False)
    assert (a - b).abs().max().item() <= F32_TOL * b.abs().max().item()


@pytest.mark.parametrize("S", [5, 400])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_padding_holds_anything(S, dt):
    """Padded events (weight 0, negative, NaN) with NaN and inf in x and gate: the state passes bit
    for bit, their gradients are 0, and nothing reaches the others."""
    from twotower.recurrence import gated_scan

    x, g, w, s0 = make(2, S, 66, dt, True, True)
    w[1] = 0.0  # a history of padding alone
    w[0, 2] = float("nan")
    pad = ~(w > 0)
    clean = [t.clone() for t in (x, g)]
    x[pad] = float("nan")
    g[pad] = float("-inf")
    dh = torch.randn(2, S, 66).to(dt)
    outs = []
    for xx, gg in (clean, (x, g)):
        xc, gc, wc, sc, dc = cu(xx, gg, w, s0, dh)
        leaves = [xc.requires_grad_(), gc.requires_grad_(), sc.requires_grad_()]
        h, last = gated_scan(xc, gc, wc, sc)
        gr = torch.autograd.grad([h, last], leaves, [dc, torch.ones_like(last)])
        outs.append([h.detach(), last.detach(), *gr])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert torch.equal(outs[1][1][1].cpu(), s0[1])
    for gr in outs[1][2:4]:
        assert not gr[pad.cuda()].any()


def test_infinite_and_extreme_gates():
    """gate +inf keeps the state, -inf replaces it; +-100 likewise in f32; an infinite weight too."""
    from twotower.recurrence import gated_scan

    x = torch.full((1, 1, 6), 3.0).cuda()
    g = torch.tensor([[[float("inf"), float("-inf"), 100.0, -100.0, 0.0, 1.0]]]).cuda()
    s0 = torch.full((1, 6), 7.0).cuda()
    for w in (None, torch.ones(1, 1).cuda(), torch.full((1, 1), 3.0).cuda()):
        _, last = gated_scan(x, g, w, s0, states=False)
        assert last[0, :4].tolist() == [7.0, 3.0, 7.0, 3.0]
    w = torch.full((1, 1), float("inf")).cuda()
    _, last = gated_scan(x[..., 4:], g[..., 4:], w, s0[:, 4:], states=False)
    assert last.tolist() == [[3.0, 3.0]]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dt):
    """Slices of wider rows (odd offsets), transposed batches, expanded rows: the same bits as
    contiguous copies, and no write outside."""
    from twotower.recurrence import gated_scan

    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(3, 50, 201, generator=gen).to(dt).cuda()
    x, g = wide[:, :, 1:97], wide[:, :, 104:200]
    w = torch.randint(0, 4, (3, 100), generator=gen).float().cuda()[:, ::2]
    a = gated_scan(x, g, w)
    b = gated_scan(x.contiguous(), g.contiguous(), w.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    xt = torch.randn(50, 3, 96, generator=gen).to(dt).cuda().transpose(0, 1)
    gx = torch.randn(1, 50, 96, generator=gen).to(dt).cuda().expand(3, 50, 96)
    a, b = gated_scan(xt, gx), gated_scan(xt.contiguous(), gx.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    xl = xt.clone().requires_grad_()
    gl = torch.randn(1, 50, 96, generator=gen).to(dt).cuda().requires_grad_()
    h, last = gated_scan(xl, gl.expand(3, 50, 96))  # a broadcast gate: its gradients are summed
    dg, = torch.autograd.grad([last.sum()], [gl])
    ref = reference(xl.detach(), gl.detach().expand(3, 50, 96), None, None, None,
                    torch.ones(3, 96))["dgate"]
    assert dg.shape == (1, 50, 96)
    err = (dg.double().cpu() - ref.sum(0, keepdim=True)).abs().max().item()
    assert err <= (F32_TOL if dt == torch.float32 else 4 * BF16_HALF) * ref.abs().max().item()


def test_one_event_at_a_time_equals_the_whole():
    """Serving form: 40 calls with S = 1 carry the state that one call over 40 events reaches."""
    from twotower.recurrence import gated_scan

    x, g, w, s0 = make(3, 40, 384, torch.float32, True, True)
    xc, gc, wc, sc = cu(x, g, w, s0)
    _, whole = gated_scan(xc, gc, wc, sc, states=False)
    st = sc
    for t in range(40):
        _, st = gated_scan(xc[:, t:t + 1], gc[:, t:t + 1], wc[:, t:t + 1], st, states=False)
    assert torch.equal(st, whole)


def test_side_stream_and_graph_replay():
    from twotower.recurrence import gated_scan

    x, g, w, s0 = make(2, 700, 96, torch.bfloat16, True, True)
    xc, gc, wc, sc = cu(x, g, w, s0)
    want = gated_scan(xc, gc, wc, sc)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = gated_scan(xc, gc, wc, sc)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs = xc.clone().requires_grad_()
    dl = torch.ones_like(sc)
    with torch.cuda.stream(st):  # warm-up on the side stream, then capture forward + backward
        for _ in range(2):
            torch.autograd.grad([gated_scan(xs, gc, wc, sc, states=False)[1]], [xs], [dl])
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        _, last = gated_scan(xs, gc, wc, sc, states=False)
        dx, = torch.autograd.grad([last], [xs], [dl])
    for k in range(3):
        with torch.no_grad():
            xs.copy_(xc * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        xe = xs.detach().clone().requires_grad_()
        le = gated_scan(xe, gc, wc, sc, states=False)[1]
        de, = torch.autograd.grad([le], [xe], [dl])
        assert torch.equal(last, le) and torch.equal(dx, de)


def test_offsets_past_32_bits():
    """A tensor of 2.2e9 elements seen through strides: the last history lies past 2^31."""
    from twotower.recurrence import gated_scan

    big = torch.zeros(2200, 1000, 1000, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(1, 40, 64, generator=gen).bfloat16().cuda()
    big[2199, :40, 900:964] = x[0]
    g = torch.zeros(2, 40, 64, dtype=torch.bfloat16, device="cuda")
    view = big[::2199][:, :40, 900:964]  # histories 0 and 2199: a stride of 2.2e9 elements
    h, last = gated_scan(view, g)
    want, wl = gated_scan(x, g[:1])
    assert torch.equal(h[1], want[0]) and torch.equal(last[1], wl[0])
    assert not h[0].any()


def test_buyer_tower_recurrent():
    """The tower's forward, its serving form and its gradients against autograd in f64."""
    from twotower import BuyerTower

    torch.manual_seed(0)
    E, B, S = 64, 5, 12
    tower = BuyerTower(E, "recurrent").cuda()
    gen = torch.Generator().manual_seed(1)
    items = torch.nn.functional.normalize(torch.randn(B, S, E, generator=gen), dim=2)
    w = torch.tensor([1.0, 5.0, 10.0])[torch.randint(0, 3, (B, S), generator=gen)]
    w[0, 7:] = 0.0
    w[3] = 0.0  # a buyer without events
    Wd = tower.gate.weight.detach().cpu().double().requires_grad_()
    bd = tower.gate.bias.detach().cpu().double().requires_grad_()
    h = torch.zeros(B, E, dtype=torch.float64)
    for t in range(S):
        la = torch.nn.functional.logsigmoid(items[:, t].double() @ Wd.t() + bd) * w[:, t:t + 1]
        h = torch.exp(la) * h - torch.expm1(la) * items[:, t].double()
    want = torch.nn.functional.normalize(h, dim=1)
    up = torch.randn(B, E, generator=gen).double()
    up[3] = 0.0  # (normalising a zero state divides its gradient by 1e-12)
    want.backward(up)
    got = tower(items.cuda(), w.cuda())
    assert (got[3] == 0).all()
    assert (got.detach().cpu().double() - want.detach()).abs().max().item() <= 2.0 ** -18
    got.backward(up.float().cuda())
    for a, b in ((tower.gate.weight.grad, Wd.grad), (tower.gate.bias.grad, bd.grad)):
        assert (a.cpu().double() - b).abs().max().item() <= 2.0 ** -16 * b.abs().max().item()
    with torch.no_grad():
        dirty = items.clone()
        dirty[w == 0] = float("nan")
        assert torch.equal(tower(dirty.cuda(), w.cuda()), got.detach())
        st = None
        for t in range(S):
            st = tower.recurrent_state(items[:, t:t + 1].cuda(), w[:, t:t + 1].cuda(), st)
        assert (tower.embed_state(st) - got.detach()).abs().max().item() <= 2.0 ** -18
        host = tower(items, w)  # host tensors in, host tensors out
    assert not host.is_cuda and torch.equal(host, got.detach().cpu())
    other = BuyerTower(E, "recurrent")
    other.load_state_dict({k: v.cpu() for k, v in tower.state_dict().items()})


def test_tower_states_of_other_types_and_no_buyers():
    from twotower import BuyerTower

    torch.manual_seed(0)
    tower = BuyerTower(64, "recurrent").cuda()
    st = torch.randn(3, 64, device="cuda").bfloat16()
    assert torch.equal(tower.embed_state(st), tower.embed_state(st.float()))
    x, w = torch.randn(3, 2, 64, device="cuda"), torch.ones(3, 2, device="cuda")
    assert torch.equal(tower.recurrent_state(x, w, st), tower.recurrent_state(x, w, st.float()))
    assert tower(x[:0], w[:0]).shape == (0, 64)
    assert torch.equal(tower.recurrent_state(x[:, :0], w[:, :0], st), st.float())
    assert not tower(x[:, :0], w[:, :0]).any()
