"""Log-probabilities over a catalog (csrc/tt_catalog.hip, twotower.losses) against their definition
in 64 bits.

Tolerances, u = 2^-24, X and W the largest row norms, s = 1 / temperature.  A logit in f32 (exact
products of bf16, f32 accumulation) is off by at most (E + 4) u s X W; lse is off by no more than the
worst logit, plus the roundings of sum, exponential and logarithm: a lane adds at most V / 8 + 64
terms one after another (fewer in large catalogs, whose shares are split).  So
  T = u ((E + 4) s X W + min(V / 8, 4096) + 64)
bounds log_prob (its own logit is summed in 64 bits) and any log p.  The entropy sum p log p moves by
at most 2 T (1 + R) for logits in a range R.  A coefficient of the gradient products is off by 4 T
of itself (in bf16 also half a step, 2^-8), and the products add at most 4096 terms in sequence
(4096 u): the bound is that times |C| |w| (in 64 bits, element by element).  Outputs in bf16 add
half a step of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


def make(N, V, E, dt, seed=0, bias=False, drop=True):
    gen = torch.Generator().manual_seed(seed + 3 * N + 5 * V + E)
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1)
    ids = torch.randint(0, V, (N,), generator=gen)
    x = torch.nn.functional.normalize(torch.randn(N, E, generator=gen) / E ** 0.5 + 0.7 * w[ids],
                                      dim=1)
    if drop and N > 2:
        ids[::5] = -1
    b = None
    if bias:
        b = torch.randn(V, generator=gen)
        out = torch.rand(V, generator=gen) < 0.2
        out[0] = V > 1
        b[out] = float("-inf")
    return x.to(dt).cuda(), w.to(dt).cuda(), ids.cuda(), b.cuda() if bias else None


def reference(x, w, ids, b, temp, g=None, ge=None):
    x, w = x.double(), w.double()
    s = 1.0 / temp
    l = x @ w.t() * s
    if b is not None:
        l = l + b.double()
    lse = torch.logsumexp(l, 1)
    lp = l - lse[:, None]
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    has = ids >= 0
    out = {"log_prob": torch.where(has, lp.gather(1, ids.clamp(min=0)[:, None])[:, 0],
                                   torch.zeros_like(ent)), "entropy": ent, "logits": l, "lp": lp}
    fin = torch.where(torch.isfinite(l), l, lse[:, None])
    out["range"] = (fin.max(1).values - fin.min(1).values).max().item()
    X, W = x.norm(dim=1).max().item(), w.norm(dim=1).max().item()
    out["T"] = U * ((x.shape[1] + 4) * s * X * W + min(w.shape[0] / 8, 4096) + 64)
    if g is not None or ge is not None:
        c = torch.zeros_like(l)
        if g is not None:
            gg = g.double() * has
            c -= gg[:, None] * p
            # (an item that is taken out has no gradient; one of vanishing probability has)
            r = torch.nonzero(has & torch.isfinite(l.gather(1, ids.clamp(min=0)[:, None])[:, 0]))[:, 0]
            c[r, ids[r]] += gg[r]
        if ge is not None:
            c -= ge.double()[:, None] * p * torch.where(p > 0, lp + ent[:, None],
                                                        torch.zeros_like(p))
        out["dx"], out["dw"] = s * (c @ w), s * (c.t() @ x)
        # what of |c| a coefficient error is taken of: its parts before they cancel
        ca = p * ((g.double().abs() if g is not None else 0) * torch.ones_like(ent)
                  + (ge.double().abs() * (out["range"] + 1 + ent.abs()) if ge is not None else 0)
                  )[:, None] + c.abs()
        out["dx_size"], out["dw_size"] = s * (ca @ w.abs()), s * (ca.t() @ x.abs())
    return out


def check_grad(got, want, size, T, dt):
    tol = size * (4 * T + 4096 * U)
    if dt == torch.bfloat16:
        tol = tol + size * BF16_HALF + BF16_HALF * want.abs()
    assert got.dtype == dt
    err = (got.double() - want).abs()
    assert (err <= tol + 1e-30).all(), f"{(err / (tol + 1e-30)).max().item()} of the bound"


SHAPES = [(1, 1, 64), (1, 5, 64), (3, 64, 64), (5, 130, 128), (128, 128, 64), (129, 257, 192),
          (300, 1000, 384), (17, 70001, 64), (2, 20, 768), (64, 4099, 1024), (33, 333, 100),
          (1000, 37, 64), (40, 500, 7),
          (129, 1, 128), (300, 31, 128), (200, 33, 256), (700, 1090, 384), (385, 64, 384),
          (257, 999, 512), (130, 641, 640), (520, 2000, 768)]


@pytest.mark.parametrize("N,V,E", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_forward_and_gradients_vs_f64(N, V, E, dt, bias):
    from twotower.losses import catalog_log_probs

    temp = 0.07
    x, w, ids, b = make(N, V, E, dt, bias=bias)
    gen = torch.Generator().manual_seed(11)
    g, ge = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    ref = reference(x, w, ids, b, temp, g, ge)
    top = min(V, 32)
    with torch.no_grad():
        r = catalog_log_probs(x, w, ids, temp, b, entropy=True, top=top)
        one = catalog_log_probs(x, w, ids, temp, b, top=1)
    T = ref["T"]
    for a in (r, one):
        lp = ref["log_prob"]
        fin = torch.isfinite(lp)
        assert torch.equal(a.log_prob[~fin].double(), lp[~fin])
        # (its own rounding to f32 besides)
        assert ((a.log_prob.double() - lp)[fin].abs() <= T + U * lp[fin].abs()).all()
    assert one.entropy is None
    assert ((r.entropy.double() - ref["entropy"]).abs() <= 2 * T * (1 + ref["range"])).all()
    # alternatives: the exact order (64-bit logits of these inputs; stable: ties to the lower id)
    val, order = torch.sort(ref["logits"], dim=1, descending=True, stable=True)
    assert torch.equal(r.top_ids, order[:, :top])
    assert torch.equal(one.top_ids, order[:, :1])
    tl = ref["lp"].gather(1, r.top_ids)
    fin = torch.isfinite(tl)
    assert torch.equal(r.top_log_probs[~fin].double(), tl[~fin])
    assert ((r.top_log_probs.double() - tl)[fin].abs() <= T + U * tl[fin].abs()).all()
    # gradients of both, then of each alone
    for use_g, use_e in ((True, True), (True, False), (False, True)):
        ref = reference(x, w, ids, b, temp, g if use_g else None, ge if use_e else None)
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        r = catalog_log_probs(xl, wl, ids, temp, b, entropy=True)
        outs, ups = [], []
        if use_g:
            outs, ups = outs + [r.log_prob], ups + [g]
        if use_e:
            outs, ups = outs + [r.entropy], ups + [ge]
        dx, dw = torch.autograd.grad(outs, [xl, wl], ups)
        check_grad(dx, ref["dx"], ref["dx_size"], T, dt)
        check_grad(dw, ref["dw"], ref["dw_size"], T, dt)


@pytest.mark.parametrize("dt,N,V,E", [
    (torch.float32, 5, 200, 768), (torch.float32, 200, 1003, 64), (torch.bfloat16, 5, 205, 768),
    (torch.bfloat16, 130, 1000, 192), (torch.bfloat16, 700, 22001, 64),
    (torch.bfloat16, 769, 50021, 384)])
@pytest.mark.parametrize("bias", [False, True])
def test_log_prob_of_likely_items_keeps_its_precision(dt, N, V, E, bias):
    """log p = -log(1 + r), r the other items' share: its own logit's error does not enter (it is the
    same on both sides), the others' only with their share, which leaves the roundings of the sums.
    Of r = p_other / p: off by T r, and the sum by its roundings (V / 8 + 64 at most)."""
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(N + V)
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1)
    ids = torch.cat([torch.tensor([V - 1, 0]), torch.randint(0, V, (N - 2,), generator=gen)])
    x = torch.nn.functional.normalize(w[ids] + 0.6 * torch.randn(N, E, generator=gen) / E ** 0.5, dim=1)
    x, w, ids = x.to(dt).cuda(), w.to(dt).cuda(), ids.cuda()
    b = torch.randn(V, generator=gen).cuda() if bias else None
    ref = reference(x, w, ids, b, 0.05)
    r = catalog_log_probs(x, w, ids, 0.05, b, entropy=True)
    p = torch.exp(ref["log_prob"])
    tol = 2 * ref["T"] * (1 - p) / p + U * (min(V / 8, 4096) + 64)
    err = (r.log_prob.double() - ref["log_prob"]).abs()
    assert (p > 0.9).any() and (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_certain_rows_stay_at_0(dt):
    """One item has all the probability (the others' is below any float): log p and entropy are 0 and
    never past it."""
    from twotower.losses import catalog_log_probs

    x, w, ids, _ = make(300, 700, 192, dt, drop=False)
    r = catalog_log_probs(w[ids], w, ids, 0.002, entropy=True, top=3)
    T = U * ((192 + 4) * 500 * 1.01 + 700 / 8 + 64)
    assert (r.log_prob <= 0).all() and (r.top_log_probs <= 0).all() and (r.entropy >= 0).all()
    assert (r.log_prob >= -U * 152).all() and (r.entropy <= U * 152).all()
    assert (r.top_log_probs[:, 0] >= -T).all() and torch.equal(r.top_ids[:, 0], ids)


@pytest.mark.parametrize("N,V,E", [(1, 70, 64), (7, 141, 192), (33, 3001, 64), (64, 500, 128),
                                   (50, 20000, 64), (40, 9, 100),
                                   (3, 2100001, 64)])  # (the catalog in two chunks)
@pytest.mark.parametrize("bias", [False, True])
def test_few_bf16_rows_have_exact_gradients(N, V, E, bias):
    """Up to 64 rows the coefficients are held in two bf16 parts (2^-16 of them at most is lost): only
    the result is rounded, by half a step."""
    from twotower.losses import catalog_log_probs

    x, w, ids, b = make(N, V, E, torch.bfloat16, bias=bias, seed=3)
    gen = torch.Generator().manual_seed(17)
    g, ge = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    ref = reference(x, w, ids, b, 0.07, g, ge)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=True)
    torch.autograd.backward([r.log_prob, r.entropy], [g, ge])
    for got, key in ((xl.grad, "dx"), (wl.grad, "dw")):
        tol = ref[key + "_size"] * (4 * ref["T"] + 4096 * U + 2.0 ** -16) + BF16_HALF * ref[key].abs()
        # (the rounded value is itself off by the first part: its half step too)
        tol = tol * (1 + BF16_HALF) + 1e-30
        assert ((got.double() - ref[key]).abs() <= tol).all()


@pytest.mark.parametrize("N,V,E", [(33, 4000, 64), (500, 2500, 128), (200, 4001, 192)])
@pytest.mark.parametrize("bias", [False, True])
def test_without_alternatives_vs_f64(N, V, E, bias):
    from twotower.losses import catalog_log_probs

    x, w, ids, b = make(N, V, E, torch.float32, bias=bias)
    gen = torch.Generator().manual_seed(13)
    g, ge = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    ref = reference(x, w, ids, b, 0.07, g, ge)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=True)
    ok = torch.isfinite(ref["log_prob"])
    assert torch.equal(torch.isfinite(r.log_prob), ok)
    err = (r.log_prob.detach().double() - ref["log_prob"]).abs()[ok]
    assert (err <= ref["T"] + U * ref["log_prob"].abs()[ok]).all()
    err = (r.entropy.detach().double() - ref["entropy"]).abs()
    assert (err <= 2 * ref["T"] * (1 + ref["range"])).all()
    torch.autograd.backward([r.log_prob, r.entropy], [g, ge])
    check_grad(xl.grad, ref["dx"], ref["dx_size"], ref["T"], torch.float32)
    check_grad(wl.grad, ref["dw"], ref["dw_size"], ref["T"], torch.float32)


@pytest.mark.parametrize("N,V,E", [
    (300, 33000, 64), (700, 22001, 192), (2049, 8200, 512),  # 256 x 256 tiles, the last ones cut
    (1281, 20100, 64),                                       # dw: some tiles whole, the rest split
    (4100, 66000, 64),                                       # and in three chunks
    (769, 50021, 384), (1152, 29200, 384)])                  # rows kept in registers
@pytest.mark.parametrize("bias", [False, True])
def test_large_tiles(N, V, E, bias):
    test_forward_and_gradients_vs_f64(N, V, E, torch.bfloat16, bias)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_catalog_in_chunks(dt):
    """More logits than one chunk of coefficients holds (256 MB): partial sums across chunks."""
    from twotower.losses import catalog_log_probs

    N, V, E = 4096, 40009 if dt == torch.bfloat16 else 17001, 64
    x, w, ids, b = make(N, V, E, dt, bias=True)
    g = torch.full((N,), 1.0 / N).cuda()
    ref = reference(x, w, ids, b, 0.1, g)
    xl, wl = x.requires_grad_(), w.requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.1, b)
    dx, dw = torch.autograd.grad([r.log_prob], [xl, wl], [g])
    check_grad(dx, ref["dx"], ref["dx_size"], ref["T"], dt)
    check_grad(dw, ref["dw"], ref["dw_size"], ref["T"], dt)
    only, = torch.autograd.grad([catalog_log_probs(xl, w.detach(), ids, 0.1, b).log_prob], [xl], [g])
    assert torch.equal(only, dx)
    only, = torch.autograd.grad([catalog_log_probs(x.detach(), wl, ids, 0.1, b).log_prob], [wl], [g])
    assert torch.equal(only, dw)


def test_gradient_vs_differences():
    """Central differences of the forward in f32: step 2^-5 in a unit direction; truncation ~
    (s step)^2 of the third derivative (s = 1 here), rounding 2^-20 / step."""
    from twotower.losses import catalog_log_probs

    x, w, ids, b = make(20, 200, 64, torch.float32, bias=True, drop=False)
    b = torch.where(torch.isinf(b), torch.zeros_like(b), b)
    up = torch.randn(20, generator=torch.Generator().manual_seed(0)).cuda()

    def f(x, w):
        r = catalog_log_probs(x, w, ids, 1.0, b, entropy=True)
        return (r.log_prob.double() * up).sum() + (r.entropy.double() * up).sum()

    xl, wl = x.requires_grad_(), w.requires_grad_()
    grads = torch.autograd.grad(f(xl, wl), [xl, wl])
    eps = 2.0 ** -5
    for i in range(2):
        v = torch.randn((x, w)[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        v /= v.norm(dim=1, keepdim=True)
        with torch.no_grad():
            a, c = [[x, w] for _ in range(2)]
            a[i], c[i] = a[i] + eps * v, c[i] - eps * v
            num = ((f(*a) - f(*c)) / (2 * eps)).item()
        ana = (grads[i] * v).double().sum().item()
        assert abs(num - ana) <= 2.0 ** -8 * max(1.0, abs(ana))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_taken_out_items_and_dead_rows_hold_anything(dt, fill):
    """Items with bias -inf / the lowest float, rows without gradients: garbage there changes no
    other result and no gradient."""
    from twotower.losses import catalog_log_probs

    x, w, ids, b = make(150, 400, 128, dt, bias=True)
    out = torch.isinf(b)
    b[out.nonzero()[::2, 0]] = torch.finfo(torch.float32).min
    ids[out[ids.clamp(min=0)] & (ids >= 0)] = 1 if not out[1] else int((~out).nonzero()[0])
    dead = torch.zeros(150, dtype=torch.bool).cuda()
    dead[::7] = True
    g = torch.randn(150, generator=torch.Generator().manual_seed(0)).cuda()
    g[dead] = 0.0
    res = []
    for dirty in (False, True):
        xx, ww = x.clone(), w.clone()
        if dirty:
            ww[out] = fill
            xx[dead] = fill
        xl, wl = xx.requires_grad_(), ww.requires_grad_()
        r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=True, top=5)
        dx, dw = torch.autograd.grad([r.log_prob], [xl, wl], [g])
        res.append((r.log_prob.detach()[~dead], r.entropy.detach()[~dead], r.top_ids[~dead],
                    r.top_log_probs[~dead], dx, dw))
    for a, c in zip(*res):
        assert torch.equal(a, c)
    assert not res[1][4][dead].any() and not res[1][5][out].any()
    assert not out[res[1][2]].any()


def test_rows_with_nothing_left_and_ids_taken_out():
    from twotower.losses import CatalogSoftmaxLoss, catalog_log_probs

    x, w, ids, _ = make(6, 50, 64, torch.float32, drop=False)
    ids[1] = -1
    b = torch.full((50,), float("-inf")).cuda()
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=True, top=3)
    want = torch.full((6,), float("-inf")).cuda()
    want[1] = 0.0
    assert torch.equal(r.log_prob, want) and not r.entropy.any()
    assert r.top_ids.tolist() == [[0, 1, 2]] * 6 and torch.isinf(r.top_log_probs).all()
    dx, dw = torch.autograd.grad([r.log_prob, r.entropy], [xl, wl], [torch.ones(6).cuda()] * 2)
    assert not dx.any() and not dw.any()
    b[7] = 0.0  # one item left: probability 1; the others' ids have none
    r = catalog_log_probs(x, w, torch.tensor([7, 7, 7, 3, -1, 7]).cuda(), 0.07, b, entropy=True,
                          top=2)
    assert (r.log_prob[[0, 1, 2, 5]].abs() <= 64 * U * 15).all() and r.log_prob[4] == 0
    assert r.log_prob[3] == float("-inf") and (r.entropy.abs() <= 64 * U * 15).all()
    assert r.top_ids.tolist() == [[7, 0]] * 6
    # the loss counts rows with an item; none at all: 0
    crit = CatalogSoftmaxLoss(0.5)
    got = crit(x, w, ids)
    ref = reference(x, w, ids, None, 0.5)
    assert abs(got.item() + ref["log_prob"].sum().item() / 5) <= ref["T"] + 8 * U * 10
    assert crit(x, w, torch.full_like(ids, -1)).item() == 0.0
    both = CatalogSoftmaxLoss(0.5, entropy_weight=0.1)(x, w, ids)
    has = ids >= 0
    assert abs(both.item() - (got.item() - 0.1 * ref["entropy"][has].mean().item())) <= 1e-5


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_equal_items_rank_by_id(dt):
    """Catalogs of equal vectors (a few kinds; one kind): equal logits in the order of their ids."""
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(0)
    for kinds, V in ((3, 5000), (1, 1000), (1, 70), (40, 9001)):
        base = torch.randn(kinds, 64, generator=gen)
        which = torch.randint(0, kinds, (V,), generator=gen)
        w = base[which].to(dt).cuda()
        x = torch.randn(4, 64, generator=gen).to(dt).cuda()
        r = catalog_log_probs(x, w, top=min(32, V))
        sc = (x.double() @ base.to(dt).cuda().double().t())[:, which.cuda()]
        order = torch.sort(sc, dim=1, descending=True, stable=True).indices
        assert torch.equal(r.top_ids, order[:, :32])


def test_nan_rows_stay_rows():
    """A NaN in a row (or in one item) gives NaN where it belongs; ids stay in range."""
    from twotower.losses import catalog_log_probs

    x, w, ids, _ = make(10, 300, 64, torch.float32, drop=False)
    x[3, 5] = float("nan")
    r = catalog_log_probs(x, w, ids, entropy=True, top=8)
    assert torch.isnan(r.log_prob[3]) and torch.isnan(r.entropy[3])
    ok = torch.arange(10) != 3
    assert torch.isfinite(r.log_prob[ok]).all() and torch.isfinite(r.top_log_probs[ok]).all()
    assert ((r.top_ids >= 0) & (r.top_ids < 300)).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dt):
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(1)
    big = torch.randn(300, 300, generator=gen).to(dt).cuda()
    x, w = big[:50, 3:131], big[50:, 100:228]
    ids = torch.arange(100, device="cuda")[::2]
    b = torch.randn(500, generator=gen).cuda()[::2]
    a = catalog_log_probs(x, w, ids, bias=b, entropy=True, top=4)
    c = catalog_log_probs(x.contiguous(), w.contiguous(), ids.contiguous(), bias=b.contiguous(),
                          entropy=True, top=4)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    xt = torch.randn(128, 50, generator=gen).to(dt).cuda().t()
    wl = w.contiguous().requires_grad_()
    xs = torch.randn(1, 128, generator=gen).to(dt).cuda().requires_grad_()
    r1 = catalog_log_probs(xt, wl, ids)
    assert torch.equal(r1.log_prob, catalog_log_probs(xt.contiguous(), wl, ids).log_prob)
    # a broadcast query: its gradient is the sum over the rows
    r = catalog_log_probs(xs.expand(50, 128), wl, ids)
    dx, = torch.autograd.grad([r.log_prob.sum()], [xs])
    ref = reference(xs.detach().expand(50, 128), w, ids, None, 0.07, torch.ones(50).cuda())
    assert dx.shape == (1, 128)
    size = ref["dx_size"].sum(0, keepdim=True)
    tol = size * (4 * ref["T"] + 4096 * U + (2 * BF16_HALF if dt == torch.bfloat16 else 0))
    want = ref["dx"].sum(0, keepdim=True)
    # (autograd's sum of 50 rows in dt)
    tol = tol + ref["dx"].abs().sum(0, keepdim=True) * (50 * U if dt == torch.float32
                                                        else 2 * BF16_HALF)
    assert ((dx.double() - want).abs() <= tol).all()


def test_no_rows_and_single_rows():
    from twotower.losses import catalog_log_probs

    w = torch.randn(10, 64).cuda().requires_grad_()
    x = torch.zeros(0, 64).cuda().requires_grad_()
    r = catalog_log_probs(x, w, torch.zeros(0, dtype=torch.int64).cuda(), entropy=True, top=3)
    assert r.log_prob.shape == (0,) and r.top_ids.shape == (0, 3)
    dx, dw = torch.autograd.grad([r.log_prob.sum()], [x, w])
    assert dx.shape == (0, 64) and not dw.any()


def test_runs_repeat_and_other_streams_and_graphs():
    from twotower.losses import catalog_log_probs

    x, w, ids, b = make(700, 5000, 128, torch.bfloat16, bias=True)
    g = torch.randn(700, generator=torch.Generator().manual_seed(0)).cuda()

    def go(x):
        xl, wl = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        r = catalog_log_probs(xl, wl, ids, 0.07, b, entropy=True, top=6)
        dx, dw = torch.autograd.grad([r.log_prob, r.entropy], [xl, wl], [g, g])
        return [r.log_prob.detach(), r.entropy.detach(), r.top_ids, r.top_log_probs, dx, dw]

    want = go(x)
    assert all(torch.equal(p, q) for p, q in zip(go(x), want))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = go(x)
    st.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    xs = x.clone()
    with torch.cuda.stream(st):
        go(xs)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = go(xs)
    for k in range(3):
        xs.copy_(x * (1 - 0.3 * k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, go(xs)))


def test_offsets_past_32_bits():
    """6M x 384 items (2.3e9 elements): the last rows' products, ids and gradients."""
    from twotower.losses import catalog_log_probs

    V, E = 6_000_000, 384
    w = torch.zeros(V, E, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(0)
    tail = torch.nn.functional.normalize(torch.randn(70, E, generator=gen), dim=1).bfloat16().cuda()
    w[-70:] = tail
    x = tail[[3, 69]].contiguous()
    ids = torch.tensor([V - 67, V - 1]).cuda()
    xl, wl = x.requires_grad_(), w.requires_grad_()
    r = catalog_log_probs(xl, wl, ids, 0.07, entropy=True, top=3)
    l = x.detach().double() @ tail.double().t() / 0.07
    lse = torch.logsumexp(torch.cat([l, torch.full((2, 1), math.log(V - 70)).cuda().double()], 1), 1)
    # (V - 70 logits of 0: an exact sum but for 4096 u)
    assert ((r.log_prob.detach().double() - (l[[0, 1], [3, 69]] - lse)).abs() <= 4096 * U).all()
    order = torch.sort(l, dim=1, descending=True).indices[:, :3] + V - 70
    assert torch.equal(r.top_ids, order)
    dx, dw = torch.autograd.grad([r.log_prob.sum()], [xl, wl])
    p = torch.exp(l - lse[:, None])
    c = -p
    c[0, 3] += 1
    c[1, 69] += 1
    want = c.t() @ x.detach().double() / 0.07
    size = (p + c.abs()).t() @ x.detach().double().abs() / 0.07
    assert ((dw[-70:].double() - want).abs() <= size * 3 * BF16_HALF).all()


def test_results_changed_in_place_before_the_backward_pass():
    from twotower.losses import catalog_log_probs

    x, w, ids, _ = make(9, 200, 64, torch.float32)
    grads = []
    for change in (False, True):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        r = catalog_log_probs(xl, wl, ids)
        lp = r.log_prob
        lp = lp.mul_(2.0) if change else lp * 2.0
        lp.sum().backward()
        grads.append((xl.grad, wl.grad))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_one_tensor_as_queries_and_items():
    from twotower.losses import catalog_log_probs

    x, _, _, _ = make(70, 5, 64, torch.float32, drop=False)
    ids = torch.arange(70, device="cuda").roll(1)
    a, b, c = (x.clone().requires_grad_() for _ in range(3))
    catalog_log_probs(a, a, ids).log_prob.sum().backward()
    catalog_log_probs(b, c, ids).log_prob.sum().backward()
    assert torch.equal(a.grad, b.grad + c.grad)


def test_ids_outside_the_catalog_are_rows_without_an_item():
    from twotower.losses import CatalogSoftmaxLoss, catalog_log_probs

    x, w, ids, _ = make(12, 50, 64, torch.float32, drop=False)
    grads = []
    for none in (-1, 50, 2 ** 62, -2 ** 62):
        i = ids.clone()
        i[3], i[7] = none, none
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = CatalogSoftmaxLoss(0.1, 0.2)(xl, wl, i)
        loss.backward()
        assert (catalog_log_probs(x, w, i).log_prob[[3, 7]] == 0).all()
        grads.append((loss.detach(), xl.grad, wl.grad))
    for g in grads[1:]:
        assert all(torch.equal(a, b) for a, b in zip(g, grads[0]))


def test_refusals_on_the_device():
    from twotower.losses import CatalogSoftmaxLoss, catalog_log_probs

    x, w, ids, b = make(4, 40, 64, torch.float32, bias=True)
    for args, kw, exc in (((x.half(), w.half()), {}, TypeError), ((x, w.bfloat16()), {}, TypeError),
                          ((x, w[:, :32]), {}, ValueError), ((x[0], w), {}, ValueError),
                          ((x, w[:0]), {}, ValueError), ((x, w), dict(ids=ids[:2]), ValueError),
                          ((x, w), dict(ids=ids.int()), ValueError),
                          ((x, w), dict(bias=b[:3]), ValueError), ((x, w), dict(top=33), ValueError),
                          ((x, w[:5]), dict(top=6), ValueError),
                          ((x, w), dict(top=-1), ValueError),
                          ((x, w), dict(temperature=0.0), ValueError),
                          ((x, w), dict(temperature=1e-39), ValueError),
                          ((x, w), dict(temperature=float("nan")), ValueError),
                          ((x, w), dict(bias=b.cpu()), ValueError)):
        with pytest.raises(exc):
            catalog_log_probs(*args, **kw)
    bg = torch.zeros(40, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError):
        catalog_log_probs(x, w, ids, bias=bg).log_prob.sum().backward()
    with pytest.raises(ValueError):
        CatalogSoftmaxLoss(0.0)
