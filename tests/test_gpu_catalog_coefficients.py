"""Gradients of bf16 catalog log-probabilities: the given item's coefficient, which is most of a row's
gradient, is not rounded to bf16.

Tolerance: a coefficient c is off by 4 T of its parts (see test_gpu_catalog), and of the other items
rounded by half a step, 2^-8 of itself; the products add at most 4096 terms in sequence (4096 u); the given
item's keeps 16 bits (2^-16, as test_gpu_catalog's two-part coefficients); the result is rounded by half a
step of itself, which may move by the rest's own half step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


def reference(x, w, ids, b, temp, g, ge):
    """dx, dw in 64 bits and their tolerances."""
    x, w = x.double(), w.double()
    s = 1.0 / temp
    l = x @ w.t() * s
    if b is not None:
        l = l + b.double()
    lse = torch.logsumexp(l, 1)
    lp = l - lse[:, None]
    p = torch.exp(lp)
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    ent = -plp.sum(1)
    has = (ids >= 0) & (ids < w.shape[0])
    rows = torch.nonzero(has)[:, 0]
    gg = g.double() * has
    c = -gg[:, None] * p - ge.double()[:, None] * (plp + p * ent[:, None])
    own = torch.zeros_like(c)
    rows = rows[torch.isfinite(l[rows, ids[rows]])]
    c[rows, ids[rows]] += gg[rows]
    own[rows, ids[rows]] = 1.0
    fin = torch.where(torch.isfinite(l), l, lse[:, None])
    rng = (fin.max(1).values - fin.min(1).values).max().item()
    T = U * ((x.shape[1] + 4) * s * x.norm(dim=1).max().item() * w.norm(dim=1).max().item()
             + min(w.shape[0] / 8, 4096) + 64)
    parts = p * (gg.abs() + ge.double().abs() * (rng + 1 + ent))[:, None] + c.abs()
    bound = parts * (4 * T + 4096 * U) + c.abs() * torch.where(own > 0, 2.0 ** -16, BF16_HALF)
    dx, dw = s * (c @ w), s * (c.t() @ x)
    tx, tw = s * (bound @ w.abs()), s * (bound.t() @ x.abs())
    half = lambda t, d: (t + BF16_HALF * d.abs()) * (1 + BF16_HALF) + 1e-30  # noqa: E731
    return dx, dw, half(tx, dx), half(tw, dw)


def check(x, w, ids, b, g, ge, temp=0.07):
    from twotower.losses import catalog_log_probs

    dx, dw, tx, tw = reference(x, w, ids, b, temp, g, ge)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = catalog_log_probs(xl, wl, ids, temp, b, entropy=True)
    torch.autograd.backward([r.log_prob, r.entropy], [g, ge])
    for got, want, tol in ((xl.grad, dx, tx), (wl.grad, dw, tw)):
        err = (got.double() - want).abs()
        assert (err <= tol).all(), (err / tol).max().item()
    only, = torch.autograd.grad([catalog_log_probs(xl, w, ids, temp, b, entropy=True).log_prob], [xl], [g])
    full = catalog_log_probs(xl, wl, ids, temp, b)
    both = torch.autograd.grad([full.log_prob], [xl, wl], [g])
    assert torch.equal(only, both[0])


def make(N, V, E, bias, kind):
    gen = torch.Generator().manual_seed(N + V + E)
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1)
    if kind == "spread":
        ids = torch.randint(0, V, (N,), generator=gen)
    elif kind == "popular":  # half of the rows share three items, the first and the last among them
        ids = torch.randint(0, V, (N,), generator=gen)
        ids[::2] = torch.tensor([0, V // 2, V - 1])[torch.randint(0, 3, ((N + 1) // 2,), generator=gen)]
    else:
        ids = torch.full((N,), V - 1)
    x = torch.nn.functional.normalize(torch.randn(N, E, generator=gen) / E ** 0.5 + 0.4 * w[ids], dim=1)
    ids[3::11] = -1
    ids[5::31] = V + 1
    b = None
    if bias:
        b = torch.randn(V, generator=gen)
        b[torch.rand(V, generator=gen) < 0.1] = float("-inf")
        b = b.cuda()
    g, ge = torch.randn(N, generator=gen), 0.05 * torch.randn(N, generator=gen)
    g[7::13] = 0.0
    return x.bfloat16().cuda(), w.bfloat16().cuda(), ids.cuda(), b, g.cuda(), ge.cuda()


@pytest.mark.parametrize("N,V,E", [
    (65, 70, 64), (100, 3000, 192), (130, 1, 64), (200, 9000, 100), (300, 33000, 64),
    (700, 22001, 192), (1281, 20100, 64), (2049, 8200, 512), (4100, 66000, 64),  # (in chunks)
    (769, 50021, 384)])                                                          # (rows in registers)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kind", ["spread", "popular", "one"])
def test_the_given_items_coefficient_is_exact(N, V, E, bias, kind):
    check(*make(N, V, E, bias, kind))


def test_in_a_graph():
    """Replays with other rows and ids in the same buffers."""
    from twotower.losses import catalog_log_probs

    x, w, ids, b, g, ge = make(300, 5000, 128, True, "popular")

    def go(x, ids):
        xl, wl = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        r = catalog_log_probs(xl, wl, ids, 0.07, b)
        return torch.autograd.grad([r.log_prob], [xl, wl], [g])

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    xs, si = x.clone(), ids.clone()
    with torch.cuda.stream(st):
        go(xs, si)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = go(xs, si)
    for k in range(3):
        xs.copy_(x.roll(k, 0))
        si.copy_(ids.roll(2 * k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, go(xs, si)))
