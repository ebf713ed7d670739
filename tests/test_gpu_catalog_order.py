"""The top alternatives of the catalog log-probabilities (csrc/tt_catalog.hip) where 32-bit logits
cannot order them: products that cancel, crowds of items closer than a 32-bit sum resolves.  The
order is that of the product in 64 bits, ties to the lower id; every place is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact(x, w, temp, b=None):
    l = x.double() @ w.double().t() * (1.0 / temp)
    return l if b is None else l + b.double()


def order(l, top):
    return torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top]


def run(x, w, temp, top, b=None):
    """catalog_log_probs' alternatives, with the freshly freed memory that its outputs may get holding
    a mark: a place that is not written shows it."""
    from twotower.losses import catalog_log_probs

    n = x.shape[0]
    junk = [torch.full((n, top), -7, dtype=torch.int64, device="cuda") for _ in range(4)]
    junk += [torch.full((n, top), 1e9, device="cuda") for _ in range(4)]
    del junk
    r = catalog_log_probs(x, w, None, temp, b, top=top)
    return r.top_ids, r.top_log_probs


def check(x, w, temp, top, b=None):
    ids, lp = run(x, w, temp, top, b)
    l = exact(x, w, temp, b)
    assert torch.equal(ids, order(l, top))
    # log p: (E + 4) roundings of the products' size, as test_gpu_catalog derives it
    T = U * ((x.shape[1] + 4) / temp * x.double().norm(dim=1).max().item()
             * w.double().norm(dim=1).max().item() + min(w.shape[0] / 8, 4096) + 64)
    want = (l - torch.logsumexp(l, 1, keepdim=True)).gather(1, ids)
    assert ((lp.double() - want).abs() <= T + U * want.abs()).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 40, 700, 5000])
def test_products_that_cancel(dt, V):
    """x = (c, c, 0, ...), w_v = (r_v, -r_v, 0, ...): every exact logit is 0, the 32-bit ones are what
    the products' rounding leaves."""
    gen = torch.Generator().manual_seed(V)
    for c in (100.0, 1e4, 1e6):
        r = torch.randn(V, generator=gen)
        w, x = torch.zeros(V, 64), torch.zeros(3, 64)
        w[:, 0], w[:, 1] = r, -r
        x[:, :2] = c * torch.tensor([1.0, 1.1, 0.9])[:, None]
        check(x.to(dt).cuda(), w.to(dt).cuda(), 0.07, min(V, 32))


@pytest.mark.parametrize("norm", [1.0, 100.0, 1000.0])
@pytest.mark.parametrize("V", [1, 2, 40, 300])
def test_items_orthogonal_to_the_query(norm, V):
    """Items orthogonal to the query but for their own rounding, at norms of 1 to 1000."""
    gen = torch.Generator().manual_seed(int(norm) + V)
    for E in (64, 448):
        for _ in range(5):
            x = torch.nn.functional.normalize(torch.randn(1, E, generator=gen).double(), dim=1)
            w = torch.randn(V, E, generator=gen).double()
            w = torch.nn.functional.normalize(w - (w @ x.t()) * x, dim=1)
            check((norm * x).float().cuda(), (norm * w).float().cuda(), 0.07, min(V, 10))


def crowd(N, V, E, members, dt, seed):
    """A catalog with ``members`` items (at random places) around each of 3 vectors, their elements a
    few last bits apart, and queries near one of the three."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1)
    centre = torch.nn.functional.normalize(torch.randn(3, E, generator=gen), dim=1)
    at = torch.randperm(V, generator=gen)[:3 * members]
    ulp = torch.finfo(dt).eps
    near = centre.repeat_interleave(members, 0)
    hit = torch.rand(near.shape, generator=gen) < (0.5 if dt == torch.float32 else 2.0 / E)
    w[at] = near * (1 + ulp * torch.randint(-2, 3, near.shape, generator=gen) * hit)
    x = torch.nn.functional.normalize(
        centre[torch.randint(0, 3, (N,), generator=gen)]
        + 0.3 * torch.randn(N, E, generator=gen) / E ** 0.5, dim=1)
    return x.to(dt).cuda(), w.to(dt).cuda(), gen


@pytest.mark.parametrize("seed", range(20))
def test_a_crowd_of_nearly_equal_items(seed):
    """60 items that differ in their last bits (one text encoded in different batches)."""
    x, w, _ = crowd(5, 3000, 384, 60, torch.float32, seed)
    check(x, w, 0.07, 10)


@pytest.mark.parametrize("dt,N,V,E,members", [
    (torch.float32, 1, 200000, 64, 3000),      # many segments of a row
    (torch.float32, 40, 9001, 100, 1500), (torch.float32, 150, 20000, 64, 700),
    (torch.bfloat16, 1, 150000, 384, 4000), (torch.bfloat16, 33, 10007, 384, 1000),
    (torch.bfloat16, 140, 25000, 256, 900),    # tiles of 128
    (torch.bfloat16, 300, 33000, 64, 1500),    # tiles of 256
    (torch.bfloat16, 384, 90000, 384, 700)])   # rows kept in registers
@pytest.mark.parametrize("bias", [False, True])
def test_large_crowds(dt, N, V, E, members, bias):
    """More of them than any fixed number of candidates, over the whole catalog."""
    x, w, gen = crowd(N, V, E, members, dt, N + V)
    b = None
    if bias:
        b = torch.where(torch.rand(V, generator=gen) < 0.3, float("-inf"),
                        2.0 ** -20 * torch.randint(0, 3, (V,), generator=gen)).cuda()
    for top in (1, 10, 32):
        check(x, w, 0.07, top, b)


def test_a_crowd_in_a_graph_and_on_another_stream():
    x, w, _ = crowd(40, 9001, 64, 800, torch.float32, 3)
    from twotower.losses import catalog_log_probs

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        r = catalog_log_probs(x, w, None, 0.07, top=12)
    st.synchronize()
    assert torch.equal(r.top_ids, order(exact(x, w, 0.07), 12))
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        r = catalog_log_probs(xs, w, None, 0.07, top=12)
    for k in range(4):  # replays with and without a crowd among the alternatives
        xs.copy_(x if k % 2 == 0 else -x)
        graph.replay()
        torch.cuda.synchronize()
        e = catalog_log_probs(xs, w, None, 0.07, top=12)
        assert torch.equal(r.top_ids, order(exact(xs, w, 0.07), 12))
        assert torch.equal(r.top_ids, e.top_ids) and torch.equal(r.top_log_probs, e.top_log_probs)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_in_parts(dt, monkeypatch):
    """More rows than the alternatives' workspace is given memory for: taken in parts, the last a shorter
    one; each row's result is its own."""
    from twotower import kernels
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(0)
    x = torch.nn.functional.normalize(torch.randn(103, 64, generator=gen), dim=1).to(dt).cuda()
    w = torch.nn.functional.normalize(torch.randn(1200, 64, generator=gen), dim=1).to(dt).cuda()
    ids = torch.randint(0, 1200, (206,), generator=gen).cuda()[::2]
    b = torch.randn(1200, generator=gen).cuda()
    want = catalog_log_probs(x, w, ids, 0.07, b, entropy=True, top=7)
    sizes = []
    make = kernels._catalog_ws_bytes
    monkeypatch.setattr(kernels, "_catalog_ws_bytes", lambda n, *a: sizes.append(n) or make(n, *a))
    row = 1200 // 4 + 7 * 16 + 64 * 15 * 8
    for limit, part in ((row * 20 + 40, 20), (1, 1)):
        sizes.clear()
        monkeypatch.setattr(kernels, "CATALOG_TOP_BYTES", limit)
        got = catalog_log_probs(x, w, ids, 0.07, b, entropy=True, top=7)
        assert sorted(sizes) == sorted({part, 103 % part} - {0})
        assert torch.equal(got.top_ids, want.top_ids)
        T = U * (68 * 1.02 / 0.07 + 150 + 64)  # (other tiles may sum in another order)
        for p, q in ((got.log_prob, want.log_prob), (got.top_log_probs, want.top_log_probs)):
            assert ((p - q).abs() <= 2 * T + 2 * U * q.abs()).all()
        assert ((got.entropy - want.entropy).abs() <= 4 * T * 40).all()
    sizes.clear()
    catalog_log_probs(x, w, ids, 0.07, b)  # (without alternatives: one call)
    assert sizes == [103]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,share", [(1, 300000, 1.0), (33, 50000, 0.5), (300, 20000, 0.2), (2, 17000, 1.0)])
def test_many_copies_of_one_item(dt, N, V, share):
    """Catalogs with thousands of copies of one vector (items without a text): the lowest ids of them."""
    gen = torch.Generator().manual_seed(V)
    w = torch.nn.functional.normalize(torch.randn(V, 64, generator=gen), dim=1)
    same = torch.rand(V, generator=gen) < share
    same[0] = True  # (the one they are copies of)
    w[same] = w[0].clone()
    x = torch.nn.functional.normalize(w[same][:1] + 0.05 * torch.randn(N, 64, generator=gen), dim=1)
    x, w = x.to(dt).cuda(), w.to(dt).cuda()
    for top in (1, 32):
        ids, _ = run(x, w, 0.07, top)
        # (their 64-bit logits are equal by construction, whatever order a sum takes)
        assert torch.equal(ids, torch.nonzero(same)[:top, 0].cuda().expand(N, top))
