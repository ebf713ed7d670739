"""The top alternatives of the catalog log-probabilities (csrc/tt_catalog.hip) where 32-bit logits
cannot order them: products that cancel.  The order is that of the product in 64 bits, ties to the lower id; every place is written."""
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
@pytest.mark.parametrize("V", [1, 2, 40])
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
@pytest.mark.parametrize("V", [1, 2, 40])
def test_items_orthogonal_to_the_query(norm, V):
    """Items orthogonal to the query but for their own rounding, at norms of 1 to 1000."""
    gen = torch.Generator().manual_seed(int(norm) + V)
    for E in (64, 448):
        for _ in range(5):
            x = torch.nn.functional.normalize(torch.randn(1, E, generator=gen).double(), dim=1)
            w = torch.randn(V, E, generator=gen).double()
            w = torch.nn.functional.normalize(w - (w @ x.t()) * x, dim=1)
            check((norm * x).float().cuda(), (norm * w).float().cuda(), 0.07, min(V, 10))
