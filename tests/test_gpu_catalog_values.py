"""Values of the catalog log-probabilities that several outputs share."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dt,N,V,E", [
    (torch.float32, 5, 50, 768), (torch.float32, 200, 1003, 64), (torch.bfloat16, 5, 205, 768),
    (torch.bfloat16, 130, 9000, 192), (torch.bfloat16, 700, 22001, 64),
    (torch.bfloat16, 769, 50021, 384)])
@pytest.mark.parametrize("bias", [False, True])
def test_an_alternative_and_the_given_item_have_one_value(dt, N, V, E, bias):
    """log_prob of the r-th alternative is its top_log_prob, from p next to 1 to the least: both come
    from one formula, rounded once.  Their 64-bit products are summed in different orders: they differ by
    up to E 2^-53 |x| |w| / temperature (log p next to 0 is a difference of two values of that size, so
    its 32-bit rounding is finer than this), and that may move the rounding by a last place."""
    from twotower.losses import catalog_log_probs

    gen = torch.Generator().manual_seed(N + V)
    w = torch.nn.functional.normalize(torch.randn(V, E, generator=gen), dim=1)
    at = torch.randint(0, V, (N,), generator=gen)
    far = torch.tensor([0.3, 0.6, 1.0])[torch.arange(N) % 3][:, None]
    x = torch.nn.functional.normalize(w[at] + far * torch.randn(N, E, generator=gen) / E ** 0.5, dim=1)
    x, w = x.to(dt).cuda(), w.to(dt).cuda()
    b = torch.randn(V, generator=gen).cuda() if bias else None
    for temp in (0.03, 0.07):
        r = catalog_log_probs(x, w, None, temp, b, top=20)
        l = x.double() @ w.double().t() / temp + (b.double() if bias else 0.0)
        lp = l - torch.logsumexp(l, 1, keepdim=True)
        assert temp > 0.03 or torch.exp(lp.max()) > 0.99
        for k in (0, 1, 2, 19):
            ids = r.top_ids[:, k].contiguous()
            one = catalog_log_probs(x, w, ids, temp, b).log_prob
            assert ((one - r.top_log_probs[:, k]).abs() 
                    <= 2 * U * one.abs() + 1.02 * E * 2.0 ** -53 / temp).all()
            # and it keeps its precision next to 0 (see test_gpu_catalog)
            want = lp.gather(1, ids[:, None])[:, 0]
            p = torch.exp(want)
            T = U * ((E + 4) / temp * 1.02 + min(V / 8, 4096) + 64)
            tol = torch.where(p > 0.5, 2 * T * (1 - p) / p, T + U * want.abs())
            tol = tol + U * (min(V / 8, 4096) + 64)
            assert ((r.top_log_probs[:, k].double() - want).abs() <= tol).all()
