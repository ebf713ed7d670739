"""The recurrence, the catalog log-probabilities and AdamW together: a sequence-aware buyer tower
trained against a whole catalog, and the evaluation and retrieval paths that read its result."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain_step(Wg, bg, items, hist, w, ids, temp):
    """The same step's loss in f64 torch operations (autograd)."""
    x = items[hist]
    h = torch.zeros(hist.shape[0], items.shape[1], dtype=torch.float64)
    for t in range(hist.shape[1]):
        la = torch.nn.functional.logsigmoid(x[:, t] @ Wg.t() + bg) * w[:, t:t + 1]
        h = torch.exp(la) * h - torch.expm1(la) * x[:, t]
    z = torch.nn.functional.normalize(h, dim=1)
    lp = torch.log_softmax(z @ items.t() / temp, dim=1)
    return -lp[torch.arange(len(ids)), ids].mean()


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_the_three_operators(bits):
    """Two steps: gate and item table both trained.  Gradients against the f64 form (f32 sums of at
    most 300 terms through four operators: 2^-14 of the largest), then the update is AdamW's."""
    from twotower import BuyerTower
    from twotower.losses import CatalogSoftmaxLoss
    from twotower.optim import AdamW

    torch.manual_seed(0)
    E, B, S, V = 64, 24, 9, 300
    tower = BuyerTower(E, "recurrent").cuda()
    gen = torch.Generator().manual_seed(1)
    table = torch.nn.Parameter(torch.nn.functional.normalize(
        torch.randn(V, E, generator=gen), dim=1).cuda())
    crit = CatalogSoftmaxLoss(0.07)
    opt = AdamW([{"params": tower.parameters(), "lr": 1e-2}, {"params": [table]}], lr=1e-3,
                state_bits=bits)
    for step in range(2):
        hist = torch.randint(0, V, (B, S), generator=gen)
        w = torch.tensor([0.0, 1.0, 5.0, 10.0])[torch.randint(0, 4, (B, S), generator=gen)]
        w[:, 0] = 1.0
        ids = torch.randint(0, V, (B,), generator=gen)
        Wd, bd, td = (p.detach().cpu().double().requires_grad_()
                      for p in (tower.gate.weight, tower.gate.bias, table))
        want = _plain_step(Wd, bd, td, hist, w.double(), ids, 0.07)
        want.backward()
        opt.zero_grad()
        loss = crit(tower(table[hist.cuda()], w.cuda()), table, ids.cuda())
        loss.backward()
        assert abs(loss.item() - want.item()) <= 2.0 ** -16 * want.item()
        params = [tower.gate.weight, tower.gate.bias, table]
        for p, r in zip(params, (Wd, bd, td)):
            assert (p.grad.cpu().double() - r.grad).abs().max() <= 2.0 ** -14 * r.grad.abs().max()
        before = [p.detach().clone() for p in params]
        opt.step()
        if step == 0:  # the first step of Adam moves every weight by about lr against its gradient
            for p, b, lr in zip(params, before, (1e-2, 1e-2, 1e-3)):
                moved = p.detach() - b * (1 - lr * 1e-2)
                big = p.grad.abs() > 1e-4
                assert torch.equal(torch.sign(moved[big]), -torch.sign(p.grad[big]))
                assert (moved[big].abs() <= lr * 1.0001).all()
                assert (moved[big].abs() >= lr * 0.999).all()


def test_trained_tower_reaches_the_serving_paths():
    """EmbeddingEncoder-style use: embeddings from the recurrent tower into VectorDatabase's
    retrieval, log_probs and the evaluator's likelihood."""
    from twotower import BuyerTower, VectorDatabase
    from twotower.evaluation import Evaluator

    E, V, B = 64, 500, 7
    rng = np.random.default_rng(0)
    emb = rng.standard_normal((V, E)).astype(np.float32)
    db = VectorDatabase(E)
    db.build_index(emb, [f"p{i}" for i in range(V)])
    torch.manual_seed(0)
    tower = BuyerTower(E, "recurrent").cuda()
    unit = emb / np.linalg.norm(emb, axis=1, keepdims=True)

    class Encoder:
        def encode_buyers(self, histories, mode="A"):
            S = max(len(h) for h in histories)
            x, w = np.zeros((len(histories), S, E), np.float32), np.zeros((len(histories), S), np.float32)
            for i, h in enumerate(histories):
                for j, ev in enumerate(h):
                    x[i, j], w[i, j] = unit[int(ev["product_id"][1:])], 1.0
            with torch.no_grad():
                return tower(torch.from_numpy(x), torch.from_numpy(w)).numpy()

    pairs = [(f"b{i}", [{"product_id": f"p{p}"} for p in rng.integers(0, V, 3 + i)],
              {f"p{p}" for p in rng.integers(0, V, 2)} | {"unknown"}) for i in range(B)]
    q = Encoder().encode_buyers([h for _, h, _ in pairs])
    l = (q.astype(np.float64) / np.linalg.norm(q, axis=1, keepdims=True)) @ unit.astype(np.float64).T / 0.07
    lse = np.log(np.exp(l).sum(1))
    lp, ent, alt = db.log_probs(q, ["p3", "nope"] + ["p9"] * (B - 2), top=5)
    assert abs(lp[0] - (l[0, 3] - lse[0])) < 1e-4 and np.isnan(lp[1])
    p = np.exp(l - lse[:, None])
    np.testing.assert_allclose(ent, -(p * np.log(p)).sum(1), atol=1e-4)
    got = db.retrieve_batch(q, k=5)
    assert [[x for x, _ in r] for r in alt] == [[x for x, _ in r] for r in got]
    assert abs(alt[2][0][1] - (l[2].max() - lse[2])) < 1e-4
    lp1, _, alt1 = db.log_probs(q[0])
    assert lp1 is None and alt1 == [[]]
    ev = Evaluator(Encoder(), db, config_path=None, batch_size=3)
    res = ev.evaluate_likelihood(pairs)
    want = [l[i, int(x[1:])] - lse[i] for i, (_, _, rel) in enumerate(pairs) for x in rel if x != "unknown"]
    assert res["items"] == len(want) and abs(res["log_prob_mean"] - np.mean(want)) < 1e-4
    assert abs(res["perplexity"] - np.exp(-np.mean(want))) < 1e-2
    assert ev.evaluate_likelihood([("b", pairs[0][1], {"unknown"})]) == {}
    for bad in ((q[:, :10], None), (q, ["p1"])):
        with pytest.raises(ValueError):
            db.log_probs(*bad)


def test_log_probs_without_queries():
    from twotower import VectorDatabase

    db = VectorDatabase(64)
    db.build_index(np.eye(5, 64, dtype=np.float32), [f"p{i}" for i in range(5)])
    lp, ent, alt = db.log_probs(np.zeros((0, 64), np.float32), [], top=3)
    assert lp.shape == ent.shape == (0,) and alt == []
    lp, ent, alt = db.log_probs(np.eye(2, 64, dtype=np.float64), ["p0", "p1"], top=9)
    assert len(alt[0]) == 5 and abs(alt[1][0][1] - lp[1]) < 1e-5
