"""VectorDatabase.log_probs and Evaluator.evaluate_likelihood with a mapping that names rows which the
index does not have (a mapping file of a larger catalog)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _db():
    from twotower import VectorDatabase

    db = VectorDatabase(64)
    db.build_index(np.random.default_rng(0).standard_normal((40, 64)).astype(np.float32),
                   [f"p{i}" for i in range(40)])
    db.id_to_index = {**db.id_to_index, "gone": 40, "far": 2 ** 40, "below": -1}
    return db


def test_rows_outside_the_index_have_no_log_prob():
    db = _db()
    q = np.eye(5, 64, dtype=np.float32)
    lp, ent, _ = db.log_probs(q, ["p1", "gone", "far", "unknown", "below"])
    assert np.isfinite(lp[0]) and np.isnan(lp[1:]).all() and np.isfinite(ent).all()


def test_the_likelihood_leaves_them_out():
    from twotower.evaluation import Evaluator

    db = _db()
    q = np.eye(3, 64, dtype=np.float32)

    class Encoder:
        def encode_buyers(self, histories, mode="A"):
            return q[[h[0] for h in histories]]

    ev = Evaluator(Encoder(), db, config_path=None, batch_size=2)
    pairs = [("a", [0], {"p3", "gone"}), ("b", [1], {"far", "below"}), ("c", [2], {"p7"})]
    res = ev.evaluate_likelihood(pairs)
    lp, ent, _ = db.log_probs(q[[0, 2]], ["p3", "p7"])
    assert res["items"] == 2 and abs(res["log_prob_mean"] - lp.mean()) < 1e-6
    assert abs(res["entropy_mean"] - ent.mean()) < 1e-6
