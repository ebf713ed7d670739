"""Refusals of the fused training step that need no GPU."""
import pytest


def test_a_recurrent_tower_is_told_where_it_trains():
    from twotower import BuyerTower
    from twotower.train import TwoTowerTrainStep

    with pytest.raises(ValueError, match="'recurrent'.*autograd"):
        TwoTowerTrainStep(None, BuyerTower(64, "recurrent"))
