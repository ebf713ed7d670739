"""BuyerTower on MI355X: drop-in for the reference module.

Reference: src/models/buyer_tower.py (class BuyerTower :9).  Same constructor, submodule
names (``attention`` = Linear(E,H) -> ReLU -> Linear(H,1), so checkpoint keys
``buyer_tower.attention.{0,2}.{weight,bias}`` load unchanged), methods and errors.  The
forward arithmetic is the HIP kernels of csrc/tt_buyer.hip (and csrc/tt_recur.hip for the
addition aggregation_method="recurrent", which the reference does not have); inputs on the host are moved
to the HIP device and results moved back, so CPU-tensor callers keep working on an MI355X
box.  There is no CPU compute path: without a HIP device the forward raises.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, kernels


class BuyerTower(nn.Module):
    """Mirror of reference ``BuyerTower`` (buyer_tower.py:9-146)."""

    def __init__(self, embedding_dim: int = 384, aggregation_method: str = "attention",
                 attention_hidden_dim: int = 128):
        super().__init__()
        self.embedding_dim = embedding_dim
        self.aggregation_method = aggregation_method
        if aggregation_method == "attention":
            self.attention = nn.Sequential(
                nn.Linear(embedding_dim, attention_hidden_dim),
                nn.ReLU(),
                nn.Linear(attention_hidden_dim, 1),
            )
        elif aggregation_method == "weighted_avg":
            pass
        elif aggregation_method == "recurrent":
            if embedding_dim % 32:
                raise ValueError("aggregation_method 'recurrent' needs an embedding_dim that is a "
                                 f"multiple of 32, got {embedding_dim}")
            self.gate = nn.Linear(embedding_dim, embedding_dim)
            nn.init.constant_(self.gate.bias, 2.0)  # starts with a memory of about 8 events
        else:
            raise ValueError(f"Unknown aggregation method: {aggregation_method}")

    @staticmethod
    def _on_device(t: torch.Tensor) -> torch.Tensor:
        return t if t.is_cuda else t.to(_lib.device())

    def weighted_average(self, item_embeddings: torch.Tensor,
                         weights: torch.Tensor) -> torch.Tensor:
        """reference :43-68 -> tt_weighted_avg_l2_f32"""
        home = item_embeddings.device
        out = kernels.weighted_avg_l2(self._on_device(item_embeddings), self._on_device(weights))
        return out.to(home)

    def attention_aggregation(self, item_embeddings: torch.Tensor,
                              weights: torch.Tensor) -> torch.Tensor:
        """reference :70-101 -> tt_attn_agg_l2_f32"""
        home = item_embeddings.device
        l0, l2 = self.attention[0], self.attention[2]
        dev = _lib.device()
        if torch.is_grad_enabled() and any(p.requires_grad for p in self.parameters()):
            from .autograd_ops import AttnAggFn  # training: HIP forward + backward

            out = AttnAggFn.apply(self._on_device(item_embeddings), self._on_device(weights),
                                  l0.weight.to(dev), l0.bias.to(dev), l2.weight.to(dev),
                                  l2.bias.to(dev))
            return out.to(home)
        out = kernels.attn_agg_l2(self._on_device(item_embeddings), self._on_device(weights),
                                  l0.weight.to(dev), l0.bias.to(dev), l2.weight.to(dev),
                                  l2.bias.to(dev))
        return out.to(home)

    # ------------------------------------------------------------ recurrent (an addition)
    def _gates(self, items: torch.Tensor) -> torch.Tensor:
        """Gate logits of item vectors [B, S, E] f32 (device, contiguous)."""
        from .autograd_ops import LinearFn

        b, s, e = items.shape
        W, bias = (t.to(items.device, torch.float32).contiguous()
                   for t in (self.gate.weight, self.gate.bias))
        return LinearFn.apply(items.view(b * s, e), W, bias).view(b, s, e)

    def recurrent_state(self, item_embeddings: torch.Tensor, weights: torch.Tensor,
                        state: torch.Tensor = None) -> torch.Tensor:
        """The buyer state [B, E] after the histories item_embeddings [B, S, E] (events in time
        order, padding marked by weight 0), starting from ``state`` (None: a new buyer).  The
        serving form: keep the state per buyer and pass each new event as S = 1."""
        from .recurrence import gated_scan

        if self.aggregation_method != "recurrent":
            raise ValueError("recurrent_state needs aggregation_method 'recurrent', this tower "
                             f"has '{self.aggregation_method}'")
        if item_embeddings.dim() != 3 or item_embeddings.shape[2] != self.embedding_dim:
            raise ValueError(f"item_embeddings must be [B, S, {self.embedding_dim}], got "
                             f"{tuple(item_embeddings.shape)}")
        home = item_embeddings.device
        items = self._on_device(item_embeddings).to(torch.float32).contiguous()
        w = self._on_device(weights).to(torch.float32)
        # a padded event's vector may hold anything: its gate logits are computed from zeros
        items = torch.where((w > 0).unsqueeze(2), items, torch.zeros_like(items))
        h0 = self._on_device(state) if state is not None else None
        if items.shape[1] == 0 or items.shape[0] == 0:
            gate = items
        else:
            gate = self._gates(items)
        return gated_scan(items, gate, w, h0, states=False)[1].to(home)

    def embed_state(self, state: torch.Tensor) -> torch.Tensor:
        """Buyer embedding of a state: its F.normalize."""
        from .autograd_ops import NormalizeFn

        home = state.device
        state = self._on_device(state).to(torch.float32).contiguous()
        return (NormalizeFn.apply(state) if state.shape[0] else state).to(home)

    def recurrent_aggregation(self, item_embeddings: torch.Tensor,
                              weights: torch.Tensor) -> torch.Tensor:
        """Gated linear recurrence over the history, then F.normalize."""
        return self.embed_state(self.recurrent_state(item_embeddings, weights))

    def forward(self, item_embeddings: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """reference :103-122"""
        if self.aggregation_method == "weighted_avg":
            return self.weighted_average(item_embeddings, weights)
        elif self.aggregation_method == "attention":
            return self.attention_aggregation(item_embeddings, weights)
        elif self.aggregation_method == "recurrent":
            return self.recurrent_aggregation(item_embeddings, weights)
        else:
            raise ValueError(f"Unknown aggregation method: {self.aggregation_method}")

    def encode_from_sequence(self, item_embeddings: torch.Tensor,
                             weights: torch.Tensor) -> torch.Tensor:
        """reference :124-144"""
        if item_embeddings.dim() == 2:
            item_embeddings = item_embeddings.unsqueeze(0)
        if weights.dim() == 1:
            weights = weights.unsqueeze(0)
        return self.forward(item_embeddings, weights)
