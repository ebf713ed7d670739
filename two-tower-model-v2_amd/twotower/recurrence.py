"""Gated linear recurrence over event histories, with its backward pass (csrc/tt_recur.hip).

    A_t = sigmoid(gate_t) ** weight_t ;  h_t = A_t h_{t-1} + (1 - A_t) x_t

The order-aware aggregation of the buyer tower (``BuyerTower(aggregation_method="recurrent")``):
h is a running average of the item vectors with a memory length of its own for every event and
channel.  An event of weight w moves the state exactly as w events of weight 1 do; weight 0 is
padding.  One event at a time (S = 1 with ``h0``) is the serving form: a buyer's state is kept
and every new event costs one launch.
"""
from __future__ import annotations

import torch

from . import kernels


class _GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weights, h0, states):
        ctx.set_materialize_grads(False)
        h, last, saved = kernels.gated_scan(x, gate, weights, h0, states=states, save=True)
        ctx.save_for_backward(x, gate, weights, saved)
        ctx.h0_dtype = h0.dtype if h0 is not None else None
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        if ctx.needs_input_grad[2]:
            raise NotImplementedError("gradients w.r.t. event weights are not computed (they are "
                                      "counts of events, not parameters)")
        x, gate, weights, saved = ctx.saved_tensors
        dx, dgate, dh0 = kernels.gated_scan_backward(x, gate, weights, saved, dh, dlast,
                                                     ctx.needs_input_grad[3])
        if dh0 is not None:
            dh0 = dh0.to(ctx.h0_dtype)
        return dx, dgate, None, dh0, None


def gated_scan(x: torch.Tensor, gate: torch.Tensor, weights: torch.Tensor = None,
               h0: torch.Tensor = None, states: bool = True):
    """x, gate [B, S, D] (f32 or bf16, device), weights [B, S] or None (all 1), h0 [B, D] or None
    (zeros) -> (h [B, S, D], or None with ``states=False``; h_last [B, D] f32).

    ``gate`` holds logits: sigmoid(gate) is the part of the state that one event of weight 1
    keeps.  A weight that is not above 0 marks padding: h repeats the state there, x and gate are
    not looked at (they may hold anything) and get zero gradients.  h_last is the state after
    the last event (h0 for S = 0).  Differentiable in x, gate and h0."""
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad
                                    or (h0 is not None and h0.requires_grad)
                                    or (weights is not None and weights.requires_grad)):
        return _GatedScanFn.apply(x, gate, weights, h0, states)
    h, last, _ = kernels.gated_scan(x, gate, weights, h0, states=states)
    return h, last
