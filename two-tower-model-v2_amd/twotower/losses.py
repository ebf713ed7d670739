"""InfoNCELoss on MI355X: drop-in for src/training/losses.py (class InfoNCELoss :8).

Same constructor (temperature=0.07) and forward(buyer_embeddings, positive_embeddings,
negative_embeddings) -> scalar loss.  Forward and backward run in one HIP call
(tt_infonce_f32, csrc/tt_loss.hip): the in-batch logits are one MFMA GEMM instead of the
reference's expanded [B, B, E] bmm (:55-61), and the gradients are two more GEMMs; autograd
receives the precomputed input gradients.  ``prec="bf16"`` runs the GEMMs on bf16 MFMA
(configs[4]'s "MFMA bf16" training step); the default "f32" matches the reference to ~1e-6.

Beside it, for a softmax over a whole catalog instead of a batch (the reference has none):
``catalog_log_probs`` (log-probabilities of given items, entropy, top alternatives; csrc/
tt_catalog.hip, the logits are never stored) and ``CatalogSoftmaxLoss`` over it.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib, kernels
from ._lib import check, lib, require_device, stream_ptr


def infonce(b: torch.Tensor, p: torch.Tensor, n: torch.Tensor, temperature: float = 0.07,
            prec: str = "f32", grads: bool = True):
    """Device tensors b [B,E], p [B,E], n [B,N,E] -> (loss [] f32, (gb, gp, gn) or None)."""
    for t, name in ((b, "buyer_embeddings"), (p, "positive_embeddings"),
                    (n, "negative_embeddings")):
        require_device(t, name)
    b, p, n = (t.detach().contiguous().to(torch.float32) for t in (b, p, n))
    B, E = b.shape
    if p.shape != (B, E) or n.dim() != 3 or n.shape[0] != B or n.shape[2] != E:
        raise ValueError("InfoNCE: expected b [B,E], p [B,E], n [B,N,E]")
    N = n.shape[1]
    pr = _lib.TT_PREC_BF16 if prec == "bf16" else _lib.TT_PREC_F32
    need = ctypes.c_int64(0)
    check(lib().tt_infonce_workspace_bytes(B, N, E, pr, int(grads), ctypes.byref(need)),
          "tt_infonce_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=b.device)
    loss = torch.empty((), dtype=torch.float32, device=b.device)
    g = tuple(torch.empty_like(t) for t in (b, p, n)) if grads else (None, None, None)
    check(lib().tt_infonce_f32(b.data_ptr(), b.stride(0), p.data_ptr(), p.stride(0),
                               n.data_ptr(), n.stride(0), n.stride(1), B, N, E,
                               ctypes.c_float(temperature), pr, loss.data_ptr(),
                               *(t.data_ptr() if t is not None else None for t in g),
                               ws.data_ptr(), ws.numel(), stream_ptr()), "tt_infonce_f32")
    return loss, (g if grads else None)


class _InfoNCEFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, b, p, n, temperature, prec):
        need = any(ctx.needs_input_grad[:3])
        loss, g = infonce(b, p, n, temperature, prec, grads=need)
        if need:
            ctx.save_for_backward(*g)
        return loss

    @staticmethod
    def backward(ctx, grad_out):
        gb, gp, gn = ctx.saved_tensors
        return grad_out * gb, grad_out * gp, grad_out * gn, None, None


class InfoNCELoss(nn.Module):
    """Mirror of reference ``InfoNCELoss`` (src/training/losses.py:8-79)."""

    def __init__(self, temperature: float = 0.07, prec: str = "f32"):
        super().__init__()
        self.temperature = temperature
        self.prec = prec

    def forward(self, buyer_embeddings: torch.Tensor, positive_embeddings: torch.Tensor,
                negative_embeddings: torch.Tensor) -> torch.Tensor:
        return _InfoNCEFn.apply(buyer_embeddings, positive_embeddings, negative_embeddings,
                                self.temperature, self.prec)


class LogProbs(NamedTuple):
    """catalog_log_probs' result; what was not asked for is None."""
    log_prob: Optional[torch.Tensor]  # [N] f32
    entropy: Optional[torch.Tensor]  # [N] f32
    top_ids: Optional[torch.Tensor]  # [N, top] int64
    top_log_probs: Optional[torch.Tensor]  # [N, top] f32


class _CatalogFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ids, bias, temperature, entropy, top):
        ctx.set_materialize_grads(False)
        dt = ctx.dt = kernels.catalog_check(x, w, ids, bias)
        xr, wr = kernels.catalog_rows(x), kernels.catalog_rows(w)
        lp, ent, lse, ti, tl = kernels.catalog_logprobs(xr, wr, ids, bias, temperature, entropy,
                                                        top, dt)
        ctx.save_for_backward(xr, wr, ids, bias, lse, ent)
        ctx.temperature, ctx.e = temperature, x.shape[1]
        if top:
            ctx.mark_non_differentiable(ti, tl)
        return lp, ent, ti, tl

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, ge, _ti, _tl):
        if ctx.needs_input_grad[3]:
            raise NotImplementedError("gradients w.r.t. bias are not computed (it is a correction "
                                      "of the sampling, not a parameter)")
        x, w, ids, bias, lse, ent = ctx.saved_tensors
        dx, dw = kernels.catalog_logprobs_backward(
            x, w, ids, bias, ctx.temperature, lse, ent, g, ge, ctx.needs_input_grad[0],
            ctx.needs_input_grad[1], ctx.dt)
        if x.shape[1] != ctx.e:
            dx, dw = (t[:, :ctx.e] if t is not None else None for t in (dx, dw))
        return dx, dw, None, None, None, None, None


def catalog_log_probs(queries: torch.Tensor, items: torch.Tensor, ids: torch.Tensor = None,
                      temperature: float = 0.07, bias: torch.Tensor = None, entropy: bool = False,
                      top: int = 0) -> LogProbs:
    """Under p(v | n) = softmax_v(queries_n . items_v / temperature + bias_v), for queries [N, E] and
    items [V, E] (both f32 or both bf16, device):

    log_prob  [N] log p(ids_n | n) for ids [N] int64; 0 for an id of -1 (a row without an item; so
              is any id outside 0 .. V - 1)
    entropy   [N] (``entropy=True``)
    top_ids, top_log_probs  [N, top]: the ``top`` (<= 32) most probable items, ordered by the
              product in 64 bits, ties to the lower id

    ``bias`` [V] f32: e.g. -log q of a sampled-softmax correction; -inf takes the item out (its
    vector may hold anything).  A row with nothing left: log_prob -inf, entropy 0.  Differentiable in
    queries and items (log_prob and entropy); the logits are never stored, so N x V is bounded by
    time alone (with ``top`` a float per 16 of them is, for as many rows at a time as 4 GB hold).  E
    is padded to a multiple of 64 where it is not one: a copy of the items in every call, which a
    caller saves by keeping them padded with zeros."""
    if (isinstance(temperature, torch.Tensor) and temperature.requires_grad
            and torch.is_grad_enabled()):
        raise NotImplementedError("gradients w.r.t. the temperature are not computed: pass a number "
                                  "(or temperature.detach())")
    if torch.is_grad_enabled() and (queries.requires_grad or items.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return LogProbs(*_CatalogFn.apply(queries, items, ids, bias, float(temperature), entropy,
                                          top))
    dt = kernels.catalog_check(queries, items, ids, bias)
    lp, ent, _, ti, tl = kernels.catalog_logprobs(
        kernels.catalog_rows(queries), kernels.catalog_rows(items), ids, bias, float(temperature),
        entropy, top, dt)
    return LogProbs(lp, ent, ti, tl)


class CatalogSoftmaxLoss(nn.Module):
    """Mean over the rows of -log p(id | buyer) over all items: InfoNCELoss's task with the whole
    catalog (or any set of items) as the negatives.  Rows with id -1 (or any outside the catalog) do
    not count."""

    def __init__(self, temperature: float = 0.07, entropy_weight: float = 0.0):
        super().__init__()
        if not temperature > 0:
            raise ValueError(f"temperature must be above 0, got {temperature}")
        self.temperature = temperature
        self.entropy_weight = entropy_weight

    def forward(self, buyer_embeddings: torch.Tensor, item_embeddings: torch.Tensor,
                ids: torch.Tensor, bias: torch.Tensor = None) -> torch.Tensor:
        """buyer_embeddings [N, E], item_embeddings [V, E], ids [N] -> scalar; entropy_weight > 0
        also rewards the mean entropy (a penalty on overconfidence)."""
        r = catalog_log_probs(buyer_embeddings, item_embeddings, ids, self.temperature, bias,
                              entropy=self.entropy_weight != 0)
        has = (ids >= 0) & (ids < item_embeddings.shape[0])
        n = has.sum().clamp(min=1)
        loss = -r.log_prob.sum() / n
        if self.entropy_weight != 0:
            loss = loss - self.entropy_weight * torch.where(
                has, r.entropy, torch.zeros_like(r.entropy)).sum() / n
        return loss
