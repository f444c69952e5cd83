"""Router of a mixture-of-experts block: top-k gate, rows per expert, balance loss, gradients.

``moe_route`` turns the router's logits into the ``topk_ids`` and ``topk_w`` that
``MoELayer`` takes, and counts on the way how many tokens chose each expert; with
``balance=True`` the same pass gives the balance loss.  The reference has no counterpart
(its callers bring ids and weights).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import native

__all__ = ["Routing", "moe_route", "moe_route_backward"]

_SCORING = {"softmax": False, "sigmoid": True}


class Routing(NamedTuple):
    """What ``moe_route`` returns."""

    weights: torch.Tensor         # FP32 [T, topk]
    ids: torch.Tensor             # int32 [T, topk], -1 = no expert
    counts: torch.Tensor          # int32 [E]: tokens that chose each expert
    tokens: torch.Tensor          # int32 [1]: valid tokens
    loss: Optional[torch.Tensor]  # FP32 [1]: balance loss, None unless asked for


def _sigmoid(scoring: str) -> bool:
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    return _SCORING[scoring]


def moe_route(logits: torch.Tensor, topk: int, *, scoring: str = "softmax", renormalize: bool = True,
              scale: float = 1.0, bias: Optional[torch.Tensor] = None, token_mask: Optional[torch.Tensor] = None,
              balance: bool = False) -> Routing:
    """Choose ``topk`` experts per token from BF16, FP16 or FP32 logits ``[T, E]`` (any row stride).

    With ``score = softmax(logits)`` or ``sigmoid(logits)`` in FP32, a token's ids are its ``topk``
    largest logits -- with ``bias`` (FP32 ``[E]``), its largest ``score + bias`` -- in falling order,
    ties to the lowest index; its weights are ``scale * score[ids]``, divided by their sum before
    scaling with ``renormalize`` (shares that sum to 1 also where the scores themselves are below FP32's
    range).  Tokens that ``token_mask`` (bool or uint8 ``[T]``) drops and slots
    for which no logit above -inf is left get id -1 and weight 0, which ``MoELayer`` passes over;
    an expert is switched off by logits of -inf.  NaN counts as -inf, +inf as the largest finite value.

    ``balance=True``: ``loss = E / (topk V^2) sum_e counts[e] sum_t p[t, e]`` over the V valid tokens,
    ``p`` the scores divided by their sum over the experts; 1 when rows and probabilities are spread
    evenly.  E up to 1024, topk up to 32; no host synchronisation.
    """
    return Routing(*native.require().moe_route(logits, topk, _sigmoid(scoring), renormalize, scale, bias, token_mask,
                                               balance))


def moe_route_backward(logits: torch.Tensor, ids: torch.Tensor, grad_weights: Optional[torch.Tensor] = None,
                       grad_loss: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                       tokens: Optional[torch.Tensor] = None, *, scoring: str = "softmax", renormalize: bool = True,
                       scale: float = 1.0) -> torch.Tensor:
    """Gradient of the logits from those of the weights (FP32 ``[T, topk]``) and the loss (FP32 ``[1]``,
    on the device; needs the forward call's ``counts`` and ``tokens``).

    ``ids`` are the forward call's.  The choice of experts and their counts are held fixed, as is
    usual; rows without an expert get zeros.  The result has the logits' dtype.
    """
    return native.require().moe_route_backward(logits, ids, grad_weights, grad_loss, counts, tokens, _sigmoid(scoring),
                                               renormalize, scale)
