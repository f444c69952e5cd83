"""A mixture-of-experts block: norm, router, routed experts, shared expert, residual stream.

``MoEBlock`` puts the package's operators together the way a decoder layer's second half uses
them::

    h = x + residual;  u = rms_norm(h) * norm_weight             add_rms_norm
    logits = u gate_weight^T                   (FP32)            linear
    ids, weights, counts, loss                                   moe_route
    y = sum_j weights_j expert_{ids_j}(u)                        MoELayer
    out = act(u up^T) down^T + y               (shared expert)   linear, linear (residual = y)

and returns ``out`` and ``h``, which the next step's ``add_rms_norm`` adds.  The forward has no host
synchronisation, so it can be captured in a CUDA graph (one rank, or the peer-memory exchange).

``router_gradients`` goes back from the gate's weights and the balance loss to the gate's and
the norm's weights and to ``h``, for training the router beside experts that stay as they are.
The reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .linear import linear, linear_backward
from .norm import add_rms_norm, add_rms_norm_backward
from .router import Routing, moe_route, moe_route_backward

__all__ = ["BlockOutput", "MoEBlock", "RouterGradients"]


class BlockOutput(NamedTuple):
    out: torch.Tensor      # [T, H], to be added to `h` by the next step
    h: torch.Tensor        # [T, H], the residual stream
    normed: torch.Tensor   # [T, H], what the experts and the router saw
    logits: torch.Tensor   # FP32 [T, E]
    routing: Routing


class RouterGradients(NamedTuple):
    gate_weight: torch.Tensor
    norm_weight: torch.Tensor
    h: torch.Tensor


class MoEBlock:
    """norm_weight ``[H]``, gate_weight BF16 ``[E, H]``, experts a ``MoELayer`` over E experts.

    shared: ``(up [I, H], down [H, I])`` BF16 weights of a dense expert that every token takes, or None.
    gate_bias: FP32 ``[E]``, moves the choice of experts alone.  The rest as in ``moe_route``.
    """

    def __init__(self, norm_weight: torch.Tensor, gate_weight: torch.Tensor, experts, topk: int, *,
                 shared: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, activation: str = "silu", eps: float = 1e-6,
                 scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                 gate_bias: Optional[torch.Tensor] = None):
        if gate_weight.dim() != 2 or gate_weight.shape[1] != norm_weight.shape[0]:
            raise ValueError(f"gate_weight must be [E, H] with H = {norm_weight.shape[0]}, got {tuple(gate_weight.shape)}")
        if experts.num_experts != gate_weight.shape[0]:
            raise ValueError("the gate and the experts must have the same number of experts")
        self.norm_weight, self.gate_weight, self.gate_bias = norm_weight, gate_weight, gate_bias
        self.experts, self.topk, self.shared, self.activation = experts, topk, shared, activation
        self.eps, self.scoring, self.renormalize, self.scale = eps, scoring, renormalize, scale

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                token_mask: Optional[torch.Tensor] = None, balance: bool = False) -> BlockOutput:
        """x, residual: BF16 ``[T, H]``.  Tokens that ``token_mask`` drops reach no routed expert."""
        norm = add_rms_norm(x, self.norm_weight, residual, eps=self.eps)
        u = norm.y
        logits = linear(u, self.gate_weight, out_dtype=torch.float32)
        routing = moe_route(logits, self.topk, scoring=self.scoring, renormalize=self.renormalize, scale=self.scale,
                            bias=self.gate_bias, token_mask=token_mask, balance=balance)
        y = self.experts(u, routing.ids, routing.weights)
        if self.shared is not None:
            up, down = self.shared
            y = linear(linear(u, up, activation=self.activation), down, residual=y)
        return BlockOutput(y, x if norm.h is None else norm.h, u, logits, routing)

    __call__ = forward

    def router_gradients(self, o: BlockOutput, grad_weights: Optional[torch.Tensor] = None,
                         grad_loss: Optional[torch.Tensor] = None) -> RouterGradients:
        """Gradients from those of the gate's weights (FP32 ``[T, topk]``) and of the balance loss
        (FP32 ``[1]``), along the router's path alone; ``h``'s is to be added to the others that reach it.  The
        logits' gradient is rounded to the rows' dtype, as an operand of the gate's two products."""
        r = o.routing
        dlogits = moe_route_backward(o.logits, r.ids, grad_weights, grad_loss, r.counts, r.tokens, scoring=self.scoring,
                                     renormalize=self.renormalize, scale=self.scale)
        du, dgate, _ = linear_backward(dlogits.to(o.normed.dtype), o.normed, self.gate_weight)
        dh, dnorm = add_rms_norm_backward(du, o.h, self.norm_weight, eps=self.eps)
        return RouterGradients(dgate, dnorm, dh)
