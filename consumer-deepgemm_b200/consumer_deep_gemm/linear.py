"""Dense product with bias, activation and residual in its epilogue, and its gradients.

The products around the routed experts: the router's logits, a shared expert, a projection
that adds the residual stream.  BF16 or FP16 operands on the tensor cores, FP32 sums.  The
reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import native

__all__ = ["linear", "linear_backward"]

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _activation(name: Optional[str]) -> int:
    if name not in _ACTIVATIONS:
        raise ValueError(f"activation must be None, 'relu', 'silu', 'gelu' or 'gelu_tanh', got {name!r}")
    return _ACTIVATIONS[name]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           out_dtype: Optional[torch.dtype] = None, preact: bool = False):
    """``y = act(x @ weight.T + bias) + residual`` with everything after the product in its epilogue.

    x ``[M, K]`` and weight ``[N, K]``: both BF16 or both FP16, any row strides (rows that do not start
    on 16-byte boundaries are copied once inside the call).  bias ``[N]`` and residual ``[M, N]``:
    x's dtype or FP32.  activation: None, ``"relu"``, ``"silu"``, ``"gelu"`` (erf) or ``"gelu_tanh"``,
    in FP32 with the fast exponential (relative error 2^-19 + 2^-21 |exponent|).
    out_dtype: x's dtype (the default) or ``torch.float32``, e.g. for router logits.  Returns ``y``, or
    with ``preact=True`` ``(y, z)``, z being the value before the activation in x's dtype, which
    ``linear_backward`` takes.
    """
    if out_dtype is None or out_dtype == x.dtype:
        out_f32 = False
    elif out_dtype == torch.float32:
        out_f32 = True
    else:
        raise ValueError(f"out_dtype must be x's dtype or torch.float32, got {out_dtype}")
    y, z = native.require().linear(x, weight, bias, residual, _activation(activation), out_f32, preact)
    return (y, z) if preact else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, z: Optional[torch.Tensor] = None, *,
                    activation: Optional[str] = None, input_grad: bool = True, weight_grad: bool = True,
                    bias_grad: bool = False):
    """``(dx, dweight, dbias)`` of ``linear`` from ``dy``; None where not asked for.

    dy, z: ``[M, N]`` of x's dtype; ``z`` is the forward call's (``preact=True``) and needed with an
    activation only.  The gradient of the residual is ``dy`` itself.  ``dz = dy * act'(z)`` is rounded
    to x's dtype, as an operand of both products (the error of ``dx`` and ``dweight`` is sqrt 2 of what their
    own rounding leaves); ``dbias`` has x's dtype and sums the unrounded values.
    """
    return native.require().linear_backward(dy, x, weight, z, _activation(activation), input_grad, weight_grad, bias_grad)
