"""RMS norm with the residual's addition and an FP8 output, and its gradient.

The step before the experts (and before every dense product) of a block: the residual
stream takes the previous step's output, and its norm goes on, in the rows' own type for the
router and ``MoELayer`` and as e4m3 codes with 1x128 scales for the grouped GEMM
(``m_grouped_fp8_fp4_gemm_nt_contiguous((q, scale), ...)``).  The reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import native

__all__ = ["AddRMSNorm", "add_rms_norm", "add_rms_norm_backward"]


class AddRMSNorm(NamedTuple):
    """What ``add_rms_norm`` returns; None where not asked for."""

    h: Optional[torch.Tensor]      # x + residual [T, H], x's dtype; only with a residual
    y: Optional[torch.Tensor]      # the norm [T, H], x's dtype
    q: Optional[torch.Tensor]      # its e4m3 codes [T, H]
    scale: Optional[torch.Tensor]  # their FP32 scales [T, ceil(H / 128)]


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 quantize: bool = False, ue8m0: bool = False, normed: bool = True) -> AddRMSNorm:
    """``h = x + residual``; ``y = h / sqrt(mean(h^2) + eps) * weight``; e4m3 codes of ``y``.

    x, residual: BF16, FP16 or FP32 ``[T, H]`` (any row stride, H up to 32,768); weight ``[H]`` of
    the same dtype or FP32.  The sum and the norm are held in FP32: ``h`` and ``y`` are each rounded
    once, and the codes are of the unrounded ``y``.  ``quantize=True`` adds ``q`` and ``scale`` (1x128
    blocks, the last one shorter when H is no multiple of 128; the amax/448 recipe of the framework's
    quantiser, whose scales these are bit for bit, or with
    ``ue8m0=True`` scales rounded up to powers of two); ``normed=False`` leaves ``y`` out.
    A row of zeros gives zeros (with ``eps`` > 0); a NaN keeps its place in ``y`` and ``q`` (its row is NaN);
    a row whose mean square passes FP32's range gives zeros.
    """
    return AddRMSNorm(*native.require().add_rms_norm(x, weight, residual, eps, quantize, ue8m0, normed))


def add_rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, dh: Optional[torch.Tensor] = None,
                          *, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dx, dweight)`` of ``add_rms_norm`` from the gradient ``dy`` of ``y``.

    ``h`` is the forward pass's ``h`` (its ``x`` where there was no residual), ``dh`` the gradient
    that reaches it by the residual stream.  ``dx`` is the gradient of ``x`` and of ``residual``
    alike; ``dweight`` has the weight's dtype and is summed over the rows in FP32, in an order that the
    sizes, the dtype, whether the rows lie on 16-byte boundaries, and the GPU's SM count fix.
    """
    dx, dw = native.require().rms_norm_backward(dy, h, weight, dh, eps)
    return dx, dw
