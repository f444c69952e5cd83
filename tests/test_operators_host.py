"""CPU checks of the operators around the experts: argument checks of the C ABI and of Python, and
the arithmetic the kernels rely on."""

import ctypes

import pytest
import torch

import cabi

P, I32, I64, F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = 1, 2, 3, 4
FAKE = 1 << 20  # an address that is never read: every call here is refused on the host
BF16, F16, FP32 = cabi.DT["bf16"], 9, cabi.DT["f32"]


class NormArgs(ctypes.Structure):
    _fields_ = [("x", P), ("x_stride", I64), ("r", P), ("r_stride", I64), ("w", P), ("dtype", I32), ("w_dtype", I32),
                ("T", I64), ("H", I64), ("eps", F32), ("scale_fmt", I32), ("h", P), ("h_stride", I64), ("y", P),
                ("y_stride", I64), ("q", P), ("q_stride", I64), ("s", P), ("s_stride_m", I64), ("s_stride_k", I64)]


class NormBackwardArgs(ctypes.Structure):
    _fields_ = [("dy", P), ("dy_stride", I64), ("h", P), ("h_stride", I64), ("w", P), ("dh", P), ("dh_stride", I64),
                ("dtype", I32), ("w_dtype", I32), ("T", I64), ("H", I64), ("eps", F32), ("dx", P), ("dx_stride", I64),
                ("dw", P)]


class RouteArgs(ctypes.Structure):
    _fields_ = [("logits", P), ("stride", I64), ("dtype", I32), ("scoring", I32), ("token_mask", P), ("bias", P),
                ("T", I64), ("E", I64), ("topk", I64), ("renormalize", I32), ("scale", F32), ("weights", P), ("ids", P),
                ("counts", P), ("tokens", P), ("loss", P)]


class LinearArgs(ctypes.Structure):
    _fields_ = [("x", P), ("x_stride", I64), ("w", P), ("w_stride", I64), ("bias", P), ("residual", P),
                ("residual_stride", I64), ("dtype", I32), ("bias_dtype", I32), ("residual_dtype", I32),
                ("out_dtype", I32), ("activation", I32), ("M", I64), ("N", I64), ("K", I64), ("y", P), ("y_stride", I64),
                ("z_out", P), ("z_stride", I64)]


def _norm(**kw):
    g = NormArgs(x=FAKE, x_stride=256, w=FAKE, dtype=BF16, w_dtype=BF16, T=4, H=256, eps=1e-6, y=FAKE, y_stride=256)
    for k, v in kw.items():
        setattr(g, k, v)
    return cabi.lib().cdg_add_rms_norm(ctypes.byref(g), None)


def test_norm_arguments():
    assert _norm(T=0) == 0
    for bad in (dict(H=0), dict(T=-1), dict(dtype=FP32 + 40), dict(w_dtype=F16), dict(eps=-1.0), dict(scale_fmt=2),
                dict(x=None), dict(w=None), dict(y=None), dict(q=FAKE, s=None), dict(eps=float("nan"))):
        assert _norm(**bad) == INVALID, bad
    assert _norm(H=32769) == UNSUPPORTED
    lib = cabi.lib()
    lib.cdg_rms_norm_backward_workspace_bytes.restype = ctypes.c_size_t
    lib.cdg_rms_norm_backward_workspace_bytes.argtypes = [I64, I64]
    assert lib.cdg_rms_norm_backward_workspace_bytes(4, 256) >= 4 * 256 * 4
    assert lib.cdg_rms_norm_backward_workspace_bytes(4, 0) == 0
    lib.cdg_rms_norm_backward.argtypes = [ctypes.POINTER(NormBackwardArgs), P, ctypes.c_size_t, P]
    g = NormBackwardArgs(dy=FAKE, dy_stride=256, h=FAKE, h_stride=256, w=FAKE, dtype=BF16, w_dtype=BF16, T=4, H=256,
                         eps=1e-6, dx=FAKE, dx_stride=256, dw=FAKE)
    assert lib.cdg_rms_norm_backward(ctypes.byref(g), None, 0, None) == WORKSPACE
    assert lib.cdg_rms_norm_backward(ctypes.byref(g), P(FAKE), 16, None) == WORKSPACE
    g.dw = None
    assert lib.cdg_rms_norm_backward(ctypes.byref(g), P(FAKE), 1 << 20, None) == INVALID


def test_route_arguments():
    lib = cabi.lib()
    lib.cdg_moe_route.argtypes = [ctypes.POINTER(RouteArgs), P, ctypes.c_size_t, P]
    lib.cdg_moe_route_workspace_bytes.restype = ctypes.c_size_t
    lib.cdg_moe_route_workspace_bytes.argtypes = [I64]

    def call(ws=FAKE, n=1 << 20, **kw):
        g = RouteArgs(logits=FAKE, stride=64, dtype=FP32, scoring=0, T=4, E=64, topk=8, renormalize=1, scale=1.0,
                      weights=FAKE, ids=FAKE, counts=FAKE, tokens=FAKE)
        for k, v in kw.items():
            setattr(g, k, v)
        return lib.cdg_moe_route(ctypes.byref(g), P(ws), n, None)

    for bad in (dict(topk=0), dict(topk=65), dict(E=0), dict(scoring=2), dict(dtype=cabi.DT["i32"]), dict(counts=None),
                dict(ids=None), dict(T=-1)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(E=1025), dict(topk=33), dict(T=(1 << 23) + 1)):
        assert call(**bad) == UNSUPPORTED, bad
    assert call(ws=None) == WORKSPACE and call(n=8) == WORKSPACE and call(ws=FAKE + 4) == ALIGNMENT
    assert lib.cdg_moe_route_workspace_bytes(256) >= 256 * 12
    assert lib.cdg_moe_route_workspace_bytes(0) == 0


def test_linear_arguments():
    lib = cabi.lib()
    lib.cdg_linear.argtypes = [ctypes.POINTER(LinearArgs), P, ctypes.c_size_t, P]
    lib.cdg_linear_workspace_bytes.argtypes = [ctypes.POINTER(LinearArgs)]
    lib.cdg_linear_workspace_bytes.restype = ctypes.c_size_t

    def args(**kw):
        g = LinearArgs(x=FAKE, x_stride=64, w=FAKE, w_stride=64, dtype=BF16, out_dtype=BF16, M=4, N=8, K=64, y=FAKE,
                       y_stride=8)
        for k, v in kw.items():
            setattr(g, k, v)
        return g

    for bad in (dict(dtype=FP32), dict(out_dtype=F16), dict(activation=5), dict(activation=-1), dict(M=-1),
                dict(bias=FAKE, bias_dtype=F16), dict(residual=FAKE, residual_dtype=F16), dict(y=None), dict(w=None)):
        assert lib.cdg_linear(ctypes.byref(args(**bad)), None, 0, None) == INVALID, bad
    assert lib.cdg_linear(ctypes.byref(args(K=(1 << 30) + 1)), None, 0, None) == UNSUPPORTED
    assert lib.cdg_linear(ctypes.byref(args(M=0)), None, 0, None) == 0
    # rows on 16-byte boundaries need no workspace; others a copy with rows padded to eight columns
    assert lib.cdg_linear_workspace_bytes(ctypes.byref(args())) == 0
    odd = args(x_stride=67, K=61)
    assert lib.cdg_linear_workspace_bytes(ctypes.byref(odd)) >= 4 * 64 * 2
    assert lib.cdg_linear(ctypes.byref(odd), None, 0, None) == WORKSPACE


def test_python_refuses_before_the_device():
    import consumer_deep_gemm as cdg

    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    for call in (lambda: cdg.linear(x, x, activation="tanh"), lambda: cdg.linear(x, x, out_dtype=torch.float64),
                 lambda: cdg.linear_backward(x, x, x, activation="selu"), lambda: cdg.moe_route(x, 2, scoring="relu"),
                 lambda: cdg.moe_route_backward(x, x, scoring="")):
        with pytest.raises(ValueError):
            call()


def test_normal_tail_formula():
    """The GELU's tail (Abramowitz and Stegun 7.1.26 in the form the kernel uses) against erfc."""
    z = torch.linspace(-12, 12, 200001, dtype=torch.float64)
    a = z.abs()
    t = 1 / (1 + 0.3275911 * 0.70710678 * a)
    poly = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429))))
    tail = 0.5 * poly * torch.exp(-0.5 * a * a)
    assert float((tail - torch.special.ndtr(-a)).abs().max()) < 0.5 * 1.5e-7 + 1e-8


def test_norm_backward_workspace_alignment():
    """Partial sums are stored 16 bytes at a time: a workspace on a lesser boundary is refused on the host."""
    lib = cabi.lib()
    lib.cdg_rms_norm_backward.argtypes = [ctypes.POINTER(NormBackwardArgs), P, ctypes.c_size_t, P]
    g = NormBackwardArgs(dy=FAKE, dy_stride=256, h=FAKE, h_stride=256, w=FAKE, dtype=BF16, w_dtype=BF16, T=4, H=256,
                         eps=1e-6, dx=FAKE, dx_stride=256, dw=FAKE)
    for off in (4, 8, 12, 1):
        assert lib.cdg_rms_norm_backward(ctypes.byref(g), P(FAKE + off), 1 << 20, None) == ALIGNMENT


class RouteBackwardArgs(ctypes.Structure):
    _fields_ = [("logits", P), ("stride", I64), ("dtype", I32), ("scoring", I32), ("ids", P), ("grad_weights", P),
                ("grad_loss", P), ("counts", P), ("tokens", P), ("T", I64), ("E", I64), ("topk", I64),
                ("renormalize", I32), ("scale", F32), ("dlogits", P), ("d_stride", I64)]


class LinearBackwardArgs(ctypes.Structure):
    _fields_ = [("dy", P), ("dy_stride", I64), ("x", P), ("x_stride", I64), ("w", P), ("w_stride", I64), ("z", P),
                ("z_stride", I64), ("dtype", I32), ("db_dtype", I32), ("activation", I32), ("M", I64), ("N", I64),
                ("K", I64), ("dx", P), ("dx_stride", I64), ("dw", P), ("dw_stride", I64), ("db", P)]


def test_pointers_off_their_types_boundary_are_refused():
    """Each pointer in turn one byte past FAKE (16-bit types) or two bytes past it (32-bit types)."""
    lib = cabi.lib()

    def each(entry, make, names, off, rest):
        fn = getattr(lib, entry)
        fn.argtypes = None
        for name in names:
            g = make()
            setattr(g, name, FAKE + off)
            assert fn(ctypes.byref(g), *rest) == ALIGNMENT, (entry, name)

    ws = (P(FAKE), ctypes.c_size_t(1 << 24), None)

    def norm(dtype=BF16):
        return NormArgs(x=FAKE, x_stride=256, r=FAKE, r_stride=256, w=FAKE, dtype=dtype, w_dtype=dtype, T=4, H=256,
                        eps=1e-6, h=FAKE, h_stride=256, y=FAKE, y_stride=256, q=FAKE, q_stride=256, s=FAKE,
                        s_stride_m=2, s_stride_k=1)

    each("cdg_add_rms_norm", norm, ["x", "r", "w", "h", "y", "s"], 1, (None,))
    each("cdg_add_rms_norm", lambda: norm(FP32), ["x", "r", "w", "h", "y", "s"], 2, (None,))

    def norm_backward(dtype=F16):
        return NormBackwardArgs(dy=FAKE, dy_stride=256, h=FAKE, h_stride=256, w=FAKE, dh=FAKE, dh_stride=256, dtype=dtype,
                                w_dtype=FP32, T=4, H=256, eps=1e-6, dx=FAKE, dx_stride=256, dw=FAKE)

    each("cdg_rms_norm_backward", norm_backward, ["dy", "h", "dh", "dx"], 1, ws)
    each("cdg_rms_norm_backward", lambda: norm_backward(FP32), ["dy", "h", "dh", "dx", "w", "dw"], 2, ws)

    def route(dtype=BF16):
        return RouteArgs(logits=FAKE, stride=64, dtype=dtype, bias=FAKE, T=4, E=64, topk=8, renormalize=1, scale=1.0,
                         weights=FAKE, ids=FAKE, counts=FAKE, tokens=FAKE, loss=FAKE)

    each("cdg_moe_route", route, ["logits"], 1, ws)
    each("cdg_moe_route", lambda: route(FP32), ["logits", "bias", "weights", "ids", "counts", "tokens", "loss"], 2, ws)

    def route_backward(dtype=BF16):
        return RouteBackwardArgs(logits=FAKE, stride=64, dtype=dtype, ids=FAKE, grad_weights=FAKE, grad_loss=FAKE,
                                 counts=FAKE, tokens=FAKE, T=4, E=64, topk=8, scale=1.0, dlogits=FAKE, d_stride=64)

    each("cdg_moe_route_backward", route_backward, ["logits", "dlogits"], 1, (None,))
    each("cdg_moe_route_backward", lambda: route_backward(FP32),
         ["logits", "dlogits", "ids", "grad_weights", "grad_loss", "counts", "tokens"], 2, (None,))

    def product(out=BF16):
        return LinearArgs(x=FAKE, x_stride=64, w=FAKE, w_stride=64, bias=FAKE, residual=FAKE, residual_stride=8,
                          dtype=BF16, bias_dtype=out, residual_dtype=out, out_dtype=out, M=4, N=8, K=64, y=FAKE,
                          y_stride=8, z_out=FAKE, z_stride=8)

    each("cdg_linear", product, ["x", "w", "bias", "residual", "y", "z_out"], 1, ws)
    each("cdg_linear", lambda: product(FP32), ["bias", "residual", "y"], 2, ws)

    def product_backward():
        return LinearBackwardArgs(dy=FAKE, dy_stride=8, x=FAKE, x_stride=64, w=FAKE, w_stride=64, z=FAKE, z_stride=8,
                                  dtype=BF16, db_dtype=FP32, activation=2, M=4, N=8, K=64, dx=FAKE, dx_stride=64,
                                  dw=FAKE, dw_stride=64, db=FAKE)

    each("cdg_linear_backward", product_backward, ["dy", "x", "w", "z", "dx", "dw"], 1, ws)
    each("cdg_linear_backward", product_backward, ["db"], 2, ws)


def test_documented_imports():
    """Every `from consumer_deep_gemm[.module] import ...` line of the README and the integration notes."""
    import importlib
    import os
    import re

    seen = set()
    for name in ("README.md", "INTEGRATION.md"):
        with open(os.path.join(cabi.REPO, name)) as f:
            text = f.read()
        for module, names in re.findall(r"^from (consumer_deep_gemm[\w.]*) import ([\w, ]+)", text, re.M):
            for each in names.split(","):
                assert hasattr(importlib.import_module(module), each.strip()), (name, module, each)
                seen.add(each.strip())
    assert {"MoEBlock", "MoELayer", "add_rms_norm", "linear", "moe_route"} <= seen
    import consumer_deep_gemm as cdg

    for each in cdg.__all__:
        assert hasattr(cdg, each), each
    assert "MoEBlock" in cdg.__all__


def test_normal_tail_fit():
    """The normal tail's fit as the kernel has it: within 1.2e-7 of the tail itself in 64 bits and, each step
    rounded to FP32, 5e-7 (eight multiplications and additions, a division and a product of 6e-8 each, the
    early ones damped by t < 1)."""
    c = [0.122044094, 0.122772254, 0.10436748, 0.118629217, -0.0330358259, 0.179384798, -0.150699764, 0.0365378037]
    a = torch.cat([torch.linspace(0, 3, 20001), torch.linspace(3, 14.5, 20001)])
    want = 0.5 * torch.special.erfcx(a.double() / 2 ** 0.5)
    for dtype, most in ((torch.float64, 1.2e-7), (torch.float32, 5e-7)):
        k = torch.tensor(c, dtype=torch.float32).to(dtype)
        t = 1 / (1 + torch.tensor(0.306, dtype=torch.float32).to(dtype) * a.to(dtype))
        p = k[7]
        for i in range(6, -1, -1):
            p = p * t + k[i]
        assert float(((t * p).double() / want - 1).abs().max()) < most
