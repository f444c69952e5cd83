"""GPU checks of the dense product with its epilogue, and of its gradients.

Against plain formulas in 64 bits on the same inputs.  Tolerances, with d the unit roundoff of the
output's type (2^-8 BF16, 2^-11 FP16) and S = sum_k |x||w| of an element:
  * The tensor cores add 16 products at a time to a 32-bit sum and may drop what lies below its
    last bit: K / 16 additions of 17 terms, each within 2^-23 of S, so a sum is within
    (K + 64) 2^-23 S however it was split.  Activations have slopes within 1.2 and are computed
    within 2^-20 of their value and argument.
  * An element is thus within d |y| + 1.2 (K + 64) 2^-23 S + 2^-20 (|act| + |z|), and the whole
    result, whose errors are independent, within 0.6 d of its norm (a rounding's mean square is
    d^2 / 3) plus 2^-18 for the sums.
  * FP32 results: no running sum covers more than 512 of K, so the norm of the error is within
    2^-19 of that of S-weighted results; checked as 2^-19 |y| in the norm and per element as above
    without d.
  * Gradients: dz is rounded to the operands' type, so an element of dx is within
    d |dx| + (d + (N + 64) 2^-23) sum |dz||w|, and the norm of the error within 0.6 sqrt(2) d.  FP16
    rounds a dz below 2^-14 to a multiple of 2^-24, and the slope of an activation is within 2^-20
    however small it is, which adds 2^-25 sum |w| (FP16) and 2^-20 sum |dy||w|.
"""

import math

import pytest
import torch

import cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(autouse=True)
def _seed():
    """The same inputs in every run and order."""
    torch.manual_seed(20)


def _cdg():
    import consumer_deep_gemm

    return consumer_deep_gemm


def _act64(z, act):
    if act == "relu":
        return z.relu()  # slope 0 at 0
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _operands(M, N, K, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    w = (torch.randn(N, K, generator=g, device=DEV) / max(1, K) ** 0.5).to(dtype)
    return x, w


def _check(got, x, w, bias, residual, act, out_dtype):
    K = x.shape[1]
    z = x.double() @ w.double().t()
    S = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        z = z + bias.double()
        S = S + bias.double().abs()
    a = _act64(z, act)
    y = a if residual is None else a + residual.double()
    assert got.dtype == out_dtype and got.shape == y.shape
    if y.numel() == 0:
        return
    err = (got.double() - y).abs()
    d = UNIT[out_dtype]
    slack = d * y.abs() + 1.2 * (K + 64) * 2.0 ** -23 * S + 2.0 ** -20 * (a.abs() + z.abs() + y.abs())
    if out_dtype == torch.float16:
        slack = slack + 2.0 ** -25
    bad = err > slack
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} out of tolerance, first {bad.nonzero()[0].tolist()}"
    if y.numel() >= 64:
        norm = 2.0 ** -19 if out_dtype == torch.float32 else 0.6 * d + 2.0 ** -18
        assert float(err.norm()) <= norm * float((y.abs() + z.abs()).norm())
    assert cabi.device_status() == (0, 0)


SHAPES = [(1, 4096, 4096), (1, 1, 1), (1, 130, 33), (2, 256, 64), (3, 1000, 520), (8, 4096, 1024), (17, 77, 200),
          (64, 512, 2048), (100, 64, 64), (128, 128, 128), (129, 257, 65), (300, 200, 72), (1000, 384, 1000),
          (513, 1030, 333), (2048, 256, 4096), (256, 2048, 511), (5, 16, 8192), (700, 3, 100), (4096, 512, 128),
          (2049, 1100, 1088), (1536, 2560, 320), (33, 8, 16)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                             (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_linear_against_64_bits(M, N, K, dtype, out_dtype):
    x, w = _operands(M, N, K, dtype)
    _check(_cdg().linear(x, w, out_dtype=out_dtype), x, w, None, None, None, out_dtype)
    bias = torch.randn(N, device=DEV).to(dtype)
    residual = torch.randn(M, N, device=DEV).to(dtype)
    got = _cdg().linear(x, w, bias, residual, activation="silu", out_dtype=out_dtype)
    _check(got, x, w, bias, residual, "silu", out_dtype)
    assert torch.equal(got, _cdg().linear(x, w, bias, residual, activation="silu", out_dtype=out_dtype))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(1, 300, 128), (200, 96, 100), (1024, 1024, 256), (4, 640, 4096)])
def test_linear_epilogues(M, N, K, act):
    x, w = _operands(M, N, K, torch.bfloat16, seed=1)
    w = w * 3
    for bias, residual in ((None, None), (torch.randn(N, device=DEV), None),
                           (torch.randn(N, device=DEV).bfloat16(), torch.randn(M, N, device=DEV)),
                           (None, torch.randn(M, N, device=DEV).bfloat16())):
        for out in (torch.bfloat16, torch.float32):
            _check(_cdg().linear(x, w, bias, residual, activation=act, out_dtype=out), x, w, bias, residual, act, out)


@pytest.mark.parametrize("M,N,K", [(4611, 2568, 130), (8200, 2600, 64), (2560, 2305, 520), (19000, 256, 72)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
def test_linear_many_tiles(M, N, K, dtype, out_dtype):
    """Enough 256 x 256 tiles for every SM pair to take several, with ragged edges."""
    x, w = _operands(M, N, K, dtype, seed=5)
    bias = torch.randn(N, device=DEV)
    for b, r, act in ((None, None, None), (bias.to(dtype), torch.randn(M, N, device=DEV).to(out_dtype), "gelu_tanh"),
                      (bias, torch.randn(M, N, device=DEV), "relu"),
                      (None, torch.randn(M, N, device=DEV).to(dtype), None)):
        got = _cdg().linear(x, w, b, r, activation=act, out_dtype=out_dtype)
        _check(got, x, w, b, r, act, out_dtype)
        assert torch.equal(got, _cdg().linear(x, w, b, r, activation=act, out_dtype=out_dtype))
    y, z = _cdg().linear(x, w, bias, activation="silu", out_dtype=out_dtype, preact=True)
    _check(z, x, w, bias, None, None, dtype)
    _check(y, x, w, bias, None, "silu", out_dtype)


@pytest.mark.parametrize("N,wide,off", [(2306, 2400, 0), (2306, 2401, 5), (2307, 2400, 1), (2307, 2307, 0), (2312, 2322, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_many_tiles_on_odd_rows(N, wide, off, dtype):
    """Rows of the result and of the residual on word boundaries, between them, and on each in turn."""
    M, K = 2593, 264
    x, w = _operands(M, N, K, dtype, seed=9)
    residual = torch.randn(M, wide, device=DEV).to(dtype)[:, off:off + N]
    for r in (None, residual, residual[:1].expand(M, N)):
        got = _cdg().linear(x, w, None, r, activation="silu")
        _check(got, x, w, None, r, "silu", dtype)


def test_linear_preactivation_output():
    x, w = _operands(130, 200, 96, torch.float16, seed=2)
    bias = torch.randn(200, device=DEV).half()
    y, z = _cdg().linear(x, w, bias, activation="gelu", preact=True)
    _check(z, x, w, bias, None, None, torch.float16)
    _check(y, x, w, bias, None, "gelu", torch.float16)


@pytest.mark.parametrize("off,width", [(0, 128), (8, 264), (1, 130), (3, 200)])
def test_linear_strides_broadcast_and_stream(off, width):
    big = torch.randn(300, 512, device=DEV).bfloat16()
    x = big[:150, off:off + width]
    w = big[100:, off:off + width][::2]
    residual = big.t()[:150].contiguous()[:, 7:107]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _cdg().linear(x, w, None, residual)
    s.synchronize()
    _check(got, x, w, None, residual, None, torch.bfloat16)
    # one row of x, and one row of the residual, for every row
    xb, rb = x[:1].expand(150, width), residual[:1].expand(150, 100)
    _check(_cdg().linear(xb, w, None, rb), xb, w, None, rb, None, torch.bfloat16)


def test_linear_empty():
    x, w = _operands(5, 7, 0, torch.bfloat16)
    bias = torch.randn(7, device=DEV)
    r = torch.randn(5, 7, device=DEV).bfloat16()
    _check(_cdg().linear(x, w, bias, r, activation="silu"), x, w, bias, r, "silu", torch.bfloat16)
    _check(_cdg().linear(x, w, out_dtype=torch.float32), x, w, None, None, None, torch.float32)
    x, w = _operands(0, 7, 16, torch.bfloat16)
    assert _cdg().linear(x, w).shape == (0, 7)
    x, w = _operands(4, 0, 16, torch.bfloat16)
    assert _cdg().linear(x, w).shape == (4, 0)


def test_linear_infinities_stay_in_their_rows():
    x, w = _operands(200, 160, 320, torch.bfloat16, seed=3)
    clean = _cdg().linear(x, w)
    x2 = x.clone()
    x2[17, 5] = math.inf
    x2[140, 300] = math.nan
    got = _cdg().linear(x2, w)
    rows = torch.ones(200, dtype=torch.bool, device=DEV)
    rows[17] = rows[140] = False
    assert torch.equal(got[rows], clean[rows])
    assert not bool(torch.isfinite(got[17]).any()) and bool(torch.isnan(got[140]).all())


def _backward64(dy, x, w, z, act):
    dz = dy.double()
    if act:
        zz = z.double().requires_grad_(True)
        dz, = torch.autograd.grad(_act64(zz, act), zz, dz)
    return dz


def _check_gradient(got, want, terms, depth, d, count, small):
    assert got.shape == want.shape
    if want.numel() == 0:
        return
    slack = d * want.abs() + (d * (1 + 2.0 ** -8) + (depth + 64) * 2.0 ** -23) * terms + 2.0 ** -24 + small
    bad = (got.double() - want).abs() > slack
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} out of tolerance"
    if want.numel() >= 256:
        err = (got.double() - want).norm()
        assert float(err) <= (0.6 * math.sqrt(2) * d + 2.0 ** -18) * float(want.norm()) * 1.1 + 2.0 ** -24 * count


@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (1, 1, 1), (128, 256, 192), (130, 70, 100), (1000, 513, 257),
                                   (2048, 256, 1024), (77, 1030, 40), (512, 2048, 512), (4099, 24, 136), (3000, 1024, 1536), (2312, 2570, 2500),
                                   (5000, 2056, 1032)])
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, None), (torch.bfloat16, "silu"), (torch.float16, "gelu"),
                                       (torch.bfloat16, "gelu_tanh"), (torch.float16, "relu")])
def test_linear_backward_against_64_bits(M, N, K, dtype, act):
    x, w = _operands(M, N, K, dtype, seed=4)
    dy = torch.randn(M, N, device=DEV).to(dtype)
    z = torch.randn(M, N, device=DEV).to(dtype) if act else None
    dx, dw, db = _cdg().linear_backward(dy, x, w, z, activation=act, bias_grad=True)
    dz = _backward64(dy, x, w, z, act)
    d = UNIT[dtype]
    count = dz.numel() ** 0.5
    under = 2.0 ** -25 if dtype == torch.float16 else 0.0
    slope = 2.0 ** -20 if act else 0.0
    aw, ax, ady = w.double().abs(), x.double().abs(), dy.double().abs()
    _check_gradient(dx, dz @ w.double(), dz.abs() @ aw, N, d, count, under * aw.sum(0) + slope * (ady @ aw))
    _check_gradient(dw, dz.t() @ x.double(), dz.abs().t() @ ax, M, d, count, under * ax.sum(0) + slope * (ady.t() @ ax))
    # db: FP32 sums of values within 2^-20
    slack = d * dz.sum(0).abs() + (M / 8 + 1100) * 2.0 ** -24 * dz.abs().sum(0) + 2.0 ** -20 * dz.abs().sum(0) + 2.0 ** -24
    assert bool(((db.double() - dz.sum(0)).abs() <= slack).all())
    again = _cdg().linear_backward(dy, x, w, z, activation=act, bias_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dw, db)))
    only = _cdg().linear_backward(dy, x, w, z, activation=act, weight_grad=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
    assert cabi.device_status() == (0, 0)


def test_linear_backward_strides():
    big = torch.randn(260, 700, device=DEV).half()
    for off in (0, 8, 5):
        dy, x, w = big[:200, off:off + 136], big[:200, 200 + off:280 + off], big[:136, 300 + off:380 + off]
        z = big[60:, 400 + off:536 + off]
        got = _cdg().linear_backward(dy, x, w, z, activation="silu", bias_grad=True)
        want = _cdg().linear_backward(dy.contiguous(), x.contiguous(), w.contiguous(), z.contiguous(), activation="silu",
                                      bias_grad=True)
        for a, b in zip(got, want):
            assert float((a.double() - b.double()).norm()) <= 2.0 ** -10 * float(b.double().norm())


def test_linear_backward_against_differences():
    """Central differences of sum(dy * y) in 64 bits; FP16 gradients within 2^-9 of the largest."""
    x, w = _operands(6, 5, 9, torch.float16, seed=7)
    dy = torch.randn(6, 5, device=DEV).half()
    bias = torch.randn(5, device=DEV).half()
    for act in ACTS[2:]:
        y, z = _cdg().linear(x, w, bias, activation=act, preact=True)
        dx, dw, db = _cdg().linear_backward(dy, x, w, z, activation=act, bias_grad=True)

        def f(a, b, c):
            return float((_act64(a @ b.t() + c, act) * dy.double()).sum())

        x64, w64, b64 = x.double(), w.double(), bias.double()
        for which, got in ((0, dx), (1, dw), (2, db)):
            for at in ((0,), (got.numel() - 1,), (got.numel() // 2,)):
                args = [x64, w64, b64]
                e = torch.zeros_like(args[which]).view(-1)
                e[at[0]] = 1e-5
                e = e.view_as(args[which])
                up = f(*(a + e if i == which else a for i, a in enumerate(args)))
                down = f(*(a - e if i == which else a for i, a in enumerate(args)))
                tol = 2.0 ** -9 * float(got.abs().max()) * 4
                assert abs((up - down) / 2e-5 - float(got.view(-1)[at[0]])) < tol


def test_linear_backward_empty():
    x, w = _operands(0, 8, 16, torch.bfloat16)
    dy = torch.empty(0, 8, device=DEV, dtype=torch.bfloat16)
    dx, dw, db = _cdg().linear_backward(dy, x, w, bias_grad=True)
    assert dx.shape == (0, 16) and float(dw.float().abs().sum()) == 0 and float(db.float().abs().sum()) == 0


def test_linear_refusals():
    cdg = _cdg()
    x, w = _operands(4, 8, 16, torch.bfloat16)
    dy = torch.zeros(4, 8, device=DEV, dtype=torch.bfloat16)
    bad = [lambda: cdg.linear(x, w.half()), lambda: cdg.linear(x.float(), w.float()), lambda: cdg.linear(x, w[:, :8]),
           lambda: cdg.linear(x, w, torch.zeros(7, device=DEV)), lambda: cdg.linear(x, w, torch.zeros(8, device=DEV).half()),
           lambda: cdg.linear(x, w, None, torch.zeros(4, 7, device=DEV)), lambda: cdg.linear(x, w, activation="tanh"),
           lambda: cdg.linear(x, w, out_dtype=torch.float16), lambda: cdg.linear(x[0], w),
           lambda: cdg.linear(x.t(), torch.zeros(8, 4, device=DEV, dtype=torch.bfloat16)),
           lambda: cdg.linear_backward(dy, x, w, activation="silu"), lambda: cdg.linear_backward(dy[:3], x, w),
           lambda: cdg.linear_backward(dy.half(), x, w), lambda: cdg.linear_backward(dy, x, w, dy[:, :4], activation="relu")]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        cdg.linear(x.cpu(), w)


@pytest.mark.parametrize("M,N,K", [(4, 0, 16), (1, 0, 8), (300, 0, 264), (5, 8, 0), (300, 0, 0), (0, 0, 8)])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("bias_grad", [False, True])
def test_linear_backward_of_empty_products(M, N, K, act, bias_grad):
    x, w = _operands(M, N, K, torch.bfloat16)
    dy = torch.randn(M, N, device=DEV).bfloat16()
    dx, dw, db = _cdg().linear_backward(dy, x, w, dy if act else None, activation=act, bias_grad=bias_grad)
    assert dx.shape == (M, K) and dw.shape == (N, K) and float(dx.float().abs().sum()) == 0
    assert (db is None) != bias_grad and (db is None or db.shape == (N,))
    if bias_grad and act is None:
        want = dy.double().sum(0)
        assert bool(((db.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * dy.double().abs().sum(0)).all())


def test_persistent_product_keeps_to_the_sm_limit():
    """set_num_sms(2) leaves one CTA pair of the 74 a B200 has: the product of 256 tiles takes many times as long
    (64 tiles a pair instead of four; a factor of four is asked for) and gives the same bits."""
    cdg = _cdg()
    x, w = _operands(4096, 4096, 1024, torch.bfloat16, seed=11)

    def timed():
        y = cdg.linear(x, w)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        start.record()
        for _ in range(5):
            y = cdg.linear(x, w)
        end.record()
        end.synchronize()
        return y, start.elapsed_time(end)

    want, whole = timed()
    cdg.set_num_sms(2)
    try:
        got, limited = timed()
    finally:
        cdg.set_num_sms(0)
    assert torch.equal(got, want)
    assert limited > 4 * whole, (limited, whole)


@pytest.mark.parametrize("rows", [1, 40, 4096])
def test_gelu_tail_is_relatively_accurate(rows):
    """GELU far below zero, y = z Phi(z), with z the operands' own values (x = 1, K = 1, no sum).

    The tail is exp(-z^2 / 2) times a fitted factor.  The factor is within 5e-7 in FP32 and its fast division
    within 2 units in the last place (2.4e-7); exp(x) is within 2 + 1.173 |x| units, its argument z^2 / 2 is
    rounded once (0.25 z^2 2^-23): together within 2^-19 + z^2 2^-23.  Results below 2^-126 may be zero."""
    z = torch.linspace(-14, 2, 2049, device=DEV).bfloat16().unique()
    x = torch.ones(rows, 1, device=DEV).bfloat16()
    want = z.double() * 0.5 * torch.special.erfc(-z.double() / math.sqrt(2))  # ndtr cancels below -5
    near = (2.0 ** -19 + z.double().square() * 2.0 ** -23) * want.abs() + 2.0 ** -126
    got = _cdg().linear(x, z[:, None].contiguous(), activation="gelu", out_dtype=torch.float32)
    assert bool(((got.double() - want).abs() <= near).all())
    got = _cdg().linear(x, z[:, None].contiguous(), activation="gelu")
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8) + near).all())


@pytest.mark.parametrize("M,N,stride,off", [(2626, 2239, 2240, 0), (2626, 2233, 2248, 8), (4096, 2045, 2056, 0),
                                            (513, 1030, 1040, 16), (300, 197, 200, 0), (40, 61, 64, 0), (3, 1001, 1008, 0),
                                            (2600, 2250, 2257, 3)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_z", [False, True])
def test_results_into_columns_of_a_wider_matrix(M, N, stride, off, out, with_z):
    """By the C ABI y and z may be columns of wider matrices: the others' columns keep their values."""
    import ctypes

    from test_operators_host import FP32, BF16, LinearArgs

    lib = cabi.lib()
    x, w = _operands(M, N, 136, torch.bfloat16, seed=15)
    wide = torch.full((off + M * stride,), 7.0, device=DEV, dtype=out)
    z_wide = torch.full((off + M * stride,), 7.0, device=DEV, dtype=torch.bfloat16)
    y, z = (t.as_strided((M, N), (stride, 1), off) for t in (wide, z_wide))
    g = LinearArgs(x=x.data_ptr(), x_stride=136, w=w.data_ptr(), w_stride=136, dtype=BF16,
                   out_dtype=FP32 if out == torch.float32 else BF16, activation=2, M=M, N=N, K=136, y=y.data_ptr(),
                   y_stride=stride, z_out=z.data_ptr() if with_z else None, z_stride=stride)
    lib.cdg_linear.argtypes = [ctypes.POINTER(LinearArgs), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    assert lib.cdg_linear(ctypes.byref(g), None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    _check(y, x, w, None, None, "silu", out)
    if with_z:
        _check(z, x, w, None, None, None, torch.bfloat16)
        z.fill_(7.0)
    y.fill_(7.0)
    assert bool((wide == 7.0).all()) and bool((z_wide == 7.0).all())


@pytest.mark.parametrize("act", ACTS[1:])
def test_activations_and_slopes_of_the_largest_values(act):
    """Far from zero an activation is z or 0 and its slope 1 or 0, up to BF16's largest value."""
    z = torch.tensor([3.3e38, 1e30, 2e19, 1e15, 300.0], device=DEV).bfloat16()
    z = torch.cat([z, -z])
    y = _cdg().linear(z[:, None].contiguous(), torch.ones(1, 1, device=DEV).bfloat16(), activation=act)
    assert torch.equal(y[:5, 0], z[:5]) and float(y[5:].float().abs().sum()) == 0
    dx, _, db = _cdg().linear_backward(torch.ones_like(y), torch.ones_like(y), torch.ones(1, 1, device=DEV).bfloat16(),
                                       z[:, None].contiguous(), activation=act, bias_grad=True)
    assert dx[:, 0].tolist() == [1.0] * 5 + [0.0] * 5 and float(db) == 5.0
