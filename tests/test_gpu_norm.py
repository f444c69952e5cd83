"""GPU checks of the RMS norm (with residual, with e4m3 output) and its gradient.

Against plain formulas in 64 bits on the same inputs.  Tolerances, from the arithmetic (u = 2^-24,
FP32's unit roundoff; d = the unit roundoff of the output's type: half the spacing above 1 of a
significand of 8 bits (BF16, 2^-8), 11 bits (FP16, 2^-11) or 24 bits (FP32, 2^-24)):
  * h is one FP32 sum and one rounding: within (d + 2u) |h|.
  * y: the mean of H squares in FP32 partial sums of at most 40 terms in a row, a square root, a
    division and two products: within (d + 40u) |y|.
  * scales: of a 32-bit y, one division: within 42u.  Codes: e4m3 of values within 44u of the exact
    ones; equal, except where the exact value lies within 44u of an e4m3 rounding point, where
    they are one step apart.
  * dx, dw: sums whose terms are each within 40u: within d |result| + 80u sum |terms|, with T
    terms a column added in FP32, at most T / grid + grid / 8 + 8 of them in a row, for dw.
"""

import pytest
import torch

import cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _seed():
    """The same inputs in every run and order."""
    torch.manual_seed(20)


def _cdg():
    import consumer_deep_gemm

    return consumer_deep_gemm


def _inputs(T, H, dtype, wdtype, residual, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, H, generator=g, device=DEV).to(dtype)
    w = (torch.randn(H, generator=g, device=DEV) * 0.3 + 1).to(wdtype)
    r = (torch.randn(T, H, generator=g, device=DEV) * 2).to(dtype) if residual else None
    return x, w, r


def _norm64(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    return h, h * torch.rsqrt((h * h).mean(1, keepdim=True) + eps) * w.double()


def _within(got, want, slack, what):
    bad = (got.double() - want).abs() > slack
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} values out of tolerance"


def _e4m3_steps(v):
    """The spacing of e4m3 values around v (64 bits)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)


def _check_quant(y64, q, scale, pow2):
    T, H = y64.shape
    kb = (H + 127) // 128
    pad = torch.nn.functional.pad(y64, (0, kb * 128 - H)).view(T, kb, 128)
    amax = pad.abs().amax(2).clamp(min=1e-12)
    want = amax / 448
    if pow2:
        want = torch.exp2(torch.ceil(torch.log2(want)))
    _within(scale, want, 42 * U * want, "scale")
    v = (pad / want[:, :, None]).view(T, kb * 128)[:, :H]
    code = q.double()
    step = _e4m3_steps(v)
    # |code - v| is at most half a step where the rounding is right, and 44u more where the
    # 32-bit value fell on the other side of the rounding point
    _within(code, v, step * 0.5 * (1 + 1e-12) + 44 * U * v.abs(), "e4m3 codes")


SHAPES = [(1, 1), (3, 7), (5, 128), (1, 4096), (300, 4096), (301, 1000), (700, 130), (64, 8192), (9, 257), (700, 2560),
          (3, 32768), (4, 9001), (1000, 64), (2, 16384), (600, 1023)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype,wdtype,residual", [(torch.bfloat16, torch.bfloat16, True),
                                                   (torch.bfloat16, torch.float32, False),
                                                   (torch.float16, torch.float16, True),
                                                   (torch.float32, torch.float32, True)])
def test_norm_against_64_bits(T, H, dtype, wdtype, residual):
    x, w, r = _inputs(T, H, dtype, wdtype, residual)
    o = _cdg().add_rms_norm(x, w, r, eps=1e-5, quantize=True)
    h, y = _norm64(x, w, r, 1e-5)
    if residual:
        _within(o.h, h, (UNIT[dtype] + 2 * U) * h.abs() + 1e-30, "h")
    else:
        assert o.h is None
    # FP16 outputs below 2^-14 are rounded to a multiple of 2^-24
    floor = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    _within(o.y, y, (UNIT[dtype] + 40 * U) * y.abs() + floor, "y")
    _check_quant(y, o.q, o.scale, pow2=False)


@pytest.mark.parametrize("T,H", [(65, 4096), (33, 1000), (7, 77)])
def test_norm_power_of_two_scales(T, H):
    x, w, _ = _inputs(T, H, torch.bfloat16, torch.float32, False, seed=3)
    o = _cdg().add_rms_norm(x, w, eps=1e-6, quantize=True, ue8m0=True, normed=False)
    assert o.y is None and o.h is None
    bits = o.scale.view(torch.int32)
    assert int((bits & 0x7FFFFF).abs().sum()) == 0
    _, y = _norm64(x, w, None, 1e-6)
    # blocks whose largest value lies at a power of two itself may take either neighbour
    _check_quant(y, o.q, o.scale, pow2=True)


def test_norm_quantised_output_feeds_the_grouped_gemm():
    """The codes and scales are the GEMM's own operand form."""
    from consumer_deep_gemm import synthetic  # noqa: F401  (package import path check)

    x, w, r = _inputs(256, 512, torch.bfloat16, torch.bfloat16, True, seed=5)
    o = _cdg().add_rms_norm(x, w, r, quantize=True)
    g = torch.Generator().manual_seed(1)
    b = torch.randint(0, 256, (1, 256, 256), generator=g, dtype=torch.uint8).to(DEV)
    sb = torch.full((1, 256, 16), 121, dtype=torch.uint8, device=DEV)
    d = torch.empty(256, 256, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(256, dtype=torch.int32, device=DEV)
    _cdg().m_grouped_fp8_fp4_gemm_nt_contiguous((o.q, o.scale), (b, sb), d, ids)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=DEV)
    wt = torch.stack([table[(b[0] & 15).long()], table[(b[0] >> 4).long()]], 2).reshape(256, 512).double() * 2.0 ** -6
    want = (o.q.double() * o.scale.double().repeat_interleave(128, 1)) @ wt.t()
    err = (d.double() - want).norm() / want.norm()
    assert float(err) < 4e-3  # BF16 roundings of the GEMM's activations and of its output
    assert cabi.device_status() == (0, 0)


def test_norm_strided_rows_other_stream_and_repeat():
    big = torch.randn(50, 3 * 520 + 4, device=DEV).to(torch.bfloat16)
    for off in (0, 3):  # rows on 16-byte boundaries or not
        x = big[:, off:off + 520]
        r = big[::1, 1040 + off:1560 + off]
        w = torch.linspace(0.5, 1.5, 520, device=DEV)
        want = _cdg().add_rms_norm(x.contiguous(), w, r.contiguous(), quantize=True)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = _cdg().add_rms_norm(x, w, r, quantize=True)
        s.synchronize()
        _, y = _norm64(x, w, r, 1e-6)
        _within(got.y, y, (UNIT[torch.bfloat16] + 40 * U) * y.abs() + 1e-30, "y")
        assert torch.equal(got.h, want.h)
        again = _cdg().add_rms_norm(x, w, r, quantize=True)
        assert torch.equal(again.y, got.y) and torch.equal(again.q.view(torch.uint8), got.q.view(torch.uint8))


def test_norm_special_rows():
    x = torch.randn(6, 300, device=DEV)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[3] = 1e-30
    x[4] = 1e18
    w = torch.ones(300, device=DEV)
    o = _cdg().add_rms_norm(x, w, quantize=True)
    assert float(o.y[0].abs().sum()) == 0 and float(o.q[0].float().abs().sum()) == 0
    assert bool(torch.isfinite(o.scale[0]).all())
    assert bool(torch.isnan(o.y[1]).all()) and bool(torch.isnan(o.q[1].float()).all())
    assert bool(torch.isnan(o.y[2, 7])) and float(o.y[2, :7].abs().sum()) == 0
    assert bool(torch.isfinite(o.y[3:]).all())
    _, y = _norm64(x[4:], w, None, 1e-6)
    _within(o.y[4:], y, (UNIT[torch.float32] + 40 * U) * y.abs(), "large and ordinary rows")


def test_norm_no_rows():
    x = torch.empty(0, 256, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(256, device=DEV, dtype=torch.bfloat16)
    o = _cdg().add_rms_norm(x, w, x, quantize=True)
    assert o.y.shape == (0, 256) and o.scale.shape == (0, 2)
    dx, dw = _cdg().add_rms_norm_backward(x, x, w)
    assert dx.shape == (0, 256) and float(dw.float().abs().sum()) == 0


def _backward64(dy, h, w, dh, eps):
    h, dy, w = h.double(), dy.double(), w.double()
    s = torch.rsqrt((h * h).mean(1, keepdim=True) + eps)
    u = w * dy
    n = h * s
    m = (u * n).mean(1, keepdim=True)
    dx = s * (u - n * m)
    parts = s * (u.abs() + n.abs() * (u * n).abs().mean(1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
        parts = parts + dh.double().abs()
    return dx, parts, (dy * n).sum(0), (dy * n).abs().sum(0)


@pytest.mark.parametrize("T,H", SHAPES + [(5000, 96), (2000, 515)])
@pytest.mark.parametrize("dtype,wdtype,residual", [(torch.bfloat16, torch.bfloat16, True),
                                                   (torch.float16, torch.float32, False),
                                                   (torch.float32, torch.float32, True)])
def test_norm_backward_against_64_bits(T, H, dtype, wdtype, residual):
    x, w, r = _inputs(T, H, dtype, wdtype, True, seed=1)
    dh = r if residual else None
    h = (x * 2).to(dtype)
    dy = _inputs(T, H, dtype, wdtype, False, seed=2)[0]
    dx, dw = _cdg().add_rms_norm_backward(dy, h, w, dh, eps=1e-5)
    want, parts, ww, wparts = _backward64(dy, h, w, dh, 1e-5)
    floor = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    _within(dx, want, UNIT[dtype] * want.abs() * (1 + 1e-6) + 80 * U * parts + floor, "dx")
    row = T / 148 + 148 * 16 / 8 + 8 + 40  # additions in a row, at most
    _within(dw, ww, UNIT[wdtype] * ww.abs() + row * U * wparts + (2.0 ** -25 if wdtype == torch.float16 else 1e-30), "dw")
    again = _cdg().add_rms_norm_backward(dy, h, w, dh, eps=1e-5)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_norm_backward_against_differences():
    """Central differences of sum(dy * y) in 64 bits, step 1e-5: their error is below 1e-8 here."""
    T, H = 3, 37
    x, w, _ = _inputs(T, H, torch.float32, torch.float32, False, seed=9)
    dy = torch.randn(T, H, device=DEV)
    dx, dw = _cdg().add_rms_norm_backward(dy, x, w, eps=1e-3)
    x64, w64, dy64 = x.double(), w.double(), dy.double()

    def f(a, b):
        return float((_norm64(a, b, None, 1e-3)[1] * dy64).sum())

    for i, j in ((0, 0), (1, 17), (2, 36)):
        e = torch.zeros_like(x64)
        e[i, j] = 1e-5
        assert abs((f(x64 + e, w64) - f(x64 - e, w64)) / 2e-5 - float(dx[i, j])) < 2e-5
    for j in (0, 36):
        e = torch.zeros_like(w64)
        e[j] = 1e-5
        assert abs((f(x64, w64 + e) - f(x64, w64 - e)) / 2e-5 - float(dw[j])) < 2e-5


def test_norm_refusals():
    cdg = _cdg()
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    bad = [lambda: cdg.add_rms_norm(x, w[:32]),
           lambda: cdg.add_rms_norm(x, w.half()),
           lambda: cdg.add_rms_norm(x, w, x.float()),
           lambda: cdg.add_rms_norm(x, w, x[:2]),
           lambda: cdg.add_rms_norm(x.t(), torch.ones(4, device=DEV, dtype=torch.bfloat16)),
           lambda: cdg.add_rms_norm(x, w, normed=False),
           lambda: cdg.add_rms_norm(x.int(), w),
           lambda: cdg.add_rms_norm(x, w, eps=-1.0),
           lambda: cdg.add_rms_norm(x[0], w),
           lambda: cdg.add_rms_norm_backward(x[:3], x, w),
           lambda: cdg.add_rms_norm_backward(x.half(), x, w),
           lambda: cdg.add_rms_norm_backward(x, x, w, x[:, :32])]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        cdg.add_rms_norm(x.cpu(), w)
    with pytest.raises(RuntimeError):
        cdg.add_rms_norm(torch.zeros(1, 32769, device=DEV), torch.ones(32769, device=DEV))


@pytest.mark.parametrize("T,H", [(3000, 1024), (5, 4096), (300, 640)])
@pytest.mark.parametrize("ue8m0", [False, True])
def test_norm_codes_are_the_quantisers(T, H, ue8m0):
    """Scales of the FP32 y bit for bit those of the framework's quantiser.  Codes: e4m3 of y * (448 / amax)
    against e4m3 of y / amax * 448, each two roundings: equal but where a rounding point of e4m3 lies
    within 4u of the value, and then one step apart; a power-of-two scale divides exactly."""
    from consumer_deep_gemm import native

    for offset in (0, 1):  # rows on 16-byte boundaries, or not
        x = torch.randn(T, H + 1, device=DEV)[:, offset:offset + H]
        w = torch.rand(H, device=DEV) + 0.5
        o = _cdg().add_rms_norm(x, w, quantize=True, ue8m0=ue8m0)
        q, scale = native.require().quant_fp8_rows(o.y, ue8m0)
        assert torch.equal(o.scale.view(torch.int32), scale.view(torch.int32))
        a, b = o.q.double(), q.view(torch.float8_e4m3fn).double()
        if ue8m0:
            assert torch.equal(a, b)
            continue
        amax = o.y.double().view(T, H // 128, 128).abs().amax(2, keepdim=True)
        v = (o.y.double().view(T, H // 128, 128) / amax * 448).view(T, H)
        apart = a != b
        assert bool(((a - b).abs() <= _e4m3_steps(v))[apart].all())
        assert bool((((a + b) / 2 - v).abs() <= 4 * U * v.abs())[apart].all())


@pytest.mark.parametrize("T,H", [(5, 136), (700, 8), (3, 392), (4, 1), (6, 129), (3, 16392)])
@pytest.mark.parametrize("ue8m0", [False, True])
def test_norm_last_blocks_of_a_few_columns(T, H, ue8m0):
    x, w, r = _inputs(T, H, torch.float32, torch.float32, True, seed=17)
    o = _cdg().add_rms_norm(x, w, r, quantize=True, ue8m0=ue8m0)
    _check_quant(_norm64(x, w, r, 1e-6)[1], o.q, o.scale, pow2=ue8m0)
