"""GPU checks of the router (top-k gate, counts, balance loss) and its gradient.

Against plain formulas in 64 bits.  Ids, counts and token numbers are exact (logits are compared
as they are).  Tolerances of the numbers, with u = 2^-24 and R the row's range of logits above -inf:
the fast exponential is within 2 + 1.2 |x| units in the last place (2u each), a fast or exact
division within 4u, sums of E terms in lanes and shuffles within (E / 32 + 5) u of the sum of
magnitudes.  So a score or probability is within e = (2 (4 + 2.4 R) + E / 32 + 16) u, a weight
within 2e, and a gradient within 6e of the sum of its terms' magnitudes.
"""

import math

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


def _logits(T, E, dtype, seed=0, off=()):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (torch.randn(T, E, generator=g, device=DEV) * 2).to(dtype)
    for e in off:
        z[:, e] = -math.inf
    mask = torch.rand(T, generator=g, device=DEV) > 0.2
    return z, mask


def _scores(z, scoring):
    z = z.double()
    s = torch.softmax(z, 1).nan_to_num(0.0) if scoring == "softmax" else torch.sigmoid(z)
    return s, s / s.sum(1, keepdim=True).clamp(min=1e-300)


def _error(z, E):
    finite = torch.where(torch.isfinite(z), z.double(), 0.0)
    R = float(finite.max() - finite.min()) if z.numel() else 0.0
    return (2 * (4 + 2.4 * R) + E / 32 + 16) * U


def _route64(z, k, scoring, renorm, scale, mask=None, bias=None):
    s, p = _scores(z, scoring)
    by = z.double() if bias is None else torch.where(z > -math.inf, s + bias.double(), -math.inf)
    v, i = torch.sort(by, dim=1, descending=True, stable=True)
    ok = v[:, :k] > -math.inf
    if mask is not None:
        ok = ok & mask.bool()[:, None]
    ids = torch.where(ok, i[:, :k], -1)
    w = torch.where(ok, s.gather(1, ids.clamp(min=0)), 0.0)
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    counts = torch.bincount(ids[ids >= 0], minlength=z.shape[1])
    valid = ok.any(1)
    n = max(1, int(valid.sum()))
    loss = float((counts.double() * p[valid].sum(0)).sum()) * z.shape[1] / k / n / n
    return ids, w * scale, counts, int(valid.sum()), loss, v


CASES = [(1, 1, 1), (1, 256, 8), (64, 256, 8), (1000, 256, 8), (77, 7, 7), (4099, 161, 6), (333, 1024, 32), (50, 33, 2),
         (20000, 64, 4), (129, 512, 16), (3, 100, 10)]


@pytest.mark.parametrize("T,E,k", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_route_against_64_bits(T, E, k, dtype, scoring, renorm):
    z, mask = _logits(T, E, dtype, off=(3,) if E > 40 else ())
    for m in (None, mask):
        o = _cdg().moe_route(z, k, scoring=scoring, renormalize=renorm, scale=1.5, token_mask=m, balance=True)
        ids, w, counts, valid, loss, _ = _route64(z, k, scoring, renorm, 1.5, m)
        assert torch.equal(o.ids.long(), ids)
        assert torch.equal(o.counts.long(), counts) and int(o.tokens) == valid
        e = _error(z, E)
        assert bool(((o.weights.double() - w).abs() <= 2 * e * w.abs() + 1e-30).all())
        # every probability within e; the sums' own error is below T / 148 u per CTA
        assert abs(float(o.loss) - loss) <= (e + (T / 148 + 16) * U) * loss + 1e-30
        again = _cdg().moe_route(z, k, scoring=scoring, renormalize=renorm, scale=1.5, token_mask=m, balance=True)
        assert torch.equal(again.weights, o.weights) and torch.equal(again.loss, o.loss)
        plain = _cdg().moe_route(z, k, scoring=scoring, renormalize=renorm, scale=1.5, token_mask=m)
        assert plain.loss is None and torch.equal(plain.ids, o.ids) and torch.equal(plain.counts, o.counts)


def test_route_ties_go_to_the_lowest_index():
    z = torch.zeros(5, 256, device=DEV)
    z[1, 200] = z[1, 100] = z[1, 101] = 1.0
    z[2, ::2] = -0.0
    z[3] = torch.arange(256, device=DEV) % 3
    o = _cdg().moe_route(z, 5)
    assert o.ids.tolist() == [[0, 1, 2, 3, 4], [100, 101, 200, 0, 1], [0, 1, 2, 3, 4], [2, 5, 8, 11, 14],
                              [0, 1, 2, 3, 4]]


def test_route_special_rows():
    inf, nan = math.inf, math.nan
    z = torch.randn(8, 40, device=DEV)
    z[0] = -inf                                   # nothing to choose
    z[1] = -inf
    z[1, 33] = 0.5                                # one expert for three slots
    z[2, 5] = nan
    z[3, 7] = inf
    z[4] = nan
    z[5] = torch.finfo(torch.float32).min         # the type's lowest value is a value
    z[6] *= 1e30
    for scoring in ("softmax", "sigmoid"):
        o = _cdg().moe_route(z, 3, scoring=scoring, balance=True)
        assert o.ids[0].tolist() == [-1, -1, -1] and o.ids[4].tolist() == [-1, -1, -1]
        assert float(o.weights[0].abs().sum()) == 0 and float(o.weights[4].abs().sum()) == 0
        assert o.ids[1].tolist() == [33, -1, -1] and o.weights[1].tolist() == [1.0, 0.0, 0.0]
        assert 5 not in o.ids[2].tolist() and int(o.ids[3, 0]) == 7
        assert o.ids[5].tolist() == [0, 1, 2]
        assert int(o.tokens) == 6 and int(o.counts.sum()) == 5 * 3 + 1
        assert bool(torch.isfinite(o.weights).all()) and bool(torch.isfinite(o.loss).all())
        g = _cdg().moe_route_backward(z, o.ids, torch.ones_like(o.weights), torch.ones(1, device=DEV), o.counts, o.tokens,
                                      scoring=scoring)
        assert bool(torch.isfinite(g).all())
        assert float(g[0].abs().sum()) == 0 and float(g[4].abs().sum()) == 0 and float(g[2, 5]) == 0


def test_route_bias_moves_the_choice_only():
    z, mask = _logits(3000, 200, torch.float32, seed=4, off=(9,))
    bias = torch.randn(200, device=DEV) * 0.05
    bias[17] = -math.inf
    for scoring in ("softmax", "sigmoid"):
        o = _cdg().moe_route(z, 6, scoring=scoring, bias=bias, token_mask=mask, balance=True)
        ids, w, counts, valid, loss, v = _route64(z, 6, scoring, True, 1.0, mask, bias)
        # rows whose scores with bias differ by more than their error have one right answer
        clear = (v[:, :6] - v[:, 1:7]).min(1).values > 4 * _error(z, 200) * v.abs().clamp(max=1.0).amax(1)
        assert float(clear.double().mean()) > 0.9
        assert torch.equal(o.ids.long()[clear], ids[clear])
        assert bool(((o.weights.double() - w).abs()[clear] <= 2 * _error(z, 200) * w.abs()[clear] + 1e-30).all())
        assert int(o.tokens) == valid and int(o.counts[17]) == 0 and int(o.counts[9]) == 0


@pytest.mark.parametrize("E", [1, 5, 64, 161, 256, 700])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_a_lone_choice_has_the_weight_one_and_no_gradient(E, scoring):
    z, mask = _logits(777, E, torch.float32, seed=6)
    o = _cdg().moe_route(z, 1, scoring=scoring, token_mask=mask)
    assert torch.equal(o.weights[:, 0], mask.float())
    g = _cdg().moe_route_backward(z, o.ids, torch.randn(777, 1, device=DEV), scoring=scoring)
    assert float(g.abs().max()) == 0


def test_route_strides_streams_and_uint8_mask():
    big = torch.randn(100, 300, device=DEV)
    z = big[:, 11:211]
    mask = (torch.arange(100, device=DEV) % 3 > 0)
    want = _cdg().moe_route(z.contiguous(), 8, token_mask=mask, balance=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _cdg().moe_route(z, 8, token_mask=mask.to(torch.uint8), balance=True)
        g = _cdg().moe_route_backward(z, got.ids, got.weights, got.loss, got.counts, got.tokens)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(g, _cdg().moe_route_backward(z.contiguous(), want.ids, want.weights, want.loss, want.counts,
                                                    want.tokens))


def test_route_no_tokens():
    z = torch.empty(0, 64, device=DEV)
    o = _cdg().moe_route(z, 4, balance=True)
    assert o.ids.shape == (0, 4) and int(o.counts.sum()) == 0 and int(o.tokens) == 0 and float(o.loss) == 0
    assert _cdg().moe_route_backward(z, o.ids, o.weights).shape == (0, 64)
    z = torch.randn(9, 64, device=DEV)
    o = _cdg().moe_route(z, 4, token_mask=torch.zeros(9, dtype=torch.bool, device=DEV), balance=True)
    assert int(o.tokens) == 0 and float(o.loss) == 0 and bool((o.ids == -1).all())


def _backward64(z, ids, gw, gl, counts, tokens, scoring, renorm, scale):
    """(gradient by autograd of the formulas in 64 bits, a bound on its terms' magnitudes)."""
    E, k = z.shape[1], ids.shape[1]
    x = z.double().clone().requires_grad_(True)
    if scoring == "softmax":
        m = torch.where(torch.isfinite(x), x, -1e300).detach().amax(1, keepdim=True)
        e = torch.exp(x - m)
        s = e / e.sum(1, keepdim=True)
        p = s
    else:
        s = torch.sigmoid(x)
        p = s / s.sum(1, keepdim=True)
    ok = ids >= 0
    c = torch.where(ok, s.gather(1, ids.clamp(min=0).long()), 0.0)
    total = c.sum(1, keepdim=True)
    w = c / torch.where(total > 0, total, 1.0) if renorm else c
    f = (w * scale * gw.double()).sum() if gw is not None else 0.0
    valid = ok.any(1)
    load = 0.0
    if gl is not None:
        n = max(1, int(tokens))
        load = float(gl) * counts.double() * E / (k * n * n)
        f = f + (load * torch.where(valid[:, None], p, 0.0)).sum()
    grad, = torch.autograd.grad(f, x)
    grad = grad * valid[:, None]
    with torch.no_grad():
        # what each gradient is a difference of
        up = torch.zeros_like(x)
        if gw is not None:
            gg = torch.where(ok, gw.double().abs() * scale, 0.0)
            t = torch.where(total > 0, total, 1.0) if renorm else 1.0
            gg = torch.where(ok, (gg + ((gg * c).sum(1, keepdim=True) / t if renorm else 0.0)) / t, 0.0)
            up.scatter_add_(1, ids.clamp(min=0).long(), gg)
        a = abs(load) if gl is not None else torch.zeros(E, device=z.device, dtype=torch.float64)
        if scoring == "softmax":
            d = up + a
            terms = p * (d + (d * p).sum(1, keepdim=True))
        else:
            S = s.sum(1, keepdim=True)
            terms = (up + (a + (a * p).sum(1, keepdim=True)) / S) * s
    return grad, terms


@pytest.mark.parametrize("T,E,k", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                            ("sigmoid", False)])
def test_route_backward_against_64_bits(T, E, k, dtype, scoring, renorm):
    z, mask = _logits(T, E, dtype, seed=2)
    o = _cdg().moe_route(z, k, scoring=scoring, renormalize=renorm, scale=2.5, token_mask=mask, balance=True)
    gw = torch.randn(T, k, device=DEV)
    gl = torch.tensor([0.7 * T], device=DEV)
    for w, l in ((gw, gl), (gw, None), (None, gl)):
        got = _cdg().moe_route_backward(z, o.ids, w, l, o.counts, o.tokens, scoring=scoring, renormalize=renorm,
                                        scale=2.5)
        want, terms = _backward64(z, o.ids, w, l, o.counts, o.tokens, scoring, renorm, 2.5)
        assert got.dtype == dtype
        slack = (UNIT[dtype] if dtype != torch.float32 else 0.0) * want.abs() + 6 * _error(z, E) * terms + 1e-30
        bad = (got.double() - want).abs() > slack
        assert not bool(bad.any()), int(bad.sum())


@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_route_backward_against_differences(scoring, renorm):
    """Central differences of the weights' and the loss's sum in 64 bits (step 1e-6; choice fixed)."""
    z, _ = _logits(4, 12, torch.float32, seed=6)
    o = _cdg().moe_route(z, 3, scoring=scoring, renormalize=renorm, scale=2.0, balance=True)
    gw = torch.randn(4, 3, device=DEV)
    gl = torch.tensor([3.0], device=DEV)
    got = _cdg().moe_route_backward(z, o.ids, gw, gl, o.counts, o.tokens, scoring=scoring, renormalize=renorm, scale=2.0)
    ids = o.ids.long()

    def f(x):
        s, p = _scores(x, scoring)
        c = s.gather(1, ids)
        w = 2.0 * (c / c.sum(1, keepdim=True) if renorm else c)
        loss = (o.counts.double() * p.sum(0)).sum() * 12 / 3 / 16
        return float((w * gw.double()).sum() + 3.0 * loss)

    for t, e in ((0, 0), (1, 5), (2, 11), (3, int(ids[3, 0]))):
        d = torch.zeros(4, 12, dtype=torch.float64, device=DEV)
        d[t, e] = 1e-6
        diff = (f(z.double() + d) - f(z.double() - d)) / 2e-6
        assert abs(diff - float(got[t, e])) < 1e-5


def test_route_feeds_the_layer_counts():
    """counts are what the layer's own count of the ids gives, masked tokens left out."""
    from consumer_deep_gemm import native

    z, mask = _logits(500, 64, torch.bfloat16, seed=8)
    o = _cdg().moe_route(z, 8, token_mask=mask)
    assert torch.equal(native.require().ep_count(o.ids, 64), o.counts)
    assert cabi.device_status() == (0, 0)


def test_route_refusals():
    cdg = _cdg()
    z = torch.zeros(4, 16, device=DEV)
    o = cdg.moe_route(z, 2, balance=True)
    bad = [lambda: cdg.moe_route(z, 0), lambda: cdg.moe_route(z, 17), lambda: cdg.moe_route(z[0], 2),
           lambda: cdg.moe_route(z.int(), 2), lambda: cdg.moe_route(z, 2, scoring="tanh"),
           lambda: cdg.moe_route(z, 2, bias=torch.zeros(15, device=DEV)),
           lambda: cdg.moe_route(z, 2, bias=torch.zeros(16, device=DEV).half()),
           lambda: cdg.moe_route(z, 2, token_mask=torch.ones(3, dtype=torch.bool, device=DEV)),
           lambda: cdg.moe_route(z, 2, token_mask=torch.ones(4, device=DEV)),
           lambda: cdg.moe_route(z.t(), 2),
           lambda: cdg.moe_route_backward(z, o.ids),
           lambda: cdg.moe_route_backward(z, o.ids.long(), o.weights),
           lambda: cdg.moe_route_backward(z, o.ids, o.weights.half()),
           lambda: cdg.moe_route_backward(z, o.ids, None, o.loss),
           lambda: cdg.moe_route_backward(z, o.ids[:2], o.weights[:2])]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cdg.moe_route(z.cpu(), 2), lambda: cdg.moe_route(torch.zeros(1, 1025, device=DEV), 2),
                 lambda: cdg.moe_route(torch.zeros(1, 64, device=DEV), 33)):
        with pytest.raises(RuntimeError):
            call()


def _low(T, E, seed, below):
    """Logits around `below` in every third row, around 0 in the others."""
    z, mask = _logits(T, E, torch.float32, seed=seed, off=(3,) if E > 40 else ())
    z[::3] += below
    return z, mask


def _row_error(E):
    """_error with a row's own range: no row's logits span more than 24 here."""
    return (2 * (4 + 2.4 * 24) + E / 32 + 16) * U


@pytest.mark.parametrize("T,E,k", [(50, 256, 8), (4099, 161, 6), (333, 700, 24), (20000, 33, 2), (9, 16, 16)])
@pytest.mark.parametrize("below", [-100.0, -83.0, -41.0, -600.0])
def test_route_sigmoid_scores_below_the_normal_range(T, E, k, below):
    """Sigmoids of logits below -87 are below 2^-126; their shares are not."""
    z, mask = _low(T, E, seed=12, below=below)
    o = _cdg().moe_route(z, k, scoring="sigmoid", scale=1.5, token_mask=mask, balance=True)
    ids, w, counts, valid, loss, _ = _route64(z, k, "sigmoid", True, 1.5, mask)
    assert torch.equal(o.ids.long(), ids) and torch.equal(o.counts.long(), counts) and int(o.tokens) == valid
    e = _row_error(E)
    assert bool(((o.weights.double() - w).abs() <= 2 * e * w.abs() + 1e-30).all())
    assert abs(float(o.loss) - loss) <= (e + (T / 148 + 16) * U) * loss + 1e-30
    gw = torch.randn(T, k, device=DEV)
    gl = torch.tensor([0.7 * T], device=DEV)
    for renorm in (True, False):
        for a, b in ((gw, gl), (gw, None), (None, gl)):
            got = _cdg().moe_route_backward(z, o.ids, a, b, o.counts, o.tokens, scoring="sigmoid", renormalize=renorm, scale=2.5)
            want, terms = _backward64(z, o.ids, a, b, o.counts, o.tokens, "sigmoid", renorm, 2.5)
            bad = (got.double() - want).abs() > 6 * e * terms + 1e-30
            assert not bool(bad.any()), int(bad.sum())


@pytest.mark.parametrize("E,k", [(64, 4), (64, 12), (600, 5)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_bias_may_choose_scores_below_the_normal_range(E, k, scoring):
    """The bias moves the choice to experts whose scores are e^-150 of the others': their shares sum to 1."""
    T = 500
    z, mask = _logits(T, E, torch.float32, seed=13)
    z[:, E // 2:] -= 150.0
    bias = -0.01 * torch.arange(E, device=DEV, dtype=torch.float32)  # decides among the low ones
    bias[:E // 2] = -20.0
    o = _cdg().moe_route(z, k, scoring=scoring, bias=bias, token_mask=mask)
    want_ids = torch.where(mask[:, None], torch.arange(E // 2, E // 2 + k, device=DEV), -1)
    assert torch.equal(o.ids.long(), want_ids)
    c = torch.softmax(z[:, E // 2:E // 2 + k].double(), 1) * mask[:, None]
    e = _row_error(E)
    assert bool(((o.weights.double() - c).abs() <= 2 * e * c + 1e-30).all())
    gw = torch.randn(T, k, device=DEV)
    got = _cdg().moe_route_backward(z, o.ids, gw, scoring=scoring)
    want, terms = _backward64(z, o.ids, gw, None, o.counts, o.tokens, scoring, True, 1.0)
    assert bool(((got.double() - want).abs() <= 6 * e * terms + 1e-30).all())


@pytest.mark.parametrize("T,E,k", [(1000, 256, 8), (77, 7, 7), (333, 700, 24)])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("sigmoid", False)])
def test_route_backward_of_fp16_logits(T, E, k, scoring, renorm):
    """As against 64 bits above; FP16 results below 2^-14 are rounded to a multiple of 2^-24."""
    z, mask = _logits(T, E, torch.float16, seed=14)
    o = _cdg().moe_route(z, k, scoring=scoring, renormalize=renorm, token_mask=mask, balance=True)
    gw = torch.randn(T, k, device=DEV)
    gl = torch.tensor([0.7 * T], device=DEV)
    got = _cdg().moe_route_backward(z, o.ids, gw, gl, o.counts, o.tokens, scoring=scoring, renormalize=renorm)
    want, terms = _backward64(z, o.ids, gw, gl, o.counts, o.tokens, scoring, renorm, 1.0)
    assert got.dtype == torch.float16
    slack = UNIT[torch.float16] * want.abs() + 6 * _error(z, E) * terms + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= slack).all())
