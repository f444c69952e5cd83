"""GPU checks of MoEBlock: the operators run together around MoELayer.

The routed experts have their own tests; here the layer is called on the block's own normed rows,
ids and weights, so that what is checked is what stands around it.  Tolerances: u, h and logits
as in the operators' tests; the block's output against the layer's plus the shared expert in 64
bits on the same u, within three BF16 roundings (the hidden row, the layer's output, the sum):
norm of the error at most 3 * 0.6 * 2^-8 of the terms' norms.  Router gradients pass two BF16
roundings (dlogits, du) and a third of their own: 3 * 0.6 * 2^-8 of the norm, times 1.5 for the
correlation of the roundings within a row.
"""

import pytest
import torch

import cabi
from moe_ref import make_layer_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
T, E, H, I, K = 96, 8, 256, 128, 2


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(21)


def _block(shared=True, **kw):
    from consumer_deep_gemm.block import MoEBlock
    from consumer_deep_gemm.moe import MoELayer

    x, _, _, w1, w1s, w2, w2s = make_layer_inputs(T, E, H, I, K)
    layer = MoELayer(w1.to(DEV), w1s.to(DEV), w2.to(DEV), w2s.to(DEV), num_experts=E)
    norm = (torch.randn(H, device=DEV) * 0.1 + 1).bfloat16()
    gate = (torch.randn(E, H, device=DEV) * 0.1).bfloat16()
    pair = ((torch.randn(I, H, device=DEV) * 0.05).bfloat16(), (torch.randn(H, I, device=DEV) * 0.05).bfloat16())
    residual = torch.randn(T, H, device=DEV).bfloat16()
    return MoEBlock(norm, gate, layer, K, shared=pair if shared else None, **kw), x.to(DEV), residual, layer, pair


@pytest.mark.parametrize("shared,scoring", [(True, "softmax"), (False, "sigmoid")])
def test_block_forward(shared, scoring):
    block, x, residual, layer, (up, down) = _block(shared, scoring=scoring, scale=1.5)
    mask = torch.rand(T, device=DEV) > 0.25
    o = block(x, residual, token_mask=mask, balance=True)
    h = x.double() + residual.double()
    assert float((o.h.double() - h).norm() / h.norm()) <= 0.6 * 2.0 ** -8
    u = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * block.norm_weight.double()
    assert float((o.normed.double() - u).norm() / u.norm()) <= 0.6 * 2.0 ** -8
    logits = o.normed.double() @ block.gate_weight.double().t()
    assert float((o.logits.double() - logits).norm() / logits.norm()) <= 2.0 ** -19
    # the gate on the block's own logits
    score = torch.softmax(o.logits.double(), 1) if scoring == "softmax" else torch.sigmoid(o.logits.double())
    ids = torch.sort(o.logits, dim=1, descending=True, stable=True).indices[:, :K]
    w = score.gather(1, ids)
    w = 1.5 * w / w.sum(1, keepdim=True)
    assert torch.equal(o.routing.ids.long(), torch.where(mask[:, None], ids, -1))
    assert bool(((o.routing.weights.double() - torch.where(mask[:, None], w, 0.0)).abs() <= 1e-5).all())
    assert int(o.routing.tokens) == int(mask.sum()) and int(o.routing.counts.sum()) == K * int(mask.sum())
    y = layer(o.normed, o.routing.ids, o.routing.weights)
    assert float(y[~mask].float().abs().sum()) == 0  # no routed expert
    want, terms = y.double(), y.double().abs()
    if shared:
        z = o.normed.double() @ up.double().t()
        dense = (z * torch.sigmoid(z)) @ down.double().t()
        want, terms = want + dense, terms + dense.abs()
    assert float((o.out.double() - want).norm()) <= 3 * 0.6 * 2.0 ** -8 * float(terms.norm())
    assert cabi.device_status() == (0, 0)


def test_block_without_residual_and_in_a_graph():
    block, x, _, _, _ = _block()
    o = block(x)
    assert o.h is x and o.routing.loss is None
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = block(x, balance=True)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.routing.ids, o.routing.ids) and torch.equal(c.logits, o.logits)
    # rows of an expert's group are placed by atomics, each computed by itself: the same values
    assert torch.equal(c.out, o.out)
    x.mul_(-1.0)
    g.replay()
    again = block(x)
    assert torch.equal(c.out, again.out) and not torch.equal(again.out, o.out)


def test_block_router_gradients():
    block, x, residual, _, _ = _block(scale=2.0)
    o = block(x, residual, balance=True)
    gw = torch.randn(T, K, device=DEV)
    gl = torch.tensor([5.0], device=DEV)
    g = block.router_gradients(o, gw, gl)
    h = o.h.double().requires_grad_(True)
    nw = block.norm_weight.double().requires_grad_(True)
    gate = block.gate_weight.double().requires_grad_(True)
    u = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * nw
    p = torch.softmax(u @ gate.t(), 1)
    c = p.gather(1, o.routing.ids.long())
    loss = (o.routing.counts.double() * p.sum(0)).sum() * E / K / T / T
    f = (2.0 * c / c.sum(1, keepdim=True) * gw.double()).sum() + 5.0 * loss
    want = torch.autograd.grad(f, (gate, nw, h))
    for a, b in zip((g.gate_weight, g.norm_weight, g.h), want):
        assert float((a.double() - b).norm()) <= 1.5 * 3 * 0.6 * 2.0 ** -8 * float(b.norm())


def test_block_refusals():
    from consumer_deep_gemm.block import MoEBlock

    block, _, _, layer, _ = _block()
    with pytest.raises(ValueError):
        MoEBlock(block.norm_weight, block.gate_weight[:, :128], layer, K)
    with pytest.raises(ValueError):
        MoEBlock(block.norm_weight, block.gate_weight[:4], layer, K)


def test_block_of_no_tokens():
    block, x, residual, _, _ = _block()
    o = block(x[:0], residual[:0], balance=True)
    assert o.out.shape == (0, H) and o.logits.shape == (0, E) and int(o.routing.tokens) == 0


def test_operators_without_programmatic_launches():
    """set_pdl(False) changes when kernels start, not what they compute."""
    import consumer_deep_gemm as cdg

    x = torch.randn(700, 1000, device=DEV).bfloat16()
    w = (torch.randn(300, 1000, device=DEV) / 32).bfloat16()
    nw = torch.rand(1000, device=DEV) + 0.5
    gw = torch.randn(700, 8, device=DEV)

    def everything():
        n = cdg.add_rms_norm(x, nw, x, quantize=True)
        dh = cdg.add_rms_norm_backward(n.y, n.h, nw, n.y)
        z = cdg.linear(n.y, w, out_dtype=torch.float32)
        r = cdg.moe_route(z, 8, balance=True)
        dz = cdg.moe_route_backward(z, r.ids, gw, r.loss, r.counts, r.tokens)
        y, pre = cdg.linear(n.y, w, activation="silu", preact=True)
        d = cdg.linear_backward(dz.bfloat16(), n.y, w, pre, activation="silu", bias_grad=True)
        odd = cdg.linear(x[:, 1:], w[:, 1:], activation="gelu")
        return [*n[:2], n.q.view(torch.uint8), n.scale, *dh, z, *r, dz, y, pre, *d, odd]

    want = everything()
    cdg.set_pdl(False)
    try:
        got = everything()
    finally:
        cdg.set_pdl(True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_products_on_two_streams_at_once():
    """Persistent and tile kernels beside each other: the bits of the calls one after the other."""
    import consumer_deep_gemm as cdg

    shapes = [(4096, 2048, 512), (300, 512, 2048), (1, 4096, 1024), (2593, 2307, 264), (64, 256, 4096)]
    calls = [((torch.randn(m, k, device=DEV).bfloat16(), (torch.randn(n, k, device=DEV) / k ** 0.5).bfloat16()))
             for m, n, k in shapes]
    want = [cdg.linear(x, w, activation="gelu_tanh") for x, w in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for x, w in calls if i == 0 else calls[::-1]:
                    got[i].append(cdg.linear(x, w, activation="gelu_tanh"))
    torch.cuda.synchronize()
    for i in range(2):
        for j, y in enumerate(got[i]):
            assert torch.equal(y, (want if i == 0 else want[::-1])[j % len(want)])
    assert cabi.device_status() == (0, 0)
