"""Cases of the operators around the routed experts of a mixture-of-experts block.

Three operators, each forward and backward:

* ``norm``    RMS norm with the residual's addition and an e4m3 output with 1x128 scales
* ``route``   top-k gate over router logits, per-expert counts and the balance loss
* ``linear``  matrix product with bias, activation and residual in its epilogue

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true,
through the entry points of ``consumer_deep_gemm``.  ``exact`` gives the same outputs from the
definitions in 64 bits.  Sizes are those of the benchmark's layer (hidden 4096, intermediate 2048,
256 experts, top-8, 32,768 tokens) and generic ones around them.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def _package():
    path = os.path.join(_ROOT, "consumer-deepgemm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import consumer_deep_gemm

    return consumer_deep_gemm


# ------------------------------------------------------------------------------------ cases
def _norm(name, T, H, dtype="bf16", weight="bf16", residual=True, quantize=True, normed=True):
    return {"name": name, "op": "norm", "T": T, "H": H, "dtype": dtype, "weight": weight, "residual": residual,
            "quantize": quantize, "normed": normed}


def _norm_backward(name, T, H, dtype="bf16", weight="bf16", residual=True):
    return {"name": name, "op": "norm_backward", "T": T, "H": H, "dtype": dtype, "weight": weight,
            "residual": residual}


def _route(name, T, E, k, dtype="fp32", scoring="softmax", renormalize=True, masked=False, balance=False,
           op="route"):
    return {"name": name, "op": op, "T": T, "E": E, "k": k, "dtype": dtype, "scoring": scoring,
            "renormalize": renormalize, "masked": masked, "balance": balance}


def _linear(name, M, N, K, dtype="bf16", out="bf16", activation="", bias=False, residual=False):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "out": out,
            "activation": activation, "bias": bias, "residual": residual}


def _linear_backward(name, M, N, K, dtype="bf16", activation="silu", bias=True):
    return {"name": name, "op": "linear_backward", "M": M, "N": N, "K": K, "dtype": dtype, "activation": activation,
            "bias": bias}


def listed():
    return [
        # the norm before the experts while decoding a small batch: latency counts
        _norm("norm decode", 8, 4096),
        # the same norm over a prefill batch of the benchmark's layer, y for the router and the
        # experts, e4m3 for a dense FP8 product
        _norm("norm prefill", 32768, 4096),
        # odd row count, a last block of 72 columns, no residual, the 8-bit output alone
        _norm("norm ragged", 6007, 2504, dtype="fp16", weight="fp32", residual=False, normed=False),
        # training: gradients of the norm, the residual stream's gradient added
        _norm_backward("norm backward", 16384, 4096),
        # the gate of 64 decoded tokens over 256 experts
        _route("route decode", 64, 256, 8),
        # the gate of the benchmark's batch in training: padding tokens, disabled experts, balance loss
        _route("route balance", 32768, 256, 8, masked=True, balance=True),
        # gradients of gate weights and balance loss, odd sizes, BF16 logits (with ties)
        _route("route backward", 16389, 161, 6, dtype="bf16", renormalize=False, masked=True, balance=True,
               op="route_backward"),
        # one token through a dense projection: the weights are read once
        _linear("linear decode", 1, 4096, 4096, activation="silu", bias=True),
        # router logits of the benchmark's batch, 32-bit output
        _linear("linear router", 32768, 256, 4096, out="fp32"),
        # odd sizes whose rows start at no 16-byte boundary
        _linear("linear odd", 1237, 2050, 1030, dtype="fp16", out="fp16", activation="gelu", bias=True),
        # a dense projection over a prefill batch with everything in the epilogue
        _linear("linear prefill", 8192, 4096, 4096, activation="gelu_tanh", bias=True, residual=True),
        # training: gradients of a shared expert's first product
        _linear_backward("linear backward", 8192, 2048, 4096),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _rounded(rng, n, to):
    """Half of the sizes are multiples of `to`, the other half stay as drawn, odd ones among them."""
    return (n + to - 1) // to * to if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "route", "route_backward", "linear", "linear", "linear_backward"])
    if op in ("norm", "norm_backward"):
        H = _rounded(rng, _log_int(rng, 64, 8192), 128)
        T = _log_int(rng, 1, min(32768, 32768 * 4096 // H))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            T = max(1, T // 2)
        weight = rng.choice([dtype, "fp32"])
        if op == "norm_backward":
            c = _norm_backward("", T, H, dtype, weight, rng.random() < 0.7)
        else:
            quantize = rng.random() < 0.7
            c = _norm("", T, H, dtype, weight, rng.random() < 0.7, quantize, not quantize or rng.random() < 0.6)
    elif op in ("route", "route_backward"):
        E = _rounded(rng, _log_int(rng, 4, 512), 32)
        k = _log_int(rng, 1, min(E, 16))
        T = _log_int(rng, 1, 65536)
        c = _route("", T, E, k, rng.choice(["fp32", "bf16"]), rng.choice(["softmax", "softmax", "sigmoid"]),
                   rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.6, op)
    else:
        most = 8192 * 4096 * 4096 // (1 if op == "linear" else 2)
        while True:
            M, N, K = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
            N, K = _rounded(rng, N, 64), _rounded(rng, K, 64)
            if M * N * K <= most:
                break
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        if op == "linear":
            c = _linear("", M, N, K, dtype, rng.choice([dtype, dtype, "fp32"]),
                        rng.choice(["", "relu", "silu", "gelu", "gelu_tanh"]), rng.random() < 0.5, rng.random() < 0.5)
        else:
            c = _linear_backward("", M, N, K, dtype, rng.choice(["", "relu", "silu", "gelu", "gelu_tanh"]),
                                 rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype="fp32", std=1.0, mean=0.0):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return (t * std + mean).to(_DTYPES[dtype])

    s = dict(case)
    op = case["op"]
    if op in ("norm", "norm_backward"):
        T, H, dt = case["T"], case["H"], case["dtype"]
        s["w"] = normal(H, dtype=case["weight"], std=0.1, mean=1.0)
        if op == "norm":
            s["x"] = normal(T, H, dtype=dt)
            s["r"] = normal(T, H, dtype=dt, std=2.0) if case["residual"] else None
        else:
            s["h"] = normal(T, H, dtype=dt, std=2.0)
            s["dy"] = normal(T, H, dtype=dt, std=0.1)
            s["dh"] = normal(T, H, dtype=dt, std=0.1) if case["residual"] else None
    elif op in ("route", "route_backward"):
        T, E, k = case["T"], case["E"], case["k"]
        # a popularity of each expert under the tokens' own preferences
        s["logits"] = (normal(T, E) + normal(E, std=0.5)).to(_DTYPES[case["dtype"]])
        s["mask"] = None
        if case["masked"]:  # padding tokens, and every 64th expert switched off
            s["mask"] = torch.rand(T, generator=g, device="cuda") >= 0.05
            s["logits"][:, 3::64] = -math.inf
        if op == "route_backward":
            # what the forward pass left: ids, counts and the number of valid tokens
            ids, _, valid = _choose(s["logits"].float(), k, s["mask"])
            s["ids"] = ids
            s["counts"] = torch.bincount(ids[ids >= 0].long(), minlength=E)[:E].to(torch.int32)
            s["tokens"] = valid.sum().to(torch.int32).reshape(1)
            s["gw"] = normal(T, k, std=0.1)
            s["gl"] = normal(1, mean=float(T), std=0.01 * T) if case["balance"] else None
    else:
        M, N, K, dt = case["M"], case["N"], case["K"], case["dtype"]
        s["x"] = normal(M, K, dtype=dt)
        s["w"] = normal(N, K, dtype=dt, std=0.02)
        if op == "linear":
            s["b"] = normal(N, dtype=dt, std=0.5) if case["bias"] else None
            s["r"] = normal(M, N, dtype=dt) if case["residual"] else None
        else:
            s["z"] = normal(M, N, dtype=dt) if case["activation"] else None
            s["dy"] = normal(M, N, dtype=dt, std=0.1)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _choose(scores, k, mask):
    """(ids, selectable, valid): the k largest of each row, ties to the lowest index; -1 where the
    token is masked or no expert above -inf is left."""
    top = torch.sort(scores, dim=1, descending=True, stable=True)
    ids = top.indices[:, :k]
    ok = top.values[:, :k] > -math.inf
    valid = top.values[:, 0] > -math.inf
    if mask is not None:
        ok = ok & mask[:, None]
        valid = valid & mask
    return torch.where(ok, ids, -1).to(torch.int32), ok, valid


def _probabilities(logits, scoring):
    """(scores, probabilities) of each row in 32 bits; rows without a value above -inf are 0."""
    if scoring == "softmax":
        m = logits.max(dim=1, keepdim=True).values
        e = torch.exp(logits - torch.where(m > -math.inf, m, 0.0))
    else:
        e = 1.0 / (1.0 + torch.exp(-logits))
    total = e.sum(dim=1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    return (p if scoring == "softmax" else e), p


def _plain_norm(s):
    x = s["x"].float()
    h = x if s["r"] is None else x + s["r"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["w"].float()
    out = {}
    if s["r"] is not None:
        out["h"] = h.to(s["x"].dtype)
    if s["normed"]:
        out["y"] = y.to(s["x"].dtype)
    if s["quantize"]:
        T, H = y.shape
        pad = -H % 128
        blocks = torch.nn.functional.pad(y, (0, pad)).view(T, (H + pad) // 128, 128)
        amax = blocks.abs().amax(dim=2, keepdim=True).clamp(min=1e-12)
        q = (blocks / amax * 448.0).to(torch.float8_e4m3fn)
        out["q"] = q.view(T, H + pad)[:, :H]
        out["scale"] = (amax / 448.0).squeeze(2)
    return out


def _plain_norm_backward(s):
    h, dy, w = s["h"].float(), s["dy"].float(), s["w"].float()
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    n, u = h * rstd, dy * w
    dx = rstd * (u - n * (u * n).mean(dim=1, keepdim=True))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["h"].dtype), "dw": (dy * n).sum(dim=0).to(s["w"].dtype)}


def _plain_route(s):
    logits, k = s["logits"].float(), s["k"]
    E = logits.shape[1]
    ids, ok, valid = _choose(logits, k, s["mask"])
    score, p = _probabilities(logits, s["scoring"])
    w = torch.where(ok, torch.gather(score, 1, ids.clamp(min=0).long()), 0.0)
    if s["renormalize"]:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    counts = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
    counts = counts.index_add_(0, torch.where(ok, ids, E).reshape(-1).long(),
                               torch.ones(ids.numel(), dtype=torch.int32, device=ids.device))[:E]
    tokens = valid.sum().to(torch.int32).reshape(1)
    out = {"weights": w * 2.5, "ids": ids, "counts": counts, "tokens": tokens}
    if s["balance"]:
        n = tokens.float().clamp(min=1.0)
        mean_p = torch.where(valid[:, None], p, 0.0).sum(dim=0) / n
        out["loss"] = (counts.float() * (E / k) / n * mean_p).sum().reshape(1)
    return out


def _plain_route_backward(s):
    logits, k = s["logits"].float(), s["k"]
    E = logits.shape[1]
    ids = s["ids"].long()
    ok = ids >= 0
    valid = ok.any(dim=1, keepdim=True)
    score, p = _probabilities(logits, s["scoring"])
    at = ids.clamp(min=0)
    g = torch.where(ok, s["gw"], 0.0) * 2.5
    if s["renormalize"]:
        chosen = torch.where(ok, torch.gather(score, 1, at), 0.0)
        total = chosen.sum(dim=1, keepdim=True)
        total = torch.where(total > 0, total, 1.0)
        g = torch.where(ok, (g - (g * chosen).sum(dim=1, keepdim=True) / total) / total, 0.0)
    dscore = torch.zeros_like(logits).scatter_add_(1, at, g)
    if s["scoring"] == "softmax":
        d = dscore
    else:
        d = 0.0
    if s["gl"] is not None:
        n = s["tokens"].float().clamp(min=1.0)
        d = d + s["gl"] * s["counts"].float() * (E / k) / n / n
    if s["scoring"] == "softmax":
        out = p * (d - (d * p).sum(dim=1, keepdim=True))
    else:
        if s["gl"] is not None:
            total = score.sum(dim=1, keepdim=True)
            dscore = dscore + (d - (d * p).sum(dim=1, keepdim=True)) / torch.where(total > 0, total, 1.0)
        out = dscore * score * (1.0 - score)
    return {"dlogits": torch.where(valid, out, 0.0).to(s["logits"].dtype)}


def _plain_act(z, kind):
    if kind == "relu":
        return torch.clamp(z, min=0.0)
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_act_slope(z, kind):
    if kind == "relu":
        return (z > 0).float()
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _plain_act(z, s["activation"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(_DTYPES[s["out"]])}


def _plain_linear_backward(s):
    dt = s["x"].dtype
    dz = s["dy"].float()
    if s["activation"]:
        dz = dz * _plain_act_slope(s["z"].float(), s["activation"])
    out = {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ s["x"].float()).to(dt)}
    if s["bias"]:
        out["db"] = dz.sum(dim=0).to(dt)
    return out


# ------------------------------------------------------------------------------------ the framework's
def _own_norm(s):
    cdg = _package()
    o = cdg.add_rms_norm(s["x"], s["w"], s["r"], eps=EPS, quantize=s["quantize"], normed=s["normed"])
    return {name: t for name, t in (("h", o.h), ("y", o.y), ("q", o.q), ("scale", o.scale)) if t is not None}


def _own_norm_backward(s):
    dx, dw = _package().add_rms_norm_backward(s["dy"], s["h"], s["w"], s["dh"], eps=EPS)
    return {"dx": dx, "dw": dw}


def _own_route(s):
    o = _package().moe_route(s["logits"], s["k"], scoring=s["scoring"], renormalize=s["renormalize"], scale=2.5,
                             token_mask=s["mask"], balance=s["balance"])
    out = {"weights": o.weights, "ids": o.ids, "counts": o.counts, "tokens": o.tokens}
    if s["balance"]:
        out["loss"] = o.loss
    return out


def _own_route_backward(s):
    return {"dlogits": _package().moe_route_backward(s["logits"], s["ids"], s["gw"], s["gl"], s["counts"], s["tokens"],
                                                     scoring=s["scoring"], renormalize=s["renormalize"], scale=2.5)}


def _own_linear(s):
    return {"y": _package().linear(s["x"], s["w"], s["b"], s["r"], activation=s["activation"] or None,
                                   out_dtype=_DTYPES[s["out"]])}


def _own_linear_backward(s):
    dx, dw, db = _package().linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=s["activation"] or None,
                                            bias_grad=s["bias"])
    return {"dx": dx, "dw": dw, "db": db} if s["bias"] else {"dx": dx, "dw": dw}


_PLAIN = {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "route": _plain_route,
          "route_backward": _plain_route_backward, "linear": _plain_linear, "linear_backward": _plain_linear_backward}
_OWN = {"norm": _own_norm, "norm_backward": _own_norm_backward, "route": _own_route,
        "route_backward": _own_route_backward, "linear": _own_linear, "linear_backward": _own_linear_backward}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------------------------------------ least work
def work(case):
    op = case["op"]
    if op in ("norm", "norm_backward"):
        n, e, w = case["T"] * case["H"], _SIZE[case["dtype"]], case["H"] * _SIZE[case["weight"]]
        if op == "norm_backward":
            return {"bytes": n * e * (4 if case["residual"] else 3) + 2 * w, "flops": 12 * n}
        moved = e + (2 * e if case["residual"] else 0) + (e if case["normed"] else 0) + (1 if case["quantize"] else 0)
        scales = 4 * case["T"] * ((case["H"] + 127) // 128) if case["quantize"] else 0
        return {"bytes": n * moved + scales + w, "flops": 8 * n}
    if op in ("route", "route_backward"):
        T, E, k, e = case["T"], case["E"], case["k"], _SIZE[case["dtype"]]
        side = 8 * T * k + 4 * E + (T if case["masked"] and op == "route" else 0)
        return {"bytes": T * E * e * (1 if op == "route" else 2) + side, "flops": 8 * T * E}
    M, N, K, e = case["M"], case["N"], case["K"], _SIZE[case["dtype"]]
    if op == "linear":
        side = (N * e if case["bias"] else 0) + (M * N * e if case["residual"] else 0)
        return {"bytes": (M * K + N * K) * e + M * N * _SIZE[case["out"]] + side, "flops": 2 * M * N * K}
    side = (N * e if case["bias"] else 0) + (M * N * e if case["activation"] else 0)
    return {"bytes": 2 * (M * K + N * K) * e + M * N * e + side, "flops": 4 * M * N * K}


# ------------------------------------------------------------------------------------ 64 bits
def _exact_norm(s):
    h = s["x"].double()
    if s["r"] is not None:
        h = h + s["r"].double()
    y = h / (h.pow(2).sum(1, keepdim=True) / s["H"] + EPS).sqrt() * s["w"].double()
    out = {"h": h if s["r"] is not None else None, "y": y if s["normed"] else None}
    if s["quantize"]:
        scales, codes = [], []
        for c in range(0, s["H"], 128):
            block = y[:, c:c + 128]
            a = block.abs().max(1, keepdim=True).values.clamp(min=1e-12)
            scales.append(a / 448)
            v = block / a * 448
            # e4m3: three bits after the leading one, exponents from -6, ties to the even code
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            codes.append(torch.round(v / step) * step)
        out["q"], out["scale"] = torch.cat(codes, 1), torch.cat(scales, 1)
    return {name: t for name, t in out.items() if t is not None}


def _exact_norm_backward(s):
    h, dy, w, H = s["h"].double(), s["dy"].double(), s["w"].double(), s["H"]
    r = (h.pow(2).sum(1, keepdim=True) / H + EPS).sqrt()
    dx = dy * w / r - h * ((dy * w * h).sum(1, keepdim=True) / H) / r.pow(3)
    if s["dh"] is not None:
        dx += s["dh"].double()
    return {"dx": dx, "dw": torch.einsum("th,th->h", dy, h / r)}


def _exact_scores(s):
    z = s["logits"].double()
    if s["scoring"] == "sigmoid":
        score = torch.sigmoid(z)
        return score, score / score.sum(1, keepdim=True).clamp(min=1e-300)
    p = torch.softmax(z, 1).nan_to_num(0.0)
    return p, p


def _exact_route(s):
    z, k, E = s["logits"].double(), s["k"], s["E"]
    T = z.shape[0]
    live = torch.ones(T, dtype=torch.bool, device=z.device) if s["mask"] is None else s["mask"]
    score, p = _exact_scores(s)
    left, hits, chosen = z.clone(), torch.zeros(E, dtype=torch.float64, device=z.device), []
    rows = torch.arange(T, device=z.device)
    column = torch.arange(E, device=z.device)
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        at = torch.where(left == best, column, E).min(1).values  # the lowest index of the largest
        good = (best[:, 0] > -math.inf) & live
        chosen.append(torch.where(good, score[rows, at], 0.0))
        hits += torch.bincount(at[good], minlength=E)
        left[rows, at] = -math.inf
    w = torch.stack(chosen, 1)
    if s["renormalize"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    out = {"weights": 2.5 * w, "ids": None, "counts": None, "tokens": None}
    if s["balance"]:
        live = live & (z > -math.inf).any(1)
        n = max(1, int(live.sum()))
        out["loss"] = ((hits / n) * p[live].sum(0) / n).sum().mul(E / k).reshape(1)
    return out


def _exact_route_backward(s):
    z, k, E, ids = s["logits"].double(), s["k"], s["E"], s["ids"].long()
    score, p = _exact_scores(s)
    pick = torch.zeros_like(z)
    up = torch.zeros_like(z)  # the gradient of each chosen score's weight, at its expert
    for j in range(k):
        on = ids[:, j] >= 0
        pick[on, ids[on, j]] = 1.0
        up[on, ids[on, j]] = 2.5 * s["gw"][on, j].double()
    if s["renormalize"]:
        total = (pick * score).sum(1, keepdim=True).clamp(min=1e-300)
        up = pick * (up / total - (up * score).sum(1, keepdim=True) / total ** 2)
    load = torch.zeros(E, dtype=torch.float64, device=z.device)
    if s["gl"] is not None:
        load = s["gl"].double() * s["counts"].double() * E / (k * max(1, int(s["tokens"])) ** 2)
    if s["scoring"] == "softmax":
        total = up + load
        d = p * total - p * (p * total).sum(1, keepdim=True)
    else:
        whole = score.sum(1, keepdim=True).clamp(min=1e-300)
        d = (up + load / whole - (load * p).sum(1, keepdim=True) / whole) * score * (1 - score)
    return {"dlogits": d * (ids >= 0).any(1, keepdim=True)}


def _exact_act(z, kind):
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return {"": z, "relu": z.relu(), "silu": z * torch.sigmoid(z)}[kind]


def _exact_linear(s):
    z = torch.matmul(s["x"].double(), s["w"].double().T)
    if s["b"] is not None:
        z += s["b"].double()
    y = _exact_act(z, s["activation"])
    return {"y": y if s["r"] is None else y + s["r"].double()}


def _exact_linear_backward(s):
    dz = s["dy"].double()
    if s["activation"]:
        z = s["z"].double().requires_grad_(True)
        dz, = torch.autograd.grad(_exact_act(z, s["activation"]), z, dz)
    out = {"dx": torch.matmul(dz, s["w"].double()), "dw": torch.matmul(dz.T, s["x"].double())}
    if s["bias"]:
        out["db"] = dz.sum(0)
    return out


_EXACT = {"norm": _exact_norm, "norm_backward": _exact_norm_backward, "route": _exact_route,
          "route_backward": _exact_route_backward, "linear": _exact_linear, "linear_backward": _exact_linear_backward}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
