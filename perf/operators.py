"""Workloads of the 16-bit linear layer with a fused epilogue, the gated feed-forward block and the Newton-Schulz
orthogonalisation: their inputs, their plain forms in elementary torch operations, and the calls that a user makes of
acmil_amd.  `own` selects the calls; `exact` gives the same values from the definitions in 64 bits.

  linear   y = act(x W^T + b) + r;  training: also dx, dW, db, dr for an incoming dy
  ffn      y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + r;  training: also every gradient
  ortho    X = G / (|G|_F + eps); five times  A = X X^T, X <- a X + (b A + c A A) X   (on G^T where G is tall)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
STEPS = 5


# ------------------------------------------------------------------------------------------------ cases
def _linear(name, M, K, N, dtype, act, bias, residual, train):
    c = {"op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "train": train}
    return dict(c, name=name) if name else c


def _ffn(name, M, D, F, dtype, act, bias, residual, train):
    c = {"op": "ffn", "M": M, "D": D, "F": F, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "train": train}
    return dict(c, name=name) if name else c


def _ortho(name, m, n, count, group, dtype):
    c = {"op": "ortho", "m": m, "n": n, "count": count, "group": group, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a served model: latency and the weight's bytes
        _linear("linear one row", 1, 4096, 4096, "bf16", "gelu_tanh", True, True, False),
        # feature projection of a 50 000-patch bag that is stored in fp16 (1536 -> 768), inference
        _linear("linear bag projection", 50000, 1536, 768, "fp16", "relu", False, False, False),
        # a residual block on a bag of 10 007 patches at width 768, training; rows fill no tile
        _linear("linear residual block train", 10007, 768, 768, "fp16", "relu", False, True, True),
        # an ordinary wide layer, training
        _linear("linear wide train", 8192, 4096, 4096, "bf16", "gelu", True, True, True),
        # one token through a small block
        _ffn("ffn one row", 1, 2048, 5632, "bf16", "silu", False, True, False),
        # a small batch of served sequences, one token each
        _ffn("ffn 24 rows", 24, 4096, 11008, "bf16", "silu", False, True, False),
        # rows, width and hidden width that no tile divides, with biases, training
        _ffn("ffn odd train", 777, 1000, 2731, "fp16", "gelu", True, True, True),
        # a training step's block
        _ffn("ffn wide train", 8192, 4096, 11008, "bf16", "silu", False, True, True),
        # the matrices of the gated-attention aggregator (projection, both attention branches) in one optimizer step
        _ortho("ortho aggregator", 256, 512, 3, "trunk", "fp32"),
        # the two to_qkv matrices of the Nystrom model
        _ortho("ortho two qkv", 1536, 512, 2, "stack", "fp32"),
        # an odd tall matrix
        _ortho("ortho odd tall", 2731, 1000, 1, "stack", "fp16"),
        # a wide layer's matrix
        _ortho("ortho wide layer", 4096, 4096, 1, "stack", "bf16"),
    ]


def _size(rng, lo, hi, even=0.5):
    """A size spread over its logarithm; half of them a multiple of 64 where that fits, the others as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < even and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("linear", "ffn", "ortho"))
    if op == "ortho":
        group = rng.choice(("stack", "stack", "trunk"))
        top = 4096 if group == "stack" else 2048
        m, n = _size(rng, 16, top), _size(rng, 16, top)
        count = 3 if group == "trunk" else rng.choice((1, 1, 2, 4, 7)) if max(m, n) <= 1536 else 1
        return _ortho(None, m, n, count, group, rng.choice(("fp32", "fp32", "bf16", "fp16")))
    train = rng.random() < 0.5
    M = _size(rng, 1, 8192, 0.3)
    dtype, act = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("silu", "gelu", "gelu_tanh", "relu", "sigmoid", "none"))
    bias, residual = rng.random() < 0.5, rng.random() < 0.5
    if op == "linear":
        return _linear(None, M, _size(rng, 32, 4096), _size(rng, 32, 4096), dtype, act, bias, residual, train)
    return _ffn(None, M, _size(rng, 32, 4096), _size(rng, 32, 11008), dtype, act, bias, residual, train)


def _shapes(case):
    """The matrices of one orthogonalisation call."""
    m, n = case["m"], case["n"]
    if case["group"] == "trunk":
        return [(m, n), (max(1, m // 2), m), (max(1, m // 2), m)]
    return [(m, n)] * case["count"]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dt)

    if case["op"] == "ortho":
        grads = []
        for m, n in _shapes(case):
            # a weight gradient: the product of an upstream gradient and features whose scales fall off
            rows = 2 * min(m, n) + 16
            up = torch.randn(rows, m, generator=gen, device="cuda") * 1e-3
            feat = torch.randn(rows, n, generator=gen, device="cuda") * torch.arange(1, n + 1, device="cuda").float().rsqrt()
            grads.append((up.t() @ feat).to(dt))
        return {"case": case, "g": grads if case["group"] == "trunk" else torch.stack(grads) if len(grads) > 1 else grads[0]}

    M = case["M"]
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        s = {"x": normal(M, K), "w": normal(N, K, scale=K ** -0.5), "b": normal(N, scale=0.5) if case["bias"] else None,
             "r": normal(M, N) if case["residual"] else None, "dy": normal(M, N) if case["train"] else None}
        leaves = ("x", "w", "b", "r")
    else:
        D, F = case["D"], case["F"]
        s = {"x": normal(M, D), "wg": normal(F, D, scale=D ** -0.5), "wu": normal(F, D, scale=D ** -0.5),
             "wd": normal(D, F, scale=F ** -0.5), "r": normal(M, D) if case["residual"] else None,
             "dy": normal(M, D) if case["train"] else None}
        s.update({"bg": normal(F, scale=0.3), "bu": normal(F, scale=0.3), "bd": normal(D, scale=0.3)} if case["bias"]
                 else {"bg": None, "bu": None, "bd": None})
        leaves = ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r")
    if case["train"]:
        for k in leaves:
            if s[k] is not None:
                s[k].requires_grad_(True)
    s["leaves"] = [k for k in leaves if s[k] is not None]
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _act(name, z):
    """act(z) and act'(z)"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if name == "sigmoid":
        s = _sigmoid(z)
        return s, s * (1.0 - s)
    if name == "silu":
        s = _sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    k = math.sqrt(2.0 / math.pi)                       # gelu_tanh: 0.5 z (1 + tanh(t)) = z sigmoid(2 t)
    s = _sigmoid(2.0 * k * (z + 0.044715 * z * z * z))
    return z * s, s + z * s * (1.0 - s) * 2.0 * k * (1.0 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y, slope = _act(case["act"], z)
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dz = dy * slope
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(dt)
        if s["r"] is not None:
            out["dr"] = dy.to(dt)
    return out


def _plain_ffn(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["bg"].detach().float(), u + s["bu"].detach().float()
    a, slope = _act(case["act"], g)
    h = a * u
    y = h @ wd.t()
    if case["bias"]:
        y = y + s["bd"].detach().float()
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"], out["dwu"], out["dwd"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)
        if case["bias"]:
            out["dbg"], out["dbu"], out["dbd"] = dg.sum(0).to(dt), du.sum(0).to(dt), dy.sum(0).to(dt)
        if s["r"] is not None:
            out["dr"] = dy.to(dt)
    return out


def _plain_ortho(g):
    a, b, c = COEFFS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        p = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * p + c * (p @ p)) @ x
    if tall:
        x = x.transpose(-2, -1).contiguous()
    return x.to(g.dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_linear(s):
    from acmil_amd import autograd, ops
    case = s["case"]
    if not case["train"]:
        return {"y": ops.linear_act(s["x"], s["w"], bias=s["b"], act=case["act"], residual=s["r"])}
    y = autograd.linear_act(s["x"], s["w"], bias=s["b"], act=case["act"], residual=s["r"])
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
    return dict({"d" + k: t for k, t in zip(s["leaves"], grads)}, y=y.detach())


def _own_ffn(s):
    from acmil_amd import autograd, ops
    case = s["case"]
    call = autograd.gated_ffn if case["train"] else ops.gated_ffn
    y = call(s["x"], s["wg"], s["wu"], s["wd"], b_gate=s["bg"], b_up=s["bu"], b_down=s["bd"], act=case["act"], residual=s["r"])
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
    return dict({"d" + k: t for k, t in zip(s["leaves"], grads)}, y=y.detach())


def run(state):
    op = state["case"]["op"]
    if op == "ortho":
        if own:
            from acmil_amd import ops
            return {"o": ops.orthogonalize(state["g"], steps=STEPS, coeffs=COEFFS, eps=EPS)}
        g = state["g"]
        return {"o": [_plain_ortho(t) for t in g] if isinstance(g, list) else _plain_ortho(g)}
    if op == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    return _own_ffn(state) if own else _plain_ffn(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "ortho":
        nbytes = flops = 0
        for m, n in _shapes(case):
            s, t = min(m, n), max(m, n)
            nbytes += 2 * e * m * n
            flops += STEPS * (3 * s * s * t + s * s * s)       # both symmetric products count for half
        return {"bytes": nbytes, "flops": flops}
    M, bias, res = case["M"], int(case["bias"]), int(case["residual"])
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        fwd = M * K + N * K + N * bias + M * N * (1 + res)
        back = M * N + M * K + N * K + N * bias + M * N * res
        return {"bytes": e * (fwd + (back if case["train"] else 0)), "flops": 2 * M * K * N * (3 if case["train"] else 1)}
    D, F = case["D"], case["F"]
    fwd = M * D + 3 * D * F + (2 * F + D) * bias + M * D * (1 + res)
    back = 2 * M * D + 3 * D * F + (2 * F + D) * bias + M * D * res
    return {"bytes": e * (fwd + (back if case["train"] else 0)), "flops": 6 * M * D * F * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _act64(name, z):
    if name == "relu":
        return torch.clamp_min(z, 0.0)
    if name == "sigmoid":
        return 0.5 * (1.0 + torch.tanh(0.5 * z))
    if name == "silu":
        return 0.5 * z * (1.0 + torch.tanh(0.5 * z))
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ortho":
        def one(g):
            x = g.double()
            turn = x.shape[0] > x.shape[1]
            x = x.t().contiguous() if turn else x
            x = x / (torch.linalg.norm(x) + EPS)
            for _ in range(STEPS):
                gram = torch.mm(x, x.t())
                y = torch.mm(gram, x)
                x = COEFFS[0] * x + COEFFS[1] * y + COEFFS[2] * torch.mm(gram, y)
            return x.t().contiguous() if turn else x
        g = s["g"]
        return {"o": [one(t) for t in g] if isinstance(g, list) else torch.stack([one(t) for t in g]) if g.dim() == 3 else one(g)}
    d = {k: s[k].detach().double().requires_grad_(case["train"]) for k in s["leaves"]}
    F = torch.nn.functional
    if case["op"] == "linear":
        y = _act64(case["act"], F.linear(d["x"], d["w"], d.get("b")))
    else:
        h = _act64(case["act"], F.linear(d["x"], d["wg"], d.get("bg"))) * F.linear(d["x"], d["wu"], d.get("bu"))
        y = F.linear(h, d["wd"], d.get("bd"))
    if "r" in d:
        y = y + d["r"]
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [d[k] for k in s["leaves"]], s["dy"].double())
    return dict({"d" + k: t for k, t in zip(s["leaves"], grads)}, y=y.detach())
