"""Plain 64-bit forms of the 16-bit linear layer and gated block, each value with a bound on what a correct kernel may be off.

How the bounds come about (u = eps / 2 of the 16-bit type, f = 2^-24):
  * a product accumulated in fp32 over K terms is off by at most 2 (K + 4) f sum |x w| (factor 2: the order and the inner rounding of the
    matrix instruction are not specified);
  * the activations are evaluated in fp32 with one exponential or erf: off by at most 2e-6 (1 + |z|), their slopes by 4e-6 (1 + |z|); an error e
    of z moves them by at most 1.2 e (largest first and second derivative of the six); relu's slope is free where |z| <= e;
  * rounding a value v to the type moves it by at most u |v| (2^-25 more for fp16, whose smallest step is 2^-24).  Where rounded values enter
    another sum their roundings are independent and centred, so (Hoeffding) the sum of e_k a_k stays below 7 sqrt(sum e_k^2 a_k^2) except
    with probability 5e-11 per element, and always below sum e_k |a_k|: the smaller of the two is used.
"""
import math

import torch

F32 = 2.0 ** -24


def act64(name, z):
    """act(z), act'(z)"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.clamp_min(z, 0.0), (z > 0).double()
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


class Val:
    """a value, the bound of its independent centred roundings, the bound of everything else"""

    def __init__(self, v, rnd=None, sys=None):
        self.v = v
        self.rnd = torch.zeros_like(v) if rnd is None else rnd
        self.sys = torch.zeros_like(v) if sys is None else sys

    @property
    def off(self):
        return self.rnd + self.sys


def product(a: Val, b: Val):
    """a @ b with fp32 accumulation; b exact"""
    k = a.v.shape[1]
    m = b.v.abs()
    rnd = torch.minimum(a.rnd @ m, 7 * torch.sqrt(a.rnd.square() @ m.square()))
    return Val(a.v @ b.v, None, rnd + a.sys @ m + 2 * (k + 4) * F32 * ((a.v.abs() + a.off) @ m))


def add(a: Val, b):
    return a if b is None else Val(a.v + b, a.rnd, a.sys + F32 * (a.v + b).abs())


def act(name, z: Val):
    a, s = act64(name, z.v)
    sys = torch.zeros_like(a) if name == "none" else 2e-6 * (1 + z.v.abs())
    slope_sys = torch.zeros_like(a) if name == "none" else 4e-6 * (1 + z.v.abs()) + 1.2 * z.off
    if name == "relu":
        slope_sys = (z.v.abs() <= z.off).double()
    return Val(a, None, sys + 1.2 * z.off), Val(s, None, slope_sys)


def mul(a: Val, b: Val):
    return Val(a.v * b.v, None, a.off * b.v.abs() + b.off * a.v.abs() + a.off * b.off + F32 * (a.v * b.v).abs())


def rounded(a: Val, dtype):
    u, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    return Val(a.v, u * (a.v.abs() + a.off) + tiny, a.off)


def colsum(a: Val):
    rnd = torch.minimum(a.rnd.sum(0), 7 * a.rnd.square().sum(0).sqrt())
    return Val(a.v.sum(0), None, rnd + a.sys.sum(0) + 2 * (a.v.shape[0] + 4) * F32 * a.v.abs().sum(0))


def T(a: Val):
    return Val(a.v.t(), a.rnd.t(), a.sys.t())


def linear_ref(x, w, b, name, r, dy=None):
    dt = x.dtype
    x, w, b, r, dy = (None if t is None else t.detach().double() for t in (x, w, b, r, dy))
    z = add(product(Val(x), Val(w.t())), b)
    a, s = act(name, z)
    out = {"y": rounded(add(a, r), dt)}
    if dy is not None:
        dz = Val(dy) if name == "none" else rounded(mul(Val(dy), s), dt)
        out["dx"] = rounded(product(dz, Val(w)), dt)
        out["dw"] = rounded(product(T(dz), Val(x)), dt)
        out["db"] = rounded(colsum(dz), dt)
    return out


def ffn_ref(x, wg, wu, wd, bg, bu, bd, name, r, dy=None):
    dt = x.dtype
    x, wg, wu, wd, bg, bu, bd, r, dy = (None if t is None else t.detach().double() for t in (x, wg, wu, wd, bg, bu, bd, r, dy))
    g, u = add(product(Val(x), Val(wg.t())), bg), add(product(Val(x), Val(wu.t())), bu)
    a, s = act(name, g)
    h = rounded(mul(a, u), dt)
    out = {"y": rounded(add(add(product(h, Val(wd.t())), bd), r), dt)}
    if dy is not None:
        dh = product(Val(dy), Val(wd))
        dg, du = rounded(mul(mul(dh, u), s), dt), rounded(mul(dh, a), dt)
        p, q = product(dg, Val(wg)), product(du, Val(wu))
        out["dx"] = rounded(Val(p.v + q.v, None, p.off + q.off + 2 * (dg.v.shape[1] + 4) * F32 * (dg.v.abs() @ wg.abs() + du.v.abs() @ wu.abs())), dt)
        out["dwg"], out["dwu"] = rounded(product(T(dg), Val(x)), dt), rounded(product(T(du), Val(x)), dt)
        hd = product(T(h), Val(dy))
        out["dwd"] = rounded(T(hd), dt)
        out["dbg"], out["dbu"], out["dbd"] = rounded(colsum(dg), dt), rounded(colsum(du), dt), rounded(colsum(Val(dy)), dt)
    return out


def check(name, got, ref: Val):
    assert got.shape == ref.v.shape, (name, tuple(got.shape), tuple(ref.v.shape))
    d = (got.detach().double().to(ref.v.device) - ref.v).abs()
    bad = ~(d <= ref.off)
    assert not bad.any(), "%s: %d of %d outside the bound; worst %.3e against %.3e" % (
        name, int(bad.sum()), bad.numel(), float(d[bad].max()), float(ref.off.flatten()[(d / (ref.off + 1e-300)).flatten().argmax()]))
