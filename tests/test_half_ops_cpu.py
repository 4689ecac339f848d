"""16-bit linear layer, gated block: what they refuse, on the CPU (nothing reaches a kernel), and the reference's own gradients."""
import ctypes

import numpy as np
import pytest
import torch

import half_reference as R
from acmil_amd import _lib, autograd, ops


def test_cpu_tensors_and_other_types_are_refused():
    x, w = torch.zeros(4, 16, dtype=torch.float16), torch.zeros(8, 16, dtype=torch.float16)
    for call in (lambda: ops.linear_act(x, w), lambda: autograd.linear_act(x, w), lambda: ops.gated_ffn(x, w, w, w.t()),
                 lambda: autograd.gated_ffn(x, w, w, w.t())):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("change, code", [
    ({}, -3), ({"dtype": 0}, -2), ({"dtype": 7}, -2), ({"act": 9}, -1), ({"M": 0}, -1), ({"K": 0}, -1), ({"N": -1}, -1), ({"K": (1 << 22) + 1}, -1),
    ({"M": (1 << 30) + 1}, -1), ({"M": 1 << 30, "N": 1 << 12}, -1),
    ({"x": 4096, "W": 4096, "ldx": 15, "ldw": 16}, -1), ({"x": 4096, "W": 4096, "ldx": 16, "ldw": 1 << 23}, -1), ({"x": 4096, "W": 4096, "ldx": 16, "ldw": 16}, -3),
    ({"x": 4096, "W": 4096, "ldx": 16, "ldw": 16, "y": 4096, "ldy": 7}, -1),
    ({"x": 4096, "W": 4096, "ldx": 16, "ldw": 16, "y": 4096, "ldy": 8, "pre": 4100}, -1),
    ({"x": 4096, "W": 4096, "ldx": 16, "ldw": 16, "y": 4096, "ldy": 8, "res": 4096, "ldr": 3}, -1)])
def test_linear_entry_refuses(change, code):
    """error codes before anything is launched; the workspace query answers 0 for the same block"""
    lib = _lib.load()
    a = _lib.LinearArgs(**{**dict(dtype=1, act=0, M=4, K=16, N=8), **change})
    assert lib.acmil_linear_act(ctypes.byref(a), None, 0, None) == code
    assert lib.acmil_linear_act_workspace_bytes(ctypes.byref(a)) == 0


def test_entries_refuse_missing_pieces():
    lib = _lib.load()
    good = dict(dtype=2, act=2, M=40, K=4096, N=8, x=4096, W=4096, ldx=4096, ldw=4096, y=4096, ldy=8)      # (K is split: needs a workspace)
    a = _lib.LinearArgs(**good)
    need = lib.acmil_linear_act_workspace_bytes(ctypes.byref(a))
    assert need > 256
    assert lib.acmil_linear_act(ctypes.byref(a), None, need, None) == -3                 # no workspace
    assert lib.acmil_linear_act(ctypes.byref(a), 4097, need, None) == -1                 # not on 256 bytes
    assert lib.acmil_linear_act(ctypes.byref(a), 4096, need - 1, None) == -1             # too small
    assert lib.acmil_linear_act(None, 4096, need, None) == -3
    assert lib.acmil_linear_act_bwd(ctypes.byref(a), 4096, 1 << 30, None) == -3          # no dy
    b = _lib.LinearArgs(**good, dy=4096, lddy=8)
    assert lib.acmil_linear_act_bwd(ctypes.byref(b), 4096, 1 << 30, None) == -3          # an activation, but no pre
    f = dict(dtype=1, act=2, M=40, D=16, F=24, x=4096, ldx=16, Wg=4096, ldwg=16, Wu=4096, ldwu=16, Wd=4096, ldwd=24, y=4096, ldy=16)
    assert lib.acmil_gated_ffn_workspace_bytes(ctypes.byref(_lib.FfnArgs(**f))) > 0
    for change, code in (({"Wu": None}, -3), ({"ldwd": 23}, -1), ({"g": 4096}, -3), ({"g": 4096, "u": 4096, "h": 4098}, -1), ({"y": None}, -3),
                         ({"F": (1 << 21) + 1, "ldwd": 1 << 22}, -1), ({"act": -1}, -1), ({"dtype": 0}, -2)):
        a = _lib.FfnArgs(**{**f, **change})
        assert lib.acmil_gated_ffn(ctypes.byref(a), 4096, 1 << 30, None) == code, change
    a = _lib.FfnArgs(**f, dy=4096, lddy=16)
    assert lib.acmil_gated_ffn_bwd(ctypes.byref(a), 4096, 1 << 30, None) == -3           # nothing kept by the forward


def test_workspace_grows_only_with_copies_and_splits():
    """rows that lie on 16 bytes need no copy; a shifted base address or an odd length does"""
    lib = _lib.load()
    base = dict(dtype=1, act=0, M=4096, K=1024, N=4096, ldx=1024, ldw=1024, y=4096, ldy=4096, W=1 << 20)
    assert lib.acmil_linear_act_workspace_bytes(ctypes.byref(_lib.LinearArgs(**base, x=1 << 20))) <= 512
    assert lib.acmil_linear_act_workspace_bytes(ctypes.byref(_lib.LinearArgs(**base, x=(1 << 20) + 2))) >= 4096 * 1024 * 2
    assert lib.acmil_linear_act_workspace_bytes(ctypes.byref(_lib.LinearArgs(**{**base, "M": 32}, x=(1 << 20) + 2))) <= 512


@pytest.mark.parametrize("act", list(_lib.ACTS))
def test_reference_gradients_are_those_of_differences(act):
    """the 64-bit reference the GPU tests trust: its gradients against central differences and autograd"""
    g = torch.Generator().manual_seed(3)
    x, w, b, r, dy = (torch.randn(*s, generator=g) for s in ((5, 6), (7, 6), (7,), (5, 7), (5, 7)))
    x, w, b, r, dy = (t.to(torch.bfloat16) for t in (x, w, b, r, dy))
    ref = R.linear_ref(x, w, b, act, r, dy)
    h = 1e-6
    for name, t, d in (("dx", x, 0), ("dw", w, 1), ("db", b, 2)):
        args = [x.double(), w.double(), b.double()]
        num = torch.zeros(t.shape, dtype=torch.float64)
        for i in range(t.numel()):
            hi, lo = [a.clone() for a in args], [a.clone() for a in args]
            hi[d].view(-1)[i] += h
            lo[d].view(-1)[i] -= h
            f = lambda a: (R.act64(act, a[0] @ a[1].t() + a[2])[0] * dy.double()).sum()
            num.view(-1)[i] = (f(hi) - f(lo)) / (2 * h)
        assert (ref[name].v - num).abs().max() < 1e-7 * (1 + num.abs().max())
    xs = [t.double().requires_grad_() for t in (x, w, w * 0.5, w.t().contiguous())]
    a, _ = R.act64(act, xs[0] @ xs[1].t())
    y = (a * (xs[0] @ xs[2].t())) @ xs[3].t()
    grads = torch.autograd.grad(y, xs, x.double())
    ref = R.ffn_ref(x, w, w * 0.5, w.t().contiguous(), None, None, None, act, None, x)
    for k, t in zip(("dx", "dwg", "dwu", "dwd"), grads):
        assert (ref[k].v - t).abs().max() < 1e-9 * (1 + t.abs().max()), k


def test_orthogonalize_entry_refuses():
    lib = _lib.load()
    co = (ctypes.c_float * 15)(*([3.4445, -4.7750, 2.0315] * 5))

    def call(m=8, n=16, ldg=16, ldo=16, dtype=0, steps=5, eps=1e-7, g=4096, o=4096, ws=4096, size=1 << 30, count=1, co=co):
        mats = (_lib.OrthoMat * 1)(_lib.OrthoMat(g, ldg, o, ldo, m, n))
        return lib.acmil_orthogonalize(count, mats, dtype, steps, co, eps, ws, size, None)

    for kw, code in ((dict(m=0), -1), (dict(n=65537, ldg=1 << 17, ldo=1 << 17), -1), (dict(ldg=15), -1), (dict(ldo=15), -1), (dict(dtype=5), -2), (dict(steps=0), -1),
                     (dict(steps=65), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(g=None), -3), (dict(o=None), -3), (dict(ws=None), -3),
                     (dict(ws=4100), -1), (dict(size=100), -1), (dict(count=0), -1), (dict(co=None), -3),
                     (dict(co=(ctypes.c_float * 15)(*([6.0, 0.0, 0.0] * 5))), -1), (dict(co=(ctypes.c_float * 15)(*([float("nan")] * 15))), -1)):
        assert call(**kw) == code, kw
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.orthogonalize(torch.zeros(4, 4))


def test_muon_entries_and_trainer_option_refuse():
    from acmil_amd import train as T
    lib = _lib.load()
    seg = (_lib.MuonSeg * 2)(_lib.MuonSeg(0, 10, 1.0), _lib.MuonSeg(10, 0, 1.0))
    assert lib.acmil_muon_momentum(2, seg, 4096, 4096, 4096, 0.9, 1, None, None, None) == -1          # an empty segment
    assert lib.acmil_muon_momentum(1, seg, 4096, 4096, None, 0.9, 1, None, None, None) == -3
    assert lib.acmil_muon_momentum(1, seg, 4096, 4096, 4096, 1.0, 1, None, None, None) == -1
    assert lib.acmil_muon_momentum(0, seg, 4096, 4096, 4096, 0.9, 1, None, None, None) == -1
    assert lib.acmil_muon_apply(1, None, 4096, 4096, 0.1, 0.0, None, None) == -3
    assert lib.acmil_muon_apply(1, seg, None, 4096, 0.1, 0.0, None, None) == -3
    with pytest.raises(RuntimeError, match="needs the GPU"):
        T.make_optimizer(torch.nn.Linear(64, 64), T.Struct(wd=0.0, optimizer="muon"), torch.device("cpu"))
    with pytest.raises(SystemExit):
        T.get_arguments(["--optimizer", "sgd"])


def _largest(a, b, c, u):
    """the largest |a s + b s^3 + c s^5| and |b s^2 + c s^4| on [0, u], from the roots of their derivatives in 64 bits"""
    def peak(p):
        s = [0.0, u] + [r.real for r in p.deriv().roots() if abs(r.imag) < 1e-12 and 0 <= r.real <= u]
        return max(abs(p(v)) for v in s)
    P = np.polynomial.Polynomial
    return peak(P([0, a, 0, b, 0, c])), peak(P([0, 0, b, 0, c]))


def test_orthogonalize_coefficients_at_their_limits():
    """Tables are accepted exactly where the polynomials stay below 3.9 and 15.5.  No workspace is given: an accepted table is refused behind the
    check (NULL), a refused one by it (SHAPE).  Two tables have a peak beyond the limit between two of 2049 even samples of [0, 1], which stay below."""
    lib = _lib.load()
    mats = (_lib.OrthoMat * 1)(_lib.OrthoMat(4096, 16, 4096, 16, 8, 16))

    def accepted(*table):
        co = (ctypes.c_float * len(table))(*table)
        rc = lib.acmil_orthogonalize(1, mats, 0, len(table) // 3, co, 1e-7, None, 0, None)
        assert rc in (-1, -3)
        return rc == -3

    for between in ((13.233685493469238, -46.426395416259766, 34.76467514038086), (9.997149467468262, -48.42892837524414, 39.40630340576172)):
        up, bp = _largest(*between, 1.0)
        s = np.arange(2049) / 2048.0
        a, b, c = between
        assert (up > 3.9 or bp > 15.5) and np.abs(a * s + b * s ** 3 + c * s ** 5).max() < 3.9 and np.abs(b * s ** 2 + c * s ** 4).max() < 15.5
        assert not accepted(*between)
        assert accepted(*(v * (1 - 1e-5) for v in between))
    assert accepted(*(ops.NS_COEFFS * 64)) and accepted(1.5, -0.5, 0.0) and accepted(0.0, 0.0, 0.0) and accepted(3.8999, 0.0, 0.0)
    assert not accepted(3.9001, 0.0, 0.0) and not accepted(0.0, 0.0, 3.9001) and not accepted(float("inf"), 0.0, 0.0)
    assert not accepted(2.0, 0.0, 0.0, 2.0, 0.0, 0.0) and accepted(2.0, 0.0, 0.0, 1.9, 0.0, 0.0)          # the second step starts where the first ends
    rng = np.random.default_rng(0)
    seen = [0, 0]
    for _ in range(3000):
        table = np.float32(rng.normal(size=3) * rng.choice([1.0, 4.0, 16.0], 3) * (rng.random(3) < 0.9))
        table = np.concatenate([table, np.float32(rng.normal(size=3))])
        u, ok, near = 1.0, True, False
        for k in (0, 3):
            up, bp = _largest(*(float(v) for v in table[k:k + 3]), u)
            near |= abs(up - 3.9) < 1e-6 or abs(bp - 15.5) < 1e-6
            ok &= up <= 3.9 and bp <= 15.5
            u = up
        if not near:
            assert accepted(*(float(v) for v in table)) == ok, table
            seen[int(ok)] += 1
    assert min(seen) > 300


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """no_grad does not switch forward mode off: a dual tensor in any place raises, and none is left unnoticed; without one the call goes on (to the
    refusal of CPU tensors)"""
    dt = torch.float16
    lin = dict(x=torch.zeros(4, 16, dtype=dt), weight=torch.zeros(16, 16, dtype=dt), bias=torch.zeros(16, dtype=dt), residual=torch.zeros(4, 16, dtype=dt))
    ffn = dict(x=torch.zeros(4, 16, dtype=dt), w_gate=torch.zeros(16, 16, dtype=dt), w_up=torch.zeros(16, 16, dtype=dt), w_down=torch.zeros(16, 16, dtype=dt),
               b_gate=torch.zeros(16, dtype=dt), b_up=torch.zeros(16, dtype=dt), b_down=torch.zeros(16, dtype=dt), residual=torch.zeros(4, 16, dtype=dt))
    with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
        for call, args in ((autograd.linear_act, lin), (autograd.gated_ffn, ffn)):
            for k, v in args.items():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(**{**args, k: torch.autograd.forward_ad.make_dual(v, torch.ones_like(v))})
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call(**args)
