"""Newton-Schulz orthogonalisation on the GPU against the definition in 64 bits.

Tolerances.  Values are held to 22 bits (half a step: 2^-23) and products drop terms of 2^-22, where fp32 holds 24: a correct kernel is off by at
most 4 times what the same iteration in fp32 is off, plus the rounding of the result, u = eps / 2 of its type.  Independently of any fp32 run:
one step adds at most 16 * 2^-22 |X| (A, B and the two products each 2^-21 of norms up to |b| + |c| <= 7), and what is there is multiplied by
at most 3.9 a step (the largest of |p'(s)| and |p(s) / s| of the polynomial on [0, 1.2]): the sum of those is the second bound."""
import pytest
import torch

from acmil_amd import ops

pytestmark = pytest.mark.gpu
CO = (3.4445, -4.7750, 2.0315)
DTS = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def iterate(g, dtype, steps=5, coeffs=CO, eps=1e-7):
    """the definition in `dtype`, and the second bound of the module's docstring"""
    x = g.to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.double().norm().to(dtype) + eps)
    bound = 0.0
    for a, b, c in ([coeffs] * steps if isinstance(coeffs[0], float) else coeffs):
        p = x @ x.t().contiguous()
        x = a * x + (b * p + c * (p @ p)) @ x
        bound = 3.9 * bound + 16 * 2.0 ** -22 * float(x.double().norm())
    return (x.t() if tall else x), bound


def check(o, g, **kw):
    assert o.shape == g.shape and o.dtype == g.dtype
    want, bound = iterate(g, torch.float64, **kw)
    fp32, _ = iterate(g, torch.float32, **kw)
    off, ref = (o.double() - want).norm(), (fp32.double() - want).norm()
    u = torch.finfo(g.dtype).eps / 2 * want.norm() if g.dtype != torch.float32 else 2.0 ** -24 * want.norm()
    assert off <= 4 * ref + u + 1e-30, (float(off), float(ref), float(u))
    assert off <= bound + u + 1e-30, (float(off), bound)


def gradient(m, n, dt, seed=0, scale=1e-3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = 2 * min(m, n) + 8
    return (torch.randn(r, m, generator=gen, device="cuda").t() @ torch.randn(r, n, generator=gen, device="cuda") * scale).to(dt)


@pytest.mark.parametrize("m, n", [(1, 1), (1, 50), (50, 1), (2, 3), (31, 32), (33, 31), (64, 64), (65, 130), (128, 256), (256, 128), (100, 1000), (777, 129), (512, 512)])
@pytest.mark.parametrize("dt", list(DTS))
def test_sizes(m, n, dt):
    check(ops.orthogonalize(gradient(m, n, DTS[dt], seed=m)), gradient(m, n, DTS[dt], seed=m))


@pytest.mark.parametrize("m, n", [(16, 40), (32, 1152), (32, 1185), (1150, 19), (50, 544), (64, 545), (96, 288), (70, 289), (271, 90), (128, 160), (101, 160), (128, 161), (150, 128)])
@pytest.mark.parametrize("dt", list(DTS))
def test_matrices_that_fit_one_workgroup_and_just_do_not(m, n, dt):
    g = gradient(m, n, DTS[dt], seed=n)
    check(ops.orthogonalize(g), g)
    many = torch.stack([gradient(m, n, DTS[dt], seed=n + k) for k in range(3)])
    got = ops.orthogonalize(many)
    assert torch.equal(got[0], ops.orthogonalize(g)) and torch.equal(got, ops.orthogonalize(many)) and torch.equal(ops.orthogonalize(many, out=many), got)


def test_small_matrices_of_all_shapes_in_one_call():
    shapes = [(1, 7), (200, 30), (64, 64), (128, 160), (96, 3), (33, 400), (90, 90)] * 19                   # more than two launches hold
    gs = [gradient(*s, torch.float32, seed=k % 7) for k, s in enumerate(shapes)]
    wide = torch.full((64, 100), 7.0, device="cuda")
    wide[:, 3:67] = gs[2]
    gs[2] = wide[:, 3:67]                                                                                  # rows on 4 bytes
    outs = ops.orthogonalize(gs)
    for k in list(range(7)) + [58, 59, 60, 61, 119, 120, 132]:
        check(outs[k], gs[k])
        assert torch.equal(outs[k], outs[k % 7])
    check(ops.orthogonalize(gs[3], steps=9, coeffs=(1.5, -0.5, 0.0)), gs[3], steps=9, coeffs=(1.5, -0.5, 0.0))


def test_small_matrices_captured_and_with_bad_values():
    gs = [gradient(20, 70, torch.float32, seed=1), gradient(128, 96, torch.float32, seed=2)]
    ops.orthogonalize(gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.orthogonalize(gs)
    for _ in range(3):
        for g in gs:
            g.normal_()
        want = ops.orthogonalize(gs)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))
    for bad in (float("nan"), float("inf")):
        g = gradient(20, 70, torch.float32, seed=1)
        g[3, 4] = bad
        o = ops.orthogonalize([g, gs[0]])
        assert o[0].isnan().all() and torch.equal(o[1], want[0])                                           # a neighbour of the same launch is not touched
    assert not ops.orthogonalize(torch.zeros(3, 20, 70, device="cuda")).any()
    one = torch.full((1, 1), -3.0, device="cuda")
    want, bound = iterate(one, torch.float64)                                                # a single value: fp32 may be off by next to nothing, by chance
    assert (ops.orthogonalize(one).double() - want).abs() <= bound + 2.0 ** -24              # (the docstring's second bound: 16 * 2^-22 |X| a step, times 3.9)


@pytest.mark.parametrize("m, n", [(1500, 1900), (2900, 2700)])
def test_larger_tiles(m, n):
    g = gradient(m, n, torch.float32)
    check(ops.orthogonalize(g), g)


def test_stacks_lists_and_many_matrices():
    g = torch.stack([gradient(40, 96, torch.float32, seed=k) for k in range(60)])          # more than one group
    o = ops.orthogonalize(g)
    for k in (0, 23, 24, 47, 59):
        check(o[k], g[k])
        assert torch.equal(o[k], ops.orthogonalize(g[k]))                                    # alone: bit for bit the same
    assert torch.equal(ops.orthogonalize(g.view(6, 10, 40, 96)).view(60, 40, 96), o)
    shapes = [(256, 512), (128, 256), (128, 256), (5, 128), (3, 7), (300, 20)]
    gs = [gradient(*s, torch.bfloat16, seed=i) for i, s in enumerate(shapes)]
    for a, b in zip(ops.orthogonalize(gs), gs):
        check(a, b)
    assert ops.orthogonalize([]) == [] and ops.orthogonalize(torch.empty(0, 4, 4, device="cuda")).shape == (0, 4, 4)
    assert ops.orthogonalize(torch.empty(3, 0, device="cuda")).shape == (3, 0)


def test_strides():
    big = gradient(200, 300, torch.float32)
    for g in (big[3:90, 7:150], big[::2, :64], big.t()[:100], big[:, ::3], big[:1].expand(40, 300)):
        check(ops.orthogonalize(g), g)


def test_low_rank_zero_and_scale():
    gen = torch.Generator(device="cuda").manual_seed(1)
    a, b = torch.randn(300, 2, generator=gen, device="cuda"), torch.randn(2, 200, generator=gen, device="cuda")
    g = a @ b
    o = ops.orthogonalize(g)
    check(o, g)
    assert not ops.orthogonalize(torch.zeros(70, 90, device="cuda")).any()
    g = gradient(96, 160, torch.float32, scale=1.0)
    for s in (1e-34, 1e-30, 1e-4, 1e20, 1e30):                                                # squares and reciprocals that leave fp32
        o = ops.orthogonalize(g * s, eps=0.0)
        assert (o - ops.orthogonalize(g, eps=0.0)).norm() <= 1e-4 * o.norm(), s              # scaling rounds every value by 2^-24, times at most 3.9^5
    g[3, 4] = float("inf")
    assert ops.orthogonalize(g).isnan().any()


def test_coefficients_and_steps():
    g = gradient(120, 200, torch.float32)
    check(ops.orthogonalize(g, steps=1), g, steps=1)
    cubic = (1.5, -0.5, 0.0)
    check(ops.orthogonalize(g, steps=14, coeffs=cubic), g, steps=14, coeffs=cubic)
    table = [(3.4445, -4.7750, 2.0315)] * 4 + [(1.875, -1.25, 0.375)] * 3
    o = ops.orthogonalize(g, steps=7, coeffs=table)
    check(o, g, steps=7, coeffs=table)
    s = torch.linalg.svdvals(o.cpu().double())
    assert (s > 0.9).all() and (s < 1.1).all()


def test_stream_graph_and_repeatability():
    gs = [gradient(130, 260, torch.float32, seed=3), gradient(64, 64, torch.float32, seed=4), gradient(500, 300, torch.float32, seed=5)]
    eager = ops.orthogonalize(gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.orthogonalize(gs)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.orthogonalize(gs)
    for _ in range(3):
        for g in gs:
            g.normal_()
        want = ops.orthogonalize(gs)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_outputs_given_by_the_caller():
    gs = [gradient(40, 64, torch.float32, seed=k) for k in range(30)]                        # two groups: the second is read when the first is written
    want = ops.orthogonalize(gs)
    outs = [torch.full((40, 64), 7.0, device="cuda") for _ in gs]
    assert ops.orthogonalize(gs, out=outs)[3] is outs[3] and all(torch.equal(a, b) for a, b in zip(want, outs))
    wide = torch.full((40, 80), 7.0, device="cuda")                                          # between rows that are not its own nothing is written
    wide[:, 8:72] = gs[0]
    assert torch.equal(ops.orthogonalize(wide[:, 8:72], out=outs[0]), want[0]) and (wide[:, :8] == 7).all() and (wide[:, 72:] == 7).all()
    buf = torch.stack(gs)
    for out in (torch.empty(30, 64, 40, device="cuda"), torch.empty(30, 64, 40, device="cuda").transpose(1, 2), outs[0], torch.empty_like(buf).half()):
        with pytest.raises(RuntimeError, match="structure"):
            ops.orthogonalize(buf, out=out)
    for a, out in ((gs, gs[1:] + gs[:1]), (gs, [outs[0]] * 30), ([buf[0], buf[1]], [buf.view(-1)[640:3200].view(40, 64), outs[1]]),
                   (wide[:, 8:72], wide.view(-1)[:2560].view(40, 64))):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.orthogonalize(a, out=out)
    assert ops.orthogonalize([gs[0], gs[0]])[1].equal(want[0])                               # read twice: allowed
    ops.orthogonalize(buf, out=buf), ops.orthogonalize(gs, out=gs)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, gs, buf))


def test_refusals():
    g = gradient(8, 8, torch.float32)
    for call in (lambda: ops.orthogonalize(g.double()), lambda: ops.orthogonalize(g[0]), lambda: ops.orthogonalize([g, g.half()]),
                 lambda: ops.orthogonalize([g[None]]), lambda: ops.orthogonalize(g, coeffs=(5.0, 0.0, 0.0)), lambda: ops.orthogonalize(g, eps=-1.0)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: ops.orthogonalize(g, steps=0), lambda: ops.orthogonalize(g, steps=2, coeffs=[CO])):
        with pytest.raises(ValueError):
            call()
