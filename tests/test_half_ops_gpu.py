"""16-bit linear layer with a fused epilogue and gated feed-forward block on the GPU, against the 64-bit reference with its bounds."""
import pytest
import torch

import half_reference as R
from acmil_amd import _lib, autograd, ops

pytestmark = pytest.mark.gpu
DTS = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = list(_lib.ACTS)


def rand(gen, dt, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)


def make_linear(M, K, N, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return rand(g, dt, M, K), rand(g, dt, N, K, scale=K ** -0.5), rand(g, dt, N), rand(g, dt, M, N), rand(g, dt, M, N)


def run_linear(x, w, b, act, r, dy):
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = autograd.linear_act(x, w, bias=b, act=act, residual=r)
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db", "dr"), (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    return dict(grads, y=y)


def check_linear(x, w, b, act, r, dy):
    out = run_linear(x, w, b, act, r, dy)
    ref = R.linear_ref(x, w, b, act, r, dy)
    for k, v in out.items():
        if k == "dr":
            assert torch.equal(v, dy)
        else:
            R.check(k, v, ref[k])
    assert torch.equal(ops.linear_act(x.detach(), w.detach(), bias=b, act=act, residual=r), out["y"])


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 64, 5), (2, 7, 3), (5, 9, 17), (16, 63, 40), (17, 65, 33), (31, 130, 127), (32, 256, 128), (33, 64, 8), (33, 1, 1),
          (64, 8, 129), (100, 130, 300), (128, 64, 128), (129, 192, 257), (257, 100, 70)]


@pytest.mark.parametrize("M, K, N", SHAPES)
@pytest.mark.parametrize("dt", list(DTS))
def test_linear_sizes(M, K, N, dt):
    x, w, b, r, dy = make_linear(M, K, N, DTS[dt], seed=M + K)
    check_linear(x, w, b, ACTS[(M + N) % len(ACTS)], r, dy)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias, residual", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("M", [3, 70])
def test_linear_epilogues(act, bias, residual, M):
    x, w, b, r, dy = make_linear(M, 72, 50, torch.float16, seed=7)
    check_linear(x * 3, w, b if bias else None, act, r if residual else None, dy)


@pytest.mark.parametrize("M, K, N", [(2500, 200, 4200), (100, 4096, 256), (70, 1000, 2050), (4200, 2500, 24), (3000, 40, 3333)])
@pytest.mark.parametrize("dt", list(DTS))
def test_linear_large_tiles_and_split_products(M, K, N, dt):
    """products of each tile size and with K split (forward, input and weight gradient take different ones)"""
    x, w, b, r, dy = make_linear(M, K, N, DTS[dt], seed=K)
    check_linear(x, w, b, "silu", r, dy)


@pytest.mark.parametrize("M, K, N", [(5000, 200, 3500), (4000, 72, 5001), (17000, 136, 1000), (300, 1000, 20000), (5000, 3500, 200)])
@pytest.mark.parametrize("dt", list(DTS))
def test_linear_rows_in_two_launches(M, K, N, dt):
    """more large tiles than CUs, and a last round that is better a product of its own: forward, dx and dW"""
    x, w, b, r, dy = make_linear(M, K, N, DTS[dt], seed=N)
    check_linear(x, w, b, "silu", r, dy)
    check_linear(x.detach(), w.detach(), None, "none", None, dy)


@pytest.mark.parametrize("M, D, F", [(5000, 200, 1700), (2600, 3300, 250)])
def test_ffn_rows_in_two_launches(M, D, F):
    check_ffn(make_ffn(M, D, F, torch.bfloat16, seed=2), "silu", bias=False)


@pytest.mark.parametrize("M, K, N", [(5, 8200, 4100), (20, 4096, 8201), (32, 4104, 8208), (33, 8200, 4104), (64, 4096, 8200)])
@pytest.mark.parametrize("dt", list(DTS))
def test_few_rows_by_streamed_weights(M, K, N, dt):
    """weights of 64 MB and more under 5 to 64 rows have tiles of their own (forward and input gradient)"""
    x, w, b, r, dy = make_linear(M, K, N, DTS[dt], seed=M)
    check_linear(x, w, b, "gelu_tanh", r, dy)


@pytest.mark.parametrize("M", [24, 50])
def test_ffn_few_rows_by_streamed_weights(M):
    check_ffn(make_ffn(M, 4096, 8200, torch.bfloat16, seed=M), "silu")


@pytest.mark.parametrize("M", [9, 90])
def test_linear_strides(M):
    """row strides, shifted bases, transposed weights, expanded rows, leading dimensions, strided bias and residual"""
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(5)
    big = rand(g, dt, M, 200)
    w, b, r, dy = rand(g, dt, 48, 96, scale=0.1), rand(g, dt, 48), rand(g, dt, M, 48), rand(g, dt, M, 48)
    for x in (big[:, 8:104], big[:, 1:97], big[:, ::2][:, :96], big[:1, :96].expand(M, 96)):
        check_linear(x, w, b, "gelu", r, dy)
    x = big[:, :96].contiguous()
    check_linear(x, rand(g, dt, 96, 48, scale=0.1).t(), rand(g, dt, 96)[::2], "silu", rand(g, dt, 48, M).t(), rand(g, dt, 1, 1).expand(M, 48))
    check_linear(x, rand(g, dt, 60, 200, scale=0.1)[4:52, 3:99], b, "relu", rand(g, dt, 1, 48).expand(M, 48), dy)
    y = ops.linear_act(x.view(3, M // 3, 96), w, bias=b, act="silu", residual=r.view(3, M // 3, 48))
    assert y.shape == (3, M // 3, 48) and torch.equal(y.view(M, 48), ops.linear_act(x, w, bias=b, act="silu", residual=r))
    assert torch.equal(ops.linear_act(x[0], w), ops.linear_act(x[:1], w)[0])


def make_ffn(M, D, F, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"x": rand(g, dt, M, D), "wg": rand(g, dt, F, D, scale=D ** -0.5), "wu": rand(g, dt, F, D, scale=D ** -0.5), "wd": rand(g, dt, D, F, scale=F ** -0.5),
            "bg": rand(g, dt, F, scale=0.3), "bu": rand(g, dt, F, scale=0.3), "bd": rand(g, dt, D, scale=0.3), "r": rand(g, dt, M, D), "dy": rand(g, dt, M, D)}


def check_ffn(t, act, bias=True, residual=True):
    t = {k: v.detach() for k, v in t.items()}
    for k in ("bg", "bu", "bd") * (not bias) + ("r",) * (not residual):
        t[k] = None
    names = [k for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r") if t[k] is not None]
    for k in names:
        t[k].requires_grad_(True)
    y = autograd.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], b_gate=t["bg"], b_up=t["bu"], b_down=t["bd"], act=act, residual=t["r"])
    out = dict(zip(["d" + k for k in names], torch.autograd.grad(y, [t[k] for k in names], t["dy"])), y=y)
    ref = R.ffn_ref(*(t[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd")), act, t["r"], t["dy"])
    for k, v in out.items():
        if k == "dr":
            assert torch.equal(v, t["dy"])
        else:
            R.check(k, v, ref[k])
    plain = {k: (None if v is None else v.detach()) for k, v in t.items()}
    assert torch.equal(ops.gated_ffn(plain["x"], plain["wg"], plain["wu"], plain["wd"], b_gate=plain["bg"], b_up=plain["bu"], b_down=plain["bd"], act=act,
                                     residual=plain["r"]), y)


@pytest.mark.parametrize("M, D, F", [(1, 1, 1), (1, 64, 40), (2, 9, 7), (16, 33, 65), (20, 128, 100), (32, 40, 129), (33, 64, 64), (40, 9, 7), (100, 72, 200),
                                     (129, 130, 131), (300, 64, 257)])
@pytest.mark.parametrize("dt", list(DTS))
def test_ffn_sizes(M, D, F, dt):
    check_ffn(make_ffn(M, D, F, DTS[dt], seed=M + F), ACTS[(M + F) % len(ACTS)])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias, residual", [(False, False), (True, False)])
@pytest.mark.parametrize("M", [5, 66])
def test_ffn_epilogues(act, bias, residual, M):
    check_ffn(make_ffn(M, 48, 80, torch.bfloat16, seed=2), act, bias, residual)


@pytest.mark.parametrize("M, D, F", [(2600, 96, 2100), (200, 1024, 700), (2100, 2100, 130), (33, 3000, 64)])
def test_ffn_large_tiles_and_split_products(M, D, F):
    check_ffn(make_ffn(M, D, F, torch.float16, seed=4), "silu")


@pytest.mark.parametrize("M", [7, 77])
def test_ffn_strides(M):
    t = make_ffn(M, 64, 96, torch.float16, seed=9)
    g = torch.Generator(device="cuda").manual_seed(1)
    both = rand(g, torch.float16, 192, 64, scale=0.1)
    wide = rand(g, torch.float16, 96, 160, scale=0.1)
    check_ffn(dict(t, wg=both[:96], wu=both[96:]), "silu")
    check_ffn(dict(t, wg=wide[:, 8:72], wd=wide.t()[:64]), "gelu")                     # leading dimensions that differ; a transposed view
    check_ffn(dict(t, wg=wide[:, 1:65], x=rand(g, torch.float16, M, 131)[:, 3:67]), "gelu_tanh")


def test_no_rows():
    for dt in DTS.values():
        x, w = torch.empty(0, 24, dtype=dt, device="cuda"), torch.ones(8, 24, dtype=dt, device="cuda")
        x.requires_grad_(), w.requires_grad_()
        y = autograd.linear_act(x, w, act="silu", bias=torch.ones(8, dtype=dt, device="cuda"))
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == (0, 8) and dx.shape == x.shape and not dw.any()
        wd = torch.ones(24, 8, dtype=dt, device="cuda", requires_grad=True)
        y = autograd.gated_ffn(x, w, w, wd)
        dw, dd = torch.autograd.grad(y.sum(), (w, wd))
        assert y.shape == (0, 24) and not dw.any() and not dd.any()


@pytest.mark.parametrize("M", [6, 200])
def test_infinities_and_nan_stay_in_their_rows(M):
    x, w, b, r, dy = make_linear(M, 64, 40, torch.bfloat16, seed=1)
    clean = ops.linear_act(x, w, bias=b, act="gelu", residual=r)
    x2 = x.clone()
    x2[2, 3], x2[4, 0] = float("inf"), float("nan")
    y = ops.linear_act(x2, w, bias=b, act="gelu", residual=r)
    keep = [i for i in range(M) if i not in (2, 4)]
    assert torch.equal(y[keep], clean[keep]) and y[4].isnan().all() and not torch.isfinite(y[2]).all()
    assert torch.isnan(ops.linear_act(x2, w, act="relu")[4]).all()
    big = torch.full((M, 64), 3e4, dtype=torch.float16, device="cuda")
    assert torch.isinf(ops.linear_act(big, torch.ones(8, 64, dtype=torch.float16, device="cuda"))).all()
    t = make_ffn(M, 64, 50, torch.bfloat16, seed=1)                                      # a hidden width with padding: NaN of one row stays there
    t["x"][3, 5] = float("nan")
    y = ops.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[i for i in range(M) if i != 3]]).all()


def test_results_are_reproducible_and_neighbours_untouched():
    x, w, b, r, dy = make_linear(300, 2048, 300, torch.bfloat16, seed=3)
    a = run_linear(x, w, b, "gelu", r, dy)
    for _ in range(3):
        c = run_linear(x, w, b, "gelu", r, dy)
        assert all(torch.equal(a[k], c[k]) for k in a)


def test_other_stream_and_graph_replays():
    """forward and backward on a side stream, then captured and replayed with new inputs between eager calls"""
    t = make_ffn(150, 256, 300, torch.bfloat16, seed=6)
    lin = make_linear(150, 256, 200, torch.bfloat16, seed=8)

    def step():
        y, saved = ops.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], residual=t["r"], keep=True)
        grads = ops.gated_ffn_bwd(t["dy"], t["x"], t["wg"], t["wu"], t["wd"], saved, need_gate_up_bias=True, need_down_bias=True)
        z, pre = ops.linear_act(lin[0], lin[1], bias=lin[2], act="gelu", residual=lin[3], keep_pre=True)
        return (y, z) + tuple(grads) + tuple(ops.linear_act_bwd(lin[4], lin[0], lin[1], pre, act="gelu")) + (ops.linear_act(lin[0][:4], lin[1]),)

    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        t["x"].normal_()
        lin[0].normal_()
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured)), k


def test_two_graphs_share_nothing():
    x, w, b, r, dy = make_linear(40, 4096, 64, torch.float16, seed=2)
    x2, w2, _, _, _ = make_linear(40, 4096, 64, torch.float16, seed=12)
    ops.linear_act(x, w)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = ops.linear_act(x, w, act="silu")
    with torch.cuda.graph(g2):
        y2 = ops.linear_act(x2, w2, act="silu")
    e1, e2 = ops.linear_act(x, w, act="silu"), ops.linear_act(x2, w2, act="silu")
    for _ in range(3):
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, e1) and torch.equal(y2, e2)


def test_two_calls_at_once():
    """two streams in turn, without waiting for each other: every call has a workspace of its own"""
    lin = [make_linear(200, 1024, 320, torch.bfloat16, seed=k) for k in (0, 1)]
    ffn = [make_ffn(200, 256, 320, torch.bfloat16, seed=k) for k in (0, 1)]

    def step(k):
        x, w, b, r, dy = lin[k]
        t = ffn[k]
        y, saved = ops.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], keep=True)
        return (ops.linear_act(x, w, bias=b, act="silu", residual=r), y) + ops.linear_act_bwd(dy, x, w) + ops.gated_ffn_bwd(
            t["dy"], t["x"], t["wg"], t["wu"], t["wd"], saved)[:4]

    want = [step(0), step(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(k))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k in (0, 1) for out in got[k] for a, b in zip(out, want[k]))


def test_one_tensor_in_two_places():
    """the weight is also the input (its gradients add up, in the tensors' type), the residual is the input, one matrix is gate and up"""
    w, dy = make_linear(96, 96, 96, torch.bfloat16)[1].detach(), make_linear(96, 96, 96, torch.bfloat16)[4]
    w.requires_grad_()
    (got,) = torch.autograd.grad(autograd.linear_act(w, w, act="silu", residual=w), w, dy)
    parts = [w.detach().clone().requires_grad_() for _ in range(3)]
    dx, dw, dr = torch.autograd.grad(autograd.linear_act(parts[0], parts[1], act="silu", residual=parts[2]), parts, dy)
    exact = dx.double() + dw.double() + dr.double()                                          # two roundings of partial sums, in any order
    assert ((got.double() - exact).abs() <= 2.0 ** -8 * (2.01 * (dx.abs() + dw.abs() + dr.abs()).double())).all()
    t = make_ffn(50, 64, 40, torch.float16)
    t["wu"] = t["wg"]
    x, wg, wd = (t[k].requires_grad_() for k in ("x", "wg", "wd"))
    (got,) = torch.autograd.grad(autograd.gated_ffn(x, wg, wg, wd), wg, t["dy"])
    wu = wg.detach().clone().requires_grad_()
    dg, du = torch.autograd.grad(autograd.gated_ffn(x, wg, wu, wd), (wg, wu), t["dy"])
    assert torch.equal(got, dg + du)


def test_offsets_beyond_32_bits():
    """Inputs, outputs and kept values of more than 2^31 elements.  Only the last rows of dy are not zero: the weight gradients are exactly those of
    these rows (zeros add nothing to a sum), and the values of these rows those of a small call."""
    M, K, N, last = 270001, 8192, 16, 150
    g = torch.Generator(device="cuda").manual_seed(9)
    dt = torch.bfloat16
    x = torch.zeros(M, K, dtype=dt, device="cuda")
    dy = torch.zeros(M, N, dtype=dt, device="cuda")
    x[-last:], dy[-last:] = rand(g, dt, last, K), rand(g, dt, last, N)
    w, b = rand(g, dt, N, K, scale=K ** -0.5), rand(g, dt, N)
    y, pre = ops.linear_act(x, w, bias=b, act="silu", keep_pre=True)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre, act="silu")
    ref = R.linear_ref(x[-last:], w, b, "silu", None, dy[-last:])
    for name, v in (("y", y[-last:]), ("dx", dx[-last:]), ("dw", dw), ("db", db)):
        R.check(name, v, ref[name])
    assert not dx[:-last].any()
    del dx, pre, y
    y = ops.linear_act(x[:, :N], w[:, :N].repeat(K // N, 1), act="relu")                    # the output is the large one
    R.check("y", y[-last:], R.linear_ref(x[-last:, :N], w[:, :N].repeat(K // N, 1), None, "relu", None)["y"])
    assert not y[:-last].any()
    del x, y
    t = make_ffn(1, N, K, dt, seed=4)
    xs = torch.zeros(M, N, dtype=dt, device="cuda")
    xs[-last:] = rand(g, dt, last, N)
    y, saved = ops.gated_ffn(xs, t["wg"], t["wu"], t["wd"], keep=True)
    dx, dg, du, dd = ops.gated_ffn_bwd(dy, xs, t["wg"], t["wu"], t["wd"], saved)[:4]
    ref = R.ffn_ref(xs[-last:], t["wg"], t["wu"], t["wd"], None, None, None, "silu", None, dy[-last:])
    for name, v in (("y", y[-last:]), ("dx", dx[-last:]), ("dwg", dg), ("dwu", du), ("dwd", dd)):
        R.check(name, v, ref[name])
    assert not dx[:-last].any() and not y[:-last].any()


def test_refusals_on_the_device():
    x, w, b, r, dy = make_linear(4, 16, 8, torch.float16)
    bad = [lambda: ops.linear_act(x.float(), w), lambda: ops.linear_act(x, w.bfloat16()), lambda: ops.linear_act(x[:, :8], w),
           lambda: ops.linear_act(x, w, bias=b[:7]), lambda: ops.linear_act(x, w, residual=r[:3]), lambda: ops.linear_act(x, w, bias=b.cpu()),
           lambda: ops.linear_act_bwd(dy, x, w, None, act="silu"), lambda: ops.linear_act_bwd(dy[:2], x, w), lambda: ops.gated_ffn(x, w, w, w),
           lambda: ops.gated_ffn(x, w, w[:4], w.t()), lambda: ops.linear_act(x, w[:0]), lambda: ops.gated_ffn(x, w, w, w.t(), residual=r)]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError, match="act"):
        ops.linear_act(x, w, act="swish")
    y = autograd.linear_act(x.requires_grad_(), w, act="gelu")
    (gx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


def test_without_gradients_nothing_is_kept():
    x, w, b, r, dy = make_linear(70, 64, 40, torch.bfloat16)
    t = make_ffn(70, 64, 40, torch.bfloat16)
    w.requires_grad_(), t["wg"].requires_grad_()
    with torch.no_grad():
        y = autograd.linear_act(x, w, bias=b, act="silu", residual=r)
        z = autograd.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"])
    assert not y.requires_grad and not z.requires_grad
    assert torch.equal(y, autograd.linear_act(x, w, bias=b, act="silu", residual=r)) and torch.equal(z, autograd.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"]))


def test_gradients_against_differences():
    """a directional derivative of the whole block against a central difference in 64 bits of the formulas: the gradients are off by at most their
    bounds (half_reference), summed along the direction"""
    t = make_ffn(40, 24, 32, torch.float16, seed=3)
    names = ("x", "wg", "wu", "wd", "bg", "bu", "bd")
    for k in names:
        t[k].requires_grad_()
    y = autograd.gated_ffn(*(t[k] for k in names), act="gelu_tanh", residual=t["r"])
    got = torch.autograd.grad(y, [t[k] for k in names], t["dy"])
    ref = R.ffn_ref(*(t[k] for k in names), "gelu_tanh", t["r"], t["dy"])
    v = {k: t[k].detach().double() for k in names}

    def value(p):
        g, u = p["x"] @ p["wg"].t() + p["bg"], p["x"] @ p["wu"].t() + p["bu"]
        return (((R.act64("gelu_tanh", g)[0] * u) @ p["wd"].t() + p["bd"]) * t["dy"].double()).sum()

    for k, d in zip(names, got):
        e = torch.randn(v[k].shape, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda", dtype=torch.float64)
        h = 1e-5
        slope = (value({**v, k: v[k] + h * e}) - value({**v, k: v[k] - h * e})) / (2 * h)
        bound = (ref["d" + k].off * e.abs()).sum() + 1e-6 * (1 + slope.abs())
        assert (slope - (d.double() * e).sum()).abs() <= bound, k


@pytest.mark.parametrize("M, D, F", [(4200, 64, 2700), (300, 72, 1000), (90, 2048, 300), (5, 40, 33)])
def test_ffn_bias_gradients_alone(M, D, F):
    """256-wide tiles, 128-wide ones, a split K, few rows; asked for alone they are what they are beside everything else, and the padding is zero"""
    t = make_ffn(M, D, F, torch.float16, seed=5)
    check_ffn(t, "gelu")
    y, saved = ops.gated_ffn(t["x"].detach(), t["wg"].detach(), t["wu"].detach(), t["wd"].detach(), keep=True)
    args = (t["dy"], t["x"].detach(), t["wg"].detach(), t["wu"].detach(), t["wd"].detach(), saved)
    alone = ops.gated_ffn_bwd(*args, need_x=False, need_gate_up=False, need_down=False, need_gate_up_bias=True)
    every = ops.gated_ffn_bwd(*args, need_gate_up_bias=True, need_down_bias=True)
    assert alone[0] is None and alone[1] is None and alone[6] is None
    assert torch.equal(alone[4], every[4]) and torch.equal(alone[5], every[5])
    whole = alone[4].as_strided((2 * ((F + 7) // 8 * 8),), (1,), 0)
    assert not whole[F:(F + 7) // 8 * 8].any() and not whole[(F + 7) // 8 * 8 + F:].any()


def test_mixed_needs():
    """only the gradients that are asked for are formed; the others are None"""
    x, w, b, r, dy = make_linear(50, 64, 40, torch.bfloat16)
    w.requires_grad_()
    y = autograd.linear_act(x, w, bias=b, act="silu", residual=r)
    y.backward(dy)
    assert w.grad is not None and x.grad is None and b.grad is None
    t = make_ffn(50, 64, 40, torch.bfloat16)
    t["wd"].requires_grad_()
    autograd.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"]).backward(t["dy"])
    R.check("dwd", t["wd"].grad, R.ffn_ref(*(t[k] for k in ("x", "wg", "wu", "wd")), None, None, None, "silu", None, t["dy"])["dwd"])


def test_a_residual_block_trains():
    """linear -> gated block -> linear with residuals, as a model would chain them: gradients of the whole against 64-bit autograd.  Chained
    roundings: each of the 4 products rounds its output and one intermediate, each by at most u relative to its norm, and the gradients pass
    the chain once more: 16 u in the norm."""
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(11)
    x = rand(g, dt, 500, 96)
    p = {"w1": rand(g, dt, 64, 96, scale=0.1), "b1": rand(g, dt, 64, scale=0.1), "wg": rand(g, dt, 160, 64, scale=0.12), "wu": rand(g, dt, 160, 64, scale=0.12),
         "wd": rand(g, dt, 64, 160, scale=0.08), "w2": rand(g, dt, 64, 64, scale=0.12)}
    for v in p.values():
        v.requires_grad_()
    h = autograd.linear_act(x, p["w1"], bias=p["b1"], act="gelu")
    h = autograd.gated_ffn(h, p["wg"], p["wu"], p["wd"], residual=h)
    y = autograd.linear_act(h, p["w2"], act="silu", residual=h)
    dy = rand(g, dt, 500, 64)
    got = torch.autograd.grad(y, list(p.values()), dy)
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    h = R.act64("gelu", x.double() @ q["w1"].t() + q["b1"])[0]
    h = h + (R.act64("silu", h @ q["wg"].t())[0] * (h @ q["wu"].t())) @ q["wd"].t()
    z = h + R.act64("silu", h @ q["w2"].t())[0]
    want = torch.autograd.grad(z, list(q.values()), dy.double())
    assert (y.double() - z).norm() <= 16 * 2 ** -8 * z.norm()
    for k, a, b in zip(p, got, want):
        assert (a.double() - b).norm() <= 16 * 2 ** -8 * b.norm(), k


@pytest.mark.parametrize("act", ACTS)
def test_far_values_have_the_slopes_of_their_sides(act):
    """single features whose pre-activations are as large as bf16 holds: outputs and gradients are those of the 64-bit form (all finite)"""
    v = [1e15, 1e19, 2e19, 1e20, 1e30, 3e38]
    x = torch.tensor([s * a for a in v for s in (1, -1)], dtype=torch.bfloat16, device="cuda")[:, None]
    one = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    for M in (3, len(x)):
        out = run_linear(x[:M].clone(), one.clone(), None, act, None, torch.ones(M, 1, dtype=torch.bfloat16, device="cuda"))
        a, slope = R.act64(act, x[:M].double())
        assert ((out["y"].double() - a).abs() <= 2.0 ** -8 * a.abs() + 1e-30).all()
        assert ((out["dx"].double() - slope).abs() <= 2.0 ** -8 * slope.abs() + 1e-30).all()
    t = {"x": x, "wg": one, "wu": torch.zeros_like(one), "wd": one}
    t = {k: w.clone().requires_grad_() for k, w in t.items()}
    y = autograd.gated_ffn(t["x"], t["wg"], t["wu"], t["wd"], b_up=torch.ones(1, dtype=torch.bfloat16, device="cuda"), act=act)       # y = act(x)
    (dx,) = torch.autograd.grad(y, t["x"], torch.ones_like(y))
    a, slope = R.act64(act, x.double())
    assert ((y.double() - a).abs() <= 2.0 ** -7 * a.abs() + 1e-30).all() and ((dx.double() - slope).abs() <= 2.0 ** -7 * slope.abs() + 1e-30).all()


@pytest.mark.parametrize("M", [2, 20, 70, 300])
def test_subnormal_values_count(M):
    """fp16 values below 2^-14, as inputs, weights, incoming gradients and results: sums of exact products by powers of two, so every
    sum is exact (a multiple of 2^-24 below 2^-12) and rounded once"""
    g = torch.Generator(device="cuda").manual_seed(M)

    def small(*shape):
        return (torch.randint(-1023, 1024, shape, generator=g, device="cuda").double() * 2.0 ** -24).half()

    def powers(*shape):
        return torch.where(torch.randint(0, 2, shape, generator=g, device="cuda") > 0, 1.0, -1.0).half()

    for x, w, dy in ((small(M, 72), powers(40, 72), powers(M, 40)), (powers(M, 72), small(40, 72), small(M, 40))):
        x[:, 3:] = 0                                                   # three products a sum
        y = ops.linear_act(x, w)
        exact = x.double() @ w.double().t()
        assert torch.equal(y, exact.half()) and bool((exact != 0).any()) and float(exact.abs().max()) < 2.0 ** -12
        dy[4:] = 0
        dy[:, 4:] = 0                                                  # dx: four products a sum; dW, db: as many rows
        dx, dw, db = ops.linear_act_bwd(dy, x, w)
        assert torch.equal(dx, (dy.double() @ w.double()).half()) and torch.equal(dw, (dy.double().t() @ x.double()).half())
        assert torch.equal(db, dy.double().sum(0).half())
