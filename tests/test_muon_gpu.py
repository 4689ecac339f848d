"""optim.FlatMuon and `train --optimizer muon`: orthogonalised momentum for the matrices, AdamW for the rest."""
import math

import pytest
import torch

from acmil_amd import autograd, ops
from acmil_amd.optim import FlatAdamW, FlatMuon
from test_ortho_gpu import iterate

pytestmark = pytest.mark.gpu
SHAPES = [(64, 96), (96,), (5, 96), (40, 40), (32, 200), (7, 3, 3), (200, 33)]
MATRICES = [0, 3, 4, 6]


def parameters(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(*s, generator=g) * 0.1).cuda()) for s in SHAPES]


def set_grads(params, seed):
    g = torch.Generator().manual_seed(100 + seed)
    for p in params:
        p.grad.copy_(torch.randn(*p.shape, generator=g) * 1e-2)


@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_follow_the_formula(nesterov):
    """Matrices against the formula in 64 bits: an update is off by at most lr scale times the orthogonalisation's own bound (test_ortho_gpu), the
    momentum and the parameter by roundings of 2^-24 each (8 of them per step are allowed).  The rest is FlatAdamW bit for bit."""
    params, twin = parameters(), parameters()
    opt = FlatMuon(params, lr=1e-2, weight_decay=0.1, nesterov=nesterov)
    ref = FlatAdamW(twin, lr=1e-2, weight_decay=0.1)
    assert opt._muon_indices == MATRICES
    want = {i: params[i].detach().double() for i in MATRICES}
    buf = {i: torch.zeros_like(want[i]) for i in MATRICES}
    slack = {i: 0.0 for i in MATRICES}
    for step in range(4):
        lr = 1e-2 / (1 + step)
        opt.param_groups[0]["lr"] = ref.param_groups[0]["lr"] = lr
        set_grads(params, step), set_grads(twin, step)
        opt.step(), ref.step()
        for i in MATRICES:
            g = params[i].grad.double()
            buf[i] = 0.95 * buf[i] + g
            o, bound = iterate(g + 0.95 * buf[i] if nesterov else buf[i], torch.float64)
            scale = 0.2 * math.sqrt(max(want[i].shape))
            want[i] = want[i] * (1 - lr * 0.1) - lr * scale * o
            slack[i] += lr * scale * (bound + 3.9 ** 5 * 2 ** -22) + 8 * 2 ** -24 * float(want[i].norm())
            assert (params[i].double() - want[i]).norm() <= slack[i], (step, i)
        for i, (p, q) in enumerate(zip(params, twin)):
            if i not in MATRICES:
                assert torch.equal(p, q), (step, i)


def test_a_raised_flag_skips_the_step():
    params = parameters()
    opt = FlatMuon(params, lr=1e-2)
    set_grads(params, 0)
    opt.guard_flag.zero_()
    opt.step(track_flag=True)
    before, momentum = opt.flat.clone(), opt.exp_avg.clone()
    opt.guard_flag.fill_(1.0)
    opt.step(track_flag=True)
    assert torch.equal(opt.flat, before) and torch.equal(opt.exp_avg, momentum)
    assert opt.poll_skipped(0) == [2] and opt.skipped_steps == 1 and opt._run_skips.tolist() == [1] * len(opt._runs)
    opt.guard_flag.zero_()
    twin = parameters()
    other = FlatMuon(twin, lr=1e-2)
    for k in (0, 1):
        set_grads(twin, k)
        other.step()
    set_grads(params, 1)
    opt.step()
    assert torch.equal(opt.flat, other.flat)                       # the skipped step left no trace, bias corrections included


def test_state_and_choice_of_matrices():
    params = parameters()
    opt = FlatMuon(params, lr=1e-2, momentum=0.9, ns_steps=3, muon=[params[0], params[2]])
    assert opt._muon_indices == [0, 2]
    for k in range(2):
        set_grads(params, k)
        opt.step()
    sd = opt.state_dict()
    again = FlatMuon(parameters(), lr=1.0, muon=None)
    with pytest.raises(RuntimeError, match="other parameters"):
        again.load_state_dict(sd)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    new = FlatMuon(twin, lr=1.0, muon=[twin[0], twin[2]])
    new.load_state_dict(sd)
    assert new.param_groups[0]["momentum"] == 0.9 and new.param_groups[0]["ns_steps"] == 3 and new.param_groups[0]["lr"] == 1e-2
    set_grads(params, 5), set_grads(twin, 5)
    opt.step(), new.step()
    assert torch.equal(opt.flat, new.flat)
    adam = FlatAdamW(parameters(), lr=1e-2)
    with pytest.raises(RuntimeError, match="FlatMuon"):
        adam.load_state_dict(sd)
    with pytest.raises(RuntimeError, match="another optimizer"):
        opt.load_state_dict(adam.state_dict())
    for bad in (dict(muon=[params[1]]), dict(muon=[torch.nn.Parameter(torch.zeros(40, 40, device="cuda"))])):
        with pytest.raises(RuntimeError):
            FlatMuon(params, **bad)
    with pytest.raises(RuntimeError, match="no weight matrix"):
        FlatMuon([torch.nn.Parameter(torch.zeros(9, device="cuda"))])
    with pytest.raises(ValueError):
        FlatMuon(parameters(), momentum=1.0)


def test_what_a_step_cannot_run_is_refused_before_anything_changes():
    """more steps than one call takes, a momentum of 1, a matrix of more than 65536 rows: by the constructor, by load_state_dict, and by step() where the
    group was changed in between -- with parameters, momentum and counters as they were"""
    for bad in (dict(ns_steps=65), dict(ns_steps=0), dict(momentum=1.0), dict(momentum=-0.1)):
        with pytest.raises(ValueError):
            FlatMuon(parameters(), **bad)
    params = parameters()
    opt = FlatMuon(params, lr=1e-2)
    set_grads(params, 0)
    opt.step()

    def seen():
        return [opt.flat.clone(), opt.exp_avg.clone(), opt.exp_avg_sq.clone()], (opt.step_count, opt._step_id, opt._launches, opt.mutations)

    tensors, counters = seen()
    for key, value in (("ns_steps", 65), ("ns_steps", 0), ("momentum", 1.0), ("momentum", float("nan"))):
        good = opt.param_groups[0][key]
        opt.param_groups[0][key] = value
        with pytest.raises(ValueError):
            opt.step()
        opt.param_groups[0][key] = good
        sd = opt.state_dict()
        sd["param_groups"][0][key] = value
        with pytest.raises(ValueError):
            opt.load_state_dict(sd)
        now, count = seen()
        assert count == counters and all(torch.equal(a, b) for a, b in zip(now, tensors)) and opt.param_groups[0][key] == good
    twin = parameters()
    other = FlatMuon(twin, lr=1e-2)
    for k in (0, 1):
        set_grads(twin, k)
        other.step()
    set_grads(params, 1)
    opt.step()
    assert torch.equal(opt.flat, other.flat)                       # the refusals left no trace
    tall = torch.nn.Parameter(torch.full((65537, 32), 0.5, device="cuda"))
    with pytest.raises(RuntimeError, match="at most 65536"):
        FlatMuon([tall], muon=[tall])
    rest = torch.nn.Parameter(torch.full((40, 32), 0.5, device="cuda"))
    opt = FlatMuon([tall, rest], lr=1e-2, weight_decay=0.0)        # left to AdamW: the first step moves every value by lr
    assert opt._muon_indices == [1]
    opt.grad[:-1].fill_(1.0)                                       # (the last slot is the range flag)
    opt.step()
    assert ((tall - 0.49).abs() <= 1e-6).all()                     # 0.5 - 1e-2 / (1 + 1e-8), three roundings of values below 1


def test_a_group_that_cannot_be_read_changes_nothing():
    """a value of the wrong kind in the group raises before the momentum moves: the step can be taken again with a right one"""
    params = parameters()
    opt = FlatMuon(params, lr=1e-2)
    set_grads(params, 0)
    flat = opt.flat.clone()
    for key, value in (("ns_steps", 2.5), ("lr", None), ("weight_decay", "much"), ("betas", (0.9, None)), ("nesterov", None)):
        good = opt.param_groups[0][key]
        opt.param_groups[0][key] = value
        with pytest.raises((TypeError, ValueError)):
            opt.step()
        opt.param_groups[0][key] = good
        assert not opt.exp_avg.any() and torch.equal(opt.flat, flat) and opt.step_count == 0 and opt._launches == 0, key
    twin = parameters()
    other = FlatMuon(twin, lr=1e-2)
    set_grads(twin, 0)
    other.step(), opt.step()
    assert torch.equal(opt.flat, other.flat)


def test_a_step_makes_its_parameters_device_the_current_one(monkeypatch):
    """every library call of a step is made while the parameters' device is entered, whatever device was current (seen here by what is entered: one
    device is enough)"""
    from acmil_amd import _lib, optim
    params = parameters()
    opt = FlatMuon(params, lr=1e-2)
    set_grads(params, 0)
    inside, calls, real = [], [], _lib.load()

    class Guard(torch.cuda.device):
        def __init__(self, device):
            super().__init__(device)
            self.asked = device

        def __enter__(self):
            inside.append(self.asked)
            return super().__enter__()

        def __exit__(self, *e):
            inside.pop()
            return super().__exit__(*e)

    class Lib:
        def __getattr__(self, name):
            calls.append((name, list(inside)))
            return getattr(real, name)

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(optim._lib, "load", Lib)
    opt.step()
    assert {n for n, _ in calls} >= {"acmil_muon_momentum", "acmil_orthogonalize", "acmil_muon_apply", "acmil_adamw_step"}
    assert all(devices and devices[0] == opt.flat.device for _, devices in calls) and not inside


def test_more_matrices_than_one_launch_holds():
    g = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter((torch.randn(32, 32 + k % 3, generator=g) * 0.1).cuda()) for k in range(70)]
    opt = FlatMuon(params, lr=1e-2, weight_decay=0.0, nesterov=False)
    start = [p.detach().clone() for p in params]
    for k, p in enumerate(params):
        p.grad.copy_(torch.randn(*p.shape, generator=g))
    opt.step()
    for k in (0, 23, 24, 63, 64, 69):
        o = ops.orthogonalize(params[k].grad)
        want = start[k] - 1e-2 * 0.2 * math.sqrt(max(params[k].shape)) * o
        assert (params[k] - want).abs().max() <= 2 ** -22 * (start[k].abs().max() + 0.1)       # two roundings of values below 0.6


def test_trains_the_16_bit_layers():
    """a residual block of linear_act and gated_ffn on bf16 copies of fp32 parameters, stepped by FlatMuon: the step is the formula's for the gradients
    that arrived (bounds as in test_steps_follow_the_formula), and those are the ones the block gives without the optimizer"""
    g = torch.Generator().manual_seed(3)
    shapes = {"w": (64, 96), "b": (64,), "wg": (160, 64), "wu": (160, 64), "wd": (64, 160)}
    p = {k: torch.nn.Parameter((torch.randn(*s, generator=g) * 0.1).cuda()) for k, s in shapes.items()}
    x, dy = torch.randn(300, 96, generator=g).cuda().bfloat16(), torch.randn(300, 64, generator=g).cuda().bfloat16()

    def block(q):
        h = autograd.linear_act(x, q["w"], bias=q["b"], act="gelu")
        return autograd.gated_ffn(h, q["wg"], q["wu"], q["wd"], residual=h)

    opt = FlatMuon(p.values(), lr=1e-2, weight_decay=0.1)
    for step in range(2):
        half = {k: v.detach().bfloat16().requires_grad_() for k, v in p.items()}
        want = torch.autograd.grad(block(half), list(half.values()), dy)
        before = {k: v.detach().double() for k, v in p.items()}
        buf = {k: opt.exp_avg[o:o + v.numel()].view(v.shape).double() for (k, v), o in zip(p.items(), _offsets(p))}
        opt.zero_grad()
        block({k: v.bfloat16() for k, v in p.items()}).backward(dy)
        for (k, v), w in zip(p.items(), want):
            assert torch.equal(v.grad, w.float()), k
        opt.step()
        for k in ("w", "wg", "wu", "wd"):
            grad = p[k].grad.double()
            o, bound = iterate(grad + 0.95 * (0.95 * buf[k] + grad), torch.float64)
            scale = 1e-2 * 0.2 * math.sqrt(max(shapes[k]))
            new = before[k] * (1 - 1e-3) - scale * o
            assert (p[k].double() - new).norm() <= scale * (bound + 3.9 ** 5 * 2 ** -22) + 8 * 2 ** -24 * float(new.norm()), (step, k)


def _offsets(p):
    at = 0
    for v in p.values():
        yield at
        at += v.numel()


@pytest.mark.parametrize("n_token, bags", [(5, 1), (1, 1), (5, 4)])
def test_trainer_runs_with_muon(n_token, bags):
    """train.train_one_epoch with the optimizer make_optimizer builds for --optimizer muon: runs, applies every step, moves every trained
    parameter, and leaves the frozen branch head of an n_token = 1 model alone"""
    from acmil_amd import train as T
    args = T.get_arguments(["--optimizer", "muon", "--n_token", str(n_token)])
    assert args.optimizer == "muon" and T.get_arguments([]).optimizer == "adamw"
    dev = torch.device("cuda", 0)
    conf = T.Struct(train_epoch=1, warmup_epoch=0, wd=1e-5, lr=1e-3, min_lr=0, n_class=3, n_token=n_token, n_masked_patch=10, mask_drop=0.6, arch="ga",
                    precision="f16x3", seed=0, D_feat=512, D_inner=256, optimizer="muon", bags_per_step=bags)
    T.set_seed(0)
    model = T.build_model(conf).to(dev).train()
    opt = T.make_optimizer(model, conf, dev, None, lr=conf.lr)
    names = [n for n, p in model.named_parameters()]
    assert [names[i] for i in opt._muon_indices] == ["dimreduction.fc1.weight", "attention.attention_V.0.weight", "attention.attention_U.0.weight"]
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    T.train_one_epoch(model, T.SyntheticBags(8, 700, 512, 3, seed=1), opt, dev, 0, conf, log_every=0)
    opt.poll_skipped(0)
    assert opt.step_count == 8 // bags and opt.skipped_steps == 0
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all()
        assert torch.equal(p, before[n]) == (n_token == 1 and n.startswith("classifier.0")), n


def test_two_ranks_on_one_bucket():
    """data-parallel training with FlatMuon: the direct reducer is closed, a flag of one rank skips the step on both, both ranks and a single process on
    the averaged gradients agree bit for bit (tests/dist_worker_muon.py)"""
    import os
    import socket
    import subprocess
    import sys
    s = socket.socket(); s.bind(("127.0.0.1", 0)); port = s.getsockname()[1]; s.close()
    env = dict(os.environ)
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "dist_worker_muon.py")
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
                        "--master-port", str(port), worker], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert r.returncode == 0 and "MUON_OK" in r.stdout, r.stdout[-3000:]
