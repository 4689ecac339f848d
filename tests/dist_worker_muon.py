"""Two ranks training with --optimizer muon on a data-parallel bucket, able to run on ONE GPU.

Launched by tests/test_muon_gpu.py::test_two_ranks_on_one_bucket as
    python -m torch.distributed.run --nnodes=1 --nproc-per-node 2 --master-addr 127.0.0.1 --master-port P tests/dist_worker_muon.py
The direct reducer is set up first, as --dp-reduce direct does: make_optimizer has to close it, because FlatMuon reads final gradients.  Three steps
of  ACMIL_GA.train_step -> mean of the bucket -> FlatMuon.step, step 1 with a bag outside the split-f16 range on rank 1 only.  The bucket is
averaged through host memory (gloo).  Checks, on every rank: (i) the reducer is closed and no optimizer owns it; (ii) bit-identical parameters and
momentum on both ranks after every step; (iii) equal to ONE process stepping on the averaged gradients of the same two bags; (iv) the flagged step, whose
flag rides in the bucket, is skipped by BOTH ranks and leaves parameters and momentum as they were.  Prints MUON_OK on rank 0.
"""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from acmil_amd import train as T  # noqa: E402
from acmil_amd.optim import FlatMuon  # noqa: E402
from dist_worker_nccl import bag_of  # noqa: E402


def setup(dev, seed, rank=None, world=1):
    conf = T.Struct(train_epoch=3, warmup_epoch=0, wd=1e-2, lr=1e-3, min_lr=0, n_class=3, n_token=5, n_masked_patch=10, mask_drop=0.6,
                    arch="ga", precision="f16x3", seed=1, D_feat=384, D_inner=128, optimizer="muon")
    T.set_seed(seed)
    model = T.build_model(conf).to(dev).train()
    bucket = T.GradBucket(list(model.parameters()))
    peer = None
    if rank is not None:
        assert bucket.enable_direct(rank, world), "direct reduction could not be set up"
        peer = bucket.peer
    opt = T.make_optimizer(model, conf, dev, bucket, lr=conf.lr)
    assert isinstance(opt, FlatMuon) and bucket.peer is None and opt.peer is None and opt.grad.data_ptr() == bucket.flat.data_ptr()
    assert peer is None or (peer._closed and getattr(peer, "owner", None) is None)
    return model, bucket, opt


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    assert world == 2
    dev = torch.device("cuda", rank % torch.cuda.device_count())
    torch.cuda.set_device(dev)
    dist.init_process_group("gloo")
    model, bucket, opt = setup(dev, 7, rank, world)               # same seed: identical initial parameters
    twin, tbucket, topt = setup(dev, 99)                          # single-process replica on this rank's GPU
    twin.load_state_dict(model.state_dict())
    uniforms = [torch.rand(5, 10, generator=torch.Generator().manual_seed(50 + s)).to(dev) for s in range(3)]
    for step in range(3):
        x, y = bag_of(rank, step, step == 1 and rank == 1)
        _, out = model.train_step(x.to(dev).unsqueeze(0), torch.tensor([y], device=dev), uniforms=uniforms[step], guard_flag=opt.guard_flag,
                                  optimizer=opt, track_flag=True)
        assert out["opt_step_id"] is None, "the step applied the optimizer ahead of the gradient reduction"
        bucket.sync_from_grads()
        mean = bucket.flat.cpu()
        dist.all_reduce(mean)
        bucket.flat.copy_(mean / world)
        before = opt.flat.clone(), opt.exp_avg.clone()
        sid = opt.step(track_flag=True)
        assert (opt.poll_skipped(0) == [sid]) == (step == 1), step
        if step == 1:
            assert torch.equal(opt.flat, before[0]) and torch.equal(opt.exp_avg, before[1])
        else:
            assert not torch.equal(opt.flat, before[0])
        for mine in (opt.flat, opt.exp_avg):
            both = [torch.empty_like(mine).cpu() for _ in range(world)]
            dist.all_gather(both, mine.cpu())
            assert torch.equal(both[0], both[1]), "ranks diverged at step %d" % step
        acc = torch.zeros_like(tbucket.flat)
        for r in range(world):
            xr, yr = bag_of(r, step, step == 1 and r == 1)
            twin.train_step(xr.to(dev).unsqueeze(0), torch.tensor([yr], device=dev), uniforms=uniforms[step], guard_flag=topt.guard_flag)
            tbucket.sync_from_grads()
            acc += tbucket.flat
        tbucket.flat.copy_(acc / world)
        topt.step(track_flag=True)
        topt.poll_skipped(0)
        assert torch.equal(topt.flat, opt.flat), "step %d: not what one process does with the averaged gradients (max diff %g)" % (
            step, (topt.flat - opt.flat).abs().max().item())
    assert opt.skipped_steps == 1 and opt.step_count == 2 and topt.skipped_steps == 1
    dist.barrier()
    if rank == 0:
        print("MUON_OK")
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
