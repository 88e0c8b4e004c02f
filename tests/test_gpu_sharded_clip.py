"""ShardedSCAO.step(max_grad_norm) on the NCCL path with the library's kernels: one rank in
a process of its own, against clipping by hand and unsharded optimizers."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu
KW = dict(lr=1e-3, sparsity=0.0, noise_std_init=0.0, async_precond=False, warmup_steps=2, precond_freq=2,
          min_precond_updates=1, blend_steps=2, k_min=4, k_max=16, max_precond_dim=48)


def _rank(rank, port, out):
    from datetime import timedelta

    import torch.distributed as dist

    from scao_b200 import SCAO, clip_grad_norm_, workloads
    from scao_b200.distributed import ShardedSCAO
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    dist.init_process_group("nccl", rank=rank, world_size=1, device_id=dev, timeout=timedelta(seconds=60))
    try:
        w = workloads.tiny()
        gen = torch.Generator(device=dev).manual_seed(3)
        new = lambda s, k=1.0: torch.randn(s.shape, generator=gen, device=dev) * k  # noqa: E731
        params = [torch.nn.Parameter(new(s, 0.1)) for s in w.params]
        plain = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt = ShardedSCAO(params, w, lambda pairs: SCAO([p for p, _ in pairs], **KW), buckets=2)
        lay = opt.layout
        each = [SCAO([plain[i] for i in opt.my if lay.bucket[i] == b], **KW) for b in range(lay.nb)]
        worst = 0.0
        for k, max_norm in enumerate((0.5, 1e6, 0.01, 2.0, 0.3)):
            grads = [new(s, 0.3) for s in w.params]
            for p, q, g in zip(params, plain, grads):
                p.grad, q.grad = g.clone(), g.clone()
            opt.flat_grad_from_params()
            opt.step(max_norm)
            total = clip_grad_norm_(plain, max_norm)
            for o in each:
                o.step()
            worst = max(worst, abs(opt.total_norm.item() / total.item() - 1))
        torch.cuda.synchronize()
        far = max(((p - q).norm() / q.norm()).item() for p, q in zip(params, plain))
        out["norm"], out["params"] = worst, far
    finally:
        dist.destroy_process_group()


def test_one_rank_clips_like_by_hand():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = mp.get_context("spawn").Manager().dict()
    mp.spawn(_rank, args=(port, out), nprocs=1, join=True)
    # the norm is squared in 64 bits and its root rounded once more (2^-24); the scaled
    # gradients follow, and the updates with them (about as much, over five steps)
    assert out["norm"] <= 2.0 ** -22 and out["params"] <= 2.0 ** -18, dict(out)
