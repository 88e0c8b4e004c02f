"""ShardedSCAO clips the averaged gradients by their norm over all ranks: 2 gloo
ranks on the CPU, with the norm and the scaling of the GPU library replaced by
torch's (the sharing between the ranks is what runs here)."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from scao_b200 import distributed, workloads
from scao_b200.distributed import ShardedSCAO


class _SGD:
    def __init__(self, pairs):
        self.ps = [p for p, _ in pairs]

    def step(self):
        for p in self.ps:
            p.data.add_(p.grad, alpha=-0.1)


def _worker(rank, world, port, hooked, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        distributed.get_total_norm = torch.nn.utils.get_total_norm
        distributed.clip_grads_with_norm_ = torch.nn.utils.clip_grads_with_norm_
        w = workloads.tiny()
        torch.manual_seed(0)
        params = [torch.nn.Parameter(torch.randn(s.shape)) for s in w.params]
        start = [p.detach().clone() for p in params]
        opt = ShardedSCAO(params, w, _SGD, buckets=2)
        errs = []
        if hooked:
            opt.attach_grad_hooks()
        for max_norm in (0.25, 1e6):
            before = [p.detach().clone() for p in params]
            if hooked:
                sum((p * (rank + 1.0) * (i + 1)).sum() for i, p in enumerate(params)).backward()
            else:
                for i, p in enumerate(params):
                    p.grad = torch.full(p.shape, (rank + 1.0) * (i + 1))
            opt.flat_grad_from_params()
            opt.step(max_norm)
            avg = [torch.full(s.shape, (1 + world) / 2 * (i + 1)) for i, s in enumerate(start)]
            norm = torch.cat([a.reshape(-1) for a in avg]).norm().item()
            c = min(1.0, max_norm / (norm + 1e-6))
            errs.append(abs(opt.total_norm.item() / norm - 1))
            errs += [(p.detach() - (b - 0.1 * c * a)).abs().max().item()
                     for p, b, a in zip(params, before, avg)]
        with pytest.raises(ValueError):
            opt.step(-1.0)
        q.put((rank, max(errs)))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("hooked", [False, True])
def test_sharded_clip(hooked):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, hooked, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
    # single-precision sums of a few thousand values: 1e-5 of values up to about 20
    assert set(got) == {0, 1} and max(got.values()) < 2e-4, got
