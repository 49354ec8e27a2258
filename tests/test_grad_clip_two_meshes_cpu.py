"""Norm and clipping of gradients that FSDP2 shards on top of tensor parallelism, on four `gloo` ranks: both mesh
dimensions hold different parts, although FSDP2's placement there is not a plain Shard."""
import os
import socket

import torch
import torch.multiprocessing as mp

from test_grad_clip_distributed_cpu import _stand_ins

WORLD = 4


def _rank(rank, port):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.fsdp import fully_shard
    from torch.distributed.tensor.parallel import ColwiseParallel, parallelize_module, RowwiseParallel

    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=WORLD)
    lib = _stand_ins()
    from float8_experimental_b200 import clip_grad_norm_, get_total_norm

    mesh = init_device_mesh("cpu", (2, 2), mesh_dim_names=("dp", "tp"))
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(6, 8), torch.nn.Linear(8, 6))
    x = torch.randn(5, 6)
    grads = torch.autograd.grad(model(x).square().sum(), list(model.parameters()))
    want = float(torch.cat([g.reshape(-1) for g in grads]).double().norm())
    parallelize_module(model, mesh["tp"], {"0": ColwiseParallel(), "1": RowwiseParallel()})
    fully_shard(model, mesh=mesh["dp"])
    model(x).square().sum().backward()
    total = get_total_norm([p.grad for p in model.parameters()])
    assert abs(float(total) - want) <= 1e-5 * want, (float(total), want)
    assert abs(float(clip_grad_norm_(model.parameters(), 0.5)) - want) <= 1e-5 * want
    for p, g in zip(model.parameters(), grads):
        assert torch.allclose(p.grad.full_tensor(), g * (0.5 / want), rtol=1e-4, atol=1e-7)
    dist.barrier()
    dist.destroy_process_group()
    del lib


def test_both_mesh_dimensions_count():
    for attempt in range(3):  # the probed port can be taken again before rank 0 listens on it
        with socket.socket() as s:
            s.bind(("127.0.0.1", 0))
            port = s.getsockname()[1]
        try:
            mp.spawn(_rank, args=(port,), nprocs=WORLD, join=True)
            return
        except Exception as exc:  # noqa: BLE001
            if "EADDRINUSE" not in str(exc) or attempt == 2:
                raise
