"""Gradient norm and clipping of sharded gradients on two `gloo` ranks, the kernels replaced by CPU stand-ins: what is
all-reduced, over which groups, and that every rank ends with the norm of the whole gradients."""
import math
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

WORLD = 2


def _stand_ins():
    """Multi-tensor norm and scaling with torch, under the CPU key of the library's operators."""
    import float8_experimental_b200._ops  # noqa: F401  (defines the schemas)

    def multi_norm(xs, kind, root):
        flat = torch.cat([x.reshape(-1).double() for x in xs])
        if kind == 0:
            v = flat.abs().max() if flat.numel() else flat.sum()
        else:
            v = (flat.abs() ** kind).sum()
            v = v.sqrt() if root and kind == 2 else v
        return v.float()

    def multi_clip_(xs, total_norm, max_norm):
        f = min(1.0, max_norm / (float(total_norm) + 1e-6))
        for x in xs:
            x.mul_(f)

    lib = torch.library.Library("f8b200", "IMPL")
    lib.impl("multi_norm", multi_norm, "CPU")
    lib.impl("multi_clip_", multi_clip_, "CPU")
    return lib


def _rank(rank, port):
    import torch.distributed as dist
    from torch.distributed._tensor import distribute_tensor, Replicate, Shard
    from torch.distributed.device_mesh import init_device_mesh

    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=WORLD)
    lib = _stand_ins()
    from float8_experimental_b200 import clip_grad_norm_, get_total_norm

    mesh = init_device_mesh("cpu", (WORLD,))
    gen = torch.Generator().manual_seed(0)  # the same whole gradients on both ranks
    whole = [torch.randn(7, 5, generator=gen), torch.randn(1, 9, generator=gen), torch.randn(12, generator=gen),
             torch.randn(3, generator=gen)]
    # 7 rows and 1 row over two ranks: uneven and empty shards; one replicated; one an ordinary tensor
    places = [[Shard(0)], [Shard(0)], [Replicate()], None]
    params = []
    for w, place in zip(whole, places):
        g = w.clone() if place is None else distribute_tensor(w.clone(), mesh, place)
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        params.append(p)
    flat = torch.cat([w.reshape(-1).double() for w in whole])
    for kind, want in ((2.0, flat.norm()), (1.0, flat.abs().sum()), (math.inf, flat.abs().max())):
        got = get_total_norm([p.grad for p in params], kind)
        assert abs(float(got) - float(want)) <= 1e-5 * float(want), (rank, kind)
    total = clip_grad_norm_(params, 0.5)
    assert abs(float(total) - float(flat.norm())) <= 1e-5 * float(flat.norm())
    for p, w, place in zip(params, whole, places):
        g = p.grad if place is None else p.grad.full_tensor()
        assert torch.allclose(g, w * (0.5 / float(flat.norm())), rtol=1e-4, atol=0)
    # a sum that is still spread over the ranks has no norm yet
    from torch.distributed._tensor import DTensor, Partial

    with pytest.raises(NotImplementedError, match="Partial"):
        get_total_norm([DTensor.from_local(torch.ones(3), mesh, [Partial()])])
    dist.barrier()
    dist.destroy_process_group()
    del lib


def test_sharded_gradients_count_once():
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
