"""The exchange around the classifier loss and the sharded gradient norm under gloo, with stand-ins for
the GPU calls (no GPU needed)."""
import os
import socket
import sys

import multiprocessing as mp
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "pytorch-retinanet_amd")


def _batch():
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(11, 6, generator=g, dtype=torch.float64), torch.randn(5, 6, generator=g, dtype=torch.float64)
    y = torch.tensor([0, 4, 2, -100, 1, 3, -100, -100, 2, -1, 5])      # the last two: outside, left out
    return x, w, y


def _mean(x, w, y, divisor):
    keep = (y >= 0) & (y < w.shape[0])
    rows = torch.nn.functional.cross_entropy(x @ w.T, torch.where(keep, y, 0), reduction="none")
    return (rows * keep).sum().reshape(1) / divisor


class _Loss(torch.nn.Module):
    """What the wrapper needs of retinahead.LinearCrossEntropy, on host tensors."""
    cfg = dict(reduction="mean", ignore_index=-100)

    def forward(self, features, weight, labels, bias=None, divisor=None):
        if divisor is None:
            divisor = ((labels >= 0) & (labels < weight.shape[0])).sum().clamp(min=1)
        return _mean(features, weight, labels, divisor)


def _worker(rank, world, port, q):
    for p in (ROOT, PKG):
        if p not in sys.path:
            sys.path.insert(0, p)
    import torch.distributed as dist
    from retinahead import dist as rdist, functional as F, _lib
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    x, w, y = _batch()
    lo, hi = rdist.shard_bounds(len(y), rank, world)
    x, w = x[lo:hi].requires_grad_(True), w.requires_grad_(True)
    loss = rdist.DataParallelLinearCrossEntropy(_Loss())(x, w, y[lo:hi])
    loss.backward()

    def grad_clip(tensors, max_norm=None, norm_type=2.0, stages=_lib.CLIP_ALL, out=None, grads=False):
        values = [t.grad for t in tensors if t.grad is not None]
        if not values:
            return None
        flat = torch.cat(values).double()
        if out is None:
            out = {"total": ((flat ** 2).sum() if norm_type == 2.0 else flat.abs().max()).reshape(1)}
        if stages & _lib.CLIP_SCALE:
            norm = out["total"].sqrt() if norm_type == 2.0 else out["total"]
            out["norm"] = norm.float().reshape(())
            for t in values:
                t.mul_(float(min(1.0, max_norm / (float(norm) + 1e-6))))
        return out

    F.grad_clip = grad_clip
    clipped = {}
    for norm in (2.0, float("inf")):
        params = [torch.nn.Parameter(torch.zeros(3)) for _ in range(2)] if rank == 0 else []      # others: none
        for i, p in enumerate(params):
            p.grad = torch.tensor([1.0, -2.0, 2.0]) * (i + 1)
        clipped[norm] = (float(rdist.clip_grad_norm_(params, 1.0, norm_type=norm)), [p.grad.tolist() for p in params])
    p = torch.nn.Parameter(torch.zeros(1))
    p.grad = torch.tensor([float("nan") if rank else 3.0])
    bad = float(rdist.clip_grad_norm_([p], 1.0, norm_type=float("inf")))
    with pytest.raises(RuntimeError, match="not finite"):
        rdist.clip_grad_norm_([p], 1.0, norm_type=float("inf"), error_if_nonfinite=True)
    q.put((rank, float(loss), x.grad.tolist(), w.grad.tolist(), clipped, bad))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_share_the_count_and_the_norm(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=120) for _ in range(world)], key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    x, w, y = _batch()
    x.requires_grad_(True), w.requires_grad_(True)
    want = _mean(x, w, y, 6.0)
    want.backward()
    for rank, loss, _, _, clipped, bad in res:
        assert abs(loss - float(want.detach())) <= 1e-6 * float(want.detach())      # the count and the value pass through float32
        norm = 45.0 ** 0.5
        assert abs(clipped[2.0][0] - norm) <= 1e-6 * norm and clipped[float("inf")][0] == 4.0
        assert bad != bad
        if rank == 0:
            assert torch.allclose(torch.tensor(clipped[2.0][1]) * norm, torch.tensor([[1.0, -2, 2], [2, -4, 4]]), rtol=1e-5)
    assert torch.allclose(torch.cat([torch.tensor(r[2], dtype=torch.float64) for r in res]), x.grad, rtol=1e-6, atol=1e-9)
    assert torch.allclose(sum(torch.tensor(r[3], dtype=torch.float64) for r in res), w.grad, rtol=1e-6, atol=1e-9)


def test_wrapper_refuses_a_sum():
    import retinahead as rh
    from retinahead import dist as rdist
    with pytest.raises(ValueError, match="sum"):
        rdist.DataParallelLinearCrossEntropy(rh.LinearCrossEntropy(reduction="sum"))
    labels = torch.tensor([3, 0, -100, -1, 7])
    assert float(rdist.count_valid(labels, 7)) == 2.0 and float(rdist.count_valid(labels, 7, ignore_index=3)) == 1.0
