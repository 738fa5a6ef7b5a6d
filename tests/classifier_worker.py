"""One rank of the multi-process test of the classifier loss and the sharded gradient norm
(tests/test_gpu_classifier_ranks.py): started as a fresh process, writes its results to an .npz file.

  python tests/classifier_worker.py RANK WORLD PORT OUT.npz
"""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "pytorch-retinanet_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

ROWS, FEATURES, CLASSES = 75, 64, 90


def batch(torch):
    """The whole batch, the same on every rank: the second rank's shard has other counts than the first's."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(ROWS, FEATURES, generator=g), torch.randn(CLASSES, FEATURES, generator=g) * 0.2
    y, b = torch.randint(0, CLASSES, (ROWS,), generator=g), torch.randn(CLASSES, generator=g) * 0.1
    y[50:70] = -100
    return x, w, y, b


def gradients(torch):
    g = torch.Generator().manual_seed(6)
    return [torch.randn(n, generator=g) for n in (7, 1000, 33, 4096)]


def main():
    rank, world, port, out_path = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3], sys.argv[4]
    import torch
    import torch.distributed as dist
    import retinahead as rh
    from retinahead import dist as rdist

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = port
    dist.init_process_group("gloo", rank=rank, world_size=world)
    dev = torch.device("cuda", 0)
    x, w, y, b = batch(torch)
    lo, hi = rdist.shard_bounds(ROWS, rank, world)
    res = {"bounds": np.array([lo, hi])}
    x, w, b = (t.to(dev).requires_grad_(True) for t in (x[lo:hi], w, b))
    mod = rdist.DataParallelLinearCrossEntropy(rh.LinearCrossEntropy())
    for step in range(2):
        x.grad = w.grad = b.grad = None
        loss = mod(x, w, y[lo:hi].to(dev), b)
        loss.backward()
        res[f"loss{step}"] = loss.detach().cpu().numpy()
        for name, t in (("d_features", x), ("d_weight", w), ("d_bias", b)):
            res[f"{name}{step}"] = t.grad.cpu().numpy()
    # an empty shard still takes part
    empty = mod(x[:0] if rank else x, w, (y[lo:hi][:0] if rank else y[lo:hi]).to(dev), b)
    res["loss_of_first"] = empty.detach().cpu().numpy()
    # every other gradient on every other rank; then all of them on the first
    for kind, share in (("half", lambda i: i % world == rank), ("all", lambda i: rank == 0)):
        for norm in (2.0, 1.0, float("inf")):
            grads = [t for i, t in enumerate(gradients(torch)) if share(i)]
            params = [torch.nn.Parameter(torch.zeros_like(t, device=dev)) for t in grads]
            for p, t in zip(params, grads):
                p.grad = t.to(dev)
            total = rdist.clip_grad_norm_(params, 0.5, norm_type=norm)
            res[f"norm_{kind}_{norm}"] = np.array([float(total)])
            for i, p in enumerate(params):
                res[f"grad_{kind}_{norm}_{i}"] = p.grad.cpu().numpy()
    p = torch.nn.Parameter(torch.zeros(4, device=dev))
    p.grad = torch.full((4,), float("nan") if rank else 1.0, device=dev)
    res["nan"] = np.array([float(rdist.clip_grad_norm_([p], 0.5, norm_type=float("inf")))])
    res["nan_grad"] = p.grad.cpu().numpy()
    np.savez(out_path, **res)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
