"""DataParallelLinearCrossEntropy and dist.clip_grad_norm_ under two ranks on one GPU (gloo, fresh
processes), against 64 bits on the whole batch."""
import os
import socket
import subprocess
import sys

import numpy as np
import pytest
import torch

import classifier_worker as worker
from test_gpu_classifier import close, oracle

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def _run_ranks(world, tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = str(s.getsockname()[1])
    outs = [str(tmp_path / f"rank{r}.npz") for r in range(world)]
    env = dict(os.environ, HSA_ENABLE_IPC_MODE_LEGACY="0")
    procs = [subprocess.Popen([sys.executable, os.path.join(HERE, "classifier_worker.py"), str(r), str(world), port,
                               outs[r]], env=env) for r in range(world)]
    try:
        codes = [p.wait(timeout=90) for p in procs]
    except subprocess.TimeoutExpired:
        for p in procs:
            p.kill()
        raise
    assert codes == [0] * world, codes
    return [np.load(o) for o in outs]


def test_two_ranks(tmp_path):
    res = _run_ranks(2, tmp_path)
    x, w, y, b = worker.batch(torch)
    count = float((y != -100).sum())
    whole = oracle(x, w, y, b)
    shards = [oracle(x[lo:hi], w, y[lo:hi], b, divisor=count) for lo, hi in (r["bounds"] for r in res)]
    for r, shard in zip(res, shards):
        for step in (0, 1):
            close("loss", torch.from_numpy(r[f"loss{step}"]), whole["loss"])
            for k in ("d_features", "d_weight", "d_bias"):
                close(k, torch.from_numpy(r[f"{k}{step}"]), shard[k])
        lo, hi = res[0]["bounds"]
        close("loss", torch.from_numpy(r["loss_of_first"]), oracle(x[lo:hi], w, y[lo:hi], b)["loss"])
    # the shards' bounds add up: the whole batch's gradients are the ranks' sum
    summed = sum(torch.from_numpy(r["d_weight0"]).double() for r in res)
    assert ((summed - whole["d_weight"][0]).abs() <= sum(s["d_weight"][1] for s in shards)).all()

    grads = worker.gradients(torch)
    flat = torch.cat(grads).double()
    for norm in (2.0, 1.0, float("inf")):
        want = float(torch.linalg.vector_norm(flat, norm))
        factor = min(1.0, 0.5 / (want + 1e-6))
        for kind in ("half", "all"):
            for rank, r in enumerate(res):
                # summed in 64 bits, rounded once to float32
                assert abs(float(r[f"norm_{kind}_{norm}"][0]) - want) <= 2.0 ** -23 * want
                mine = [t for i, t in enumerate(grads) if (i % 2 == rank if kind == "half" else rank == 0)]
                for i, t in enumerate(mine):
                    got = torch.from_numpy(r[f"grad_{kind}_{norm}_{i}"]).double()
                    # the factor (norm + 1e-6, division, product: a rounding each) on float32 values
                    assert ((got - t.double() * factor).abs() <= 2.0 ** -22 * t.double().abs() * factor).all()
    for r in res:       # a NaN on one rank is everyone's
        assert np.isnan(r["nan"][0]) and np.isnan(r["nan_grad"]).all()
