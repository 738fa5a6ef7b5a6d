"""What the gradient norm and clipping refuse, and their host-side logic (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest
import torch

import retinahead as rh
from retinahead import _lib


def test_refuses_host_tensors_and_values():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(rh.RetinaHeadError, match="HIP device"):
        rh.clip_grad_norm_([p], 1.0)
    with pytest.raises(rh.RetinaHeadError, match="HIP device"):
        rh.grad_norm(p.grad)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            rh.clip_grad_norm_([p], bad)
    with pytest.raises(ValueError, match="norm_type"):
        rh.clip_grad_norm_([p], 1.0, norm_type=0.5)
    assert float(rh.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0
    assert float(rh.grad_norm([])) == 0.0
    with pytest.raises(rh.RetinaHeadError, match="list of tensors"):
        rh.grad_norm([1.0])
    with pytest.raises(TypeError):
        rh.grad_norm(3)


REF = np.dtype([("data", np.uint64), ("count", np.int64), ("dtype", np.int32), ("reserved", np.int32)])


def _refs(*items):
    assert REF.itemsize == C.sizeof(_lib.TensorRef)
    a = np.zeros(len(items), REF)
    for i, it in enumerate(items):
        a[i] = tuple(it) + (0,)
    return a


def _args(refs, **kw):
    a = _lib.GradClipArgs(refs.ctypes.data, len(refs), 0, _lib.CLIP_ALL, 1.0, 4096, 8192, 16384, 1 << 20)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("items,kw,code,text", [
    ([(4096, 4, 3)], {}, -1, "element type"),
    ([(4096, -1, 0)], {}, -2, "element count"),
    ([(0, 4, 0)], {}, -1, "null pointer"),
    ([(4098, 4, 0)], {}, -5, "aligned"),
    ([(4097, 4, 1)], {}, -5, "aligned"),
    ([(4096, 100, 0), (4096, 100, 0)], {}, -1, "share memory"),
    ([(8192, 100, 0), (4096, 1025, 0)], {}, -1, "share memory"),
    ([(4096, 4, 0)], dict(stages=0), -1, "stages"),
    ([(4096, 4, 0)], dict(stages=4), -1, "stages"),
    ([(4096, 4, 0)], dict(norm_type=3), -1, "norm"),
    ([(4096, 4, 0)], dict(total=None), -1, "null"),
    ([(4096, 4, 0)], dict(workspace_bytes=8), -4, "workspace"),
    ([(4096, 4, 0)], dict(workspace=None), -4, "workspace"),
    ([(4096, 4, 0)], dict(workspace=16400), -5, "256"),
])
def test_entry_point_refuses(items, kw, code, text):
    refs = _refs(*items)
    assert rh.load_library().rh_grad_clip(C.byref(_args(refs, **kw)), None) == code
    assert text in _lib.last_error()


def test_workspace_query():
    q = rh.load_library().rh_grad_clip_workspace_bytes
    one = _refs((4096, 5, 0))
    assert q(one.ctypes.data, 1) == 256 and q(None, 0) == 256
    assert q(None, 1) == 0 and q(one.ctypes.data, -1) == 0
    big = _refs((4096, 1 << 34, 0))
    assert q(big.ctypes.data, 1) < 1 << 20


def test_refuses_tangents():
    """Forward-mode differentiation has no rule here: a tangent must not count as zero."""
    import torch.autograd.forward_ad as forward_ad
    p = torch.nn.Parameter(torch.ones(4))
    with forward_ad.dual_level():
        p.grad = forward_ad.make_dual(torch.ones(4), torch.ones(4))
        with pytest.raises(rh.RetinaHeadError, match="forward-mode"):
            rh.grad_norm(p.grad)
        with pytest.raises(rh.RetinaHeadError, match="forward-mode"):
            rh.clip_grad_norm_([p], 1.0)


def test_stages_refuse_what_they_cannot_use():
    F = rh.functional
    p = torch.ones(4)
    with pytest.raises(ValueError, match="as out"):      # its total would be anything
        F.grad_clip([p], 1.0, stages=_lib.CLIP_SCALE)
    total, norm = torch.ones(1, dtype=torch.float64), torch.ones(())
    for out in (dict(total=total.float(), norm=norm), dict(total=total, norm=norm.double()),
                dict(total=total.expand(2), norm=norm)):
        with pytest.raises(ValueError, match="one float64 total"):
            F.grad_clip([p], 1.0, stages=_lib.CLIP_SCALE, out=out)
