"""What the classifier loss refuses, and its host-side sizes (no GPU needed)."""
import ctypes as C

import pytest
import torch

import retinahead as rh
from retinahead import _lib
from retinahead import functional as F


def _call(**kw):
    a = dict(features=torch.zeros(4, 8), weight=torch.zeros(5, 8), labels=torch.zeros(4, dtype=torch.int64),
             bias=torch.zeros(5))
    a.update(kw)
    return F.linear_cross_entropy(**a)


def test_refuses_host_tensors():
    with pytest.raises(rh.RetinaHeadError, match="HIP device"):
        _call()


@pytest.mark.parametrize("kw,error,text", [
    (dict(features=torch.zeros(4, 8, dtype=torch.float64)), rh.RetinaHeadError, "float32, bfloat16 or float16"),
    (dict(weight=torch.zeros(5, 8, dtype=torch.bfloat16)), rh.RetinaHeadError, "one element type"),
    (dict(bias=torch.zeros(5, dtype=torch.float16)), rh.RetinaHeadError, "one element type"),
    (dict(weight=torch.zeros(5, 7)), rh.RetinaHeadError, "expected features"),
    (dict(weight=torch.zeros(8)), rh.RetinaHeadError, "expected features"),
    (dict(labels=torch.zeros(3, dtype=torch.int64)), rh.RetinaHeadError, "labels must have"),
    (dict(labels=torch.zeros(4)), rh.RetinaHeadError, "int64 or int32"),
    (dict(bias=torch.zeros(4)), rh.RetinaHeadError, "bias must be"),
    (dict(weight=torch.zeros(0, 8), bias=None), rh.RetinaHeadError, "at least one class"),
    (dict(reduction="none"), ValueError, "reduction"),
    (dict(divisor=torch.ones(2)), rh.RetinaHeadError, "divisor"),
    (dict(expected_grad=0.0), ValueError, "expected_grad"),
])
def test_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        _call(**kw)


def test_module_refuses():
    with pytest.raises(ValueError):
        rh.LinearCrossEntropy(reduction="none")
    with pytest.raises(ValueError):
        rh.LinearCrossEntropy(expected_grad=0)


def test_workspace_query():
    lib = rh.load_library()
    q = lib.rh_linear_ce_workspace_bytes
    full = _lib.CE_GRAD_X | _lib.CE_GRAD_W | _lib.CE_GRAD_B
    assert q(0, 8, 5, 0, 0) == 0 and "rows" in _lib.last_error()
    assert q(4, 0, 5, 0, 0) == 0 and "features" in _lib.last_error()
    assert q(4, 8, 0, 0, 0) == 0 and "classes" in _lib.last_error()
    assert q(4, 8, 5, 3, 0) == 0 and "element type" in _lib.last_error()
    assert 0 < q(400, 8, 500, 0, 0) < q(400, 8, 500, 0, full)
    assert 0 < q(400, 8, 500, 1, 0) < q(400, 8, 500, 1, full) < q(400, 8, 500, 1, full | _lib.CE_COPY_WEIGHT)
    assert 0 < q(4, 8, 5, 0, 0) < q(4, 8, 5, 0, full)
    # the logits of this call would take 8 GiB in 16 bits
    assert q(1 << 15, 1024, 1 << 17, _lib.RH_BF16, full) < 3 << 30


def _args(**kw):
    host = torch.zeros(1 << 16, dtype=torch.uint8)       # never read: every call below is refused
    at = (host.data_ptr() + 255) // 256 * 256
    a = _lib.LinearCeArgs()
    for k in ("x", "w", "labels", "row_loss", "small", "workspace"):
        setattr(a, k, at)
    a.n, a.v, a.d, a.ldx, a.ldw, a.grad, a.workspace_bytes = 4, 5, 8, 8, 8, 1.0, 1 << 30
    for k, v in kw.items():
        setattr(a, k, at + 4 if v == "unaligned" else at if v == "there" else v)
    return a, host


@pytest.mark.parametrize("kw,code,text", [
    (dict(x=None), -1, "null"),
    (dict(reduction=2), -1, "reduction"),
    (dict(dtype=7), -1, "element type"),
    (dict(db="there"), -1, "bias"),
    (dict(n=0), -2, "rows"),
    (dict(ldx=7), -2, "stride"),
    (dict(ldw=7), -2, "stride"),
    (dict(w="unaligned"), -5, "RH_CE_COPY_WEIGHT"),
    (dict(d=7), -5, "RH_CE_COPY_WEIGHT"),
    (dict(dw="unaligned"), -5, "gradients"),
    (dict(workspace_bytes=16), -4, "workspace"),
    (dict(workspace=None), -4, "workspace"),
    (dict(workspace="unaligned"), -5, "256"),
])
def test_entry_point_refuses(kw, code, text):
    a, host = _args(**kw)
    assert rh.load_library().rh_linear_ce(C.byref(a), None) == code
    assert text in _lib.last_error()


def test_scale_gradient_refuses():
    lib = rh.load_library()
    assert lib.rh_scale_gradient(None, 4, 0, None, 1.0, None) == -1
    assert lib.rh_scale_gradient(None, -1, 0, None, 1.0, None) == -2
    assert lib.rh_scale_gradient(None, 4, 0, None, 0.0, None) == -1
    assert lib.rh_scale_gradient(None, 0, 0, None, 1.0, None) == 0


@pytest.mark.parametrize("which", ["features", "weight", "bias", "divisor"])
def test_refuses_tangents(which):
    """Forward-mode differentiation has no rule here: a tangent must not count as zero."""
    import torch.autograd.forward_ad as forward_ad
    args = dict(features=torch.ones(4, 8), weight=torch.ones(5, 8), labels=torch.zeros(4, dtype=torch.int64),
                bias=torch.ones(5), divisor=torch.ones(1))
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(rh.RetinaHeadError, match="forward-mode"):
            F.linear_cross_entropy(**args)
        with pytest.raises(rh.RetinaHeadError, match="forward-mode"):
            rh.LinearCrossEntropy()(**args)


@pytest.mark.parametrize("n,d,v", [(49104, 256, 601), (850_176, 24, 600), (100_000, 512, 512)])
def test_workspace_of_whole_rows(n, d, v):
    """The placed features, P, the places and the sums of columns: nothing of what the logits by tiles need."""
    q = rh.load_library().rh_linear_ce_workspace_bytes
    columns = (v + 63) // 64 * 64
    p, x, rows = n * columns * 2, n * ((d + 31) // 32 * 64), n * 12 + n
    sums = (n + 63) // 64 * v * 4
    got = q(n, d, v, _lib.RH_BF16, _lib.CE_GRAD_X | _lib.CE_GRAD_B)
    assert got <= p + x + rows + sums + (1 << 20), (got, p, x, rows, sums)
