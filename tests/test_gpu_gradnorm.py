"""The global gradient norm and clipping (retinahead.grad_norm, clip_grad_norm_) against 64 bits.

Bounds.  Squares, magnitudes and their sums are float64 (relative error of a sum of N positive terms:
below N 2^-52), the norm is rounded to float32 once: 2^-24, and 2^-23 covers both.  The factor c takes a
float32 addition and a division on top: (2^-23 + 2 * 2^-24) = 2^-22; a scaled value one rounding to its
type more, and half the type's smallest step where it is that small.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NORMS = [2.0, 1.0, math.inf]


@pytest.fixture(scope="module")
def rh():
    import retinahead
    retinahead.load_library()
    return retinahead


def norm64(ts, p):
    flat = torch.cat([t.detach().double().reshape(-1) for t in ts])
    if flat.numel() == 0:
        return 0.0
    return float(flat.abs().max() if p == math.inf else flat.abs().pow(p).sum().pow(1.0 / p))


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


def check_clip(rh, grads, max_norm, p):
    want = norm64(grads, p)
    before = [g.clone() for g in grads]
    got = rh.clip_grad_norm_(params_of(grads), max_norm, norm_type=p)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    c = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        if max_norm / (want + 1e-6) >= 1.0 + 2.0 ** -22:
            assert torch.equal(g, b)
            continue
        exact = b.double() * c
        f = torch.finfo(g.dtype)
        tol = exact.abs() * (f.eps / 2 + 2.0 ** -22) + f.smallest_normal * f.eps / 2
        assert ((g.double() - exact).abs() <= tol).all()


def rand(n, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, generator=g) * scale).to(TYPES[dtype]).cuda()


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sizes", [[1], [7], [0, 3, 0], [8192], [8191, 8193, 16384, 16385], [64] * 170 + [5] * 170,
                                   [1_000_003, 2, 77], [9_000_000]])
def test_sizes(rh, dtype, sizes, p):
    grads = [rand(n, dtype, i) for i, n in enumerate(sizes)]
    assert abs(float(rh.grad_norm(grads, p)) - norm64(grads, p)) <= 2.0 ** -23 * norm64(grads, p)
    check_clip(rh, grads, 0.1, p)


@pytest.mark.parametrize("p", NORMS)
def test_mixed_types_at_any_address(rh, p):
    """Views back to back in flat buffers; what lies around and between them stays as it was."""
    grads, guards = [], []
    for i, dtype in enumerate(list(TYPES) * 4):
        buf = rand(70000, dtype, 100 + i)
        at = 1 + i
        for n in (1, 3, 8, 40001 + i, 9):
            grads.append(buf[at:at + n])
            at += n + (i % 2)
        mask = torch.ones(70000, dtype=torch.bool, device="cuda")
        a = 1 + i
        for n in (1, 3, 8, 40001 + i, 9):
            mask[a:a + n] = False
            a += n + (i % 2)
        guards.append((buf, mask, buf.clone()))
    check_clip(rh, grads, 1.0, p)
    for buf, mask, was in guards:
        assert torch.equal(buf[mask], was[mask])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_not_clipped_below_the_bound(rh, dtype):
    grads = [rand(1000, dtype, 1), rand(50001, dtype, 2)]
    check_clip(rh, grads, 1e6, 2.0)
    check_clip(rh, grads, math.inf, 2.0)
    check_clip(rh, grads, 0.0, 2.0)
    zero = [torch.zeros(100, dtype=TYPES[dtype], device="cuda")]
    check_clip(rh, zero, 1.0, 2.0)


def test_matches_torch_on_a_model(rh):
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.ReLU(), torch.nn.Conv2d(16, 24, 3), torch.nn.Flatten(),
                              torch.nn.Linear(24 * 144, 10)).cuda().to(memory_format=torch.channels_last)
    net(torch.randn(4, 3, 16, 16, device="cuda")).square().sum().backward()
    net[0].bias.grad = None
    mine = [None if p.grad is None else p.grad.clone(memory_format=torch.preserve_format) for p in net.parameters()]
    want = torch.nn.utils.clip_grad_norm_(net.parameters(), 0.1)
    theirs = [p.grad for p in net.parameters()]
    for p, g in zip(net.parameters(), mine):
        p.grad = g
    got = rh.clip_grad_norm_(net.parameters(), 0.1)
    assert torch.allclose(got, want, rtol=1e-5)      # torch sums in float32
    for g, t in zip(mine, theirs):
        assert g is None and t is None or torch.allclose(g, t, rtol=1e-5, atol=0)


def test_far_values(rh):
    """Squares that leave float32: sums in 64 bits."""
    for v in (1e30, 1e-30):
        g = [torch.full((3000,), v, device="cuda"), torch.full((77,), v, device="cuda", dtype=torch.bfloat16)]
        check_clip(rh, g, 1.0, 2.0)
    top = [torch.full((100,), torch.finfo(torch.float32).max, device="cuda")]
    assert float(rh.grad_norm(top)) == math.inf
    assert float(rh.grad_norm(top, math.inf)) == torch.finfo(torch.float32).max


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_nan_and_inf(rh, dtype, p):
    for bad in (math.nan, math.inf, -math.inf):
        a, b = rand(20000, dtype, 3), rand(33, dtype, 4)
        a[11111] = bad
        if bad != bad:
            b[3] = math.inf
        t, kept = [x.clone() for x in (a, b)], [x.clone() for x in (a, b)]
        got = rh.clip_grad_norm_(params_of([a, b]), 1.0, norm_type=p)
        if bad != bad:
            assert math.isnan(float(got)) and torch.isnan(a).all() and torch.isnan(b).all()
        else:
            assert float(got) == math.inf
            assert torch.isnan(a[11111]) and (b == 0).all() and (a[:11111] == 0).all()
        with pytest.raises(RuntimeError, match="not finite"):
            rh.clip_grad_norm_(params_of(t), 1.0, norm_type=p, error_if_nonfinite=True)
        for x, k in zip(t, kept):      # refused before anything was scaled
            assert torch.equal(x.nan_to_num(7.0), k.nan_to_num(7.0))
    good = [rand(100, dtype, 5)]
    want = norm64(good, p)
    assert abs(float(rh.clip_grad_norm_(params_of(good), 0.5, p, error_if_nonfinite=True)) - want) <= 2.0 ** -23 * want


def test_orders_of_dimensions_and_refusals(rh):
    base = rand(2 * 3 * 5 * 7, "f32", 6)
    x = base.view(2, 3, 5, 7)
    for g in (x, x.clone().permute(3, 1, 0, 2), x.clone().to(memory_format=torch.channels_last), x.clone()[:, :, :, None]):
        check_clip(rh, [g], 0.1, 2.0)
    with pytest.raises(rh.RetinaHeadError, match="fill their memory"):
        rh.grad_norm([rand(100, "f32", 7)[::2]])
    with pytest.raises(rh.RetinaHeadError, match="fill their memory"):
        rh.grad_norm([rand(1, "f32", 7).expand(5)])
    with pytest.raises(rh.RetinaHeadError, match="sparse"):
        rh.grad_norm([torch.eye(3, device="cuda").to_sparse()])
    with pytest.raises(rh.RetinaHeadError, match="float32, bfloat16 or float16"):
        rh.grad_norm([torch.zeros(3, device="cuda", dtype=torch.float64)])
    g = rand(100, "f32", 8)
    keep = g.clone()
    for pair in ([g, g], [g[:60], g[50:]]):
        with pytest.raises(rh.RetinaHeadError, match="share memory"):
            rh.clip_grad_norm_(params_of(pair), 0.1)
    assert torch.equal(g, keep)
    assert abs(float(rh.grad_norm([g, g])) - norm64([g, g], 2.0)) <= 2.0 ** -23 * norm64([g, g], 2.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            rh.clip_grad_norm_(params_of([g]), bad)
    with pytest.raises(ValueError, match="norm_type"):
        rh.grad_norm([g], 3.0)
    assert float(rh.grad_norm([])) == 0.0 and float(rh.clip_grad_norm_([torch.nn.Parameter(g)], 1.0)) == 0.0


def test_repeats_and_streams_agree(rh):
    grads = [rand(300_001, "bf16", i) for i in range(20)]
    first = rh.grad_norm(grads)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s):
            a = rh.grad_norm(grads)
        b = rh.grad_norm(grads)
        torch.cuda.synchronize()
        assert torch.equal(a, first) and torch.equal(b, first)


def test_captured(rh):
    grads = [rand(n, d, 9) for n, d in ((70001, "f32"), (33, "bf16"), (5000, "f16"))]
    params = params_of(grads)
    rh.clip_grad_norm_(params, 1e9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = rh.clip_grad_norm_(params, 0.5)
    for seed in range(4):
        new = [rand(g.numel(), d, 50 + seed, 1.0 + seed) for g, d in zip(grads, ("f32", "bf16", "f16"))]
        for g, n in zip(grads, new):
            g.copy_(n)
        graph.replay()
        eager = [n.clone() for n in new]
        want = rh.clip_grad_norm_(params_of(eager), 0.5)
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        for g, e in zip(grads, eager):
            assert torch.equal(g, e)


# ------------------------------------------------------------------ the operators as a training step uses them
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_training_step_of_a_classifier(rh, dtype):
    """Projection loss, backward, clipping, a plain update: every step against 64 bits on the same weights."""
    from test_gpu_classifier import close, make, oracle
    x, w, y, b = make(200, 96, 700, dtype, True, ignored=0.2, seed=30)
    pw, pb = torch.nn.Parameter(w.clone()), torch.nn.Parameter(b.clone())
    fn = rh.LinearCrossEntropy()
    losses = []
    for step in range(3):
        xin = x.clone().requires_grad_(True)
        pw.grad = pb.grad = None
        loss = fn(xin, pw, y, pb)
        loss.backward()
        want = oracle(x, pw.detach(), y, pb.detach())
        for k, g in (("d_features", xin.grad), ("d_weight", pw.grad), ("d_bias", pb.grad)):
            close(k, g, want[k])
        raw = [pw.grad.clone(), pb.grad.clone()]
        norm = rh.clip_grad_norm_([pw, pb], 0.05)
        exact = norm64(raw, 2.0)
        assert abs(float(norm) - exact) <= 2.0 ** -23 * exact
        c = min(1.0, 0.05 / (exact + 1e-6))
        for g, r in zip((pw.grad, pb.grad), raw):
            f = torch.finfo(g.dtype)
            tol = (r.double() * c).abs() * (f.eps / 2 + 2.0 ** -22) + f.smallest_normal * f.eps / 2
            assert ((g.double() - r.double() * c).abs() <= tol).all()
        with torch.no_grad():
            pw -= pw.grad
            pb -= pb.grad
        losses.append(float(loss.detach()))
    assert all(math.isfinite(v) for v in losses)


def test_tensor_larger_than_an_entry_of_the_table(rh):
    n = (1 << 30) + (1 << 29) + 12345
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    g[-1] = 3.0
    want = math.sqrt((n - 1) * 0.25 + 9.0)
    got = rh.clip_grad_norm_(params_of([g]), 100.0)
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    scaled = torch.tensor(0.5 * (100.0 / (want + 1e-6)), dtype=torch.float64)
    assert (g[:-1] == g[0]).all() and abs(float(g[0]) - float(scaled)) <= 2.0 ** -8 * float(scaled)
    assert abs(float(g[-1]) - 6.0 * float(scaled)) <= 2.0 ** -8 * 6.0 * float(scaled)


def test_sharded_stages(rh):
    """The two stages apart, with a sum over ranks put between them."""
    F = rh.functional
    from retinahead import _lib
    a = [rand(1000, "f32", 40), rand(33, "bf16", 41)]
    other = [rand(500, "f16", 42)]
    both = norm64(a + other, 2.0)
    out = F.grad_clip(a, stages=_lib.CLIP_NORM)
    out["total"] += F.grad_clip(other, stages=_lib.CLIP_NORM)["total"]
    before = [t.clone() for t in a]
    F.grad_clip(a, 1.0, stages=_lib.CLIP_SCALE, out=out)
    assert abs(float(out["norm"]) - both) <= 2.0 ** -23 * both
    for t, b in zip(a, before):
        exact = b.double() * (1.0 / (both + 1e-6))
        assert ((t.double() - exact).abs() <= exact.abs() * (torch.finfo(t.dtype).eps / 2 + 2.0 ** -22)).all()


@pytest.mark.parametrize("p,total,norm", [(2.0, 9.0, 3.0), (1.0, 5.0, 5.0), (math.inf, 7.0, 7.0)])
def test_scaling_of_empty_tensors_writes_the_norm(rh, p, total, norm):
    """A rank whose shards are all of size 0 has the norm that the ranks' totals make."""
    from retinahead import _lib
    from retinahead.modules import _clip
    F = rh.functional
    empty = [torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda", dtype=torch.bfloat16)]
    out = F.grad_clip(empty, norm_type=p, stages=_lib.CLIP_NORM)
    assert float(out["norm"]) == 0.0 and float(out["total"]) == 0.0
    out["total"].fill_(total)
    F.grad_clip(empty, 1.0, p, stages=_lib.CLIP_SCALE, out=out)
    assert float(out["norm"]) == norm and float(out["total"]) == total
    got = _clip(params_of(empty), 1.0, p, False, lambda t: t.add_(total))      # as the ranks' reduction adds to it
    assert float(got) == norm
    assert float(rh.clip_grad_norm_(params_of(empty), 1.0, p, error_if_nonfinite=True)) == 0.0
    assert float(rh.clip_grad_norm_(params_of(empty), 1.0, p)) == 0.0


@pytest.mark.parametrize("p", [2.0, 1.0])
def test_a_norm_beyond_float32_is_not_finite(rh, p):
    """It is infinity where it clips, so that is what error_if_nonfinite asks about."""
    top = torch.finfo(torch.float32).max
    g = torch.full((100,), top, device="cuda")
    kept = g.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        rh.clip_grad_norm_(params_of([g]), 1.0, p, error_if_nonfinite=True)
    assert torch.equal(g, kept)
    one = g[:1].clone()      # the largest that is finite
    assert float(rh.clip_grad_norm_(params_of([one]), math.inf, p, error_if_nonfinite=True)) == top
    assert float(rh.clip_grad_norm_(params_of([g]), 1.0, p)) == math.inf and (g == 0).all()


@pytest.mark.parametrize("p", NORMS)
def test_the_factor_is_rounded_once(rh, p):
    """min(1, max_norm / (norm + 1e-6)) in 64 bits, then to float32 (2^-24), times a float32 value (2^-24); the norm's
    own 64-bit sums are granted 2^-40."""
    for seed in range(24):
        g = rand(3001 + seed, "f32", 60 + seed, 1.0 + seed)
        was = g.double()
        c = 0.125 / (norm64([g], p) + 1e-6)
        rh.clip_grad_norm_(params_of([g]), 0.125, p)
        off = ((g.double() - was * c).abs() / (was.abs() * c).clamp(min=1e-30)).max()
        assert float(off) <= 2.0 ** -23 + 2.0 ** -40, seed


def test_scaling_refuses_an_out_of_the_host(rh):
    from retinahead import _lib
    g = rand(100, "f32", 90)
    kept = g.clone()
    with pytest.raises(rh.RetinaHeadError, match="HIP device"):
        rh.functional.grad_clip([g], 1.0, stages=_lib.CLIP_SCALE,
                                out=dict(total=torch.ones(1, dtype=torch.float64), norm=torch.ones(())))
    assert torch.equal(g, kept)
