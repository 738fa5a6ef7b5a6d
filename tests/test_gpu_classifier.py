"""The softmax classifier loss over a large label set (retinahead.LinearCrossEntropy) against a plain
64-bit implementation, element by element, with bounds derived from the arithmetic.

Bounds.  Let e = 2^-23 (a float32 operation is off by at most 2^-24 of its result; the matrix units'
internal additions are granted twice that) and u = eps/2 of the element type.
  logits      |dz| <= (D + 1) e sum_i |x_i w_i| + e |b|      =: Z (its largest over the classes of a row)
  lse         a sum of positive terms, each off by its exponent's error, its exp and V additions (pairwise
              within tiles, but V e bounds any order):  |d lse| <= Z + (V + 16) e + e (|max| + |lse|)
  row loss    Z + |d lse| + e |row|
  P           |dP| <= p (exp(Z + |d lse| + 8 e + 4 e |z - lse| + k) - 1) + e + u |P|
              (the e: p - 1 in float32, and what is so far below its row's largest that it counts as 0;
              k: half a step of the kept logit, 2^-12 for bfloat16 and 2^-13 for float16)
  dX = s P W  s (|dP| |W| + (V + 2) e |P| |W|) + (u + 2 e) |dX| + half the type's smallest step
and dW, db in the same way over the rows.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -23


@pytest.fixture(scope="module")
def rh():
    import retinahead
    retinahead.load_library()
    return retinahead


def make(n, d, v, dtype, bias, ignored=0.0, seed=0, scale=2.0, label_type=torch.int64):
    g = torch.Generator().manual_seed(seed * 1009 + n * 7 + d * 3 + v)
    w = (torch.randn(v, d, generator=g) * scale / math.sqrt(d)).to(TYPES[dtype])
    y = torch.randint(0, v, (n,), generator=g)
    x = torch.randn(n, d, generator=g)
    x[::2] += 1.5 * w[y[::2]].float()
    x = x.to(TYPES[dtype])
    if ignored:
        y[torch.rand(n, generator=g) < ignored] = -100
    b = (torch.randn(v, generator=g) * 0.5).to(TYPES[dtype]) if bias else None
    return x.cuda(), w.cuda(), y.to(label_type).cuda(), None if b is None else b.cuda()


def oracle(x, w, y, b, reduction="mean", upstream=1.0, divisor=None, ignore=-100):
    """Results in 64 bits and the bound of each (see the module's docstring)."""
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    u = torch.finfo(x.dtype).eps / 2
    n, d = x.shape
    v = w.shape[0]
    keep = (y != ignore) & (y >= 0) & (y < v)
    X = torch.where(keep[:, None], x, torch.zeros_like(x)).double()
    W, Y = w.double(), torch.where(keep, y, 0).long()
    z = X @ W.T
    Z = X.abs() @ W.abs().T * ((d + 1) * E)
    if b is not None:
        z = z + b.double()
        Z = Z + E * b.double().abs()
    Z = Z.amax(1, keepdim=True) + E * z.abs()
    lse = torch.logsumexp(z, 1, keepdim=True)
    zy = z.gather(1, Y[:, None])
    dlse = Z.amax(1, keepdim=True) + (v + 16) * E + E * (z.amax(1, keepdim=True).abs() + lse.abs())
    row = torch.where(keep, (lse - zy)[:, 0], 0.0)
    drow = torch.where(keep, (Z.gather(1, Y[:, None]) + dlse)[:, 0] + E * row.abs(), 0.0)
    count = float(keep.sum())
    s = 1.0 / max(1.0, count if divisor is None else divisor) if reduction == "mean" else 1.0
    loss = row.sum() * s
    p = (z - lse).exp()
    k = keep.double()[:, None]
    P = p.clone()
    P.scatter_add_(1, Y[:, None], torch.full_like(zy, -1.0))
    kept = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -12, torch.float16: 2.0 ** -13}[x.dtype]
    dP = (p * torch.expm1(Z + dlse + 8 * E + 4 * E * (z - lse).abs() + kept) + E + u * P.abs()) * k
    P = P * k
    s *= upstream
    a = abs(s)
    out = {"loss": (loss, drow.sum() * abs(s / upstream) + 2 * E * loss.abs()), "row_loss": (row, drow)}
    for name, left, dleft, right, terms in (("d_features", P, dP, W, v), ("d_weight", P.T, dP.T, X, n),
                                            ("d_bias", P.T, dP.T, torch.ones(n, 1, dtype=torch.float64, device=x.device), n)):
        want = s * (left @ right)
        tol = a * (dleft @ right.abs() + (terms + 2) * E * (left.abs() @ right.abs())) + (u + 2 * E) * want.abs() + tiny
        if name == "d_bias":
            want, tol = want[:, 0], tol[:, 0]
        out[name] = (want, tol)
    return out


def close(name, got, want):
    value, tol = want
    got = got.double().reshape(value.shape)
    bad = ~((got - value).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), bad.numel(), float(((got - value).abs() / tol).nan_to_num(1e9).max()))


def check_all(rh, x, w, y, b, **kw):
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, b is not None), **kw)
    want = oracle(x, w, y, b, reduction=kw.get("reduction", "mean"), upstream=kw.get("expected_grad", 1.0))
    for name in ("loss", "row_loss", "d_features", "d_weight") + (("d_bias",) if b is not None else ()):
        close(name, out[name], want[name])
    return out


SIZES = [(1, 8, 1), (1, 64, 2), (2, 1, 3), (3, 17, 5), (31, 33, 63), (64, 64, 64), (128, 128, 128), (129, 72, 257),
         (300, 100, 1000), (257, 256, 601), (65, 520, 4099), (1000, 40, 70)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_matches_64_bits(rh, n, d, v, dtype, bias):
    x, w, y, b = make(n, d, v, dtype, bias, ignored=0.3 if n > 2 else 0.0)
    out = check_all(rh, x, w, y, b)
    assert float(out["num_valid"]) == float((y != -100).sum())
    assert int(out["status"]) == 0
    assert out["d_features"].dtype == x.dtype and out["row_loss"].dtype == torch.float32
    assert (out["d_features"][y == -100] == 0).all() and (out["row_loss"][y == -100] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,v", [(4099, 264, 70001), (8200, 1032, 300), (70000, 24, 90)])
def test_large_tiles_pieces_and_many_rows(rh, n, d, v, dtype):
    if dtype == "f32" and v > 1000:
        n = 2051
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.1, seed=3)
    check_all(rh, x, w, y, b)


SIZES_WIDE = [(5, 512, 33), (130, 520, 1), (129, 1000, 2049), (700, 513, 4100), (64, 1544, 129)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,d,v", SIZES_WIDE)
def test_wide_features(rh, n, d, v, dtype, bias):
    """The logits are kept between the passes from a feature width on."""
    x, w, y, b = make(n, d, v, dtype, bias, ignored=0.3, seed=11, scale=4.0)
    check_all(rh, x, w, y, b)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,d,v", [(17, 8, 1), (64, 256, 80), (63, 40, 127), (129, 33, 128), (65, 257, 129), (200, 264, 256),
                                   (127, 512, 300), (130, 72, 384), (70, 300, 385), (128, 500, 512), (66, 256, 513),
                                   (193, 256, 601), (100, 31, 640), (100, 64, 641), (1000, 2048, 100)])
def test_whole_rows(rh, n, d, v, dtype):
    """Around the sizes whose logits a workgroup holds whole: each gradient by itself too, in every reduction."""
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.3, seed=18)
    got = check_all(rh, x, w, y, b)
    check_all(rh, x, w, y, None, reduction="sum")
    for i, k in enumerate(("d_features", "d_weight", "d_bias")):
        only = rh.functional.linear_cross_entropy(x, w, y, b, grads=tuple(j == i for j in range(3)))
        assert torch.equal(only[k], got[k]) and torch.equal(only["loss"], got["loss"]), k
    low = b.clone()
    low[: v // 2] = float("-inf")
    y = torch.where(y >= 0, y.clamp(min=v // 2), y)
    got = rh.functional.linear_cross_entropy(x, w, y, low, grads=(True, True, True))
    want = oracle(x, w[v // 2:], torch.where(y >= 0, y - v // 2, y), b[v // 2:])
    for k in ("loss", "row_loss", "d_features"):
        close(k, got[k], want[k])
    for k in ("d_weight", "d_bias"):
        assert (got[k][: v // 2] == 0).all()
        close(k, got[k][v // 2:], want[k])
    keep = torch.full((v, d + 24), float("nan"), dtype=x.dtype, device="cuda")      # NaN between the rows
    keep[:, 8:d + 8] = w
    again = rh.functional.linear_cross_entropy(x, keep[:, 8:d + 8], y, low, grads=(True, True, True))
    for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
        assert torch.equal(again[k], got[k]), k


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("d,v", [(8, 17), (33, 200), (2048, 40), (2056, 3000), (5000, 130), (256, 40001)])
def test_few_rows(rh, n, d, v, dtype):
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.25 if n > 4 else 0.0, seed=13)
    check_all(rh, x, w, y, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d", [(1, 4096), (1, 2056), (2, 1032), (2, 4096), (3, 1024), (4, 2048), (4, 520), (7, 1024)])
def test_few_rows_masked_and_strided(rh, n, d, dtype):
    """The first classes masked (workgroups that see nothing else), a row left out that holds anything,
    rows of any stride, and the gradients that a frozen weight leaves."""
    v = 1500
    x, w, y, b = make(n, d, v, dtype, True, seed=17)
    for low in (float("-inf"), torch.finfo(b.dtype).min):
        b[:700] = low
        y.clamp_(min=700)
        got = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
        want = oracle(x, w[700:], y - 700, b[700:])
        for k in ("loss", "row_loss", "d_features"):
            close(k, got[k], want[k])
        for k in ("d_weight", "d_bias"):
            assert (got[k][:700] == 0).all()
            close(k, got[k][700:], want[k])
    only = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, False, False))
    assert torch.equal(only["d_features"], got["d_features"]) and torch.equal(only["loss"], got["loss"])
    odd = torch.full((n, d + 3), float("nan"), dtype=x.dtype, device="cuda")
    odd[:, 1:d + 1] = x
    ww = torch.full((v, d + 5), float("nan"), dtype=x.dtype, device="cuda")
    ww[:, 3:d + 3] = w
    for xs, ws in ((odd[:, 1:d + 1], w), (x, ww[:, 3:d + 3])):
        again = rh.functional.linear_cross_entropy(xs, ws, y, b, grads=(True, True, True))
        for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
            assert torch.equal(again[k], got[k]), k
    y[n - 1] = -100
    want = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    for value in (float("nan"), float("inf"), torch.finfo(x.dtype).min):
        x[n - 1] = value
        got = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
        for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
            assert torch.equal(got[k], want[k]), k
        assert (got["d_features"][n - 1] == 0).all()


def test_few_rows_of_very_many_classes(rh):
    """More classes than the waves take in one go, and a workspace row past 2^31 bytes of weights."""
    x, w, y, b = make(3, 16, 300_001, "bf16", True, seed=14)
    check_all(rh, x, w, y, b)
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(600_000, 2048, generator=g, device="cuda").mul_(0.03).bfloat16()      # 2.4 GB
    x = torch.randn(2, 2048, generator=g, device="cuda").bfloat16()
    y = torch.tensor([599_999, 3], device="cuda")
    out = rh.functional.linear_cross_entropy(x, w, y, grads=(True, True, False))
    z = torch.cat([x.double() @ w[i:i + 50_000].double().T for i in range(0, 600_000, 50_000)], 1)
    row = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    assert ((out["row_loss"].double() - row).abs() <= 4096 * E * row).all()
    p = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
    p[torch.arange(2), y] -= 1.0
    for c in (0, 3, 299_999, 599_999):
        want = (p[:, c, None] * x.double()).sum(0) / 2
        assert ((out["d_weight"][c].double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-9).all()


def test_rows_in_chunks(rh):
    """More rows than logits may be kept of: the same sums as the two halves by themselves."""
    x, w, y, b = make(17001, 520, 70001, "bf16", True, seed=12)
    y[:9000:3] = -100
    kw = dict(reduction="sum", grads=(True, True, True))
    both = rh.functional.linear_cross_entropy(x, w, y, b, **kw)
    halves = [rh.functional.linear_cross_entropy(x[i], w, y[i], b, **kw) for i in (slice(0, 8000), slice(8000, 17001))]
    assert torch.allclose(both["row_loss"], torch.cat([h["row_loss"] for h in halves]), rtol=64 * E, atol=64 * E)
    for part in (slice(0, 300), slice(8500, 9000), slice(16800, 17001)):      # a row's results need that row alone
        close("d_features", both["d_features"][part], oracle(x[part], w, y[part], b, reduction="sum")["d_features"])
    assert abs(float(both["loss"]) - sum(float(h["loss"]) for h in halves)) <= 3 * 2.0 ** -24 * float(both["loss"])
    u = 2.0 ** -8
    for k, rows in (("d_weight", x), ("d_bias", torch.ones(17001, 1, device="cuda"))):
        a, c = (h[k].double() for h in halves)
        # each side rounds once per result; the sums inside are float32 in another order: 17001 terms of
        # |P| |x| <= |P| max|x|, and sum_n |P| <= 2 (count of the label) + the class's probability mass
        mass = 2.0 * torch.bincount(y[y >= 0], minlength=70001).double() + halves[0]["d_bias"].double().abs() \
            + halves[1]["d_bias"].double().abs() + 1.0
        slack = 64 * E * float(rows.abs().max()) * (mass[:, None] if k == "d_weight" else mass)
        bad = (both[k].double() - (a + c)).abs() > u * (a.abs() + c.abs() + (a + c).abs()) + slack
        assert not bad.any(), (k, int(bad.sum()))
    y[:] = -100
    y[16000:] = 5
    some = rh.functional.linear_cross_entropy(x, w, y, b, **kw)
    want = oracle(x[16000:], w, y[16000:], b, reduction="sum")
    close("d_features", some["d_features"][16000:], want["d_features"])
    assert (some["d_features"][:16000] == 0).all()
    for k in ("loss", "d_weight", "d_bias"):
        close(k, some[k], want[k])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,v", [(17, 4001, 70), (40, 3000, 700), (300, 2100, 130), (130, 4096, 1000), (70, 1030, 65),
                                   (600, 2048, 641), (33, 8200, 3)])
def test_long_sums_of_few_logits(rh, n, d, v, dtype):
    """Logits of few tiles and many features, whose sums are split; forward alone too."""
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.2, seed=22)
    check_all(rh, x, w, y, b)
    alone = rh.functional.linear_cross_entropy(x, w, y, b)
    close("row_loss", alone["row_loss"], oracle(x, w, y, b)["row_loss"])
    y[:] = -100
    y[n - 1] = v - 1      # one row counts: its tile's sum in as many parts as there are workgroups
    check_all(rh, x, w, y, b)
    b[: v - 1] = float("-inf")
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    assert float(out["loss"]) == 0.0 and (out["d_weight"] == 0).all() and (out["d_features"] == 0).all()


@pytest.mark.parametrize("n,d,v,dtype", [(9001, 72, 70001, "f32"), (1_700_001, 24, 600, "bf16")])
def test_rows_in_chunks_of_other_ways(rh, n, d, v, dtype):
    """float32, whose P lies beside the logits, and whole rows of few classes: more than one chunk of each."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(n, d, generator=g, device="cuda").to(TYPES[dtype])
    w = (torch.randn(v, d, generator=g, device="cuda") * 0.3).to(TYPES[dtype])
    b = (torch.randn(v, generator=g, device="cuda") * 0.1).to(TYPES[dtype])
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[5::7] = -100
    out = rh.functional.linear_cross_entropy(x, w, y, b, reduction="sum", grads=(True, True, True))
    for part in (slice(0, 200), slice(n // 2, n // 2 + 200), slice(n - 200, n)):
        want = oracle(x[part], w, y[part], b, reduction="sum")
        close("row_loss", out["row_loss"][part], want["row_loss"])
        close("d_features", out["d_features"][part], want["d_features"])
    # the sums over all rows, in 64 bits piece by piece; the bounds of the pieces add up
    total = {k: [0.0, 0.0] for k in ("loss", "d_weight", "d_bias")}
    step = 2 ** 27 // v
    for lo in range(0, n, step):
        want = oracle(x[lo:lo + step], w, y[lo:lo + step], b, reduction="sum")
        for k, sums in total.items():
            sums[0] = sums[0] + want[k][0]
            sums[1] = sums[1] + want[k][1]
    for k, sums in total.items():
        close(k, out[k], sums)


def test_two_threads_on_one_stream(rh):
    """They share a workspace: a call's launches do not fall between another's."""
    import threading
    cases = [make(200, 96, 700, "bf16", True, seed=19), make(90, 64, 5000, "f32", True, seed=20),
             make(3, 1024, 900, "f16", True, seed=21)]
    want = [rh.functional.linear_cross_entropy(*c, grads=(True, True, True)) for c in cases]
    wrong = []

    def work(i):
        for k in range(40):
            j = (i + k) % len(cases)
            got = rh.functional.linear_cross_entropy(*cases[j], grads=(True, True, True))
            torch.cuda.current_stream().synchronize()
            wrong.extend(q for q in ("loss", "row_loss", "d_features", "d_weight", "d_bias")
                         if not torch.equal(got[q], want[j][q]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("reduction,grad", [("sum", 1.0), ("mean", 0.25)])
def test_reductions_and_expected_gradient(rh, dtype, reduction, grad):
    x, w, y, b = make(50, 48, 37, dtype, True, ignored=0.2, seed=1)
    check_all(rh, x, w, y, b, reduction=reduction, expected_grad=grad)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_left_out_may_hold_anything(rh, dtype):
    x, w, y, b = make(140, 72, 300, dtype, True, ignored=0.4, seed=2)
    want = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    x2 = x.clone()
    out_rows = (y == -100).nonzero()[:, 0]
    x2[out_rows[0::3]] = float("nan")
    x2[out_rows[1::3]] = float("inf")
    x2[out_rows[2::3]] = torch.finfo(x.dtype).min
    got = rh.functional.linear_cross_entropy(x2, w, y, b, grads=(True, True, True))
    for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype", list(TYPES))
def test_no_row_counts(rh, dtype):
    x, w, y, b = make(70, 72, 300, dtype, True)
    y.fill_(-100)
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    assert float(out["loss"]) == 0.0 and float(out["num_valid"]) == 0.0
    for k in ("row_loss", "d_features", "d_weight", "d_bias"):
        assert (out[k] == 0).all(), k
    e = rh.functional.linear_cross_entropy(x[:0], w, y[:0], b, grads=(True, True, True))
    assert float(e["loss"]) == 0.0 and e["d_features"].shape == (0, 72) and (e["d_weight"] == 0).all()


def test_labels_outside_are_left_out_and_reported(rh):
    x, w, y, b = make(40, 64, 30, "f32", True)
    bad = y.clone()
    bad[3], bad[7], bad[11] = 30, -1, 1 << 40
    ref = y.clone()
    ref[[3, 7, 11]] = -100
    got = rh.functional.linear_cross_entropy(x, w, bad, b, grads=(True, True, True))
    want = rh.functional.linear_cross_entropy(x, w, ref, b, grads=(True, True, True))
    assert int(got["status"]) == 1 and int(want["status"]) == 0
    for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
        assert torch.equal(got[k], want[k])
    with pytest.raises(IndexError):
        rh.LinearCrossEntropy(check_labels=True)(x, w, bad, b)
    rh.LinearCrossEntropy(check_labels=True)(x, w, ref, b)


@pytest.mark.parametrize("value", [float("-inf"), "lowest"])
def test_classes_masked_by_the_bias(rh, value):
    x, w, y, b = make(90, 64, 200, "bf16", True, seed=4)
    y.clamp_(max=99)
    low = torch.finfo(b.dtype).min if value == "lowest" else value
    b[100:] = low
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    want = rh.functional.linear_cross_entropy(x, w[:100].contiguous(), y, b[:100].contiguous(), grads=(True, True, True))
    for k in ("loss", "row_loss"):
        assert torch.allclose(out[k], want[k], rtol=1e-5)     # other tiles: sums in another order (10 e)
    assert (out["d_weight"][100:] == 0).all() and (out["d_bias"][100:] == 0).all()
    # lse may differ in its last bits, and with it now and then which way an entry of P rounds (a
    # step of 2^-8 |P| <= 2^-8): two such entries in one sum, and one step of the result
    flips = 2 * 2.0 ** -8 * float(x.abs().max()) / 90
    assert torch.allclose(out["d_weight"][:100].float(), want["d_weight"].float(), rtol=2.0 ** -7, atol=flips)


def test_nan_and_inf_reach_the_loss(rh):
    x, w, y, b = make(40, 64, 30, "f32", True)
    x[5, 3] = float("nan")
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    assert torch.isnan(out["loss"]).all() and torch.isnan(out["row_loss"][5])
    good = torch.arange(40, device="cuda") != 5
    assert torch.isfinite(out["row_loss"][good]).all() and torch.isfinite(out["d_features"][good]).all()
    x[5, 3] = 0.0
    b[2] = float("inf")
    assert torch.isnan(rh.functional.linear_cross_entropy(x, w, y, b)["loss"]).all()


def test_strides_and_label_types(rh):
    x, w, y, b = make(60, 72, 130, "bf16", True, ignored=0.2, seed=5)
    want = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    wide = torch.full((60, 200), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 8:80] = x
    odd = torch.full((60, 201), float("nan"), dtype=x.dtype, device="cuda")
    odd[:, 3:75] = x
    ww = torch.full((130, 160), float("nan"), dtype=x.dtype, device="cuda")
    ww[:, 16:88] = w
    wo = torch.full((130, 161), float("nan"), dtype=x.dtype, device="cuda")
    wo[:, 5:77] = w
    yy = torch.full((60, 3), -7, dtype=torch.int32, device="cuda")
    yy[:, 1] = y
    for xs in (x, wide[:, 8:80], odd[:, 3:75], x.t().contiguous().t()):
        for ws in (w, ww[:, 16:88], wo[:, 5:77], w.t().contiguous().t()):
            got = rh.functional.linear_cross_entropy(xs, ws, yy[:, 1], b, grads=(True, True, True))
            for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
                assert torch.equal(got[k], want[k]), k
    batched = rh.functional.linear_cross_entropy(x.view(5, 12, 72), w, y.view(5, 12), b, grads=(True, False, False))
    assert batched["row_loss"].shape == (5, 12) and batched["d_features"].shape == (5, 12, 72)
    assert torch.equal(batched["d_features"].view(60, 72), want["d_features"]) and "d_weight" not in batched
    broad = rh.functional.linear_cross_entropy(x[:1].expand(60, 72), w, y, b)
    copied = rh.functional.linear_cross_entropy(x[:1].repeat(60, 1), w, y, b)
    assert torch.equal(broad["row_loss"], copied["row_loss"])


# ------------------------------------------------------------------ the module
def test_module_gradients_and_upstream(rh):
    x, w, y, b = make(80, 64, 200, "f32", True, ignored=0.1, seed=6)
    want = oracle(x, w, y, b)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    fn = rh.LinearCrossEntropy()
    loss = fn(leaves[0], leaves[1], y, leaves[2])
    loss.backward()
    close("loss", loss.detach(), want["loss"])
    for t, k in zip(leaves, ("d_features", "d_weight", "d_bias")):
        close(k, t.grad, want[k])
    assert torch.equal(fn.last["row_loss"], rh.functional.linear_cross_entropy(x, w, y, b)["row_loss"])
    with pytest.raises(RuntimeError):
        loss.backward()
    # any other upstream gradient, through other operations: exact powers of two
    first = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad = None
    (fn(leaves[0], leaves[1], y, leaves[2]) * 0.5 + 1.0).backward()
    for t, g in zip(leaves, first):
        assert torch.equal(t.grad, g * 0.5)
    # gradients accumulate, and only where they are asked for
    leaves[0].grad = None
    fn(leaves[0], w, y, b).backward()
    fn(leaves[0], w, y, b).backward()
    assert torch.equal(leaves[0].grad, first[0] * 2)
    with torch.no_grad():
        assert not fn(leaves[0], leaves[1], y, leaves[2]).requires_grad


def test_backward_of_the_node(rh):
    """Some of the leaves, a graph of the gradients, a kept graph, a loss changed in place."""
    x, w, y, b = make(40, 64, 90, "f32", True, seed=16)
    want = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    fn = rh.LinearCrossEntropy()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = fn(leaves[0], leaves[1], y, leaves[2])
    loss.backward(inputs=[leaves[1]])
    assert torch.equal(leaves[1].grad, want["d_weight"]) and leaves[0].grad is None and leaves[2].grad is None
    # the gradients themselves cannot be differentiated, and say so instead of counting as constants
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (g,) = torch.autograd.grad(fn(leaves[0], leaves[1], y, leaves[2]), leaves[0], create_graph=True)
    assert torch.equal(g.detach(), want["d_features"])
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    # one set of gradients, kept graph or not
    loss = fn(leaves[0], leaves[1], y, leaves[2])
    loss.backward(retain_graph=True)
    with pytest.raises(rh.RetinaHeadError, match="once"):
        loss.backward()
    # in place, and a non-leaf input
    for t in leaves:
        t.grad = None
    loss = fn(leaves[0] * 2.0, leaves[1], y, leaves[2])
    loss /= 4
    loss.backward()
    double = rh.functional.linear_cross_entropy(x * 2.0, w, y, b, grads=(True, True, True))
    assert torch.equal(leaves[0].grad, double["d_features"] * 0.5)
    assert torch.equal(leaves[1].grad, double["d_weight"] * 0.25)
    # under inference mode and without any tensor that requires gradients
    with torch.inference_mode():
        assert torch.equal(fn(x, w, y, b), want["loss"])
    assert fn(x, w, y, b).grad_fn is None


def test_gradient_against_differences(rh):
    x, w, y, b = make(12, 16, 20, "f32", True, seed=7)
    out = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    h = 2.0 ** -6
    # central differences of the 64-bit loss: h^2/6 |f'''|, with |f'''| <= 2 max|w|^3 (softmax cumulants)
    for t, k in ((x, "d_features"), (w, "d_weight"), (b, "d_bias")):
        flat = t.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 7)):
            keep = flat[i].clone()
            flat[i] = keep + h
            up = oracle(x, w, y, b)["loss"][0]
            hi = flat[i].double()
            flat[i] = keep - h
            down = oracle(x, w, y, b)["loss"][0]
            lo = flat[i].double()
            flat[i] = keep
            slope = float((up - down) / (hi - lo))
            reach = max(1.0, float(x.abs().max()), float(w.abs().max()))
            assert abs(slope - float(out[k].view(-1)[i])) <= h * h / 3 * reach ** 3 + 1e-5, (k, i)


def test_tied_weight_and_frozen_parts(rh):
    """The same weight feeds an embedding and the loss: both gradients arrive."""
    x, w, y, _ = make(30, 32, 50, "f32", False, seed=8)
    w = w.requires_grad_(True)
    emb = w[y]
    rh.LinearCrossEntropy()(emb, w, y).backward()
    got = w.grad.clone()
    want = oracle(emb.detach(), w.detach(), y, None)
    expect = want["d_weight"][0].clone()
    expect.index_add_(0, y, want["d_features"][0])
    tol = want["d_weight"][1].clone()
    tol.index_add_(0, y, want["d_features"][1] + 4 * E * want["d_features"][0].abs())
    assert ((got.double() - expect).abs() <= tol + 4 * E * expect.abs()).all()


def test_streams_and_repeated_calls_agree(rh):
    x, w, y, b = make(500, 256, 3001, "bf16", True, ignored=0.1, seed=9)
    first = rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(rh.functional.linear_cross_entropy(x, w, y, b, grads=(True, True, True)))
    torch.cuda.synchronize()
    for o in outs:
        for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
            assert torch.equal(o[k], first[k]), k


def test_captured_training_step(rh):
    """Forward and backward in one graph, replayed with new inputs between eager calls."""
    x, w, y, b = make(200, 64, 300, "bf16", True, ignored=0.1, seed=10)
    fn = rh.LinearCrossEntropy()
    sx = x.clone().requires_grad_(True)
    sw = w.clone().requires_grad_(True)
    sy = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sx.grad = sw.grad = None
        loss = fn(sx, sw, sy)
        loss.backward()
        del loss
        sx.grad = sw.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = fn(sx, sw, sy)
        static.backward()
    for seed in range(4):
        x2, w2, y2, _ = make(200, 64, 300, "bf16", False, ignored=0.1 * seed, seed=20 + seed)
        with torch.no_grad():
            sx.copy_(x2)
            sw.copy_(w2)
            sy.copy_(y2)
        graph.replay()
        want = rh.functional.linear_cross_entropy(x2, w2, y2, grads=(True, True, False))
        torch.cuda.synchronize()
        assert torch.equal(static.detach(), want["loss"])
        assert torch.equal(sx.grad, want["d_features"]) and torch.equal(sw.grad, want["d_weight"])


# ------------------------------------------------------------------ what an earlier call leaves in the workspace
def with_spoilt_workspaces(rh, call):
    """``call`` with every byte of the workspaces that it uses 0xFF before it (a NaN in every type)."""
    call()      # it has its workspace now
    torch.cuda.synchronize()
    for room in rh.functional._workspaces.values():
        room.fill_(255)
    return call()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d,v", [(1, 2056, 900), (4, 1032, 700), (13, 72, 300), (70, 40, 200), (193, 256, 601), (300, 100, 1000),
                                   (40, 3000, 700), (3000, 64, 129)])
def test_nothing_is_read_that_the_call_did_not_write(rh, n, d, v, dtype):
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.3 if n > 4 else 0.0, seed=23)
    kw = dict(grads=(True, True, True))
    first = rh.functional.linear_cross_entropy(x, w, y, b, **kw)
    again = with_spoilt_workspaces(rh, lambda: rh.functional.linear_cross_entropy(x, w, y, b, **kw))
    want = oracle(x, w, y, b)
    for k in ("loss", "row_loss", "d_features", "d_weight", "d_bias"):
        assert torch.equal(again[k], first[k]), k
        close(k, again[k], want[k])
    alone = with_spoilt_workspaces(rh, lambda: rh.functional.linear_cross_entropy(x, w, y, b))
    close("row_loss", alone["row_loss"], want["row_loss"])


@pytest.mark.parametrize("n,d,v", [(1_700_001, 8, 600), (1_680_000, 8, 640)])
def test_nothing_is_read_that_a_shorter_last_chunk_did_not_write(rh, n, d, v):
    """Whole rows in two chunks, the last with fewer workgroups than the first."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, d, generator=g, device="cuda").bfloat16()
    w, b = torch.randn(v, d, generator=g, device="cuda").bfloat16(), torch.randn(v, generator=g, device="cuda").bfloat16()
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[3::11] = -100
    out = with_spoilt_workspaces(rh, lambda: rh.functional.linear_cross_entropy(x, w, y, b, reduction="sum",
                                                                                grads=(True, True, True)))
    total = {k: [0.0, 0.0] for k in ("loss", "d_weight", "d_bias")}
    step = 2 ** 27 // v
    for lo in range(0, n, step):      # the bounds of the pieces add up
        want = oracle(x[lo:lo + step], w, y[lo:lo + step], b, reduction="sum")
        for k, sums in total.items():
            sums[0] = sums[0] + want[k][0]
            sums[1] = sums[1] + want[k][1]
    for k, sums in total.items():
        close(k, out[k], sums)


# ------------------------------------------------------------------ upstream gradients other than the expected one
def leaves_of(*tensors):
    return [None if t is None else t.clone().requires_grad_(True) for t in tensors]


UPSTREAM = [(1, 2056, 900, 64.0), (4, 1032, 5000, 256.0), (4, 40, 5000, 256.0), (13, 72, 30000, 1024.0), (16, 2048, 300, 512.0),
            (300, 40, 601, 65536.0), (4096, 256, 601, 65536.0), (700, 1001, 20011, 65536.0), (2100, 64, 9000, 65536.0),
            (40, 3000, 700, 2048.0)]


@pytest.mark.parametrize("n,d,v,up", UPSTREAM)
def test_float16_under_a_loss_scale(rh, n, d, v, up):
    """A scaled loss's gradients are those that were made for its scale, whatever 1 would have left of them."""
    x, w, y, b = make(n, d, v, "f16", True, ignored=0.2 if n > 4 else 0.0, seed=24, scale=3.0)
    want = oracle(x, w, y, b, upstream=up)
    made = rh.functional.linear_cross_entropy(x, w, y, b, expected_grad=up, grads=(True, True, True))
    for how in range(3):
        leaves = leaves_of(x, w, b)
        fn = rh.LinearCrossEntropy(expected_grad=(1.0, 1.0, 8.0)[how])
        loss = fn(leaves[0], leaves[1], y, leaves[2])
        if how == 1:
            loss.backward(torch.full((1,), up, device="cuda"))
        else:
            (loss * up).backward()
        close("loss", loss.detach(), want["loss"])
        for t, k in zip(leaves, ("d_features", "d_weight", "d_bias")):
            close(k, t.grad, want[k])
            assert torch.equal(t.grad, made[k]), (k, how)
        assert torch.equal(fn.last["row_loss"], made["row_loss"]) and torch.equal(loss.detach(), made["loss"])


@pytest.mark.parametrize("n,d,v", [(2, 1032, 700), (13, 72, 300), (193, 256, 601), (300, 100, 1000), (40, 3000, 700)])
def test_float16_gradients_made_for_the_loss_scale_stay(rh, n, d, v):
    """expected_grad is the loss scale: what forward made is what backward hands out, of any leaves."""
    x, w, y, b = make(n, d, v, "f16", True, ignored=0.2 if n > 4 else 0.0, seed=25)
    fn = rh.LinearCrossEntropy(expected_grad=512.0)
    for need in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        for up in (512.0, 96.0):
            # (other leaves may be other kernels)
            ref = rh.functional.linear_cross_entropy(x, w, y, b, expected_grad=up, grads=need)
            args = [t.clone().requires_grad_(r) for t, r in zip((x, w, b), need)]
            torch.cuda.synchronize()
            for room in rh.functional._workspaces.values():
                room.fill_(255)
            (fn(args[0], args[1], y, args[2]) * up).backward()
            for t, r, k in zip(args, need, ("d_features", "d_weight", "d_bias")):
                assert t.grad is None if not r else torch.equal(t.grad, ref[k]), (k, need, up)


def test_float16_upstream_of_special_calls(rh):
    fn = rh.LinearCrossEntropy()
    # rows left out that hold anything; a sum beyond the type's range that the upstream gradient brings back
    x, w, y, _ = make(3000, 72, 90, "f16", False, ignored=0.4, seed=26)
    x[(y == -100).nonzero()[::2, 0]] = float("nan")
    for reduction, up in (("mean", 4096.0), ("sum", 2.0 ** -10)):
        px, pw = leaves_of(x, w)
        (rh.LinearCrossEntropy(reduction=reduction)(px, pw, y) * up).backward()
        want = oracle(torch.where((y == -100)[:, None], 0.0, x), w, y, None, reduction=reduction, upstream=up)
        close("d_features", px.grad, want["d_features"])
        close("d_weight", pw.grad, want["d_weight"])
        assert (px.grad[y == -100] == 0).all()
    y5 = torch.full_like(y, 5)
    x5 = torch.full_like(x, 100.0)
    x5[:, 0] = -100.0      # dW of class 5 is about -3000 x
    px, pw = leaves_of(x5, w)
    (rh.LinearCrossEntropy(reduction="sum")(px, pw, y5) * 2.0 ** -10).backward()
    close("d_weight", pw.grad, oracle(x5, w, y5, None, reduction="sum", upstream=2.0 ** -10)["d_weight"])
    # no row counts; no rows
    px, pw = leaves_of(x, w)
    (fn(px, pw, torch.full_like(y, -100)) * 3.0).backward()
    assert (px.grad == 0).all() and (pw.grad == 0).all()
    px, pw = leaves_of(x[:0], w)
    (fn(px, pw, y[:0]) * 3.0).backward()
    assert px.grad.shape == (0, 72) and (pw.grad == 0).all()
    # a divisor, strided and batched features, int32 labels, a label outside
    x, w, y, b = make(60, 72, 130, "f16", True, seed=27)
    y[7] = 130
    wide = torch.full((60, 100), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 5:77] = x
    leaf = wide.requires_grad_(True)
    pw, pb = leaves_of(w, b)
    div = torch.full((1,), 50.0, device="cuda")
    (fn(leaf[:, 5:77].reshape(5, 12, 72), pw, y.view(5, 12).int(), pb, divisor=div) * 1000.0).backward()
    ref = rh.functional.linear_cross_entropy(x, w, y, b, divisor=div, expected_grad=1000.0, grads=(True, True, True))
    assert torch.equal(leaf.grad[:, 5:77], ref["d_features"]) and (leaf.grad[:, 77:] == 0).all()
    assert torch.equal(pw.grad, ref["d_weight"]) and torch.equal(pb.grad, ref["d_bias"])
    # inputs changed in between are refused, and one set of gradients it stays
    px, pw = leaves_of(x, w)
    loss = fn(px, pw, y)
    with torch.no_grad():
        pw += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (loss * 2.0).backward()
    px, pw = leaves_of(x, w)
    loss = fn(px, pw, y)
    (loss * 2.0).backward(retain_graph=True)
    with pytest.raises(rh.RetinaHeadError, match="once"):
        (loss * 2.0).backward()
    # labels made under inference mode
    with torch.inference_mode():
        seen = y.clone()
    first = pw.grad.clone()
    px, pw = leaves_of(x, w)
    (fn(px, pw, seen) * 2.0).backward()
    assert torch.equal(pw.grad, first)


def test_float16_scaled_step_captured(rh):
    """A graph of forward and scaled backward, replayed with other inputs and scales, the expected one among them."""
    x, w, y, _ = make(200, 64, 300, "f16", False, ignored=0.1, seed=28)
    fn = rh.LinearCrossEntropy(expected_grad=128.0)
    sx, sw, sy = x.clone().requires_grad_(True), w.clone().requires_grad_(True), y.clone()
    scale = torch.full((1,), 64.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = fn(sx, sw, sy)
        (loss * scale).backward()
        del loss
        sx.grad = sw.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = fn(sx, sw, sy)
        (static * scale).backward()
    for i, up in enumerate((128.0, 4096.0, 1.0, 128.0, 65536.0)):
        x2, w2, y2, _ = make(200, 64, 300, "f16", False, ignored=0.1 * i, seed=40 + i)
        with torch.no_grad():
            sx.copy_(x2)
            sw.copy_(w2)
            sy.copy_(y2)
            scale.fill_(up)
        graph.replay()
        want = rh.functional.linear_cross_entropy(x2, w2, y2, expected_grad=up, grads=(True, True, False))
        torch.cuda.synchronize()
        assert torch.equal(static.detach(), want["loss"])
        assert torch.equal(sx.grad, want["d_features"]) and torch.equal(sw.grad, want["d_weight"]), up


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,d,v", [(3, 1032, 700), (13, 72, 300), (193, 256, 601), (300, 101, 1000)])
def test_upstream_of_the_other_types(rh, n, d, v, dtype):
    """Stored gradients times the upstream one: its quotient, the product and the result are rounded once more."""
    x, w, y, b = make(n, d, v, dtype, True, ignored=0.2 if n > 4 else 0.0, seed=29)
    want = oracle(x, w, y, b, upstream=300.0)
    leaves = leaves_of(x, w, b)
    (rh.LinearCrossEntropy(expected_grad=7.0)(leaves[0], leaves[1], y, leaves[2]) * 300.0).backward()
    for t, k in zip(leaves, ("d_features", "d_weight", "d_bias")):
        value, tol = want[k]
        more = torch.finfo(t.dtype).eps / 2 + 2 * E
        close(k, t.grad, (value, tol * (1 + more) + more * value.abs()))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [0, 1, 255, 100_003])
def test_scale_gradient(rh, n, dtype):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g).to(TYPES[dtype]).cuda()
    was = x.clone()
    F = rh.functional
    assert F.scale_gradient_(x, torch.full((1,), 2.5, device="cuda"), 2.5) is x and torch.equal(x, was)
    F.scale_gradient_(x, torch.full((1,), 6.0, device="cuda"), 0.5)
    exact = was.double() * 12.0
    f = torch.finfo(x.dtype)
    assert ((x.double() - exact).abs() <= f.eps / 2 * exact.abs() + f.smallest_normal * f.eps / 2).all()


def test_float16_scaled_backward_from_other_streams_and_threads(rh):
    """The gradients are made anew on the forward call's stream, wherever backward is called from."""
    import threading
    cases = [make(200, 96, 700, "f16", True, seed=50), make(90, 64, 5000, "f16", True, seed=51),
             make(3, 1032, 900, "f16", True, seed=52)]
    want = [rh.functional.linear_cross_entropy(*c, expected_grad=96.0, grads=(True, True, True)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)] + [torch.cuda.default_stream()]
    wrong = []

    def work(i):
        fn = rh.LinearCrossEntropy()
        for k in range(12):
            j, s = (i + k) % 3, streams[(i + k // 3) % 3]
            x, w, y, b = cases[j]
            leaves = leaves_of(x, w, b)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                loss = fn(leaves[0], leaves[1], y, leaves[2])
                scaled = loss * 96.0
            torch.cuda.current_stream().wait_stream(s)
            scaled.backward()
            torch.cuda.synchronize()
            wrong.extend((j, q) for t, q in zip(leaves, ("d_features", "d_weight", "d_bias")) if not torch.equal(t.grad, want[j][q]))

    work(0)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_float16_as_a_scaler_and_checkpointing_call_it(rh):
    from torch.utils.checkpoint import checkpoint
    x, w, y, b = make(150, 72, 400, "f16", True, ignored=0.1, seed=53)
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 14)
    want = rh.functional.linear_cross_entropy(x, w, y, b, expected_grad=2.0 ** 14, grads=(True, True, True))
    for expected in (1.0, 2.0 ** 14):
        fn = rh.LinearCrossEntropy(expected_grad=expected)
        leaves = leaves_of(x, w, b)
        scaler.scale(fn(leaves[0], leaves[1], y, leaves[2])).backward()
        for t, k in zip(leaves, ("d_features", "d_weight", "d_bias")):
            assert torch.equal(t.grad, want[k]), (k, expected)
        for reentrant in (False, True):
            leaves = leaves_of(x, w, b)
            loss = checkpoint(lambda p, q, r: fn(p, q, y, r), *leaves, use_reentrant=reentrant)
            scaler.scale(loss).backward()
            for t, k in zip(leaves, ("d_features", "d_weight", "d_bias")):
                assert torch.equal(t.grad, want[k]), (k, expected, reentrant)
    # two calls of one weight: their gradients add up
    fn = rh.LinearCrossEntropy()
    leaves = leaves_of(x, w, b)
    ((fn(leaves[0], leaves[1], y, leaves[2]) + fn(leaves[0], leaves[1], y, leaves[2])) * 2.0 ** 14).backward()
    assert torch.equal(leaves[1].grad, want["d_weight"] * 2.0)
    # a graph of the gradients still refuses to be differentiated
    leaves = leaves_of(x, w, b)
    (g,) = torch.autograd.grad(fn(leaves[0], leaves[1], y, leaves[2]) * 2.0 ** 14, leaves[0], create_graph=True)
    assert torch.equal(g.detach(), want["d_features"])
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.float().sum().backward()
