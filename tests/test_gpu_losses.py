"""Losses on class scores (log probabilities of labels with entropy and best
classes; distillation) against plain 64-bit implementations.

Tolerances follow from the arithmetic.  With d = (z - max) / temperature an
exponential is within 2^-22 (the hardware's) and the roundings of d, 2^-23 |d|
each way; a row's sum of n terms passes through at most n / 512 + 64 additions
of one thread or tree, 2^-24 each; results are rounded once to their type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
INF = math.inf


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def ints(low, high, shape, seed, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, shape, device="cuda", generator=g).to(dtype)


def strided(t, pad, offset):
    """t's values in rows `pad` elements longer, starting `offset` elements into the buffer; NaN around them."""
    rows, cols = t.shape
    buf = torch.full((rows * (cols + pad) + offset + 1,), float("nan"), dtype=t.dtype, device=t.device)
    v = torch.as_strided(buf, (rows, cols), (cols + pad, 1), offset)
    v.copy_(t)
    return v


def assert_within(got, ref, tol, what=""):
    got = got.double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~(same | ((got - ref).abs() <= tol))
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} outside; first at {i}: {got[i]} vs {ref[i]}")


# ── plain implementations in 64 bits ─────────────────────────────────────────
def softmax64(z, temperature=1.0):
    """(d, log s, log p, p) of rows with at least one class left; a row without one: p = 0, log p = NaN."""
    z = z.double()
    top = z.amax(1, keepdim=True)
    d = (z - torch.where(top == -INF, 0.0, top)) / temperature
    logs = d.exp().sum(1, keepdim=True).log()
    log = d - logs
    return d, torch.where(logs == -INF, 0.0, logs), log, torch.where(logs == -INF, 0.0, log.exp())


def chain(n):
    return n / 512 + 64


def label64(z, labels):
    """log prob of the label, entropy, and their tolerances."""
    n = z.shape[1]
    d, logs, log, p = softmax64(z)
    has = (labels >= 0) & (labels < n)
    at = torch.where(has, labels, 0).long()[:, None]
    lp = torch.where(has, log.gather(1, at)[:, 0], 0.0)
    entropy = -torch.special.xlogy(p, p).sum(1)
    ln = math.log(n) + 1
    rel = 2.0 ** -22 + 2.0 ** -24 * (chain(n) + 4 + 2 * ln)           # of the sum
    far = torch.where(has, d.gather(1, at)[:, 0], 0.0).abs().nan_to_num(posinf=0.0)
    tol_lp = rel + 2.0 ** -24 * (2 * far + 2 * logs[:, 0] + 2)
    # t = sum d e^d / s: each term's and the sum's relative errors, |d| at most ln on average (ln + 1 squared)
    tol_h = 2 * (1 + ln) * (rel + 2.0 ** -23 * (ln + 2))
    return lp, entropy, tol_lp, tol_h


def best64(z, top):
    """The `top` best classes: equal scores in the order of their classes, NaN greatest."""
    key = z.float() + 0.0
    key = torch.where(key.isnan(), INF, key)
    # a NaN above +inf: two stable sorts, the second by being one
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan = z.isnan().gather(1, order)
    order = order.gather(1, torch.sort(nan.int(), dim=1, descending=True, stable=True).indices)
    return order[:, :top].to(torch.int32)


def check_label(tg, z, labels, top, what=""):
    n = z.shape[1]
    out = tg.label_log_probs(z, labels, top)
    lp, entropy, tol_lp, tol_h = label64(z, labels)
    assert_within(out[0], lp, tol_lp, f"{what} log_probs")
    assert_within(out[1], entropy, tol_h, f"{what} entropy")
    assert (out[1] >= 0).logical_or(out[1].isnan()).all()
    if top:
        want = best64(z, top)
        assert torch.equal(out[4], want), f"{what} classes"
        _, logs, log, _ = softmax64(z)
        log = log.gather(1, want.long())
        ln = math.log(n) + 1
        tol = 2.0 ** -22 + 2.0 ** -24 * (chain(n) + 8 + 2 * ln + 2 * log.abs().nan_to_num(posinf=0.0) + 4 * logs)
        assert_within(out[3], log, tol, f"{what} top log probs")
    return out


def label_grad64(z, labels, a, b):
    n = z.shape[1]
    d, logs, log, p = softmax64(z)
    has = ((labels >= 0) & (labels < n) & (z.double().amax(1) > -INF))[:, None]
    at = torch.where(has, labels.long()[:, None], 0)
    a = torch.where(has, a.double()[:, None], 0.0)
    b = b.double()[:, None] if b is not None else torch.zeros_like(a)
    entropy = -torch.special.xlogy(p, p).sum(1, keepdim=True)
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    logz = torch.where(p == 0, 0.0, log)
    want = a * hot - p * (a + b * (logz + entropy))
    ln = math.log(n) + 1
    rel = 2.0 ** -21 + 2.0 ** -24 * (chain(n) + 8 + 2 * ln + 4 * (d.nan_to_num(neginf=0.0).abs() + logs))
    mag = p * (a.abs() + b.abs() * (logz.abs() + entropy + 1))
    tol = U[z.dtype] * want.abs() + (rel + 2.0 ** -22) * mag + hot * a.abs() * 2.0 ** -24 + TINY[z.dtype]
    return want, tol


def check_label_grad(tg, z, labels, out, seed, what="", entropy=True):
    rows = z.shape[0]
    a, b = rand(rows, seed=seed), rand(rows, seed=seed + 1) if entropy else None
    dz = tg.label_log_probs_backward(a, z, labels, out[2], b, out[1] if entropy else None)
    want, tol = label_grad64(z, labels, a, b)
    assert_within(dz, want, tol, f"{what} dlogits")
    return dz


# Around every step of the rules: lanes and scores of narrow rows, narrow and wide, threads, CTAs that share a row.
CLASSES = [1, 2, 7, 15, 16, 17, 41, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 1025, 1026, 1032, 4099, 8191, 8192, 8193,
           16385, 40000, 65537]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_label(tg, dtype, classes):
    for rows, layout, kind, top in ((0, None, torch.int64, 1), (1, None, torch.int64, min(classes, 128)),
                                    (3, None, torch.int32, min(classes, 5)), (70, None, torch.int64, 0),
                                    (37, (5, 3), torch.int32, min(classes, 20))):
        z = rand(rows, classes, seed=classes + rows, scale=3.0, dtype=dtype)
        labels = ints(-1, classes + 1, (rows,), seed=classes, dtype=kind)   # some rows without a label
        if layout:
            z = strided(z, *layout)
        out = check_label(tg, z, labels, top, f"{rows} rows")
        check_label_grad(tg, z, labels, out, seed=classes, what=f"{rows} rows")
    check_label_grad(tg, z, labels, out, seed=1, what="no entropy", entropy=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [257, 512, 1000, 1030, 2011, 4096, 4097, 4104])
def test_label_of_many_rows(tg, dtype, classes):
    """Rows enough for a warp each, several rows a warp, aligned and not."""
    for rows, layout in ((1500, None), (163, (3, 1))):
        z = rand(rows, classes, seed=classes, scale=3.0, dtype=dtype)
        z[rows // 2] = -INF
        z[rows // 3] = torch.finfo(dtype).min
        labels = ints(-1, classes + 1, (rows,), seed=classes)
        if layout:
            z = strided(z, *layout)
        for top in (0, 1, 7, 16, 17, 100):
            out = check_label(tg, z, labels, top, f"{rows} rows, top {top}")
        check_label_grad(tg, z, labels, out, seed=classes)


@pytest.mark.parametrize("dtype", DTYPES)
def test_label_of_many_wide_rows(tg, dtype):
    """More rows than a wave of warps of more than 4,096 classes, and more than a wave of clusters."""
    for rows, classes in ((2400, 5001), (2400, 16384), (700, 16385)):
        z = rand(rows, classes, seed=classes, scale=3.0, dtype=dtype)
        labels = ints(-1, classes + 1, (rows,), seed=classes)
        out = check_label(tg, z, labels, 0, f"{rows} x {classes}")
        check_label_grad(tg, z, labels, out, seed=classes)
    check_label(tg, z, labels, 30, "30 best")


@pytest.mark.parametrize("dtype,classes", [(torch.float32, 140001), (torch.bfloat16, 300007), (torch.float16, 1200000)])
def test_the_widest_rows(tg, dtype, classes):
    """Rows that eight CTAs cannot hold: the distillation reads them twice."""
    for rows in (1, 3, 40):
        if rows * classes > 2 ** 24:
            continue
        z = rand(rows, classes, seed=rows, scale=3.0, dtype=dtype)
        labels = ints(0, classes, (rows,), seed=1)
        out = check_label(tg, z, labels, 50, f"{rows} rows")
        check_label_grad(tg, z, labels, out, seed=1)
        check_distill(tg, z, ints(-2, classes + 2, (rows, 60), 3), rand(rows, 60, seed=4, dtype=dtype), 1.3, rand(rows, seed=5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [5, 41, 300, 1024, 5003, 33000])
def test_label_masks(tg, dtype, classes):
    """Masked classes (-inf and the type's lowest value), rows of them alone, NaN, +inf, constant rows, and k larger
    than what the mask leaves."""
    rows = 13
    z = rand(rows, classes, seed=classes, scale=2.0, dtype=dtype)
    mask = torch.rand(rows, classes, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.6
    low = torch.finfo(dtype).min
    z[:4].masked_fill_(mask[:4], -INF)
    z[4:7].masked_fill_(mask[4:7], low)
    z[7] = -INF
    z[8] = low
    z[9] = 1.5
    z[10, classes // 2] = float("nan")
    z[11, classes - 1] = INF
    z[12] = -INF
    z[12, classes - 2] = -3.0
    labels = ints(0, classes, (rows,), seed=3)
    labels[12] = classes - 2
    for top in (0, 1, min(classes, 30)):
        out = check_label(tg, z, labels, top, f"top {top}")
    finite = [i for i in range(rows) if i not in (10, 11)]
    check_label_grad(tg, z[finite].contiguous(), labels[finite], [out[0][finite], out[1][finite], out[2][finite].contiguous()], seed=7)
    dz = tg.label_log_probs_backward(rand(rows, seed=1), z, labels, out[2], rand(rows, seed=2), out[1])
    assert dz[7].eq(0).all() and dz[10].isnan().all()
    assert out[0][12] == 0 and out[1][12] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [64, 700, 1500, 20000, 131072])
def test_best_classes_in_hard_orders(tg, dtype, classes):
    """Rows whose best classes crowd: rising, falling, all equal, few different values, the best in one thread's
    columns, signed zeros."""
    j = torch.arange(classes, device="cuda")
    rows = [j / classes, -j / classes, 0 * j, j % 3, (j // 7) % 2, -(j % 2) * 0.0,
            torch.where(j % 4096 < 8, j % 97, -j % 5), torch.where(j % 1024 < 8, 50.0 + j / classes, j % 11 * 0.1),
            torch.where(j >= classes - 40, 9.0, 0.0), torch.where(j < 3, 9.0, 1.0)]
    z = torch.stack([r.float() for r in rows]).to(dtype)
    labels = ints(0, classes, (len(rows),), seed=1)
    for top in (1, 2, min(classes, 37), min(classes, 128)):
        check_label(tg, z, labels, top, f"top {top}")
        one = z[6:8].contiguous()
        check_label(tg, one[:, 1:], labels[6:8] - 1, min(top, classes - 1), "unaligned")


def test_label_large_scores(tg):
    """Scores near the type's limits: the distance to the maximum passes its range."""
    for dtype in DTYPES:
        big = torch.finfo(dtype).max
        for classes in (40, 3000):
            z = torch.zeros(3, classes, device="cuda", dtype=dtype)
            z[0, 5], z[0, 6] = big, -big
            z[1] = big
            z[2] = -big
            z[2, 3] = 0.0
            labels = torch.tensor([5, 7, 3], device="cuda")
            out = check_label(tg, z, labels, 5)
            check_label_grad(tg, z, labels, out, seed=2)


def test_label_gradient_against_differences(tg):
    """Central differences of sum a log p + b H along a direction; the step's error is its square, 2^-12, and fp32's
    rounding of the sums (about 2^-22 of their size over the step 2^-6) below it."""
    for rows, classes in ((24, 50), (5, 3001)):
        z, v = rand(rows, classes, seed=1), rand(rows, classes, seed=2)
        labels = ints(0, classes, (rows,), seed=3)
        a, b = rand(rows, seed=4), rand(rows, seed=5)

        def loss(z):
            lp, h, _ = tg.label_log_probs(z, labels)
            return float((a.double() * lp.double() + b.double() * h.double()).sum())
        out = tg.label_log_probs(z, labels)
        dz = tg.label_log_probs_backward(a, z, labels, out[2], b, out[1])
        step = 2.0 ** -6
        diff = (loss(z + step * v) - loss(z - step * v)) / (2 * step)
        want = float((dz.double() * v.double()).sum())
        assert abs(diff - want) <= 2e-3 * (abs(want) + float((dz.double() * v.double()).norm()))


def test_label_gradient_sums_to_zero_and_repeats(tg):
    z = rand(300, 2011, seed=1, scale=2.0)
    labels = ints(0, 2011, (300,), seed=2)
    out, again = tg.label_log_probs(z, labels, 9), tg.label_log_probs(z, labels, 9)
    assert all(torch.equal(p, q) for p, q in zip(out, again))
    a = rand(300, seed=3)
    dz = tg.label_log_probs_backward(a, z, labels, out[2])
    # p's errors, 2^-20 of it at most for scores within 30 of the maximum, and each value's rounding
    assert (dz.double().sum(1).abs() <= 2.0 ** -18 * a.double().abs()).all()


# ── distillation ─────────────────────────────────────────────────────────────
def distill64(z, classes, teacher, temperature, weights):
    rows, n = z.shape
    has = (classes >= 0) & (classes < n) & (teacher.double() > -INF)
    t = torch.where(has, teacher.double() / temperature, -INF)
    some = has.any(1, keepdim=True)
    q = torch.where(has, torch.softmax(t, 1), 0.0)
    at = torch.where(has, classes.long(), 0)
    d, logs, log, p = softmax64(z, temperature)
    lc = log.gather(1, at)
    loss = temperature ** 2 * torch.where(q > 0, q * (torch.where(q > 0, q, 1.0).log() - lc), 0.0).sum(1)
    loss = torch.where(loss > torch.finfo(torch.float32).max, INF, loss)  # (a lowest score's loss may pass fp32's range)
    w = torch.where(some & (z.double().amax(1, keepdim=True) > -INF), temperature * (1.0 if weights is None else weights.double()[:, None]), 0.0)
    qs = torch.zeros_like(p).scatter_add_(1, at, q)
    want = w * (p - qs)
    ln = math.log(n) + 1
    rel = 2.0 ** -21 + 2.0 ** -24 * (chain(n) + 12 + 2 * ln + 6 * (d.nan_to_num(neginf=0.0).abs() + logs))
    if z.dtype != torch.float32:
        # w p may be one power of two, its exponent's addend K = max / temperature + log s - log w rounded to fp32 (|K| < 256)
        k = (z.double().amax(1, keepdim=True).nan_to_num(neginf=0.0).abs() / temperature + logs + w.abs().clamp(min=2.0 ** -64).log().abs()) * 1.4427
        rel = rel + 2.0 ** -24 * 2 * k.clamp(max=256)
    tq = 2.0 ** -24 * 24 * (1 + (t - t.amax(1, keepdim=True)).nan_to_num(neginf=0.0, nan=0.0).abs().amax(1, keepdim=True))
    tol = U[z.dtype] * want.abs() + w.abs() * (rel * p + (tq + 2.0 ** -23) * qs) + TINY[z.dtype]
    mag = torch.where(q > 0, q * (torch.where(q > 0, q, 1.0).log().abs() + lc.abs() + 1), 0.0).nan_to_num(posinf=0.0).sum(1)
    tol_loss = temperature ** 2 * (2.0 ** -22 + 2.0 ** -24 * (chain(n) + classes.shape[1] + 16 + 2 * ln) + tq[:, 0]) * mag * 2
    return loss, want, tol_loss, tol


def check_distill(tg, z, classes, teacher, temperature, weights, what=""):
    loss, dz = tg.distill_loss(z, classes, teacher, temperature, weights)
    want_loss, want, tol_loss, tol = distill64(z, classes, teacher, temperature, weights)
    assert_within(loss, want_loss, tol_loss, f"{what} loss")
    assert_within(dz, want, tol, f"{what} dlogits")
    alone = tg.distill_loss(z, classes, teacher, temperature, weights, grad=False)
    # (not the same bits: without a gradient a row is shared by other threads, and its sum is in another order)
    assert_within(alone, want_loss, tol_loss, f"{what} loss alone")
    return loss, dz


def pick(rows, classes, k, seed, dtype):
    """k classes of each row: some twice, some outside, some rows without any."""
    c = ints(-2, classes + 2, (rows, k), seed=seed, dtype=dtype)
    if k > 2:
        c[:, 2] = c[:, 0]
    c[rows // 2] = -1
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_distill(tg, dtype, classes):
    for rows, layout, kind, k, temperature in ((0, None, torch.int32, 3, 1.0), (1, None, torch.int64, 1, 1.0),
                                               (70, None, torch.int32, 8, 2.0), (37, (5, 3), torch.int64, 128, 0.7),
                                               (5, (1, 0), torch.int32, 33, 4.0)):
        z = rand(rows, classes, seed=classes + rows, scale=3.0, dtype=dtype)
        if layout:
            z = strided(z, *layout)
        if rows == 0:
            loss, dz = tg.distill_loss(z, torch.zeros(0, k, dtype=kind, device="cuda"), rand(0, k, dtype=dtype))
            assert loss.shape == (0,) and dz.shape == z.shape
            continue
        teacher = rand(rows, k, seed=classes + 1, scale=2.0, dtype=dtype if rows % 2 else torch.float32)
        weights = rand(rows, seed=5) if rows != 5 else None
        check_distill(tg, z, pick(rows, classes, k, classes, kind) if rows > 1 else ints(0, classes, (1, 1), 1, kind), teacher,
                      temperature, weights, f"{rows} rows")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [16, 48, 257, 512, 1001, 2048, 4096, 4099, 9000, 40001])
def test_distill_of_many_rows(tg, dtype, classes):
    """Rows enough for a warp each and for several rounds of every block and cluster; few and many entries."""
    for rows, k, kind, layout in ((1500, 8, torch.int32, None), (1100, 32, torch.int64, (3, 1)), (333, 128, torch.int64, None)):
        if rows * classes > 2 ** 25:
            continue
        z = rand(rows, classes, seed=classes + k, scale=3.0, dtype=dtype)
        z[rows // 3] = -INF
        if layout:
            z = strided(z, *layout)
        check_distill(tg, z, pick(rows, classes, k, classes, kind), rand(rows, k, seed=2, scale=2.0, dtype=dtype), 1.7,
                      rand(rows, seed=3), f"{rows} rows, {k} entries")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [6, 41, 900, 5003, 33000])
def test_distill_masks(tg, dtype, classes):
    rows, k = 9, 4
    z = rand(rows, classes, seed=classes, scale=2.0, dtype=dtype)
    mask = torch.rand(rows, classes, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.6
    z[:3].masked_fill_(mask[:3], -INF)
    z[3].masked_fill_(mask[3], torch.finfo(dtype).min)
    z[4] = -INF                      # nothing is left
    z[5] = torch.finfo(dtype).min
    classes_of = ints(0, classes, (rows, k), seed=2)
    teacher = rand(rows, k, seed=3, dtype=dtype)
    teacher[:, 1] = -INF             # one entry is none
    teacher[6] = -INF                # all are
    z.scatter_(1, torch.where(classes_of >= 0, classes_of, 0)[:3], torch.ones(3, k, device="cuda", dtype=dtype))
    loss, dz = check_distill(tg, z, classes_of, teacher, 1.5, rand(rows, seed=4))
    assert loss[4].isnan() and dz[4].eq(0).all() and loss[6] == 0 and dz[6].eq(0).all()
    z[7, classes - 1] = float("nan")
    teacher[8, 0] = float("nan")
    loss, dz = tg.distill_loss(z, classes_of, teacher, 1.5)
    assert loss[7].isnan() and dz[7].isnan().all() and loss[8].isnan()
    # a class that the student masks and the teacher does not: infinite loss, the formula's gradient
    z = torch.zeros(1, classes, device="cuda", dtype=dtype)
    z[0, 2] = -INF
    check_distill(tg, z, torch.tensor([[2, 3]], device="cuda"), torch.zeros(1, 2, device="cuda"), 1.0, None)


def test_distill_gradient_against_differences(tg):
    for rows, classes, k in ((24, 50, 5), (5, 3001, 40)):
        z, v = rand(rows, classes, seed=1), rand(rows, classes, seed=2)
        ids, teacher = pick(rows, classes, k, 3, torch.int64), rand(rows, k, seed=4)
        w = rand(rows, seed=5)
        dz = tg.distill_loss(z, ids, teacher, 2.0, w)[1]
        loss = lambda z: float((w.double() * tg.distill_loss(z, ids, teacher, 2.0, grad=False).double()).sum())  # noqa: E731
        step = 2.0 ** -6
        diff = (loss(z + step * v) - loss(z - step * v)) / (2 * step)
        want = float((dz.double() * v.double()).sum())
        assert abs(diff - want) <= 2e-3 * (abs(want) + float((dz.double() * v.double()).norm()))


def test_distilled_from_own_logits_has_no_loss(tg):
    """A teacher that knows all classes and equals the student: loss and gradient vanish (within roundings of q and p)."""
    z = rand(50, 100, seed=1, scale=2.0)
    best, ids = tg.label_log_probs(z, ints(0, 100, (50,), 2), 100)[3:]
    loss, dz = tg.distill_loss(z, ids, best, 2.0)
    assert loss.abs().max() <= 4 * 2.0 ** -19 and dz.abs().max() <= 2 * 2.0 ** -19


# ── streams, graphs, refusals ────────────────────────────────────────────────
def _everything(tg, z, labels, a):
    out = tg.label_log_probs(z, labels, 7)
    dz = tg.label_log_probs_backward(a, z, labels, out[2], a, out[1])
    return [*out, dz, *tg.distill_loss(z, out[4], out[3], 2.0, a)]


def _inputs(classes):
    return rand(40, classes, seed=1, scale=2.0, dtype=torch.bfloat16), ints(0, classes, (40,), 2), rand(40, seed=3)


@pytest.mark.parametrize("classes", [41, 30000])
def test_losses_run_on_the_current_stream(tg, classes):
    args = _inputs(classes)
    want = _everything(tg, *args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        got = _everything(tg, *[t.clone() for t in args])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("classes", [41, 30000])
def test_losses_capture_into_a_graph(tg, classes):
    args = _inputs(classes)
    want = _everything(tg, *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _everything(tg, *args)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):   # two graphs of the same calls share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = _everything(tg, *args)
        graphs.append((g, got))
    for g, got in graphs + graphs[:1]:
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("classes", [16, 41, 1025])
def test_nothing_outside_the_rows_is_written(tg, classes):
    """The C entry points with strided results: the columns between the rows stay as they were."""
    from tinygnn_b200 import _lib
    rows, ld = 11, classes + 3
    for dtype, kind in ((torch.float32, _lib.F32), (torch.bfloat16, _lib.BF16)):
        z = rand(rows, classes, seed=1, dtype=dtype)
        labels = ints(0, classes, (rows,), 2)
        out = tg.label_log_probs(z, labels, 3)
        a = rand(rows, seed=3)
        s = torch.cuda.current_stream().cuda_stream
        buf = torch.full((rows * ld + 2,), 7.0, dtype=dtype, device="cuda")
        view = torch.as_strided(buf, (rows, classes), (ld, 1), 1)
        st = _lib.lib.tg_label_log_probs_grad(rows, classes, kind, a.data_ptr(), None, z.data_ptr(), classes, labels.data_ptr(), 8,
                                              out[2].data_ptr(), None, view.data_ptr(), ld, s)
        assert st == _lib.OK
        assert torch.equal(view, tg.label_log_probs_backward(a, z, labels, out[2]))
        ids, best = out[4], out[3].contiguous()
        loss = torch.empty(rows, device="cuda")
        view.fill_(7.0)
        st = _lib.lib.tg_distill_loss(rows, classes, kind, z.data_ptr(), classes, 3, ids.data_ptr(), 4, 3, _lib.F32,
                                      best.data_ptr(), 3, 1.0, None, loss.data_ptr(), view.data_ptr(), ld, s)
        assert st == _lib.OK
        assert torch.equal(view, tg.distill_loss(z, ids, best)[1])
        view.fill_(7.0)
        assert buf.eq(7.0).all()


def test_refusals(tg):
    z, labels, a = rand(6, 20, seed=1), ints(0, 20, (6,), 2), rand(6, seed=3)
    lp, h, stats, best, ids = tg.label_log_probs(z, labels, 4)
    bad = [
        lambda: tg.label_log_probs(z.double(), labels),
        lambda: tg.label_log_probs(z[0], labels),
        lambda: tg.label_log_probs(z[:, :0], labels),
        lambda: tg.label_log_probs(z.cpu(), labels),
        lambda: tg.label_log_probs(z, labels.cpu()),
        lambda: tg.label_log_probs(z, labels.float()),
        lambda: tg.label_log_probs(z, labels[:5]),
        lambda: tg.label_log_probs(z, labels[:, None]),
        lambda: tg.label_log_probs(z, labels, -1),
        lambda: tg.label_log_probs(z, labels, 21),
        lambda: tg.label_log_probs(rand(2, 500), labels[:2], 129),
        lambda: tg.label_log_probs(z, labels, 1.5),
        lambda: tg.label_log_probs_backward(a[:5], z, labels, stats),
        lambda: tg.label_log_probs_backward(a.double(), z, labels, stats),
        lambda: tg.label_log_probs_backward(a, z, labels, stats[:5]),
        lambda: tg.label_log_probs_backward(a, z, labels, stats.t()),
        lambda: tg.label_log_probs_backward(a, z, labels, stats, a),
        lambda: tg.label_log_probs_backward(a, z, labels, stats, a, h[:5]),
        lambda: tg.distill_loss(z, ids[:5], best),
        lambda: tg.distill_loss(z, ids, best[:, :3]),
        lambda: tg.distill_loss(z, ids.float(), best),
        lambda: tg.distill_loss(z, ids, best.half()),
        lambda: tg.distill_loss(z, ids[:, :0], best[:, :0]),
        lambda: tg.distill_loss(z, ids, best, 0.0),
        lambda: tg.distill_loss(z, ids, best, -1.0),
        lambda: tg.distill_loss(z, ids, best, float("nan")),
        lambda: tg.distill_loss(z, ids, best, float("inf")),
        lambda: tg.distill_loss(z, ids, best, 1.0, a[:5]),
        lambda: tg.distill_loss(z, ids.repeat(1, 33), best.repeat(1, 33)),
    ]
    for k, f in enumerate(bad):
        with pytest.raises((ValueError, tg.InvalidArgument)):
            f()
            raise RuntimeError(f"call {k} was not refused")


def test_c_abi_refusals(tg):
    from tinygnn_b200 import _lib
    lib = _lib.lib
    p = rand(64).data_ptr()
    calls = [
        lib.tg_label_log_probs(4, 8, 5, p, 8, p, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 8, 0, p, 7, p, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 8, 0, p, 8, p, 2, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 8, 0, None, 8, p, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 8, 0, p, 8, None, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 8, 0, p, 8, p, 8, 9, p, p, p, p, p, None),
        lib.tg_label_log_probs(4, 8, 0, p, 8, p, 8, 2, p, p, p, None, p, None),
        lib.tg_label_log_probs(4, 8, 0, p, 8, p, 8, 0, p, p, p + 4, None, None, None),
        lib.tg_label_log_probs(-1, 8, 0, p, 8, p, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs(4, 0, 0, p, 8, p, 8, 0, p, p, p, None, None, None),
        lib.tg_label_log_probs_grad(4, 8, 0, None, None, p, 8, p, 8, p, None, p, 8, None),
        lib.tg_label_log_probs_grad(4, 8, 0, p, p, p, 8, p, 8, p, None, p, 8, None),
        lib.tg_label_log_probs_grad(4, 8, 0, p, None, p, 8, p, 8, p, None, p, 7, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 0, p, 4, 1, 0, p, 1, 1.0, None, p, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 4, 1, 0, p, 2, 1.0, None, p, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 4, 2, 1, p, 2, 1.0, None, p, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 3, 2, 0, p, 2, 1.0, None, p, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 4, 2, 0, p, 2, 0.0, None, p, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 4, 2, 0, p, 2, 1.0, None, None, p, 8, None),
        lib.tg_distill_loss(4, 8, 0, p, 8, 2, p, 4, 2, 0, p, 2, 1.0, None, p, p, 7, None),
    ]
    assert calls == [_lib.INVALID_ARGUMENT] * len(calls)
