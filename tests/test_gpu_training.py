"""Training operators (layer norm, typed linear maps, 8-bit saved activations)
against plain 64-bit implementations.

Tolerances follow from the arithmetic: results are rounded once to their type
(unit roundoff u: 2^-24, 2^-8, 2^-11 for float32, bfloat16, float16), sums are
fp32.  A product of length K is held to u |y| + (K + 16) 2^-23 sum |x| |w|
elementwise (2^-23 per step: the tensor cores may truncate) and to
1.5 u + 2^-23 (8 + sqrt K) of its norm (rounding errors of random sign).
8-bit codes of a given matrix are exact, bit for bit.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# The smallest step near zero: half of the least subnormal is lost.
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
ACTS = [("relu", 0.0), ("leaky_relu", 0.2), ("elu", 0.7), ("sigmoid", 0.0), ("tanh", 0.0), ("gelu", 0.0), (None, 0.0)]


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def rand(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


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
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} outside; first at {i}: {got[i]} vs {ref[i]}")


# ── plain implementations in 64 bits ─────────────────────────────────────────
def act64(z, act, alpha):
    if act == "relu":
        return torch.relu(z)  # slope 0 at 0
    if act == "leaky_relu":
        return torch.where(z >= 0, z, alpha * z)
    if act == "elu":
        return torch.where(z < 0, alpha * torch.expm1(z), z)
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(0.7978845608 * (z + 0.044715 * z ** 3)))
    return z


def slope64(z, act, alpha):
    z = z.detach().clone().requires_grad_(True)
    act64(z, act, alpha).sum().backward()
    return z.grad


def exponents64(x, dtype):
    """The saved form's exponents of x (float64), by comparison alone."""
    rows, cols = x.shape
    nb = (cols + 127) // 128
    top = torch.nn.functional.pad(x.abs(), (0, nb * 128 - cols)).view(rows, nb, 128).amax(2)
    e = torch.full_like(top, -24.0 if dtype == torch.float16 else -126.0)
    while bool((127 * torch.exp2(e) < top).any()):
        e = torch.where(127 * torch.exp2(e) < top, e + 1, e)
    return e


def spread(e, cols):
    return e.repeat_interleave(128, 1)[:, :cols]


def norm64(x, eps):
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean) ** 2).mean(1, keepdim=True).add(eps) ** -0.5
    return (x - mean) * rstd, mean, rstd


def spans(sizes):
    o = np.concatenate([[0], np.cumsum(sizes)]).astype(int).tolist()
    return [(t, a, b) for t, (a, b) in enumerate(zip(o, o[1:]))]


def offsets_of(sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


# ── 8-bit saved form ─────────────────────────────────────────────────────────
SHAPES = [(1, 1), (3, 7), (5, 41), (17, 128), (9, 129), (4, 200), (33, 256), (2, 1000), (7, 4099)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("layout", [None, (3, 1), (8, 8)])
def test_save8_codes_are_exact(tg, dtype, shape, layout):
    x = rand(*shape, seed=1, dtype=dtype) * torch.exp2(rand(shape[0], 1, seed=2) * 4).to(dtype)
    if layout:
        x = strided(x, *layout)
    s = tg.save8(x)
    e = exponents64(x.double(), dtype)
    assert torch.equal(s.exponents.double() - 127, e)
    codes = torch.round(x.double() / torch.exp2(spread(e, shape[1])))
    assert torch.equal(s.codes.double(), codes)
    back = s.restore()
    want = codes * torch.exp2(spread(e, shape[1]))
    assert back.dtype == dtype and torch.equal(back.double(), want)
    # bfloat16 holds every saved value exactly, whatever was saved
    assert torch.equal(s.restore(torch.bfloat16).double(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_save8_special_values(tg, dtype):
    x = torch.zeros(6, 300, dtype=dtype, device="cuda")
    x[1, 5] = float("inf")
    x[2, 130] = float("nan")
    x[3, 299] = -float("inf")
    x[4, :] = torch.finfo(dtype).max
    x[5, 0], x[5, 200] = 2.0 ** -24, -torch.finfo(dtype).max
    s = tg.save8(x)
    e = s.exponents.cpu()
    assert e[1, 0] == 255 and e[2, 1] == 255 and e[3, 2] == 255
    v = s.restore().double()
    assert v[0].eq(0).all()
    for row, block in ((1, 0), (2, 1), (3, 2)):
        assert v[row, block * 128:block * 128 + 128].isnan().all()
        others = torch.ones(300, dtype=torch.bool)
        others[block * 128:block * 128 + 128] = False
        assert v[row][others.cuda()].eq(0).all()
    top = torch.finfo(dtype).max
    assert ((v[4] - top).abs() <= top / 64).all() and v[4].isfinite().all()
    assert v[5, 0] == 2.0 ** -24 and (v[5, 200] + top).abs() <= top / 64


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,alpha", ACTS)
@pytest.mark.parametrize("shape,layout", [((9, 41), None), ((5, 384), None), ((6, 256), (1, 1))])
def test_activation_and_its_backward(tg, dtype, act, alpha, shape, layout):
    x, dy = rand(*shape, seed=3, scale=3.0, dtype=dtype), rand(*shape, seed=4, dtype=dtype)
    if layout:
        x, dy = strided(x, *layout), strided(dy, *layout)
    y, s = tg.activation_save8(x, act, alpha)
    ref = act64(x.double(), act, alpha)
    # exponential, reciprocal and products: 16 roundings of fp32, of a value at most max(|x|, 1)
    slack = 2.0 ** -20 * x.double().abs().clamp(min=1)
    assert_within(y, ref, U[dtype] * ref.abs() + slack + TINY[dtype], "y")
    assert torch.equal(s.codes, tg.save8(x).codes)
    for given, at in ((s, s.restore(torch.float32).double()), (x, x.double())):
        dx = tg.activation_backward(dy, given, act, alpha)
        want = dy.double() * slope64(at, act, alpha)
        assert_within(dx, want, U[dtype] * want.abs() + slack * dy.double().abs() + TINY[dtype], "dx")


def test_activation_extremes(tg):
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 88.0, -88.0, 200.0, -200.0, 1e20, -1e20, big, -big]], device="cuda")
    one = torch.ones_like(x)
    for act, alpha in ACTS:
        y, _ = tg.activation_save8(x, act, alpha)
        d = tg.activation_backward(one, x, act, alpha)
        assert y.isfinite().all() and d.isfinite().all(), act
        # the exponent's argument is rounded: 88 * 2^-24 relative
        want = act64(x.double().clamp(-1e6, 1e6), act, alpha)
        inside = x.abs() <= 1e6
        assert_within(y[inside], want[inside], 2.0 ** -16 * want[inside].abs() + 1e-30, act)
    nan = torch.full_like(x, float("nan"))
    for act, alpha in ACTS:
        assert tg.activation_save8(nan, act, alpha)[0].isnan().all(), act
        if act is not None:
            assert tg.activation_backward(one, nan, act, alpha).isnan().all(), act


# ── layer norm ───────────────────────────────────────────────────────────────
WIDTHS = [1, 2, 7, 16, 31, 32, 33, 64, 128, 129, 200, 256, 257, 602, 1000, 1024, 1025, 1280, 2048, 2560, 4096,
          4099, 4104, 5119, 5120, 5128, 8192, 8193, 20000]


def norm_slack(x, cols):
    """What fp32 statistics may move h by, in units of 1 + |h|: sums of at most 64 terms a thread and 10 joins, of
    values up to max|x|, against the row's deviation."""
    h, mean, rstd = norm64(x, 1e-5)
    return 2.0 ** -24 * 96 * (1 + x.abs().amax(1, keepdim=True) * rstd)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_layer_norm(tg, dtype, cols):
    for rows, layout, pdtype in ((0, None, dtype), (1, None, torch.float32), (37, None, dtype), (6, (5, 3), torch.float32)):
        x = rand(rows, cols, seed=cols, scale=2.0, shift=1.5, dtype=dtype)
        dy = rand(rows, cols, seed=cols + 1, dtype=dtype)
        if layout:
            x, dy = strided(x, *layout), strided(dy, *layout)
        gamma = rand(cols, seed=5, scale=0.3, shift=1.0, dtype=pdtype)
        beta = rand(cols, seed=6, dtype=pdtype)
        y, stats = tg.layer_norm(x, gamma, beta)
        y2, stats2, saved = tg.layer_norm(x, gamma, beta, save8=True)
        assert torch.equal(y, y2) and torch.equal(stats, stats2)
        g, b = gamma.double(), beta.double()
        if rows == 0:
            dx, dg, db = tg.layer_norm_backward(dy, x, stats, gamma)
            assert dx.shape == (0, cols) and dg.eq(0).all() and db.eq(0).all()
            continue
        xd, dyd = x.double(), dy.double()
        h, mean, rstd = norm64(xd, 1e-5)
        slack = norm_slack(xd, cols)
        ref = h * g + b
        assert_within(y, ref, U[dtype] * ref.abs() + slack * (g.abs() * (1 + h.abs()) + b.abs()) + TINY[dtype], "y")
        assert_within(stats[:, 1:], rstd, slack * rstd, "rstd")
        # the copy: within half a step (and fp32's error) of h, on the exponent that h's own magnitude gives
        held = saved.restore(torch.float32).double()
        step = torch.exp2(spread(saved.exponents.double() - 127, cols))
        assert_within(held, h, 0.5 * step + 2 * slack * (1 + h.abs()), "h in 8 bits")
        nb = (cols + 127) // 128
        top = torch.nn.functional.pad(h.abs(), (0, nb * 128 - cols)).view(rows, nb, 128).amax(2)
        e = torch.exp2(saved.exponents.double() - 127)
        least = 2.0 ** (-24 if dtype == torch.float16 else -126)
        room = 4 * slack * (1 + top)
        assert (127 * e >= top - room).all() and ((e == least) | (63.5 * e <= top + room)).all()
        for given, hh, rough in ((x, h, slack), (saved, held, 0 * slack + 2.0 ** -24 * 96)):
            dx, dg, db = tg.layer_norm_backward(dy, given, stats, gamma)
            gy = dyd * g
            m1, m2 = gy.mean(1, keepdim=True), (gy * hh).mean(1, keepdim=True)
            want = rstd * (gy - m1 - hh * m2)
            mag = gy.abs() + gy.abs().mean(1, keepdim=True) + hh.abs() * (gy * hh).abs().mean(1, keepdim=True)
            assert_within(dx, want, U[dtype] * want.abs() + rstd * 4 * (rough + slack) * (1 + hh.abs()) * mag + TINY[dtype], "dx")
            wg, wb = (dyd * hh).sum(0), dyd.sum(0)
            n = (rows + 16) * 2.0 ** -24
            tol_g = ((dyd * hh).abs() * n + dyd.abs() * (rough * (1 + hh.abs()))).sum(0)
            assert_within(dg, wg, U[pdtype] * wg.abs() + tol_g + TINY[pdtype], "dgamma")
            assert_within(db, wb, U[pdtype] * wb.abs() + n * dyd.abs().sum(0) + TINY[pdtype], "dbeta")


def test_layer_norm_many_rows_and_repeats(tg):
    """More rows than one wave of blocks; the same bits again."""
    for cols in (16, 128, 600, 4096):
        x, dy = rand(20011, cols, seed=1, dtype=torch.bfloat16), rand(20011, cols, seed=2, dtype=torch.bfloat16)
        gamma, beta = rand(cols, seed=3), rand(cols, seed=4)
        y, stats = tg.layer_norm(x, gamma, beta)
        first = tg.layer_norm_backward(dy, x, stats, gamma)
        again = tg.layer_norm_backward(dy, x, stats, gamma)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        h, _, _ = norm64(x.double(), 1e-5)
        want = (dy.double() * h).sum(0)
        tol = 2.0 ** -24 * (256 * (dy.double() * h).abs().sum(0) + 96 * 8 * dy.double().abs().sum(0))
        assert_within(first[1], want, tol, "dgamma")


def test_layer_norm_constant_and_nan_rows(tg):
    x = torch.full((3, 96), 2.5, device="cuda")
    x[1, 7] = float("nan")
    gamma, beta = rand(96, seed=1), rand(96, seed=2)
    y, stats, saved = tg.layer_norm(x, gamma, beta, save8=True)
    assert torch.equal(y[0], beta) and torch.equal(y[2], beta)
    assert y[1].isnan().all() and saved.restore()[1].isnan().all()
    assert saved.restore()[0].eq(0).all()


def test_layer_norm_gradient_against_differences(tg):
    """Central differences of L = sum(y * dy) along random directions; step 2^-6, the third derivative's term and
    fp32's rounding of L both below 1e-3 of |L'|'s scale."""
    rows, cols = 24, 200
    x, dy = rand(rows, cols, seed=1), rand(rows, cols, seed=2)
    gamma, beta = rand(cols, seed=3, scale=0.2, shift=1.0), rand(cols, seed=4)
    _, stats = tg.layer_norm(x, gamma, beta)
    grads = tg.layer_norm_backward(dy, x, stats, gamma)
    loss = lambda *a: float((tg.layer_norm(*a)[0].double() * dy.double()).sum())  # noqa: E731
    for k, p in enumerate((x, gamma, beta)):
        v = rand(*p.shape, seed=10 + k)
        hs = 2.0 ** -6
        up, down = [x, gamma, beta], [x, gamma, beta]
        up[k], down[k] = p + hs * v, p - hs * v
        diff = (loss(*up) - loss(*down)) / (2 * hs)
        want = float((grads[k].double() * v.double()).sum())
        scale = float(grads[k].double().norm() * v.double().norm()) / math.sqrt(p.numel())
        assert abs(diff - want) <= 1e-3 * (abs(want) + scale * math.sqrt(p.numel())), (k, diff, want)


# ── typed linear maps ────────────────────────────────────────────────────────
TYPED = [  # sizes of the types, K, N
    ([1], 1, 1),
    ([3], 16, 8),
    ([0, 1, 0, 2, 0], 7, 5),
    ([5, 0, 130, 1], 41, 43),
    ([64, 64], 64, 64),
    ([127, 1, 128, 129], 128, 256),
    ([300, 0, 17], 602, 41),
    ([33, 700], 200, 136),
    ([1] * 40, 96, 264),
    ([257], 136, 600),
    ([2, 1030, 3], 320, 128),
]


def typed_inputs(sizes, K, N, dtype, layout=None):
    rows, T = sum(sizes), len(sizes)
    x, dy = rand(rows, K, seed=1, dtype=dtype), rand(rows, N, seed=2, dtype=dtype)
    if layout:
        x, dy = strided(x, *layout), strided(dy, *layout)
    w = rand(T, K, N, seed=3, scale=K ** -0.5, dtype=dtype)
    return x, dy, w, rand(T, N, seed=4), offsets_of(sizes)


def assert_product(got, ref, mags, K, dtype, what):
    u = U[dtype]
    assert_within(got, ref, u * ref.abs() + (K + 16) * 2.0 ** -23 * mags + TINY[dtype], what)
    norm = float(ref.norm())
    if norm > 0 and ref.numel() >= 64:
        off = float((got.double() - ref).norm()) / float(mags.norm())
        assert off <= 1.5 * u * norm / float(mags.norm()) + 2.0 ** -23 * (8 + math.sqrt(K)), f"{what}: {off} of the norm"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(TYPED)))
@pytest.mark.parametrize("layout", [None, (3, 1), (8, 8)])
def test_typed_linear_and_gradients(tg, dtype, case, layout):
    sizes, K, N = TYPED[case]
    x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype, layout)
    xd, dyd, wd = x.double(), dy.double(), w.double()
    rows = sum(sizes)
    z, mz = torch.empty(rows, N, device="cuda", dtype=torch.float64), torch.empty(rows, N, device="cuda", dtype=torch.float64)
    dx, mdx = torch.empty(rows, K, device="cuda", dtype=torch.float64), torch.empty(rows, K, device="cuda", dtype=torch.float64)
    for t, a, b in spans(sizes):
        z[a:b], mz[a:b] = xd[a:b] @ wd[t], xd[a:b].abs() @ wd[t].abs()
        dx[a:b], mdx[a:b] = dyd[a:b] @ wd[t].T, dyd[a:b].abs() @ wd[t].abs().T
    assert_product(tg.typed_linear(x, w, off), z, mz, K, dtype, "y")
    b_rows = torch.cat([bias[t].double().expand(b - a, N) for t, a, b in spans(sizes)])
    assert_product(tg.typed_linear(x, w, off, bias), z + b_rows, mz + b_rows.abs(), K, dtype, "y + bias")
    y = tg.typed_linear(x, w, off, bias, "gelu")
    ref = act64(z + b_rows, "gelu", 0.0)
    slack = (K + 48) * 2.0 ** -23 * (mz + b_rows.abs() + 1) * 1.2
    assert_within(y, ref, U[dtype] * ref.abs() + slack + TINY[dtype], "gelu(y)")
    got_dx, got_dw, got_db = tg.typed_linear_backward(dy, x, w, off)
    assert_product(got_dx, dx, mdx, N, dtype, "dx")
    got_dw32, none = tg.typed_linear_grad_weight(x, dy, off, dtype=torch.float32, bias=False)
    assert none is None and got_dw32.dtype == torch.float32
    # the same with x in 8 bits
    s = tg.save8(x)
    sd = s.restore(torch.float32).double()
    got_s, got_sdb = tg.typed_linear_grad_weight(s, dy, off)
    assert torch.equal(got_sdb, got_db)
    for t, a, b in spans(sizes):
        n = b - a
        want, mag = xd[a:b].T @ dyd[a:b], xd[a:b].abs().T @ dyd[a:b].abs()
        assert_product(got_dw[t], want, mag, n, dtype, f"dw[{t}]")
        assert_product(got_dw32[t], want, mag, n, torch.float32, f"fp32 dw[{t}]")
        assert_within(got_db[t], dyd[a:b].sum(0), (n + 16) * 2.0 ** -24 * dyd[a:b].abs().sum(0), f"db[{t}]")
        want, mag = sd[a:b].T @ dyd[a:b], sd[a:b].abs().T @ dyd[a:b].abs()
        assert_product(got_s[t], want, mag, n, dtype, f"dw[{t}] from 8 bits")
        if n == 0:
            assert got_dw[t].eq(0).all() and got_db[t].eq(0).all() and got_s[t].eq(0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,alpha", ACTS)
def test_typed_linear_saves_its_preactivation(tg, dtype, act, alpha):
    for sizes, K, N in (([5, 0, 130, 1], 41, 43), ([70, 200], 64, 256), ([3], 24, 129)):
        x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
        y, s = tg.typed_linear(x, w, off, bias, act, alpha, save8=True)
        assert torch.equal(y, tg.typed_linear(x, w, off, bias, act, alpha))
        z = torch.cat([x[a:b].double() @ w[t].double() + bias[t].double() for t, a, b in spans(sizes)])
        mag = torch.cat([x[a:b].double().abs() @ w[t].double().abs() + bias[t].double().abs() for t, a, b in spans(sizes)])
        err = (K + 16) * 2.0 ** -23 * mag
        step = torch.exp2(spread(s.exponents.double() - 127, N))
        assert_within(s.restore(torch.float32), z, 0.5 * step + err, "saved")
        e = exponents64(z, dtype)
        # one step coarser or finer only where the block's largest value is at the boundary, within fp32's error
        assert ((s.exponents.double() - 127 - e).abs() <= 1).all()
        assert (s.exponents.double() - 127 == e).double().mean() > 0.99 or e.numel() < 100
        dx = tg.activation_backward(dy, s, act, alpha)
        want = dy.double() * slope64(s.restore(torch.float32).double(), act, alpha)
        slack = 2.0 ** -20 * dy.double().abs() * z.abs().clamp(min=1)
        assert_within(dx, want, U[dtype] * want.abs() + slack + TINY[dtype], "dz")


@pytest.mark.parametrize("dtype", DTYPES)
def test_typed_single_rows(tg, dtype):
    """Serving: a few rows, most types without any."""
    for rows, T, K, N in ((1, 1, 256, 256), (1, 64, 512, 320), (8, 64, 256, 512), (16, 4, 1000, 64), (5, 3, 33, 1001)):
        sizes = [0] * T
        for r in range(rows):
            sizes[(7 * r + 3) % T] += 1
        x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
        z = torch.cat([x[a:b].double() @ w[t].double() + bias[t].double() for t, a, b in spans(sizes)])
        mag = torch.cat([x[a:b].double().abs() @ w[t].double().abs() + bias[t].double().abs() for t, a, b in spans(sizes)])
        assert_product(tg.typed_linear(x, w, off, bias), z, mag, K, dtype, "y")
        dx = torch.cat([dy[a:b].double() @ w[t].double().T for t, a, b in spans(sizes)])
        mag = torch.cat([dy[a:b].double().abs() @ w[t].double().abs().T for t, a, b in spans(sizes)])
        assert_product(tg.typed_linear_grad_input(dy, w, off), dx, mag, N, dtype, "dx")


LONG = [  # sizes of the types, K, N: sums of more than one part, forward and for dX; limits between few rows and tiles
    ([40, 0, 90], 1700, 72),
    ([40, 0, 90], 1699, 41),
    ([130, 1, 70], 72, 1604),
    ([33, 64], 770, 1537),
    ([0, 17, 0], 801, 130),
    ([0, 31, 1, 0], 200, 1000),
    ([16, 17, 18], 1024, 1024),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(LONG)))
def test_typed_long_sums(tg, dtype, case):
    """Long inner lengths: fp32 products add several parts in the output."""
    sizes, K, N = LONG[case]
    x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
    z = torch.cat([x[a:b].double() @ w[t].double() + bias[t].double() for t, a, b in spans(sizes)])
    mag = torch.cat([x[a:b].double().abs() @ w[t].double().abs() + bias[t].double().abs() for t, a, b in spans(sizes)])
    assert_product(tg.typed_linear(x, w, off, bias), z, mag, K, dtype, "y")
    y, s = tg.typed_linear(x, w, off, bias, "elu", 0.5, save8=True)
    assert torch.equal(y, tg.typed_linear(x, w, off, bias, "elu", 0.5))
    err = (K + 16) * 2.0 ** -23 * mag
    ref = act64(z, "elu", 0.5)
    assert_within(y, ref, U[dtype] * ref.abs() + err * 1.2 + 2.0 ** -20 + TINY[dtype], "elu(y)")
    assert_within(s.restore(torch.float32), z, 0.5 * torch.exp2(spread(s.exponents.double() - 127, N)) + err, "saved")
    dx = torch.cat([dy[a:b].double() @ w[t].double().T for t, a, b in spans(sizes)])
    mag = torch.cat([dy[a:b].double().abs() @ w[t].double().abs().T for t, a, b in spans(sizes)])
    assert_product(tg.typed_linear_grad_input(dy, w, off), dx, mag, N, dtype, "dx")


def test_typed_rows_of_other_types_do_not_leak(tg):
    """NaN and infinity in one type's rows and weight stay there."""
    for dtype in DTYPES:
        sizes, K, N = [70, 3, 190], 96, 160
        x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
        clean = tg.typed_linear(x, w, off, bias), *tg.typed_linear_backward(dy, x, w, off)
        x[70:73], dy[70:73] = float("nan"), float("inf")
        w[1] = float("nan")
        y, dx, dw, db = tg.typed_linear(x, w, off, bias), *tg.typed_linear_backward(dy, x, w, off)
        for got, want in ((y, clean[0]), (dx, clean[1])):
            assert torch.equal(got[:70], want[:70]) and torch.equal(got[73:], want[73:]) and got[70:73].isnan().all()
        for got, want in ((dw, clean[2]), (db, clean[3])):
            assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and not got[1].isfinite().any()
        s = tg.save8(x)
        dws, _ = tg.typed_linear_grad_weight(s, dy, off)
        assert dws[0].isfinite().all() and dws[2].isfinite().all() and dws[1].isnan().all()


def test_typed_weight_views_and_repeats(tg):
    """Weights in a larger buffer, a transposed view; the same bits again."""
    sizes, K, N = [70, 0, 190], 96, 160
    for dtype in DTYPES:
        x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
        want = tg.typed_linear(x, w, off), *tg.typed_linear_backward(dy, x, w, off)
        big = torch.full((3, K + 2, N + 8), float("nan"), dtype=dtype, device="cuda")
        big[:, 1:K + 1, 8:] = w
        odd = torch.full((3, K + 2, N + 3), float("nan"), dtype=dtype, device="cuda")
        odd[:, 1:K + 1, 3:] = w
        flipped = w.transpose(1, 2).contiguous().transpose(1, 2)
        for v in (big[:, 1:K + 1, 8:], odd[:, 1:K + 1, 3:], flipped, w):
            got = tg.typed_linear(x, v, off), *tg.typed_linear_backward(dy, x, v, off)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_typed_gradient_against_differences(tg):
    """L = sum(y * dy) is linear in x, w and bias: differences along a direction give the gradient, but for rounding."""
    sizes, K, N = [40, 0, 90], 64, 48
    x, dy, w, bias, off = typed_inputs(sizes, K, N, torch.float32)
    grads = tg.typed_linear_backward(dy, x, w, off)
    loss = lambda *a: float((tg.typed_linear(a[0], a[1], off, a[2]).double() * dy.double()).sum())  # noqa: E731
    for k, p in enumerate((x, w, bias)):
        v = rand(*p.shape, seed=20 + k)
        up, down = [x, w, bias], [x, w, bias]
        up[k], down[k] = p + v, p - v
        diff = (loss(*up) - loss(*down)) / 2
        want = float((grads[k].double() * v.double()).sum())
        # fp32 rounding of the products' terms: 2^-23 (K + 16) of sums of about rows * N terms of random sign
        tol = 2.0 ** -23 * (K + 16) * math.sqrt(130 * N) * 8
        assert abs(diff - want) <= tol, (k, diff, want)


def test_typed_more_rows_than_a_wave(tg):
    sizes = [12000, 1, 0, 8009, 130]
    for dtype in DTYPES:
        for K, N in ((128, 256), (72, 41)):
            x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
            y = tg.typed_linear(x, w, off, bias, "relu")
            dx, dw, db = tg.typed_linear_backward(dy, x, w, off)
            for t, a, b in spans(sizes):
                xd, dyd, wd = x[a:b].double(), dy[a:b].double(), w[t].double()
                ref = torch.clamp(xd @ wd + bias[t].double(), min=0)
                mag = xd.abs() @ wd.abs() + bias[t].double().abs()
                assert_within(y[a:b], ref, U[dtype] * ref.abs() + (K + 16) * 2.0 ** -23 * mag + TINY[dtype], "y")
                assert_product(dx[a:b], dyd @ wd.T, dyd.abs() @ wd.abs().T, N, dtype, "dx")
                assert_product(dw[t], xd.T @ dyd, xd.abs().T @ dyd.abs(), b - a, dtype, "dw")
                assert_within(db[t], dyd.sum(0), 512 * 2.0 ** -24 * dyd.abs().sum(0), "db")
            again = tg.typed_linear_backward(dy, x, w, off)
            assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,N", [(264, 328), (263, 329), (520, 160), (136, 640)])
def test_typed_large_products(tg, dtype, K, N):
    """Sizes that run on pairs of CTAs (aligned copies first where rows are not aligned): uneven types, one of a row,
    one empty, one whose NaN and infinity must stay its own."""
    sizes = [30001, 0, 1, 25000, 300, 14755, 130]
    x, dy, w, bias, off = typed_inputs(sizes, K, N, dtype)
    bad = sum(sizes[:4])
    x[bad:bad + 300], dy[bad:bad + 300] = float("nan"), float("inf")
    y, z8 = tg.typed_linear(x, w, off, bias, "relu", save8=True)
    dx, dw, db = tg.typed_linear_backward(dy, x, w, off)
    dw32, _ = tg.typed_linear_grad_weight(x, dy, off, dtype=torch.float32, bias=False)
    s = tg.save8(x)
    dws, dbs = tg.typed_linear_grad_weight(s, dy, off)
    held = s.restore(torch.float32)
    for t, a, b in spans(sizes):
        if t == 4:
            assert y[a:b].isnan().all() and dx[a:b].isnan().all()
            continue
        xd, dyd, wd = x[a:b].double(), dy[a:b].double(), w[t].double()
        pre, mag = xd @ wd + bias[t].double(), xd.abs() @ wd.abs() + bias[t].double().abs()
        ref = torch.clamp(pre, min=0)
        err = (K + 16) * 2.0 ** -23 * mag
        assert_within(y[a:b], ref, U[dtype] * ref.abs() + err + TINY[dtype], f"y[{t}]")
        part = tg.Saved8(z8.codes[a:b], z8.exponents[a:b], dtype)
        step = torch.exp2(spread(part.exponents.double() - 127, N))
        assert_within(part.restore(torch.float32), pre, 0.5 * step + err, f"saved[{t}]")
        assert_product(dx[a:b], dyd @ wd.T, dyd.abs() @ wd.abs().T, N, dtype, f"dx[{t}]")
        want, mag = xd.T @ dyd, xd.abs().T @ dyd.abs()
        assert_product(dw[t], want, mag, b - a, dtype, f"dw[{t}]")
        assert_product(dw32[t], want, mag, b - a, torch.float32, f"fp32 dw[{t}]")
        hd = held[a:b].double()
        assert_product(dws[t], hd.T @ dyd, hd.abs().T @ dyd.abs(), b - a, dtype, f"dw[{t}] from 8 bits")
        assert_within(db[t], dyd.sum(0), 1024 * 2.0 ** -24 * dyd.abs().sum(0), f"db[{t}]")
        assert_within(dbs[t], dyd.sum(0), 1024 * 2.0 ** -24 * dyd.abs().sum(0), f"db[{t}] from 8 bits")
    again = tg.typed_linear(x, w, off, bias, "relu"), *tg.typed_linear_backward(dy, x, w, off)
    for p, q in zip((y, dx, dw, db), again):
        assert torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0))


def test_typed_offsets_out_of_range_stay_inside(tg):
    """Offsets are clamped: nothing outside the outputs is touched and no address past the inputs is read."""
    x, dy, w, bias, _ = typed_inputs([40, 50], 32, 24, torch.float32)
    for off in ([0, 40, 5000], [-7, 40, 90], [0, 80, 20], [90, 90, 90]):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        assert tg.typed_linear(x, w, o, bias).shape == (90, 24)
        tg.typed_linear_backward(dy, x, w, o)
        with pytest.raises(tg.InvalidArgument):
            tg.check_row_offsets(o, 90)
    torch.cuda.synchronize()
    good = offsets_of([40, 50])
    assert tg.check_row_offsets(good, 90) is good


def test_typed_offsets_that_overlap_stay_inside(tg):
    """Types that own the same rows, or leave rows out: the partial sums stay within their buffers, and types whose rows
    are their own (or owned twice) still get their gradients."""
    M, K, N = 30000, 256, 384  # weight gradients by TMA (bf16), and by loaders (fp32)
    for dtype, out in ((torch.bfloat16, torch.float32), (torch.bfloat16, None), (torch.float32, None)):
        x, dy, w, bias, _ = typed_inputs([M] + [0] * 31, K, N, dtype)
        twice = torch.tensor([0, M] * 16 + [0], dtype=torch.int32, device="cuda")
        assert tg.typed_linear(x, w, twice, bias).shape == (M, N)
        dx, dw, db = tg.typed_linear_backward(dy, x, w, twice, dtype=out)
        part = offsets_of([1000] + [0] * 30 + [500])  # rows from 1500 on are no type's
        _, dw, db = tg.typed_linear_backward(dy, x, w, part, dtype=out)
        for t, a, b in ((0, 0, 1000), (31, 1000, 1500)):
            xd, dyd = x[a:b].double(), dy[a:b].double()
            assert_product(dw[t], xd.T @ dyd, xd.abs().T @ dyd.abs(), b - a, dw.dtype, f"dw[{t}]")
            assert_within(db[t], dyd.sum(0), (b - a + 16) * 2.0 ** -24 * dyd.abs().sum(0), f"db[{t}]")
        assert dw[1:31].eq(0).all() and db[1:31].eq(0).all()
    torch.cuda.synchronize()


# ── streams, graphs, refusals ────────────────────────────────────────────────
def _everything(tg, x, dy, gamma, beta, w, w2, off):
    y, stats, h8 = tg.layer_norm(x, gamma, beta, save8=True)
    z, z8 = tg.typed_linear(y, w, off, None, "gelu", save8=True)
    out = tg.typed_linear(z, w2, off)
    da, dw2, db2 = tg.typed_linear_backward(dy, tg.save8(z), w2, off)
    dz = tg.activation_backward(da, z8, "gelu")
    dn, dw, db = tg.typed_linear_backward(dz, y, w, off)
    return [out, dw2, db2, dw, db, *tg.layer_norm_backward(dn, h8, stats, gamma)]


def _everything_inputs():
    sizes = [70, 0, 190]
    x, dy = rand(260, 96, seed=1, dtype=torch.bfloat16), rand(260, 96, seed=2, dtype=torch.bfloat16)
    w, w2 = rand(3, 96, 160, seed=3, scale=0.1, dtype=torch.bfloat16), rand(3, 160, 96, seed=4, scale=0.1, dtype=torch.bfloat16)
    return x, dy, rand(96, seed=5), rand(96, seed=6), w, w2, offsets_of(sizes)


def test_operators_run_on_the_current_stream(tg):
    args = _everything_inputs()
    want = _everything(tg, *args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        late = [a.clone() for a in args]   # written on s, after the wait
        got = _everything(tg, *late)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_capture_into_a_graph(tg):
    args = _everything_inputs()
    want = _everything(tg, *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _everything(tg, *args)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _everything(tg, *args)
    for _ in range(2):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_example_trains_and_8_bits_keep_up(tg):
    """examples/train_typed_block.py: the loss falls, and with the saved activations in 8 bits it follows the run that
    keeps them whole (each step's gradients are perturbed by about 1 %)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_typed_block.py")
    spec = importlib.util.spec_from_file_location("train_typed_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    kept = example.train(nodes=3000, width=96, types=5, steps=25, save8=True, report=None)
    whole = example.train(nodes=3000, width=96, types=5, steps=25, save8=False, report=None)
    assert kept[-1] < 0.8 * kept[0] and whole[-1] < 0.8 * whole[0]
    assert abs(kept[-1] - whole[-1]) < 0.05 * whole[-1]


def test_block_gradients_against_the_whole_formula(tg):
    """The example's block, fp32, against automatic differentiation in 64 bits."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_typed_block.py")
    spec = importlib.util.spec_from_file_location("train_typed_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    sizes = [40, 0, 90]
    block = example.TypedBlock(3, 64, 128, dtype=torch.float32, save8=False, seed=3)
    x, dy, off = rand(130, 64, seed=1), rand(130, 64, seed=2), offsets_of(sizes)
    y, kept = block.forward(x, off)
    dx, grads = block.backward(dy, kept)
    p = {k: v.double().requires_grad_(True) for k, v in block.params.items()}
    xd = x.double().requires_grad_(True)
    h, _, _ = norm64(xd, 1e-5)
    n = h * p["gamma"] + p["beta"]
    out = torch.cat([xd[a:b] + act64(n[a:b] @ p["w1"][t] + p["b1"][t], "gelu", 0.0) @ p["w2"][t] + p["b2"][t]
                     for t, a, b in spans(sizes)])
    out.backward(dy.double())
    # a chain of two products of 64 and 128 terms and a norm: 2^-23 (8 + sqrt K) each of their terms' norm, which is
    # within a factor of 8 of the result's for these inputs of random sign
    tol = 8 * 4 * 2.0 ** -23 * (8 + math.sqrt(128))
    for name, got, want in (("y", y, out.detach()), ("dx", dx, xd.grad), *((k, grads[k], p[k].grad) for k in grads)):
        off_by = float((got.double() - want).norm() / want.norm())
        assert off_by <= tol, f"{name}: {off_by}"


def test_refusals(tg):
    x, dy, w, bias, off = typed_inputs([40, 50], 32, 24, torch.float32)
    g, b = rand(32, seed=1), rand(32, seed=2)
    y, stats = tg.layer_norm(x, g, b)
    s = tg.save8(x)
    bad = [
        lambda: tg.layer_norm(x, g[:31], b),
        lambda: tg.layer_norm(x.double(), g, b),
        lambda: tg.layer_norm(x[0], g, b),
        lambda: tg.layer_norm(x.cpu(), g, b),
        lambda: tg.layer_norm(x, g.bfloat16(), b.bfloat16()),
        lambda: tg.layer_norm(x, g, b, eps=-1.0),
        lambda: tg.layer_norm(x[:, :0], g[:0], b[:0]),
        lambda: tg.layer_norm_backward(dy, x, stats, g),
        lambda: tg.layer_norm_backward(x, x, stats[:3], g),
        lambda: tg.layer_norm_backward(x.bfloat16(), s, stats, g),
        lambda: tg.typed_linear(x, w[:, :31], off),
        lambda: tg.typed_linear(x, w.bfloat16(), off),
        lambda: tg.typed_linear(x, w, off.long()),
        lambda: tg.typed_linear(x, w, off[:2]),
        lambda: tg.typed_linear(x, w, off, bias[:1]),
        lambda: tg.typed_linear(x, w, off, bias.double()),
        lambda: tg.typed_linear(x, w, off, bias, "softplus"),
        lambda: tg.typed_linear(x, w[0], off),
        lambda: tg.typed_linear_grad_input(x, w, off),
        lambda: tg.typed_linear_grad_weight(x[:80], dy, off),
        lambda: tg.typed_linear_grad_weight(x, dy, off, dtype=torch.bfloat16),
        lambda: tg.typed_linear_grad_weight(s, dy.bfloat16(), off),
        lambda: tg.typed_linear_backward(dy, x, w[:, :31], off),
        lambda: tg.activation_backward(dy, s, "relu"),
        lambda: tg.activation_save8(x, "softplus"),
        lambda: tg.typed_linear(x, torch.zeros(1025, 32, 24, device="cuda"), torch.zeros(1026, dtype=torch.int32, device="cuda")),
        lambda: s.restore(torch.float64),
        lambda: tg.Saved8(s.codes[:, :31], s.exponents[:, :0], s.dtype).restore(),
        lambda: tg.Saved8(torch.zeros(4, 24, dtype=torch.int8, device="cuda"), s.exponents[:4], s.dtype).restore(),
        lambda: tg.check_row_offsets(off, 91),
    ]
    for k, f in enumerate(bad):
        with pytest.raises((ValueError, tg.InvalidArgument)):
            f()
            raise RuntimeError(f"call {k} was not refused")


def test_c_abi_refusals(tg):
    """The C entry points refuse by status and message, before any launch."""
    from tinygnn_b200 import _lib
    lib = _lib.lib
    x = rand(4, 8)
    p = x.data_ptr()
    calls = [
        (lib.tg_save8(4, 8, 7, p, 8, 0, 0.0, None, 0, p, 16, p, 1, None), "type"),
        (lib.tg_save8(4, 8, 0, p, 7, 0, 0.0, None, 0, p, 16, p, 1, None), "leading dimension"),
        (lib.tg_save8(4, 8, 0, p, 8, 9, 0.0, None, 0, p, 16, p, 1, None), "activation"),
        (lib.tg_save8(4, 8, 0, None, 8, 0, 0.0, None, 0, p, 16, p, 1, None), "NULL"),
        (lib.tg_save8(4, 8, 0, p, 8, 0, 0.0, None, 0, p, 8, p, 1, None), "16-byte"),
        (lib.tg_save8(-1, 8, 0, p, 8, 0, 0.0, None, 0, p, 16, p, 1, None), "outside"),
        (lib.tg_activation_grad(4, 8, 0, p, 8, p, 8, p, 16, p, 1, 0, 0.0, p, 8, None), "exactly one"),
        (lib.tg_layer_norm_grad(4, 8, 0, p, 8, None, 0, None, 0, None, 0, p, 0, p, p, 8, p, p, None), "exactly one"),
        (lib.tg_typed_linear(4, 8, 8, 0, 0, p, 8, p, 8, 64, p, None, 0, 0.0, p, 8, None, 0, None, 0, None), "types"),
        (lib.tg_typed_linear(4, 8, 8, 2, 0, p, 8, p, 8, 63, p, None, 0, 0.0, p, 8, None, 0, None, 0, None), "overlap"),
        (lib.tg_typed_linear(4, 0, 8, 2, 0, p, 8, p, 8, 64, p, None, 0, 0.0, p, 8, None, 0, None, 0, None), "outside"),
        (lib.tg_typed_linear_grad_weight(4, 8, 8, 1, 1, p, 8, None, 0, None, 0, p, 8, p, 2, p, 8, 64, None, None),
         "float32 or of the rows"),
    ]
    for k, (status, word) in enumerate(calls):
        assert status == _lib.INVALID_ARGUMENT, k
    assert lib.tg_save8(4, 8, 0, p, 7, 0, 0.0, None, 0, p, 16, p, 1, None) == _lib.INVALID_ARGUMENT
    assert "leading dimension of x" in _lib.last_error()
