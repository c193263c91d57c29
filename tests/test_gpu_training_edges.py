"""Training operators at arguments and values where they went wrong once:
refusals, values near zero and far from it, rows and types at the edges of a
rule.  Each against a plain 64-bit implementation.

Tolerances follow from the arithmetic and stand beside each test.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# The smallest step near zero: half of the least subnormal is lost.
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def rand(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def test_codes_without_exponents_are_refused(tg):
    """Every entry point that takes a saved matrix refuses codes with no exponents beside them, before any launch."""
    from tinygnn_b200 import _lib
    lib = _lib.lib
    x = rand(4, 64)
    p = x.data_ptr()
    before = lib.tg_kernel_launch_count()
    calls = [
        lambda: lib.tg_layer_norm(4, 8, 0, p, 8, 0, p, p, 1e-5, p, 8, p, p, 16, None, 1, None),
        lambda: lib.tg_typed_linear(4, 8, 8, 1, 0, p, 8, p, 8, 64, p, None, 0, 0.0, p, 8, p, 16, None, 1, None),
        lambda: lib.tg_save8(4, 8, 0, p, 8, 0, 0.0, None, 0, p, 16, None, 1, None),
        lambda: lib.tg_restore8(4, 8, p, 16, None, 1, 0, p, 8, None),
        lambda: lib.tg_activation_grad(4, 8, 0, p, 8, None, 0, p, 16, None, 1, 0, 0.0, p, 8, None),
        lambda: lib.tg_layer_norm_grad(4, 8, 0, p, 8, None, 0, p, 16, None, 1, p, 0, p, p, 8, p, p, None),
        lambda: lib.tg_typed_linear_grad_weight(4, 8, 8, 1, 0, None, 0, p, 16, None, 1, p, 8, p, 0, p, 8, 64, None, None),
    ]
    for k, call in enumerate(calls):
        assert call() == _lib.INVALID_ARGUMENT, k
        assert "exponents is NULL" in _lib.last_error(), k
    assert lib.tg_kernel_launch_count() == before


def test_layer_norm_gradient_of_large_constant_rows(tg):
    """Rows whose mean times 1 / sqrt(eps) overflows fp32: h is 0, so dx = rstd * (g - mean g) and dgamma = 0, whatever
    the number of rows (a block's threads may have fewer rows than they could take).  Sums of 16 and 3 terms: 2^-20."""
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (1, 2, 3, 33):
            x = torch.full((rows, 16), 2.0 ** 121, dtype=dtype, device="cuda")
            dy, gamma, beta = rand(rows, 16, seed=1, dtype=dtype), rand(16, seed=2), rand(16, seed=3)
            y, stats = tg.layer_norm(x, gamma, beta)
            assert torch.equal(y, beta.to(dtype).expand(rows, 16))
            dx, dg, db = tg.layer_norm_backward(dy, x, stats, gamma)
            assert dg.eq(0).all(), rows
            want = dy.double().sum(0)
            assert ((db - want).abs() <= 2.0 ** -20 * dy.double().abs().sum(0)).all()
            g = dy.double() * gamma.double()
            want = 1e-5 ** -0.5 * (g - g.mean(1, keepdim=True))
            mag = 1e-5 ** -0.5 * (g.abs() + g.abs().mean(1, keepdim=True))
            assert ((dx.double() - want).abs() <= U[dtype] * want.abs() + 2.0 ** -20 * mag).all()


def small_and_large(dtype, most):
    """Values of both signs, evenly spread over their exponents from 2^-30 to `most`, as one row per 64 values."""
    n = 64 * 64
    g = torch.Generator(device="cuda").manual_seed(3)
    low, high = -30.0, torch.tensor(float(most)).log2().item()
    x = torch.exp2(low + (high - low) * torch.rand(n, device="cuda", generator=g))
    return torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, x, -x).to(dtype).view(64, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_elu_keeps_its_digits_near_zero(tg, dtype):
    """ELU to a relative tolerance, by the activation kernels and by a typed product's epilogue (x times 1: few rows and
    tiles).  fp32: 1 - e^x by CUDA's function (1 ulp), a product with alpha, and two sums of the three parts a tile's
    product has: 2^-21.  16 bits: the rounding and 2^-16 (the exponential's 2^-22 against 1/16, and alpha)."""
    x = small_and_large(dtype, 20.0)
    for alpha in (1.0, 0.7):
        xd = x.double()
        want = torch.where(xd < 0, alpha * torch.expm1(xd), xd)
        tol = (2.0 ** -21 if dtype == torch.float32 else U[dtype] + 2.0 ** -16) * want.abs() + TINY[dtype]
        got = [tg.activation_save8(x, "elu", alpha)[0],
               tg.activation_save8(x[:, :61], "elu", alpha)[0]]  # rows that end inside 16 bytes
        one = torch.ones(1, 1, 1, dtype=dtype, device="cuda")
        for rows in (16, 64 * 64):
            off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
            y = tg.typed_linear(x.view(-1, 1)[:rows].contiguous(), one, off, None, "elu", alpha)
            got.append(y)
        for y, w, t in zip(got, (want, want[:, :61], want.view(-1, 1)[:16], want.view(-1, 1)),
                           (tol, tol[:, :61], tol.view(-1, 1)[:16], tol.view(-1, 1))):
            bad = ~((y.double() - w).abs() <= t)
            assert not bad.any(), (alpha, y[bad][:4], w[bad][:4])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
def test_slopes_far_from_zero_keep_their_digits(tg, dtype, act):
    """Slopes of sigmoid and tanh to a relative tolerance where they are small.  e^-a with a up to 40 in fp32: its
    argument's rounding is 40 2^-24 of it, and six more roundings: 2^-18.  Results of 16 bits add their rounding."""
    most = 40.0 if act == "sigmoid" else 20.0
    x = small_and_large(dtype, most)
    xd = x.double()
    e = torch.exp(-xd.abs() * (1 if act == "sigmoid" else 2))
    slope = (1 if act == "sigmoid" else 4) * e / (1 + e) ** 2
    # scaled, so that fp16 (least step 2^-24) can tell more of the small ones from zero
    dy = torch.full_like(x, 2.0 ** 14)
    want = 2.0 ** 14 * slope
    tol = (2.0 ** -18 if dtype == torch.float32 else U[dtype] + 2.0 ** -18) * want + TINY[dtype]
    for cols in (64, 61):
        got = tg.activation_backward(dy[:, :cols], x[:, :cols], act)
        bad = ~((got.double() - want[:, :cols]).abs() <= tol[:, :cols])
        assert not bad.any(), (x[:, :cols][bad][:4], got[bad][:4], want[:, :cols][bad][:4])
    # infinities, NaN and zeros
    v = torch.tensor([[float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 200.0, -200.0, 3.0]], device="cuda").to(dtype)
    got = tg.activation_backward(torch.ones_like(v), v, act)
    assert got[0, :2].eq(0).all() and got[0, 2].isnan() and got[0, 3:5].eq(0.25 if act == "sigmoid" else 1.0).all()
    assert got[0, 5:7].eq(0).all() and got[0, 7] > 0


class Guarded:
    """A matrix (or a batch) in a buffer with `room` sentinel elements before it, after it and between its rows."""

    def __init__(self, shape, dtype, pad=8, room=4096):
        self.rows, self.cols = 1, shape[-1]
        for n in shape[:-1]:
            self.rows *= n
        self.ld = self.cols + pad
        self.buf = torch.full((2 * room + self.rows * self.ld,), 77.0, dtype=dtype, device="cuda")
        self.all = self.buf[room:room + self.rows * self.ld].view(self.rows, self.ld)
        self.t = self.all[:, :self.cols].unflatten(0, shape[:-1]) if len(shape) > 2 else self.all[:, :self.cols]
        self.p = self.all.data_ptr()
        self.room = room

    def check(self, what):
        assert self.buf[:self.room].eq(77).all() and self.buf[-self.room:].eq(77).all(), what
        assert self.all[:, self.cols:].eq(77).all(), what


def typed_calls(lib, x, dy, w, bias, off, y, dx, dw, db):
    """The three typed products by the C entry points into guarded buffers (db has no leading dimension: pad 0)."""
    (M, K), N, T, d = x.shape, dy.shape[1], w.shape[0], {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    st = torch.cuda.current_stream().cuda_stream
    assert lib.tg_typed_linear(M, K, N, T, d, x.data_ptr(), K, w.data_ptr(), N, K * N, off.data_ptr(), bias.data_ptr(), 0,
                               0.0, y.p, y.ld, None, 0, None, 0, st) == 0
    assert lib.tg_typed_linear_grad_input(M, K, N, T, d, dy.data_ptr(), N, w.data_ptr(), N, K * N, off.data_ptr(), dx.p,
                                          dx.ld, st) == 0
    assert lib.tg_typed_linear_grad_weight(M, K, N, T, d, x.data_ptr(), K, None, 0, None, 0, dy.data_ptr(), N,
                                           off.data_ptr(), d, dw.p, dw.ld, K * dw.ld, db.p, st) == 0
    torch.cuda.synchronize()
    for what, g in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        g.check(what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(60000, 256, 384), (30000, 256, 384), (3000, 72, 41), (40, 24, 136)])
def test_types_that_overlap(tg, dtype, M, K, N):
    """Sixteen types that each own all rows (and sixteen that own none): every one gets the whole gradients, with the
    same weight everywhere the rows' products are right too, and nothing around the outputs is written.  Sums of n terms
    to n 2^-23 of their magnitude (the tensor cores may truncate)."""
    from tinygnn_b200 import _lib
    T = 32
    x, dy = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype)
    w = rand(1, K, N, seed=3, scale=K ** -0.5, dtype=dtype).repeat(T, 1, 1)
    bias = rand(1, N, seed=4).repeat(T, 1)
    off = torch.tensor([0, M] * 16 + [0], dtype=torch.int32, device="cuda")
    y, dx = Guarded((M, N), dtype), Guarded((M, K), dtype)
    dw, db = Guarded((T, K, N), dtype), Guarded((T, N), torch.float32, pad=0)
    typed_calls(_lib.lib, x, dy, w, bias, off, y, dx, dw, db)
    xd, dyd, wd = x.double(), dy.double(), w[0].double()

    def near(got, want, mag, terms, u):
        bad = ~((got.double() - want).abs() <= u * want.abs() + (terms + 16) * 2.0 ** -23 * mag + TINY[got.dtype])
        assert not bad.any(), (int(bad.sum()), got[bad][:3], want[bad][:3])

    near(y.t, xd @ wd + bias[0].double(), xd.abs() @ wd.abs() + bias[0].double().abs(), K, U[dtype])
    near(dx.t, dyd @ wd.T, dyd.abs() @ wd.abs().T, N, U[dtype])
    dw_want, dw_mag, db_want, db_mag = xd.T @ dyd, xd.abs().T @ dyd.abs(), dyd.sum(0), dyd.abs().sum(0)
    for t in range(T):
        if t % 2:
            assert dw.t[t].eq(0).all() and db.t[t].eq(0).all(), t
        else:
            near(dw.t[t], dw_want, dw_mag, M, U[dtype])
            near(db.t[t], db_want, db_mag, M, U[torch.float32])


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_out_of_range_write_nothing_outside(tg, dtype):
    """Bounds outside [0, rows], decreasing ones, rows of no type: nothing around the outputs is written, and rows of no
    type stay as they were."""
    from tinygnn_b200 import _lib
    for M in (20, 90, 700):
        for off in ([0, 40, 5000], [-7, 10, M], [0, M - 5, 12], [M, M, M], [3, 9, M - 4], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
            K, N = 32, 24
            x, dy, w, bias = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype), rand(2, K, N, seed=3, dtype=dtype), rand(2, N, seed=4)
            y, dx = Guarded((M, N), dtype), Guarded((M, K), dtype)
            dw, db = Guarded((2, K, N), dtype), Guarded((2, N), torch.float32, pad=0)
            typed_calls(_lib.lib, x, dy, w, bias, torch.tensor(off, dtype=torch.int32, device="cuda"), y, dx, dw, db)
            c = [min(max(o, 0), M) for o in off]
            own = torch.zeros(M, dtype=torch.bool, device="cuda")
            for t in range(2):
                own[c[t]:max(c[t], c[t + 1])] = True
                n = max(0, c[t + 1] - c[t])
                want = dy[c[t]:c[t] + n].double().sum(0)
                assert ((db.t[t] - want).abs() <= (n + 16) * 2.0 ** -24 * dy[c[t]:c[t] + n].double().abs().sum(0)).all()
            assert y.t[~own].eq(77).all() and dx.t[~own].eq(77).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_type_are_written_whatever_follows_them(tg, dtype):
    """Types whose bounds fall again after their rows: by the few-row kernels (20 rows, 3 for dX) as by tiles (90)."""
    K, N = 32, 24
    for M in (3, 20, 90):
        x, dy, w = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype), rand(3, K, N, seed=3, dtype=dtype)
        off = torch.tensor([0, M - 1, 1, 1], dtype=torch.int32, device="cuda")  # type 0 owns all rows but the last
        y, dx = tg.typed_linear(x, w, off)[:M - 1], tg.typed_linear_grad_input(dy, w, off)[:M - 1]
        xd, dyd, wd = x[:M - 1].double(), dy[:M - 1].double(), w[0].double()
        for got, a, b in ((y, xd, wd), (dx, dyd, wd.T)):
            tol = U[dtype] * (a @ b).abs() + 48 * 2.0 ** -23 * (a.abs() @ b.abs()) + TINY[dtype]
            assert ((got.double() - a @ b).abs() <= tol).all(), M


def lay_out(rows, types, spread):
    """Offsets of `rows` rows over `types` types: a few rows each, or all in the third (first, of fewer) type."""
    if spread:
        o = [rows * t // types for t in range(types + 1)]
    else:
        at = min(2, types - 1)
        o = [0] * (at + 1) + [rows] * (types - at)
    return torch.tensor(o, dtype=torch.int32, device="cuda"), o


# rows, types, K, N at and past the limits between the few-row kernels and tiles (forward, dX, dW), 16-bit and fp32
LIMITS = [(4, 1, 2048, 2048), (5, 1, 2560, 2624), (8, 3, 2048, 2048), (9, 3, 2048, 2048), (32, 2, 1024, 1024),
          (32, 40, 1024, 1032), (4, 5, 1024, 1024), (4, 5, 1024, 1025), (32, 7, 128, 256), (32, 7, 129, 257), (8, 1, 520, 2056),
          (32, 1, 4096, 4096), (32, 1, 4096, 4104), (32, 2, 4096, 4104), (33, 40, 264, 136), (40, 40, 264, 136), (41, 40, 264, 136),
          (200, 200, 41, 43), (1000, 1024, 72, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,types,K,N", LIMITS)
@pytest.mark.parametrize("spread", [True, False])
def test_few_rows_at_the_limits(tg, dtype, rows, types, K, N, spread):
    """Sums of n terms to (n + 16) 2^-23 of their magnitude, and the result's rounding."""
    off, o = lay_out(rows, types, spread)
    x, dy = rand(rows, K, seed=1, dtype=dtype), rand(rows, N, seed=2, dtype=dtype)
    w, bias = rand(types, K, N, seed=3, scale=K ** -0.5, dtype=dtype), rand(types, N, seed=4)

    def near(got, want, mag, terms, u):
        bad = ~((got.double() - want).abs() <= u * want.abs() + (terms + 16) * 2.0 ** -23 * mag + TINY[got.dtype])
        assert not bad.any(), (int(bad.sum()), got[bad][:3], want[bad][:3])

    y, (dx, dw, db) = tg.typed_linear(x, w, off, bias), tg.typed_linear_backward(dy, x, w, off)
    for t in range(types):
        a, b = o[t], o[t + 1]
        if a == b:
            assert dw[t].eq(0).all() and db[t].eq(0).all()
            continue
        xd, dyd, wd = x[a:b].double(), dy[a:b].double(), w[t].double()
        near(y[a:b], xd @ wd + bias[t].double(), xd.abs() @ wd.abs() + bias[t].double().abs(), K, U[dtype])
        near(dx[a:b], dyd @ wd.T, dyd.abs() @ wd.abs().T, N, U[dtype])
        near(dw[t], xd.T @ dyd, xd.abs().T @ dyd.abs(), b - a, U[dtype])
        near(db[t], dyd.sum(0), dyd.abs().sum(0), b - a, U[torch.float32])


def device_us(f, n=5):
    """Median device time of f in us."""
    f()
    times = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[n // 2]


def test_few_rows_have_no_cliffs(tg):
    """Time, to a factor that a busy machine does not reach: rows that share a large weight take no longer than a tile
    of them (33 rows); rows that all lie in one of many types no longer than a few times what they take when spread."""
    w = rand(1, 4096, 4096, seed=1, dtype=torch.bfloat16)
    x = rand(33, 4096, seed=2, dtype=torch.bfloat16)
    off = [torch.tensor([0, r], dtype=torch.int32, device="cuda") for r in range(34)]
    for f, few in ((tg.typed_linear, 32), (tg.typed_linear_grad_input, 4)):
        tile = device_us(lambda: f(x, w, off[33]))
        assert device_us(lambda: f(x[:few], w, off[few])) <= 2 * tile + 10, few
    rows = 256
    x, dy = rand(rows, 1024, seed=3, dtype=torch.bfloat16), rand(rows, 1024, seed=4, dtype=torch.bfloat16)
    one, spread = (device_us(lambda o=lay_out(rows, 256, s)[0]: tg.typed_linear_grad_weight(x, dy, o)) for s in (False, True))
    assert one <= 6 * spread, (one, spread)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [513, 2049, 2056, 2304, 3071, 3073, 4095, 4112, 5121, 5632, 6143, 6144, 6145, 6152, 8191])
def test_layer_norm_at_the_steps_of_its_row_split(tg, dtype, cols):
    """Widths on both sides of every step, aligned and not, more rows than blocks, all outputs.  Sums of at most 32 terms a
    thread and 12 joins of values up to max |x|: 2^-24 * 48 against the row's deviation, doubled for the gradient's."""
    for rows, pad in ((700, 0), (3, 3)):
        x, dy = rand(rows, cols + pad, seed=1, scale=2.0, shift=0.5, dtype=dtype)[:, :cols], rand(rows, cols + pad, seed=2, dtype=dtype)[:, :cols]
        gamma, beta = rand(cols, seed=3, scale=0.3, shift=1.0, dtype=dtype), rand(cols, seed=4, dtype=dtype)
        y, stats, saved = tg.layer_norm(x, gamma, beta, save8=True)
        assert torch.equal(y, tg.layer_norm(x, gamma, beta)[0])
        xd, dyd, g, b = x.double(), dy.double(), gamma.double(), beta.double()
        mean = xd.mean(1, keepdim=True)
        rstd = ((xd - mean) ** 2).mean(1, keepdim=True).add(1e-5) ** -0.5
        h = (xd - mean) * rstd
        slack = 2.0 ** -24 * 48 * (1 + xd.abs().amax(1, keepdim=True) * rstd)
        want = h * g + b
        assert ((y.double() - want).abs() <= U[dtype] * want.abs() + slack * (g.abs() * (1 + h.abs()) + b.abs()) + TINY[dtype]).all()
        held = saved.restore(torch.float32).double()
        step = torch.exp2(saved.exponents.double() - 127).repeat_interleave(128, 1)[:, :cols]
        assert ((held - h).abs() <= 0.5 * step + 2 * slack * (1 + h.abs())).all()
        for given, hh, rough in ((x, h, slack), (saved, held, torch.full_like(slack, 2.0 ** -24 * 48))):
            dx, dg, db = tg.layer_norm_backward(dy, given, stats, gamma)
            gy = dyd * g
            want = rstd * (gy - gy.mean(1, keepdim=True) - hh * (gy * hh).mean(1, keepdim=True))
            mag = gy.abs() + gy.abs().mean(1, keepdim=True) + hh.abs() * (gy * hh).abs().mean(1, keepdim=True)
            tol = U[dtype] * want.abs() + rstd * 4 * (rough + slack) * (1 + hh.abs()) * mag + TINY[dtype]
            assert ((dx.double() - want).abs() <= tol).all()
            n = (rows + 16) * 2.0 ** -24
            for got, want, mag in ((dg, (dyd * hh).sum(0), (dyd * hh).abs() * n + dyd.abs() * rough * (1 + hh.abs())),
                                   (db, dyd.sum(0), dyd.abs() * n)):
                assert ((got.double() - want).abs() <= U[dtype] * want.abs() + mag.sum(0) + TINY[dtype]).all()


def test_what_is_no_truth_value_is_refused(tg):
    """A flag whose truth cannot be told (several elements), and an x of the wrong rank: InvalidArgument, like the others."""
    x, g, off = rand(4, 8), rand(8, seed=1), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    w, several = rand(1, 8, 8, seed=2), torch.zeros(2)
    for call in (lambda: tg.layer_norm(x, g, g, save8=several), lambda: tg.typed_linear(x, w, off, save8=several),
                 lambda: tg.typed_linear_grad_weight(x, x, off, bias=several),
                 lambda: tg.typed_linear_backward(x, x[0], w, off)):
        with pytest.raises(tg.InvalidArgument):
            call()


# Sizes of the types, K, N: products on pairs of CTAs in both directions, more than one tile of 256 columns: last tiles
# of 88 and 8 columns, of 89 and 7 (rows that TMA cannot read: aligned copies first), of one column and of half a tile,
# and whole tiles; types of one row, of none, and one whose values are its own.
PAIRS = [([6001, 0, 1, 5000, 300, 4755, 130], 776, 600), ([6001, 0, 1, 5000, 300, 4755, 130], 775, 601),
         ([9001, 7000, 0, 300], 640, 513), ([20000], 1024, 768)]


def last_kernel():
    from tinygnn_b200 import _lib
    return _lib.lib.tg_last_kernel_name().decode()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(PAIRS)))
def test_products_on_pairs_of_ctas(tg, dtype, case):
    """Sums of n terms to (n + 16) 2^-23 of their magnitude (the tensor cores may truncate) and the result's rounding; the
    8-bit copy to half a step more."""
    sizes, K, N = PAIRS[case]
    M, T = sum(sizes), len(sizes)
    o = [0]
    for n in sizes:
        o.append(o[-1] + n)
    off = torch.tensor(o, dtype=torch.int32, device="cuda")
    x, dy = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype)
    w, bias = rand(T, K, N, seed=3, scale=K ** -0.5, dtype=dtype), rand(T, N, seed=4)
    bad = next((t for t, n in enumerate(sizes) if n == 300), None)
    if bad is not None:
        x[o[bad]:o[bad + 1]], dy[o[bad]:o[bad + 1]] = float("nan"), float("inf")
    y, saved = tg.typed_linear(x, w, off, bias, "relu", save8=True)
    assert last_kernel() == "typed_rows_pair"
    plain = tg.typed_linear(x, w, off)
    assert last_kernel() == "typed_rows_pair"
    dx = tg.typed_linear_grad_input(dy, w, off)
    assert last_kernel() == "typed_rows_pair"

    def near(got, want, tol, what):
        off_by = ~((got.double() - want).abs() <= tol)
        assert not off_by.any(), (what, int(off_by.sum()), off_by.nonzero()[:3], got[off_by][:3], want[off_by][:3])

    for t in range(T):
        r = slice(o[t], o[t + 1])
        if t == bad:
            assert y[r].isnan().all() and dx[r].isnan().all() and plain[r].isnan().all() and saved.exponents[r].eq(255).all()
            continue
        xd, dyd, wd, b = x[r].double(), dy[r].double(), w[t].double(), bias[t].double()
        z, mag = xd @ wd, xd.abs() @ wd.abs()
        near(plain[r], z, U[dtype] * z.abs() + (K + 16) * 2.0 ** -23 * mag + TINY[dtype], f"plain {t}")
        z, err = z + b, (K + 16) * 2.0 ** -23 * (mag + b.abs())
        want = z.clamp(min=0)
        near(y[r], want, U[dtype] * want + err + TINY[dtype], f"y {t}")
        held = tg.Saved8(saved.codes[r], saved.exponents[r], dtype).restore(torch.float32)
        step = torch.exp2(saved.exponents[r].double() - 127).repeat_interleave(128, 1)[:, :N]
        near(held, z, 0.5 * step + err, f"saved {t}")
        top = torch.nn.functional.pad(z.abs(), (0, -N % 128)).view(z.shape[0], (N + 127) // 128, 128).amax(2)
        room = torch.nn.functional.pad(err, (0, -N % 128)).view(z.shape[0], (N + 127) // 128, 128).amax(2)
        e = torch.exp2(saved.exponents[r].double() - 127)
        assert (127 * e >= top - room).all() and (63.5 * e <= top + room).all(), f"exponents {t}"
        near(dx[r], dyd @ wd.T, U[dtype] * (dyd @ wd.T).abs() + (N + 16) * 2.0 ** -23 * (dyd.abs() @ wd.abs().T) + TINY[dtype], f"dx {t}")
    again = tg.typed_linear(x, w, off, bias, "relu"), tg.typed_linear_grad_input(dy, w, off)
    assert torch.equal(again[0].nan_to_num(7.0), y.nan_to_num(7.0)) and torch.equal(again[1].nan_to_num(7.0), dx.nan_to_num(7.0))


def test_routes_of_the_typed_products(tg):
    """Which kernels run on which sides of the rules, so that a test of one of them cannot silently test another."""
    def rows(M, T, K, N, dtype):
        off, _ = lay_out(M, T, True)
        tg.typed_linear(rand(M, K, dtype=dtype), rand(T, K, N, dtype=dtype), off)
        return last_kernel()
    b, f = torch.bfloat16, torch.float32
    assert rows(32, 1, 1024, 1024, b) == "typed_few" and rows(33, 1, 1024, 1024, b) == "typed_rows"
    assert rows(32, 1, 2048, 2048, b) == "typed_rows" and rows(32, 2, 2048, 2048, f) == "typed_few"
    assert rows(33, 2, 256, 256, f) == "typed_any" and rows(20000, 4, 512, 512, b) == "typed_rows"
    assert rows(20000, 4, 520, 512, b) == "typed_rows_pair" and rows(20000, 40, 520, 512, b) == "typed_rows"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,alpha", [("relu", 0.0), ("gelu", 0.0), ("elu", 0.7), (None, 0.0)])
@pytest.mark.parametrize("rows,cols,pad", [(20011, 1000, 0), (20011, 1003, 0), (6001, 1000, 1), (70001, 41, 0), (3, 9000, 0)])
def test_activations_over_many_steps(tg, dtype, act, alpha, rows, cols, pad):
    """More rows than the activation kernels' groups take at once, blocks of columns that do not divide the groups: codes
    and exponents bit for bit, values to the exponential's 2^-20 of max(|x|, 1) and the result's rounding."""
    x, dy = rand(rows, cols + pad, seed=1, scale=2.0, dtype=dtype)[:, :cols], rand(rows, cols + pad, seed=2, dtype=dtype)[:, :cols]
    y, saved = tg.activation_save8(x, act, alpha)
    nb = (cols + 127) // 128
    m, e = torch.frexp(torch.nn.functional.pad(x.float().abs(), (0, nb * 128 - cols)).view(rows, nb, 128).amax(2))
    e = (e - 7 + (m > 127 / 128).int()).clamp(min=-24 if dtype == torch.float16 else -126)
    assert torch.equal(saved.exponents.int(), e + 127)
    scale = torch.exp2(e.double()).repeat_interleave(128, 1)[:, :cols]
    assert torch.equal(saved.codes.double(), torch.round(x.double() / scale))
    assert torch.equal(saved.restore(torch.float32).double(), saved.codes.double() * scale)

    def forms(z):
        zd = z.double().requires_grad_(True)
        v = {"relu": torch.relu, "elu": lambda a: torch.where(a < 0, alpha * torch.expm1(a), a), None: lambda a: a * 1,
             "gelu": lambda a: 0.5 * a * (1 + torch.tanh(0.7978845608 * (a + 0.044715 * a ** 3)))}[act](zd)
        return v.detach(), torch.autograd.grad(v.sum(), zd)[0]

    want, slope = forms(x)
    slack = 2.0 ** -20 * x.double().abs().clamp(min=1)
    assert ((y.double() - want).abs() <= U[dtype] * want.abs() + slack + TINY[dtype]).all()
    for given, s in ((x, slope), (saved, forms(saved.restore(torch.float32))[1])):
        got, want = tg.activation_backward(dy, given, act, alpha), dy.double() * s
        assert ((got.double() - want).abs() <= U[dtype] * want.abs() + slack * dy.double().abs() + TINY[dtype]).all()


def scratch_high(f):
    """The most bytes of the device's default memory pool (the library's scratch) in use while f runs."""
    import ctypes
    cu = ctypes.CDLL("libcuda.so.1")
    pool, value = ctypes.c_void_p(), ctypes.c_uint64(0)
    assert cu.cuDeviceGetDefaultMemPool(ctypes.byref(pool), torch.cuda.current_device()) == 0
    high = 8  # CU_MEMPOOL_ATTR_USED_MEM_HIGH
    torch.cuda.synchronize()
    assert cu.cuMemPoolSetAttribute(pool, high, ctypes.byref(value)) == 0
    f()
    torch.cuda.synchronize()
    assert cu.cuMemPoolGetAttribute(pool, high, ctypes.byref(value)) == 0
    return value.value


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_scratch_is_for_cut_types(tg, dtype):
    """400 types of 512 x 512, one of them long enough to be cut: partial sums for its pieces, not for every type."""
    T, K, N = 400, 512, 512
    sizes = [3] * T
    sizes[7] = 6000
    M = sum(sizes)
    off = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    x, dy = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype)
    out = []
    used = scratch_high(lambda: out.append(tg.typed_linear_grad_weight(x, dy, off)))
    # 2 (148 / 8 tiles + 1) pieces of a MiB and the aligned copies that the route makes (none here)
    assert 0 < used <= 64 << 20, used
    dw, db = out[0]
    for t in (0, 6, 7, 8, 399):
        a, b = int(off[t]), int(off[t + 1])
        xd, dyd = x[a:b].double(), dy[a:b].double()
        want, mag = xd.T @ dyd, xd.abs().T @ dyd.abs()
        assert ((dw[t].double() - want).abs() <= U[dtype] * want.abs() + (b - a + 16) * 2.0 ** -23 * mag + TINY[dtype]).all(), t
        assert ((db[t].double() - dyd.sum(0)).abs() <= (b - a + 16) * 2.0 ** -24 * dyd.abs().sum(0)).all(), t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("types", [37, 300])
@pytest.mark.parametrize("K,N", [(40, 72), (264, 200)])
def test_weight_gradients_of_cut_whole_and_empty_types(tg, dtype, types, K, N):
    """Types of every kind in one call (more than 256 keep their order, fewer run longest first): each whole type's
    gradient and each cut one's sum of pieces, from both forms of x, dW of both types."""
    g = torch.Generator().manual_seed(types)
    sizes = [(0, 1, 63, 64, 65, 200, 1500, 9000)[int(k)] for k in torch.randint(8, (types,), generator=g)]
    if types > 256:
        sizes = [n if t % 9 == 0 else n % 64 for t, n in enumerate(sizes)]
    M = sum(sizes)
    o = [0] + torch.tensor(sizes).cumsum(0).tolist()
    off = torch.tensor(o, dtype=torch.int32, device="cuda")
    x, dy = rand(M, K, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype)
    saved = tg.save8(x)
    for given, wide in ((x, None), (saved, None), (x, torch.float32)):
        dw, db = tg.typed_linear_grad_weight(given, dy, off, dtype=wide)
        xs = given.double() if given is x else given.restore(torch.float32).double()
        for t in range(types):
            xd, dyd, n = xs[o[t]:o[t + 1]], dy[o[t]:o[t + 1]].double(), sizes[t]
            want, mag = xd.T @ dyd, xd.abs().T @ dyd.abs()
            assert ((dw[t].double() - want).abs() <= U[dw.dtype] * want.abs() + (n + 16) * 2.0 ** -23 * mag + TINY[dw.dtype]).all(), t
            assert ((db[t].double() - dyd.sum(0)).abs() <= (n + 16) * 2.0 ** -24 * dyd.abs().sum(0)).all(), t
        again = tg.typed_linear_grad_weight(given, dy, off, dtype=wide)
        assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_a_refused_cuda_call_is_not_reported_again(tg):
    """A call that the CUDA runtime refuses (a synchronisation inside a capture) fails by itself; the next call, which
    has nothing wrong, succeeds."""
    import ctypes
    from tinygnn_b200 import _lib
    cu, lib = ctypes.CDLL("libcuda.so.1"), _lib.lib
    off, x = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), rand(4, 8)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    handle, graph = ctypes.c_void_p(stream.cuda_stream), ctypes.c_void_p()
    assert cu.cuStreamBeginCapture_v2(handle, 2) == 0  # relaxed: this stream only
    try:
        status = lib.tg_typed_check_offsets(4, 1, off.data_ptr(), stream.cuda_stream)
    finally:
        cu.cuStreamEndCapture(handle, ctypes.byref(graph))
    assert status == _lib.CUDA
    y = x.clone()
    tg.relu_(y)  # (checks the runtime's last error after its launch)
    assert torch.equal(y, x.clamp(min=0))
    tg.check_row_offsets(off, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_very_wide_outputs(tg, dtype):
    """More columns than 65,535 tiles of any kernel: products of one input column, exact but for the result's rounding;
    sums of nine rows."""
    M, N = 9, 65536 * 256 + 300
    x, dy = rand(M, 1, seed=1, dtype=dtype), rand(M, N, seed=2, dtype=dtype)
    w, off = rand(1, 1, N, seed=3, dtype=dtype), torch.tensor([0, M], dtype=torch.int32, device="cuda")
    dw, db = tg.typed_linear_grad_weight(x, dy, off)
    for c in (slice(0, 1000), slice(N - 1000, N)):
        xd, dyd = x.double(), dy[:, c].double()
        want, mag = (xd * dyd).sum(0), (xd * dyd).abs().sum(0)
        assert ((dw[0, 0, c].double() - want).abs() <= U[dtype] * want.abs() + 25 * 2.0 ** -23 * mag + TINY[dtype]).all()
        assert ((db[0, c].double() - dyd.sum(0)).abs() <= 25 * 2.0 ** -24 * dyd.abs().sum(0)).all()
    for rows in (M, 40):
        xs = rand(rows, 1, seed=4, dtype=dtype)
        y = tg.typed_linear(xs, w, torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
        want = xs.double() * w[0, 0, -1000:].double()
        assert ((y[:, -1000:].double() - want).abs() <= (U[dtype] + 2.0 ** -22) * want.abs() + TINY[dtype]).all()
        del y
