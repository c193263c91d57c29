"""Group norm with an activation over the rows of graphs, and its gradient,
against a plain 64-bit implementation.

Tolerances follow from the arithmetic: statistics are fp32 sums of at most 64
terms of a thread and 32 lanes, and of a graph's parts (64 a thread and 8
joins), 2^-24 of the values each; results are rounded once to their type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
ACTS = [(None, 0.0), ("relu", 0.0), ("leaky_relu", 0.2), ("elu", 0.7), ("sigmoid", 0.0), ("tanh", 0.0), ("gelu", 0.0)]
EPS = 1e-5


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def rand(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def strided(t, pad, offset):
    rows, cols = t.shape
    buf = torch.full((rows * (cols + pad) + offset + 1,), float("nan"), dtype=t.dtype, device=t.device)
    v = torch.as_strided(buf, (rows, cols), (cols + pad, 1), offset)
    v.copy_(t)
    return v


def offsets_of(sizes):
    o = [0]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def assert_within(got, ref, tol, what=""):
    got = got.double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} outside; first at {i}: {got[i]} vs {ref[i]}")


def act64(u, act, alpha):
    if act == "relu":
        return torch.relu(u)
    if act == "leaky_relu":
        return torch.where(u >= 0, u, alpha * u)
    if act == "elu":
        return torch.where(u < 0, alpha * torch.expm1(u), u)
    if act == "sigmoid":
        return torch.sigmoid(u)
    if act == "tanh":
        return torch.tanh(u)
    if act == "gelu":
        return torch.nn.functional.gelu(u, approximate="tanh")
    return u


def slope64(u, act, alpha):
    u = u.detach().requires_grad_(True)
    return torch.autograd.grad(act64(u, act, alpha).sum(), u)[0]


class Plain:
    """The formulas, graph by graph."""

    def __init__(self, x, gamma, beta, sizes, groups, act, alpha, eps=EPS):
        self.sizes, self.groups, self.act, self.alpha = sizes, groups, act, alpha
        self.x, self.gamma, self.beta = x.double(), gamma.double(), beta.double()
        self.mean, self.r = torch.zeros_like(self.x), torch.zeros_like(self.x)
        self.stats = torch.zeros(len(sizes), groups, 2, dtype=torch.float64, device=x.device)
        for g, (a, b) in enumerate(self.spans()):
            if a == b:
                continue
            v = self.x[a:b].view(b - a, groups, -1)
            m = v.mean((0, 2), keepdim=True)
            r = ((v - m) ** 2).mean((0, 2), keepdim=True).add(eps).rsqrt()
            self.stats[g, :, 0], self.stats[g, :, 1] = m.flatten(), r.flatten()
            self.mean[a:b], self.r[a:b] = m.expand_as(v).reshape(b - a, -1), r.expand_as(v).reshape(b - a, -1)
        self.h = (self.x - self.mean) * self.r
        self.u = self.h * self.gamma + self.beta
        self.y = act64(self.u, act, alpha)

    def spans(self):
        o = 0
        for s in self.sizes:
            yield o, o + s
            o += s

    def over(self, v):
        """The mean over each graph's rows and each group's columns, at each row and column."""
        out = torch.zeros_like(v)
        for a, b in self.spans():
            if a < b:
                w = v[a:b].view(b - a, self.groups, -1)
                out[a:b] = w.mean((0, 2), keepdim=True).expand_as(w).reshape(b - a, -1)
        return out

    def largest(self, v):
        out = torch.zeros_like(v)
        for a, b in self.spans():
            if a < b:
                w = v[a:b].abs().view(b - a, self.groups, -1)
                out[a:b] = w.amax((0, 2), keepdim=True).expand_as(w).reshape(b - a, -1)
        return out

    def slack(self):
        """What the statistics' roundings move h by, in units of 1 + |h|: about 2^-24 (64 + 32 + 64 + 8) of the
        values' distance from the part's first, which is at most twice the largest from the mean."""
        return 2.0 ** -24 * 168 * (1 + 2 * self.largest(self.x - self.mean) * self.r) + 2.0 ** -23 * self.mean.abs() * self.r

    def grad(self, dy):
        self.s = slope64(self.u, self.act, self.alpha)
        du = dy.double() * self.s
        g = du * self.gamma
        return du, g, self.r * (g - self.over(g) - self.h * self.over(g * self.h))


def check(tg, x, dy, gamma, beta, sizes, groups, act, alpha, offsets="make", what=""):
    dtype, pdtype = x.dtype, gamma.dtype
    off = offsets_of(sizes) if offsets == "make" else offsets
    y, stats = tg.group_norm(x, gamma, beta, groups, off, act, alpha, EPS)
    ref = Plain(x, gamma, beta, sizes, groups, act, alpha)
    slack = ref.slack()
    # the activation's slope is at most 1.13, its own error 2^-16 of its value (16 bits) or 2^-20 (fp32)
    own = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -16
    tol_u = slack * (ref.gamma.abs() * (1 + ref.h.abs()) + ref.beta.abs())
    assert_within(y, ref.y, U[dtype] * ref.y.abs() + 1.13 * tol_u + own * ref.y.abs() + TINY[dtype], f"{what} y")
    full = [i for i, s in enumerate(sizes) if s]
    assert stats.shape == (len(sizes), groups, 2)
    for g in range(len(sizes)):
        if g not in full:
            assert stats[g].eq(0).all()
    dx, dg, db = tg.group_norm_backward(dy, x, stats, gamma, beta, groups, off, act, alpha)
    du, gg, want = ref.grad(dy)
    # the slope's error: its change over u's error (a second derivative is at most 1.2, but relu's and elu's slopes jump
    # at 0: values within u's error of it are left out), and its own
    kink = (ref.u.abs() <= tol_u) if act in ("relu", "leaky_relu", "elu") else torch.zeros_like(ref.u, dtype=torch.bool)
    tol_du = dy.double().abs() * (1.2 * tol_u + own) + du.abs() * 2.0 ** -22 + torch.where(kink, dy.double().abs(), 0.0)
    tol_g = tol_du * ref.gamma.abs()
    count = 2.0 ** -24 * 168
    mean_tol = ref.over(tol_g) + count * ref.over(gg.abs())
    h_tol = ref.over(tol_g * ref.h.abs() + gg.abs() * slack * (1 + ref.h.abs())) + count * ref.over((gg * ref.h).abs())
    mag = gg.abs() + ref.over(gg.abs()) + ref.h.abs() * ref.over((gg * ref.h).abs())
    tol = ref.r * (tol_g + mean_tol + ref.h.abs() * h_tol + 4 * slack * (1 + ref.h.abs()) * mag)
    assert_within(dx, want, U[dtype] * want.abs() + tol + TINY[dtype], f"{what} dx")
    rows = x.shape[0]
    n = 2.0 ** -24 * (rows / 32 + 168)
    wg, wb = (du * ref.h).sum(0), du.sum(0)
    tol_dg = (tol_du * ref.h.abs() + du.abs() * slack * (1 + ref.h.abs()) + n * (du * ref.h).abs()).sum(0)
    assert_within(dg, wg, U[pdtype] * wg.abs() + tol_dg + TINY[pdtype], f"{what} dgamma")
    assert_within(db, wb, U[pdtype] * wb.abs() + (tol_du + n * du.abs()).sum(0) + TINY[pdtype], f"{what} dbeta")
    return y, stats, dx, dg, db


def inputs(rows, cols, dtype, pdtype, seed):
    return (rand(rows, cols, seed=seed, scale=2.0, shift=1.5, dtype=dtype), rand(rows, cols, seed=seed + 1, dtype=dtype),
            rand(cols, seed=5, scale=0.3, shift=1.0, dtype=pdtype), rand(cols, seed=6, dtype=pdtype))


# (columns, groups): every width of a vector and of a block's rows, odd groups, groups of one column, several blocks wide.
SHAPES = [(1, 1), (3, 3), (8, 1), (8, 8), (24, 3), (64, 1), (64, 16), (96, 4), (128, 8), (130, 2), (320, 32), (513, 1), (1024, 8),
          (2048, 4), (4104, 1), (4104, 513), (5000, 8)]
SIZES = [[1], [5, 0, 1, 0, 40, 3], [300], [2, 2, 2, 500, 1, 1, 129]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,groups", SHAPES)
def test_group_norm(tg, dtype, cols, groups):
    for k, sizes in enumerate(SIZES):
        rows = sum(sizes)
        act, alpha = ACTS[(k + cols) % len(ACTS)]
        x, dy, gamma, beta = inputs(rows, cols, dtype, dtype if k % 2 else torch.float32, seed=cols + k)
        if k == 1:
            x, dy = strided(x, 5, 3), strided(dy, 5, 3)
        if k == 3:
            x, dy = strided(x, 8, 0), strided(dy, 16, 8)
        check(tg, x, dy, gamma, beta, sizes, groups, act, alpha, what=f"{sizes} {act}")
    check(tg, x, dy, gamma, beta, [rows], groups, None, 0.0, offsets=None, what="no offsets")


@pytest.mark.parametrize("act,alpha", ACTS)
def test_activations(tg, act, alpha):
    for dtype in DTYPES:
        x, dy, gamma, beta = inputs(700, 48, dtype, torch.float32, seed=3)
        check(tg, x, dy, gamma, beta, [100, 250, 350], 6, act, alpha, what=f"{dtype}")


def test_many_graphs_and_repeats(tg):
    """More chunks than blocks, more graphs than a warp finds in one step, a graph of most rows; the same bits again."""
    g = torch.Generator().manual_seed(1)
    for cols, groups, dtype in ((64, 1, torch.float32), (16, 4, torch.bfloat16), (128, 8, torch.float16)):
        sizes = torch.randint(0, 12, (3000,), generator=g).tolist()
        sizes[1234] = 40000
        rows = sum(sizes)
        x, dy, gamma, beta = inputs(rows, cols, dtype, torch.float32, seed=7)
        first = check(tg, x, dy, gamma, beta, sizes, groups, "gelu", 0.0)
        off = offsets_of(sizes)
        y, stats = tg.group_norm(x, gamma, beta, groups, off, "gelu")
        again = (y, stats, *tg.group_norm_backward(dy, x, stats, gamma, beta, groups, off, "gelu"))
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize("cols,groups,dtype", [(64, 1, torch.float32), (48, 16, torch.bfloat16), (37, 37, torch.float16),
                                               (320, 32, torch.float16), (1000, 8, torch.bfloat16)])
def test_large_graphs_among_small_ones(tg, cols, groups, dtype):
    """Several graphs larger than a block's among many of few rows or none, neighbours and apart, first and last; all in
    one; and all alike, at the block's limit and one past it."""
    g = torch.Generator().manual_seed(cols)
    limit = max(65536 // (cols * (4 if dtype == torch.float32 else 2)), 1)
    small = torch.randint(0, 6, (700,), generator=g).tolist()
    mixed = [3 * limit] + small[:200] + [limit + 1, 2 * limit + 5, 0, limit, limit - 1] + small[200:] + [5 * limit + 1]
    for sizes in (mixed, [0] * 50 + [4 * limit + 3] + [1] * 300, [limit] * 3 + [0] * 40, [limit + 1] * 3 + [0] * 40):
        x, dy, gamma, beta = inputs(sum(sizes), cols, dtype, torch.float32, seed=cols)
        check(tg, x, dy, gamma, beta, sizes, groups, "gelu", 0.0, what=f"{len(sizes)} graphs")


def test_one_large_graph(tg):
    for dtype in (torch.float32, torch.bfloat16):
        x, dy, gamma, beta = inputs(100003, 40, dtype, dtype, seed=2)
        check(tg, x, dy, gamma, beta, [100003], 5, "relu", 0.0)


def test_means_far_from_zero(tg):
    """A mean of 1000 deviations, and one value of 10,000: the deviations are not lost."""
    x = rand(5000, 32, seed=1) + 1000.0
    ref = Plain(x, torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"), [5000], 4, None, 0.0)
    _, stats = tg.group_norm(x, torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"), 4)
    # the mean is a number of 2^10: half a step of it, and of each of the sums' 168 steps over deviations of a few
    assert ((stats[..., 0].double() - ref.stats[..., 0]).abs() <= 2.0 ** -14 * 2).all()
    assert ((stats[..., 1].double() / ref.stats[..., 1] - 1).abs() <= 2.0 ** -24 * 400).all()
    x = rand(5000, 32, seed=1)
    x[0] = 10000.0
    ref = Plain(x, torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"), [5000], 4, None, 0.0)
    _, stats = tg.group_norm(x, torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"), 4)
    assert ((stats[..., 1].double() / ref.stats[..., 1] - 1).abs() <= 2.0 ** -24 * 400).all()


def test_constant_and_nan_graphs(tg):
    x = torch.full((30, 16), 2.5, device="cuda")
    x[12, 3] = float("nan")
    gamma, beta = rand(16, seed=1), rand(16, seed=2)
    y, stats = tg.group_norm(x, gamma, beta, 2, offsets_of([10, 10, 10]))
    assert torch.equal(y[:10], beta.expand(10, 16)) and torch.equal(y[20:], beta.expand(10, 16))
    assert y[10:20, :8].isnan().all() and torch.equal(y[10:20, 8:], beta[8:].expand(10, 8))


def test_layer_norm_is_the_group_norm_of_single_rows(tg):
    """Graphs of one row each and one group are layer norm (within both's roundings)."""
    x, dy, gamma, beta = inputs(64, 200, torch.float32, torch.float32, seed=1)
    off = torch.arange(65, dtype=torch.int32, device="cuda")
    y, stats = tg.group_norm(x, gamma, beta, 1, off)
    z, zstats = tg.layer_norm(x, gamma, beta)
    assert (y - z).abs().max() <= 2.0 ** -24 * 168 * 8
    assert (stats[:, 0] - zstats).abs().max() <= 2.0 ** -24 * 168


def test_gradient_against_differences(tg):
    """Central differences of sum(y dy) along random directions (see layer norm's)."""
    sizes, groups = [7, 0, 20, 13], 4
    x, dy, gamma, beta = inputs(40, 48, torch.float32, torch.float32, seed=1)
    off = offsets_of(sizes)
    _, stats = tg.group_norm(x, gamma, beta, groups, off, "gelu")
    grads = tg.group_norm_backward(dy, x, stats, gamma, beta, groups, off, "gelu")
    loss = lambda x, g, b: float((tg.group_norm(x, g, b, groups, off, "gelu")[0].double() * dy.double()).sum())  # noqa: E731
    for k, p in enumerate((x, gamma, beta)):
        v = rand(*p.shape, seed=10 + k)
        hs = 2.0 ** -6
        up, down = [x, gamma, beta], [x, gamma, beta]
        up[k], down[k] = p + hs * v, p - hs * v
        diff = (loss(*up) - loss(*down)) / (2 * hs)
        want = float((grads[k].double() * v.double()).sum())
        scale = float(grads[k].double().norm() * v.double().norm())
        assert abs(diff - want) <= 2e-3 * (abs(want) + scale), (k, diff, want)


def test_no_rows_and_no_graphs(tg):
    x, dy, gamma, beta = inputs(0, 16, torch.bfloat16, torch.bfloat16, seed=1)
    for off, graphs in ((None, 1), (offsets_of([0, 0]), 2), (offsets_of([]), 0)):
        y, stats = tg.group_norm(x, gamma, beta, 4, off)
        assert y.shape == (0, 16) and stats.shape == (graphs, 4, 2) and stats.eq(0).all()
        dx, dg, db = tg.group_norm_backward(dy, x, stats, gamma, beta, 4, off)
        assert dx.shape == (0, 16) and dg.eq(0).all() and db.eq(0).all()


def test_rows_of_no_graph_are_left_alone(tg):
    """Rows before the first offset and after the last, and offsets out of range: nothing else is written."""
    from tinygnn_b200 import _lib
    x, dy, gamma, beta = inputs(200, 32, torch.float32, torch.float32, seed=4)
    s = torch.cuda.current_stream().cuda_stream
    for off, spans in (([10, 60, 150], [(10, 60), (60, 150)]), ([-5, 60, 900], [(0, 60), (60, 200)])):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        y = torch.full((200, 40), 7.0, device="cuda")
        stats = torch.empty(2, 4, 2, device="cuda")
        st = _lib.lib.tg_group_norm(200, 32, 4, 2, o.data_ptr(), _lib.F32, x.data_ptr(), 32, _lib.F32, gamma.data_ptr(),
                                    beta.data_ptr(), EPS, 0, 0.0, y.data_ptr(), 40, stats.data_ptr(), s)
        assert st == _lib.OK
        dx = torch.full((200, 40), 7.0, device="cuda")
        dg, db = torch.empty(32, device="cuda"), torch.empty(32, device="cuda")
        st = _lib.lib.tg_group_norm_grad(200, 32, 4, 2, o.data_ptr(), _lib.F32, dy.data_ptr(), 32, x.data_ptr(), 32, stats.data_ptr(),
                                         _lib.F32, gamma.data_ptr(), beta.data_ptr(), 0, 0.0, dx.data_ptr(), 40, dg.data_ptr(),
                                         db.data_ptr(), s)
        assert st == _lib.OK
        inside = torch.zeros(200, dtype=torch.bool, device="cuda")
        for a, b in spans:
            inside[a:b] = True
            want = tg.group_norm(x[a:b], gamma, beta, 4)[0]
            assert (y[a:b, :32] - want).abs().max() <= 2.0 ** -24 * 168 * 8
        assert y[~inside].eq(7.0).all() and y[:, 32:].eq(7.0).all()
        assert dx[~inside].eq(7.0).all() and dx[:, 32:].eq(7.0).all()
        assert (dg - tg.group_norm_backward(dy[inside], x[inside], stats, gamma, beta, 4,
                                            offsets_of([b - a for a, b in spans]))[1]).abs().max() <= 2.0 ** -24 * 168 * 200


# ── streams, graphs, refusals ────────────────────────────────────────────────
def _everything(tg, x, dy, gamma, beta, off):
    y, stats = tg.group_norm(x, gamma, beta, 8, off, "gelu")
    return [y, stats, *tg.group_norm_backward(dy, x, stats, gamma, beta, 8, off, "gelu")]


def test_runs_on_the_current_stream_and_captures(tg):
    args = (*inputs(1000, 64, torch.bfloat16, torch.float32, seed=1), offsets_of([10, 0, 490, 500]))
    want = _everything(tg, *args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        got = _everything(tg, *[t.clone() for t in args])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = []
    for _ in range(2):
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


def test_refusals(tg):
    x, dy, gamma, beta = inputs(30, 24, torch.float32, torch.float32, seed=1)
    off = offsets_of([10, 20])
    y, stats = tg.group_norm(x, gamma, beta, 4, off)
    bad = [
        lambda: tg.group_norm(x, gamma, beta, 5, off),
        lambda: tg.group_norm(x, gamma, beta, 0, off),
        lambda: tg.group_norm(x, gamma, beta, -4, off),
        lambda: tg.group_norm(x, gamma[:23], beta, 4, off),
        lambda: tg.group_norm(x, gamma, beta.bfloat16(), 4, off),
        lambda: tg.group_norm(x, gamma.half(), beta.half(), 4, off),
        lambda: tg.group_norm(x.double(), gamma, beta, 4, off),
        lambda: tg.group_norm(x.cpu(), gamma, beta, 4, off),
        lambda: tg.group_norm(x, gamma, beta, 4, off.long()),
        lambda: tg.group_norm(x, gamma, beta, 4, off.cpu()),
        lambda: tg.group_norm(x, gamma, beta, 4, off[:0]),
        lambda: tg.group_norm(x, gamma, beta, 4, off, "softplus"),
        lambda: tg.group_norm(x, gamma, beta, 4, off, None, 0.0, -1.0),
        lambda: tg.group_norm_backward(dy[:29], x, stats, gamma, beta, 4, off),
        lambda: tg.group_norm_backward(dy, x.half(), stats, gamma, beta, 4, off),
        lambda: tg.group_norm_backward(dy, x, stats[:1], gamma, beta, 4, off),
        lambda: tg.group_norm_backward(dy, x, stats, gamma, beta, 8, off),
        lambda: tg.group_norm_backward(dy, x, stats, gamma, beta, 4),
        lambda: tg.group_norm_backward(dy, x, stats.double(), gamma, beta, 4, off),
    ]
    for k, f in enumerate(bad):
        with pytest.raises((ValueError, tg.InvalidArgument)):
            f()
            raise RuntimeError(f"call {k} was not refused")


def test_c_abi_refusals(tg):
    from tinygnn_b200 import _lib
    lib = _lib.lib
    p = rand(64).data_ptr()

    def fwd(rows=4, cols=8, groups=2, graphs=1, off=None, dtype=0, x=p, ldx=8, pd=0, act=0, ldy=8, stats=p):
        return lib.tg_group_norm(rows, cols, groups, graphs, off, dtype, x, ldx, pd, p, p, EPS, act, 0.0, p, ldy, stats, None)

    def bwd(groups=2, graphs=1, off=None, dtype=0, dy=p, lddy=8, lddx=8, act=0, stats=p):
        return lib.tg_group_norm_grad(4, 8, groups, graphs, off, dtype, dy, lddy, p, 8, stats, 0, p, p, act, 0.0, p, lddx, p, p, None)
    calls = [fwd(rows=-1), fwd(rows=2 ** 31 - 1), fwd(cols=0), fwd(groups=3), fwd(graphs=2), fwd(graphs=-1), fwd(graphs=1 << 25, off=p), fwd(dtype=4),
             fwd(x=None), fwd(ldx=7), fwd(pd=1), fwd(act=9), fwd(ldy=7), fwd(stats=None), fwd(stats=p + 4), bwd(groups=3),
             bwd(graphs=0), bwd(dtype=9), bwd(dy=None), bwd(lddy=7), bwd(lddx=7), bwd(act=-1), bwd(stats=None)]
    assert calls == [_lib.INVALID_ARGUMENT] * len(calls)
