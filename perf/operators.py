"""The training operators' workloads: layer norm, typed (grouped) linear maps and
8-bit activation checkpoints.

Each case is one pass a training or serving program makes.  ``own`` False
computes it with elementary torch operations in 32 bits, rounded once at the
end; ``own`` True makes the calls of :mod:`tinygnn_b200`.  ``exact`` computes
the same from the definitions in 64 bits.

The passes (``op``):

* ``norm``     layer norm forward and its backward pass, from the input or
               (``saved8``) from an 8-bit copy of the normalised rows.
* ``act``      an activation that saves its input in 8 bits, and its backward
               pass from that copy.
* ``typed``    rows sorted by type through their type's weight, bias and
               activation; with ``saved8`` also the pre-activation kept in
               8 bits and the activation's backward pass from it.
* ``typed_grad``  the gradients of input, weight and bias of a typed linear
               map; with ``saved8`` its input is held in 8 bits.

An 8-bit copy holds, for each row and each block of 128 columns, the least
power of two 2^e with max|x| <= 127 2^e, and round-to-even(x / 2^e).
"""
import itertools
import math

import numpy as np
import torch

own = False

BLOCK = 128  # columns that share an exponent in an 8-bit copy
TILE = 512   # rows of one type that the plain form multiplies at a time

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ── cases ────────────────────────────────────────────────────────────────────
def listed():
    return [
        # A small citation graph's hidden rows in fp32: latency.
        dict(name="norm small", op="norm", rows=2708, cols=16, dtype="float32", saved8=False),
        # The hidden rows of a graph of 232,965 nodes.
        dict(name="norm nodes", op="norm", rows=232965, cols=128, dtype="bfloat16", saved8=False),
        # Wide rows of an odd width, the normalised rows kept in 8 bits.
        dict(name="norm wide saved8", op="norm", rows=8191, cols=4099, dtype="float16", saved8=True),
        # Class scores of a small graph (41 columns) through an activation.
        dict(name="act small", op="act", rows=2708, cols=41, dtype="float32", act="elu"),
        # The hidden activations of a large feed-forward layer.
        dict(name="act large", op="act", rows=131072, cols=1024, dtype="bfloat16", act="gelu"),
        # Serving: eight rows, one token or node each, through 64 experts' weights.
        dict(name="typed serve", op="typed", rows=8, k=1024, n=1024, types=64, skew=1.0, dtype="bfloat16",
             act="gelu", saved8=False),
        # Raw features of 602 columns, five node types, fp32.
        dict(name="typed nodes f32", op="typed", rows=232965, k=602, n=128, types=5, skew=1.0, dtype="float32",
             act="relu", saved8=False),
        # The largest forward product: sixteen experts.
        dict(name="typed large", op="typed", rows=65536, k=2048, n=2048, types=16, skew=0.5, dtype="bfloat16",
             act="gelu", saved8=True),
        # A minibatch of a graph with many relation types, fp16.
        dict(name="typed relations", op="typed", rows=20011, k=128, n=256, types=40, skew=2.0, dtype="float16",
             act="relu", saved8=False),
        # Its gradients in fp32, a narrow odd output.
        dict(name="grad relations f32", op="typed_grad", rows=20011, k=128, n=41, types=7, skew=1.5,
             dtype="float32", saved8=False),
        # Gradients of an expert layer.
        dict(name="grad large", op="typed_grad", rows=32768, k=1024, n=2048, types=8, skew=0.5, dtype="bfloat16",
             saved8=False),
        # Gradients of an expert layer whose input was kept in 8 bits.
        dict(name="grad large saved8", op="typed_grad", rows=65536, k=1024, n=1024, types=8, skew=1.0,
             dtype="bfloat16", saved8=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    w = _spread(rng, low, high)
    return w if rng.random() < 0.34 else max(8, w // 8 * 8)


def draw(rng):
    op = rng.choice(["norm", "act", "typed", "typed", "typed_grad", "typed_grad"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    half = dtype != "float32"
    acts = ["relu", "elu", "leaky_relu", "sigmoid", "tanh", "gelu"]
    if op in ("norm", "act"):
        cols = _width(rng, 8, 8192)
        rows = _spread(rng, 1, min(262144, 2 ** 27 // cols))
        if op == "norm":
            return dict(op=op, rows=rows, cols=cols, dtype=dtype, saved8=half and rng.random() < 0.5)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, act=rng.choice(acts))
    k, n = _width(rng, 16, 2048), _width(rng, 16, 2048)
    rows = _spread(rng, 1, min(262144, int((2.5e11 if half else 1.2e11) / (k * n))))
    case = dict(op=op, rows=rows, k=k, n=n, types=_spread(rng, 1, 64), skew=round(rng.uniform(0.0, 2.5), 2), dtype=dtype)
    if op == "typed":
        return dict(case, act=rng.choice(acts), saved8=half and rng.random() < 0.3)
    return dict(case, saved8=rng.random() < 0.4)


def _sizes(case):
    """Rows of each type: uneven (weights spread evenly over (0, 1], to the power `skew`), in no order, some zero."""
    t, rows = case["types"], case["rows"]
    w = [(((i + 1) * 0.6180339887) % 1.0) ** case["skew"] for i in range(t)]
    ends = [min(rows, int(rows * acc / sum(w))) for acc in itertools.accumulate(w)]
    ends[-1] = rows
    return [b - a for a, b in zip([0] + ends, ends)]


# ── inputs ───────────────────────────────────────────────────────────────────
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _hidden(rows, cols, dtype, g):
    """Hidden activations: normal values around a mean of each column's own, some columns several times larger."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= 0.5 + torch.rand(cols, device="cuda", generator=g) * 1.5
    x += torch.randn(cols, device="cuda", generator=g) * 0.5
    x *= 1.0 + 7.0 * (torch.rand(cols, device="cuda", generator=g) < 0.02)
    return x.to(dtype)


def _least(dtype):
    """The least exponent of a block: fp16 rows keep theirs where fp16 can hold the values."""
    return -24 if dtype == torch.float16 else -126


def _saved8(x, emin):
    """(codes int8, exponents uint8) of x."""
    rows, cols = x.shape
    nb = (cols + BLOCK - 1) // BLOCK
    v = torch.zeros(rows, nb * BLOCK, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, nb, BLOCK)
    m, e = torch.frexp(v.abs().amax(2))
    e = (e - 7 + (m > 127 / 128).int()).clamp(min=emin)
    codes = torch.round(v * _pow2(-e)[:, :, None]).to(torch.int8).view(rows, nb * BLOCK)[:, :cols]
    return codes, (e + 127).to(torch.uint8)


def _pow2(e):
    """2^e of integers e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values8(codes, exponents):
    scale = _pow2(exponents.to(torch.int32) - 127).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * scale


def prepare(case, seed):
    g = _generator(seed)
    dtype, rows = DTYPES[case["dtype"]], case["rows"]
    s = dict(case=dict(case))
    if case["op"] == "norm":
        c = case["cols"]
        s["x"] = _hidden(rows, c, dtype, g)
        s["dy"] = torch.randn(rows, c, device="cuda", generator=g).mul_(0.1).to(dtype)
        s["gamma"] = (1.0 + 0.2 * torch.randn(c, device="cuda", generator=g)).to(dtype)
        s["beta"] = (0.2 * torch.randn(c, device="cuda", generator=g)).to(dtype)
        return s
    if case["op"] == "act":
        s["x"] = _hidden(rows, case["cols"], dtype, g)
        s["dy"] = torch.randn(rows, case["cols"], device="cuda", generator=g).mul_(0.1).to(dtype)
        return s
    k, n, types = case["k"], case["n"], case["types"]
    sizes = _sizes(case)
    s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")
    s["w"] = (torch.randn(types, k, n, device="cuda", generator=g) / math.sqrt(k)).to(dtype)
    x = _hidden(rows, k, dtype, g)
    s["dy"] = torch.randn(rows, n, device="cuda", generator=g).mul_(0.1).to(dtype)
    if case["op"] == "typed":
        s["x"] = x
        s["bias"] = 0.1 * torch.randn(types, n, device="cuda", generator=g)
    elif case["saved8"]:
        # Rows of codes start at multiples of 16 bytes, as the library lays them out.
        ld = (k + 15) // 16 * 16
        codes, s["exponents"] = _saved8(x, _least(dtype))
        buf = torch.zeros(rows, ld, dtype=torch.int8, device="cuda")
        buf[:, :k] = codes
        s["codes"] = buf[:, :k]
    else:
        s["x"] = x
    # The plain form's plan: the rows of each type in tiles of at most TILE rows.
    tile_type, tile_row, where, start = [], [], [], 0
    for t, m in enumerate(sizes):
        for r in range(0, m, TILE):
            where.append(np.arange(min(TILE, m - r)) + len(tile_type) * TILE)
            tile_type.append(t)
            tile_row.append(start + r)
        start += m
    ends = torch.cumsum(torch.tensor(sizes), 0)
    tt = torch.tensor(tile_type)
    idx = torch.tensor(tile_row)[:, None] + torch.arange(TILE)
    inside = idx < ends[tt][:, None]
    s["tile_type"], s["tile_inside"] = tt.cuda(), inside.cuda()
    s["tile_rows"] = torch.where(inside, idx, 0).cuda()
    s["row_place"] = torch.tensor(np.concatenate(where)).cuda()
    s["row_type"] = torch.repeat_interleave(torch.arange(types), torch.tensor(sizes)).cuda()
    return s


# ── the passes ───────────────────────────────────────────────────────────────
def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "leaky_relu":
        return torch.where(z >= 0, z, 0.01 * z)
    if act == "elu":
        return torch.where(z < 0, torch.exp(z) - 1, z)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    return 0.5 * z * (1 + torch.tanh(0.7978845608 * (z + 0.044715 * z * z * z)))


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "leaky_relu":
        return torch.where(z >= 0, 1.0, 0.01).to(z.dtype)
    if act == "elu":
        return torch.where(z < 0, torch.exp(z), 1.0)
    if act == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 - p)
    if act == "tanh":
        p = torch.tanh(z)
        return 1 - p * p
    p = torch.tanh(0.7978845608 * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + p) + 0.5 * z * (1 - p * p) * 0.7978845608 * (1 + 3 * 0.044715 * z * z)


ALPHA = {"leaky_relu": 0.01, "elu": 1.0}
EPS = 1e-5


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import tinygnn_b200 as tg
    c = s["case"]
    if c["op"] == "norm":
        if c["saved8"]:
            y, stats, saved = tg.layer_norm(s["x"], s["gamma"], s["beta"], EPS, save8=True)
        else:
            y, stats = tg.layer_norm(s["x"], s["gamma"], s["beta"], EPS)
            saved = s["x"]
        dx, dgamma, dbeta = tg.layer_norm_backward(s["dy"], saved, stats, s["gamma"])
        return y, dx, dgamma, dbeta
    if c["op"] == "act":
        alpha = ALPHA.get(c["act"], 0.0)
        y, saved = tg.activation_save8(s["x"], c["act"], alpha)
        return y, tg.activation_backward(s["dy"], saved, c["act"], alpha)
    if c["op"] == "typed":
        alpha = ALPHA.get(c["act"], 0.0)
        if not c["saved8"]:
            return tg.typed_linear(s["x"], s["w"], s["offsets"], s["bias"], c["act"], alpha)
        y, saved = tg.typed_linear(s["x"], s["w"], s["offsets"], s["bias"], c["act"], alpha, save8=True)
        return y, tg.activation_backward(s["dy"], saved, c["act"], alpha)
    x = tg.Saved8(s["codes"], s["exponents"], s["dy"].dtype) if c["saved8"] else s["x"]
    return tg.typed_linear_backward(s["dy"], x, s["w"], s["offsets"])


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        x, dy, gamma, beta = (s[k].float() for k in ("x", "dy", "gamma", "beta"))
        centred = x - x.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
        h = centred * rstd
        y = h * gamma + beta
        if c["saved8"]:
            h = _values8(*_saved8(h, _least(s["x"].dtype)))
        gdy = dy * gamma
        dx = rstd * (gdy - gdy.mean(1, keepdim=True) - h * (gdy * h).mean(1, keepdim=True))
        return [v.to(s["x"].dtype) for v in (y, dx, (dy * h).sum(0), dy.sum(0))]
    if c["op"] == "act":
        x = s["x"].float()
        y = _act(x, c["act"])
        dx = s["dy"].float() * _act_slope(_values8(*_saved8(s["x"], _least(s["x"].dtype))), c["act"])
        return y.to(s["x"].dtype), dx.to(s["x"].dtype)
    w = s["w"].float()
    if c["op"] == "typed":
        tiles = s["x"].float()[s["tile_rows"]]
        z = torch.matmul(tiles, w[s["tile_type"]]).view(-1, c["n"])[s["row_place"]]
        z = z + s["bias"][s["row_type"]]
        y = _act(z, c["act"]).to(s["x"].dtype)
        if not c["saved8"]:
            return y
        z = _values8(*_saved8(z, _least(y.dtype)))
        return y, (s["dy"].float() * _act_slope(z, c["act"])).to(y.dtype)
    x = _values8(s["codes"], s["exponents"]) if c["saved8"] else s["x"].float()
    dy = s["dy"].float()
    dy_tiles = dy[s["tile_rows"]] * s["tile_inside"][:, :, None]
    dx = torch.matmul(dy_tiles, w[s["tile_type"]].transpose(1, 2)).view(-1, c["k"])[s["row_place"]]
    part = torch.matmul(x[s["tile_rows"]].transpose(1, 2), dy_tiles)
    dw = torch.zeros_like(w).index_add_(0, s["tile_type"], part)
    db = torch.zeros(c["types"], c["n"], device=dy.device).index_add_(0, s["tile_type"], dy_tiles.sum(1))
    return dx.to(s["dy"].dtype), dw.to(s["dy"].dtype), db


# ── the definitions in 64 bits ───────────────────────────────────────────────
def _rounded8(x, emin):
    """x (float64) as its 8-bit copy holds it."""
    cols = x.shape[1]
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(x.shape[0], -1, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -140) / 127))
    e = torch.where(127 * torch.exp2(e) < top, e + 1, e)       # the logarithm is rounded
    e = torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e)
    step = torch.exp2(torch.clamp(e, min=emin))
    return (torch.round(x / step) * step).flatten(1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    emin = _least(DTYPES[case["dtype"]])
    if case["op"] == "norm":
        x, dy, gamma, beta = (s[k].double() for k in ("x", "dy", "gamma", "beta"))
        mean = x.sum(1, keepdim=True) / case["cols"]
        var = ((x - mean) ** 2).sum(1, keepdim=True) / case["cols"]
        rstd = (var + EPS) ** -0.5
        h = (x - mean) * rstd
        y = gamma * h + beta
        if case["saved8"]:
            h = _rounded8(h, emin)
        g = gamma * dy
        dx = rstd * (g - g.sum(1, keepdim=True) / case["cols"] - h * (g * h).sum(1, keepdim=True) / case["cols"])
        return y, dx, (dy * h).sum(0), dy.sum(0)
    if case["op"] == "act":
        x = s["x"].double()
        return _act(x, case["act"]), s["dy"].double() * _act_slope(_rounded8(x, emin), case["act"])
    o = np.concatenate([[0], np.cumsum(_sizes(case))]).tolist()
    spans = list(zip(range(case["types"]), o, o[1:]))
    if case["op"] == "typed":
        z = torch.cat([s["x"][a:b].double() @ s["w"][t].double() + s["bias"][t].double() for t, a, b in spans])
        y = _act(z, case["act"])
        if not case["saved8"]:
            return y
        return y, s["dy"].double() * _act_slope(_rounded8(z, emin), case["act"])
    if case["saved8"]:
        step = torch.exp2(s["exponents"].double() - 127)
        x = s["codes"].double() * step.repeat_interleave(BLOCK, 1)[:, :case["k"]]
    else:
        x = s["x"].double()
    dy = s["dy"].double()
    dx = torch.cat([dy[a:b] @ s["w"][t].double().T for t, a, b in spans])
    dw = torch.stack([x[a:b].T @ dy[a:b] for _, a, b in spans])
    db = torch.stack([dy[a:b].sum(0) for _, a, b in spans])
    return dx, dw, db


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    rows = case["rows"]
    if case["op"] in ("norm", "act"):
        values = rows * case["cols"]
        # x, dy in; y, dx out.
        return {"bytes": 4 * values * size, "flops": (20 if case["op"] == "norm" else 16) * values}
    k, n = case["k"], case["n"]
    used = sum(m > 0 for m in _sizes(case))
    if case["op"] == "typed":
        # x, the used weights and biases in, y out; with the backward pass dy in, dz out.
        by = rows * k * size + used * (k * n * size + n * 4) + rows * n * size * (3 if case["saved8"] else 1)
        return {"bytes": by, "flops": 2 * rows * k * n}
    x = rows * k + rows * ((k + BLOCK - 1) // BLOCK) if case["saved8"] else rows * k * size
    by = x + rows * n * size + rows * k * size + used * k * n * size + case["types"] * (k * n * size + n * 4)
    return {"bytes": by, "flops": 4 * rows * k * n}
