"""Workloads of the classification operators: log probabilities of labels with
entropy and top alternatives, distillation from a teacher's top logits, and
group norm over the rows of batched graphs.

Each case is one pass a training or serving program makes.  ``own`` False
computes it with elementary torch operations in 32 bits (long sums in 64),
rounded once at the end; ``own`` True makes the calls of :mod:`tinygnn_b200`.
``exact`` computes the same from the definitions in 64 bits.

The passes (``op``):

* ``label``    log probability of each row's label, the entropy of the row and
               its ``top`` best classes (none for 0); with ``grad`` also the
               logits' gradient for given gradients of the first two.
* ``distill``  the loss against a teacher's ``k`` best logits of each row and
               its gradient; without ``grad`` (evaluation) the loss alone.
* ``group``    group norm with an activation, over the rows of each graph and
               the columns of each group; with ``grad`` also its gradients.

A label outside the classes is none: log probability 0 and no gradient from
it.  A masked class (-inf) has the probability 0; a row of masked classes alone
has the log probability -inf, the entropy 0 and no gradient.  Equal logits are
ranked by class.  A teacher's class outside the classes is none.
"""
import itertools
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


# ── cases ────────────────────────────────────────────────────────────────────
def listed():
    return [
        # Class scores of a small citation graph, trained with an entropy term: latency.
        dict(name="label small", op="label", rows=2708, classes=7, dtype="float32", top=3, grad=True, mask="none"),
        # The 41 classes of a graph of 232,965 nodes, some classes masked, some rows entirely.
        dict(name="label nodes", op="label", rows=232965, classes=41, dtype="float32", top=5, grad=True, mask="inf"),
        # Serving: the next token of four sequences with its 20 alternatives.
        dict(name="label serve", op="label", rows=4, classes=131072, dtype="bfloat16", top=20, grad=False, mask="none"),
        # Scoring a prompt, a vocabulary of an odd size, masked by the type's lowest value.
        dict(name="label score odd", op="label", rows=2011, classes=49999, dtype="float16", top=10, grad=False,
             mask="lowest"),
        # The loss of a training step over a large vocabulary.
        dict(name="label large", op="label", rows=8192, classes=131072, dtype="bfloat16", top=0, grad=True, mask="none"),
        # A student of a few hundred classes on the nodes of a minibatch, fp32.
        dict(name="distill nodes", op="distill", rows=20011, classes=349, dtype="float32", k=8, temperature=2.0, grad=True),
        # A few rows of a large vocabulary, many alternatives, evaluated only.
        dict(name="distill few", op="distill", rows=16, classes=65537, dtype="float32", k=128, temperature=1.0, grad=False),
        # The largest: distillation over a large vocabulary.
        dict(name="distill large", op="distill", rows=8192, classes=131072, dtype="bfloat16", k=64, temperature=1.5,
             grad=True),
        # Serving one small graph.
        dict(name="group serve", op="group", graphs=1, rows=60, cols=256, groups=8, skew=0.0, dtype="bfloat16", act="relu",
             grad=False),
        # A training batch of many small graphs, all columns in one group.
        dict(name="group molecules", op="group", graphs=2048, rows=50021, cols=64, groups=1, skew=1.0, dtype="float32",
             act="gelu", grad=True),
        # The hidden rows of one large graph.
        dict(name="group one graph", op="group", graphs=1, rows=232965, cols=128, groups=8, skew=0.0, dtype="bfloat16",
             act="relu", grad=True),
        # Sixteen grids of 64 x 64 points, 320 columns in 32 groups.
        dict(name="group grids", op="group", graphs=16, rows=65536, cols=320, groups=32, skew=0.0, dtype="float16",
             act="gelu", grad=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["label", "label", "distill", "group", "group"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "group":
        groups = rng.choice([1, 1, 2, 4, 8, 16, 32])
        per = max(1, _spread(rng, 8, 1024) // groups)
        cols = groups * (per if rng.random() < 0.34 else max(8, per // 8 * 8))
        rows = _spread(rng, 1, min(262144, 2 ** 25 // cols))
        graphs = min(4096, _spread(rng, 1, max(1, rows)))
        return dict(op=op, graphs=graphs, rows=rows, cols=cols, groups=groups, skew=round(rng.uniform(0.0, 2.0), 2),
                    dtype=dtype, act=rng.choice(["none", "relu", "elu", "sigmoid", "gelu"]), grad=rng.random() < 0.7)
    classes = _spread(rng, 2, 131072)
    if rng.random() < 0.6:
        classes = max(8, classes // 8 * 8)
    rows = _spread(rng, 1, min(262144, 2 ** 29 // classes))
    if op == "label":
        top = rng.choice([0, 0, 1, 5, 20, 64])
        return dict(op=op, rows=rows, classes=classes, dtype=dtype, top=min(top, classes), grad=rng.random() < 0.5,
                    mask=rng.choice(["none", "inf", "lowest"]))
    return dict(op=op, rows=rows, classes=classes, dtype=dtype, k=min(classes, _spread(rng, 1, 128)),
                temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), grad=rng.random() < 0.8)


def _sizes(case):
    """Rows of each graph: uneven (weights spread evenly over (0, 1], to the power `skew`), in no order, some zero."""
    n, rows = case["graphs"], case["rows"]
    w = [(((i + 1) * 0.6180339887) % 1.0) ** case["skew"] for i in range(n)]
    ends = [min(rows, int(rows * acc / sum(w))) for acc in itertools.accumulate(w)]
    ends[-1] = rows
    return [b - a for a, b in zip([0] + ends, ends)]


# ── inputs ───────────────────────────────────────────────────────────────────
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _logits(rows, classes, dtype, g):
    """Normal scores around a common bias of each class, and one class of each row well above the rest."""
    z = torch.randn(rows, classes, device="cuda", generator=g, dtype=torch.float32 if rows * classes < 2 ** 26 else dtype)
    z *= 2.0
    z += torch.randn(classes, device="cuda", generator=g).to(z.dtype)
    best = torch.randint(0, classes, (rows, 1), device="cuda", generator=g)
    lift = 2.0 + 8.0 * torch.rand(rows, 1, device="cuda", generator=g)
    z.scatter_add_(1, best, lift.to(z.dtype))
    return z.to(dtype), best


def prepare(case, seed):
    g = _generator(seed)
    dtype, rows = DTYPES[case["dtype"]], case["rows"]
    s = dict(case=dict(case))
    if case["op"] == "group":
        cols = case["cols"]
        x = torch.randn(rows, cols, device="cuda", generator=g)
        x *= 0.5 + torch.rand(cols, device="cuda", generator=g) * 1.5
        x += torch.randn(cols, device="cuda", generator=g) * 0.5
        s["x"] = x.to(dtype)
        s["dy"] = torch.randn(rows, cols, device="cuda", generator=g).mul_(0.1).to(dtype)
        s["gamma"] = (1.0 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
        s["beta"] = (0.2 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
        sizes = _sizes(case)
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")
        # The plain form's plan: the graph of each row, the group of each column, the values of each graph's groups.
        s["row_graph"] = torch.repeat_interleave(torch.arange(case["graphs"]), torch.tensor(sizes)).cuda()
        s["count"] = (torch.tensor(sizes).double() * (cols // case["groups"])).clamp(min=1).cuda()[:, None]
        return s
    classes = case["classes"]
    s["z"], best = _logits(rows, classes, dtype, g)
    if case["op"] == "label":
        label = torch.where(torch.rand(rows, 1, device="cuda", generator=g) < 0.7, best,
                            torch.randint(0, classes, (rows, 1), device="cuda", generator=g))
        if case["mask"] != "none":
            low = -math.inf if case["mask"] == "inf" else torch.finfo(dtype).min
            masked = torch.rand(classes, device="cuda", generator=g) < 0.2
            keep = s["z"].gather(1, label)
            s["z"].masked_fill_(masked[None, :], low)
            s["z"].scatter_(1, label, keep)
            s["z"].masked_fill_(torch.rand(rows, 1, device="cuda", generator=g) < 0.01, low)
        none = torch.rand(rows, device="cuda", generator=g) < 0.05
        s["labels"] = torch.where(none, -1, label[:, 0])
        if case["grad"]:
            s["dlog"] = -torch.rand(rows, device="cuda", generator=g) / math.sqrt(rows)
            s["dent"] = torch.full((rows,), -0.01 / math.sqrt(rows), device="cuda")
        return s
    k = case["k"]
    # k different classes of each row, the teacher's logits of them in falling order; some rows have fewer, some none.
    start = torch.randint(0, classes, (rows, 1), device="cuda", generator=g)
    step = next(p for p in (7919, 104729, 1) if classes % p)
    s["classes"] = ((start + torch.arange(k, device="cuda") * step) % classes).to(torch.int32)
    s["classes"][:, 0] = best[:, 0].to(torch.int32)
    t = torch.randn(rows, k, device="cuda", generator=g) * 2.0
    s["teacher"] = (t.sort(1, descending=True).values + 6.0).to(dtype)
    have = torch.where(torch.rand(rows, 1, device="cuda", generator=g) < 0.05,
                       torch.randint(0, k + 1, (rows, 1), device="cuda", generator=g), k)
    s["classes"].masked_fill_(torch.arange(k, device="cuda")[None, :] >= have, -1)
    s["weights"] = torch.rand(rows, device="cuda", generator=g) / math.sqrt(rows)
    return s


# ── the passes ───────────────────────────────────────────────────────────────
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import tinygnn_b200 as tg
    c = s["case"]
    if c["op"] == "label":
        out = tg.label_log_probs(s["z"], s["labels"], c["top"])
        if not c["grad"]:
            return out[:2] + out[3:]
        dz = tg.label_log_probs_backward(s["dlog"], s["z"], s["labels"], out[2], s["dent"], out[1])
        return out[:2] + out[3:] + (dz,)
    if c["op"] == "distill":
        return tg.distill_loss(s["z"], s["classes"], s["teacher"], c["temperature"], s["weights"], c["grad"])
    act = None if c["act"] == "none" else c["act"]
    alpha = 1.0 if c["act"] == "elu" else 0.0
    y, stats = tg.group_norm(s["x"], s["gamma"], s["beta"], c["groups"], s["offsets"], act, alpha, EPS)
    if not c["grad"]:
        return y
    return (y, *tg.group_norm_backward(s["dy"], s["x"], stats, s["gamma"], s["beta"], c["groups"], s["offsets"], act, alpha))


def _plain(s):
    c = s["case"]
    if c["op"] == "label":
        return _plain_label(s, c)
    if c["op"] == "distill":
        return _plain_distill(s, c)
    return _plain_group(s, c)


def _plain_label(s, c):
    z, n = s["z"].float(), c["classes"]
    top = z.amax(1, keepdim=True)
    empty = top == -math.inf
    d = z - torch.where(empty, 0.0, top)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log = d - torch.log(total)                                   # all classes' log probabilities
    p = e / torch.where(empty, 1.0, total)
    entropy = -torch.where(p > 0, p * log, 0.0).sum(1)
    label = s["labels"][:, None]
    has = (label >= 0) & (label < n)
    at = torch.where(has, label, 0)
    out = [torch.where(has, log.gather(1, at), 0.0)[:, 0], entropy]
    if c["top"]:
        # The value's rank in the upper half of a key, the class in the lower: equal values in the classes' order.
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 31 + (n - 1 - torch.arange(n, device=z.device))
        best = torch.topk(key, c["top"], 1).values
        best = n - 1 - (best & (2 ** 31 - 1))
        out += [log.gather(1, best), best.to(torch.int32)]
    if c["grad"]:
        a = torch.where(has[:, 0], s["dlog"], 0.0)[:, None]
        dz = -p * (a + s["dent"][:, None] * torch.where(p > 0, log + entropy[:, None], 0.0))
        dz.scatter_add_(1, at, torch.where(empty, 0.0, a))
        out.append(dz.to(s["z"].dtype))
    return out


def _plain_distill(s, c):
    warmth, n = c["temperature"], c["classes"]
    has = (s["classes"] >= 0) & (s["classes"] < n)
    at = torch.where(has, s["classes"].long(), 0)
    t = torch.where(has, s["teacher"].float() / warmth, -math.inf)
    some = has.any(1, keepdim=True)
    q = torch.exp(t - torch.where(some, t.amax(1, keepdim=True), 0.0))
    q = q / torch.where(some, q.sum(1, keepdim=True), 1.0)
    d = s["z"].float()
    d = (d - d.amax(1, keepdim=True)) / warmth
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log = d.gather(1, at) - torch.log(total)
    loss = warmth * warmth * torch.where(q > 0, q * (torch.log(q) - log), 0.0).sum(1)
    if not c["grad"]:
        return loss
    dz = torch.where(some, e / total, 0.0).scatter_add_(1, at, -q) * (warmth * s["weights"][:, None])
    return loss, dz.to(s["z"].dtype)


def _act(u, act):
    if act == "none":
        return u
    if act == "relu":
        return torch.clamp(u, min=0)
    if act == "elu":
        return torch.where(u < 0, torch.expm1(u), u)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-u))
    return 0.5 * u * (1 + torch.tanh(0.7978845608 * (u + 0.044715 * u * u * u)))


def _act_slope(u, act):
    if act == "none":
        return torch.ones_like(u)
    if act == "relu":
        return (u > 0).to(u.dtype)
    if act == "elu":
        return torch.where(u < 0, torch.exp(u), 1.0)
    if act == "sigmoid":
        p = 1 / (1 + torch.exp(-u))
        return p * (1 - p)
    p = torch.tanh(0.7978845608 * (u + 0.044715 * u * u * u))
    return 0.5 * (1 + p) + 0.5 * u * (1 - p * p) * 0.7978845608 * (1 + 3 * 0.044715 * u * u)


def _plain_group(s, c):
    x, gamma, beta = s["x"].float(), s["gamma"].float(), s["beta"].float()
    graphs, groups = c["graphs"], c["groups"]

    def mean(v):
        """The mean over each graph's rows and each group's columns, for each row and column."""
        rows = v.double().view(v.shape[0], groups, -1).sum(2)
        m = torch.zeros(graphs, groups, device=v.device, dtype=torch.float64).index_add_(0, s["row_graph"], rows)
        return (m / s["count"])[s["row_graph"]].repeat_interleave(c["cols"] // groups, 1).float()

    centred = x - mean(x)
    r = 1 / torch.sqrt(mean(centred * centred) + EPS)
    h = centred * r
    u = h * gamma + beta
    y = _act(u, c["act"]).to(s["x"].dtype)
    if not c["grad"]:
        return y
    du = s["dy"].float() * _act_slope(u, c["act"])
    g = du * gamma
    dx = r * (g - mean(g) - h * mean(g * h))
    return [y] + [v.to(y.dtype) for v in (dx, (du * h).double().sum(0), du.double().sum(0))]


# ── the definitions in 64 bits ───────────────────────────────────────────────
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "label":
        return _exact_label(s, case)
    if case["op"] == "distill":
        return _exact_distill(s, case)
    return _exact_group(s, case)


def _exact_label(s, c):
    rows, n = s["z"].shape
    lp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    entropy, kept, classes, grads = torch.zeros_like(lp), [], [], []
    block = max(1, 2 ** 27 // n)
    for r0 in range(0, rows, block):
        z = s["z"][r0:r0 + block].double()
        labels = s["labels"][r0:r0 + block]
        lse = torch.logsumexp(z, 1, keepdim=True)
        log = torch.where(lse == -math.inf, -math.inf, z - lse)
        p = log.exp()
        plogp = torch.special.xlogy(p, p)
        entropy[r0:r0 + block] = -plogp.sum(1)
        has = ((labels >= 0) & (labels < n)).nonzero()[:, 0]
        lp[r0 + has] = log[has, labels[has]]
        if c["top"]:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :c["top"]]
            kept.append(log.gather(1, order))
            classes.append(order.to(torch.int32))
        if c["grad"]:
            a, b = s["dlog"][r0:r0 + block].double(), s["dent"][r0:r0 + block].double()
            dz = -b[:, None] * (plogp + p * entropy[r0:r0 + block, None])
            some = has[lse[has, 0] > -math.inf]
            dz[some] -= a[some, None] * p[some]
            dz[some, labels[some]] += a[some]
            grads.append(dz.float())  # (within half a step of fp32)
    out = [lp, entropy]
    if c["top"]:
        out += [torch.cat(kept), torch.cat(classes)]
    if c["grad"]:
        out.append(torch.cat(grads))
    return out


def _exact_distill(s, c):
    rows, n = s["z"].shape
    warmth, losses, grads = c["temperature"], [], []
    block = max(1, 2 ** 27 // n)
    for r0 in range(0, rows, block):
        z = s["z"][r0:r0 + block].double() / warmth
        ids = s["classes"][r0:r0 + block].long()
        there = (ids >= 0) & (ids < n)
        some = there.any(1)
        t = (s["teacher"][r0:r0 + block].double() / warmth).masked_fill(~there, -math.inf)
        q = torch.softmax(t, 1).masked_fill(~there, 0.0)
        log = z - torch.logsumexp(z, 1, keepdim=True)
        ids = ids.masked_fill(~there, 0)
        losses.append(warmth ** 2 * (torch.special.xlogy(q, q) - q * log.gather(1, ids)).sum(1))
        if c["grad"]:
            dz = log.exp()
            dz[~some] = 0
            dz.scatter_add_(1, ids, -q)
            grads.append((dz * (warmth * s["weights"][r0:r0 + block, None].double())).float())  # (as above)
    return (torch.cat(losses), torch.cat(grads)) if c["grad"] else torch.cat(losses)


def _exact_group(s, c):
    groups = c["groups"]
    graph, count = s["row_graph"], s["count"]
    x = s["x"].double().view(c["rows"], groups, -1)
    gamma, beta = (s[k].double().view(groups, -1) for k in ("gamma", "beta"))

    def over_graph(v):
        """The mean of v over each graph and group, for each row."""
        return torch.stack([torch.bincount(graph, v[:, j].sum(1), c["graphs"]) for j in range(groups)], 1).div(count)[graph][:, :, None]

    x = x - over_graph(x)
    r = (over_graph(x ** 2) + EPS) ** -0.5
    h = x * r
    u = h * gamma + beta
    y = _act(u, c["act"]).view(c["rows"], -1)
    if not c["grad"]:
        return y
    du = s["dy"].double().view(u.shape) * _act_slope(u, c["act"])
    dgamma, dbeta = (du * h).sum(0).flatten(), du.sum(0).flatten()
    g = du * gamma
    dx = r * (g - over_graph(g) - h * over_graph(g * h))
    return y, dx.view(c["rows"], -1), dgamma, dbeta


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    rows = case["rows"]
    if case["op"] == "group":
        values = rows * case["cols"]
        # x (and dy) in; y (and dx) out.
        return {"bytes": (4 if case["grad"] else 2) * values * size, "flops": (30 if case["grad"] else 12) * values}
    values = rows * case["classes"]
    by = (2 if case["grad"] else 1) * values * size  # the logits in, their gradient out
    if case["op"] == "label":
        by += rows * (8 + 8 + 8 * case["top"] + (8 if case["grad"] else 0))
        return {"bytes": by, "flops": (14 if case["grad"] else 8) * values}
    by += rows * (case["k"] * (4 + size) + 8)
    return {"bytes": by, "flops": (10 if case["grad"] else 6) * values}
