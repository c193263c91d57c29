"""A student's step on a batch of graphs -- linear, group norm with GELU, linear,
the teacher's best classes, both losses -- and the example that trains one."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("distill_student", os.path.join(ROOT, "examples", "distill_student.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g) * scale


def step64(p, x, sizes, groups, labels, ids, best, mix=0.7, temperature=2.0, entropy=0.01):
    """The mean loss in 64 bits, from the formulas, for automatic differentiation."""
    a = x @ p["w1"][0] + p["b1"][0]
    parts, o = [], 0
    for s in sizes:
        if s:
            v = a[o:o + s].view(s, groups, -1)
            o += s
            m = v.mean((0, 2), keepdim=True)
            parts.append(((v - m) / (((v - m) ** 2).mean((0, 2), keepdim=True) + 1e-5).sqrt()).reshape(s, -1))
    h = torch.nn.functional.gelu(torch.cat(parts) * p["gamma"] + p["beta"], approximate="tanh")
    z = h @ p["w2"][0] + p["b2"][0]
    q = torch.softmax(best.double() / temperature, 1)
    soft = torch.log_softmax(z / temperature, 1).gather(1, ids.long())
    distill = temperature ** 2 * (q * (q.log() - soft)).sum(1)
    log = torch.log_softmax(z, 1)
    has = labels >= 0
    lp = torch.where(has, log.gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
    return (mix * distill - (1 - mix) * lp + entropy * (log.exp() * log).sum(1)).mean(), z


def test_step_against_the_whole_formula(tg, example):
    """fp32, against automatic differentiation in 64 bits.  The chain: two products of 64 and 48 terms, a norm, two
    softmaxes; 2^-23 (8 + sqrt K) of each one's terms' norm, which is within a factor of 8 of the result's here."""
    sizes, classes = [30, 0, 1, 69], 33
    student = example.Student(64, 48, classes, 6, torch.float32, seed=3)
    for k in ("gamma", "beta", "b1", "b2"):
        student.params[k] = student.params[k] + rand(*student.params[k].shape, seed=len(k), scale=0.2)
    x = rand(100, 64, seed=1)
    offsets = torch.tensor([0, 30, 30, 31, 100], dtype=torch.int32, device="cuda")
    labels = torch.randint(-1, classes, (100,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    best, ids = tg.label_log_probs(rand(100, classes, seed=2, scale=2.0), labels, 4)[3:]
    z, kept = student.forward(x, offsets)
    loss, dz = example.loss_and_gradient(z, labels, ids, best)
    grads = student.backward(dz, kept)
    p = {k: v.double().requires_grad_(True) for k, v in student.params.items()}
    want, z64 = step64(p, x.double(), sizes, 6, labels, ids, best)
    want.backward()
    tol = 8 * 5 * 2.0 ** -23 * (8 + math.sqrt(64))
    assert abs(float(loss) - float(want.detach())) <= tol * abs(float(want.detach()))
    for name, got, ref in (("z", z, z64.detach()), *((k, grads[k].view_as(p[k]), p[k].grad) for k in grads)):
        off_by = float((got.double() - ref).norm() / ref.norm())
        assert off_by <= tol, f"{name}: {off_by}"


def test_captured_step_replays(tg, example):
    """The whole step as one CUDA graph: the same bits as eager, on new inputs too."""
    student = example.Student(64, 96, 500, 8, torch.bfloat16, seed=1)
    x, offsets = rand(300, 64, seed=1).bfloat16(), torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    all_rows = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    labels = torch.arange(300, device="cuda") % 500
    teacher = rand(300, 500, seed=2, scale=3.0)
    w1, w2 = student.params["w1"].bfloat16(), student.params["w2"].bfloat16()
    p = student.params

    def step():
        best, ids = tg.label_log_probs(teacher, labels, 9)[3:]
        a = tg.typed_linear(x, w1, all_rows, p["b1"])
        h, stats = tg.group_norm(a, p["gamma"], p["beta"], 8, offsets, "gelu")
        z = tg.typed_linear(h, w2, all_rows, p["b2"])
        loss, dz = tg.distill_loss(z, ids, best, 2.0)
        lp, e, s = tg.label_log_probs(z, labels)
        dz2 = tg.label_log_probs_backward(lp, z, labels, s, lp, e)
        return [loss, lp, e, dz, dz2, *student.backward(dz + dz2, (x, a, h, stats, w1, w2, all_rows, offsets)).values()]
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (1, 9):
        x.copy_(rand(300, 64, seed=seed))
        teacher.copy_(rand(300, 500, seed=seed + 1, scale=3.0))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_example_runs(example):
    for dtype in (torch.bfloat16, torch.float32):
        losses = example.train(graphs=9, nodes=700, features=32, hidden=64, classes=13, top=4, steps=3, dtype=dtype, report=None)
        assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
