"""Group norm and the losses on class scores without a GPU: refusals, the C entry
points' status, the workloads' sizes, the package's names."""
import importlib.util
import os
import random

import pytest
import torch

import tinygnn_b200 as tg
from tinygnn_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load(*path):
    spec = importlib.util.spec_from_file_location(path[-1][:-3], os.path.join(ROOT, *path))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_names_are_offered():
    for name in ("group_norm", "group_norm_backward", "label_log_probs", "label_log_probs_backward", "distill_loss"):
        assert name in dir(tg) and callable(getattr(tg, name)) and getattr(tg, name).__doc__


def test_cpu_tensors_and_wrong_kinds_are_refused():
    x, labels, rows = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: tg.group_norm(x, x[0], x[0], 2), lambda: tg.group_norm(x, x[0], x[0], 2, None, "softplus"),
                 lambda: tg.group_norm_backward(x, x, torch.zeros(1, 2, 2), x[0], x[0], 2),
                 lambda: tg.label_log_probs(x, labels), lambda: tg.label_log_probs(x.tolist(), labels),
                 lambda: tg.label_log_probs_backward(rows, x, labels, torch.zeros(4, 2)),
                 lambda: tg.distill_loss(x, ids, x[:, :2]), lambda: tg.distill_loss(x, ids, None)):
        with pytest.raises(tg.InvalidArgument):
            call()


def test_entry_points_without_a_device_say_so():
    if _lib.lib.tg_device_count() > 0:
        pytest.skip("a device is present")
    lib = _lib.lib
    calls = [lib.tg_group_norm(1, 1, 1, 1, None, 0, None, 1, 0, None, None, 1e-5, 0, 0.0, None, 1, None, None),
             lib.tg_group_norm_grad(1, 1, 1, 1, None, 0, None, 1, None, 1, None, 0, None, None, 0, 0.0, None, 1, None, None, None),
             lib.tg_label_log_probs(1, 1, 0, None, 1, None, 8, 0, None, None, None, None, None, None),
             lib.tg_label_log_probs_grad(1, 1, 0, None, None, None, 1, None, 8, None, None, None, 1, None),
             lib.tg_distill_loss(1, 1, 0, None, 1, 1, None, 4, 1, 0, None, 1, 1.0, None, None, None, 1, None)]
    assert calls == [_lib.NO_DEVICE] * len(calls)


def test_workloads():
    """The listed and drawn cases are within the operators' limits, and their graphs' sizes add up."""
    ops = load("perf", "more_operators.py")
    rng = random.Random(3)
    cases = ops.listed() + [ops.draw(rng) for _ in range(300)]
    largest = max(ops.work(c)["bytes"] for c in ops.listed())
    for c in cases:
        assert ops.work(c)["bytes"] <= largest and c["rows"] >= 1
        if c["op"] == "group":
            sizes = ops._sizes(c)
            assert len(sizes) == c["graphs"] and sum(sizes) == c["rows"] and min(sizes) >= 0 and c["cols"] % c["groups"] == 0
        elif c["op"] == "label":
            assert 0 <= c["top"] <= min(128, c["classes"])
        else:
            assert 1 <= c["k"] <= min(128, c["classes"])


def test_example_imports():
    assert load("examples", "distill_student.py").train
