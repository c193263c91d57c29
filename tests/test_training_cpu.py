"""Training operators without a GPU: refusals that need none, the saved form's
definition, and the example's import."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import tinygnn_b200 as tg
from tinygnn_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    off = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: tg.save8(x), lambda: tg.activation_save8(x, "relu"), lambda: tg.layer_norm(x, x[0], x[0]),
                 lambda: tg.typed_linear(x, torch.zeros(1, 8, 8), off),
                 lambda: tg.typed_linear_grad_input(x, torch.zeros(1, 8, 8), off),
                 lambda: tg.typed_linear_grad_weight(x, x, off), lambda: tg.activation_backward(x, x, "relu"),
                 lambda: tg.check_row_offsets(off, 4)):
        with pytest.raises(tg.InvalidArgument):
            call()


def test_wrong_kinds_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: tg.activation_save8(x, "softplus"), lambda: tg.save8(np.zeros((2, 2), np.float32).tolist()),
                 lambda: tg.activation_backward(x, tg.Saved8(x, x, torch.float16), "relu"),
                 lambda: tg.Saved8(x, x, torch.float64).restore(),
                 lambda: tg.typed_linear_grad_weight(x, x, x, dtype=torch.float64)):
        with pytest.raises((ValueError, AttributeError)):
            call()


def test_entry_points_without_a_device_say_so():
    if _lib.lib.tg_device_count() > 0:
        pytest.skip("a device is present")
    lib = _lib.lib
    calls = [lib.tg_save8(1, 1, 0, None, 1, 0, 0.0, None, 0, None, 16, None, 1, None),
             lib.tg_restore8(1, 1, None, 16, None, 1, 0, None, 1, None),
             lib.tg_activation_grad(1, 1, 0, None, 1, None, 1, None, 0, None, 0, 0, 0.0, None, 1, None),
             lib.tg_layer_norm(1, 1, 0, None, 1, 0, None, None, 1e-5, None, 1, None, None, 0, None, 0, None),
             lib.tg_layer_norm_grad(1, 1, 0, None, 1, None, 1, None, 0, None, 0, None, 0, None, None, 1, None, None,
                                    None),
             lib.tg_typed_linear(1, 1, 1, 1, 0, None, 1, None, 1, 1, None, None, 0, 0.0, None, 1, None, 0, None, 0,
                                 None),
             lib.tg_typed_linear_grad_input(1, 1, 1, 1, 0, None, 1, None, 1, 1, None, None, 1, None),
             lib.tg_typed_linear_grad_weight(1, 1, 1, 1, 0, None, 1, None, 0, None, 0, None, 1, None, 0, None, 1, 1,
                                             None, None),
             lib.tg_typed_check_offsets(1, 1, None, None)]
    assert calls == [_lib.NO_DEVICE] * len(calls)


def test_saved_form_bytes():
    rows, cols = 10, 300
    s = tg.Saved8(torch.zeros(rows, cols, dtype=torch.int8), torch.zeros(rows, 3, dtype=torch.uint8), torch.bfloat16)
    assert s.shape == (rows, cols) and s.nbytes == rows * (cols + 3)


def test_workloads_plain_8_bit_form_matches_its_definition():
    """The workloads' plain form of the 8-bit copy against the one by logarithms, in 64 bits."""
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 300, generator=g) * torch.exp2(torch.randn(40, 1, generator=g) * 6)
    x[3] = 0
    x[4, 7] = 127.0  # a block's largest value exactly 127 * 2^0
    for emin in (-126, -24):
        assert torch.equal(ops._values8(*ops._saved8(x, emin)).double(), ops._rounded8(x.double(), emin))


def test_workloads_type_sizes():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    for rows, types, skew in ((1, 64, 2.5), (8, 64, 1.0), (20011, 40, 2.0), (5, 1, 0.0)):
        sizes = ops._sizes(dict(rows=rows, types=types, skew=skew))
        assert len(sizes) == types and sum(sizes) == rows and min(sizes) >= 0
