"""Group norm's statistics where one column, one row or one part of a graph stands
apart from the rest: their error is of the deviations, not of how far that part is
from the others.
"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_group_norm import Plain, offsets_of, rand  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def check_stats(tg, x, sizes, groups, what, steps):
    one, zero = torch.ones(x.shape[1], device="cuda"), torch.zeros(x.shape[1], device="cuda")
    _, stats = tg.group_norm(x, one, zero, groups, offsets_of(sizes))
    ref = Plain(x, one, zero, sizes, groups, None, 0.0).stats
    # A mean is off by its own last bit, and by `steps` roundings of values within a part of it (sd 1: |x - k| < 10).
    off = (stats[..., 0].double() - ref[..., 0]).abs()
    assert (off <= 2.0 ** -24 * (2 * ref[..., 0].abs() + 10 * steps)).all(), f"{what}: mean off by {float(off.max())}"
    off = (stats[..., 1].double() / ref[..., 1] - 1).abs()
    assert (off <= 2.0 ** -24 * steps).all(), f"{what}: rstd off by {float(off.max()) * 2 ** 24} units"


# A thread's sum of squares about its first value has at most as many roundings as it has rows (7 of 4,096 x 1,024, 25
# of 60,000 x 256; 2 each), and is about twice the deviations; means add 2, each; the quotient and the root 4: half of all
# that for the root.
@pytest.mark.parametrize("shift", [10.0, 100.0, 1000.0, 30000.0])
@pytest.mark.parametrize("rows,cols,groups,steps", [(4096, 1024, 1, 32), (60000, 256, 2, 64)])
def test_parts_that_stand_apart(tg, shift, rows, cols, groups, steps):
    x = rand(rows, cols, seed=1)
    for what, at in (("first column", (slice(None), slice(0, 1))), ("first columns of all groups", (slice(None), slice(0, None, cols // groups))),
                     ("first row", (slice(0, 1), slice(None))), ("first rows", (slice(0, 9), slice(None))),
                     ("last column", (slice(None), slice(cols - 1, None))), ("first value", (slice(0, 1), slice(0, 1)))):
        for sign in (1.0, -1.0):
            y = x.clone()
            y[at] += sign * shift
            check_stats(tg, y, [rows], groups, what, steps)


@pytest.mark.parametrize("shift", [1000.0, 30000.0])
def test_graphs_whose_first_row_stands_apart(tg, shift):
    """Graphs that begin anywhere in a chunk: the first part of one may be a single row."""
    sizes = [5, 9001, 6, 8003, 7, 11000, 1, 1, 12001]
    for cols, groups in ((512, 4), (96, 1)):
        x = rand(sum(sizes), cols, seed=2)
        o = 0
        for s in sizes:
            x[o] += shift
            o += s
        check_stats(tg, x, sizes, groups, f"{cols} columns", 128)


def test_large_graph_among_small_ones(tg):
    """The chunks' join of a graph that is no block's."""
    sizes = [3] * 2000 + [30011] + [2] * 3000
    x = rand(sum(sizes), 64, seed=3)
    x[6000, :] += 3000.0
    x[:, 0] += 500.0
    check_stats(tg, x, sizes, 1, "64 columns", 128)
