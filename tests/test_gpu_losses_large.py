"""More than 2^31 scores or values: the rows past that give the same bits as by
themselves (a graph's rows, as in a batch without the others)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_losses import rand  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def scores(rows, classes):
    """Random rows, repeated (a block of them is made)."""
    z = torch.empty(rows, classes, dtype=torch.bfloat16, device="cuda")
    some = rand(1009, classes, seed=1, scale=3.0, dtype=torch.bfloat16)
    for r in range(0, rows, 1009):
        z[r:r + 1009] = some[:min(1009, rows - r)]
    return z


@pytest.mark.parametrize("rows,classes", [(2 ** 31 // 41 + 5000, 41), (2 ** 31 // 1003 + 999, 1003), (16500, 131072)])
def test_scores_past_2_31(tg, rows, classes):
    z = scores(rows, classes)
    labels = torch.arange(rows, device="cuda") % classes
    a = torch.ones(rows, device="cuda")
    out = tg.label_log_probs(z, labels, 2)
    # Rows that a launch of these alone shares out alike: one of the repeated ones near the start against the last
    # rows' copy of it, whose place among the 1,009 is the same.
    n = min(2018, rows)
    first, last = slice(0, n), slice((rows - n) // 1009 * 1009, (rows - n) // 1009 * 1009 + n)
    for k in (1, 2, 3):
        assert torch.equal(out[k][first], out[k][last])
    assert torch.equal(out[4][first], out[4][last])
    want = torch.log_softmax(z[last].float(), 1).gather(1, labels[last][:, None])[:, 0]
    assert (out[0][last] - want).abs().max() <= 2.0 ** -24 * 40 * (classes / 512 + 64)
    same = labels.clone()
    same[last] = labels[first]
    dz = tg.label_log_probs_backward(a, z, same, out[2], a, out[1])
    assert torch.equal(dz[first], dz[last])
    del dz
    ids = torch.arange(4, device="cuda", dtype=torch.int32).expand(rows, 4).contiguous()
    loss, dz = tg.distill_loss(z, ids, rand(1, 4, seed=2).expand(rows, 4), 2.0, a)
    assert torch.equal(loss[first], loss[last]) and torch.equal(dz[first], dz[last])


def test_values_past_2_31(tg):
    rows, cols = 2 ** 31 // 64 + 70000, 64
    x = scores(rows, cols)
    gamma, beta = rand(cols, seed=3), rand(cols, seed=4)
    for cuts in ([0, 20 * 1009, 40 * 1009, rows - 30 * 1009, rows], None):
        off = torch.tensor(cuts, dtype=torch.int32, device="cuda") if cuts else torch.arange(0, rows + 1, 1, dtype=torch.int32, device="cuda")[::500].contiguous()
        y, stats = tg.group_norm(x, gamma, beta, 8, off, "gelu")
        dx, _, _ = tg.group_norm_backward(y, x, stats, gamma, beta, 8, off, "gelu")
        for a, b in ((0, 1), (-2, -1)):
            b0, b1 = int(off[a]), int(off[b])
            one, st = tg.group_norm(x[b0:b1].clone(), gamma, beta, 8, None, "gelu")
            # (rows shared out otherwise: the statistics within 2^-24 of a few hundred sums, y to a step of its type)
            assert (stats[a if a >= 0 else -1] - st[0]).abs().max() <= 2.0 ** -24 * 400 * 4
            assert ((y[b0:b1].float() - one.float()).abs() <= 2.0 ** -7 * one.float().abs() + 1e-4).all()
            grad = tg.group_norm_backward(one, x[b0:b1].clone(), st, gamma, beta, 8, None, "gelu")[0]
            assert ((dx[b0:b1].float() - grad.float()).abs() <= 2.0 ** -6 * (grad.float().abs() + 1)).all()
        del y, dx
