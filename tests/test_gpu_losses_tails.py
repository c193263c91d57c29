"""Best classes among the scores before the first and after the last 16-byte vector
of a row, which other lanes look at before the vectors; the same bits each time."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_losses import DTYPES, best64, rand  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes,rows", [(1030, 1500), (4093, 700), (5003, 300), (40001, 20)])
def test_best_classes_beside_the_vectors(tg, dtype, classes, rows):
    buf = rand(rows * (classes + 5) + 9, seed=classes).to(dtype)
    labels = torch.zeros(rows, dtype=torch.int64, device="cuda")
    for offset, pad in ((0, 0), (1, 0), (3, 5), (7, 2)):
        z = torch.as_strided(buf, (rows, classes), (classes + pad, 1), offset).clone().contiguous()
        for at, value in ((slice(0, 7), 9.0), (slice(classes - 7, classes), 9.0)):
            z[:, at] += value
        z[::3, :5] = 20.0                     # equal ones
        z[1::3, classes - 6:] = 20.0
        into = torch.as_strided(buf, (rows, classes), (classes + pad, 1), offset)
        into.copy_(z)
        for top in (1, 3, 9, 16):
            want = best64(z, top)
            first = tg.label_log_probs(into, labels, top)
            assert torch.equal(first[4], want), f"offset {offset}, top {top}"
            for _ in range(20):
                assert all(torch.equal(a, b) for a, b in zip(tg.label_log_probs(into, labels, top), first))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [5, 16, 41, 64, 100, 256])
def test_last_rows_of_a_block(tg, dtype, classes):
    """Narrow rows whose block has lanes without a row beside theirs: the same bits as among more rows."""
    z = rand(300, classes, seed=classes, scale=3.0, dtype=dtype)
    ids = torch.arange(300 * 6, device="cuda").view(300, 6) * 7 % classes
    teacher, w = rand(300, 6, seed=1), rand(300, seed=2)
    loss, dz = tg.distill_loss(z, ids, teacher, 2.0, w)
    for rows in (1, 2, 3, 7, 8, 9, 31, 33, 63, 65, 100, 127, 257):
        part = tg.distill_loss(z[:rows], ids[:rows], teacher[:rows], 2.0, w[:rows])
        assert torch.equal(part[0], loss[:rows]) and torch.equal(part[1], dz[:rows]), f"{rows} rows"
        assert torch.equal(tg.distill_loss(z[:rows], ids[:rows], teacher[:rows], 2.0, grad=False), loss[:rows])
