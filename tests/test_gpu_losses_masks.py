"""Distillation of scores masked by large finite numbers, and of scores whose
maxima are far from zero, against the 64-bit form of test_gpu_losses.py (which
takes the maximum off first; its tolerances hold unchanged: a masked class has
the probability 0 on both sides, and a row's origin, however large, falls out
of the differences that the tolerances are of).
"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_losses import DTYPES, INF, assert_within, check_label, check_label_grad, distill64, ints, rand  # noqa: E402

pytestmark = pytest.mark.gpu

TEMPERATURES = [0.7, 1.0, 2.0, 4.0, 5.0, 8.0, 20.0]
# Narrow rows of 4 and 8 lanes, rows of a warp, blocks' rows, rows of a cluster; rows that a CTA holds and not.
CLASSES = [2, 7, 41, 349, 5003, 33000, 65537]


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def check_distill(tg, z, classes, teacher, temperature, weights, what=""):
    loss, dz = tg.distill_loss(z, classes, teacher, temperature, weights)
    alone = tg.distill_loss(z, classes, teacher, temperature, weights, grad=False)
    want_loss, want, tol_loss, tol = distill64(z, classes, teacher, temperature, weights)
    # p = 2^x of the hardware is 0 below 2^-126, so dlogits = w T (p - q) may lack w T 2^-126 of them (at
    # p = 1.03 x 2^-127 and w T = 2 the gradient is 1.03 x 2^-126, and 0 here).
    lost = 2.0 ** -126 * temperature * (1.0 if weights is None else weights.double().abs()[:, None])
    assert_within(loss, want_loss, tol_loss, f"{what} loss")
    assert_within(alone, want_loss, tol_loss, f"{what} loss alone")
    assert_within(dz, want, tol + lost, f"{what} dlogits")
    return loss, dz


def masks(classes):
    """Which classes a row masks: at random, a lane's (every 4th to 32nd), a vector's, ranges of them, all but one, all."""
    j = torch.arange(classes, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(classes)
    rows = [torch.rand(classes, device="cuda", generator=g) < 0.6, j % 4 == 3, j % 8 == 1, j % 16 == 0, j % 32 == 5, j % 32 != 5,
            (j // 8) % 2 == 0, (j // 2048) % 2 == 0, j >= classes // 2, j < classes // 2, j >= classes - 9, j != classes // 3]
    rows = [r if not r.all() else j != 0 for r in rows] + [torch.ones_like(j, dtype=torch.bool)]
    return torch.stack(rows)


def masked_scores(classes, dtype, copies):
    """Scores with every mask by every value, and which are masked."""
    low = torch.finfo(dtype).min
    values = [v for v in (-1e4, -1e9, -1e10, -1e20, -1e30) if v > low] + [low]
    m = masks(classes).repeat(copies, 1)
    z = [rand(m.shape[0], classes, seed=k, scale=3.0, dtype=dtype).masked_fill_(m, v) for k, v in enumerate(values)]
    return torch.cat(z), m.repeat(len(values), 1)


def unmasked_entries(m, k, seed):
    """k classes a row that it does not mask (any, where it masks all), the same one more than once."""
    order = torch.where(m, 0.0, 1.0) + torch.rand(m.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    ids = order.topk(min(k, m.shape[1]), 1).indices
    free = (~m).sum(1, keepdim=True)
    place = torch.arange(ids.shape[1], device="cuda")[None, :]
    return ids.gather(1, torch.where(free > 0, place % free.clamp(min=1), place))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_distill_of_finite_masks(tg, dtype, classes):
    z, m = masked_scores(classes, dtype, 3 if classes == 349 else 1)  # (349 classes: rows enough for a warp each)
    rows = z.shape[0]
    ids = unmasked_entries(m, 6, seed=1)
    teacher, weights = rand(rows, ids.shape[1], seed=2, scale=2.0, dtype=dtype), rand(rows, seed=3)
    for t in TEMPERATURES:
        loss, dz = check_distill(tg, z, ids, teacher, t, weights, f"T {t}")
        assert loss.isfinite().all() and dz.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_label_of_finite_masks(tg, dtype, classes):
    z, m = masked_scores(classes, dtype, 3 if classes == 349 else 1)
    labels = unmasked_entries(m, 1, seed=1)[:, 0]
    for top in (0, min(classes, 5)):
        out = check_label(tg, z, labels, top)
    check_label_grad(tg, z, labels, out, seed=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_distill_of_scores_far_from_zero(tg, dtype, classes):
    """Maxima of either sign and any size, rows whose lanes' maxima lie on both sides of any limit of size, and
    differences of the type's step there."""
    top = torch.finfo(dtype).max
    rows = []
    for k, (at, spread) in enumerate(((100, 3), (360, 8), (720, 16), (740, 40), (1400, 32), (2900, 64), (1e4, 100), (6e4, 300), (1e6, 2e4),
                                      (1e9, 1e7), (1e10, 1e8), (1e30, 1e28), (3e38, 1e36))):
        if at + 8 * spread < top:
            for sign in (1, -1):
                for scale in (1.0, 0.02):
                    rows.append((sign * at + rand(1, classes, seed=k, scale=spread * scale).clamp(-6 * spread, 6 * spread)).to(dtype))
    z = torch.cat(rows * (6 if classes == 349 else 1))
    ids = ints(0, classes, (z.shape[0], 3), seed=1)
    teacher = rand(z.shape[0], 3, seed=2, dtype=dtype)
    for t in TEMPERATURES[:4] + [1000.0]:
        check_distill(tg, z, ids, teacher, t, None, f"T {t}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_at_small_temperatures(tg, dtype):
    """Maxima of ordinary scores over a temperature that makes them large."""
    for classes in (7, 41, 349, 5003):
        z = rand(170, classes, seed=classes, scale=3.0, dtype=dtype)
        ids = z.float().topk(2, 1).indices
        for t in (1e-3, 1e-6, 1e-9, 1e-12):
            loss, dz = check_distill(tg, z, ids, rand(170, 2, seed=1, dtype=dtype), t, None, f"T {t}")
            assert not loss.isnan().any() and not dz.isnan().any()
    assert INF > loss.abs().max()
