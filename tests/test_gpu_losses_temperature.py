"""The distillation loss over its whole range of temperatures (1e-30 to 1e30), and
against a teacher that names a class of a far lower score.

loss = T (T sum q log q - sum q T log p), T log p = (z - max) - T log s: neither
T^2 nor a log p of more than fp32's range stands between finite scores and a
finite loss.  Tolerances are those of test_gpu_losses.py.
"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_losses import DTYPES, assert_within, check_distill, distill64, ints, rand  # noqa: E402

pytestmark = pytest.mark.gpu
CLASSES = [7, 41, 349, 5003, 65537]


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_teacher_of_masked_classes(tg, dtype, classes):
    """The teacher gives a class probability whose score is the type's lowest, or 1e30 below the others: the loss is
    that large, and finite."""
    rows = 160
    low = torch.finfo(dtype).min
    z = rand(rows, classes, seed=classes, scale=2.0, dtype=dtype)
    ids = torch.stack([torch.randperm(classes, generator=torch.Generator().manual_seed(r))[:4] for r in range(rows)]).cuda()
    z[torch.arange(rows), ids[:, 1]] = torch.where(torch.arange(rows, device="cuda") % 2 == 0, low, max(low, -1e30)).to(dtype)
    teacher = rand(rows, 4, seed=2, dtype=dtype)
    for t in (0.7, 1.0, 1.5):
        loss, _ = check_distill(tg, z, ids, teacher, t, None, f"T {t}")
        assert loss.isfinite().all() and (loss > 0.001 * -max(low, -1e30)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_extreme_temperatures(tg, dtype, classes):
    rows = 160
    z = rand(rows, classes, seed=classes, scale=3.0, dtype=dtype)
    ids, teacher = ints(0, classes, (rows, 5), seed=1), rand(rows, 5, seed=2, dtype=dtype)
    ids[::7] = -1
    teacher[3::7] = -float("inf")
    none = torch.zeros(rows, dtype=torch.bool, device="cuda")
    none[::7] = none[3::7] = True
    for t in (1e-30, 1e-25, 1e-20, 1e-15, 1e12, 1e18, 1e25, 1e30):
        want, grad, tol_loss, tol = distill64(z, ids, teacher, t, None)
        alone = tg.distill_loss(z, ids, teacher, t, grad=False)
        loss, dz = tg.distill_loss(z, ids, teacher, t)
        if t < 1e20:  # (above, only rows whose teacher names every class have a loss below fp32's limit)
            assert_within(alone, want, tol_loss, f"T {t} loss alone")
            assert_within(loss, want, tol_loss, f"T {t} loss")
        if dtype != torch.float16 or t < 1:  # (a gradient of T's size)
            assert_within(dz, grad, tol, f"T {t} dlogits")
        for v in (alone, loss):
            assert v[none].eq(0).all() and not v.isnan().any(), f"T {t}"
        assert dz[none].eq(0).all() and not dz.isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_factors_of_the_temperature(tg, dtype):
    """The loss of (z, teacher) at T is T^2 / U^2 times that of (z U / T, teacher U / T) at U, for powers of two."""
    z, ids, teacher = rand(50, 300, seed=1, dtype=dtype), ints(0, 300, (50, 4), 2), rand(50, 4, seed=3, dtype=dtype)
    at = {t: tg.distill_loss(z * t, ids, teacher * t, t)[0].double() / t ** 2 for t in (0.5, 1.0, 4.0)}
    # 2^-24 of a few numbers up to log 300 and the differences of the scores (within 10)
    for t in (0.5, 4.0):
        assert (at[t] - at[1.0]).abs().max() <= 2.0 ** -24 * 2 * 40


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_teacher_of_masked_classes_alone(tg, dtype, classes):
    """All of the teacher's probability at the type's lowest score: the sum over its entries is the largest there is,
    and the loss T times that."""
    rows, k = 160, min(classes - 2, 46)
    low = torch.finfo(dtype).min
    z = rand(rows, classes, seed=classes, scale=2.0, dtype=dtype)
    z[:, :k] = low
    ids = torch.arange(k, device="cuda").expand(rows, k)
    teacher = rand(rows, k, seed=2, dtype=torch.float32)
    for t in (0.1, 0.5, 0.9):
        loss, _ = check_distill(tg, z, ids, teacher, t, None, f"T {t}")
        assert loss.isfinite().all()
