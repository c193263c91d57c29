"""Training operators at arguments and values where they went wrong once:
refusals, values near zero and far from it, rows and types at the edges of a
rule.  Each against a plain 64-bit implementation.

Tolerances follow from the arithmetic and stand beside each test.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# The smallest step near zero: half of the least subnormal is lost.
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def tg():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import tinygnn_b200
    return tinygnn_b200


def rand(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def test_codes_without_exponents_are_refused(tg):
    """Every entry point that takes a saved matrix refuses codes with no exponents beside them, before any launch."""
    from tinygnn_b200 import _lib
    lib = _lib.lib
    x = rand(4, 64)
    p = x.data_ptr()
    before = lib.tg_kernel_launch_count()
    calls = [
        lambda: lib.tg_layer_norm(4, 8, 0, p, 8, 0, p, p, 1e-5, p, 8, p, p, 16, None, 1, None),
        lambda: lib.tg_typed_linear(4, 8, 8, 1, 0, p, 8, p, 8, 64, p, None, 0, 0.0, p, 8, p, 16, None, 1, None),
        lambda: lib.tg_save8(4, 8, 0, p, 8, 0, 0.0, None, 0, p, 16, None, 1, None),
        lambda: lib.tg_restore8(4, 8, p, 16, None, 1, 0, p, 8, None),
        lambda: lib.tg_activation_grad(4, 8, 0, p, 8, None, 0, p, 16, None, 1, 0, 0.0, p, 8, None),
        lambda: lib.tg_layer_norm_grad(4, 8, 0, p, 8, None, 0, p, 16, None, 1, p, 0, p, p, 8, p, p, None),
        lambda: lib.tg_typed_linear_grad_weight(4, 8, 8, 1, 0, None, 0, p, 16, None, 1, p, 8, p, 0, p, 8, 64, None, None),
    ]
    for k, call in enumerate(calls):
        assert call() == _lib.INVALID_ARGUMENT, k
        assert "exponents is NULL" in _lib.last_error(), k
    assert lib.tg_kernel_launch_count() == before
