"""Training operators on torch tensors: layer norm, typed linear maps and 8-bit
saved activations, each with its backward pass.

Matrices are 2-D CUDA tensors of float32, bfloat16 or float16 with unit column
stride (any row stride; other orders are copied).  Every function runs on
torch's current stream, allocates its results with torch and never waits for
the GPU (:func:`check_row_offsets` does).  Gradients are explicit calls;
nothing here records an autograd graph.  The checks of arguments and the calls
of the C ABI are in ``_torch_ops`` (csrc/api/torchops.cpp); a refusal raises
:class:`InvalidArgument`, a ``ValueError``.

``save8=True`` keeps a matrix for the backward pass in 8 bits
(:class:`Saved8`): a layer norm its normalised rows, a typed linear map its
pre-activation.  The backward functions take the :class:`Saved8` wherever they
take the matrix itself.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from . import build as _build
from .ops import ACT

_build.ensure_built(torchops=True)
from . import _torch_ops as _ops  # noqa: E402

_ops.set_errors(_lib.InvalidArgument, _lib.TinyGNNError)

BLOCK8 = 128  # columns that share an exponent in the saved form
DTYPE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _bad(msg: str) -> _lib.InvalidArgument:
    return _lib.InvalidArgument(_lib.INVALID_ARGUMENT, msg)


def _act(fn: str, act) -> int:
    kind = ACT.get(act)
    if kind is None:
        raise _bad(f"{fn}: unknown activation {act!r}")
    return kind


class Saved8(NamedTuple):
    """A matrix in 8 bits: value = code * 2^(exponent - 127).

    ``codes``: int8, rows x cols, rows starting at multiples of 16 bytes.
    ``exponents``: uint8, rows x ceil(cols / 128), one per row and block of
    128 columns (255: the block held an infinity or a NaN; all NaN).
    ``dtype``: the type of the matrix that was saved."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.shape[0] * (self.codes.shape[1] + self.exponents.shape[1])

    def restore(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The saved values (float32, bfloat16 and the saved type hold them exactly)."""
        kind = DTYPE.get(self.dtype if dtype is None else dtype)
        if kind is None:
            raise _bad("restore: dtype must be float32, bfloat16 or float16")
        return _ops.restore8(self.codes, self.exponents, kind)


Matrix = Union[torch.Tensor, Saved8]


def _parts(fn: str, x: Matrix, dtype: torch.dtype):
    """(matrix, codes, exponents) of a matrix given as it was or in 8 bits."""
    if isinstance(x, Saved8):
        if x.dtype != dtype:
            raise _bad(f"{fn}: the saved matrix was {x.dtype}, {dtype} is needed")
        return None, x.codes, x.exponents
    return x, None, None


# ── 8-bit saved activations ──────────────────────────────────────────────────
def save8(x: torch.Tensor) -> Saved8:
    """x in 8 bits."""
    return Saved8(*_ops.save8(x), x.dtype)


def activation_save8(x: torch.Tensor, act, alpha: float = 0.0):
    """(act(x), x in 8 bits) in one pass."""
    y, codes, exponents = _ops.activation_save8(x, _act("activation_save8", act), alpha)
    return y, Saved8(codes, exponents, x.dtype)


def activation_backward(dy: torch.Tensor, x: Matrix, act, alpha: float = 0.0) -> torch.Tensor:
    """dy * act'(x), x given as it was or in 8 bits."""
    fn = "activation_backward"
    return _ops.activation_backward(dy, *_parts(fn, x, dy.dtype), _act(fn, act), alpha)


# ── layer norm ───────────────────────────────────────────────────────────────
def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, save8: bool = False):
    """(y, stats): y = h * gamma + beta, h = (x - mean) * rstd over each row's
    columns; stats (rows x 2, float32) holds (mean, rstd) for the backward
    pass.  gamma and beta are float32 or of x's type.  With ``save8``,
    (y, stats, h in 8 bits)."""
    out = _ops.layer_norm(x, gamma, beta, eps, save8)
    return (out[0], out[1], Saved8(out[2], out[3], x.dtype)) if save8 else out


def layer_norm_backward(dy: torch.Tensor, saved: Matrix, stats: torch.Tensor, gamma: torch.Tensor):
    """(dx, dgamma, dbeta).  ``saved``: the forward pass's x, or the 8-bit copy
    of its normalised rows.  dgamma and dbeta have gamma's type."""
    return _ops.layer_norm_backward(dy, *_parts("layer_norm_backward", saved, dy.dtype), stats, gamma)


# ── typed linear maps ────────────────────────────────────────────────────────
def check_row_offsets(offsets: torch.Tensor, rows: int) -> torch.Tensor:
    """offsets, after checking on the host that they start at 0, never decrease
    and end at ``rows`` (waits for the GPU; the operators themselves do not
    check, and clamp what is out of range)."""
    _ops.check_row_offsets(offsets, rows)
    return offsets


def typed_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act=None, alpha: float = 0.0, save8: bool = False):
    """act(x[r] @ w[t] + bias[t]) for the rows r of each type t, rows
    offsets[t] .. offsets[t + 1] of x (sorted by type; a type may have none).

    x: rows x K.  w: types x K x N, x's type, at most 1024 types.  offsets:
    types + 1 int32 (:func:`check_row_offsets`).  bias: types x N, float32.
    With ``save8``, (y, pre-activation in 8 bits)."""
    out = _ops.typed_linear(x, w, offsets, bias, _act("typed_linear", act), alpha, save8)
    return (out[0], Saved8(out[1], out[2], x.dtype)) if save8 else out[0]


def typed_linear_grad_input(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """dx[r] = dy[r] @ w[t]^T."""
    return _ops.typed_linear_grad_input(dy, w, offsets)


def typed_linear_grad_weight(x: Matrix, dy: torch.Tensor, offsets: torch.Tensor,
                             dtype: Optional[torch.dtype] = None, bias: bool = True):
    """(dw, db): dw[t] = sum over the type's rows of x[r]^T dy[r] (``dtype``:
    float32 or the rows' type, the default), db[t] = sum of dy[r] (float32;
    None without ``bias``).  x is given as it was or in 8 bits."""
    fn = "typed_linear_grad_weight"
    if dtype is not None and dtype not in (torch.float32, dy.dtype):
        raise _bad(f"{fn}: dw must be float32 or {dy.dtype}, got {dtype}")
    return _ops.typed_linear_grad_weight(dy, *_parts(fn, x, dy.dtype), offsets, dtype == torch.float32, bias)


def typed_linear_backward(dy: torch.Tensor, x: Matrix, w: torch.Tensor, offsets: torch.Tensor,
                          dtype: Optional[torch.dtype] = None, bias: bool = True):
    """(dx, dw, db) of ``x @ w + bias`` (dy: the gradient before the activation,
    :func:`activation_backward`)."""
    if w.dim() == 3 and (len(x.shape) != 2 or w.shape[1] != x.shape[1]):
        raise _bad(f"typed_linear_backward: dimension mismatch — x has shape {tuple(x.shape)}, w {tuple(w.shape)}")
    dx = _ops.typed_linear_grad_input(dy, w, offsets)
    dw, db = typed_linear_grad_weight(x, dy, offsets, dtype, bias)
    return dx, dw, db
