"""Training operators on torch tensors: layer norm, typed linear maps and 8-bit
saved activations, each with its backward pass.

Matrices are 2-D CUDA tensors of float32, bfloat16 or float16 with unit column
stride (any row stride; other orders are copied).  Like :mod:`.ops`, every
function calls entry points of the C ABI on torch's current stream, allocates
its results with torch and never waits for the GPU.  Gradients are explicit
calls; nothing here records an autograd graph.

``save8=True`` keeps a matrix for the backward pass in 8 bits
(:class:`Saved8`): a layer norm its normalised rows, a typed linear map its
pre-activation.  The backward functions take the :class:`Saved8` wherever they
take the matrix itself.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib
from ._lib import check, lib
from .ops import ACT

BLOCK8 = 128  # columns that share an exponent in the saved form
DTYPE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _bad(msg: str) -> _lib.InvalidArgument:
    return _lib.InvalidArgument(_lib.INVALID_ARGUMENT, msg)


def _matrix(t: torch.Tensor, fn: str, name: str, dtype=None, shape=None) -> torch.Tensor:
    """t as a 2-D CUDA matrix with unit column stride, of the given type and shape."""
    if t.dim() != 2 or not t.is_cuda or t.dtype not in DTYPE:
        raise ValueError(f"{fn}: {name} must be a 2-D float32, bfloat16 or float16 CUDA tensor")
    if dtype is not None and t.dtype != dtype:
        raise _bad(f"{fn}: {name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise _bad(f"{fn}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.shape[1] < 1:
        raise _bad(f"{fn}: {name} has no columns")
    # Rows that overlap or run backwards (an expanded row) are laid out first.
    if not t.is_contiguous() and ((t.stride(1) != 1 and t.shape[1] > 1)
                                  or (t.stride(0) < t.shape[1] and t.shape[0] > 1)):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    ld, cols = t.stride(0), t.shape[1]
    return ld if ld >= cols else cols  # the stride of a single row is arbitrary


def _stream(t: torch.Tensor) -> int:
    """The current stream's handle, by the calls under torch.cuda.current_stream
    (which builds two objects a call: 7 us of a small operator's 20)."""
    dev = t.get_device()
    if dev != torch._C._cuda_getDevice():
        raise ValueError(f"the tensors are on {t.device}, which is not the current CUDA device")
    return torch._C._cuda_getCurrentRawStream(dev)


def _act(fn: str, act) -> int:
    if act not in ACT:
        raise _bad(f"{fn}: unknown activation {act!r}")
    return ACT[act]


def _same_device(fn: str, a: torch.Tensor, *others) -> None:
    dev = a.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{fn}: tensors on {a.device} and {t.device}")


@dataclass
class Saved8:
    """A matrix in 8 bits: value = code * 2^(exponent - 127).

    ``codes``: int8, rows x cols, rows starting at multiples of 16 bytes.
    ``exponents``: uint8, rows x ceil(cols / 128), one per row and block of
    128 columns (255: the block held an infinity or a NaN; all NaN).
    ``dtype``: the type of the matrix that was saved."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype

    @classmethod
    def empty(cls, rows: int, cols: int, dtype: torch.dtype, device) -> "Saved8":
        ld = (cols + 15) // 16 * 16
        codes = torch.empty((rows, ld), dtype=torch.int8, device=device)
        exponents = torch.empty((rows, (cols + BLOCK8 - 1) // BLOCK8), dtype=torch.uint8, device=device)
        return cls(codes if ld == cols else codes[:, :cols], exponents, dtype)

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.shape[0] * (self.codes.shape[1] + self.exponents.shape[1])

    def restore(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The saved values (exact in float32 and bfloat16)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in DTYPE:
            raise ValueError("restore: dtype must be float32, bfloat16 or float16")
        s = self._checked("restore", dtype=self.dtype)
        rows, cols = s.shape
        y = torch.empty((rows, cols), dtype=dtype, device=s.codes.device)
        check(lib.tg_restore8(rows, cols, *s._args(), DTYPE[dtype], y.data_ptr(), _ld(y), _stream(y)))
        return y

    def _checked(self, fn: str, dtype, shape=None) -> "Saved8":
        c, e = self.codes, self.exponents
        if c.dim() != 2 or e.dim() != 2 or c.dtype != torch.int8 or e.dtype != torch.uint8 or not (
                c.is_cuda and e.is_cuda):
            raise ValueError(f"{fn}: a Saved8 holds a 2-D int8 and a 2-D uint8 CUDA tensor")
        if self.dtype not in DTYPE or self.dtype != dtype:
            raise _bad(f"{fn}: the saved matrix was {self.dtype}, {dtype} is needed")
        if shape is not None and c.shape != shape:
            raise _bad(f"{fn}: the saved matrix must have shape {tuple(shape)}, got {tuple(c.shape)}")
        if e.shape[0] != c.shape[0] or e.shape[1] != (c.shape[1] + BLOCK8 - 1) // BLOCK8:
            raise _bad(f"{fn}: exponents of shape {tuple(e.shape)} do not fit codes of shape {tuple(c.shape)}")
        if c.shape[0] and (c.stride(1) != 1 and c.shape[1] > 1 or _ld(c) % 16 or c.data_ptr() % 16
                           or e.stride(1) != 1 and e.shape[1] > 1):
            raise _bad(f"{fn}: rows of codes must be contiguous and start at multiples of 16 bytes")
        return self

    def _args(self):
        c, e = self.codes, self.exponents
        ld = c.stride(0) if c.shape[0] > 1 else (c.shape[1] + 15) // 16 * 16
        return c.data_ptr(), ld, e.data_ptr(), max(_ld(e), e.shape[1])


def _saved_or_matrix(x: Union[torch.Tensor, Saved8], fn: str, name: str, dtype, shape):
    """(pointer, ld, codes, ld, exponents, ld) of a matrix or its saved form."""
    if isinstance(x, Saved8):
        return x, (None, 0, *x._checked(fn, dtype, shape)._args())
    x = _matrix(x, fn, name, dtype, shape)
    return x, (x.data_ptr(), _ld(x), None, 0, None, 0)


# ── 8-bit saved activations ──────────────────────────────────────────────────
def save8(x: torch.Tensor) -> Saved8:
    """x in 8 bits."""
    x = _matrix(x, "save8", "x")
    rows, cols = x.shape
    s = Saved8.empty(rows, cols, x.dtype, x.device)
    check(lib.tg_save8(rows, cols, DTYPE[x.dtype], x.data_ptr(), _ld(x), _lib.ACT_NONE, 0.0, None, 0, *s._args(),
                       _stream(x)))
    return s


def activation_save8(x: torch.Tensor, act, alpha: float = 0.0):
    """(act(x), x in 8 bits) in one pass."""
    x = _matrix(x, "activation_save8", "x")
    kind = _act("activation_save8", act)
    rows, cols = x.shape
    y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    s = Saved8.empty(rows, cols, x.dtype, x.device)
    check(lib.tg_save8(rows, cols, DTYPE[x.dtype], x.data_ptr(), _ld(x), kind, alpha, y.data_ptr(), _ld(y),
                       *s._args(), _stream(x)))
    return y, s


def activation_backward(dy: torch.Tensor, x: Union[torch.Tensor, Saved8], act, alpha: float = 0.0) -> torch.Tensor:
    """dy * act'(x), x given as it was or in 8 bits."""
    dy = _matrix(dy, "activation_backward", "dy")
    kind = _act("activation_backward", act)
    x, xargs = _saved_or_matrix(x, "activation_backward", "x", dy.dtype, dy.shape)
    _same_device("activation_backward", dy, x.codes if isinstance(x, Saved8) else x)
    rows, cols = dy.shape
    dx = torch.empty((rows, cols), dtype=dy.dtype, device=dy.device)
    check(lib.tg_activation_grad(rows, cols, DTYPE[dy.dtype], dy.data_ptr(), _ld(dy), *xargs, kind, alpha,
                                 dx.data_ptr(), _ld(dx), _stream(dy)))
    return dx


# ── layer norm ───────────────────────────────────────────────────────────────
def _param(t: torch.Tensor, fn: str, name: str, dtype, cols: int) -> torch.Tensor:
    if t.numel() != cols:
        raise _bad(f"{fn}: {name} must have {cols} elements, got {t.numel()}")
    if not t.is_cuda or t.dtype not in (torch.float32, dtype):
        raise ValueError(f"{fn}: {name} must be a float32 or {dtype} CUDA tensor")
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, save8: bool = False):
    """(y, stats): y = h * gamma + beta, h = (x - mean) * rstd over each row's
    columns; stats (rows x 2, float32) holds (mean, rstd) for the backward
    pass.  With ``save8``, (y, stats, h in 8 bits)."""
    fn = "layer_norm"
    x = _matrix(x, fn, "x")
    rows, cols = x.shape
    gamma, beta = _param(gamma, fn, "gamma", x.dtype, cols), _param(beta, fn, "beta", x.dtype, cols)
    if gamma.dtype != beta.dtype:
        raise _bad(f"{fn}: gamma is {gamma.dtype} and beta {beta.dtype}")
    _same_device(fn, x, gamma, beta)
    y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
    s = Saved8.empty(rows, cols, x.dtype, x.device) if save8 else None
    check(lib.tg_layer_norm(rows, cols, DTYPE[x.dtype], x.data_ptr(), _ld(x), DTYPE[gamma.dtype], gamma.data_ptr(),
                            beta.data_ptr(), eps, y.data_ptr(), _ld(y), stats.data_ptr(),
                            *(s._args() if save8 else (None, 0, None, 0)), _stream(x)))
    return (y, stats, s) if save8 else (y, stats)


def layer_norm_backward(dy: torch.Tensor, saved: Union[torch.Tensor, Saved8], stats: torch.Tensor,
                        gamma: torch.Tensor):
    """(dx, dgamma, dbeta).  ``saved``: the forward pass's x, or the 8-bit copy
    of its normalised rows.  dgamma and dbeta have gamma's type."""
    fn = "layer_norm_backward"
    dy = _matrix(dy, fn, "dy")
    rows, cols = dy.shape
    saved, sargs = _saved_or_matrix(saved, fn, "saved", dy.dtype, dy.shape)
    gamma = _param(gamma, fn, "gamma", dy.dtype, cols)
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise _bad(f"{fn}: stats must be a contiguous float32 tensor of shape ({rows}, 2)")
    _same_device(fn, dy, gamma, stats, saved.codes if isinstance(saved, Saved8) else saved)
    dx = torch.empty((rows, cols), dtype=dy.dtype, device=dy.device)
    dgamma = torch.empty((cols,), dtype=gamma.dtype, device=dy.device)
    dbeta = torch.empty((cols,), dtype=gamma.dtype, device=dy.device)
    check(lib.tg_layer_norm_grad(rows, cols, DTYPE[dy.dtype], dy.data_ptr(), _ld(dy), *sargs, stats.data_ptr(),
                                 DTYPE[gamma.dtype], gamma.data_ptr(), dx.data_ptr(), _ld(dx), dgamma.data_ptr(),
                                 dbeta.data_ptr(), _stream(dy)))
    return dx, dgamma, dbeta


# ── typed linear maps ────────────────────────────────────────────────────────
def check_row_offsets(offsets: torch.Tensor, rows: int) -> torch.Tensor:
    """offsets, after checking on the host that they start at 0, never decrease
    and end at ``rows`` (waits for the GPU; the operators themselves do not
    check, and clamp what is out of range)."""
    _offsets("check_row_offsets", offsets, offsets.numel() - 1)
    check(lib.tg_typed_check_offsets(rows, offsets.numel() - 1, offsets.data_ptr(), _stream(offsets)))
    return offsets


def _offsets(fn: str, offsets: torch.Tensor, types: int) -> None:
    if offsets.dtype != torch.int32 or not offsets.is_cuda or offsets.dim() != 1 or not offsets.is_contiguous():
        raise ValueError(f"{fn}: offsets must be a contiguous 1-D int32 CUDA tensor")
    if offsets.numel() != types + 1:
        raise _bad(f"{fn}: {types} types need {types + 1} offsets, got {offsets.numel()}")


def _weight(fn: str, w: torch.Tensor, dtype, K: Optional[int] = None, N: Optional[int] = None) -> torch.Tensor:
    if w.dim() != 3 or not w.is_cuda:
        raise ValueError(f"{fn}: w must be a 3-D CUDA tensor (types x inputs x outputs)")
    if w.dtype != dtype:
        raise _bad(f"{fn}: w must be {dtype}, got {w.dtype}")
    if (K is not None and w.shape[1] != K) or (N is not None and w.shape[2] != N) or min(w.shape) < 1:
        raise _bad(f"{fn}: dimension mismatch — the rows need w of shape (types, "
                   f"{w.shape[1] if K is None else K}, {w.shape[2] if N is None else N}), got {tuple(w.shape)}")
    k, n = w.shape[1], w.shape[2]
    if (w.stride(2) != 1 and n > 1) or (w.stride(1) < n and k > 1) or (
            w.stride(0) < (k - 1) * w.stride(1) + n and w.shape[0] > 1):
        w = w.contiguous()
    return w


def _wargs(w: torch.Tensor):
    k, n = w.shape[1], w.shape[2]
    ldw = w.stride(1) if k > 1 else max(w.stride(1), n)
    return w.data_ptr(), ldw, w.stride(0) if w.shape[0] > 1 else max(w.stride(0), (k - 1) * ldw + n)


def typed_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act=None, alpha: float = 0.0, save8: bool = False):
    """act(x[r] @ w[t] + bias[t]) for the rows r of each type t, rows
    offsets[t] .. offsets[t + 1] of x (sorted by type; a type may have none).

    x: rows x K.  w: types x K x N, x's type.  offsets: types + 1 int32
    (:func:`check_row_offsets`).  bias: types x N, float32.  With ``save8``,
    (y, pre-activation in 8 bits)."""
    fn = "typed_linear"
    x = _matrix(x, fn, "x")
    rows, K = x.shape
    w = _weight(fn, w, x.dtype, K=K)
    types, _, N = w.shape
    _offsets(fn, offsets, types)
    kind = _act(fn, act)
    if bias is not None:
        if bias.shape != (types, N) or bias.dtype != torch.float32:
            raise _bad(f"{fn}: bias must be float32 of shape ({types}, {N}), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    _same_device(fn, x, w, offsets, bias)
    y = torch.empty((rows, N), dtype=x.dtype, device=x.device)
    s = Saved8.empty(rows, N, x.dtype, x.device) if save8 else None
    check(lib.tg_typed_linear(rows, K, N, types, DTYPE[x.dtype], x.data_ptr(), _ld(x), *_wargs(w), offsets.data_ptr(),
                              None if bias is None else bias.data_ptr(), kind, alpha, y.data_ptr(), _ld(y),
                              *(s._args() if save8 else (None, 0, None, 0)), _stream(x)))
    return (y, s) if save8 else y


def typed_linear_grad_input(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """dx[r] = dy[r] @ w[t]^T."""
    fn = "typed_linear_grad_input"
    dy = _matrix(dy, fn, "dy")
    rows, N = dy.shape
    w = _weight(fn, w, dy.dtype, N=N)
    types, K, _ = w.shape
    _offsets(fn, offsets, types)
    _same_device(fn, dy, w, offsets)
    dx = torch.empty((rows, K), dtype=dy.dtype, device=dy.device)
    check(lib.tg_typed_linear_grad_input(rows, K, N, types, DTYPE[dy.dtype], dy.data_ptr(), _ld(dy), *_wargs(w),
                                         offsets.data_ptr(), dx.data_ptr(), _ld(dx), _stream(dy)))
    return dx


def typed_linear_grad_weight(x: Union[torch.Tensor, Saved8], dy: torch.Tensor, offsets: torch.Tensor,
                             dtype: Optional[torch.dtype] = None, bias: bool = True):
    """(dw, db): dw[t] = sum over the type's rows of x[r]^T dy[r] (``dtype``:
    float32 or the rows' type, the default), db[t] = sum of dy[r] (float32;
    None without ``bias``).  x is given as it was or in 8 bits."""
    fn = "typed_linear_grad_weight"
    dy = _matrix(dy, fn, "dy")
    rows, N = dy.shape
    types = offsets.numel() - 1
    _offsets(fn, offsets, types)
    if types < 1:
        raise _bad(f"{fn}: offsets need at least two elements")
    if x.shape[0] != rows:
        raise _bad(f"{fn}: x has {x.shape[0]} rows and dy {rows}")
    K = x.shape[1]
    x, xargs = _saved_or_matrix(x, fn, "x", dy.dtype, (rows, K))
    dtype = dy.dtype if dtype is None else dtype
    if dtype not in (torch.float32, dy.dtype):
        raise _bad(f"{fn}: dw must be float32 or {dy.dtype}, got {dtype}")
    _same_device(fn, dy, offsets, x.codes if isinstance(x, Saved8) else x)
    dw = torch.empty((types, K, N), dtype=dtype, device=dy.device)
    db = torch.empty((types, N), dtype=torch.float32, device=dy.device) if bias else None
    check(lib.tg_typed_linear_grad_weight(rows, K, N, types, DTYPE[dy.dtype], *xargs, dy.data_ptr(), _ld(dy),
                                          offsets.data_ptr(), DTYPE[dtype], dw.data_ptr(), N, K * N,
                                          db.data_ptr() if bias else None, _stream(dy)))
    return dw, db


def typed_linear_backward(dy: torch.Tensor, x: Union[torch.Tensor, Saved8], w: torch.Tensor, offsets: torch.Tensor,
                          dtype: Optional[torch.dtype] = None, bias: bool = True):
    """(dx, dw, db) of ``x @ w + bias`` (dy: the gradient before the activation,
    :func:`activation_backward`)."""
    if w.dim() == 3 and w.shape[1] != x.shape[1]:
        raise _bad(f"typed_linear_backward: dimension mismatch — x has {x.shape[1]} columns, w {tuple(w.shape)}")
    dx = typed_linear_grad_input(dy, w, offsets)
    dw, db = typed_linear_grad_weight(x, dy, offsets, dtype, bias)
    return dx, dw, db
