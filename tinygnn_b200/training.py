"""Training operators on torch tensors: layer norm, group norm, typed linear maps,
8-bit saved activations and the losses on class scores, each with its backward
pass.

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


# ── group norm ───────────────────────────────────────────────────────────────
def group_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, groups: int,
               offsets: Optional[torch.Tensor] = None, act=None, alpha: float = 0.0, eps: float = 1e-5):
    """(y, stats): y = act(h * gamma + beta), h = (x - mean) * rstd over the rows
    of each graph and the cols / groups neighbouring columns of each group.

    x: rows x cols.  offsets: graphs + 1 int32 (:func:`check_row_offsets`),
    graph g has the rows offsets[g] .. offsets[g + 1]; without them all rows are
    one graph.  (A batch of N images or sequences of L places, channels last, is
    ``x.view(N * L, C)`` with the offsets 0, L, 2 L, ...; ``groups=1`` normalises
    whole graphs, ``groups=cols`` each column of a graph.)  gamma and beta are
    float32 or of x's type.  stats (graphs x groups x 2, float32) holds (mean,
    rstd) for the backward pass."""
    return _ops.group_norm(x, gamma, beta, groups, offsets, _act("group_norm", act), alpha, eps)


def group_norm_backward(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, gamma: torch.Tensor,
                        beta: torch.Tensor, groups: int, offsets: Optional[torch.Tensor] = None, act=None,
                        alpha: float = 0.0):
    """(dx, dgamma, dbeta) from the forward pass's x, stats and arguments (the
    pre-activation is computed again).  dgamma and dbeta have gamma's type."""
    return _ops.group_norm_backward(dy, x, stats, gamma, beta, groups, offsets, _act("group_norm_backward", act), alpha)


# ── losses on class scores ───────────────────────────────────────────────────
def label_log_probs(logits: torch.Tensor, labels: torch.Tensor, top: int = 0):
    """(log_probs, entropy, stats), with ``top`` also (top_log_probs, top_classes):
    of each row of scores the log probability of its label, the entropy of its
    probabilities and its ``top`` (at most 128) best classes in falling order,
    equal scores in the order of their classes.

    logits: rows x classes.  labels: int32 or int64; one outside the classes is
    none (log probability 0).  -inf masks a class; a row of masked classes alone
    has NaNs for log probabilities, the entropy 0 and no gradient, a row with a NaN
    or +inf NaNs throughout.
    Results are float32 (top_classes int32); stats (rows x 2) holds (max, log of
    the sum of e^(z - max)) for the backward pass."""
    return _ops.label_log_probs(logits, labels, top)


def label_log_probs_backward(dlog_probs: torch.Tensor, logits: torch.Tensor, labels: torch.Tensor,
                             stats: torch.Tensor, dentropy: Optional[torch.Tensor] = None,
                             entropy: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dlogits from the gradients of log_probs (cross entropy: minus the rows'
    weights) and, with ``dentropy``, of entropy (both float32, one a row; then the
    forward pass's ``entropy`` is needed too).  The top alternatives take none."""
    return _ops.label_log_probs_backward(dlog_probs, logits, labels, stats, dentropy, entropy)


def distill_loss(logits: torch.Tensor, top_classes: torch.Tensor, top_logits: torch.Tensor, temperature: float = 1.0,
                 weights: Optional[torch.Tensor] = None, grad: bool = True):
    """(loss, dlogits), or the loss alone without ``grad``: each row's divergence
    from a teacher of which its best logits are known,

        temperature^2 sum_i q_i (log q_i - log p[c_i]),
        q = softmax(top_logits / temperature), p = softmax(logits / temperature),

    and ``weights`` (float32, one a row; 1 without them) times its gradient: for
    the mean over the rows they are 1 / rows each.

    top_classes, top_logits: rows x k, k at most 128 (:func:`label_log_probs` with
    ``top`` gives both: log probabilities will do).  A class outside the logits'
    classes, or one with a logit of -inf, is none; a row without any has loss and
    gradient 0; a class that occurs twice has both its probabilities.  A row of
    masked logits (-inf) alone has a NaN for its loss and no gradient.
    ``temperature`` is between 1e-30 and 1e30."""
    return _ops.distill_loss(logits, top_classes, top_logits, temperature, weights, grad)
