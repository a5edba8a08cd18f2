"""Training operators of a transformer step on sm_100a kernels: layer norm of
a residual stream, activation checkpoints in 8 bits with the backward passes
that read them, and the softmax cross entropy with its gradient.

Everything here takes CUDA tensors of float32, bfloat16 or float16, works on
the current stream, computes in 32 bits and rounds once at the end. (Inside the
tensor cores, 32-bit sums are cut off rather than rounded; the weight gradient
keeps what that costs under 3e-6 of a sum of one sign for float32 results, and
under a tenth of their own rounding for 16-bit ones.) The last
dimension is a row; rows may lie apart (a slice of a wider tensor), other
orders are copied first, once for both passes. Gradients come through autograd; a
second derivative is refused. What the 8-bit form itself is made of or gives
(``pack8``, ``Act8.unpack``, ``weight_grad8``) carries no gradient: its results
are detached, whether or not its arguments require one.

An 8-bit checkpoint holds a row's groups of 32 neighbours with one power-of-two
step each (33/32 bytes an element): the step s is the smallest with 127 s >=
the group's largest magnitude, a value x is held as rint(x / s), so it is off
by at most s / 2, which is under 1/127 of that magnitude. A finite value stays
finite (63 s and 65504 in the places of 2^128 and float16's 2^16). A group with
an infinity or NaN stands for NaN throughout, so an overflow stays visible.

Waits inside the kernels of ``cross_entropy`` and the weight gradient are
bounded (``COMMUX_KERNEL_WAIT_MS``, 2000 by default). One that runs out leaves
NaN in the results that were not finished, and every operator raises from then
on until ``commux_b200.ops.kernel_status(reset=True)``.
"""

from __future__ import annotations

import torch

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _native():
    from . import _need_native

    return _need_native()


class Act8:
    """A tensor held in 8 bits: ``q`` (int8, [rows, cols rounded up to 32]),
    ``scale`` (uint8, [rows, groups of 32]; 2^(scale - 127) is a group's step),
    the tensor's ``shape`` and ``dtype``. A packed :func:`layer_norm` holds the
    normalised input, before ``weight`` and ``bias``, which then belong to the
    form: the values it stands for are ``held * weight + bias``, with the
    parameters themselves, so an optimizer's step changes them."""

    __slots__ = ("q", "scale", "shape", "dtype", "weight", "bias")

    def __init__(self, q, scale, shape, dtype, weight=None, bias=None):
        self.q, self.scale = q, scale
        self.shape, self.dtype = torch.Size(shape), dtype
        self.weight, self.bias = weight, bias

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.scale.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values as a tensor (of the held tensor's dtype by default), without a gradient."""
        det = [t.detach() if t is not None else None for t in (self.weight, self.bias)]
        return _native().unpack8(self.q, self.scale, list(self.shape), dtype or self.dtype, *det)

    def __repr__(self):
        return f"Act8({tuple(self.shape)}, {self.dtype}, {self.nbytes} bytes)"


def layer_norm(x, weight, bias=None, eps=1e-5, *, residual=None, out_dtype=None, pack=False):
    """Layer norm over the last dimension, of ``x`` or of the stream ``s = x + residual``.

    Returns ``y``; ``(y, s)`` with a residual (``s`` in x's dtype, which is
    what the norm reads); and last, with ``pack``, the :class:`Act8` of ``y``,
    whose held values also replace the stream in what the backward pass keeps.
    ``out_dtype`` is y's dtype: by default autocast's, else x's.
    """
    if out_dtype is None:
        out_dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    got = _native().layer_norm(x, residual, weight, bias, float(eps), out_dtype, bool(pack))
    if residual is None and not pack:
        return got[0]
    out = tuple(got[:1 if residual is None else 2])
    if pack:
        out += (Act8(got[-2], got[-1], x.shape, out_dtype, weight, bias),)
    return out


def pack8(x) -> Act8:
    """``x`` held in 8 bits, without a gradient."""
    q, scale = _native().pack8(x.detach())
    return Act8(q, scale, x.shape, x.dtype)


def gelu8(x, *, approximate="tanh", pack=False):
    """GELU that keeps its input in 8 bits for the backward pass.

    ``approximate`` is "tanh" or "none", as in torch. With ``pack`` the result
    is ``(y, Act8 of y)``, from the same pass, for a :func:`linear8` that follows.
    """
    if approximate not in ("tanh", "none"):
        raise ValueError(f"gelu8: approximate is 'tanh' or 'none', got {approximate!r}")
    got = _native().gelu8(x, approximate == "tanh", bool(pack))
    return (got[0], Act8(got[1], got[2], x.shape, x.dtype)) if pack else got[0]


def linear8(x, weight, bias=None, *, act8=None):
    """``x @ weight.T + bias`` that keeps its input in 8 bits for the weight's gradient.

    ``act8`` is x's 8-bit form where it is there already (from
    :func:`layer_norm` or :func:`gelu8`); x is packed otherwise. Under autocast
    x is cast to its dtype; the weight and the bias may be of other dtypes than
    x, and their gradients are formed in their own.
    """
    if torch.is_autocast_enabled("cuda"):
        x = x.to(torch.get_autocast_dtype("cuda"))
    if act8 is None:
        return _native().linear8(x, weight, bias, None, None, None, None)
    if act8.shape != x.shape:
        raise ValueError(f"linear8: act8 holds {tuple(act8.shape)}, x is {tuple(x.shape)}")
    det = [t.detach() if t is not None else None for t in (act8.weight, act8.bias)]
    return _native().linear8(x, weight, bias, act8.q, act8.scale, *det)


def weight_grad8(dy, act8, *, bias=False, out_dtype=None):
    """Gradient of a linear layer's weight from its output's gradient ``dy``
    ([..., outputs]) and its input's 8-bit form: ``dy.T @ values``, [outputs,
    columns]. With ``bias``, ``(that, dy summed over the rows)``. ``out_dtype``
    is dy's dtype by default. The result carries no gradient."""
    if dy.shape[:-1] != act8.shape[:-1]:
        raise ValueError(f"weight_grad8: dy is {tuple(dy.shape)}, act8 holds {tuple(act8.shape)}")
    det = [t.detach() if t is not None else None for t in (act8.weight, act8.bias)]
    dw, db = _native().weight_grad8(dy, act8.q, act8.scale, act8.shape[-1], *det, bool(bias), out_dtype or dy.dtype)
    return (dw, db) if bias else dw


def cross_entropy(logits, targets, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``logits`` [..., classes] and int64 ``targets`` [...], in float32.

    ``reduction`` is "mean" (over the targets that are not ``ignore_index``),
    "sum" or "none". For the first two the gradient is formed in the forward
    pass, while the logits are on chip; the backward pass hands it out, and
    forms it again only where the upstream gradient is not one. An ignored row
    has a gradient of zero; a target that names no class makes its row NaN.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"cross_entropy: reduction is 'mean', 'sum' or 'none', got {reduction!r}")
    return _native().cross_entropy(logits, targets, int(ignore_index), _REDUCTIONS[reduction])
