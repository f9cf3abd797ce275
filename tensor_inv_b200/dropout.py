"""Dropout whose mask comes from a counter-based generator and is never stored.

Element (row, column) of the mask is a pure function of (seed, offset, row, column): the block
Philox4x32-10 with key ``seed`` and counter ``(column // 8, row, offset)`` gives 16 bits to each
of 8 columns.  Whoever needs the mask makes it again: ``dropout``, its gradient, and the kernels
of ``low_rank_matmul`` and its backward pass.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import numbers

import torch
from torch.autograd import forward_ad

from . import _native as nat

_TYPE_CODES = {
    torch.float16: nat.TI_TYPE_F16,
    torch.bfloat16: nat.TI_TYPE_BF16,
    torch.float32: nat.TI_TYPE_F32,
    torch.float64: nat.TI_TYPE_F64,
}


def drop_numbers(p, seed, offset, device):
    """The fields (cut, seed, seed_ptr, offset) of ti_dropout_spec_t; a seed tensor must outlive the
    launch."""
    if type(p) is not float and not isinstance(p, numbers.Real) or not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be a number in [0, 1], got {p!r}")
    cut = round(65536 * float(p))
    if type(offset) is not int and not isinstance(offset, numbers.Integral) or \
            not 0 <= offset < 2**64:
        raise ValueError(f"offset must be an integer in [0, 2^64), got {offset!r}")
    if seed is None:
        if cut:
            raise ValueError("dropout needs a seed: an integer or a one-element int64 CUDA tensor")
        return cut, 0, None, int(offset)
    if type(seed) is not int and isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed tensor must be one int64 on {device}, got {seed.dtype} "
                             f"{tuple(seed.shape)} on {seed.device}")
        return cut, 0, seed.data_ptr(), int(offset)
    if type(seed) is not int and not isinstance(seed, numbers.Integral) or not 0 <= seed < 2**64:
        raise ValueError(f"seed must be an integer in [0, 2^64) or a one-element int64 CUDA "
                         f"tensor, got {seed!r}")
    return cut, int(seed), None, int(offset)


def refuse_capture(what):
    """Autograd nodes keep the stream they were made on: a backward pass captured while an
    earlier graph of the same leaves lives would join streams that are not being captured,
    which ends the process.  Inside a capture the gradients are asked for by name instead."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} does not record gradients inside a CUDA graph capture; "
                           f"call it under torch.no_grad() and call {what}_backward")


def refuse_tangents(what, *operands):
    """The kernels read a dual tensor's value only, so its tangent would be lost without a word."""
    if forward_ad._current_level < 0:  # no dual_level is open
        return
    for M in operands:
        if isinstance(M, torch.Tensor) and M.is_floating_point() and \
                forward_ad.unpack_dual(M).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative: an operand has a tangent")


def _dropout(X, p, seed, offset):
    numbers_ = drop_numbers(p, seed, offset, X.device)
    if not X.is_cuda:
        raise ValueError("dropout takes a CUDA tensor; it has no CPU path")
    out = X.new_empty(X.shape)
    if X.numel() == 0:
        return out
    X = X.resolve_neg()  # a negative view holds its values unnegated
    flat = X if X.dim() == 2 else X.reshape(-1, X.shape[-1])  # a view where the strides allow it
    rows, cols = flat.shape
    if rows >= 2**32 or cols >= 2**34:
        raise ValueError(f"dropout counts rows in 32 bits and columns in 34: {rows} x {cols}")
    index = X.get_device()
    with nat.on_device(index):
        st = nat.lib().ti_dropout(_TYPE_CODES[X.dtype], flat.data_ptr(), *flat.stride(),
                                  out.data_ptr(), cols, rows, cols,
                                  ctypes.byref(nat.DropoutSpec(*numbers_)), nat.stream_ptr(index))
    nat.check("ti_dropout", st)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, p, seed, offset):
        # a seed tensor is saved, so that a change of it before the backward pass is an error
        ctx.p, ctx.offset = p, offset
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
        return _dropout(X, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dY):
        refuse_capture("dropout")
        seed = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.seed
        return _dropout(dY, ctx.p, seed, ctx.offset), None, None, None


def _check_input(X, name):
    if not isinstance(X, torch.Tensor) or X.dtype not in _TYPE_CODES:
        raise TypeError(f"{name} takes a {', '.join(map(str, _TYPE_CODES))} tensor, got "
                        f"{getattr(X, 'dtype', type(X))}")
    if X.dim() == 0:
        raise ValueError(f"{name} takes a tensor of one dimension or more")


def dropout(X, p, seed=None, offset=0):
    """``X`` with each element dropped (set to 0, whatever it held) with probability ``p`` and
    the others multiplied by ``1 / (1 - p)``.

    ``X``: a CUDA tensor of fp16, bf16, fp32 or fp64, any shape and strides; its last dimension
    counts the columns, the others the rows.  ``p`` is rounded to a multiple of 2^-16 (the factor
    uses the rounded value).  The mask depends on ``seed``, ``offset``, row and column only, not
    on the type.  ``seed``: an integer in [0, 2^64), or a one-element int64 CUDA tensor that is
    read when the kernel runs (a captured graph then draws another mask at each replay whose seed
    was changed).  ``offset``: an integer in [0, 2^64) that tells apart the calls of one seed.

    Differentiable in reverse mode: the gradient is ``dropout_backward``.  Returns a new contiguous tensor.
    """
    _check_input(X, "dropout")
    refuse_tangents("dropout", X)
    if torch.is_grad_enabled() and X.requires_grad:
        if X.is_cuda:
            refuse_capture("dropout")
        return _Dropout.apply(X, p, seed, offset)
    return _dropout(X, p, seed, offset)


def dropout_backward(dY, p, seed=None, offset=0):
    """The gradient of ``dropout`` with respect to its input: the same map applied to ``dY``."""
    _check_input(dY, "dropout_backward")
    refuse_tangents("dropout_backward", dY)
    with torch.no_grad():
        return _dropout(dY, p, seed, offset)
