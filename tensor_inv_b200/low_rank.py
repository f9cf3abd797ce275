"""Low-rank products beside a shared one: adapters of many requests, forward and backward.

``rsvd`` finds the factors of a matrix; these functions apply such factors.  With
``i = index[t]`` the adapter of row t:

    Y[t] = X[t] W + alpha * scale[i] * dropout(X)[t] A[i] B[i]

A weight difference ``D = W1 - W0`` becomes an adapter through ``U, S, Vt = rsvd(D, r)``:
``A = U * S``, ``B = Vt`` serve ``X W1`` as ``low_rank_matmul(X, W0, A, B)``.  The shared product
runs on tcgen05 tensor cores; the low-rank term joins the same accumulator, so Y is written once.
The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import numbers

import torch

from . import _native as nat
from .dropout import drop_numbers, refuse_capture, refuse_tangents

_TYPE_CODES = {torch.float16: nat.TI_TYPE_F16, torch.bfloat16: nat.TI_TYPE_BF16}
MAX_RANK = 256


def _refuse(X, W, A, B):
    """Says what is wrong with the types, shapes or devices of the operands (if anything is)."""
    tensors = {"X": X, "W": W, "A": A, "B": B}
    for name, M in tensors.items():
        if not isinstance(M, torch.Tensor) or M.dtype not in _TYPE_CODES:
            raise TypeError(f"low_rank_matmul takes {' or '.join(map(str, _TYPE_CODES))} "
                            f"tensors, got {name} of {getattr(M, 'dtype', type(M))}")
        if M.dtype != X.dtype:
            raise TypeError(f"X is {X.dtype} and {name} is {M.dtype}: one type for all operands")
        if M.device != X.device:
            raise ValueError(f"X is on {X.device} and {name} is on {M.device}")
    if X.dim() != 2 or W.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise ValueError(f"X (T, K), W (K, N), A (S, K, r), B (S, r, N) expected, got "
                         f"{tuple(X.shape)}, {tuple(W.shape)}, {tuple(A.shape)}, "
                         f"{tuple(B.shape)}")
    (T, K), N, (S, _, r) = X.shape, W.shape[1], A.shape
    if W.shape[0] != K or A.shape[1] != K or B.shape != (S, r, N):
        raise ValueError(f"low_rank_matmul: shapes {tuple(X.shape)}, {tuple(W.shape)}, "
                         f"{tuple(A.shape)}, {tuple(B.shape)} do not fit together")
    if S < 1 or not 1 <= r <= MAX_RANK:
        raise ValueError(f"one adapter or more of rank 1 to {MAX_RANK}, got S = {S}, r = {r}")
    if max(T, K, N, S) >= 2**31:
        raise ValueError("low_rank_matmul takes dimensions below 2^31")


def _describe(X, W, A, B, index, scale, alpha, p, seed, offset):
    """Checks the operands and describes them as a ti_low_rank_t.  Returns it and the tensors
    that it points into (they must outlive the launch)."""
    try:  # the usual case in one look; what is wrong, if anything, is found out below
        (T, K), (K1, N), (S, K2, r), (S1, r1, N1) = X.shape, W.shape, A.shape, B.shape
        dtype, at = X.dtype, X.get_device()
        fits = (K1 == K and K2 == K and S1 == S and r1 == r and N1 == N and 1 <= r <= MAX_RANK and
                1 <= S < 2**31 and T < 2**31 and K < 2**31 and N < 2**31 and
                dtype in _TYPE_CODES and W.dtype is dtype and A.dtype is dtype and
                B.dtype is dtype and
                at == W.get_device() == A.get_device() == B.get_device())
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        _refuse(X, W, A, B)
        raise ValueError("low_rank_matmul: operands do not fit together")
    # a negative view (such as the imaginary part of a conjugate) holds its values unnegated
    if X.is_neg() or W.is_neg() or A.is_neg() or B.is_neg():
        X, W, A, B = X.resolve_neg(), W.resolve_neg(), A.resolve_neg(), B.resolve_neg()
    if index is None:
        if S != 1:
            raise ValueError(f"{S} adapters need an index that says which one each row takes")
        index_ptr, index_bytes = None, 0
    else:
        if not isinstance(index, torch.Tensor) or index.dtype not in (torch.int64, torch.int32):
            raise TypeError("index must be an int32 or int64 tensor")
        if index.dim() != 1 or len(index) != T or index.get_device() != at:
            raise ValueError(f"index must have shape ({T},) on {X.device}, got "
                             f"{tuple(index.shape)} on {index.device}")
        index = index.contiguous()
        index_ptr, index_bytes = index.data_ptr(), index.element_size()
    if scale is None:
        scale_ptr = None
    else:
        if not isinstance(scale, torch.Tensor) or scale.dtype is not torch.float32:
            raise TypeError("scale must be a float32 tensor (one factor for all adapters: alpha)")
        if scale.dim() != 1 or len(scale) != S or scale.get_device() != at:
            raise ValueError(f"scale must have shape ({S},) on {X.device}, got "
                             f"{tuple(scale.shape)} on {scale.device}")
        scale = (scale.resolve_neg() if scale.is_neg() else scale).contiguous()
        scale_ptr = scale.data_ptr()
    if type(alpha) is not float and not isinstance(alpha, numbers.Real):
        raise TypeError("alpha must be a number")
    drop = drop_numbers(p, seed, offset, X.device)
    if at < 0:
        raise ValueError("low_rank_matmul takes CUDA tensors; it has no CPU path")
    op = nat.LowRank(_TYPE_CODES[dtype], T, K, N, S, r, X.data_ptr(), *X.stride(), W.data_ptr(),
                     *W.stride(), A.data_ptr(), *A.stride(), B.data_ptr(), *B.stride(), index_ptr,
                     index_bytes, scale_ptr, alpha, drop)
    return op, (X, W, A, B, index, scale, seed)


def _workspace(op, X, dY=None):
    return X.new_empty(max(nat.low_rank_workspace_size(op, dY), 256), dtype=torch.uint8)


def _forward(X, W, A, B, index, scale, alpha, p, seed, offset, want_p):
    op, keep = _describe(X, W, A, B, index, scale, alpha, p, seed, offset)
    rows, cols, at = op.t, op.n, X.get_device()
    Y = X.new_empty((rows, cols))
    P = X.new_empty((rows, op.r), dtype=torch.float32) if want_p else None
    if rows == 0:
        return Y, P
    with nat.on_device(at):
        ws = _workspace(op, X)
        st = nat.lib().ti_low_rank_matmul(
            ctypes.byref(op), Y.data_ptr(), cols, None if P is None else P.data_ptr(),
            ws.data_ptr(), ws.numel(), nat.stream_ptr(at))
    nat.check("ti_low_rank_matmul", st)
    del keep
    return Y, P


def _backward(dY, X, W, A, B, index, scale, alpha, p, seed, offset, P, needs):
    op, keep = _describe(X, W, A, B, index, scale, alpha, p, seed, offset)
    dev = X.device
    if not isinstance(dY, torch.Tensor) or dY.dtype != X.dtype:
        raise TypeError(f"dY must be a {X.dtype} tensor like X")
    if dY.shape != (op.t, op.n) or dY.device != dev:
        raise ValueError(f"dY must have shape {(op.t, op.n)} on {dev}, got "
                         f"{tuple(dY.shape)} on {dY.device}")
    dY = dY.resolve_neg()
    want_x, want_a, want_b = needs
    if P is None and want_b:
        P = _forward(X, W[:, :0], A, B[:, :, :0], index, scale, alpha, p, seed, offset, True)[1]
    if P is not None:
        if not isinstance(P, torch.Tensor) or P.dtype != torch.float32:
            raise TypeError("P must be the float32 projection that low_rank_matmul returns")
        if P.shape != (op.t, op.r) or P.device != dev:
            raise ValueError(f"P must have shape {(op.t, op.r)} on {dev}, got {tuple(P.shape)} "
                             f"on {P.device}")
        P = P.resolve_neg().contiguous()
    dX = torch.empty((op.t, op.k), dtype=X.dtype, device=dev) if want_x else None
    # the gradients take the layout of A and B (their strides, where those are dense)
    dA = torch.empty_like(A) if want_a else None
    dB = torch.empty_like(B) if want_b else None
    with nat.on_device(dev.index):
        ws = _workspace(op, X, dY)
        st = nat.lib().ti_low_rank_backward(
            ctypes.byref(op), dY.data_ptr(), *dY.stride(), None if P is None else P.data_ptr(),
            None if dX is None else dX.data_ptr(), op.k,
            *((None, 0, 0, 0) if dA is None else (dA.data_ptr(), *dA.stride())),
            *((None, 0, 0, 0) if dB is None else (dB.data_ptr(), *dB.stride())),
            ws.data_ptr(), ws.numel(), nat.stream_ptr(dev.index))
    nat.check("ti_low_rank_backward", st)
    del keep
    return dX, dA, dB


class _LowRank(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W, A, B, index, scale, alpha, p, seed, offset):
        Y, P = _forward(X, W, A, B, index, scale, alpha, p, seed, offset, True)
        ctx.rest = (alpha, p, offset)
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        # index, scale and a seed tensor are saved too: changed in place before the backward
        # pass, they raise like any other saved tensor
        ctx.save_for_backward(X, W, A, B, index, scale, P,
                              seed if isinstance(seed, torch.Tensor) else None)
        ctx.mark_non_differentiable(P)
        return Y, P

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dY, _):
        refuse_capture("low_rank_matmul")
        X, W, A, B, index, scale, P, seed = ctx.saved_tensors
        alpha, p, offset = ctx.rest
        need = ctx.needs_input_grad
        dX, dA, dB = _backward(dY, X, W, A, B, index, scale, alpha, p,
                               ctx.seed if seed is None else seed, offset, P,
                               (need[0], need[2], need[3]))
        return dX, None, dA, dB, None, None, None, None, None, None


def _batched(A, B):
    """One adapter may come without its leading dimension."""
    if isinstance(A, torch.Tensor) and isinstance(B, torch.Tensor) and A.dim() == B.dim() == 2:
        return A.unsqueeze(0), B.unsqueeze(0), True
    return A, B, False


def low_rank_matmul(X, W, A, B, index=None, scale=None, *, alpha=1.0, p=0.0, seed=None, offset=0,
                    return_projection=False):
    """``Y[t] = X[t] W + alpha * scale[i] * dropout(X)[t] A[i] B[i]`` with ``i = index[t]``.

    ``X`` (T, K), ``W`` (K, N), ``A`` (S, K, r), ``B`` (S, r, N): fp16 or bf16 CUDA tensors of one
    type, any strides (a weight stored outputs x inputs is passed as its transposed view); one
    adapter may be given as ``A`` (K, r), ``B`` (r, N).  Rank r from 1 to 256.  ``index`` (T,)
    int32 or int64: the adapter of each row, in any order; a value outside [0, S), such as -1,
    gives the row no low-rank term.  It may be left out when S is 1.  (With several hundred rows
    or more, rows of one adapter next to each other are faster: a tile of rows multiplies with
    every adapter that any of them takes.)  ``scale`` (S,) float32 and
    the number ``alpha`` multiply the term.  ``p``, ``seed``, ``offset``: dropout on X in the
    low-rank term only, with ``dropout``'s mask.

    Sums are held in float32, Y is rounded once.  A row is touched by its own adapter only: NaN
    or infinities in another adapter do not reach it.  The result does not change from run to run.

    Differentiable in reverse mode in X, A and B (W is fixed and may not require a gradient, nor may ``scale``).
    ``return_projection=True`` returns ``(Y, P)``: P (T, r) float32 is what ``low_rank_matmul_backward``
    reads; ``torch.no_grad()`` code, such as a captured training step, passes it there itself.
    """
    refuse_tangents("low_rank_matmul", X, W, A, B, scale)
    A, B, _ = _batched(A, B)
    if torch.is_grad_enabled() and any(getattr(M, "requires_grad", False)
                                       for M in (X, A, B, W, scale)):
        if any(getattr(M, "requires_grad", False) for M in (W, scale)):
            raise ValueError("W and scale are fixed in low_rank_matmul: it computes no gradient "
                             "of them (detach them)")
        if X.is_cuda:
            refuse_capture("low_rank_matmul")
        Y, P = _LowRank.apply(X, W, A, B, index, scale, alpha, p, seed, offset)
    else:
        Y, P = _forward(X, W, A, B, index, scale, alpha, p, seed, offset, return_projection)
    return (Y, P) if return_projection else Y


def low_rank_matmul_backward(dY, X, W, A, B, index=None, scale=None, *, P=None, alpha=1.0, p=0.0,
                             seed=None, offset=0, needs=(True, True, True)):
    """The gradients ``(dX, dA, dB)`` of ``low_rank_matmul`` for the gradient ``dY`` of Y.

    The operands, ``alpha``, ``p``, ``seed`` and ``offset`` are those of the forward call; ``P`` is the
    projection it returned (made again when left out).  ``needs`` says which of the three are
    computed; the others are None.  dX is (T, K); dA and dB have the shapes and the layout of A and
    B and are zero for an adapter that no row takes.  Sums over rows are held in float32 in a
    fixed order; infinities and NaN appear where the formula has them.
    """
    if len(needs) != 3:
        raise ValueError("needs has three entries: dX, dA, dB")
    refuse_tangents("low_rank_matmul_backward", dY, X, W, A, B, scale, P)
    A, B, single = _batched(A, B)
    with torch.no_grad():
        dX, dA, dB = _backward(dY, X, W, A, B, index, scale, alpha, p, seed, offset, P,
                               tuple(map(bool, needs)))
    if single:
        dA, dB = (None if G is None else G[0] for G in (dA, dB))
    return dX, dA, dB
