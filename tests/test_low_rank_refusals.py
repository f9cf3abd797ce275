"""What the low-rank products and dropout refuse beside wrong shapes and types, and operands in unusual
forms that they take."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import tensor_inv_b200 as ti
from tensor_inv_b200 import _native as nat
from test_low_rank import operands


@pytest.mark.parametrize("at", [0, 1, 2, 3, 5, 6, 7])
def test_tangents(at):
    """Forward-mode derivatives are refused, not dropped: X, W, A, B, scale, dY, P."""
    X, W, A, B, index, scale, dY = operands(6, 16, 24, 3, 4, device="cpu")
    ops = [X, W, A, B, index, scale, dY, torch.zeros(6, 4)]
    with forward_ad.dual_level():
        plain = list(ops)
        ops[at] = forward_ad.make_dual(ops[at], torch.ones_like(ops[at]))
        if at < 6:
            with pytest.raises(RuntimeError, match="forward-mode"):
                ti.low_rank_matmul(*ops[:6])
        with pytest.raises(RuntimeError, match="forward-mode"):
            ti.low_rank_matmul_backward(ops[6], *ops[:6], P=ops[7])
        for fn in (ti.dropout, ti.dropout_backward):
            with pytest.raises(RuntimeError, match="forward-mode"):
                fn(ops[at], 0.5, 1)
        with pytest.raises(ValueError, match="CUDA"):  # an open level alone refuses nothing
            ti.low_rank_matmul(*plain[:6])


@pytest.mark.gpu
def test_negative_views():
    """Tensors that hold their values unnegated (torch marks them so) count as what they stand for."""
    ops = operands(40, 64, 72, 2, 8)
    X, W, A, B, index, scale, dY = ops
    P = torch.arange(40.0 * 8, device="cuda").view(40, 8)
    want = (ti.low_rank_matmul(X, W, A, B, index, scale),
            *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, P=P), ti.dropout(X, 0.5, 1))
    X, W, A, B, scale, dY, P = (torch._neg_view(-M) for M in (X, W, A, B, scale, dY, P))
    assert X.is_neg() and torch.equal(X, ops[0])
    got = (ti.low_rank_matmul(X, W, A, B, index, scale),
           *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, P=P), ti.dropout(X, 0.5, 1))
    for G, E in zip(got, want):
        assert torch.equal(G, E)
    Z = torch.randn(6, 10, dtype=torch.complex64, device="cuda")
    assert torch.equal(ti.dropout(Z.conj().imag, 0.5, 1), -ti.dropout(Z.imag, 0.5, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_negative_strides_at_the_c_entry(T):
    """Every dimension of every operand walked backwards; torch's tensors cannot say that."""
    K, N, S, r = 72, 136, 3, 16
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=1)
    want = (ti.low_rank_matmul(X, W, A, B, index, scale),
            *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale))
    stream = torch.cuda.current_stream().cuda_stream

    def backwards(M, dims):
        """M's values in reversed order along `dims`, the address of the first and the strides."""
        turned = M.flip(dims).contiguous()
        strides = [-s if d in dims else s for d, s in enumerate(turned.stride())]
        at = sum(-strides[d] * (M.shape[d] - 1) for d in dims)
        return turned, turned.data_ptr() + at * M.element_size(), strides

    for dims2, dims3 in (((), (0,)), ((0,), (1,)), ((1,), (2,)), ((0, 1), (0, 1, 2))):
        kept, ptr, strides = zip(*(backwards(M, dims3 if M.dim() == 3 else dims2)
                                   for M in (X, W, A, B, dY)))
        op = nat.LowRank(nat.TI_TYPE_BF16, T, K, N, S, r, ptr[0], *strides[0], ptr[1], *strides[1],
                         ptr[2], *strides[2], ptr[3], *strides[3], index.data_ptr(), 8,
                         scale.data_ptr(), 1.0, nat.DropoutSpec())
        size = ctypes.c_size_t(0)
        Y, P = torch.empty_like(want[0]), torch.empty(T, r, device="cuda")
        assert nat.lib().ti_low_rank_workspace_size(ctypes.byref(op), ctypes.byref(size)) == 0
        ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        assert nat.lib().ti_low_rank_matmul(ctypes.byref(op), Y.data_ptr(), N, P.data_ptr(),
                                            ws.data_ptr(), size.value, stream) == nat.TI_OK
        assert torch.equal(Y, want[0])
        dX, dA, dB = torch.empty_like(X), torch.empty_like(A), torch.empty_like(B)
        assert nat.lib().ti_low_rank_backward_workspace_size(
            ctypes.byref(op), ptr[4], *strides[4], ctypes.byref(size)) == nat.TI_OK
        ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        assert nat.lib().ti_low_rank_backward(
            ctypes.byref(op), ptr[4], *strides[4], P.data_ptr(), dX.data_ptr(), K, dA.data_ptr(),
            *dA.stride(), dB.data_ptr(), *dB.stride(), ws.data_ptr(), size.value, stream) == nat.TI_OK
        for G, E in zip((dX, dA, dB), want[1:]):
            assert torch.equal(G, E)
