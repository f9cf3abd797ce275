"""What the low-rank products and dropout refuse beside wrong shapes and types (no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

import tensor_inv_b200 as ti
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
