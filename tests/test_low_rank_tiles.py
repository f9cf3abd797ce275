"""Low-rank products of more tiles, passes and segments than one CTA holds at a time.

Whole numbers throughout: every sum is exact in float32, so a result is the exact value rounded
once, and calls repeat bit for bit.
"""

import pytest
import torch

import low_rank_reference as ref
import tensor_inv_b200 as ti
from test_low_rank import TYPES, no_device_error, operands  # noqa: F401 (a fixture)


def repeats(call, exact, times=4):
    for _ in range(times):
        got = call()
        assert torch.equal(got.cpu(), exact.to(got.dtype))


# Rows of the result that are aligned to 2, 4, 8 and 16 bytes, in 150 tiles of 256 x 256 or more:
# each of the 74 CTA pairs of a B200 takes several, so that the copies of a tile's operands run
# while the tile before it is stored.
COLUMNS = [4001, 4002, 4004, 4008]


@pytest.mark.gpu
@pytest.mark.parametrize("outer", [False, True])
@pytest.mark.parametrize("N", COLUMNS)
@pytest.mark.parametrize("T, K", [(4096, 136), (2500, 520)])
def test_forward_of_many_tiles(T, K, N, outer):
    X, W, A, B, index, scale, _ = operands(T, K, N, 3, 16, dtype=TYPES[N % 8 // 4], outer=outer,
                                           seed=N)
    exact, _ = ref.forward(X, W, A, B, index, scale)
    repeats(lambda: ti.low_rank_matmul(X, W, A, B, index, scale), exact)


@pytest.mark.gpu
@pytest.mark.parametrize("outer", [False, True])
@pytest.mark.parametrize("K", COLUMNS)
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_gradient_of_many_tiles(p, K, outer):
    X, W, A, B, index, scale, dY = operands(4096, K, 136, 3, 16, dtype=TYPES[K % 8 // 4],
                                            outer=outer, seed=K)
    rest = dict(p=p, seed=5)
    exact = ref.backward(dY, X, W, A, B, index, scale, **rest)[0]
    repeats(lambda: ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale,
                                                needs=(True, False, False), **rest)[0], exact)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("T, K, S, r", [
    (1024, 40, 300, 64), (1024, 64, 700, 8),  # a step per pass: 32 passes of 4 adapters, 8 of 16
    (700, 1088, 200, 64), (520, 1088, 300, 16),  # 17 steps for clusters of 8: two CTAs have none
])
def test_projection_of_many_short_passes(T, K, S, r, p):
    """Tiles whose rows take more adapters than a pass holds: P of the forward pass and, with the
    inner dimension N, of the backward pass (seen through dX)."""
    X, W, A, B, index, scale, dY = operands(T, K, K, S, r, seed=T + r)
    rest = dict(p=p, seed=2)
    exact, exact_p = ref.forward(X, W, A, B, index, scale, **rest)
    dx = ref.backward(dY, X, W, A, B, index, scale, **rest)[0]
    for _ in range(5):
        Y, P = ti.low_rank_matmul(X, W, A, B, index, scale, return_projection=True, **rest)
        assert torch.equal(P.cpu(), exact_p.float())
        assert torch.equal(Y.cpu(), exact.to(Y.dtype))
        dX = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale,
                                         needs=(True, False, False), **rest)[0]
        assert torch.equal(dX.cpu(), dx.to(dX.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [64, 1000])
def test_gradients_of_values_that_cancel(T, dtype):
    """P and dP of 22 bits (fp16: 21) whose column sums cancel to their last one: whole numbers below
    2^24 in every partial sum, so the small sum is exact."""
    K, N, r, top = 80, 96, 8, 2.0**21 if dtype is torch.bfloat16 else 2.0**20
    X, W, A, B, _, _, dY = operands(T, K, N, 1, r, dtype=dtype, seed=T)
    big = top + 2.0**10 + 1
    for M in (X, dY):
        M.zero_()
    X[3], X[T - 2] = 1, -1
    dY[3], dY[T - 2] = 1, -1
    P = torch.zeros(T, r, device="cuda")
    P[3], P[T - 2] = big, big - 1
    dB = ti.low_rank_matmul_backward(dY, X, W, A, B, P=P)[2]
    assert (dB == 1).all()
    # dP of the same values: dY B with the three parts of the number in three columns of dY
    B.zero_()
    B[0, :, :3] = 1
    dY.zero_()
    dY[3, 0], dY[3, 1], dY[3, 2] = 2.0**11, 2.0**10, 1
    dY[T - 2, 0], dY[T - 2, 1] = 2.0**11, 2.0**10
    B[0, :, 0] = top / 2.0**11
    dA = ti.low_rank_matmul_backward(dY, X, W, A, B, P=P)[1]
    assert (dA == 1).all()


@pytest.mark.gpu
def test_results_past_32_bits():
    """Y and dX of more than 2^31 elements (4.3 GB), in rows that are not 16-byte aligned: the first
    rows, those around element 2^31 and the last against float64."""
    T, wide, r = 33000, 66001, 8
    X, W, A, B, index, scale, dY = operands(T, 40, wide, 2, r, seed=1)
    near = 2**31 // wide
    rows = torch.cat([torch.arange(at, at + 5) for at in (0, near - 2, T - 5)]).cuda()
    Y = ti.low_rank_matmul(X, W, A, B, index, scale)
    exact, _ = ref.forward(X[rows], W, A, B, index[rows], scale)
    assert torch.equal(Y[rows].cpu(), exact.to(Y.dtype))
    del Y
    back = W.t(), B.transpose(1, 2), A.transpose(1, 2)  # the same product as a gradient
    dX = ti.low_rank_matmul_backward(X, dY, *back, index, scale, needs=(True, False, False))[0]
    assert torch.equal(dX[rows].cpu(), exact.to(dX.dtype))
