"""Infinities and NaN in the gradients of low-rank products: each place holds what float64 gives."""

import pytest
import torch

import low_rank_reference as ref
import tensor_inv_b200 as ti
from test_low_rank import TYPES, no_device_error, operands  # noqa: F401 (a fixture)

INF = float("inf")


def same(got, exact):
    """Bit for bit, infinities with their signs, NaN in the same places."""
    got, want = got.cpu().double(), exact.to(got.dtype).double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])


# few rows (one chunk, results written directly) and several chunks that are joined; one adapter
# and several; a column block that ends inside a vector; ranks in one and in two blocks
SIZES = [(40, 72, 136, 1, 8), (90, 264, 75, 3, 16), (700, 520, 257, 4, 24), (1500, 72, 64, 1, 5),
         (600, 136, 300, 5, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("size", SIZES)
def test_gradients_with_infinities(size, p, dtype):
    """Infinities of both signs in X, in dY and in both: a column of dA (a row of dB) is infinite
    where its infinity meets values other than zero and of one sign, NaN where it meets a zero or
    both signs.  A and B are positive, so that dP and P have few zeros; the float64 form gives the
    places."""
    X, W, A, B, index, scale, dY = operands(*size, dtype=dtype, seed=sum(size))
    A, B = A.abs() + 1, B.abs() + 1
    T, K, N = size[:3]
    at = [(T // 3, 1), (T - 1, K // 2), (T // 2, K - 1), (5, 7), (6, 7)]
    X1, dY1 = X.clone(), dY.clone()
    for i, (t, c) in enumerate(at):
        X1[t, c] = INF if i % 2 else -INF
        dY1[t, c % N] = -INF if i % 2 else INF
    for x, dy in ((X1, dY), (X, dY1), (X1, dY1)):
        exact = ref.backward(dy, x, W, A, B, index, scale, p=p, seed=3)
        got = ti.low_rank_matmul_backward(dy, x, W, A, B, index, scale, p=p, seed=3)
        for G, E in zip(got[1:], exact[1:]):
            same(G, E)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [50, 1000])
def test_infinities_that_stay_infinite(T, dtype):
    """Everything positive: no NaN at all, infinities in the column that holds one."""
    X, W, A, B, index, scale, dY = operands(T, 80, 96, 2, 8, dtype=dtype, seed=1)
    X, W, A, B, dY = (M.abs() + 1 for M in (X, W, A, B, dY))
    index = torch.arange(T, device="cuda") % 2
    X[4, 9] = INF    # adapter 0
    dY[7, 11] = INF  # adapter 1
    P = torch.ones(T, 8, device="cuda")
    _, dA, dB = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, P=P)
    assert not torch.isnan(dA).any() and not torch.isnan(dB).any()
    # (dB is checked against P as given, dA against float64.  The finite sums of 1000 rows reach
    # 500 rows x 96 columns x 1 x 1 x scale 1/2 = 24000 at least and pass fp16's 65504 for most
    # places: those round to infinity, in the exact form too.)
    same(dA, ref.backward(dY, X, W, A, B, index, scale)[1])
    if dtype is torch.bfloat16:
        infinite = torch.zeros_like(dA, dtype=torch.bool)
        infinite[0, 9] = True
        infinite[1] = True  # row 7's dP is infinite, and X has no zeros
        assert torch.equal(torch.isinf(dA), infinite)
    infinite = torch.zeros_like(dB, dtype=torch.bool)
    infinite[1, :, 11] = True
    assert torch.equal(torch.isinf(dB), infinite)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [50, 1000])
def test_projections_at_the_end_of_float32(T):
    """A finite P that bf16 would round to an infinity: the sum is finite."""
    X, W, A, B, index, scale, dY = operands(T, 40, 48, 1, 8, seed=1)
    dY.zero_()
    P = torch.zeros(T, 8, device="cuda")
    dY[3, 5], P[3, 2] = 0.5, torch.finfo(torch.float32).max
    dB = ti.low_rank_matmul_backward(dY, X, W, A, B, index * 0, scale, P=P)[2]
    exact = torch.zeros(dB.shape, dtype=torch.float64)
    exact[0, 2, 5] = P[3, 2].item() / 2
    same(dB, exact)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_nothing_but_nan(p):
    X, W, A, B, index, scale, dY = operands(3000, 520, 264, 2, 72, seed=1)
    X.fill_(float("nan"))
    dY.fill_(float("nan"))
    index = torch.arange(3000, device="cuda") % 2
    for G in ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, p=p, seed=1):
        assert torch.isnan(G).all()
