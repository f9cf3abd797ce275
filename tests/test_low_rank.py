"""low_rank_matmul and its backward pass: values, isolation of rows, refusals, capture, streams.

Two kinds of values.  Small whole numbers: every product and sum is exact in float32 (far below
2^24), so the result is the exact value rounded once, bit for bit.  Normal numbers: within a bound
made of the roundings that the kernels do (``bound`` below).
"""

import ctypes
import subprocess
import sys
import threading

import pytest
import torch

import low_rank_reference as ref
import tensor_inv_b200 as ti
from conftest import ROOT
from tensor_inv_b200 import _native as nat

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def no_device_error(request):
    """No kernel gave up on a wait."""
    yield
    if request.node.get_closest_marker("gpu"):
        assert nat.device_error() == 0


def operands(T, K, N, S, r, dtype=torch.bfloat16, whole=True, outer=False, pad=0, seed=0,
             device="cuda", rows="mixed"):
    """X, W, A, B, index, scale, dY; outer: factors stored transposed; pad: rows of X and dY cut out
    of a wider buffer."""
    g = torch.Generator().manual_seed(seed)

    def values(*shape):
        if whole:
            return torch.randint(-2, 3, shape, generator=g).to(dtype).to(device)
        return torch.randn(shape, generator=g).to(dtype).to(device)

    def factor(*shape):
        if outer:
            return values(*shape[:-2], shape[-1], shape[-2]).transpose(-1, -2)
        return values(*shape)

    X, dY = values(T, K + pad)[:, pad // 2: pad // 2 + K], values(T, N + pad)[:, :N]
    W, A, B = factor(K, N), factor(S, K, r), factor(S, r, N)
    if rows == "mixed":
        index = torch.randint(-1, S, (T,), generator=g)
    else:  # runs
        index = torch.arange(T) * (S + 1) // max(T, 1) - 1
    scale = 2.0 ** torch.randint(-1, 2, (S,), generator=g) if whole else torch.rand(S, generator=g)
    return X, W, A, B, index.to(device), scale.float().to(device), dY


def bound(exact, magnitude, dtype, terms):
    """One rounding of the result to `dtype`, half a step; before it, sums of at most `terms`
    products in float32 along any path (a projection, then the sum that takes it), each
    addition off by at most one unit 2^-23 of the sum of magnitudes (a tensor core may cut off
    instead of rounding), and the projection split into two 11-bit parts: 2^-21."""
    before = (terms * 2.0**-23 + 2.0**-21) * magnitude
    u = ref.half_step(dtype)
    return u * (exact.abs() + before) + before + torch.finfo(dtype).smallest_normal * u * 2


def check(got, exact, magnitude, terms):
    off = (got.detach().cpu().double() - exact).abs()
    assert (off <= bound(exact, magnitude, got.dtype, terms)).all(), float(off.max())


def check_forward(ops, p=0.0, seed=0, offset=0, alpha=1.0, whole=True):
    X, W, A, B, index, scale, _ = ops
    Y, P = ti.low_rank_matmul(X, W, A, B, index, scale, alpha=alpha, p=p, seed=seed,
                              offset=offset, return_projection=True)
    exact, exact_p = ref.forward(X, W, A, B, index, scale, alpha, p, seed, offset)
    assert Y.shape == exact.shape and Y.dtype == X.dtype and Y.is_contiguous()
    if whole:
        assert torch.equal(P.cpu(), exact_p.float())
        assert torch.equal(Y.cpu(), exact.to(X.dtype))
    else:
        mag, mag_p = ref.forward(X, W, A, B, index, scale, alpha, p, seed, offset, absolute=True)
        (T, K), r = X.shape, A.shape[2]
        check(P, exact_p, mag_p, K + 4)
        check(Y, exact, mag, 2 * K + r + 8)
    return Y, P


def check_backward(ops, p=0.0, seed=0, offset=0, alpha=1.0, whole=True):
    X, W, A, B, index, scale, dY = ops
    rest = dict(alpha=alpha, p=p, seed=seed, offset=offset)
    got = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, **rest)
    exact = ref.backward(dY, X, W, A, B, index, scale, **rest)
    for G, E, M in zip(got, exact, (X, A, B)):
        assert G.shape == M.shape and G.dtype == M.dtype
        if whole:
            assert torch.equal(G.cpu(), E.to(M.dtype))
    if not whole:
        mags = ref.backward(dY, X, W, A, B, index, scale, absolute=True, **rest)
        (T, K), N, r = X.shape, W.shape[1], A.shape[2]
        for G, E, m, terms in zip(got, exact, mags, (2 * N + r + 8, N + T + 8, K + T + 8)):
            check(G, E, m, terms)
    return got


# T, K, N, S, r: one row, odd sizes, sizes around tiles, ranks around 8 and 16, more adapters
# than rows, more rows than a tile
SIZES = [
    (1, 64, 64, 1, 1), (1, 1, 1, 1, 1), (1, 200, 300, 3, 8), (2, 129, 65, 2, 5), (7, 96, 40, 9, 16),
    (16, 256, 128, 4, 32), (31, 72, 520, 40, 3), (33, 1000, 264, 2, 64), (64, 64, 64, 64, 8),
    (100, 333, 77, 3, 13), (129, 128, 256, 2, 16), (200, 511, 129, 5, 17), (257, 64, 513, 3, 128),
    (300, 40, 1000, 2, 256), (384, 320, 192, 1, 24), (777, 257, 255, 6, 12),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("outer", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_whole_numbers(size, outer, dtype):
    check_forward(operands(*size, dtype=dtype, outer=outer, seed=sum(size)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("outer", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_backward_whole_numbers(size, outer, dtype):
    check_backward(operands(*size, dtype=dtype, outer=outer, seed=sum(size)))


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
def test_dropout_whole_numbers(size):
    """p = 1/2: the factor is 2, everything stays exact."""
    ops = operands(*size, outer=size[0] % 2 == 1, seed=3 + sum(size), pad=3)
    check_forward(ops, p=0.5, seed=2**63 + 11, offset=2**40 + 1)
    check_backward(ops, p=0.5, seed=2**63 + 11, offset=2**40 + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 500, 300, 2, 16), (40, 1024, 136, 8, 8), (150, 257, 260, 3, 24),
                                  (600, 384, 512, 4, 40)])
def test_normal_numbers(size, dtype):
    for outer, rows in ((False, "mixed"), (True, "runs")):
        ops = operands(*size, dtype=dtype, whole=False, outer=outer, rows=rows, seed=5)
        check_forward(ops, whole=False, alpha=0.37)
        check_backward(ops, whole=False, alpha=0.37, p=0.2, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2000, 520, 392, 3, 16), (1024, 2048, 640, 1, 32),
                                  (515, 4096, 1032, 2, 64), (4100, 136, 264, 7, 8)])
def test_larger_whole_numbers(size):
    """More rows than one wave of tiles and longer sums; |sums| <= 4096 * 4 + 64 * 2^14 * 8, and
    entries of A are thinned out to keep them below 2^24."""
    X, W, A, B, index, scale, dY = operands(*size, rows="runs", outer=True, seed=9)
    g = torch.Generator("cuda").manual_seed(1)
    A = torch.where(torch.rand(A.shape, device="cuda", generator=g) < 0.05, A, 0)
    B = torch.where(torch.rand(B.shape, device="cuda", generator=g) < 0.2, B, 0)
    ops = X, W, A, B, index, scale, dY
    check_forward(ops)
    check_backward(ops, p=0.5, seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 70, 300])
def test_strides(T):
    """Every operand in odd layouts: both strides above 1, rows that start at odd addresses,
    an adapter shared by all (stride 0), an index of stride 2, transposed X and dY."""
    K, N, S, r = 72, 136, 4, 16
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=1)

    def spread(M, step):
        wide = torch.full([step * d for d in M.shape], float("nan"), device="cuda", dtype=M.dtype)
        view = wide[tuple(slice(None, None, step) for _ in M.shape)]
        return view.copy_(M)

    def odd(M):
        flat = torch.empty(M.numel() + M.shape[0] * 9 + 1, device="cuda", dtype=M.dtype)
        n = M[0].numel()
        return torch.as_strided(flat, M.shape, (n + 9, *M.stride()[1:]), 1).copy_(M)

    index2 = torch.stack([index, index * 0 + 99], 1)[:, 0]
    turned = (X.t().contiguous().t(), W, A, B, index.int(), scale, dY.t().contiguous().t())
    for ops in ((spread(X, 2), spread(W, 3), spread(A, 2), spread(B, 2), index2, scale,
                 spread(dY, 2)),
                (odd(X), odd(W), odd(A.contiguous()), odd(B.contiguous()), index, scale, odd(dY)),
                turned,
                (X, W, A[:1].expand(S, K, r), B[1:2].expand(S, r, N), index, scale, dY)):
        check_forward(ops)
        check_backward(ops, p=0.5, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 64, 400])
def test_rows_see_their_own_adapter_only(T):
    """NaN and infinities in one adapter, and in rows without a term or of other adapters, reach
    nothing else; the rows that do take that adapter get what the formula gives."""
    K, N, S, r = 200, 264, 3, 16
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=2)
    index = (torch.arange(T, device="cuda") % 4) - 1
    clean = ti.low_rank_matmul(X, W, A, B, index, scale)
    clean_grads = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale)
    A2, B2 = A.clone(), B.clone()
    A2[1, 3, 2] = float("nan")
    B2[1, 5, 7] = float("inf")
    Y = ti.low_rank_matmul(X, W, A2, B2, index, scale)
    other = index != 1
    assert torch.equal(Y[other], clean[other])
    grads = ti.low_rank_matmul_backward(dY, X, W, A2, B2, index, scale)
    assert torch.equal(grads[0][other], clean_grads[0][other])
    for G, C in zip(grads[1:], clean_grads[1:]):
        assert torch.equal(G[[0, 2]], C[[0, 2]])
    # an infinity in B: only column 7 of that adapter's rows, with the sign of P
    Y, P = ti.low_rank_matmul(X, W, A, B2, index, scale, return_projection=True)
    exact, _ = ref.forward(X, W, A, B2, index, scale)
    assert torch.equal(torch.nan_to_num(Y.cpu().double(), 1e9), torch.nan_to_num(
        exact.to(X.dtype).double(), 1e9))
    assert torch.isinf(Y).any()
    # rows of X and dY that hold NaN touch their own rows and their own adapter's gradients
    X3, dY3 = X.clone(), dY.clone()
    X3[2] = float("nan")     # adapter 1
    dY3[2] = float("inf")
    Y = ti.low_rank_matmul(X3, W, A, B, index, scale)
    rest = torch.arange(T, device="cuda") != 2
    assert torch.equal(Y[rest], clean[rest]) and torch.isnan(Y[2]).all()
    grads = ti.low_rank_matmul_backward(dY3, X3, W, A, B, index, scale)
    assert torch.equal(grads[0][rest], clean_grads[0][rest])
    for G, C in zip(grads[1:], clean_grads[1:]):
        assert torch.equal(G[[0, 2]], C[[0, 2]]) and not torch.isfinite(G[1]).all()


@pytest.mark.gpu
def test_infinite_projection():
    """An infinite row of X: what float64 gives, infinities and NaN in the same places."""
    X, W, A, B, index, scale, _ = operands(70, 64, 40, 2, 4, seed=8)
    A, B = A.abs() + 1, B.abs() + 1
    W = W.abs() + 1
    X[3, 5], X[69, 1] = float("inf"), float("-inf")
    Y = ti.low_rank_matmul(X, W, A, B, index, scale)
    exact, _ = ref.forward(X, W, A, B, index, scale)
    assert torch.equal(Y.cpu().double(), exact.to(X.dtype).double())
    assert torch.isinf(Y[3]).all() and torch.isinf(Y[69]).all()


@pytest.mark.gpu
def test_projections_beyond_half_precision():
    """fp16 operands whose projection leaves fp16's range at both ends: it is held in float32."""
    X, W, A, B, index, scale, dY = operands(300, 256, 64, 1, 8, dtype=torch.float16, whole=False)
    for big, small in ((60.0, 2.0**-12), (2.0**-14, 4096.0)):
        ops = (X * big, W * 0, A * big, B * small, index, scale, dY)
        check_forward(ops, whole=False)
        check_backward((X * big, W, A * small, B * small, index, scale, dY * big), whole=False)


@pytest.mark.gpu
def test_empty_and_unused():
    X, W, A, B, index, scale, dY = operands(10, 32, 24, 3, 4)
    Y = ti.low_rank_matmul(X[:0], W, A, B, index[:0], scale)
    assert Y.shape == (0, 24)
    grads = ti.low_rank_matmul_backward(dY[:0], X[:0], W, A, B, index[:0], scale)
    assert grads[0].shape == (0, 32) and (grads[1] == 0).all() and (grads[2] == 0).all()
    assert ti.low_rank_matmul(X, W[:, :0], A, B[:, :, :0], index, scale).shape == (10, 0)
    Y = ti.low_rank_matmul(X[:, :0], W[:0], A[:, :0], B, index, scale)
    assert Y.shape == (10, 24) and (Y == 0).all()
    none = torch.full_like(index, -1)
    assert torch.equal(ti.low_rank_matmul(X, W, A, B, none, scale),
                       (X.double() @ W.double()).to(X.dtype))
    far = torch.where(index >= 0, index, 2**40)  # values outside [0, S) mean none, like -1
    assert torch.equal(ti.low_rank_matmul(X, W, A, B, far, scale),
                       ti.low_rank_matmul(X, W, A, B, index, scale))
    only = torch.full_like(index, 1)
    _, dA, dB = ti.low_rank_matmul_backward(dY, X, W, A, B, only, scale)
    assert (dA[[0, 2]] == 0).all() and (dB[[0, 2]] == 0).all() and (dA[1] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 300])
def test_one_adapter_without_its_leading_dimension(T):
    X, W, A, B, _, _, dY = operands(T, 64, 48, 1, 4, seed=4)
    Y = ti.low_rank_matmul(X, W, A[0], B[0])
    assert torch.equal(Y.cpu(), ref.forward(X, W, A, B, None, None)[0].to(X.dtype))
    dX, dA, dB = ti.low_rank_matmul_backward(dY, X, W, A[0], B[0])
    for G, E in zip((dX, dA, dB), ref.backward(dY, X, W, A, B, None, None)):
        assert torch.equal(G.cpu(), E.to(X.dtype).reshape(G.shape))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
def test_autograd_and_differences(T):
    """Autograd gives the named backward pass; and since Y is linear in each operand alone, a
    difference of exact values is exact: <dY, Y(M + E) - Y(M)> = <dM, E>."""
    X, W, A, B, index, scale, dY = operands(T, 80, 56, 3, 8, seed=6)
    leaves = [M.detach().clone().requires_grad_() for M in (X, A, B)]
    rest = dict(alpha=0.5, p=0.5, seed=3, offset=1)
    Y, P = ti.low_rank_matmul(leaves[0], W, leaves[1], leaves[2], index, scale,
                              return_projection=True, **rest)
    assert not P.requires_grad
    Y.backward(dY)
    named = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, P=P, **rest)
    for M, G in zip(leaves, named):
        assert torch.equal(M.grad, G)
    some = ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, needs=(False, True, False),
                                       **rest)
    assert some[0] is None and some[2] is None and torch.equal(some[1], named[1])
    exact = ref.backward(dY, X, W, A, B, index, scale, **rest)
    g = torch.Generator().manual_seed(0)
    for k, M in enumerate((X, A, B)):
        E = torch.randint(-1, 2, M.shape, generator=g).to(M.dtype).cuda()
        moved = [X, A, B]
        moved[k] = M + E
        before = ref.forward(X, W, A, B, index, scale, 0.5, 0.5, 3, 1)[0]
        after = ref.forward(moved[0], W, moved[1], moved[2], index, scale, 0.5, 0.5, 3, 1)[0]
        slope = ((after - before) * dY.cpu().double()).sum()
        assert slope == (exact[k] * E.cpu().double()).sum()


@pytest.mark.gpu
def test_repeats_bit_for_bit():
    ops = operands(700, 264, 520, 5, 16, whole=False, seed=1)
    X, W, A, B, index, scale, dY = ops
    first = (ti.low_rank_matmul(X, W, A, B, index, scale),
             *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, p=0.1, seed=1))
    for _ in range(3):
        again = (ti.low_rank_matmul(X, W, A, B, index, scale),
                 *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, p=0.1, seed=1))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 300])
def test_capture(T):
    """A training step captured through the named calls, replayed with other inputs and seeds;
    two graphs side by side keep their own workspaces; autograd inside a capture is refused."""
    X, W, A, B, index, scale, dY = operands(T, 136, 72, 3, 8, seed=3)
    seed = torch.tensor([1], device="cuda")

    def step():
        with torch.no_grad():
            Y, P = ti.low_rank_matmul(X, W, A, B, index, scale, p=0.5, seed=seed,
                                      return_projection=True)
            return (Y, *ti.low_rank_matmul_backward(dY, X, W, A, B, index, scale, P=P, p=0.5,
                                                    seed=seed))

    step()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    leaf = A.detach().clone().requires_grad_()
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
            with pytest.raises(RuntimeError, match="capture"):
                ti.low_rank_matmul(X, W, leaf, B, index, scale)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in (4, 9):
        seed.fill_(s)
        X.copy_(torch.randint(-2, 3, X.shape))
        index.copy_(torch.randint(-1, 3, index.shape))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):  # may run at the same time
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        expect = step()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, expect))


@pytest.mark.gpu
def test_two_calls_at_once_on_two_streams():
    ops = operands(500, 520, 264, 3, 16, seed=2)
    X, W, A, B, index, scale, dY = ops
    expect = ti.low_rank_matmul(X, W, A, B, index, scale)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ti.low_rank_matmul(X, W, A, B, index, scale))
    torch.cuda.synchronize()
    assert all(torch.equal(Y, expect) for Y in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 130])
def test_offsets_past_32_bits(T):
    """Rows of X more than 2^31 elements from its start, and adapters whose offset passes 2^31."""
    K, N, S, r = 64, 72, 3, 8
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=5)
    step = (2**31 // (T - 1) + 8) // 8 * 8
    far = torch.empty(T * step + K, dtype=X.dtype, device="cuda").as_strided((T, K), (step, 1))
    far.copy_(X)
    gap = 2**31 + 64
    farA = torch.empty(2 * gap + K * r, dtype=X.dtype, device="cuda").as_strided(
        (S, K, r), (gap, r, 1))
    farA.copy_(A)
    ops = far, W, farA, B, index, scale, dY
    check_forward(ops)
    dX, dA, dB = ti.low_rank_matmul_backward(dY, far, W, farA, B, index, scale)
    for G, E in zip((dX, dA, dB), ref.backward(dY, X, W, A, B, index, scale)):
        assert torch.equal(G.cpu(), E.to(X.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 50, 300])
def test_what_lies_beside_the_output_is_left(T):
    """The C entry with a leading dimension wider than n and rows behind the last one."""
    K, N, S, r = 64, 75, 2, 8
    X, W, A, B, index, scale, _ = operands(T, K, N, S, r, seed=7)
    from tensor_inv_b200.low_rank import _describe, _workspace

    op, keep = _describe(X, W, A, B, index, scale, 1.0, 0.0, None, 0)
    for ld in (N, N + 5, 80, 96):
        out = torch.full((T + 4, ld), 7.0, dtype=X.dtype, device="cuda")
        ws = _workspace(op, X)
        st = nat.lib().ti_low_rank_matmul(ctypes.byref(op), out.data_ptr(), ld, None,
                                          ws.data_ptr(), ws.numel(),
                                          torch.cuda.current_stream().cuda_stream)
        assert st == nat.TI_OK
        assert torch.equal(out[:T, :N], ti.low_rank_matmul(X, W, A, B, index, scale))
        assert (out[T:] == 7).all() and (out[:, N:] == 7).all()


@pytest.mark.gpu
def test_factors_of_a_weight_difference():
    """The run as it is used: rsvd factors W1 - W0, the factors serve X W1 beside the shared
    W0 together with a second adapter, and a descent step on them by autograd runs."""
    g = torch.Generator("cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64)

    K, N, r, T = 192, 160, 8, 96
    W0 = randn(K, N).bfloat16()
    D = randn(K, r) @ randn(r, N) / 8
    U, S, Vt = ti.rsvd(D, r)
    A = torch.stack([U * S.sqrt(), randn(K, r) / 10]).bfloat16()
    B = torch.stack([S.sqrt()[:, None] * Vt, torch.zeros_like(Vt)]).bfloat16()
    X = randn(T, K).bfloat16()
    index = torch.arange(T, device="cuda") % 3 - 1
    Y = ti.low_rank_matmul(X, W0, A, B, index)
    want = X.double() @ W0.double()
    own = index == 0
    # rounding A and B to bf16 moves D by less than 2^-8 (each by half a step, 2^-9, and the
    # product of both is below 2^-17) of |A||B|; Y itself is rounded by half a step
    low = X.double() @ D
    slack = X.double().abs() @ ((U * S.sqrt()).abs() @ (S.sqrt()[:, None] * Vt).abs())
    want[own] += low[own]
    tol = 2.0**-7 * (1 + 2.0**-6) * slack + 2.0**-8 * (want.abs() + 2.0**-7 * slack) + \
        (2 * K + r + 8) * 2.0**-22 * (X.double().abs() @ W0.double().abs() + slack)
    assert ((Y.double() - want).abs() <= tol).all()
    A.requires_grad_()
    B.requires_grad_()
    Y = ti.low_rank_matmul(ti.dropout(X, 0.1, 1), W0, A, B, index, p=0.1, seed=1, offset=1)
    Y.float().square().mean().backward()
    assert torch.isfinite(A.grad).all() and torch.isfinite(B.grad).all()
    assert (B.grad[1] != 0).any() and (A.grad[1] == 0).all()  # B[1] is zero, so A[1] has no slope
    assert nat.device_error() == 0

@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("N", [73, 74, 75, 76])
def test_factor_cut_from_a_wider_buffer(T, N):
    """Columns that end inside a vector, in rows that are aligned for one: what stands behind them
    (NaN here) is not used, on either side."""
    K, S, r = 75, 3, 8
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=7)
    wide = torch.full((S, r, 80), float("nan"), dtype=B.dtype, device=B.device)
    wide[:, :, :N] = B
    tall = torch.full((S, r, 80), float("nan"), dtype=A.dtype, device=A.device)
    tall[:, :, :K] = A.transpose(1, 2)
    for a, b in ((A, wide[:, :, :N]), (tall[:, :, :K].transpose(1, 2), B),
                 (tall[:, :, :K].transpose(1, 2), wide[:, :, :N])):
        check_forward((X, W, a, b, index, scale, dY))
        check_backward((X, W, a, b, index, scale, dY), p=0.5, seed=1)



@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_odd_layouts_of_factors(T):
    """Adapters whose ranks or columns are the slowest dimension, and operands that repeat one row or
    column (stride 0)."""
    K, N, S, r = 72, 136, 4, 16
    X, W, A, B, index, scale, dY = operands(T, K, N, S, r, seed=1)
    for a, b in ((A.permute(2, 0, 1).contiguous().permute(1, 2, 0),
                  B.permute(2, 0, 1).contiguous().permute(1, 2, 0)),
                 (A.permute(1, 0, 2).contiguous().permute(1, 0, 2),
                  B.permute(1, 0, 2).contiguous().permute(1, 0, 2)),
                 (A[:, :, :1].expand(S, K, r), B[:, :, :1].expand(S, r, N)),
                 (A[:, :1].expand(S, K, r), B[:, :1].expand(S, r, N))):
        check_forward((X, W, a, b, index, scale, dY))
        check_backward((X, W, a, b, index, scale, dY), p=0.5, seed=1)
    ops = X[:1].expand(T, K), W[:, :1].expand(K, N), A, B, index, scale, dY[:, :1].expand(T, N)
    check_forward(ops)
    check_backward(ops, p=0.5, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 100, 300])
def test_everything_dropped(T):
    ops = operands(T, 72, 136, 4, 16, seed=1)
    check_forward(ops, p=1.0, seed=3)
    check_backward(ops, p=1.0, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [10, 300])
def test_gradients_of_empty_dimensions(T):
    X, W, A, B, index, scale, dY = operands(T, 32, 24, 3, 4)
    for K, N in ((0, 24), (32, 0)):
        a, b = A[:, :K], B[:, :, :N]
        grads = ti.low_rank_matmul_backward(dY[:, :N], X[:, :K], W[:K, :N], a, b, index, scale)
        for G, shape in zip(grads, ((T, K), a.shape, b.shape)):
            assert G.shape == shape and (G == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("outer", [False, True])
@pytest.mark.parametrize("size", [
    (256, 200, 136, 32, 16), (257, 200, 136, 32, 16), (320, 328, 257, 40, 13), (321, 328, 257, 40, 13),
    (512, 256, 392, 64, 24), (513, 256, 392, 64, 24), (512, 72, 64, 500, 8)])
def test_borders_between_forms(size, outer):
    """With many adapters the form for few rows reaches further: both sides of its borders."""
    for rows in ("mixed", "runs"):
        ops = operands(*size, outer=outer, rows=rows, seed=4, pad=3)
        check_forward(ops)
        check_backward(ops, p=0.5, seed=8)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [
    (300, 64, 72, 300, 8), (1000, 72, 64, 1000, 5), (600, 264, 136, 3, 256), (40000, 64, 72, 5, 8),
    (5000, 40, 24, 1, 16), (129, 64, 64, 1, 16), (8200, 64, 64, 9, 16)])
def test_many_adapters_many_rows(size):
    """As many adapters as rows, the largest rank, many tiles of few columns, the first rows past a
    rule's border."""
    ops = operands(*size, seed=3, pad=5)
    check_forward(ops)
    check_backward(ops, p=0.5, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(300, 70000, 8, 2, 4), (20, 70000, 8, 2, 4), (300, 8, 70000, 2, 4)])
def test_long_dimensions(size):
    """Inner and outer dimensions past 2^16; factors thinned out so that sums stay below 2^24."""
    X, W, A, B, index, scale, dY = operands(*size, seed=3)
    g = torch.Generator("cuda").manual_seed(1)
    A = torch.where(torch.rand(A.shape, device="cuda", generator=g) < 0.02, A, 0)
    B = torch.where(torch.rand(B.shape, device="cuda", generator=g) < 0.02, B, 0)
    check_forward((X, W, A, B, index, scale, dY))
    check_backward((X, W, A, B, index, scale, dY), p=0.5, seed=2)


@pytest.mark.gpu
def test_a_broadcast_gradient():
    """Y.sum() hands an expanded gradient (strides 0) to the backward pass."""
    X, W, A, B, index, scale, dY = operands(300, 72, 136, 4, 16, seed=1)
    A.requires_grad_()
    X.requires_grad_()
    ti.low_rank_matmul(X, W, A, B, index, scale).sum().backward()
    exact = ref.backward(torch.ones_like(dY), X, W, A, B, index, scale)
    assert torch.equal(X.grad.cpu(), exact[0].to(X.dtype))
    assert torch.equal(A.grad.cpu(), exact[1].to(X.dtype))


@pytest.mark.gpu
def test_calls_from_several_threads():
    ops = [operands(300 + i, 72, 136, 4, 16, seed=i) for i in range(4)]
    want = [(ti.low_rank_matmul(*o[:6]), *ti.low_rank_matmul_backward(o[6], *o[:6])) for o in ops]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = (ti.low_rank_matmul(*ops[i][:6]),
                       *ti.low_rank_matmul_backward(ops[i][6], *ops[i][:6]))
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


CAPTURES = """
import sys, torch
sys.path.insert(0, {root!r})
import tensor_inv_b200 as ti
def ones(*shape):
    return torch.ones(*shape, device="cuda").bfloat16()
X, W, A, B = ones(300, 64), ones(64, 64), ones(2, 64, 8), ones(2, 8, 64)
index = torch.zeros(300, dtype=torch.int64, device="cuda")
if {first}:  # the process's first calls are captured ones
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Y = ti.low_rank_matmul(X, W, A, B, index)
        y = ti.low_rank_matmul(X[:3], W, A, B, index[:3])
        grads = ti.low_rank_matmul_backward(X, X, W, A, B, index)
    graph.replay()
    assert (Y == 576).all() and (y == 576).all() and (grads[0] == 576).all()
else:  # a backward pass captured while an eager graph of the same leaves lives
    A.requires_grad_()
    kept = ti.low_rank_matmul(X, W, A, B, index)
    Y = ti.low_rank_matmul(X, W, A, B, index)
    kept.backward(torch.ones_like(Y), retain_graph=True)
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            Y.backward(torch.ones_like(Y))
        raise SystemExit("captured")
    except RuntimeError:
        pass
    assert (ti.low_rank_matmul(X, W, A, B, index) == 576).all()
torch.cuda.synchronize()
print("fine")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("first", [True, False])
def test_captures_in_a_process_of_their_own(first):
    code = CAPTURES.format(root=str(ROOT), first=first)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


# ---------------------------------------------------------------------------------------
# refusals (no GPU needed: arguments are checked before the device)
# ---------------------------------------------------------------------------------------
def cpu_operands(**kw):
    return operands(6, 16, 24, 3, 4, device="cpu", **kw)


def test_refused_arguments():
    X, W, A, B, index, scale, dY = cpu_operands()
    good = [X, W, A, B, index, scale]
    cases = [
        (TypeError, 0, X.float()), (TypeError, 1, W.half()), (TypeError, 2, A.double()),
        (TypeError, 0, [[1.0]]), (ValueError, 0, X[0]), (ValueError, 0, X[:, :8]),
        (ValueError, 1, W[:8]), (ValueError, 1, W[:, :8]), (ValueError, 2, A[:2]),
        (ValueError, 2, A[:, :8]), (ValueError, 2, A[:, :, :2]), (ValueError, 3, B[:, :, :8]),
        (ValueError, 2, A[0]), (ValueError, 4, index[:3]), (TypeError, 4, index.float()),
        (TypeError, 4, [0] * 6), (ValueError, 4, None), (TypeError, 5, scale.double()),
        (TypeError, 5, 2.0), (ValueError, 5, scale[:2]),
        (ValueError, 0, X),  # nothing wrong but the device
    ]
    for error, at, value in cases:
        args = list(good)
        args[at] = value
        with pytest.raises(error):
            ti.low_rank_matmul(*args)
        with pytest.raises(error):
            ti.low_rank_matmul_backward(dY, *args)
    with pytest.raises(TypeError):
        ti.low_rank_matmul(*good, alpha="1")
    with pytest.raises(ValueError, match="seed"):
        ti.low_rank_matmul(*good, p=0.5)
    with pytest.raises(ValueError, match="needs"):
        ti.low_rank_matmul_backward(dY, *good, needs=(True,))
    wide = torch.zeros(3, 16, 257, dtype=X.dtype), torch.zeros(3, 257, 24, dtype=X.dtype)
    with pytest.raises(ValueError, match="rank"):
        ti.low_rank_matmul(X, W, *wide, index, scale)
    with pytest.raises(ValueError, match="rank"):
        ti.low_rank_matmul(X, W, A[:, :, :0], B[:, :0], index, scale)


def test_refused_gradients():
    X, W, A, B, index, scale, _ = cpu_operands()
    for at in (1, 5):
        args = [X, W, A, B, index, scale]
        args[at] = args[at].clone().requires_grad_()
        with pytest.raises(ValueError, match="fixed"):
            ti.low_rank_matmul(*args)


@pytest.mark.gpu
def test_refused_gradient_operands():
    X, W, A, B, index, scale, dY = operands(6, 16, 24, 3, 4)
    P = torch.zeros(6, 4, device="cuda")
    for bad in (dict(dY=dY[:3]), dict(dY=dY[:, :8]), dict(dY=dY.cpu()), dict(P=P[:3]),
                dict(P=P.cpu())):
        with pytest.raises(ValueError):
            ti.low_rank_matmul_backward(bad.get("dY", dY), X, W, A, B, index, scale, P=bad.get("P"))
    for bad in (dict(dY=dY.float()), dict(P=P.double())):
        with pytest.raises(TypeError):
            ti.low_rank_matmul_backward(bad.get("dY", dY), X, W, A, B, index, scale, P=bad.get("P"))


def test_c_entry_statuses():
    """The C entry points refuse by status before they touch a device."""
    size = ctypes.c_size_t(0)

    def ask(**kw):
        op = nat.LowRank()
        for name, value in dict(dtype=1, t=4, k=8, n=8, s=2, r=4, index_bytes=8, **{}).items():
            setattr(op, name, value)
        cut = kw.pop("cut", 0)
        for name, value in kw.items():
            setattr(op, name, value)
        op.drop.cut = cut
        return nat.lib().ti_low_rank_workspace_size(ctypes.byref(op), ctypes.byref(size))

    assert ask() == nat.TI_OK and size.value > 0
    for bad in (dict(dtype=2), dict(dtype=-1), dict(t=-1), dict(k=-1), dict(n=-1), dict(s=0),
                dict(r=0), dict(cut=-1), dict(cut=65537), dict(index=64, index_bytes=2)):
        assert ask(**bad) == nat.TI_ERR_INVALID_ARGUMENT, bad
    for big in (dict(r=257), dict(t=2**31), dict(k=2**31), dict(n=2**31), dict(s=2**31)):
        assert ask(**big) == nat.TI_ERR_UNSUPPORTED, big
    assert nat.lib().ti_low_rank_workspace_size(None, ctypes.byref(size)) == \
        nat.TI_ERR_INVALID_ARGUMENT
    spec = nat.DropoutSpec(cut=70000)
    assert nat.lib().ti_dropout(1, None, 1, 1, None, 1, 1, 1, ctypes.byref(spec), None) == \
        nat.TI_ERR_INVALID_ARGUMENT
    spec = nat.DropoutSpec(cut=1)
    for args in ((4, 1, 1, 1), (-1, 1, 1, 1), (1, -1, 1, 1), (1, 1, -1, 1), (1, 1, 4, 3)):
        dtype, rows, cols, ld = args
        assert nat.lib().ti_dropout(dtype, None, 1, 1, None, ld, rows, cols, ctypes.byref(spec),
                                    None) == nat.TI_ERR_INVALID_ARGUMENT
