"""dropout: the mask against the generator's definition, values, refusals, gradient, capture."""

import numpy as np
import pytest
import torch

import low_rank_reference as ref
import tensor_inv_b200 as ti
from tensor_inv_b200.dropout import drop_numbers

SEED, OFFSET = 0x9E3779B97F4A7C15 - 2**63, 5_000_000_007


def test_reference_generator_known_answers():
    """The published test vectors of Philox4x32-10 (counter and key all zeros / all ones)."""
    zeros = ref.philox_halves(1, 8, 0, 0)[0]
    words = zeros[0::2] | zeros[1::2] << 16
    assert [int(w) for w in words] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("bad", [
    dict(p=-0.1, seed=1), dict(p=1.5, seed=1), dict(p=float("nan"), seed=1), dict(p="x", seed=1),
    dict(p=0.5), dict(p=0.5, seed=-1), dict(p=0.5, seed=2**64), dict(p=0.5, seed=1.5),
    dict(p=0.5, seed=1, offset=-1), dict(p=0.5, seed=1, offset=2**64),
    dict(p=0.5, seed=1, offset=0.5), dict(p=0.5, seed=torch.zeros(2, dtype=torch.int64)),
    dict(p=0.5, seed=torch.zeros(1, dtype=torch.int32)), dict(p=0.5, seed=1)])
def test_refusals(bad):
    """Bad arguments raise ValueError; the last one is good but for its CPU tensor."""
    for fn in (ti.dropout, ti.dropout_backward):
        with pytest.raises(ValueError):
            fn(torch.zeros(4, 4), **bad)


def test_refused_types():
    for X in (torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.complex64), [1.0]):
        with pytest.raises(TypeError):
            ti.dropout(X, 0.5, 1)
    with pytest.raises(ValueError, match="one dimension"):
        ti.dropout(torch.tensor(1.0), 0.5, 1)


def test_probability_steps():
    assert drop_numbers(0.5, 1, 0, torch.device("cpu"))[0] == 32768
    assert drop_numbers(1.0, 1, 0, torch.device("cpu"))[0] == 65536
    assert drop_numbers(2.0**-18, None, 0, torch.device("cpu"))[0] == 0


def want(X, p, seed=SEED, offset=OFFSET):
    flat = X.detach().cpu().reshape(-1, X.shape[-1])
    kept = ref.mask(*flat.shape, p, seed, offset)
    return torch.where(kept, flat.double() * ref.keep_factor(p), 0.0).reshape(X.shape), kept


def check(got, X, p, seed=SEED, offset=OFFSET):
    """fp32: the factor is rounded once and the product once: two half steps (their product
    below 2^-40); 16-bit types: that in fp32, then one half step of the type; fp64: two half
    steps.  Where the factor is exact (p = 1/2) the same bound holds with room."""
    exact, kept = want(X, p, seed, offset)
    u = ref.half_step(X.dtype)
    tol = {torch.float64: 2 * u, torch.float32: 2 * u}.get(X.dtype, u + 3 * 2.0**-24)
    got = got.cpu().double()
    # an exact value that rounds below the type's normal range is off by half a subnormal step
    tiny = torch.finfo(X.dtype).smallest_normal * u * 2
    assert ((got - exact).abs() <= tol * 1.0001 * exact.abs() + tiny).all()
    assert (got.reshape(kept.shape)[~kept] == 0).all()


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 9), (48, 1001), (2, 3, 65), (17,), (300, 512), (1, 4099)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("shape", SHAPES)
def test_values(shape, dtype):
    g = torch.Generator().manual_seed(1)
    X = torch.randn(shape, generator=g).to(dtype).cuda()
    for p in (0.1, 0.5, 0.93):
        check(ti.dropout(X, p, SEED, OFFSET), X, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
def test_strides_and_alignment(dtype):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(70, 333, generator=g).to(dtype).cuda()
    for X in (wide[:, :64], wide[:, 1:258], wide.T, wide[::3, ::2], wide[5:6], wide[:, 4:4],
              wide[3].expand(9, 333), wide[:, :320].reshape(70, 5, 64).transpose(0, 1)):
        Y = ti.dropout(X, 0.3, SEED, OFFSET)
        assert Y.shape == X.shape and Y.is_contiguous()
        if X.numel():
            check(Y, X, 0.3)


@pytest.mark.gpu
def test_ends_of_the_probability():
    X = torch.tensor([[1.5, float("nan"), float("inf"), -0.0, 2.0] * 7]).cuda()
    assert (ti.dropout(X, 1.0, 3) == 0).all()
    Y = ti.dropout(X, 0.0)
    assert torch.equal(Y.view(torch.int32), X.view(torch.int32)) and Y.data_ptr() != X.data_ptr()


@pytest.mark.gpu
def test_dropped_places_hold_zero_whatever_they_held():
    X = torch.full((64, 100), float("nan"), device="cuda", dtype=torch.bfloat16)
    kept = ref.mask(64, 100, 0.5, 9, 0)
    Y = ti.dropout(X, 0.5, 9).cpu()
    assert torch.isnan(Y[kept]).all() and (Y[~kept] == 0).all()


@pytest.mark.gpu
def test_one_mask_for_every_type_and_a_device_seed():
    X = torch.ones(33, 130, device="cuda")
    masks = [ti.dropout(X.to(t), 0.4, 77, 5) != 0 for t in
             (torch.float16, torch.bfloat16, torch.float32, torch.float64)]
    seed = torch.tensor([77], dtype=torch.int64, device="cuda")
    masks.append(ti.dropout(X, 0.4, seed, 5) != 0)
    assert all(torch.equal(m, masks[0]) for m in masks)
    assert not torch.equal(masks[0], ti.dropout(X, 0.4, 77, 6) != 0)
    assert not torch.equal(masks[0], ti.dropout(X, 0.4, 78, 5) != 0)


@pytest.mark.gpu
def test_share_of_kept_elements():
    """1e7 independent bits: the share is within 6 standard deviations of 1 - p."""
    Y = ti.dropout(torch.ones(1000, 10000, device="cuda", dtype=torch.float16), 0.1, 12)
    share = (Y != 0).double().mean().item()
    assert abs(share - (1 - round(6553.6) / 65536)) < 6 * np.sqrt(0.09 / 1e7)


@pytest.mark.gpu
def test_gradient():
    X = torch.randn(20, 50, device="cuda", dtype=torch.float64, requires_grad=True)
    dY = torch.randn(50, 20, device="cuda", dtype=torch.float64).T
    ti.dropout(X, 0.5, 4, 2).backward(dY)
    assert torch.equal(X.grad, ti.dropout_backward(dY, 0.5, 4, 2))
    # the map is linear: a difference quotient is exact up to rounding
    E = torch.randn_like(X.detach())
    with torch.no_grad():
        slope = (ti.dropout(X + E, 0.5, 4, 2) - ti.dropout(X, 0.5, 4, 2)).mul(dY).sum()
    terms = (E * X.grad).abs().sum() + (X.detach() * X.grad).abs().sum()
    assert (slope - (E * X.grad).sum()).abs() <= 1100 * 2.0**-52 * terms


@pytest.mark.gpu
def test_changed_seed_before_the_backward_pass_is_an_error():
    X = torch.randn(4, 4, device="cuda", requires_grad=True)
    seed = torch.tensor([7], device="cuda")
    Y = ti.dropout(X, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        Y.sum().backward()


@pytest.mark.gpu
def test_capture_reads_the_seed_at_replay_and_refuses_gradients():
    X = torch.randn(65, 77, device="cuda")
    seed = torch.tensor([1], device="cuda")
    leaf = X.clone().requires_grad_()
    ti.dropout(X, 0.5, seed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Y = ti.dropout(X, 0.5, seed)
        with pytest.raises(RuntimeError, match="capture"):
            ti.dropout(leaf, 0.5, 1)
    for s in (5, 6):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(Y, ti.dropout(X, 0.5, s))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows 2^31 + 8 elements apart (12 GB), and the last rows of a very tall matrix."""
    step = 2**31 + 8
    X = torch.empty(2 * step + 64, dtype=torch.float16, device="cuda").as_strided((3, 33), (step, 1))
    X.copy_(torch.randn(3, 33))
    check(ti.dropout(X, 0.25, SEED, OFFSET), X, 0.25)
    del X
    rows = 2**28 + 3
    X = torch.ones(rows, 9, dtype=torch.bfloat16, device="cuda")
    Y = ti.dropout(X, 0.5, 3)
    kept = torch.from_numpy(ref.philox_halves(5, 9, 3, 0, rows - 5) >= 32768)
    assert torch.equal(Y[-5:].cpu() != 0, kept)


@pytest.mark.gpu
def test_another_stream():
    X = torch.randn(500, 1000, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        Y = ti.dropout(X, 0.5, 8)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(Y, ti.dropout(X, 0.5, 8))
