"""Cases of the low-rank products and of dropout, with their plain forms.

The operators:

* forward: ``Y[t] = X[t] W + scale[i] (M X)[t] A[i] B[i] / (1 - p)`` with ``i = index[t]`` (-1:
  the row takes no low-rank term) and M the dropout mask of a counter-based generator;
* backward: the gradients of X, A and B for a given dY (W is shared and fixed);
* dropout: ``M X / (1 - p)`` alone; on a gradient it is its own backward pass.

The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
as 1, 2, 3", 2011) with the seed as its key and the counter (column // 8, row, offset): the
element takes 16 of the block's 128 bits and is kept when they are at least round(65536 p).
"""

import functools

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _product(name, op, T, K, N, S, r, dtype, p, layout, rows, pad=0):
    return {"name": name, "op": op, "T": T, "K": K, "N": N, "S": S, "r": r, "dtype": dtype,
            "p": p, "layout": layout, "rows": rows, "pad": pad}


def _dropout(name, T, K, dtype, p, pad=0):
    return {"name": name, "op": "dropout", "T": T, "K": K, "dtype": dtype, "p": p, "pad": pad}


def listed():
    return [
        # one token of one request, the smallest call of serving
        _product("forward-1", "forward", 1, 4096, 4096, 8, 16, "bf16", 0.0, "outer", "mixed"),
        # one token each of many requests, each with an adapter of its own, some with none
        _product("forward-48", "forward", 48, 4096, 8192, 64, 16, "fp16", 0.0, "outer", "mixed"),
        # a small ragged prompt against odd sizes, in the layout of a factorization (U S, Vt)
        _product("forward-ragged", "forward", 333, 1001, 1500, 5, 7, "bf16", 0.0, "inner", "runs"),
        # prompts of several requests in one batch
        _product("forward-prompts", "forward", 4096, 4096, 4096, 16, 64, "bf16", 0.0, "outer",
                 "runs"),
        # the largest product: a full batch of long prompts
        _product("forward-large", "forward", 8192, 8192, 8192, 4, 32, "fp16", 0.0, "inner",
                 "runs"),
        # the forward pass of training one adapter with dropout on its input
        _product("forward-dropout", "forward", 2048, 4096, 4096, 1, 32, "bf16", 0.1, "outer",
                 "one"),
        # a training step's backward pass: one adapter, dropout
        _product("backward-one", "backward", 4096, 4096, 4096, 1, 16, "bf16", 0.1, "outer", "one"),
        # several adapters trained in one batch, odd sizes
        _product("backward-ragged", "backward", 1500, 2000, 1001, 6, 24, "fp16", 0.0, "inner",
                 "runs"),
        # a small step, where launches count
        _product("backward-small", "backward", 128, 1024, 1024, 2, 8, "bf16", 0.05, "outer",
                 "mixed"),
        # activations of one small step, rows cut out of a wider buffer
        _dropout("dropout-small", 48, 1001, "fp32", 0.5, pad=23),
        # hidden states of one batch
        _dropout("dropout", 4096, 4096, "fp16", 0.1),
        # the largest hidden states of a batch
        _dropout("dropout-large", 16384, 8192, "bf16", 0.1),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; one in three is odd, the others a multiple of 8."""
    n = int(round(low * (high / low) ** rng.random()))
    return max(low, n | 1) if rng.random() < 1 / 3 else max(low, n // 8 * 8, 1)


def draw(rng):
    op = rng.choice(["forward", "forward", "backward", "dropout"])
    dtype = rng.choice(["bf16", "fp16"])
    pad = rng.choice([0, 0, 8, 13])
    p = rng.choice([0.0, 0.0, round(0.02 + 0.5 * rng.random(), 3)])
    if op == "dropout":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "T": _size(rng, 1, 16384), "K": _size(rng, 64, 8192), "dtype": dtype,
                "p": p or 0.1, "pad": pad}
    T = _size(rng, 1 if op == "forward" else 16, 8192)
    S = rng.choice([1, 2, 5, 16, 64])
    r = rng.choice([1, 4, 8, 13, 16, 24, 32, 64, 128])
    if S * r > 2048:
        S = 2048 // r
    return {"op": op, "T": T, "K": _size(rng, 64, 8192), "N": _size(rng, 64, 8192), "S": S, "r": r,
            "dtype": dtype, "p": p if op == "backward" or T > 256 else 0.0,
            "layout": rng.choice(["outer", "inner"]),
            "rows": "one" if S == 1 else rng.choice(["mixed", "runs"]), "pad": pad}


def _index(case, generator):
    """Which adapter each row takes: ``one`` (every row the same), ``runs`` (requests of ragged
    lengths one after another) or ``mixed`` (each row its own); -1 for rows without one."""
    T, S = case["T"], case["S"]
    if case["rows"] == "one":
        return torch.zeros(T, dtype=torch.int64, device="cuda")
    if case["rows"] == "mixed":
        return torch.randint(-1, S, (T,), generator=generator, device="cuda") if T > 1 else \
            torch.randint(0, S, (T,), generator=generator, device="cuda")
    runs = min(T, S + 2)
    ends = torch.randint(0, T + 1, (runs - 1,), generator=generator, device="cuda").sort().values
    run = torch.searchsorted(ends, torch.arange(T, device="cuda"), right=True)
    return torch.randint(-1, S, (runs,), generator=generator, device="cuda")[run]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def rows_of(T, K, pad):
        # with a pad: the columns [0, K) of a wider buffer
        return torch.randn(T, K + pad, generator=generator, device="cuda").to(dtype)[:, :K]

    def matrix(rows, columns, std, batch=()):
        # "inner": rows x columns as the product reads them; "outer": stored transposed, as
        # checkpoints keep weights (outputs x inputs), and passed as a transposed view
        shape = (rows, columns) if case["layout"] == "inner" else (columns, rows)
        M = (std * torch.randn(*batch, *shape, generator=generator, device="cuda")).to(dtype)
        return M if case["layout"] == "inner" else M.transpose(-1, -2)

    T, K, p = case["T"], case["K"], case["p"]
    state = {"op": case["op"], "p": p, "seed": (seed * 0x9E3779B97F4A7C15 + 1) % 2 ** 63,
             "offset": seed % 1000, "X": rows_of(T, K, case["pad"])}
    if case["op"] == "dropout":
        return state
    N, S, r = case["N"], case["S"], case["r"]
    state["W"] = matrix(K, N, K ** -0.5)
    state["A"] = matrix(K, r, K ** -0.5, (S,))
    state["B"] = matrix(r, N, r ** -0.5, (S,))
    state["scale"] = 0.5 + torch.rand(S, generator=generator, device="cuda")
    state["index"] = _index(case, generator)
    if case["op"] == "backward":
        # the projection that the forward pass of a training step returns beside Y
        state["P"] = _projection(state)
        state["dY"] = rows_of(T, N, case["pad"])
    return state


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------
def _philox_round(words, key):
    c0, c1, c2, c3 = words
    low = 0xFFFFFFFF
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return ((b >> 32) & low) ^ c1 ^ key[0], b & low, ((a >> 32) & low) ^ c3 ^ key[1], a & low


def _kept(X, state):
    """The mask of the kept elements of X (rows x columns)."""
    T, K = X.shape
    seed, offset = state["seed"], state["offset"]
    keys = [((seed + i * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
            for i in range(10)]
    blocks = (K + 7) // 8
    column = torch.arange(blocks, device=X.device).expand(T, blocks)
    row = torch.arange(T, device=X.device)[:, None].expand(T, blocks)
    start = (column, row, torch.full_like(column, offset & 0xFFFFFFFF),
             torch.full_like(column, offset >> 32))
    words = torch.stack(functools.reduce(_philox_round, keys, start), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(T, 8 * blocks)[:, :K]
    return halves >= round(65536 * state["p"])


def _dropped(X, state):
    """M X / (1 - p) in 32 bits (X's own values when p is 0)."""
    X = X.float()
    if state["p"] == 0:
        return X
    dropped = round(65536 * state["p"])
    return torch.where(_kept(X, state), X * (65536 / (65536 - dropped)), 0.0)


def _chosen(state):
    """(T, S, 1): the scale of the row's adapter at that adapter, 0 elsewhere."""
    S = state["A"].shape[0]
    hit = state["index"][:, None] == torch.arange(S, device="cuda")
    return torch.where(hit, state["scale"], 0.0)[:, :, None]


def _columns(F):
    """(S, K, r) factors side by side as one (K, S r) matrix, in 32 bits."""
    S, K, r = F.shape
    return F.float().transpose(0, 1).reshape(K, S * r)


def _wide_projection(state, X):
    """scale X A of the row's adapter at that adapter's r columns, 0 at the others'."""
    S, _, r = state["A"].shape
    return ((X @ _columns(state["A"])).view(-1, S, r) * _chosen(state)).view(-1, S * r)


def _projection(state):
    S, _, r = state["A"].shape
    return _wide_projection(state, _dropped(state["X"], state)).view(-1, S, r).sum(1)


def _forward(state):
    B = state["B"].float()
    S, r, N = B.shape
    P = _wide_projection(state, _dropped(state["X"], state))
    return (state["X"].float() @ state["W"].float() + P @ B.reshape(S * r, N)).to(
        state["X"].dtype)


def _backward(state):
    dtype = state["X"].dtype
    dY, X, A, B = state["dY"].float(), _dropped(state["X"], state), state["A"], state["B"]
    S, K, r = A.shape
    hit = (state["index"][:, None] == torch.arange(S, device="cuda"))[:, :, None]
    P = torch.where(hit, state["P"][:, None, :], 0.0).view(-1, S * r)
    dP = ((dY @ _columns(B.transpose(1, 2))).view(-1, S, r) * _chosen(state)).view(-1, S * r)
    dX = dY @ state["W"].float().T + _dropped(dP @ _columns(A).T, state)
    dA = (X.T @ dP).view(K, S, r).transpose(0, 1)
    dB = (P.T @ dY).view(S, r, -1)
    return {"dX": dX.to(dtype), "dA": dA.to(dtype), "dB": dB.to(dtype)}


def run(state):
    if own:
        import tensor_inv_b200 as ti

        drop = {"p": state["p"], "seed": state["seed"], "offset": state["offset"]}
        if state["op"] == "dropout":
            return ti.dropout(state["X"], **drop)
        operands = [state[name] for name in ("X", "W", "A", "B", "index", "scale")]
        if state["op"] == "forward":
            return ti.low_rank_matmul(*operands, **drop)
        dX, dA, dB = ti.low_rank_matmul_backward(state["dY"], *operands, P=state["P"], **drop)
        return {"dX": dX, "dA": dA, "dB": dB}
    if state["op"] == "dropout":
        return _dropped(state["X"], state).to(state["X"].dtype)
    return _forward(state) if state["op"] == "forward" else _backward(state)


# ---------------------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    T, K = case["T"], case["K"]
    if case["op"] == "dropout":
        return {"bytes": 2 * size * T * K, "flops": T * K}
    N, r = case["N"], case["r"]
    adapters = size * min(T, case["S"]) * r * (K + N)
    matrices = size * (T * K + K * N + T * N) + 8 * T
    if case["op"] == "forward":
        return {"bytes": matrices + adapters, "flops": 2 * T * K * N + 2 * T * r * (K + N)}
    return {"bytes": matrices + size * T * K + 2 * adapters + 4 * T * r,
            "flops": 2 * T * K * N + 4 * T * r * (K + N)}


def _philox_reference(T, K, seed, offset):
    """The 16-bit numbers of a T x K matrix, with numpy's unsigned integers."""
    blocks = -(-K // 8)
    c = [np.tile(np.arange(blocks, dtype=np.uint32), (T, 1)),
         np.repeat(np.arange(T, dtype=np.uint32)[:, None], blocks, axis=1),
         np.full((T, blocks), offset % 2 ** 32, dtype=np.uint32),
         np.full((T, blocks), offset >> 32, dtype=np.uint32)]
    k0, k1 = seed % 2 ** 32, seed >> 32
    for _ in range(10):
        first = c[0].astype(np.uint64) * np.uint64(0xD2511F53)
        second = c[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
        c = [(second >> np.uint64(32)).astype(np.uint32) ^ c[1] ^ np.uint32(k0),
             second.astype(np.uint32),
             (first >> np.uint64(32)).astype(np.uint32) ^ c[3] ^ np.uint32(k1),
             first.astype(np.uint32)]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    words = np.ascontiguousarray(np.stack(c, axis=-1).astype("<u4"))
    return words.view("<u2").reshape(T, 8 * blocks)[:, :K]


def exact(case, seed):
    state = prepare(case, seed)
    T, K, p = case["T"], case["K"], case["p"]
    cut = int(round(65536 * p))
    keep = 1.0
    if cut:
        u = _philox_reference(T, K, state["seed"], state["offset"])
        keep = torch.from_numpy(np.where(u < cut, 0.0, 65536 / (65536 - cut))).cuda()
    X = state["X"].double()
    if case["op"] == "dropout":
        return X * keep
    index, scale = state["index"], state["scale"].double()
    W, A, B = state["W"].double(), state["A"].double(), state["B"].double()
    if case["op"] == "forward":
        Y = X @ W
        for s in range(case["S"]):
            t = torch.nonzero(index == s)[:, 0]
            Y[t] += scale[s] * ((X * keep)[t] @ A[s]) @ B[s]
        return Y
    dY = state["dY"].double()
    dX, dA, dB = torch.zeros_like(X), torch.zeros_like(A), torch.zeros_like(B)
    for s in range(case["S"]):
        t = torch.nonzero(index == s)[:, 0]
        dP = scale[s] * (dY[t] @ B[s].T)
        dX[t] = dP @ A[s].T
        dA[s] = (X * keep)[t].T @ dP
        dB[s] = state["P"][t].double().T @ dY[t]
    return {"dX": dX * keep + dY @ W.T, "dA": dA, "dB": dB}
