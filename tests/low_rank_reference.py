"""Plain float64 forms of the low-rank products and of dropout's mask, for the tests."""

import numpy as np
import torch


def philox_halves(rows, cols, seed, offset, row0=0):
    """The 16-bit numbers of a rows x cols matrix: Philox4x32-10 (Salmon et al. 2011)."""
    blocks = -(-cols // 8)
    u64 = np.uint64
    c = [np.broadcast_to(np.arange(blocks, dtype=np.uint32), (rows, blocks)),
         np.broadcast_to((row0 + np.arange(rows, dtype=np.uint64)).astype(np.uint32)[:, None],
                         (rows, blocks)),
         np.full((rows, blocks), offset % 2**32, np.uint32),
         np.full((rows, blocks), offset >> 32, np.uint32)]
    k0, k1 = seed % 2**32, seed >> 32
    for _ in range(10):
        a, b = c[0].astype(u64) * u64(0xD2511F53), c[2].astype(u64) * u64(0xCD9E8D57)
        c = [(b >> u64(32)).astype(np.uint32) ^ c[1] ^ np.uint32(k0), b.astype(np.uint32),
             (a >> u64(32)).astype(np.uint32) ^ c[3] ^ np.uint32(k1), a.astype(np.uint32)]
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    words = np.stack(c, axis=-1).astype("<u4")
    return words.reshape(rows, 4 * blocks).view("<u2")[:, :cols].astype(np.int64)


def mask(rows, cols, p, seed, offset):
    return torch.from_numpy(philox_halves(rows, cols, seed, offset) >= round(65536 * p))


def keep_factor(p):
    cut = round(65536 * p)
    return 65536 / (65536 - cut) if cut < 65536 else 0.0


def forward(X, W, A, B, index, scale, alpha=1.0, p=0.0, seed=0, offset=0, absolute=False):
    """(Y, P) in float64; absolute: of the operands' magnitudes, for error bounds."""
    X, W, A, B = (M.detach().double().cpu() for M in (X, W, A, B))
    if absolute:
        X, W, A, B = (M.abs() for M in (X, W, A, B))
        alpha = abs(alpha)
    T, (S, _, r) = X.shape[0], A.shape
    index = torch.zeros(T, dtype=torch.int64) if index is None else index.long().cpu()
    scale = torch.ones(S, dtype=torch.float64) if scale is None else scale.double().cpu()
    if absolute:
        scale = scale.abs()
    D = X if round(65536 * p) == 0 else \
        torch.where(mask(T, X.shape[1], p, seed, offset), X * keep_factor(p), 0.0)
    P = torch.zeros(T, r, dtype=torch.float64)
    Y = X @ W
    for s in range(S):
        t = torch.nonzero(index == s)[:, 0]
        P[t] = alpha * scale[s] * (D[t] @ A[s])
        Y[t] += P[t] @ B[s]
    return Y, P


def backward(dY, X, W, A, B, index, scale, alpha=1.0, p=0.0, seed=0, offset=0, absolute=False):
    """(dX, dA, dB) in float64."""
    dY, X, W, A, B = (M.detach().double().cpu() for M in (dY, X, W, A, B))
    if absolute:
        dY, X, W, A, B = (M.abs() for M in (dY, X, W, A, B))
        alpha = abs(alpha)
    T, S = X.shape[0], A.shape[0]
    index = torch.zeros(T, dtype=torch.int64) if index is None else index.long().cpu()
    scale = torch.ones(S, dtype=torch.float64) if scale is None else scale.double().cpu()
    if absolute:
        scale = scale.abs()
    kept, factor = torch.ones(X.shape, dtype=torch.bool), 1.0
    if round(65536 * p):
        kept, factor = mask(T, X.shape[1], p, seed, offset), keep_factor(p)
    D = torch.where(kept, X * factor, 0.0)
    dX, dA, dB = dY @ W.T, torch.zeros_like(A), torch.zeros_like(B)
    for s in range(S):
        t = torch.nonzero(index == s)[:, 0]
        dP = alpha * scale[s] * (dY[t] @ B[s].T)
        dX[t] += torch.where(kept[t], (dP @ A[s].T) * factor, 0.0)
        dA[s] = D[t].T @ dP
        dB[s] = (alpha * scale[s] * (D[t] @ A[s])).T @ dY[t]
    return dX, dA, dB


def half_step(dtype):
    return torch.finfo(dtype).eps / 2
