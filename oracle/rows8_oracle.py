"""CPU oracle of rows in 8 bits, in 64 bits, from the format's definition.

Blocks of 32 columns share 2^e, the smallest power of two at which the block's
largest finite magnitude is at most ``room`` (448 for e4m3, 127 for int8) times
it, e in [-127, 127], 0 for a block of zeros; values beside it are rounded to
nearest even to four significant bits, at least 2^-9 apart (e4m3), or to
integers (int8).  Values that are not finite become NaN.
"""

from __future__ import annotations

import numpy as np
import torch

ROOM = {"e4m3": 448.0, "int8": 127.0}


def _round_half_even(v: np.ndarray) -> np.ndarray:
    return np.rint(v)


def block_exponents(x: np.ndarray, fmt: str) -> np.ndarray:
    """e of every block of 32 columns of x [R, N] (float64): int [R, ceil(N / 32)]."""
    R, N = x.shape
    nb = -(-N // 32)
    v = np.zeros((R, nb * 32))
    v[:, :N] = np.where(np.isfinite(x), np.abs(x), 0.0)
    most = v.reshape(R, nb, 32).max(-1)
    e = np.zeros((R, nb), dtype=np.int64)
    for r, b in np.argwhere(most > 0):
        k = -160
        while most[r, b] > ROOM[fmt] * 2.0**k:
            k += 1
        e[r, b] = min(max(k, -127), 127)
    return e


def quantize(x: torch.Tensor, fmt: str):
    """x [R, N] -> (values that 8 bits hold, float64 numpy with NaN; scales uint8 [B, R, 16])."""
    v = x.double().numpy()
    R, N = v.shape
    e = block_exponents(v, fmt)
    unit = np.repeat(2.0 ** e.astype(np.float64), 32, axis=1)[:, :N]
    with np.errstate(invalid="ignore"):
        y = v / unit
    y = np.where(np.isfinite(v), y, np.nan)
    if fmt == "int8":
        q = _round_half_even(y)
    else:
        # spacing of four significant bits: 2^(floor(log2|y|) - 3), 2^-9 at least
        _, k = np.frexp(np.where(np.isfinite(y), y, 0.0))  # |y| = m 2^k, m in [0.5, 1)
        step = 2.0 ** np.maximum(k - 1 - 3, -9)
        q = _round_half_even(y / step) * step
    B = -(-N // 512)
    bytes_ = np.full((R, B * 16), 127, dtype=np.uint8)
    bytes_[:, : e.shape[1]] = (e + 127).astype(np.uint8)
    return q * unit, torch.from_numpy(np.ascontiguousarray(bytes_.reshape(R, B, 16).transpose(1, 0, 2)))


def values(codes: torch.Tensor, scales: torch.Tensor) -> np.ndarray:
    """What codes [R, N] with scales [B, R, 16] stand for, float64."""
    R, N = codes.shape
    e = scales.permute(1, 0, 2).reshape(R, -1).numpy().astype(np.int64) - 127
    unit = np.repeat(2.0 ** e.astype(np.float64), 32, axis=1)[:, :N]
    v = codes.double().numpy() if codes.dtype != torch.int8 else np.where(codes.numpy() == -128, np.nan, codes.double().numpy())
    return v * unit


def swiglu_backward(d_act: np.ndarray, gu: np.ndarray, w: np.ndarray):
    """(dG1, act_w, dw per row) in 64 bits; d_act [R, I], gu [R, 2I], w [R]."""
    I = d_act.shape[1]
    g, u = gu[:, :I], gu[:, I:]
    with np.errstate(over="ignore"):
        sig = 1.0 / (1.0 + np.exp(-g))
    s = g * sig
    d = d_act * w[:, None]
    dg1 = np.concatenate([d * u * (sig + s * (1 - sig)), d * s], axis=1)
    return dg1, w[:, None] * s * u, (d_act * s * u).sum(1)


def grouped_nt(a: np.ndarray, b: np.ndarray, offsets: np.ndarray):
    """(C, sum over blocks of 64 columns of the largest |product|), in 64 bits:
    a [M, K], b [G, N, K]."""
    M, K = a.shape
    N = b.shape[1]
    c, big = np.zeros((M, N)), np.zeros((M, N))
    for g in range(b.shape[0]):
        rows = slice(int(offsets[g]), int(offsets[g + 1]))
        if rows.stop <= rows.start:
            continue
        c[rows] = a[rows] @ b[g].T
        for k in range(0, K, 64):
            p = np.abs(a[rows, None, k : k + 64] * b[g][None, :, k : k + 64])
            big[rows] += p.max(-1)
    return c, big
