"""CPU oracle of rows in 4 bits, in 64 bits, from the format's definition.

Blocks of 32 columns share 2^e, the smallest power of two with the block's
largest magnitude below 7 * 2^e, e in [-127, 127], 0 for a block of zeros;
values beside it are rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives, ties to the even code.  A block that holds a value that is not
finite is NaN.
"""

from __future__ import annotations

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _blocks(v: np.ndarray) -> np.ndarray:
    """[R, N] -> [R, ceil(N / 32), 32], zeros past the last column."""
    R, N = v.shape
    out = np.zeros((R, -(-N // 32) * 32))
    out[:, :N] = v
    return out.reshape(R, -1, 32)


def quantize(x: torch.Tensor):
    """x [R, N] -> (values that 4 bits hold, float64 numpy with NaN; scales uint8 [B, R, 16])."""
    v = _blocks(x.double().numpy())
    R, nb, _ = v.shape
    N = x.shape[1]
    bad = ~np.isfinite(v).all(-1)
    most = np.abs(np.where(bad[..., None], 0.0, v)).max(-1)
    e = np.zeros((R, nb), dtype=np.int64)
    for r, b in np.argwhere(most > 0):
        k = -160
        while most[r, b] >= 7 * 2.0**k:
            k += 1
        e[r, b] = min(max(k, -127), 127)
    unit = 2.0 ** e[..., None].astype(np.float64)
    y = np.where(bad[..., None], 0.0, v) / unit
    far = np.abs(np.abs(y)[..., None] - LEVELS)
    # the nearest level; of two as near the one of the even code
    code = np.array([0, 2, 4, 6, 1, 3, 5, 7])[far[..., [0, 2, 4, 6, 1, 3, 5, 7]].argmin(-1)]
    q = np.where(bad[..., None], np.nan, np.copysign(LEVELS[code], y) * unit).reshape(R, -1)[:, :N]
    B = -(-N // 512)
    bytes_ = np.full((R, B * 16), 127, dtype=np.uint8)
    bytes_[:, :nb] = np.where(bad, 255, e + 127)
    return q, torch.from_numpy(np.ascontiguousarray(bytes_.reshape(R, B, 16).transpose(1, 0, 2)))


def values(codes: torch.Tensor, scales: torch.Tensor, N: int) -> np.ndarray:
    """What codes [R, ceil(N / 2)] with scales [B, R, 16] stand for, float64."""
    R = codes.shape[0]
    c = codes.numpy()
    half = np.stack([c & 15, c >> 4], -1).reshape(R, -1)[:, :N]
    byte = np.repeat(scales.permute(1, 0, 2).reshape(R, -1).numpy().astype(np.int64), 32, axis=1)[:, :N]
    v = LEVELS[half & 7] * np.where(half & 8, -1.0, 1.0) * 2.0 ** (byte - 127).astype(np.float64)
    return np.where(byte == 255, np.nan, v)
