"""Rows in 4 bits: weights, products, and the expert layer over 4-bit weights.

As rows in 8 bits (``rows8``), with e2m1 values, two to a byte: blocks of 32
neighbouring columns of a row share a power of two, and each value is 0, 0.5,
1, 1.5, 2, 3, 4 or 6 of it, with a sign (``Rows4``).  This is the microscaling
format of 4-bit checkpoints; only the order in which the exponents lie is this
library's.

* ``quantize_rows4`` / ``dequantize_rows4`` write such rows and read them back.
* ``group_gemm_nt_rows4`` multiplies ragged groups of rows, in 8 bits
  (``Rows8``, e4m3) or in 4, with one 4-bit weight matrix per group, on the
  matrix instruction that takes the codes and their powers of two (at four times
  the rate of bf16 where both are in 4 bits).
* ``expert_layer_rows4`` is the whole expert layer over weights kept in 4 bits
  (``Experts4``), for serving: half the weight bytes of ``expert_layer_rows8``.
  Tokens and activations are held in 8 bits as there.

Streams, checks and errors are those of ``rows8``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .kernels import HALF, _check_dev, _half, _ptr
from .rows8 import GROUP, Rows8, _e4m3, _empty, _indices, _launch, _serving_layer, scales_shape


@dataclass(frozen=True)
class Rows4:
    """Rows in 4 bits.

    codes: uint8 [..., R, ceil(N / 2)], column 2 j in the low half of byte j;
    bit 3 of a half is the sign, bits 2 and 1 the exponent, bit 0 the mantissa.
    scales: uint8 [..., ceil(N / 512), R, 16]; byte [b, r, j] is e + 127 of the
    power of two 2^e beside columns 512 b + 32 j .. + 31 of row r, 127 past the
    last column; 255 stands for NaN in all of them.
    columns: N.
    dtype: bfloat16 or float16, what the rows were and are read back as.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    columns: int
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.columns))

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> "Rows4":
        return Rows4(self.codes.to(device), self.scales.to(device), self.columns, self.dtype)


def _kind(name: str, q, *kinds: type) -> None:
    assert isinstance(q, kinds), f"{name} must be {' or '.join(k.__name__ for k in kinds)}, got {type(q).__name__}"


def _rows4(name: str, q: Rows4, dims: int, like: torch.dtype | None = None) -> torch.dtype:
    """Check an operand's parts against each other; returns its dtype."""
    _kind(name, q, Rows4)
    assert q.codes.dtype == torch.uint8, f"{name} codes must be uint8, got {q.codes.dtype}"
    assert q.dtype in HALF, f"{name} must stand for bfloat16 or float16 rows, got {q.dtype}"
    assert like is None or q.dtype == like, f"{name} must stand for {like} like the other operands, got {q.dtype}"
    assert q.scales.dtype == torch.uint8, f"{name} scales must be uint8, got {q.scales.dtype}"
    assert q.codes.dim() == dims, f"{name} must have {dims} dimensions, got {q.codes.dim()}"
    assert q.codes.shape[-1] == (q.columns + 1) // 2, f"{name} codes of {q.columns} columns must be {(q.columns + 1) // 2} wide, got {q.codes.shape[-1]}"
    assert q.scales.shape == scales_shape(q.shape), f"{name} scales must be {scales_shape(q.shape)}, got {tuple(q.scales.shape)}"
    assert q.codes.is_contiguous() and q.scales.is_contiguous(), f"{name} must be contiguous"
    return q.dtype


def quantize_rows4(x: torch.Tensor) -> Rows4:
    """x [R, N] or [G, R, N] (bfloat16 or float16) in 4 bits.

    Each block of 32 columns takes the smallest power of two 2^e at which its
    largest magnitude is below 7 * 2^e, and every value is rounded to the
    nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 beside it (ties to the even code): to
    within 2^-2 of itself, down to 2^e.  A block with a value that is not finite
    becomes NaN as a whole.

    The rows of a 2-D x may lie apart (stride(0) >= N); nothing needs to be aligned.
    """
    dev = _check_dev(x)
    assert x.dtype in HALF, f"x must be bfloat16 or float16, got {x.dtype}"
    assert x.dim() in (2, 3), f"x must be [R, N] or [G, R, N], got {tuple(x.shape)}"
    *lead, R, N = x.shape
    G, ld = (lead[0] if lead else 1), N
    if not x.is_contiguous():
        assert not lead and (N <= 1 or x.stride(1) == 1) and (R <= 1 or x.stride(0) >= N), (
            "columns must be contiguous and the rows of a 2-D x apart"
        )
        ld = max(N, x.stride(0))
    q = Rows4(x.new_empty((*lead, R, (N + 1) // 2), dtype=torch.uint8),
              x.new_empty((*lead, -(-N // GROUP), R, 16), dtype=torch.uint8), N, x.dtype)
    _launch("pmx_rows4_quantize", x.dtype, dev, _ptr(x), ld, R * N, G, R, N, _ptr(q.codes), _ptr(q.scales))
    return q


def dequantize_rows4(q: Rows4) -> torch.Tensor:
    """The rows of q [R, N] or [G, R, N], as its dtype.  Exact (values beyond
    the type's range become its largest finite one)."""
    dims = q.codes.dim() if isinstance(q, Rows4) and q.codes.dim() == 3 else 2
    dt = _rows4("q", q, dims)
    dev = _check_dev(q.codes, q.scales)
    *lead, R, N = q.shape
    out = q.codes.new_empty((*lead, R, N), dtype=dt)
    _launch("pmx_rows4_dequantize", dt, dev, _ptr(q.codes), _ptr(q.scales), lead[0] if lead else 1, R, N, _ptr(out))
    return out


def group_gemm_nt_rows4(a: Rows8 | Rows4, b: Rows4, offsets: torch.Tensor) -> torch.Tensor:
    """C[rows of g] = a[rows of g] @ b[g]^T, rounded once to the operands'
    dtype: a [M, K] in 4 bits or in e4m3, b [G, N, K] in 4 bits; rows of g:
    offsets[g] .. offsets[g+1]-1 (int32 [G + 1], ascending; rows that no group
    has are not written).  K a multiple of 32, N of 8.

    With both in 4 bits sums are good to fp32.  With a in 8 bits, as in
    ``group_gemm_nt_rows8``: off by less than 7 * 2^-13 of the largest product
    of each eight neighbouring columns.
    """
    _kind("a", a, Rows8, Rows4), _kind("b", b, Rows4)
    _check_dev(a.codes, a.scales, b.codes, b.scales, offsets)
    dev = offsets.device
    bits = 4 if isinstance(a, Rows4) else 8
    dt = _rows4("a", a, 2) if bits == 4 else _e4m3("a", a, 2)
    _rows4("b", b, 3, dt)
    G, N, K = b.shape
    M = a.shape[0]
    assert a.shape[1] == K, "a and b disagree on K"
    _indices("offsets", offsets, G + 1)
    c = torch.empty((M, N), dtype=dt, device=dev)
    _launch("pmx_rows4_group_gemm_nt", dt, dev, _ptr(a.codes), _ptr(a.scales), bits, _ptr(b.codes), _ptr(b.scales),
            _ptr(offsets), G, M, N, K, _ptr(c))
    return c


def gemm_fc1_swiglu_rows4(x: Rows8, w: Rows4, offsets: torch.Tensor, row_token: torch.Tensor | None = None,
                          row_w: torch.Tensor | None = None) -> Rows8:
    """act[r] = silu(gate) * up * row_w[r], in e4m3 again, with (gate | up) =
    x[row_token[r]] @ w[g]^T: x [T, H] in e4m3, w [G, 2I, H] in 4 bits (gate rows
    first); row_token int32 [A] (None: row r is x[r]), row_w [A] (None: ones).
    fp32 up to the rounding to 8 bits (2^128, to which 4 bits round the topmost
    eighth of bfloat16's range and 8 bits its topmost 3%, counts as infinite).
    H a multiple of 32, I of 16."""
    _kind("x", x, Rows8), _kind("w", w, Rows4)
    dev = _check_dev(x.codes, x.scales, w.codes, w.scales, offsets, row_token, row_w)
    dt = _e4m3("x", x, 2)
    _rows4("w", w, 3, dt)
    G, I2, H = w.shape
    T = x.shape[0]
    assert x.shape[1] == H, "x and w disagree on the hidden size"
    assert I2 % 2 == 0, "w must hold as many gate as up rows"
    _indices("offsets", offsets, G + 1)
    A = T
    if row_token is not None:
        _indices("row_token", row_token)
        A = row_token.numel()
    if row_w is not None:
        _half("row weights", row_w, dt)
        assert row_w.numel() == A, "one weight per row"
    act = _empty((A, I2 // 2), torch.float8_e4m3fn, dt, dev)
    _launch("pmx_rows4_gemm_fc1_swiglu", dt, dev, _ptr(x.codes), _ptr(x.scales), T, _ptr(row_token), _ptr(w.codes),
            _ptr(w.scales), _ptr(offsets), G, A, H, I2 // 2, _ptr(row_w), _ptr(act.codes), _ptr(act.scales))
    return act


@dataclass(frozen=True)
class Experts4:
    """The weights of a layer's physical copies in 4 bits: gate_up [C, 2I, H]
    (gate rows first) and down [C, H, I]."""

    gate_up: Rows4
    down: Rows4

    @classmethod
    def quantize(cls, gate_up: torch.Tensor, down: torch.Tensor) -> "Experts4":
        """From merged 16-bit weights, once, when they are loaded."""
        C, H, I = down.shape
        assert tuple(gate_up.shape) == (C, 2 * I, H), (
            f"gate_up shape {tuple(gate_up.shape)} does not match down {tuple(down.shape)} (expected {(C, 2 * I, H)})"
        )
        assert gate_up.dtype == down.dtype, "gate_up and down must have one dtype"
        return cls(quantize_rows4(gate_up.detach()), quantize_rows4(down.detach()))


def expert_layer_rows4(hidden: torch.Tensor, routing_weights: torch.Tensor, selected_experts: torch.Tensor,
                       weights: Experts4, mapping: torch.Tensor | None = None, sources: torch.Tensor | None = None,
                       source: int = 0, recorder=None) -> torch.Tensor:
    """The full layer on one GPU over weights in 4 bits: [T, H] -> [T, H], forward only.

    The arguments are those of ``expert_layer``; ``weights`` from
    ``Experts4.quantize``.  The steps and what is held between them are those of
    ``expert_layer_rows8``.  H and I multiples of 32.
    """
    _kind("weights", weights, Experts4), _kind("gate_up", weights.gate_up, Rows4), _kind("down", weights.down, Rows4)
    return _serving_layer("expert_layer_rows4", "pmx_rows4_layer", 32, _rows4, hidden, routing_weights, selected_experts, weights,
                          mapping, sources, source, recorder)
