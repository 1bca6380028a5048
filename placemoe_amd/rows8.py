"""Rows in 8 bits: activation checkpoints, and the expert layer over 8-bit weights.

Blocks of 32 neighbouring columns of a row share a power of two, and each
value is held beside it as an e4m3 float or an int8 (``Rows8``).  Two things
are built on it:

* **Activation checkpoints.**  ``quantize_rows`` writes one in the forward;
  the backward reads it with ``dequantize_rows`` (in order, or spread to the
  rows of the expert copies) and ``swiglu_bwd_rows8`` (the SwiGLU backward from
  8-bit gate and up rows).  ``expert_layer(activation_checkpoint=...)`` and
  ``set_activation_checkpoint`` use them.
* **Products.**  ``group_gemm_nt_rows8`` multiplies ragged row groups with one
  8-bit weight matrix per group; ``expert_layer_rows8`` is the whole expert
  layer over weights kept in 8 bits (``Experts8``), for serving: half the
  weight bytes of bf16, and twice its matrix rate in fc2 (fc1, whose results are
  rounded to 8 bits, multiplies exactly, at the rate of bf16).

Every function enqueues gfx950 kernels on the current stream of its tensors'
device and waits for nothing.  Wrong devices, dtypes and shapes raise
``AssertionError``, limits of the kernels ``ValueError``, both before anything
is launched; there is no CPU fallback.  Results do not depend on the other
rows of a call, nor on the slot that holds a copy.
"""

from __future__ import annotations

import contextlib
from dataclasses import dataclass

import torch

from . import _capi, kernels
from .kernels import HALF, _check_dev, _half, _ptr, _stream, _sym

FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_FORMAT_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}
BLOCK = 32  # columns that share a power of two
GROUP = 512  # columns whose 16 exponent bytes lie together


def _format(fmt: str) -> torch.dtype:
    if fmt not in FORMATS:
        raise ValueError(f"8-bit format must be one of {sorted(FORMATS)}, got {fmt!r}")
    return FORMATS[fmt]


@dataclass(frozen=True)
class Rows8:
    """Rows in 8 bits.

    codes: [..., R, N] ``float8_e4m3fn`` or ``int8`` (-128 stands for NaN).
    scales: uint8 [..., ceil(N / 512), R, 16]; byte [b, r, j] is e + 127 of the
    power of two 2^e beside columns 512 b + 32 j .. + 31 of row r.
    dtype: bfloat16 or float16, what the rows were and are read back as.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> "Rows8":
        return Rows8(self.codes.to(device), self.scales.to(device), self.dtype)


def scales_shape(shape) -> tuple:
    """The shape of the exponent bytes of rows of the given shape."""
    *lead, R, N = shape
    return (*lead, -(-N // GROUP), R, 16)


def _rows8(name: str, q: Rows8, dims: int) -> torch.dtype:
    """Check an operand's parts against each other; returns its dtype."""
    assert isinstance(q, Rows8), f"{name} must be Rows8, got {type(q).__name__}"
    assert q.codes.dtype in _FORMAT_CODES, f"{name} codes must be float8_e4m3fn or int8, got {q.codes.dtype}"
    assert q.dtype in HALF, f"{name} must stand for bfloat16 or float16 rows, got {q.dtype}"
    assert q.scales.dtype == torch.uint8, f"{name} scales must be uint8, got {q.scales.dtype}"
    assert q.codes.dim() == dims, f"{name} must have {dims} dimensions, got {q.codes.dim()}"
    assert q.scales.shape == scales_shape(q.codes.shape), (
        f"{name} scales must be {scales_shape(q.codes.shape)}, got {tuple(q.scales.shape)}"
    )
    assert q.codes.is_contiguous() and q.scales.is_contiguous(), f"{name} must be contiguous"
    return q.dtype


def _e4m3(name: str, q: Rows8, dims: int, like: torch.dtype | None = None) -> torch.dtype:
    dt = _rows8(name, q, dims)
    assert q.codes.dtype == torch.float8_e4m3fn, f"{name} must be e4m3 for a product, got {q.codes.dtype}"
    assert like is None or dt == like, f"{name} must stand for {like} like the other operands, got {dt}"
    return dt


def _indices(name: str, t: torch.Tensor, numel: int | None = None) -> None:
    assert t.dtype == torch.int32 and t.is_contiguous(), f"{name} must be contiguous int32"
    assert numel is None or t.numel() == numel, f"{name} must have {numel} entries, got {t.numel()}"


def _on(dev: torch.device):
    """The launch device: a kernel starts on the current one, whatever its stream."""
    return contextlib.nullcontext() if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _launch(name: str, dtype: torch.dtype, dev: torch.device, *args) -> None:
    if dev.index == torch._C._cuda_getDevice():
        _capi.call(_sym(name, dtype), *args, _stream(dev))
        return
    with torch.cuda.device(dev):
        _capi.call(_sym(name, dtype), *args, _stream(dev))


def _empty(shape, fmt: torch.dtype, dtype: torch.dtype, dev: torch.device) -> Rows8:
    *lead, R, N = shape
    return Rows8(torch.empty(shape, dtype=fmt, device=dev),
                 torch.empty((*lead, -(-N // GROUP), R, 16), dtype=torch.uint8, device=dev), dtype)


# ---------------------------------------------------------------------------
# Activation checkpoints
# ---------------------------------------------------------------------------


def quantize_rows(x: torch.Tensor, fmt: str = "e4m3") -> Rows8:
    """x [R, N] or [G, R, N] (bfloat16 or float16) in 8 bits.

    Each block of 32 columns takes the smallest power of two 2^e at which its
    largest finite magnitude is at most 448 (e4m3) or 127 (int8) times 2^e, and
    every value is rounded to nearest even beside it: to within 2^-4 of itself
    (e4m3, down to 2^-6 times 2^e) or 2^-1 times 2^e (int8, about 4 times as exact for
    blocks without an outlier).  Infinities and NaN become NaN.

    The rows of a 2-D x may lie apart (stride(0) >= N); nothing needs to be aligned.
    """
    dev = _check_dev(x)
    code = _format(fmt)
    assert x.dtype in HALF, f"x must be bfloat16 or float16, got {x.dtype}"
    assert x.dim() in (2, 3), f"x must be [R, N] or [G, R, N], got {tuple(x.shape)}"
    *lead, R, N = x.shape
    G, ld = (lead[0] if lead else 1), N
    if not x.is_contiguous():
        assert not lead and (N <= 1 or x.stride(1) == 1) and (R <= 1 or x.stride(0) >= N), (
            "columns must be contiguous and the rows of a 2-D x apart"
        )
        ld = max(N, x.stride(0))
    # (the cheapest allocations: a small call's time is the host's)
    q = Rows8(torch.empty_like(x, dtype=code) if ld == N else x.new_empty((R, N), dtype=code),
              x.new_empty((*lead, -(-N // GROUP), R, 16), dtype=torch.uint8), x.dtype)
    _launch("pmx_rows8_quantize", x.dtype, dev, _ptr(x), ld, R * N, G, R, N, _FORMAT_CODES[code], _ptr(q.codes),
            _ptr(q.scales))
    return q


def dequantize_rows(q: Rows8, pos: torch.Tensor | None = None) -> torch.Tensor:
    """The rows of q [R, N], as its dtype: [R, N], or with ``pos`` (int32
    [R, K], a permutation of 0 .. R*K-1 such as a routing's) row r at each
    pos[r, k] of [R*K, N].  Exact (values beyond float16's range become its
    largest finite one)."""
    dev = _check_dev(q.codes, q.scales, pos)
    dt = _rows8("q", q, 2)
    R, N = q.codes.shape
    K = 0
    if pos is not None:
        assert pos.dim() == 2 and pos.shape[0] == R and pos.shape[1] > 0, "pos must be [rows, K]"
        _indices("pos", pos)
        K = pos.shape[1]
    out = torch.empty((R * max(K, 1), N), dtype=dt, device=dev)
    _launch("pmx_rows8_dequantize", dt, dev, _ptr(q.codes), _ptr(q.scales), _ptr(pos), R, K, N,
            _FORMAT_CODES[q.codes.dtype], _ptr(out))
    return out


def swiglu_bwd_rows8(d_act: torch.Tensor, gu: Rows8, row_w: torch.Tensor | None = None,
                     row_src: torch.Tensor | None = None, num_assign: int | None = None):
    """SwiGLU backward from gate and up rows in 8 bits -> (dG1, act_w, dw).

    d_act [R, I]: the gradient of the weighted activations act_w = row_w * silu(gate) * up,
    gu [R, 2I] (gate columns, then up columns), row_w [R] (None: ones).
    dG1 [R, 2I] is the gradient of (gate | up), act_w [R, I] the activations
    themselves (for the weight gradient of fc2), and with ``row_src`` (int32 [R], no
    entry twice) dw [num_assign] the weights' gradient, dw[row_src[r]] = sum_j d_act * silu(gate) * up
    (entries that no row names are not written; None without ``row_src``).
    Computed in fp32, each result rounded once.
    """
    dev = _check_dev(d_act, gu.codes, gu.scales, row_w, row_src)
    dt = _half("d_act", d_act)
    assert _rows8("gu", gu, 2) == dt, f"gu must stand for {dt} rows like d_act, got {gu.dtype}"
    assert d_act.dim() == 2, "d_act must be [R, I]"
    R, I = d_act.shape
    assert tuple(gu.shape) == (R, 2 * I), f"gu must be {(R, 2 * I)}, got {tuple(gu.shape)}"
    if row_w is not None:
        _half("row weights", row_w, dt)
        assert row_w.numel() == R, "one weight per row"
    dw = None
    if row_src is not None:
        assert row_w is not None, "row_src names the rows' weights: row_w is needed"
        _indices("row_src", row_src, R)
        num_assign = R if num_assign is None else int(num_assign)
        dw = d_act.new_empty(num_assign)
        if I == 0:
            dw.zero_()
    dg1, act_w = d_act.new_empty((R, 2 * I)), torch.empty_like(d_act)
    _launch("pmx_rows8_swiglu_bwd", dt, dev, _ptr(d_act), _ptr(gu.codes), _ptr(gu.scales), _ptr(row_w), _ptr(row_src),
            R, I, dw.numel() if dw is not None else 0, _FORMAT_CODES[gu.codes.dtype], _ptr(dg1), _ptr(act_w), _ptr(dw))
    return dg1, act_w, dw


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------


def group_gemm_nt_rows8(a: Rows8, b: Rows8, offsets: torch.Tensor) -> torch.Tensor:
    """C[rows of g] = a[rows of g] @ b[g]^T, rounded once to the operands'
    dtype: a [M, K], b [G, N, K], both e4m3; rows of g: offsets[g] .. offsets[g+1]-1
    (int32 [G + 1], ascending; rows that no group has are not written).  K a
    multiple of 16, N of 8.

    The 8-bit matrix instruction adds products in eights of neighbouring columns,
    each cut below 2^-13 of the largest of its eight, and the eights in fp32: a sum is off
    by less than 7 * 2^-13 of the largest product of each eight, of random
    values by 1.5e-5 of itself (bf16's half step: 2^-9 to 2^-8, fp16's: 2^-12 to 2^-11)."""
    dev = _check_dev(a.codes, a.scales, b.codes, b.scales, offsets)
    dt = _e4m3("a", a, 2)
    _e4m3("b", b, 3, dt)
    G, N, K = b.shape
    M = a.shape[0]
    assert a.shape[1] == K, "a and b disagree on K"
    _indices("offsets", offsets, G + 1)
    c = torch.empty((M, N), dtype=dt, device=dev)
    _launch("pmx_rows8_group_gemm_nt", dt, dev, _ptr(a.codes), _ptr(a.scales), _ptr(b.codes), _ptr(b.scales), _ptr(offsets),
            G, M, N, K, _ptr(c))
    return c


def gemm_fc1_swiglu_rows8(x: Rows8, w: Rows8, offsets: torch.Tensor, row_token: torch.Tensor | None = None,
                          row_w: torch.Tensor | None = None) -> Rows8:
    """act[r] = silu(gate) * up * row_w[r], in 8 bits again, with (gate | up) =
    x[row_token[r]] @ w[g]^T: x [T, H], w [G, 2I, H] (gate rows first), both e4m3;
    row_token int32 [A] (None: row r is x[r]), row_w [A] (None: ones).  fp32
    up to the rounding to 8 bits (2^128, to which 8 bits round the topmost 3% of
    bfloat16's range, counts as infinite).  H and I multiples of 16."""
    dev = _check_dev(x.codes, x.scales, w.codes, w.scales, offsets, row_token, row_w)
    dt = _e4m3("x", x, 2)
    _e4m3("w", w, 3, dt)
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
    _launch("pmx_rows8_gemm_fc1_swiglu", dt, dev, _ptr(x.codes), _ptr(x.scales), T, _ptr(row_token), _ptr(w.codes),
            _ptr(w.scales), _ptr(offsets), G, A, H, I2 // 2, _ptr(row_w), _ptr(act.codes), _ptr(act.scales))
    return act


def quantize_rows_routed(x: torch.Tensor, pos: torch.Tensor, w: torch.Tensor):
    """(x [T, H] in e4m3, row_token [T*K], row_w [T*K]): token and weight of each
    row of the copies, row_token[pos[t, k]] = t and row_w[pos[t, k]] = w[t, k]."""
    dev = _check_dev(x, pos, w)
    dt = _half("x", x)
    _half("routing weights", w, dt)
    T, H = x.shape
    K = pos.shape[1]
    _indices("pos", pos, T * K)
    assert w.numel() == T * K, "routing weights: one per (token, k)"
    q = _empty((T, H), torch.float8_e4m3fn, dt, dev)
    row_token = torch.empty(T * K, dtype=torch.int32, device=dev)
    row_w = torch.empty(T * K, dtype=dt, device=dev)
    _launch("pmx_rows8_quantize_routed", dt, dev, _ptr(x), _ptr(pos), _ptr(w), T, K, H, _ptr(q.codes), _ptr(q.scales),
            _ptr(row_token), _ptr(row_w))
    return q, row_token, row_w


@dataclass(frozen=True)
class Experts8:
    """The weights of a layer's physical copies in e4m3: gate_up [C, 2I, H] (gate
    rows first) and down [C, H, I]."""

    gate_up: Rows8
    down: Rows8

    @classmethod
    def quantize(cls, gate_up: torch.Tensor, down: torch.Tensor) -> "Experts8":
        """From merged 16-bit weights, once, when they are loaded."""
        C, H, I = down.shape
        assert tuple(gate_up.shape) == (C, 2 * I, H), (
            f"gate_up shape {tuple(gate_up.shape)} does not match down {tuple(down.shape)} (expected {(C, 2 * I, H)})"
        )
        assert gate_up.dtype == down.dtype, "gate_up and down must have one dtype"
        return cls(quantize_rows(gate_up.detach()), quantize_rows(down.detach()))


def expert_layer_rows8(hidden: torch.Tensor, routing_weights: torch.Tensor, selected_experts: torch.Tensor,
                       weights: Experts8, mapping: torch.Tensor | None = None, sources: torch.Tensor | None = None,
                       source: int = 0, recorder=None) -> torch.Tensor:
    """The full layer on one GPU over weights in 8 bits: [T, H] -> [T, H], forward only.

    The arguments are those of ``expert_layer``; ``weights`` from
    ``Experts8.quantize``.  Tokens are quantised once, fc1 reads each where it
    lies for every copy that it is routed to, and the activations, weighted by
    the router, leave its epilogue in 8 bits for fc2 (router weights on the fc2
    input, as in the non-EP arithmetic); a token's rows, held in 24 bits (each value to
    2^-16 of itself), are then summed and rounded once.  H and I multiples of 16.
    """
    assert isinstance(weights, Experts8), f"weights must be Experts8, got {type(weights).__name__}"
    return _serving_layer("expert_layer_rows8", "pmx_rows8_layer", 16, _e4m3, hidden, routing_weights, selected_experts, weights,
                          mapping, sources, source, recorder)


def _serving_layer(name: str, entry: str, multiple: int, check_weights, hidden: torch.Tensor, routing_weights: torch.Tensor,
                   selected_experts: torch.Tensor, weights, mapping: torch.Tensor | None, sources: torch.Tensor | None,
                   source: int, recorder) -> torch.Tensor:
    """The layer ``name`` over weights in 8 or 4 bits; ``check_weights`` looks one matrix over, ``entry`` is the C-ABI's call."""
    from . import experts  # experts itself uses this module's checkpoints

    if torch.is_grad_enabled() and (hidden.requires_grad or routing_weights.requires_grad):
        raise ValueError(f"{name} has no backward; call it under torch.no_grad()")
    _check_dev(hidden, routing_weights, selected_experts, weights.gate_up.codes, weights.gate_up.scales, weights.down.codes,
               weights.down.scales, mapping, sources)
    dt = _half("hidden states", hidden)
    _half("routing weights", routing_weights, dt)
    assert hidden.dim() == 2, "hidden states must be [tokens, hidden size]"
    check_weights("gate_up", weights.gate_up, 3, dt)
    check_weights("down", weights.down, 3, dt)
    C, H, I = weights.down.shape
    assert tuple(weights.gate_up.shape) == (C, 2 * I, H), "gate_up and down describe different layers"
    T = hidden.shape[0]
    assert hidden.shape[1] == H, f"hidden size {hidden.shape[1]} != down's hidden size {H}"
    sel = selected_experts if selected_experts.dim() == 2 else selected_experts.reshape(-1, 1)
    assert sel.shape[0] == T and routing_weights.numel() == sel.numel(), "one expert and one weight per (token, k)"
    sel = sel.to(torch.int64).contiguous()
    K = sel.shape[1]
    if mapping is not None:
        mapping = mapping.to(torch.int64).contiguous()
        assert mapping.dim() == 2, "mapping must be [num_sources, num_experts]"
        S, E = mapping.shape
    else:
        S, E = 1, C
    if sources is not None:
        assert mapping is not None, "per-token sources need a mapping table"
        sources = sources.to(torch.int64).contiguous().reshape(-1)
        assert sources.numel() == T, "sources must have one entry per token"
    if T == 0 or K == 0:
        if recorder is not None:
            recorder(torch.zeros(C, dtype=torch.int32, device=hidden.device))
        return torch.zeros_like(hidden)
    ws_bytes = getattr(_capi.load(), entry + "_workspace_bytes")(T, K, H, I, C)
    if ws_bytes == 0:
        raise ValueError(f"{name}: {T} tokens, {K} each, through {C} copies of {H} x {I} are not supported (sizes "
                         f"must be multiples of {multiple}, copies at most 2048, and tokens, a copy's weights and each tensor's "
                         "scales below 2 GiB)")
    dev = hidden.device
    with _on(dev):
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        out = torch.empty_like(hidden)
        counts = None if recorder is None else torch.empty(C, dtype=torch.int32, device=dev)
        experts._poll_pending_checks()
        check = kernels.RouteCheck()
        status_host = check.arm(dev)
        try:
            _capi.call(
                _sym(entry, dt), _ptr(hidden), _ptr(routing_weights), _ptr(sel), _ptr(mapping), _ptr(sources),
                int(source), S, E, _ptr(weights.gate_up.codes), _ptr(weights.gate_up.scales), _ptr(weights.down.codes),
                _ptr(weights.down.scales), T, K, H, I, C, _ptr(out), _ptr(counts), _ptr(ws), ws_bytes, status_host, _stream(dev),
            )
        except ValueError:  # arguments refused: nothing was launched
            check.refused()
            raise
        except _capi.PmxError:  # a launch failed, others of the call may run
            check.launch_failed()
            raise
        experts.note_routing(check)
        if recorder is not None:
            recorder(counts)
    return out
