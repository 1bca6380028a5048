"""The dense gated block: what every token passes beside the routed experts
(a model's shared experts) or in their place (its dense layers).

``gated_ffn`` is differentiable in the tokens and both weights; a handful of
tokens (serving) run on kernels of their own.  Kernels are enqueued on the
current stream of the tensors' device and waited for by nobody.  Wrong devices,
dtypes and shapes raise ``AssertionError``, limits of the kernels
``ValueError``, both before anything is launched; there is no CPU fallback.
"""

from __future__ import annotations

import torch

from . import _capi
from .kernels import _check_dev, _half, _ptr
from .rows8 import _launch

GATES = {"silu": 0, "gelu_tanh": 1, "quick_gelu": 2}


def _forward(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, gate: int, keep_gates: bool, keep_act: bool):
    """(out, what is kept): the bytes of the gate and up sums in fp32 and, behind them, of act; of either alone where
    the other is not wanted (one tensor: each takes some microseconds of a small call)."""
    T, H = x.shape
    N, I = down.shape
    out = x.new_empty((T, N))
    behind = 8 * T * I if keep_gates else 0
    alone = keep_gates and not keep_act
    size = (2 if T <= 16 else 1) * T * I  # act's
    kept = x.new_empty(behind if alone else behind + 2 * size, dtype=torch.uint8)
    passing = x.new_empty(size) if alone else None  # act, on its way to fc2 only
    gates = kept.data_ptr() if keep_gates else None
    act = passing.data_ptr() if alone else kept.data_ptr() + behind
    _launch("pmx_gated_ffn_fwd", x.dtype, x.device, _ptr(x), _ptr(gate_up), _ptr(down), T, H, I, N, gate, gates, act, _ptr(out))
    return out, kept


class _NoSecond(torch.autograd.Function):
    """A gradient as it is, differentiable by nobody."""

    @staticmethod
    def forward(ctx, grad, _):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("gated_ffn has no second derivative")


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up, down, gate):
        need_x, need_up, need_down = ctx.needs_input_grad[:3]
        out, kept = _forward(x, gate_up, down, gate, need_x or need_up, need_down)
        ctx.gate = gate
        # what the wanted gradients read
        ctx.save_for_backward(x if need_up else None, gate_up if need_x else None, down if need_x or need_up else None, kept)
        ctx.has_gates = need_x or need_up  # (in the backward these flags say what the one call wants)
        ctx.sizes = (*x.shape, down.shape[1])
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x, gate_up, down, kept = ctx.saved_tensors
        T, H, I = ctx.sizes
        N = grad_out.shape[1]
        grad_out = grad_out.contiguous()
        if grad_out.data_ptr() % 16:  # a part of a larger gradient
            grad_out = grad_out.clone()
        need_x, need_up, need_down = ctx.needs_input_grad[:3]
        new = grad_out.new_empty
        dx = new((T, H)) if need_x else None
        dup = new((2 * I, H)) if need_up else None
        ddown = new((N, I)) if need_down else None
        if T == 0:
            for d in (dup, ddown):
                if d is not None:
                    d.zero_()
            return dx, dup, ddown, None
        gates = kept.data_ptr()
        act = gates + (T * I * 8 if ctx.has_gates else 0)
        ws_bytes = _capi.load().pmx_gated_ffn_workspace_bytes(T, H, I, N)
        ws = new(ws_bytes, dtype=torch.uint8)
        _launch("pmx_gated_ffn_bwd", grad_out.dtype, grad_out.device, _ptr(grad_out), _ptr(x), _ptr(gate_up), _ptr(down),
                gates if ctx.has_gates else None, act if need_down else None, T, H, I, N, ctx.gate, _ptr(dx), _ptr(dup), _ptr(ddown), _ptr(ws), ws_bytes)
        if torch.is_grad_enabled():  # create_graph: a loss over these gradients must not miss its terms silently
            mark = torch.empty(0, requires_grad=True)
            dx, dup, ddown = (None if d is None else _NoSecond.apply(d, mark) for d in (dx, dup, ddown))
        return dx, dup, ddown, None


def gated_ffn(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """out = (gate(x @ Wg^T) * (x @ Wu^T)) @ down^T, [..., H] -> [..., N].

    x [..., H], gate_up [2I, H] (the rows of Wg, then those of Wu) and down
    [N, I], all bfloat16 or all float16, contiguous; H, I and N multiples of 8.
    ``activation``: "silu", "gelu_tanh" (GELU's tanh form) or "quick_gelu"
    (g sigmoid(1.702 g)).

    Sums are held in fp32; the gated products, and in the backward the gradients
    of gate and up, are rounded to the tensors' dtype, being operands of
    products (up to 16 tokens, for fc2 and the weights' gradients, to two such
    values each).  In float16 those beyond 65504 are infinite, and what is below
    2^-25 is lost, also where an output or a gradient itself would be in range:
    scale the loss as for any float16 training; bfloat16 has fp32's range.  For
    the backward x, the gate and up sums [tokens, 2I] in fp32 and their products
    [tokens, I] are kept, as far as the gradients that are wanted read them.
    """
    if activation not in GATES:
        raise ValueError(f"activation must be one of {sorted(GATES)}, got {activation!r}")
    _check_dev(x, gate_up, down)
    dt = _half("x", x)
    _half("gate_up", gate_up, dt)
    _half("down", down, dt)
    assert gate_up.dim() == 2 and down.dim() == 2, "gate_up and down must be matrices"
    N, I = down.shape
    H = gate_up.shape[1]
    assert gate_up.shape[0] == 2 * I, f"gate_up must have {2 * I} rows, twice the columns of down, got {gate_up.shape[0]}"
    assert x.dim() >= 1 and x.shape[-1] == H, f"x must be [..., {H}], got {tuple(x.shape)}"
    rows = x.reshape(-1, H) if x.dim() != 2 else x
    if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad):
        out = _GatedFFN.apply(rows, gate_up, down, GATES[activation])
    else:
        out = _forward(rows, gate_up, down, GATES[activation], False, False)[0]
    return out if x.dim() == 2 else out.view(*x.shape[:-1], N)
