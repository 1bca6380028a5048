"""The dense gated block on the GPU against its definition in 64 bits.

Tolerances are carried through the block as its kernels compute it, in the
worst case: sums in fp32 (a rounding of half a step, 2^-24 of what has been
added up, per product), a rounding to the tensors' type (eps / 2 of the value)
where a value is kept or a product reads it, a sigmoid good to 2^-17 of itself,
and gates whose slope is at most 1.2 and their slopes' slopes 1.
"""

import math

import pytest
import torch

import placemoe_amd
from tests.helpers import assert_exact

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
GATES = ["silu", "gelu_tanh", "quick_gelu"]
ROUND = 2.0**-24


def _randn(shape, seed, dtype=BF, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _case(cuda, T, H, I, N, dtype, seed=0):
    x, dout = _randn((T, H), seed + 1, dtype), _randn((T, N), seed + 4, dtype, 0.1)
    if H > 5:
        x[:, 5] *= 10
    up, down = _randn((2 * I, H), seed + 2, dtype, 1 / math.sqrt(H)), _randn((N, I), seed + 3, dtype, 1 / math.sqrt(I))
    return [t.to(cuda) for t in (x, up, down, dout)]


def _gate(g, kind):
    """(gate, its slope) in 64 bits, from the definitions."""
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g**3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    k = 1.0 if kind == "silu" else 1.702
    s = torch.sigmoid(k * g)
    return g * s, s + k * g * s * torch.sigmoid(-k * g)


def _reference(x, up, down, dout, kind, two=False):
    """[(value, tolerance)] of out, dx, dgate_up, ddown; two: fc2 of the forward and the weights' gradients
    read act and the gradients of gate and up in two values."""
    half = torch.finfo(x.dtype).eps / 2
    tiny = 2.0**-133 if x.dtype == BF else 2.0**-24
    x, up, down, dout = (t.detach().double() for t in (x, up, down, dout))
    T, H = x.shape
    N, I = down.shape
    gu, d_gu = x @ up.t(), x.abs() @ up.abs().t() * (H * ROUND)
    g, u, d_g, d_u = gu[:, :I], gu[:, I:], d_gu[:, :I], d_gu[:, I:]
    a, slope = _gate(g, kind)
    h = a * u
    d_h = 1.2 * d_g * u.abs() + a.abs() * d_u + 1.2 * d_g * d_u + h.abs() * 2.0**-17
    d_h2 = d_h + (h.abs() + d_h) * half * half + tiny
    d_h = d_h + (h.abs() + d_h) * half + tiny
    out = h @ down.t()
    d_out = (d_h2 if two else d_h) @ down.abs().t() + h.abs() @ down.abs().t() * (3 * I * ROUND)
    # backward: gate and up sums as the forward left them, dh from the accumulators
    dh = dout @ down
    d_dh = dout.abs() @ down.abs() * (N * ROUND)
    dg, du = dh * u * slope, dh * a
    most = dh.abs() + d_dh
    d_dg = d_dh * u.abs() * slope.abs() + most * (d_u * 1.2 + (u.abs() + d_u) * (d_g + 2.0**-15))
    d_dg2, d_dg = (d_dg + (dg.abs() + d_dg) * r + tiny for r in (half * half, half))
    d_du = d_dh * a.abs() + most * (1.2 * d_g + a.abs() * 2.0**-16)
    d_du2, d_du = (d_du + (du.abs() + d_du) * r + tiny for r in (half * half, half))
    dgu, d_dgu = torch.cat((dg, du), 1), torch.cat((d_dg, d_du), 1)
    dx, d_dx = dgu @ up, d_dgu @ up.abs() + dgu.abs() @ up.abs() * (4 * I * ROUND)
    d_dgu2 = torch.cat((d_dg2, d_du2), 1)
    dup, d_dup = dgu.t() @ x, (d_dgu2 if two else d_dgu).t() @ x.abs() + dgu.abs().t() @ x.abs() * (2 * T * ROUND)
    ddown = dout.t() @ h
    d_ddown = dout.abs().t() @ (d_h2 if two else d_h) + dout.abs().t() @ h.abs() * (2 * T * ROUND)
    return [(v, t + (v.abs() + t) * half + tiny) for v, t in ((out, d_out), (dx, d_dx), (dup, d_dup), (ddown, d_ddown))]


def _run(x, up, down, dout, kind, **kw):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, up, down)]
    out = placemoe_amd.gated_ffn(*leaves, activation=kind, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _check(got, want, eps, size=1 << 12):
    for name, a, (v, tol) in zip(("out", "dx", "dgate_up", "ddown"), got, want):
        assert a.shape == v.shape, name
        off = (a.double() - v).abs()
        assert torch.isfinite(a).all(), name
        assert (off <= tol * 1.0001).all(), f"{name}: {off.max().item()} off, {(off - tol).max().item()} over its tolerance"
        if a.numel() >= size:
            # two roundings on the way, an operand's and its own, each of root mean square at most eps / sqrt(12) of its values
            far = off.norm() / v.norm()
            assert far <= math.sqrt(2) * eps / math.sqrt(12), f"{name}: {far.item()} from the definition"


SIZES = [(1, 8, 8, 8), (3, 24, 40, 16), (7, 64, 8, 72), (16, 200, 120, 328), (17, 264, 136, 520), (33, 1000, 264, 1000), (65, 128, 512, 128),
         (130, 1416, 1000, 1416), (257, 512, 256, 264), (600, 72, 2056, 80), (1531, 520, 328, 520), (2100, 264, 72, 1024)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,H,I,N", SIZES)
def test_against_the_definition(cuda, T, H, I, N, dtype):
    kind = GATES[(T + H // 8) % 3]
    print(f"gated {T} {H} {I} {N} {kind} {dtype}", flush=True)
    case = _case(cuda, T, H, I, N, dtype)
    _check(_run(*case, kind), _reference(*case, kind), torch.finfo(dtype).eps)


@pytest.mark.parametrize("kind", GATES)
@pytest.mark.parametrize("T", [1, 5, 16, 17, 64, 300, 3000])
def test_every_gate(cuda, T, kind):
    case = _case(cuda, T, 512, 264, 384, BF, seed=T)
    print(f"gated {kind} {T}", flush=True)
    got = _run(*case, kind)
    _check(got, _reference(*case, kind), torch.finfo(BF).eps)
    with torch.no_grad():  # nothing kept: the same output
        assert_exact(placemoe_amd.gated_ffn(*case[:3], activation=kind), got[0], "without gradients")


def test_large(cuda):
    case = _case(cuda, 4096, 2048, 768, 2048, BF)
    _check(_run(*case, "silu"), _reference(*case, "silu"), torch.finfo(BF).eps)


@pytest.mark.parametrize("kind", GATES)
def test_gradients_against_differences(cuda, kind):
    """(f(p + h v) - f(p - h v)) / 2h of the sum f of out * dout in 64 bits, along v = the gradient, against |gradient|^2."""
    x, up, down, dout = _case(cuda, 40, 64, 48, 56, BF)
    _, *grads = _run(x, up, down, dout, kind)
    base = [t.double() for t in (x, up, down)]

    def f(p):
        gu = p[0] @ p[1].t()
        I = gu.shape[1] // 2
        return ((_gate(gu[:, :I], kind)[0] * gu[:, I:]) @ p[2].t() * dout.double()).sum()

    for k, grad in enumerate(grads):
        v, h = grad.double() / grad.double().norm(), 1e-5
        plus, minus = list(base), list(base)
        plus[k], minus[k] = base[k] + h * v, base[k] - h * v
        slope = (f(plus) - f(minus)) / (2 * h)
        # the gradient is within 2 eps / sqrt(12) of the true one (see _check), h^2 terms far below
        assert abs(slope / grad.double().norm() - 1) <= 2 * torch.finfo(BF).eps / math.sqrt(12), (k, slope, grad.norm())


@pytest.mark.parametrize("kind", GATES)
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T", [8, 40])
def test_extreme_gates(cuda, kind, dtype, T):
    """Gate values from the smallest to the largest of the type: sigmoids of 0 and 1, squares past fp32."""
    I = H = N = 16
    big = float(torch.finfo(dtype).max)
    values = torch.tensor([0.0, 1e-6, 0.5, -0.5, 3, -3, 11, -11, 30, -30, 90, -90, 300, -300, big, -big])
    x = torch.zeros((T, H), dtype=dtype)
    x[:, 0] = values[torch.arange(T) % 16].to(dtype)
    x[:, 1] = 1
    up = torch.zeros((2 * I, H), dtype=dtype)
    up[:I, 0] = 1  # gate = x0
    up[I:, 1] = 0.25  # up = 1/4
    down = torch.eye(N, I, dtype=dtype)
    dout = torch.full((T, N), 0.5, dtype=dtype)
    case = [t.to(cuda) for t in (x, up, down, dout)]
    got = _run(*case, kind)
    g = x[:, :1].double()
    a, slope = _gate(g, kind)
    slope = torch.where(g.abs() > 200, (g > 0).double(), slope)  # 0 * inf in the definition
    a = torch.where(g > 200, g, torch.where(g < -200, 0.0, a))
    eps = torch.finfo(dtype).eps
    out = (a * 0.25).expand(T, N)
    # (dx1 of the largest gate, 16 * 0.125 = 2 times it, is past the type: infinite, compared below where it fits)
    assert torch.isfinite(got[0]).all() and not got[1].isnan().any() and torch.isfinite(got[1][:, 0]).all()
    # a sigmoid below 2^-126, fp32's smallest normal, may count as 0: off by |gate| 2^-126, at most 2^-119 for the |gate| <= 90
    # where it is not 0 in 64 bits either
    tiny = 2.0**-119 if dtype == BF else 2.0**-23
    assert ((got[0].cpu().double() - out).abs() <= out.abs() * (eps + 2.0**-15) + tiny).all()
    # dx0 = sum over I columns of 0.5 * 0.25 * slope, dx1 = 0.25 * sum of 0.5 * a
    want = torch.cat((I * 0.125 * slope, I * 0.125 * a), 1)
    tol = want.abs() * (2.5 * eps + 2.0**-14) + I * 0.125 * 2.0**-14 * torch.tensor([[1.0, 0.0]]) + I * tiny
    if dtype == F16:  # 2 * 65504 is past the type
        want, tol = want[g[:, 0].abs() < 1e4], tol[g[:, 0].abs() < 1e4]
        assert ((got[1].cpu().double()[g[:, 0].abs() < 1e4, :2] - want).abs() <= tol).all()
    else:
        fits = want.abs() < 3e38
        assert ((got[1].cpu().double()[:, :2] - want).abs() <= tol)[fits].all()


@pytest.mark.parametrize("T", [5, 200])
def test_what_is_not_finite_stays_with_its_token(cuda, T):
    case = _case(cuda, T, 136, 72, 88, BF)
    ref = _run(*case, "silu")
    case[0][2, 7], case[0][4, 100] = math.nan, math.inf
    got = _run(*case, "silu")
    bad = torch.zeros(T, dtype=torch.bool, device=cuda)
    bad[[2, 4]] = True
    assert got[0][bad].isnan().any(1).all() and got[1][bad].isnan().any(1).all()
    for k in (0, 1):
        assert_exact(got[k][~bad], ref[k][~bad], "the others")


def test_leading_dimensions_and_layouts(cuda):
    x, up, down, dout = _case(cuda, 60, 64, 48, 56, BF)
    flat = _run(x, up, down, dout, "silu")
    for lead in ((60,), (5, 12), (3, 4, 5), (1, 60, 1)):
        got = _run(x.view(*lead, 64), up, down, dout.view(*lead, 56), "silu")
        assert got[0].shape == (*lead, 56) and got[1].shape == (*lead, 64)
        for a, b in zip(got, flat):
            assert_exact(a.reshape(b.shape), b)
    one = placemoe_amd.gated_ffn(x[3], up, down)
    assert one.shape == (56,)
    assert_exact(one, placemoe_amd.gated_ffn(x[3:4], up, down)[0])
    # a gradient that is not contiguous, and one that is broadcast
    out = _run(x, up, down, dout.t().contiguous().t(), "silu")
    assert_exact(out[1], flat[1])
    leaves = [t.clone().requires_grad_(True) for t in (x, up, down)]
    placemoe_amd.gated_ffn(*leaves).sum().backward()
    ones = _run(x, up, down, torch.ones_like(dout), "silu")
    for leaf, b in zip(leaves, ones[1:]):
        assert_exact(leaf.grad, b)


@pytest.mark.parametrize("T", [3, 120, 1000])
def test_only_the_wanted_gradients(cuda, T):
    x, up, down, dout = _case(cuda, T, 136, 72, 88, BF)
    full = _run(x, up, down, dout, "gelu_tanh")
    for mask in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, up, down))]
        out = placemoe_amd.gated_ffn(*leaves, activation="gelu_tanh")
        out.backward(dout)
        assert_exact(out, full[0])
        for k, leaf in enumerate(leaves):
            if mask >> k & 1:
                assert_exact(leaf.grad, full[1 + k], f"mask {mask}, leaf {k}")
            else:
                assert leaf.grad is None


@pytest.mark.parametrize("kind", GATES)
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,H,I,N", [(1, 520, 264, 520), (2, 280, 64, 280), (7, 1416, 1000, 1416), (16, 128, 1000, 72), (16, 2048, 768, 2048)])
def test_few_tokens_are_rounded_once(cuda, T, H, I, N, dtype, kind):
    """Of up to 16 tokens out and the weights' gradients alone are rounded: to half a step and what their sums are off."""
    case = _case(cuda, T, H, I, N, dtype, seed=T)
    got, want, eps = _run(*case, kind), _reference(*case, kind, two=True), torch.finfo(dtype).eps
    for k in (0, 2, 3):
        (v, tol), off = want[k], (got[k].double() - want[k][0]).abs()
        assert (off <= tol * 1.0001).all(), k
        # one rounding, of root mean square at most eps / sqrt(12) of its values, and what the sums are off
        assert off.norm() <= eps / math.sqrt(12) * v.norm() + (tol - v.abs() * eps / 2).clamp(min=0).norm(), k
    with torch.no_grad():
        assert_exact(placemoe_amd.gated_ffn(*case[:3], activation=kind), got[0], "without gradients")


@pytest.mark.parametrize("T", [3, 120])
def test_some_gradients_of_a_graph_that_has_all(cuda, T):
    case = _case(cuda, T, 264, 136, 200, BF)
    full = _run(*case, "silu")
    leaves = [t.clone().requires_grad_(True) for t in case[:3]]
    out = placemoe_amd.gated_ffn(*leaves)
    for mask in (1, 2, 4, 3, 5, 6, 7):
        wanted = [k for k in range(3) if mask >> k & 1]
        for k, d in zip(wanted, torch.autograd.grad(out, [leaves[k] for k in wanted], case[3], retain_graph=True)):
            assert_exact(d, full[1 + k], f"mask {mask}, leaf {k}")


def test_under_checkpoints_and_saved_elsewhere(cuda):
    """Recomputed in the backward, and with what is kept moved to the host meanwhile."""
    from torch.utils.checkpoint import checkpoint

    x, up, down, dout = _case(cuda, 90, 264, 136, 200, BF)
    want = _run(x, up, down, dout, "silu")
    for way in ("reentrant", "not", "host"):
        leaves = [t.clone().requires_grad_(True) for t in (x, up, down)]
        if way == "host":
            with torch.autograd.graph.save_on_cpu():
                out = placemoe_amd.gated_ffn(*leaves)
        else:
            out = checkpoint(placemoe_amd.gated_ffn, *leaves, use_reentrant=way == "reentrant")
        out.backward(dout)
        for a, w in zip([out.detach(), *(t.grad for t in leaves)], want):
            assert_exact(a, w, way)


def test_a_leaf_used_twice_and_two_backwards(cuda):
    """Tied tokens and weights accumulate; a retained graph gives its gradients again."""
    x, up, down, dout = _case(cuda, 50, 64, 48, 64, BF)
    a, b, c = (t.clone().requires_grad_(True) for t in (x, up, down))
    mid = placemoe_amd.gated_ffn(a, b, c)
    out = placemoe_amd.gated_ffn(mid, b, c)
    got = torch.autograd.grad(out, (a, b, c), dout, retain_graph=True)
    again = torch.autograd.grad(out, (a, b, c), dout)
    second = _run(mid.detach(), up, down, dout, "silu")
    first = _run(x, up, down, second[1], "silu")
    assert_exact(got[0], first[1])
    for k in (1, 2):
        assert_exact(got[k], first[1 + k] + second[1 + k])
    for u, v in zip(got, again):
        assert_exact(u, v)
    with pytest.raises(RuntimeError):  # no second derivative
        out = placemoe_amd.gated_ffn(a, b, c)
        (d,) = torch.autograd.grad(out, a, dout, create_graph=True)
        d.sum().backward()


def test_a_gradient_at_an_odd_address(cuda):
    """Out's gradient as a part of a larger one, two bytes past a boundary."""
    x, up, down, dout = _case(cuda, 20, 64, 48, 56, BF)
    want = _run(x, up, down, dout, "silu")
    leaves = [t.clone().requires_grad_(True) for t in (x, up, down)]
    both = torch.cat([leaves[0].detach().flatten()[:1], placemoe_amd.gated_ffn(*leaves).flatten()])
    both.backward(torch.cat([dout.flatten()[:1], dout.flatten()]))
    for leaf, w in zip(leaves, want[1:]):
        assert_exact(leaf.grad, w)


def test_a_loss_over_gradients_is_refused(cuda):
    x, up, down, dout = _case(cuda, 20, 64, 48, 56, BF)
    a = x.clone().requires_grad_(True)
    for weights in ((up, down), tuple(t.clone().requires_grad_(True) for t in (up, down))):
        out = placemoe_amd.gated_ffn(a, *weights)
        (d,) = torch.autograd.grad(out, a, dout, create_graph=True)
        assert_exact(d, _run(x, up, down, dout, "silu")[1])
        with pytest.raises(RuntimeError, match="second"):
            (out.sum() + d.square().sum()).backward()


def test_no_tokens(cuda):
    x, up, down, dout = _case(cuda, 4, 64, 48, 56, BF)
    got = _run(x[:0], up, down, dout[:0], "silu")
    assert got[0].shape == (0, 56) and got[1].shape == (0, 64)
    assert (got[2] == 0).all() and (got[3] == 0).all() and got[2].shape == up.shape and got[3].shape == down.shape
    assert placemoe_amd.gated_ffn(x.view(2, 2, 64)[:, :0], up, down).shape == (2, 0, 56)


def test_refusals(cuda):
    x, up, down, _ = _case(cuda, 4, 64, 48, 56, BF)
    f = placemoe_amd.gated_ffn
    for bad in (
        lambda: f(x.half(), up, down),
        lambda: f(x, up.half(), down),
        lambda: f(x.float(), up.float(), down.float()),
        lambda: f(x, up.cpu(), down),
        lambda: f(x, up[:-1], down),
        lambda: f(x[:, :56].contiguous(), up, down),
        lambda: f(x, up, down[:, :40].contiguous()),
        lambda: f(x.t().contiguous().t(), up, down),
        lambda: f(x, up.t().contiguous().t(), down),
        lambda: f(x, up[None], down),
        lambda: f(x[0, 0], up, down),
    ):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(ValueError):
        f(_randn((4, 60), 1).to(cuda), _randn((96, 60), 1).to(cuda), down)  # H
    with pytest.raises(ValueError):  # alignment
        f(torch.zeros(4 * 64 + 4, dtype=BF, device=cuda)[4:].view(4, 64), up, down)


def test_on_two_streams_at_once(cuda):
    cases = [_case(cuda, T, 264, 136, 200, BF, seed=T) for T in (9, 700)]
    want = [_run(*c, "silu") for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k, _run(*cases[k], "silu")))
    torch.cuda.synchronize()
    for k, outs in got:
        for j, (a, b) in enumerate(zip(outs, want[k])):
            assert_exact(a, b, f"case {k}, output {j}")


@pytest.mark.parametrize("T", [2, 900])
def test_in_a_graph(cuda, T):
    """Forward and backward captured; replays with other inputs between eager calls."""
    case = _case(cuda, T, 264, 136, 200, BF)
    _run(*case, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _run(*case, "silu")
    for k in range(3):
        case[0].copy_(_randn((T, 264), 80 + k).to(cuda))
        graph.replay()
        eager = _run(*case, "silu")
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(outs, eager)):
            assert_exact(a, b, f"replay {k}, output {j}")


def test_results_do_not_change_from_call_to_call(cuda):
    case = _case(cuda, 3000, 520, 264, 520, BF)
    first = _run(*case, "silu")
    for _ in range(3):
        for a, b in zip(_run(*case, "silu"), first):
            assert_exact(a, b)


def test_nothing_waits_for_the_gpu(cuda):
    cases = [_case(cuda, T, 64, 48, 56, BF) for T in (3, 500)]
    for c in cases:
        _run(*c, "silu")
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for c in cases:
            _run(*c, "silu")
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()


def test_offsets_past_32_bits(cuda):
    """gu of more than 2^31 elements: 4096 tokens over and over, each repeat the same as the first."""
    n, times, H, I, N = 4096, 260, 64, 1024, 64
    assert n * times * 2 * I > 2**31
    x, up, down, dout = _case(cuda, n, H, I, N, BF)
    ref = _run(x, up, down, dout, "silu")
    got = _run(x.repeat(times, 1), up, down, dout.repeat(times, 1), "silu")
    for k in (0, 1):
        assert_exact(got[k][-n:], ref[k])
    want = _reference(x, up, down, dout, "silu")
    for k in (2, 3):
        # sums of all repeats: the partial ones grow to the last, one rounding of 2^-24 for each 16 tokens
        v = want[k][0] * times
        far = (got[k].double() - v).norm() / v.norm()
        assert far <= 2 * torch.finfo(BF).eps / math.sqrt(12) + n * times / 16 * ROUND, far


def test_one_block_beside_the_routed_experts(cuda):
    """Routed experts and the block that every token passes, summed, with one backward through both."""
    from placemoe_amd.workloads import make_workload

    wl = make_workload("qwen3", tokens=64)
    leaf = lambda t: t.to(cuda).requires_grad_(True)  # noqa: E731
    x, w, fc1, fc2 = leaf(wl.hidden), leaf(wl.routing_weights), leaf(wl.fc1), leaf(wl.fc2)
    up, down = leaf(_randn((2 * 768, wl.H), 5, BF, 0.02)), leaf(_randn((wl.H, 768), 6, BF, 0.02))
    dout = _randn((wl.T, wl.H), 7).to(cuda)

    def routed():
        return placemoe_amd.expert_layer(x, w, wl.selected.to(cuda), fc2, fc1_1_2_weight=fc1, mapping=wl.mapping.to(cuda),
                                         sources=wl.sources.to(cuda))

    both = torch.autograd.grad(routed() + placemoe_amd.gated_ffn(x, up, down), (x, up, down), dout)
    (dx_routed,) = torch.autograd.grad(routed(), (x,), dout)
    dx, dup, ddown = torch.autograd.grad(placemoe_amd.gated_ffn(x, up, down), (x, up, down), dout)
    assert_exact(both[0], dx_routed + dx)
    assert_exact(both[1], dup)
    assert_exact(both[2], ddown)
