"""Infinite and undefined values in the dense gated block's operands reach what the definition says, at every number of tokens."""

import math

import pytest
import torch

from tests.helpers import assert_exact
from tests.test_gpu_gated import BF, F16, _case, _gate, _run

pytestmark = pytest.mark.gpu


def _kinds(t):
    """0 finite, 1 and -1 infinite, 2 NaN."""
    return torch.where(t.isnan(), 2, torch.where(t.isinf(), torch.sign(t.nan_to_num(0.0, 1.0, -1.0)), 0)).to(torch.int8)


def _definition(x, up, down, dout):
    x, up, down, dout = (t.double() for t in (x, up, down, dout))
    I = down.shape[1]
    gu = x @ up.t()
    g, u = gu[:, :I], gu[:, I:]
    a, slope = _gate(g, "silu")
    dh = dout @ down
    dgu = torch.cat((dh * u * slope, dh * a), 1)
    return (a * u) @ down.t(), dgu @ up, dgu.t() @ x, dout.t() @ (a * u)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 40, 300])
@pytest.mark.parametrize("where", ["down", "dout", "down and dout", "gate_up"])
def test_infinities_and_nan(cuda, where, T, dtype):
    H, I, N = 136, 72, 88
    case = _case(cuda, T, H, I, N, dtype, seed=T)
    clean = _run(*case, "silu")
    x, up, down, dout = case
    if "down" in where:
        down[3, 10], down[7, 20], down[9, 4] = math.inf, -math.inf, math.nan
        down[11, 30], down[11, 31] = math.inf, math.inf  # of one sign or NaN, by act's
    if "dout" in where:
        dout[T // 2, 5], dout[0, 6], dout[T - 1, 8] = math.inf, -math.inf, math.nan
    if where == "gate_up":
        up[I + 40, 9] = math.inf  # u of column 40
    print(f"gated infinite {where} {T} {dtype}", flush=True)
    got, want = _run(*case, "silu"), _definition(*case)
    for name, a, c, v in zip(("out", "dx", "dgate_up", "ddown"), got, clean, want):
        kinds = _kinds(v)
        assert torch.equal(_kinds(a), kinds), f"{name}: {(_kinds(a) != kinds).sum().item()} of {v.numel()} of another kind"
        assert_exact(a[kinds == 0], c[kinds == 0], f"{name}: the others")


@pytest.mark.parametrize("T", [3, 16, 17, 200])
def test_the_range_between_the_products_is_the_types(cuda, T):
    """Gated products of 300 * 300 and of 2^-14 * 2^-13 beside weights that bring them back."""
    I = H = N = 8
    for dtype, keeps in ((BF, True), (F16, False)):
        for size, back in ((300.0, 2.0**-10), (2.0**-13, 2.0**10)):
            x = torch.full((T, H), 0.0, dtype=dtype)
            x[:, 0] = 1
            up = torch.zeros((2 * I, H), dtype=dtype)
            up[:, 0] = size  # g = u = size
            down = torch.full((N, I), back, dtype=dtype)
            print(f"gated range {T} {dtype} {size}", flush=True)
            got = _run(*(t.to(cuda) for t in (x, up, down, torch.ones((T, N), dtype=dtype))), "silu")
            g = torch.tensor(size, dtype=dtype).double()
            h = _gate(g, "silu")[0] * g
            if keeps:
                want = (I * h * back).expand(T, N)
                # act's rounding and out's
                assert ((got[0].double().cpu() - want).abs() <= want.abs() * (2.0**-7 + 2.0**-15)).all()
            else:  # fp16: the product alone is past the type's range
                assert h > 65504 or h < 2.0**-25
                assert (got[0] == (math.inf if h > 1 else 0)).all() and (got[3] == (math.inf if h > 1 else 0)).all()
