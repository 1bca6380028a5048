"""The serving layer over 8-bit weights on every tiling of its two products.

The tilings that the cases reach are checked on the host by
tests/test_rows8.py."""

import math

import numpy as np
import pytest
import torch

import placemoe_amd
from placemoe_amd import kernels, rows8
from tests.helpers import assert_bf16_close, assert_exact
from tests.test_gpu_rows8 import SUBNORMAL, _layer_oracle, _randn

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16

# name: (tokens, experts per token, copies, hidden size, intermediate size); widths that end inside every tile
LAYERS = {
    "narrow": (10, 3, 6, 1040, 272),
    "few": (120, 4, 96, 1040, 528),
    "mid": (600, 2, 12, 2064, 272),
    "large": (4000, 2, 6, 1040, 272),
    "large wide": (4096, 4, 5, 2064, 272),
    "large, many copies": (6000, 4, 96, 1040, 528),
}


def _case(cuda, name, dtype=BF):
    """(hidden, weights, selected, 16-bit gate_up and down): ragged, one copy without tokens."""
    T, K, C, H, I = LAYERS[name]
    print(f"layer rows8 {name} {dtype}", flush=True)
    g = torch.Generator().manual_seed(T + C)
    share = torch.exp(torch.randn(C, generator=g))
    share[C // 2] = 0
    sel = torch.multinomial(share.expand(T, C), K, generator=g)
    w = torch.softmax(torch.randn((T, K), generator=g), -1).to(dtype)
    gate_up, down = _randn((C, 2 * I, H), 1, dtype, 1 / math.sqrt(H)), _randn((C, H, I), 2, dtype, 1 / math.sqrt(I))
    return _randn((T, H), 3, dtype).to(cuda), w.to(cuda), sel.to(cuda), gate_up.to(cuda), down.to(cuda)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("name", LAYERS)
def test_layer_against_64_bits(cuda, name, dtype):
    """Some tokens, the last among them, against the definition, and their bits in calls of their own."""
    x, w, sel, gate_up, down = _case(cuda, name, dtype)
    q = rows8.Experts8.quantize(gate_up, down)
    got = placemoe_amd.expert_layer_rows8(x, w, sel, q)
    some = torch.linspace(0, x.shape[0] - 1, 10).long().to(cuda)
    exact, tol = _layer_oracle(x[some].cpu(), w[some].cpu(), sel[some].cpu().numpy(), q, torch.finfo(dtype).eps)
    off = np.abs(got[some].double().cpu().numpy() - exact)
    assert (off <= tol * 1.0001 + SUBNORMAL[dtype]).all(), (off - tol).max()
    assert_bf16_close(got[some], torch.from_numpy(exact), name="out")
    assert_exact(placemoe_amd.expert_layer_rows8(x[some], w[some], sel[some], q), got[some], "a few tokens")


@pytest.mark.parametrize("name", LAYERS)
def test_loud_columns_leave_the_others_alone(cuda, name):
    """fc2's rows hold every column to a share of itself: some outputs 2^10 times as loud (an exact factor, as the
    down projections of trained models have) change no bit of the others beside them."""
    x, w, sel, gate_up, down = _case(cuda, name)
    plain = placemoe_amd.expert_layer_rows8(x, w, sel, rows8.Experts8.quantize(gate_up, down))
    loud = torch.zeros(down.shape[1], dtype=torch.bool, device=cuda)
    loud[5::32] = True
    louder = torch.where(loud.view(1, -1, 1), down * 1024, down)
    got = placemoe_amd.expert_layer_rows8(x, w, sel, rows8.Experts8.quantize(gate_up, louder))
    assert_exact(got[:, ~loud], plain[:, ~loud], "columns beside the loud ones")
    assert_exact(got[:, loud], plain[:, loud] * 1024, "loud columns")


@pytest.mark.parametrize("name", LAYERS)
def test_layer_keeps_nan_to_its_token(cuda, name):
    x, w, sel, gate_up, down = _case(cuda, name)
    q = rows8.Experts8.quantize(gate_up, down)
    want = placemoe_amd.expert_layer_rows8(x, w, sel, q)
    bad, w2, T = x.clone(), w.clone(), x.shape[0]
    bad[2, 7], bad[T // 2, 50], w2[T - 1, 1] = math.nan, -math.inf, math.nan
    got = placemoe_amd.expert_layer_rows8(bad, w2, sel, q)
    hit = torch.tensor([2, T // 2, T - 1], device=cuda)
    assert got[hit].isnan().all()
    rest = torch.ones(T, dtype=torch.bool, device=cuda)
    rest[hit] = False
    assert_exact(got[rest], want[rest], "the other tokens")


def test_the_layer_in_steps(cuda):
    """Routing, tokens to 8 bits, fc1, fc2 and the sum as calls of their own: the layer, but for fc2's rows, which
    the public product rounds to the tensors' dtype."""
    x, w, sel, gate_up, down = _case(cuda, "mid")
    q, C = rows8.Experts8.quantize(gate_up, down), down.shape[0]
    r = kernels.route(sel, C)
    tokens, row_token, row_w = rows8.quantize_rows_routed(x, r.pos, w)
    act = rows8.gemm_fc1_swiglu_rows8(tokens, q.gate_up, r.offsets, row_token, row_w)
    y = rows8.group_gemm_nt_rows8(act, q.down, r.offsets)
    got, want = kernels.moe_gather(y, r.pos).double(), placemoe_amd.expert_layer_rows8(x, w, sel, q).double()
    # half a step of each row, and of each sum
    rows = y.double().abs()[r.pos.long()].sum(1)
    tol = (rows + got.abs() + want.abs()) * torch.finfo(BF).eps / 2
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() - tol).max()
