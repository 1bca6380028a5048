"""What the checkpointed expert layer keeps, and its SwiGLU backward where gates saturate."""

import numpy as np
import pytest
import torch

from oracle import rows8_oracle as O
from placemoe_amd import experts, rows8
from placemoe_amd.workloads import make_workload
from tests.test_gpu_rows8 import _near, _randn

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("split", [False, True])
def test_frozen_fc1_keeps_no_hidden_states(cuda, split):
    """Only fc1's weight gradient reads the hidden states' 8 bits: frozen, they are not kept."""
    wl = make_workload("qwen3", device=cuda, tokens=512)
    T, A, H, I = wl.T, wl.T * wl.K, wl.H, wl.I

    def kept(trained):
        x, fc1 = wl.hidden.clone().requires_grad_(), wl.fc1.clone()
        w = dict(fc1_1_weight=fc1[:, :I].contiguous(), fc1_2_weight=fc1[:, I:].contiguous()) if split else dict(fc1_1_2_weight=fc1)
        for t in w.values():
            t.requires_grad_(trained)
        total = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (total.append(t), t)[1], lambda t: t):
            experts.expert_layer(x, wl.routing_weights, wl.selected, wl.fc2, mapping=wl.mapping, sources=wl.sources,
                                 activation_checkpoint="int8", **w)
        return sum(t.numel() * t.element_size() for t in total if t.numel() < wl.C * I * H)

    # codes and a byte per 32 of them (padded to 512 columns); positions, sources and weights of the rows
    gate_up, hidden = 2 * A * I + A * 16 * -(-2 * I // 512), T * H + T * 16 * -(-H // 512)
    assert kept(False) <= gate_up + 32 * A
    assert gate_up + hidden <= kept(True) <= gate_up + hidden + 32 * A


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_swiglu_backward_of_saturated_gates(cuda, dtype, fmt):
    """A gate per row, around the exponential's ends (e^-g passes fp32's range at -88.7, is lost beside 1 at 17.4)
    and at the type's; their own blocks, so that 8 bits hold each of them."""
    gates = [-5e37, -1e4, -104.0, -96.0, -90.0, -88.0, -87.0, -80.0, -64.0, -30.0, 17.0, 18.0, 30.0, 64.0, 88.0, 104.0, 1e4, 5e37]
    R, I = len(gates), 32
    gu = _randn((R, 2 * I), 5, dtype)
    most = 6e4 if dtype == F16 else 1e38
    gu[:, :I] = torch.tensor(gates).clamp(-most, most).unsqueeze(1)
    d = _randn((R, I), 6, dtype, 2.0**-6)
    w = (0.05 + torch.rand(R, generator=torch.Generator().manual_seed(7))).to(dtype)
    q = rows8.quantize_rows(gu.to(cuda), fmt)
    v = O.values(q.codes.cpu(), q.scales.cpu())
    g, u = v[:, :I], v[:, I:]
    assert (np.abs(g) >= 16).all() and (g[:10] < 0).all() and (g[10:] > 0).all(), "8 bits hold the gates"
    dn, wn = d.double().numpy(), w.double().numpy()[:, None]
    # (the oracle's own exp(-g) passes the range of 64 bits: those gates' sigmoid is 0)
    e_dg1, e_act, e_dw = O.swiglu_backward(dn, v, wn[:, 0])
    dg1, act_w, dw = rows8.swiglu_bwd_rows8(d.to(cuda), q, w.to(cuda), torch.arange(R, dtype=torch.int32, device=cuda), R)
    # The exponential's argument, up to 2^7 in base 2, is good to 2^-17, and so is the sigmoid; below fp32's normal
    # numbers it is 0.  From 16 on it is 1 to 2^-23, and silu's slope 1 to 16 times that.
    with np.errstate(over="ignore"):
        sig = 1 / (1 + np.exp(-g))
    off = np.where(g > 0, 2.0**-20, np.where(sig < 2.0**-125, sig, sig * 2.0**-16))
    slope = np.where(g < 0, (1 + np.abs(g)) * off, 2.0**-18)
    _near(dg1[:, :I], e_dg1[:, :I], np.abs(dn * wn * u) * slope, dtype, "d gate")
    _near(dg1[:, I:], e_dg1[:, I:], np.abs(dn * wn * g) * off, dtype, "d up")
    _near(act_w, e_act, np.abs(wn * u * g) * off, dtype, "act_w")
    _near(dw, e_dw, (np.abs(dn * u * g) * (off + sig * (I + 8) * 2.0**-24)).sum(1), dtype, "dw")
