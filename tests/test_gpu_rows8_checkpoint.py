"""What the checkpointed expert layer keeps."""

import pytest
import torch

from placemoe_amd import experts
from placemoe_amd.workloads import make_workload

pytestmark = pytest.mark.gpu


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
