"""A 4-bit checkpoint's exponents, row by row, in this library's order: the integration guide's code, run as written."""

import re
from pathlib import Path

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import rows4_oracle as O
from placemoe_amd import rows8
from tests import test_rows4

DOC = Path(__file__).resolve().parent.parent / "INTEGRATION.md"


def _snippet() -> str:
    blocks = [b for b in re.findall(r"```python\n(.*?)```", DOC.read_text(), flags=re.S) if "def rows4_scales" in b]
    assert len(blocks) == 1, "the guide converts exponents in one place"
    return blocks[0]


@pytest.mark.parametrize("C,H,I", [((), 5, 32), ((), 3, 768), ((), 4, 512), ((3,), 7, 768), ((2,), 1, 1056), ((2, 3), 4, 544)])
def test_exponents_of_a_checkpoint(C, H, I):
    g = torch.Generator().manual_seed(I)
    x = (torch.randn((*C, H, I), generator=g) * torch.logspace(-6, 4, H).unsqueeze(1)).bfloat16().view(-1, H, I)
    want = torch.stack([O.quantize(m)[1] for m in x])  # [copies, ceil(I / 512), H, 16]
    e = torch.empty((len(x), H, I // 32), dtype=torch.uint8)
    for j in range(I // 32):
        e[:, :, j] = want[:, j // 16, :, j % 16]
    codes = torch.from_numpy(np.zeros((*C, H, I // 2), dtype=np.uint8))
    ns = {"torch": torch, "placemoe_amd": placemoe_amd, "codes": codes, "e": e.view(*C, H, I // 32), "I": I}
    exec(compile(_snippet(), str(DOC), "exec"), ns)
    down = ns["down"]
    assert down.scales.shape == rows8.scales_shape((*C, H, I)) and down.scales.is_contiguous()
    assert torch.equal(down.scales.view(want.shape), want)
    assert down.shape == (*C, H, I) and down.dtype == test_rows4.BF
