"""The dense gated block on 128- and 256-row tiles whose last rows and columns are part of one.

Sizes at which the rule (gated_rule.h) takes these tiles, so that every product
runs on each of them with a short last tile in both directions, with a depth of
whole K-tiles and with one that ends inside; tests/test_gated_tiles.py holds
the sizes to the rule.  Against the definition in 64 bits, with the tolerances
of tests/test_gpu_gated.py.
"""

import pytest
import torch

import placemoe_amd
from placemoe_amd import _capi
from tests.helpers import assert_exact
from tests.test_gpu_gated import BF, F16, GATES, _case, _check, _reference, _run

pytestmark = pytest.mark.gpu

# T, H, I, N -> rows of the tiles of fc1, fc2, fc1's dgrad and fc2's dgrad; T is 1, 15, 17 or 33 past a multiple of 64
TILES = {
    (12417, 320, 344, 320): (256, 128, 128, 128),
    (16385, 368, 448, 192): (128, 128, 256, 256),
    (14543, 320, 320, 624): (256, 256, 128, 128),
    (16001, 576, 136, 832): (128, 256, 256, 64),
    (14497, 128, 832, 64): (256, 64, 64, 256),
    (16657, 128, 704, 512): (256, 256, 64, 256),
    (14031, 128, 576, 64): (64, 64, 64, 256),
}


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("size", TILES, ids=str)
def test_short_last_tiles(cuda, size, dtype):
    kind = GATES[size[0] % 3]
    print(f"gated tiles {size} {kind} {dtype}", flush=True)
    case = _case(cuda, *size, dtype)
    got = _run(*case, kind)
    _check(got, _reference(*case, kind), torch.finfo(dtype).eps)
    with torch.no_grad():  # no gate and up sums are kept: the same output
        assert_exact(placemoe_amd.gated_ffn(*case[:3], activation=kind), got[0], "without gradients")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("size", [*TILES, (1, 72, 40, 24), (17, 264, 136, 520), (65, 128, 520, 128), (1531, 520, 328, 520),
                                  (3001, 264, 520, 264)], ids=str)
def test_what_lies_behind_a_tensor_is_left_alone(cuda, size, dtype):
    """Through the C ABI, every tensor with NaN behind it: outputs' have to stay, inputs' reach no result."""
    print(f"gated canaries {size} {dtype}", flush=True)
    T, H, I, N = size
    case = _case(cuda, *size, dtype)
    planes = 2 if T <= 16 else 1
    lib, suffix = _capi.load(), "_f16" if dtype == F16 else ""
    stream = torch.cuda.current_stream().cuda_stream
    behind = 64 * 8 * max(H, 2 * I, N) + 4096  # more than 64 rows of anything
    need = {"gates": T * I * 8, "act": planes * T * I * 2, "out": T * N * 2, "dx": T * H * 2, "dup": 4 * I * H, "ddown": 2 * N * I,
            "ws": lib.pmx_gated_ffn_workspace_bytes(T, H, I, N)}
    # 0xff throughout is NaN in 16 and in 32 bits
    buf = {k: torch.full((n + behind,), 0xFF, dtype=torch.uint8, device=cuda) for k, n in need.items()}
    x, up, down, dout = (torch.full((t.numel() + behind,), float("nan"), dtype=dtype, device=cuda) for t in case)
    for wide, t in zip((x, up, down, dout), case):
        wide[:t.numel()] = t.flatten()
    at = {k: b.data_ptr() for k, b in buf.items()}

    def forward(gates):
        rc = getattr(lib, "pmx_gated_ffn_fwd" + suffix)(x.data_ptr(), up.data_ptr(), down.data_ptr(), T, H, I, N, 0, gates, at["act"],
                                                        at["out"], stream)
        assert rc == _capi.PMX_OK
        return buf["act"][:need["act"]].clone(), buf["out"][:need["out"]].clone()

    first = forward(None)
    assert (buf["gates"] == 0xFF).all()
    for a, b in zip(forward(at["gates"]), first):
        assert torch.equal(a, b), "with the sums kept"
    rc = getattr(lib, "pmx_gated_ffn_bwd" + suffix)(
        dout.data_ptr(), x.data_ptr(), up.data_ptr(), down.data_ptr(), at["gates"], at["act"], T, H, I, N, 0, at["dx"], at["dup"],
        at["ddown"], at["ws"], need["ws"], stream)
    assert rc == _capi.PMX_OK
    for k, b in buf.items():
        assert (b[need[k]:] == 0xFF).all(), f"behind {k}"
    for wide, t in zip((x, up, down, dout), case):
        assert_exact(wide[:t.numel()].view(t.shape), t, "an input")
        assert wide[t.numel():].isnan().all()
    want = _run(*case, "silu")
    for k, w in zip(("out", "dx", "dup", "ddown"), want):
        assert_exact(buf[k][:need[k]].view(dtype).view(w.shape), w, k)
