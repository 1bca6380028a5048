"""The expert layer over 4-bit weights on every tiling of its two products.

Sizes at which the rule (rows8_rule.h) takes them; tests/test_rows4_tiles.py
holds the sizes to the rule.  A token's output has the same bits in a call of a
few tokens, whose tiles tests/test_gpu_rows4.py holds to the definition; two
tokens of each size are held to it here too.
"""

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import moe_oracle
from placemoe_amd import _capi, rows4, rows8
from tests.helpers import assert_exact
from tests.test_gpu_rows4 import BF, F16, RESTS, _as8, _layer_oracle, _offsets, _randn

pytestmark = pytest.mark.gpu

# T, K, copies, H, I -> rows of fc1's and fc2's tiles (0: 32 x 64 ones; 384: 256 with the short rests on 128)
LAYERS = {
    (96, 8, 160, 2048, 768): (32, 32),
    (364, 3, 117, 992, 224): (32, 32),
    (200, 3, 160, 640, 160): (0, 32),
    (400, 1, 49, 288, 544): (32, 0),
    (598, 4, 70, 544, 96): (0, 128),
    (1358, 2, 93, 352, 288): (32, 128),
    (1348, 6, 53, 736, 96): (128, 256),
    (2254, 8, 102, 160, 160): (256, 128),
    (5485, 5, 123, 224, 96): (256, 256),
    (9521, 5, 59, 928, 736): (384, 256),
    (15951, 6, 108, 672, 800): (256, 384),
    (9666, 5, 144, 992, 864): (384, 384),
    (8192, 8, 160, 2048, 768): (384, 384),
}


def _weights4(cuda, shape, seed, dtype, std):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return rows4.quantize_rows4((torch.randn(shape, generator=g, device=cuda) * std).to(dtype))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("size", LAYERS, ids=str)
def test_a_layer_on_every_tiling(cuda, size, dtype):
    T, K, C, H, I = size
    E, S = C - C // 4, 4
    print(f"rows4 layer {size} {dtype}", flush=True)
    g = torch.Generator().manual_seed(T)
    hidden = _randn((T, H), T, dtype)
    # uneven: every eighth expert is chosen three times as often
    score = torch.rand((T, E), generator=g) ** torch.where(torch.arange(E) % 8 == 0, 1 / 3, 1.0)
    sel = score.topk(K).indices
    w = torch.softmax(torch.randn((T, K), generator=g), -1).to(dtype)
    src = torch.randint(0, S, (T,), generator=g)
    e, s = torch.arange(E), torch.arange(S).unsqueeze(1)
    mapping = torch.where((e < C - E) & (s % 2 == 1), E + e, e).contiguous()
    weights = rows4.Experts4(_weights4(cuda, (C, 2 * I, H), 1, dtype, H**-0.5), _weights4(cuda, (C, H, I), 2, dtype, I**-0.5))
    on = [t.to(cuda) for t in (hidden, w, sel, src)]

    def call(part):
        h, rw, se, so = (t[part].contiguous() for t in on)
        return placemoe_amd.expert_layer_rows4(h, rw, se, weights, mapping=mapping.to(cuda), sources=so)

    out = call(slice(None))
    for part in (slice(0, 1), slice(7, 9), slice(T // 2, T // 2 + 5), slice(T - 3, T)):
        assert_exact(out[part], call(part), f"tokens {part}")
    two = slice(T // 3, T // 3 + 2)
    phys = moe_oracle.map_logical_to_physical(mapping.numpy(), src[two].numpy(), sel[two].numpy())
    used = np.unique(phys)
    some = lambda q: _as8(rows4.Rows4(q.codes[used].contiguous(), q.scales[used].contiguous(), q.columns, dtype))  # noqa: E731
    exact, tol = _layer_oracle(hidden[two], w[two], np.searchsorted(used, phys), rows8.Experts8(some(weights.gate_up), some(weights.down)),
                               torch.finfo(dtype).eps)
    tiny = 2.0**-133 if dtype == BF else 2.0**-24
    assert (np.abs(out[two].double().cpu().numpy() - exact) <= tol * 1.0001 + tiny).all()
    # The oracle's worst case lets fc1 be off by 2^-11 of the largest product of each 64, added up over H / 64 of them; at
    # H = 2048 that is 1.6e-3 of a gate or up value, moves one activation's code in 25 and, added up over I = 768 columns, is
    # a third of the outputs.  The kernel's fc1 is good to fp32: 2^-24 sqrt(H) or so, at most 3e-6, moves a code in 10^4 by a
    # twelfth of its value, sqrt(1e-4) / 12 < 2^-10 of the outputs in root mean square; fc2's cut and 24-bit rows are
    # below 2^-15.  With the last rounding's 2^-8 (at most) that is less than 2^-7.
    off = out[two].double().cpu().numpy() - exact
    assert np.linalg.norm(off) <= 2.0**-7 * np.linalg.norm(exact), np.linalg.norm(off) / np.linalg.norm(exact)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_rests_apart_with_tokens_and_weights_of_rows(cuda, dtype):
    """fc1 as the layer calls it: rows from the tokens that a map names, each with a weight."""
    counts, N, K = RESTS
    before, behind, T = 3, 5, 1777
    G, M, I = len(counts), before + sum(counts) + behind, N // 2
    off = (_offsets(counts) + before).to(torch.int32)
    g = torch.Generator().manual_seed(3)
    x = rows8.quantize_rows(_randn((T, K), 11, dtype).to(cuda))
    w = rows4.quantize_rows4(_randn((G, N, K), 12, dtype, 0.06).to(cuda))
    token = torch.randint(0, T, (M,), generator=g).to(torch.int32).to(cuda)
    row_w = (0.05 + torch.rand(M, generator=g)).to(dtype).to(cuda)
    act = torch.full((M, I), 0x55, dtype=torch.uint8, device=cuda)
    scales = torch.full((1, M, 16), 0x55, dtype=torch.uint8, device=cuda)
    on = off.to(cuda)
    print(f"rows4 rests apart, mapped {dtype}", flush=True)
    assert getattr(_capi.load(), "pmx_rows4_gemm_fc1_swiglu" + ("_f16" if dtype == F16 else ""))(
        x.codes.data_ptr(), x.scales.data_ptr(), T, token.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), on.data_ptr(), G, M, K, I,
        row_w.data_ptr(), act.data_ptr(), scales.data_ptr(), torch.cuda.current_stream().cuda_stream) == _capi.PMX_OK
    for rows in (slice(0, before), slice(M - behind, M)):
        assert (act[rows] == 0x55).all() and (scales[:, rows] == 0x55).all()
    for c, n in enumerate(counts):
        rows = slice(int(off[c]), int(off[c]) + n)
        one = rows4.Rows4(w.codes[c:c + 1].contiguous(), w.scales[c:c + 1].contiguous(), K, dtype)
        ref = rows4.gemm_fc1_swiglu_rows4(x, one, _offsets([n]).to(cuda), token[rows].clone(), row_w[rows].clone())
        assert torch.equal(act[rows], ref.codes.view(torch.uint8)) and torch.equal(scales[:, rows], ref.scales), f"copy {c}"
