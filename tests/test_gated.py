"""The dense gated block without a GPU: the C ABI's refusals, the wrapper's checks, the rules."""

import ctypes

import pytest
import torch

import placemoe_amd
from placemoe_amd import _capi

BF = torch.bfloat16
P = ctypes.c_void_p(256)
ARG, SHAPE, OK = _capi.PMX_ERR_ARG, _capi.PMX_ERR_SHAPE, _capi.PMX_OK
BIG = 1 << 40


@pytest.mark.parametrize("suffix", ["", "_f16"])
def test_c_abi_refusals(suffix):
    lib = _capi.load()
    fwd, bwd = getattr(lib, "pmx_gated_ffn_fwd" + suffix), getattr(lib, "pmx_gated_ffn_bwd" + suffix)
    sizes = dict(T=4, H=16, I=24, N=32)

    def forward(gate=0, at=(P,) * 6, **kw):
        s = {**sizes, **kw}
        return fwd(*at[:3], s["T"], s["H"], s["I"], s["N"], gate, *at[3:], None)

    def backward(gate=0, at=(P,) * 9, ws=P, ws_bytes=BIG, **kw):
        s = {**sizes, **kw}
        return bwd(*at[:6], s["T"], s["H"], s["I"], s["N"], gate, *at[6:], ws, ws_bytes, None)

    for call in (forward, backward):
        for gate in (-1, 3, 100):
            assert call(gate) == ARG
        for name in "THIN":
            assert call(**{name: -8}) == ARG
            assert name == "T" or call(**{name: 0}) == ARG
            assert name == "T" or call(**{name: 20}) == SHAPE  # not a multiple of 8
        assert call(H=1 << 20, I=1 << 10) == SHAPE  # weights of 4 GiB
        assert call(N=1 << 20, I=1 << 10) == SHAPE
        assert call(T=1 << 31) == SHAPE
        assert call(T=0, at=(None,) * 9 if call is backward else (None,) * 6) == OK
    for k in range(6):  # x, gate_up, down, gu, act, out
        at = [P] * 6
        at[k] = ctypes.c_void_p(264)
        assert forward(at=at) == SHAPE, k
        at[k] = None
        if k != 3:  # gu may be left out
            assert forward(at=at) == ARG, k
    dx, dup, ddown = 6, 7, 8
    for wanted, needs in (((dx,), (0, 2, 3, 4)), ((dup,), (0, 1, 3, 4)), ((ddown,), (0, 5))):
        for k in needs:  # dout, x, gate_up, down, gu, act
            at = [P] * 6 + [P if i in wanted else None for i in (6, 7, 8)]
            at[k] = None
            assert backward(at=at) == ARG, (wanted, k)
    for k in range(9):
        at = [P] * 9
        at[k] = ctypes.c_void_p(264)
        assert backward(at=at) == SHAPE, k
    assert backward(at=[P] * 6 + [None] * 3) == ARG
    assert backward(ws=None) == ARG and backward(ws=ctypes.c_void_p(264)) == SHAPE
    need = lib.pmx_gated_ffn_workspace_bytes(4, 16, 24, 32)
    assert need >= 4 * 48 * 2 and backward(ws_bytes=need - 1) == ARG


def test_workspace():
    ws = _capi.load().pmx_gated_ffn_workspace_bytes
    assert ws(0, 16, 24, 32) == 0 and ws(-1, 16, 24, 32) == 0 and ws(4, 12, 24, 32) == 0
    # small weights, many tokens: their gradients' rows are cut into chunks
    assert ws(16384, 2048, 768, 2048) >= 16384 * 1536 * 2 + 2 * 1536 * 2048 * 4
    # a gradient that passes one descriptor is not cut (the sums alone would be 24 GB)
    assert ws(16384, 16384, 32768, 16384) < 16384 * 65536 * 2 + (1 << 32)


def test_wrapper_refuses():
    x, up, down = torch.zeros((2, 16), dtype=BF), torch.zeros((48, 16), dtype=BF), torch.zeros((16, 24), dtype=BF)
    with pytest.raises(AssertionError, match="GPU tensors"):
        placemoe_amd.gated_ffn(x, up, down)
    with pytest.raises(ValueError, match="activation"):
        placemoe_amd.gated_ffn(x, up, down, activation="relu")
