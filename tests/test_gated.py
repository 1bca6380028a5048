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
        for name in "HIN":  # 256 rows of an operand pass one descriptor
            assert call(**{**dict(H=8, I=8, N=8), name: 1 << 22}) == SHAPE
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


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path_factory.mktemp("rule") / "gated_rule"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", str(Path(__file__).with_name("gated_rule_main.cpp")), "-o", str(exe)],
                   check=True)

    def ask(*lines):
        out = subprocess.run([str(exe)], input="\n".join(lines), capture_output=True, text=True, check=True).stdout.split("\n")
        return [[int(v) for v in line.split()] for line in out if line]

    return ask


def test_tilings_are_the_measured_best(rule):
    """Of calls whose times lie well apart (gated_rule.h): kind, rows, N, K -> height of the fastest tiles."""
    best = {(0, 256, 1536, 2048): 64, (0, 8192, 1536, 2048): 256, (1, 1024, 7168, 2048): 128, (2, 1024, 7168, 4096): 128,
            (3, 1024, 2048, 7168): 64, (3, 8192, 768, 2048): 128, (0, 8192, 4096, 7168): 256, (1, 2048, 4096, 11008): 128,
            (2, 1536, 4096, 22016): 128, (3, 17, 264, 512): 64}
    got = rule(*(f"tiling {k} {r} {n} {d}" for k, r, n, d in best))
    assert [g[0] for g in got] == list(best.values())


def test_few_tokens(rule):
    asked = {(1, 7168, 2048, 7168): 1, (64, 7168, 2048, 7168): 1, (65, 7168, 2048, 7168): 0, (64, 2048, 768, 2048): 1,
             (16, 4096, 11008, 4096): 1, (64, 4096, 11008, 4096): 0, (1, 8, 8, 8): 1}
    assert [g[0] for g in rule(*(f"few {t} {h} {i} {n}" for t, h, i, n in asked))] == list(asked.values())


def test_weight_gradients(rule):
    import random

    rng = random.Random(5)
    cases = [(16384, 1536, 2048), (16384, 2048, 768), (8192, 4096, 7168), (17, 2000, 1416), (1, 8, 8), (1 << 31, 8, 8)]
    cases += [(rng.randint(1, 20000), 8 * rng.randint(1, 1000), 8 * rng.randint(1, 1000)) for _ in range(300)]
    for (K, M, N), (small, splits, chunk) in zip(cases, rule(*(f"wgrad {k} {m} {n} 0" for k, m, n in cases))):
        # chunks of whole K-tiles that cover the rows, the last of them with some; small tiles take them whole
        count = -(-K // chunk)
        assert chunk % 64 == 0 and count <= splits <= 32 and (count - 1) * chunk < K, (K, M, N)
        assert not (small and splits > 1)
    assert rule("wgrad 8192 4096 7168 0")[0][:2] == [0, 1] and rule("wgrad 17 2000 1416 0")[0][:2] == [1, 1]
    assert rule("wgrad 16384 1536 2048 0")[0][:2] == [0, 5] and rule("wgrad 16384 2048 768 0")[0][:2] == [0, 10]
