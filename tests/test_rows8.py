"""Rows in 8 bits without a GPU: the oracle against the format's own float
type, the C ABI's refusals, and the wrappers' checks (all before any launch)."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import rows8_oracle as O
from placemoe_amd import _capi, experts, rows8
from tests import test_gpu_rows8, test_gpu_rows8_layer

ROOT = Path(__file__).resolve().parents[1]

BF = torch.bfloat16


@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_oracle_rounds_like_the_e4m3_type(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((40, 100), generator=g) * torch.logspace(-6, 4, 40).unsqueeze(1)).to(dtype)
    x[3] = 0
    v, scales = O.quantize(x, "e4m3")
    e = scales.permute(1, 0, 2).reshape(40, -1).to(torch.int64) - 127
    unit = torch.exp2(e.double()).repeat_interleave(32, 1)[:, :100]
    want = (x.double() / unit).float().to(torch.float8_e4m3fn).double() * unit
    assert np.array_equal(v, want.numpy())
    # the smallest power: half of it would not hold the block's largest value
    most = torch.nn.functional.pad(x.double().abs(), (0, 28)).view(40, 4, 32).amax(-1)
    u = torch.exp2(e[:, :4].double())
    assert (most <= 448 * u).all() and ((most > 224 * u) | (most == 0)).all()


def test_oracle_int8_is_within_half_a_step():
    x = torch.randn((9, 70), generator=torch.Generator().manual_seed(4)).to(BF)
    v, scales = O.quantize(x, "int8")
    e = scales.permute(1, 0, 2).reshape(9, -1).to(torch.int64) - 127
    unit = torch.exp2(e.double()).repeat_interleave(32, 1)[:, :70].numpy()
    assert (np.abs(v - x.double().numpy()) <= unit / 2).all() and (np.abs(v) <= 127 * unit).all()


P = ctypes.c_void_p(256)
ARG, SHAPE, OK = _capi.PMX_ERR_ARG, _capi.PMX_ERR_SHAPE, _capi.PMX_OK


@pytest.mark.parametrize("suffix", ["", "_f16"])
def test_c_abi_refusals(suffix):
    lib = _capi.load()
    quantize, routed = getattr(lib, "pmx_rows8_quantize" + suffix), getattr(lib, "pmx_rows8_quantize_routed" + suffix)
    dequantize, swiglu = getattr(lib, "pmx_rows8_dequantize" + suffix), getattr(lib, "pmx_rows8_swiglu_bwd" + suffix)
    nt, fc1 = getattr(lib, "pmx_rows8_group_gemm_nt" + suffix), getattr(lib, "pmx_rows8_gemm_fc1_swiglu" + suffix)
    assert quantize(P, 8, 0, 1, 4, 8, 2, P, P, None) == ARG  # no such format
    assert quantize(P, 7, 0, 1, 4, 8, 0, P, P, None) == ARG  # rows overlap
    assert quantize(P, 8, 0, 1, -1, 8, 0, P, P, None) == ARG
    assert quantize(None, 8, 0, 1, 4, 8, 0, P, P, None) == ARG
    assert quantize(None, 8, 0, 1, 0, 8, 0, None, None, None) == OK
    assert quantize(P, 1 << 40, 0, 1 << 20, 1 << 20, 8, 0, P, P, None) == SHAPE
    assert routed(P, P, P, 1 << 30, 4, 8, P, P, P, P, None) == SHAPE
    assert routed(P, None, P, 4, 2, 8, P, P, P, P, None) == ARG
    assert routed(P, P, P, 4, 0, 8, P, P, P, P, None) == ARG
    assert dequantize(P, P, P, 4, 0, 8, 0, P, None) == ARG  # positions, but none per row
    assert dequantize(P, P, P, 1 << 30, 4, 8, 0, P, None) == SHAPE
    assert dequantize(P, P, None, 4, 0, 8, 5, P, None) == ARG
    assert dequantize(None, None, None, 0, 0, 8, 0, None, None) == OK
    assert swiglu(P, P, P, P, None, 4, 8, 4, 0, P, P, P, None) == ARG  # dw without row_src
    assert swiglu(P, P, P, P, P, 4, 8, 4, 0, P, P, None, None) == ARG
    assert swiglu(None, P, P, P, P, 4, 8, 4, 0, P, P, P, None) == ARG
    assert swiglu(P, P, P, P, P, 1 << 40, 1 << 30, 4, 0, P, P, P, None) == SHAPE
    assert nt(P, P, P, P, P, 0, 8, 8, 16, P, None) == ARG
    assert nt(P, P, P, P, P, 4096, 8, 8, 16, P, None) == ARG
    assert nt(P, P, P, P, P, 4, 8, 8, 24, P, None) == SHAPE  # K
    assert nt(P, P, P, P, P, 4, 8, 12, 16, P, None) == SHAPE  # N
    assert nt(P, P, P, P, P, 4, 8, 1 << 20, 1 << 12, P, None) == SHAPE  # 4 GiB per group
    assert nt(P, P, P, P, P, 4, 1 << 31, 8, 16, P, None) == SHAPE
    assert nt(ctypes.c_void_p(8), P, P, P, P, 4, 8, 8, 16, P, None) == SHAPE  # alignment
    assert nt(None, P, P, P, P, 4, 8, 8, 16, P, None) == ARG
    assert nt(None, None, None, None, None, 4, 0, 8, 16, None, None) == OK
    assert fc1(P, P, 8, None, P, P, P, 4, 16, 32, 32, P, P, P, None) == ARG  # rows without a map
    assert fc1(P, P, 8, P, P, P, P, 4, 16, 32, 24, P, P, P, None) == SHAPE  # I
    assert fc1(P, P, 1 << 20, P, P, P, P, 4, 16, 1 << 11, 32, P, P, P, None) == SHAPE  # 2 GiB of tokens
    assert fc1(P, P, 8, P, P, P, P, 4, 16, 32, 0, P, P, P, None) == ARG


def test_grids_past_one_launch_are_refused():
    """Of 2^32 threads or more a launch runs what is left modulo 2^32, and reports success."""
    lib = _capi.load()
    rows = 1 << 24  # blocks of 256 threads
    assert lib.pmx_rows8_quantize(P, 1, 0, 1, 32 * rows, 1, 0, P, P, None) == SHAPE
    assert lib.pmx_rows8_quantize(P, 8, 0, 32 * rows // 4, 4, 8, 0, P, P, None) == SHAPE  # a block per group
    assert lib.pmx_rows8_dequantize(P, P, None, 16 * rows, 0, 8, 0, P, None) == SHAPE
    assert lib.pmx_rows8_dequantize(P, P, P, 16 * rows, 4, 8, 0, P, None) == SHAPE
    assert lib.pmx_rows8_swiglu_bwd(P, P, P, P, P, 4 * rows, 8, 4, 0, P, P, P, None) == SHAPE
    ws = lib.pmx_rows8_layer_workspace_bytes  # the sum over a token's rows: 64 threads per token
    assert ws(4 * rows - 1, 1, 16, 16, 1) > 0 and ws(4 * rows, 1, 16, 16, 1) == 0


def _rows(shape, fmt="e4m3", dtype=BF):
    return rows8.Rows8(torch.zeros(shape, dtype=rows8.FORMATS[fmt]),
                       torch.full(rows8.scales_shape(shape), 127, dtype=torch.uint8), dtype)


def test_size_and_moving():
    q = _rows((3, 5, 600))
    assert q.shape == (3, 5, 600) and q.nbytes == 3 * 5 * (600 + 2 * 16)
    moved = q.to("cpu")
    assert moved.dtype == BF and torch.equal(moved.scales, q.scales) and moved.codes.shape == q.codes.shape


def test_wrappers_refuse_host_tensors():
    i32 = torch.zeros(3, dtype=torch.int32)
    for call in (
        lambda: rows8.quantize_rows(torch.zeros((2, 8), dtype=BF)),
        lambda: rows8.dequantize_rows(_rows((2, 8))),
        lambda: rows8.swiglu_bwd_rows8(torch.zeros((2, 8), dtype=BF), _rows((2, 16))),
        lambda: rows8.group_gemm_nt_rows8(_rows((2, 16)), _rows((2, 8, 16)), i32),
        lambda: rows8.gemm_fc1_swiglu_rows8(_rows((2, 16)), _rows((2, 32, 16)), i32),
    ):
        with pytest.raises(AssertionError, match="GPU tensors"):
            call()


def test_operand_checks():
    assert rows8._rows8("q", _rows((3, 4, 600)), 3) == BF
    assert rows8.scales_shape((4, 600)) == (2, 4, 16)
    q = _rows((4, 600))
    for bad, match in (
        (q.codes, "must be Rows8"),
        (rows8.Rows8(q.codes.float(), q.scales, BF), "codes must be"),
        (rows8.Rows8(q.codes, q.scales, torch.float32), "stand for"),
        (rows8.Rows8(q.codes, q.scales.int(), BF), "uint8"),
        (rows8.Rows8(q.codes, q.scales[:1], BF), "scales must be"),
        (_rows((3, 4, 600)), "2 dimensions"),
        (rows8.Rows8(q.codes.t().contiguous().t(), q.scales, BF), "contiguous"),
    ):
        with pytest.raises(AssertionError, match=match):
            rows8._rows8("q", bad, 2)
    with pytest.raises(AssertionError, match="e4m3 for a product"):
        rows8._e4m3("q", _rows((4, 600), "int8"), 2)
    with pytest.raises(ValueError, match="8-bit format"):
        rows8._format("e5m2")


def test_checkpoint_settings_are_checked():
    with pytest.raises(ValueError, match="activation checkpoint"):
        placemoe_amd.set_activation_checkpoint("fp8")
    assert placemoe_amd.set_activation_checkpoint("int8") is None
    assert placemoe_amd.set_activation_checkpoint(None) == "int8"
    z = torch.zeros((2, 16), dtype=BF)
    with pytest.raises(ValueError, match="activation checkpoint"):
        experts.expert_layer(z, z[:, :1], torch.zeros((2, 1), dtype=torch.int64), z, fc1_1_2_weight=z,
                             activation_checkpoint="bf16")


@pytest.fixture(scope="module")
def tiling(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path_factory.mktemp("rule") / "rows8_rule"
    subprocess.run([cxx, "-O2", "-std=c++17", f"-I{ROOT / 'placemoe_amd' / 'csrc'}", str(ROOT / "tests" / "rows8_rule_main.cpp"),
                    "-o", str(exe)], check=True)

    def ask(calls):
        """calls: (kind, rows, copies, N, K) -> tile heights, on 256 CUs."""
        lines = "\n".join(f"{('nt', 'fc1').index(k)} {' '.join(map(str, c))} 256" for k, *c in calls)
        out = subprocess.run([str(exe)], input=lines, check=True, capture_output=True, text=True).stdout
        return [int(x) for x in out.split()]

    return ask


def test_tiling_rule_takes_the_faster_one(tiling):
    measured = {  # us with 32 x 256 (or 32 x 64), 128 x 128 and 256 x 256 tiles
        ("nt", 640, 160, 1536, 2048): (91, 96, 121), ("nt", 10240, 160, 1536, 2048): (149, 105, 127),
        ("nt", 96000, 160, 1536, 2048): (857, 421, 355), ("nt", 2304, 12, 1000, 1104): (20, 13, 20),
        ("nt", 32000, 16, 4096, 7168): (2439, 1136, 848), ("nt", 64, 16, 4096, 7168): (80, 81, 105),
        ("fc1", 640, 160, 1536, 2048): (95, 119, 196), ("fc1", 10240, 160, 1536, 2048): (171, 131, 205),
        ("fc1", 96000, 160, 1536, 2048): (1146, 653, 606), ("fc1", 1536, 8, 1536, 2048): (36, 25, 51),
        ("fc1", 32000, 16, 4096, 7168): (2997, 1722, 1502),
    }
    for call, height in zip(measured, tiling(list(measured))):
        us = dict(zip((32, 128, 256, 0), measured[call] + measured[call][:1]))
        assert us[height] <= 1.05 * min(us.values()), (call, height)


# us on 32 x 64, 32 x 256, 128 x 128 and 256 x 256 tiles (log-normal counts with sigma 0.4)
FOUR_TILINGS = {
    ("nt", 1, 16, 7168, 2048): (10.8, 14.0, 14.9, 27.7), ("fc1", 1, 16, 7168, 2048): (14.4, 17.1, 20.8, 47.2),
    ("nt", 256, 8, 1536, 2048): (11.9, 13.9, 15.2, 27.9), ("fc1", 256, 8, 1536, 2048): (17.3, 17.9, 21.6, 48.3),
    ("nt", 640, 160, 1536, 2048): (89.2, 89.9, 97.1, 110.9), ("fc1", 640, 160, 1536, 2048): (92.4, 91.7, 116.5, 187.2),
    ("nt", 2560, 160, 1536, 2048): (99.9, 94.3, 99.8, 112.8), ("fc1", 2560, 160, 1536, 2048): (101.8, 94.2, 119.7, 189.7),
    ("nt", 5120, 160, 1536, 2048): (114.0, 106.4, 102.3, 114.6), ("fc1", 5120, 160, 1536, 2048): (123.9, 110.6, 124.1, 192.6),
    ("nt", 5120, 160, 2048, 768): (56.0, 55.3, 49.5, 67.4), ("fc1", 5120, 160, 2048, 768): (74.1, 64.3, 68.1, 112.6),
    ("nt", 10240, 160, 1536, 2048): (152.1, 146.3, 108.8, 117.2), ("fc1", 10240, 160, 1536, 2048): (178.4, 156.4, 133.9, 193.0),
    ("nt", 64, 16, 4096, 7168): (89.2, 78.2, 81.1, 92.3), ("fc1", 64, 16, 4096, 7168): (94.2, 79.6, 94.3, 150.6),
    ("nt", 256, 16, 4096, 7168): (91.8, 84.0, 85.6, 95.0), ("fc1", 256, 16, 4096, 7168): (96.2, 84.9, 96.2, 156.1),
    ("nt", 160, 160, 1536, 2048): (46.6, 54.5, 59.8, 79.9), ("fc1", 80, 160, 2048, 768): (26.4, 22.6, 30.2, 48.7),
}


def test_tiling_rule_on_four_tilings(tiling):
    """Each tiling at its own time: none of these calls loses more than 5% to the best one."""
    for call, height in zip(FOUR_TILINGS, tiling(list(FOUR_TILINGS))):
        us = dict(zip((0, 32, 128, 256), FOUR_TILINGS[call]))
        assert us[height] <= 1.05 * min(us.values()), (call, height, us)


def test_gpu_cases_reach_every_tiling(tiling):
    def heights(kind, cases):
        return {n: h for n, h in zip(cases, tiling([(kind, sum(c), len(c), N, K) for c, N, K in cases.values()]))}

    def even(cases):
        return {n: (c, N // 32 * 32, K) for n, (c, N, K) in cases.items()}

    assert 0 in heights("nt", test_gpu_rows8.LAYOUTS).values()
    assert set(heights("nt", test_gpu_rows8.WIDE).values()) == {32, 128}
    assert set(heights("fc1", even(test_gpu_rows8.WIDE)).values()) == {32, 128}
    assert 256 in heights("nt", test_gpu_rows8.LARGE).values()
    assert 256 in heights("fc1", even(test_gpu_rows8.LARGE)).values()
    # test_wide_fc1_equals_single_copies' other side
    alone = [("fc1", 1300, 1, 512, 112), ("fc1", 255, 1, 320, 272)]
    assert tiling(alone) == [0, 0]
    # one row of the same copy in calls of several tilings (test_a_row_depends_on_itself_and_its_copy_alone)
    calls = [(25600, 1), (2600, 1), (1, 1), (400, 200), (6400, 10)]
    assert tiling([("nt", *c, 248, 1104) for c in calls]) == [128, 0, 0, 32, 128]
    # test_every_tiling_gives_the_same_bits
    for kind, N in (("nt", 4096), ("fc1", 4096)):
        assert tiling([(kind, rows, 1, N, 1024) for rows in (4096, 1000, 10)]) == [256, 128, 0]
    few = [(k, sum(c), len(c), N, K) for k in ("nt", "fc1") for c, N, K in test_gpu_rows8.FEW.values()]
    assert tiling(few) == [0, 32] * 2


def test_layer_cases_reach_every_tiling(tiling):
    layers = test_gpu_rows8_layer.LAYERS.values()
    assert tiling([("nt", T * K, C, H, I) for T, K, C, H, I in layers]) == [0, 32, 128, 256, 256, 256]
    assert set(tiling([("fc1", T * K, C, 2 * I, H) for T, K, C, H, I in layers])) == {0, 32, 128, 256}


def test_layer_workspace(tiling):
    lib = _capi.load()
    ws = lib.pmx_rows8_layer_workspace_bytes
    A, H, I, C = 96 * 8, 2048, 768, 160
    assert ws(96, 8, H, I, C) >= 96 * H + A * I + 2 * A * H + lib.pmx_route_workspace_bytes(A, C)
    assert ws(96, 8, H + 8, I, C) == 0 and ws(96, 0, H, I, C) == 0 and ws(96, 8, H, I, 5000) == 0
    assert ws(1 << 20, 8, 1 << 12, I, C) == 0  # 4 GiB of tokens
    layer = lib.pmx_rows8_layer
    args = [P] * 5 + [0, 1, C] + [P] * 4 + [96, 8, H, I, C, P, None]
    assert layer(*args, P, ws(96, 8, H, I, C) - 1, None, None) == ARG
    assert layer(*args, None, 1 << 40, None, None) == ARG
    assert layer(*args, ctypes.c_void_p(8), 1 << 40, None, None) == SHAPE
    assert layer(None, *args[1:], P, 1 << 40, None, None) == ARG
    assert layer(*args[:15], 100, *args[16:], P, 1 << 40, None, None) == SHAPE
