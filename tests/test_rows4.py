"""Rows in 4 bits without a GPU: the oracle's own properties, the C ABI's
refusals, and the wrappers' checks (all before any launch)."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import rows4_oracle as O
from placemoe_amd import _capi, rows4, rows8
from tests import test_gpu_rows4

ROOT = Path(__file__).resolve().parent.parent
BF = torch.bfloat16
P = ctypes.c_void_p(256)
ARG, SHAPE, OK = _capi.PMX_ERR_ARG, _capi.PMX_ERR_SHAPE, _capi.PMX_OK


@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_oracle_is_within_half_a_step_of_the_smallest_power(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((40, 100), generator=g) * torch.logspace(-6, 4, 40).unsqueeze(1)).to(dtype)
    x[3] = 0
    v, scales = O.quantize(x)
    e = scales.permute(1, 0, 2).reshape(40, -1).to(torch.int64) - 127
    unit = torch.exp2(e.double()).repeat_interleave(32, 1)[:, :100].numpy()
    y = np.abs(x.double().numpy()) / unit
    step = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))
    assert (np.abs(v - x.double().numpy()) <= step / 2 * unit).all()
    most = torch.nn.functional.pad(x.double().abs(), (0, 28)).view(40, 4, 32).amax(-1)
    u = torch.exp2(e[:, :4].double())
    assert (most < 7 * u).all() and ((most >= 3.5 * u) | (most == 0)).all()
    assert (e[:, 4:] == 0).all()


def test_oracle_ties_and_the_end_of_the_range():
    x = torch.zeros((2, 32), dtype=BF)
    x[0, :9] = torch.tensor([6.75, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75])
    x[1, 0] = 7.0  # as far from 6 as from 8: the next power of two
    v, scales = O.quantize(x)
    assert v[0, :9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -1.0]
    assert scales[0, 0, 0] == 127 and scales[0, 1, 0] == 128 and v[1, 0] == 8.0


@pytest.mark.parametrize("suffix", ["", "_f16"])
def test_c_abi_refusals(suffix):
    lib = _capi.load()
    quantize, dequantize = getattr(lib, "pmx_rows4_quantize" + suffix), getattr(lib, "pmx_rows4_dequantize" + suffix)
    nt, fc1 = getattr(lib, "pmx_rows4_group_gemm_nt" + suffix), getattr(lib, "pmx_rows4_gemm_fc1_swiglu" + suffix)
    assert quantize(P, 7, 0, 1, 4, 8, P, P, None) == ARG  # rows overlap
    assert quantize(P, 8, 0, 1, -1, 8, P, P, None) == ARG
    assert quantize(None, 8, 0, 1, 4, 8, P, P, None) == ARG
    assert quantize(None, 8, 0, 1, 0, 8, None, None, None) == OK
    assert quantize(P, 1 << 40, 0, 1 << 20, 1 << 20, 8, P, P, None) == SHAPE
    assert quantize(P, 1, 0, 1, 1 << 29, 1, P, P, None) == SHAPE  # 2^32 threads
    assert dequantize(P, P, 1, -4, 8, P, None) == ARG
    assert dequantize(P, None, 1, 4, 8, P, None) == ARG
    assert dequantize(None, None, 0, 4, 8, None, None) == OK
    assert dequantize(P, P, 1, 1 << 29, 1, P, None) == SHAPE
    for bits in (8, 4):
        assert nt(P, P, bits, P, P, P, 0, 8, 8, 32, P, None) == ARG
        assert nt(P, P, bits, P, P, P, 4096, 8, 8, 32, P, None) == ARG
        assert nt(P, P, bits, P, P, P, 4, 8, 8, 48, P, None) == SHAPE  # K
        assert nt(P, P, bits, P, P, P, 4, 8, 12, 32, P, None) == SHAPE  # N
        assert nt(P, P, bits, P, P, P, 4, 8, 1 << 20, 1 << 13, P, None) == SHAPE  # 4 GiB per group
        assert nt(P, P, bits, P, P, P, 4, 1 << 31, 8, 32, P, None) == SHAPE
        for k in range(6):
            at = [P] * 6
            at[k] = ctypes.c_void_p(264)  # alignment (offsets are int32: any)
            a, a_s, b, b_s, off, c = at
            assert k == 4 or nt(a, a_s, bits, b, b_s, off, 4, 8, 8, 32, c, None) == SHAPE, k
            at[k] = None
            a, a_s, b, b_s, off, c = at
            assert nt(a, a_s, bits, b, b_s, off, 4, 8, 8, 32, c, None) == ARG, k
        assert nt(None, None, bits, None, None, None, 4, 0, 8, 32, None, None) == OK
    for bits in (0, 5, 16, -4):
        assert nt(P, P, bits, P, P, P, 4, 8, 8, 32, P, None) == ARG
    assert fc1(P, P, 8, None, P, P, P, 4, 16, 32, 32, P, P, P, None) == ARG  # rows without a map
    assert fc1(P, P, 8, P, P, P, P, 4, 16, 32, 24, P, P, P, None) == SHAPE  # I
    assert fc1(P, P, 8, P, P, P, P, 4, 16, 48, 32, P, P, P, None) == SHAPE  # H
    assert fc1(P, P, 1 << 20, P, P, P, P, 4, 16, 1 << 11, 32, P, P, P, None) == SHAPE  # 2 GiB of tokens
    assert fc1(P, P, 8, P, P, P, P, 4, 16, 32, 0, P, P, P, None) == ARG


def test_layer_sizes():
    ws = _capi.load().pmx_rows4_layer_workspace_bytes
    assert ws(1, 8, 2048, 768, 160) > 0
    assert ws(1, 8, 2048 + 16, 768, 160) == 0 and ws(1, 8, 2048, 768 + 16, 160) == 0
    assert ws(1, 8, 2048, 768, 2049) == 0 and ws(1, 0, 2048, 768, 160) == 0
    assert ws(1 << 21, 1, 2048, 768, 160) == 0  # 2 GiB or more of tokens
    # twice the rows of an 8-bit matrix: 2 GiB are as many bytes
    assert ws(1, 1, 32768, 65504, 1) > 0 and _capi.load().pmx_rows8_layer_workspace_bytes(1, 1, 32768, 65504, 1) == 0


def _rows(shape, dtype=BF):
    return rows4.Rows4(torch.zeros((*shape[:-1], (shape[-1] + 1) // 2), dtype=torch.uint8),
                       torch.full(rows8.scales_shape(shape), 127, dtype=torch.uint8), shape[-1], dtype)


def _rows8(shape, dtype=BF):
    return rows8.Rows8(torch.zeros(shape, dtype=torch.float8_e4m3fn), torch.full(rows8.scales_shape(shape), 127, dtype=torch.uint8), dtype)


def test_size_and_moving():
    q = _rows((3, 5, 601))
    assert q.shape == (3, 5, 601) and q.nbytes == 3 * 5 * (301 + 2 * 16)
    moved = q.to("cpu")
    assert moved.dtype == BF and torch.equal(moved.scales, q.scales) and moved.shape == q.shape


def test_wrappers_refuse_host_tensors():
    i32 = torch.zeros(3, dtype=torch.int32)
    w = rows4.Experts4(_rows((2, 64, 32)), _rows((2, 32, 32)))
    for call in (
        lambda: rows4.quantize_rows4(torch.zeros((2, 8), dtype=BF)),
        lambda: rows4.dequantize_rows4(_rows((2, 8))),
        lambda: rows4.group_gemm_nt_rows4(_rows8((2, 32)), _rows((2, 8, 32)), i32),
        lambda: rows4.group_gemm_nt_rows4(_rows((2, 32)), _rows((2, 8, 32)), i32),
        lambda: rows4.gemm_fc1_swiglu_rows4(_rows8((2, 32)), _rows((2, 32, 32)), i32),
        lambda: placemoe_amd.expert_layer_rows4(torch.zeros((2, 32), dtype=BF), torch.zeros((2, 1), dtype=BF),
                                                torch.zeros((2, 1), dtype=torch.int64), w),
    ):
        with pytest.raises(AssertionError, match="GPU tensors"):
            call()


# us on 32 x 64, 32 x 256, 128 x 128 and 256 x 256 tiles (log-normal counts with sigma 0.4):
# NT of 8-bit rows, NT of 4-bit rows, fc1
MEASURED = {
    (64, 160, 1536, 2048): ((20, 23, 26, 50), (18, 20, 21, 34), (30, 32, 39, 88)),
    (640, 160, 1536, 2048): ((45, 44, 58, 95), (40, 42, 45, 64), (67, 59, 103, 170)),
    (1600, 160, 1536, 2048): ((46, 46, 60, 95), (41, 42, 46, 64), (68, 59, 103, 171)),
    (5120, 160, 1536, 2048): ((67, 62, 64, 97), (46, 50, 47, 66), (97, 84, 105, 172)),
    (20480, 160, 1536, 2048): ((192, 162, 101, 115), (112, 104, 64, 81), (284, 228, 162, 194)),
    (81920, 160, 1536, 2048): ((684, 559, 296, 280), (392, 354, 192, 188), (1035, 811, 516, 505)),
    (1, 16, 4096, 7168): ((20, 26, 30, 70), (12, 18, 20, 42), (31, 42, 52, 132)),
    (256, 16, 4096, 7168): ((44, 38, 46, 74), (39, 38, 39, 46), (61, 46, 88, 139)),
    (16000, 16, 4096, 7168): ((996, 830, 436, 409), (550, 490, 275, 253), (1603, 1276, 820, 763)),
}


# ... and on 256 x 256 ones with the short rests on 128 x 128 ones, in the same order
APART = {
    (16000, 160, 1536, 2048): ((94.8, 109.2, 92.5), (173.9, 200.8, 150.8)),
    (40960, 160, 1536, 2048): ((163.8, 175.4, 152.0), (306.7, 293.9, 260.6)),
    (81920, 160, 1536, 2048): ((312.6, 283.8, 269.9), (535.7, 486.0, 465.8)),
    (65600, 160, 2048, 768): ((135.4, 149.1, 135.8), (259.4, 242.1, 219.8)),
    (81920, 160, 2048, 768): ((166.7, 172.2, 153.7), (313.3, 284.8, 261.0)),
    (5760, 16, 4096, 7168): ((181.5, 177.7, 208.2), (336.4, 317.8, 381.8)),
    (16000, 16, 4096, 7168): ((453.8, 409.7, 385.9), (823.1, 769.9, 710.0)),
    (2048, 8, 2048, 1024): ((12.2, 17.9, 26.1), (19.1, 29.3, 40.8)),
    (179200, 256, 512, 512): ((80.2, 82.6, 85.1), (139.8, 136.4, 133.7)),
    (32000, 32, 2816, 4096): ((362.0, 338.8, 329.2), (669.2, 647.4, 619.8)),
}


@pytest.fixture(scope="module")
def tiling(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path_factory.mktemp("rule") / "rows4_rule"
    subprocess.run([cxx, "-O2", "-std=c++17", f"-I{ROOT / 'placemoe_amd' / 'csrc'}", str(ROOT / "tests" / "rows4_rule_main.cpp"),
                    "-o", str(exe)], check=True)

    def ask(calls):
        """calls: (line, rows, copies, N, K) -> tile heights, on 256 CUs."""
        asked = "\n".join(f"{' '.join(map(str, c))} 256" for c in calls)
        return [int(x) for x in subprocess.run([str(exe)], input=asked, check=True, capture_output=True, text=True).stdout.split()]

    return ask


def test_tiling_rule_takes_a_fast_one(tiling):
    """None of these calls loses more than a twelfth to its best tiling."""
    calls = [(line, call, us) for call, lines in MEASURED.items() for line, us in zip((0, 2, 1), lines)]
    taken = set()
    for (line, call, us), height in zip(calls, tiling([(line, *call) for line, call, _ in calls])):
        taken.add(height)
        if height == 384:  # timed in APART
            assert min(us) in us[2:]
            continue
        t = dict(zip((0, 32, 128, 256), us))
        assert t[height] <= 13 / 12 * min(us), (line, call, height, t)
    assert taken == {0, 32, 128, 256, 384}


def test_rests_are_apart_where_that_is_fast(tiling):
    calls = [(line, call, us) for call, lines in APART.items() for line, us in enumerate(lines)]
    apart = 0
    for (line, call, us), height in zip(calls, tiling([(line, *call) for line, call, _ in calls])):
        t = dict(zip((128, 256, 384), us))
        # where copies have fewer than 256 rows, rests are not looked at
        assert t[height] <= (13 / 12 if call[0] >= 256 * call[1] else 1.25) * min(us), (line, call, height, t)
        apart += height == 384
    assert apart >= 8
    counts, N, K = test_gpu_rows4.RESTS
    assert tiling([(line, 8 + sum(counts), len(counts), N, K) for line in (0, 1)]) == [384, 384]
