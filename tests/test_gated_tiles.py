"""The rule takes the tiles that tests/test_gpu_gated_tiles.py means to run."""

import shutil
import subprocess
from pathlib import Path

import pytest

from tests.test_gpu_gated_tiles import TILES


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path_factory.mktemp("rule") / "gated_rule"
    subprocess.run([cxx, "-O1", "-std=c++17", str(Path(__file__).with_name("gated_rule_main.cpp")), "-o", str(exe)], check=True)

    def ask(products):
        """products: (kind, rows, N, K) -> heights of their tiles."""
        asked = "\n".join(f"tiling {k} {r} {n} {d}" for k, r, n, d in products)
        return [int(v) for v in subprocess.run([str(exe)], input=asked, check=True, capture_output=True, text=True).stdout.split()]

    return ask


def _products(T, H, I, N):
    return (0, T, 2 * I, H), (1, T, N, I), (2, T, H, 2 * I), (3, T, I, N)


def test_tiles_of_the_sizes(rule):
    run = set()
    for size, heights in TILES.items():
        assert tuple(rule(_products(*size))) == heights, size
        for (kind, rows, N, K), height in zip(_products(*size), heights):
            columns = N // 2 % 128 if kind == 0 else N % 256
            if height > 64 and columns and rows % height:
                run.add((kind, height, K % 64 == 0))
    assert run >= {(k, 128, whole) for k in range(4) for whole in (True, False)}
    assert run >= {(k, 256, True) for k in range(4)} | {(1, 256, False), (2, 256, False)}
    for kind in (0, 3):  # the four-wave kernel: 1, 15, 17 and 33 rows in the last 64
        assert {s[0] % 64 for s, h in TILES.items() if h[kind] == 256} == {1, 15, 17, 33}


def test_no_256_rows_with_a_short_last_k_tile_for_fc1_and_fc2_dgrad(rule):
    """Their 256-row kernel takes whole K-tiles alone."""
    import random

    rng = random.Random(7)
    calls = [(rng.choice((0, 3)), int(2 ** rng.uniform(5, 24)), 8 * int(2 ** rng.uniform(0, 11)), 8 * int(2 ** rng.uniform(0, 11)))
             for _ in range(4000)]
    calls = [(k, r, n, d + 8 if d % 64 == 0 else d) for k, r, n, d in calls]
    assert set(rule(calls)) == {64, 128}
    whole = [(k, r, n, (d + 63) // 64 * 64) for k, r, n, d in calls]
    assert set(rule(whole)) == {64, 128, 256}


def test_no_kernel_is_built_that_no_call_reaches(tmp_path):
    """The gated build has the eight-wave kernel for fc2, fc1's dgrad and the weight gradients, not for the other two."""
    from placemoe_amd import build
    from tests.test_build_resources import _compile_remarks

    names = [r["name"] for r in _compile_remarks(build.CSRC / "grouped_gemm.hip", tmp_path, build.EXTRA_OBJECTS["grouped_gemm.gated"][1])]
    eight = {n.split("grouped_gemm_kernelILi")[1][0] for n in names if "119grouped_gemm_kernelILi" in n}
    four = {n.split("grouped_gemm_w4_kernelILi")[1][0] for n in names if "grouped_gemm_w4_kernelILi" in n}
    assert (eight, four) == ({"1", "2", "4"}, {"0", "3", "4"}), names


def test_kernels_for_few_tokens_are_held_to_registers(tmp_path):
    """fc1 and fc2 of up to 16, 32 and 64 tokens in both types; the build refuses one that spills."""
    from placemoe_amd import build
    from tests.test_build_resources import _compile_remarks

    few = [r for r in _compile_remarks(build.CSRC / "gated_ffn.hip", tmp_path) if build.RESOURCE_CHECKED["gated_ffn.hip"].search(r["name"])]
    assert len(few) == 12
    build.check_no_scratch(few, build.RESOURCE_CHECKED["gated_ffn.hip"], "gated_ffn.hip")
    with pytest.raises(RuntimeError, match="spill"):
        build.check_no_scratch([dict(few[0], vgpr_spill=1), *few[1:]], build.RESOURCE_CHECKED["gated_ffn.hip"], "gated_ffn.hip")
