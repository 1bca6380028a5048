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
