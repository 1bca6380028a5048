"""The rule takes the tilings that tests/test_gpu_rows4_tiles.py means to run."""

from tests.test_gpu_rows4_tiles import LAYERS
from tests.test_rows4 import tiling  # noqa: F401  (a fixture)


def test_tilings_of_the_layers(tiling):  # noqa: F811
    for (T, K, C, H, I), heights in LAYERS.items():
        assert tuple(tiling([(1, T * K, C, 2 * I, H), (0, T * K, C, H, I)])) == heights, (T, K, C, H, I)
    for product in (0, 1):
        assert {h[product] for h in LAYERS.values()} == {0, 32, 128, 256, 384}
