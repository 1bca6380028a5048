"""Rows in 8 bits on the GPU against the 64-bit oracle.

Tolerances, from the arithmetic:

* writing and reading back are exact by definition (one rounding to nearest
  even, powers of two): codes, exponents and values must be equal;
* SwiGLU backward: one rounding of each result (half a step, eps / 2), beside
  fp32 arithmetic whose sigmoid is good to 2^-18 for |gate| <= 32 (the
  exponential's argument, up to 46 in base 2, is rounded to 2^-19);
* products of small integers, whose every sum is exact in fp32, must be equal
  after the one rounding; products of arbitrary values carry up to 2^-11 of
  the largest product of each 64 columns (a matrix instruction adds its 64
  products to about 2^-12 of the largest, measured) and the result's half step.
"""

import math

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import moe_oracle
from oracle import rows8_oracle as O
from placemoe_amd import _capi, experts, kernels, rows8
from placemoe_amd.workloads import make_workload
from tests.helpers import BF16_REL, assert_bf16_close, assert_exact

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
SUBNORMAL = {BF: 2.0**-133, F16: 2.0**-24}


def _randn(shape, seed, dtype=BF, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _same(got, want, name):
    """Equal as 64-bit values, NaN where NaN."""
    got = got.detach().double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    bad = np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))
    assert bad.size == 0, f"{name}: {len(bad)} differ, first at {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


def _check_written(q, x, fmt, name):
    v, scales = O.quantize(x, fmt)
    assert torch.equal(q.scales.cpu(), scales), f"{name}: exponents"
    _same(O.values(q.codes.cpu(), q.scales.cpu()), v, name)
    return v


def _spiky(shape, seed, dtype):
    """Blocks of every size, zeros, one loud column, values at the edges of the type."""
    R, N = shape
    x = _randn(shape, seed, torch.float32) * torch.logspace(-7 if dtype == F16 else -30, 4, R).unsqueeze(1)
    if N > 3:
        x[:, 3] *= 100
    x[R // 2] = 0
    x = x.to(dtype)
    info = torch.finfo(dtype)
    x[0, N // 2] = info.max
    x[-1, :] = info.smallest_normal
    x[-1, N - 1] = info.smallest_normal * 2.0 ** (-7 if dtype == BF else -10)  # the smallest subnormal
    return x


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("R,N", [(1, 1), (1, 8), (3, 31), (5, 33), (33, 512), (31, 513), (65, 1411), (4, 2048), (40, 100)])
def test_written_and_read_back_exactly(cuda, R, N, fmt, dtype):
    print(f"rows8 {R}x{N} {fmt} {dtype}", flush=True)
    x = _spiky((R, N), R * 31 + N, dtype)
    q = rows8.quantize_rows(x.to(cuda), fmt)
    assert q.shape == (R, N) and q.dtype == dtype and q.codes.dtype == rows8.FORMATS[fmt]
    v = _check_written(q, x, fmt, f"{R}x{N}")
    most = float(torch.finfo(dtype).max)
    _same(rows8.dequantize_rows(q), np.clip(v, -most, most), "read back")


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_values_that_are_not_finite(cuda, fmt, dtype):
    x = _randn((6, 96), 5, dtype)
    x[0, 3], x[1, 40], x[2, 95] = math.inf, -math.inf, math.nan
    x[3, 32:64] = math.inf  # a block with nothing finite
    x[4] = math.nan
    q = rows8.quantize_rows(x.to(cuda), fmt)
    _check_written(q, x, fmt, "not finite")
    back = rows8.dequantize_rows(q).cpu()
    assert torch.equal(back.isnan(), ~x.isfinite())


def test_ties_round_to_even(cuda):
    # beside 2^0 (the block holds 448): 17 and 19 lie halfway between multiples of 2
    x = torch.zeros((1, 32), dtype=BF)
    x[0, :6] = torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0**-10, 3 * 2.0**-10])
    back = rows8.dequantize_rows(rows8.quantize_rows(x.to(cuda))).cpu()[0, :6]
    assert back.tolist() == [448.0, 16.0, 20.0, -16.0, 0.0, 2.0**-8]
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5])
    back = rows8.dequantize_rows(rows8.quantize_rows(x.to(cuda), "int8")).cpu()[0, :6]
    assert back.tolist() == [127.0, 0.0, 2.0, 2.0, 0.0, -2.0]


def test_strided_unaligned_and_grouped_rows(cuda):
    big = _randn((70, 1500), 6)
    dev = big.to(cuda)
    for part in (slice(0, 700), slice(1, 702), slice(3, 4)):
        _check_written(rows8.quantize_rows(dev[:, part]), big[:, part], "e4m3", f"columns {part}")
    _check_written(rows8.quantize_rows(dev[::3, 5:600]), big[::3, 5:600], "e4m3", "every third row")
    one = rows8.quantize_rows(dev.view(-1)[7: 7 + 2 * 515].view(2, 515))
    _check_written(one, big.view(-1)[7: 7 + 2 * 515].view(2, 515), "e4m3", "odd address")
    w = _randn((3, 37, 130), 7)
    q = rows8.quantize_rows(w.to(cuda))
    assert q.scales.shape == (3, 1, 37, 16)
    for g in range(3):
        v, s = O.quantize(w[g], "e4m3")
        assert torch.equal(q.scales[g].cpu(), s)
        _same(O.values(q.codes[g].cpu(), q.scales[g].cpu()), v, f"group {g}")
    for bad in (dev.t(), dev[:, ::2], dev[0].expand(4, 1500), w.to(cuda).transpose(1, 2)):
        with pytest.raises(AssertionError):
            rows8.quantize_rows(bad)
    with pytest.raises(AssertionError):
        rows8.quantize_rows(dev.float())


def test_nothing_to_write(cuda):
    for shape in ((0, 64), (5, 0), (0, 0), (0, 4, 64), (2, 0, 64)):
        q = rows8.quantize_rows(torch.empty(shape, dtype=BF, device=cuda))
        assert q.shape == shape and tuple(q.scales.shape) == rows8.scales_shape(shape)
        if len(shape) == 2:
            assert rows8.dequantize_rows(q).shape == shape


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,K,N", [(1, 1, 40), (37, 2, 1000), (50, 8, 515), (7, 4, 16)])
def test_read_back_into_copies_rows(cuda, T, K, N, dtype):
    print(f"read back T={T} K={K} N={N}", flush=True)
    q = rows8.quantize_rows(_randn((T, N), T, dtype).to(cuda), "int8")
    pos = torch.randperm(T * K, generator=torch.Generator().manual_seed(T)).to(torch.int32).view(T, K).to(cuda)
    assert_exact(rows8.dequantize_rows(q, pos), kernels.moe_scatter(rows8.dequantize_rows(q), pos), "rows")


def test_positions_outside_are_skipped(cuda):
    q = rows8.quantize_rows(_randn((4, 64), 1).to(cuda))
    pos = torch.tensor([[0], [9], [-1], [3]], dtype=torch.int32, device=cuda)
    out = torch.full((4, 64), 7.0, dtype=BF, device=cuda)
    _capi.call("pmx_rows8_dequantize", q.codes.data_ptr(), q.scales.data_ptr(), pos.data_ptr(), 4, 1, 64, 0, out.data_ptr(),
               torch.cuda.current_stream().cuda_stream)
    want = rows8.dequantize_rows(q)
    assert_exact(out[[0, 3]], want[[0, 3]], "named rows")
    assert (out[[1, 2]] == 7.0).all()


def test_routed_rows(cuda):
    T, K, H = 75, 3, 528
    x, w = _randn((T, H), 8), torch.rand((T, K), generator=torch.Generator().manual_seed(9)).to(BF)
    pos = torch.randperm(T * K, generator=torch.Generator().manual_seed(10)).to(torch.int32).view(T, K)
    q, row_token, row_w = rows8.quantize_rows_routed(x.to(cuda), pos.to(cuda), w.to(cuda))
    _check_written(q, x, "e4m3", "tokens")
    want = torch.empty(T * K, dtype=torch.int64)
    want[pos.view(-1).long()] = torch.arange(T * K)
    assert_exact(row_token, want // K, "row_token")
    assert_exact(row_w, w.view(-1)[want], "row_w")


# ---------------------------------------------------------------------------
# SwiGLU backward
# ---------------------------------------------------------------------------


def _near(got, exact, slack, dtype, name):
    """Within half a step of the exact value and the slack."""
    got = got.detach().double().cpu().numpy()
    tol = np.abs(exact) * torch.finfo(dtype).eps / 2 + slack + SUBNORMAL[dtype]
    off = np.abs(got - exact) - tol * 1.0001
    assert np.isfinite(got).all(), name
    assert (off <= 0).all(), f"{name}: {np.abs(got - exact).max()} off, {off.max()} over its tolerance"


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("R,I", [(1, 1), (2, 16), (5, 33), (64, 96), (33, 513), (130, 1411), (7, 2048), (300, 100)])
def test_swiglu_backward_from_8_bits(cuda, R, I, fmt, dtype):
    print(f"swiglu_bwd_rows8 {R}x{I} {fmt} {dtype}", flush=True)
    gu = _randn((R, 2 * I), R + I, torch.float32, 3.0).clamp(-30, 30).to(dtype)
    d = _randn((R, I), R + I + 1, dtype)
    w = (0.05 + torch.rand(R, generator=torch.Generator().manual_seed(I))).to(dtype)
    src = torch.randperm(R, generator=torch.Generator().manual_seed(R)).to(torch.int32)
    q = rows8.quantize_rows(gu.to(cuda), fmt)
    dg1, act_w, dw = rows8.swiglu_bwd_rows8(d.to(cuda), q, w.to(cuda), src.to(cuda), R)
    v = O.values(q.codes.cpu(), q.scales.cpu())
    dn, wn = d.double().numpy(), w.double().numpy()
    e_dg1, e_act, e_dw = O.swiglu_backward(dn, v, wn)
    g, u = v[:, :I], v[:, I:]
    sig = 1 / (1 + np.exp(-g))
    size = np.abs(np.concatenate([dn * wn[:, None] * u * (sig + np.abs(g) * sig), dn * wn[:, None] * g * sig], 1))
    _near(dg1, e_dg1, size * 2.0**-17, dtype, "dG1")
    _near(act_w, e_act, np.abs(e_act) * 2.0**-17, dtype, "act_w")
    terms = np.abs(dn * g * sig * u).sum(1)
    got_dw = torch.empty(R, dtype=dtype)
    got_dw = dw.cpu()[src.long()]
    _near(got_dw, e_dw, terms * (2.0**-17 + (I + 8) * 2.0**-24), dtype, "dw")
    # without weights: ones
    dg1, act, none = rows8.swiglu_bwd_rows8(d.to(cuda), q)
    e_dg1, e_act, _ = O.swiglu_backward(dn, v, np.ones(R))
    assert none is None
    _near(dg1, e_dg1, size / wn[:, None] * 2.0**-17, dtype, "dG1 unweighted")
    _near(act, e_act, np.abs(e_act) * 2.0**-17, dtype, "act")


def test_swiglu_gradient_against_differences(cuda):
    """d/dg and d/du of sum(d * silu(g) * u) in 64 bits, by central differences."""
    R, I = 6, 40
    q = rows8.quantize_rows(_randn((R, 2 * I), 1).to(cuda))
    d = _randn((R, I), 2).to(cuda)
    dg1, _, _ = rows8.swiglu_bwd_rows8(d, q)
    v, dn = O.values(q.codes.cpu(), q.scales.cpu()), d.double().cpu().numpy()

    def f(x):  # per element of (g | u), only its own term changes
        g, u = x[:, :I], x[:, I:]
        return dn * g / (1 + np.exp(-g)) * u

    h = 1e-5
    num = np.empty_like(v)
    for half in (slice(0, I), slice(I, 2 * I)):
        up, down = v.copy(), v.copy()
        up[:, half] += h
        down[:, half] -= h
        num[:, half] = (f(up) - f(down)) / (2 * h)
    # differences are good to h^2 times a third derivative of a few units, and 1e-16 / h
    _near(dg1, num, np.abs(np.concatenate([dn, dn], 1)) * (2.0**-16 + 1e-8) * (1 + np.abs(v).max()), BF, "gradient")


def test_swiglu_extreme_gates(cuda):
    """Saturated gates: silu -> 0 or g, no NaN from infinities on the way; a NaN stays in its row."""
    gu = torch.zeros((3, 64), dtype=BF)
    gu[0, :32] = torch.tensor([-3e38, -1e4, -100.0, -90.0, 100.0, 1e4] + [0.0] * 26)
    gu[0, 32:] = 1.0
    gu[1, :] = 2.0
    gu[1, 5] = math.nan
    gu[2, :] = 0.5
    q = rows8.quantize_rows(gu.to(cuda))
    d = torch.ones((3, 32), dtype=BF, device=cuda)
    dg1, act, _ = rows8.swiglu_bwd_rows8(d, q)
    assert dg1[0].isfinite().all() and act[0].isfinite().all() and dg1[2].isfinite().all()
    v = rows8.dequantize_rows(q)[0, :6].float()
    assert torch.equal(act[0, :6].float()[v <= -1e4], torch.zeros_like(v[v <= -1e4]))
    assert torch.equal(act[0, 5:6].float(), v[5:6])
    assert dg1[1].isnan().nonzero().view(-1).tolist() == [5, 37] and act[1].isnan().nonzero().view(-1).tolist() == [5]


def test_swiglu_skips_unnamed_weights(cuda):
    R, I, A = 8, 40, 12
    q = rows8.quantize_rows(_randn((R, 2 * I), 3).to(cuda))
    d, w = _randn((R, I), 4).to(cuda), torch.ones(R, dtype=BF, device=cuda)
    src = torch.tensor([0, 2, 4, 6, 8, 10, 12, -1], dtype=torch.int32, device=cuda)
    dg1, act = torch.empty((R, 2 * I), dtype=BF, device=cuda), torch.empty((R, I), dtype=BF, device=cuda)
    dw = torch.full((A,), 7.0, dtype=BF, device=cuda)
    _capi.call("pmx_rows8_swiglu_bwd", d.data_ptr(), q.codes.data_ptr(), q.scales.data_ptr(), w.data_ptr(), src.data_ptr(), R, I,
               A, 0, dg1.data_ptr(), act.data_ptr(), dw.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert (dw.cpu()[1::2] == 7.0).all() and (dw.cpu()[::2] != 7.0).all()


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------


def _offsets(counts):
    return torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32)


def _ints(shape, seed, dtype=BF):
    """Small integers times a power of two per block of 32 columns: exact in 8 bits."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, shape, generator=g).float()
    nb = -(-shape[-1] // 32)
    p = torch.exp2(torch.randint(0, 3, (*shape[:-1], nb), generator=g).float()).repeat_interleave(32, -1)[..., : shape[-1]]
    return (x * p).to(dtype)


LAYOUTS = {
    "one row": ([1], 8, 16),
    "one row each": ([1] * 5, 40, 48),
    "empty groups": ([0, 3, 0, 0, 17, 0], 64, 128),
    "only the last": ([0, 0, 0, 33], 256, 512),
    "ragged": ([5, 31, 32, 33, 64, 1, 0, 70], 200, 1104),
    "long K": ([9, 40], 72, 2320),
    "mid": ([130, 61, 0, 255, 128], 328, 144),
    "mid wide": ([100, 90], 1000, 656),
    "large": ([256, 257, 511, 300], 264, 272),
    "large odd": ([700, 0, 301], 520, 1040),
    "many groups": ([2, 0, 1] * 400, 16, 32),
    "one K-tile": ([300, 100, 0, 40], 264, 112),
    "one full K-tile": ([70, 33], 136, 128),
    "two K-tiles": ([70, 33], 136, 144),
    "three K-tiles": ([150, 33], 136, 384),
}

# the same with more tiles than the narrowest tiling has blocks: the wider ones
WIDE = {
    "ragged": ([5, 31, 32, 33, 64, 1, 0, 70, 129, 40] * 30, 200, 1104),
    "ragged few": ([5, 31, 2, 33, 4, 1, 0, 7] * 60, 232, 1104),
    "short K": ([70, 0, 33, 150] * 60, 136, 112),
    "two K-tiles": ([70, 33, 90] * 60, 264, 144),
    "three K-tiles": ([150, 33] * 100, 136, 384),
    "odd N": ([130, 61, 0, 255, 128] * 30, 328, 272),
    "deep": ([90, 40] * 60, 264, 2320),
    "many rows": ([1300, 700] * 24, 520, 112),
}


@pytest.mark.parametrize("name", WIDE)
def test_wide_products_of_integers_are_exact(cuda, name):
    counts, N, K = WIDE[name]
    print(f"rows8 wide {name}", flush=True)
    M, G = sum(counts), len(counts)
    a, b = _ints((M, K), 1).to(cuda), _ints((G, N, K), 2).to(cuda)
    off = _offsets(counts)
    got = rows8.group_gemm_nt_rows8(rows8.quantize_rows(a), rows8.quantize_rows(b), off.to(cuda))
    want = torch.cat([(a[off[g]:off[g + 1]].double() @ b[g].double().t()).float().to(BF) for g in range(G)])
    assert_exact(got, want, name)


@pytest.mark.parametrize("name", WIDE)
def test_wide_fc1_equals_single_copies(cuda, name):
    """A copy's rows among those of many others, and alone on narrow tiles (tested against 64 bits): the same bits."""
    counts, N, K = WIDE[name]
    print(f"rows8 wide fc1 {name}", flush=True)
    A, G, I, T = sum(counts), len(counts), N // 32 * 16, 333
    x = rows8.quantize_rows(_randn((T, K), 3).to(cuda))
    w = rows8.quantize_rows(_randn((G, 2 * I, K), 4, std=0.06).to(cuda))
    token = torch.randint(0, T, (A,), generator=torch.Generator().manual_seed(5)).to(torch.int32).to(cuda)
    row_w = torch.rand(A, generator=torch.Generator().manual_seed(6)).to(BF).to(cuda)
    off = _offsets(counts)
    act = rows8.gemm_fc1_swiglu_rows8(x, w, off.to(cuda), token, row_w)
    for g in (0, 1, 3, G // 2, G - 2, G - 1):
        rows = slice(int(off[g]), int(off[g + 1]))
        one = rows8.Rows8(w.codes[g:g + 1].contiguous(), w.scales[g:g + 1].contiguous(), BF)
        ref = rows8.gemm_fc1_swiglu_rows8(x, one, _offsets([rows.stop - rows.start]).to(cuda), token[rows].clone(), row_w[rows].clone())
        assert torch.equal(act.codes.view(torch.uint8)[rows], ref.codes.view(torch.uint8)), f"copy {g}"
        assert torch.equal(act.scales[:, rows], ref.scales), f"copy {g}"


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("name", LAYOUTS)
def test_products_of_integers_are_exact(cuda, name, dtype):
    counts, N, K = LAYOUTS[name]
    print(f"rows8 gemm {name} {dtype}", flush=True)
    M, G = sum(counts), len(counts)
    a, b = _ints((M, K), 1, dtype), _ints((G, N, K), 2, dtype)
    off = _offsets(counts)
    qa, qb = rows8.quantize_rows(a.to(cuda)), rows8.quantize_rows(b.to(cuda))
    got = rows8.group_gemm_nt_rows8(qa, qb, off.to(cuda))
    want = torch.cat([a[off[g]:off[g + 1]].double() @ b[g].double().t() for g in range(G)])
    # |sum| <= K * (3 * 4)^2 < 2^24: fp32 holds it, and one rounding follows
    assert_exact(got, want.float().to(dtype), name)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("counts,N,K", [([7, 0, 40], 48, 400), ([150, 170], 136, 1008), ([300, 260], 264, 528)])
def test_products_of_activations(cuda, counts, N, K, dtype):
    M, G = sum(counts), len(counts)
    a, b = _randn((M, K), 11, dtype), _randn((G, N, K), 12, dtype, 0.05)
    a[:, 5] *= 30
    off = _offsets(counts)
    print(f"rows8 gemm {counts} {N} {K} {dtype}", flush=True)
    qa, qb = rows8.quantize_rows(a.to(cuda)), rows8.quantize_rows(b.to(cuda))
    got = rows8.group_gemm_nt_rows8(qa, qb, off.to(cuda))
    va = O.values(qa.codes.cpu(), qa.scales.cpu())
    vb = np.stack([O.values(qb.codes[g].cpu(), qb.scales[g].cpu()) for g in range(G)])
    c, big = O.grouped_nt(va, vb, off.numpy())
    _near(got, c, big * 2.0**-11, dtype, "C")


# (rows, copies, N, K): the calls' tile heights are checked on the host by tests/test_rows8.py
LARGE = {"one group": ([4096], 4096, 1024), "ragged large": ([1500, 0, 2400, 300, 1], 4096, 1040), "many tiles": ([700] * 12, 1000, 2064)}


@pytest.mark.parametrize("name", LARGE)
def test_large_products_of_integers_are_exact(cuda, name):
    counts, N, K = LARGE[name]
    print(f"rows8 gemm {name}", flush=True)
    M, G = sum(counts), len(counts)
    a, b = _ints((M, K), 1).to(cuda), _ints((G, N, K), 2).to(cuda)
    off = _offsets(counts)
    got = rows8.group_gemm_nt_rows8(rows8.quantize_rows(a), rows8.quantize_rows(b), off.to(cuda))
    want = torch.cat([(a[off[g]:off[g + 1]].double() @ b[g].double().t()).float().to(BF) for g in range(G)])
    assert_exact(got, want, name)


@pytest.mark.parametrize("name", LARGE)
def test_large_fc1_of_integers(cuda, name):
    """Every gate and up value is exact in fp32, so that the activations are known to the sigmoid's 2^-17."""
    counts, N, K = LARGE[name]
    print(f"rows8 fc1 {name}", flush=True)
    A, G, I, T = sum(counts), len(counts), N // 32 * 16, 777
    x, w = (_ints((T, K), 3) * 0.03125).to(cuda), (_ints((G, 2 * I, K), 4) * 0.03125).to(cuda)
    token = torch.randint(0, T, (A,), generator=torch.Generator().manual_seed(5)).to(torch.int32).to(cuda)
    off = _offsets(counts)
    act = rows8.gemm_fc1_swiglu_rows8(rows8.quantize_rows(x), rows8.quantize_rows(w), off.to(cuda), token)
    gu = torch.cat([x[token[off[g]:off[g + 1]].long()].double() @ w[g].double().t() for g in range(G)])
    exact = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]
    got = rows8.dequantize_rows(act).double()
    # at a block's power of two a value is off by half a step, 2^-4 of it, at least 2^-10 of the power
    e = act.scales.permute(1, 0, 2).reshape(A, -1)[:, : -(-I // 32)].double() - 127
    unit = torch.exp2(e).repeat_interleave(32, 1)[:, :I]
    tol = exact.abs() * (2.0**-4 + 2.0**-16) + unit * 2.0**-10
    assert ((got - exact).abs() <= tol).all(), ((got - exact).abs() - tol).max()
    most = torch.nn.functional.pad(exact.abs(), (0, -I % 32)).view(A, -1, 32).amax(-1)
    low, high = most * (1 - 2.0**-16), most * (1 + 2.0**-16)
    assert ((low <= 448 * torch.exp2(e)) & ((high > 224 * torch.exp2(e)) | (most == 0))).all(), "exponents"


def test_rows_of_no_group_are_left_alone(cuda):
    a, b = rows8.quantize_rows(_ints((300, 64), 1).to(cuda)), rows8.quantize_rows(_ints((2, 32, 64), 2).to(cuda))
    for offsets in ([3, 20, 290], [0, 300, 300], [5, 5, 5]):
        c = torch.full((300, 32), 7.0, dtype=BF, device=cuda)
        off = torch.tensor(offsets, dtype=torch.int32, device=cuda)
        _capi.call("pmx_rows8_group_gemm_nt", a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(),
                   off.data_ptr(), 2, 300, 32, 64, c.data_ptr(), torch.cuda.current_stream().cuda_stream)
        out = torch.ones(300, dtype=torch.bool)
        out[offsets[0]:offsets[2]] = False
        assert (c.cpu()[out] == 7.0).all()
        full = rows8.dequantize_rows(a).float()
        w = rows8.dequantize_rows(rows8.Rows8(b.codes.view(64, 64), b.scales.permute(1, 0, 2, 3).reshape(1, 64, 16).contiguous(), BF))
        for g in range(2):
            rows = slice(offsets[g], offsets[g + 1])
            assert_exact(c[rows], (full[rows].double() @ w.view(2, 32, 64)[g].double().t()).to(BF), f"group {g}")


def test_offsets_past_the_rows_are_clamped(cuda):
    """Offsets that leave [0, M] are clamped; where they descend nothing is written."""
    a, b = rows8.quantize_rows(_ints((40, 64), 1).to(cuda)), rows8.quantize_rows(_ints((3, 32, 64), 2).to(cuda))
    want = rows8.group_gemm_nt_rows8(a, b, torch.tensor([0, 10, 10, 40], dtype=torch.int32, device=cuda))
    got = rows8.group_gemm_nt_rows8(a, b, torch.tensor([-7, 10, 10, 1 << 30], dtype=torch.int32, device=cuda))
    assert_exact(got, want, "clamped")
    for bad in ([40, 30, 20, 10], [0, 30, 20, 40]):
        c = torch.full((40, 32), 7.0, dtype=BF, device=cuda)
        off = torch.tensor(bad, dtype=torch.int32, device=cuda)
        _capi.call("pmx_rows8_group_gemm_nt", a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(),
                   off.data_ptr(), 3, 40, 32, 64, c.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert (c == 7.0).all()


def test_a_row_depends_on_itself_and_its_copy_alone(cuda):
    """The same row in calls of one, a few, and many rows, in any slot: the same bits."""
    K, N = 1104, 248
    a, w = _randn((6400, K), 1).to(cuda), _randn((1, N, K), 2, std=0.05).to(cuda)
    ref = rows8.group_gemm_nt_rows8(rows8.quantize_rows(a.repeat(4, 1)), rows8.quantize_rows(w),
                                    torch.tensor([0, 25600], dtype=torch.int32, device=cuda))[:6400]
    for rows, slots in ((1, 1), (16, 1), (20, 3), (130, 2), (300, 5), (400, 200), (2600, 1), (6400, 10)):
        part = rows8.quantize_rows(a[:rows])
        counts = [0] * slots
        counts[slots // 2] = rows
        ww = torch.randn((slots, N, K), device=cuda).to(BF)
        ww[slots // 2] = w[0]
        got = rows8.group_gemm_nt_rows8(part, rows8.quantize_rows(ww), _offsets(counts).to(cuda))
        assert_exact(got, ref[:rows], f"{rows} rows in slot {slots // 2}")


# few rows: 32 x 64 tiles, and 32 x 256 ones
FEW = {"few tiles": ([2] * 100, 448, 272), "many tiles": ([3, 0, 7] * 100, 1016, 272)}


@pytest.mark.parametrize("name", FEW)
def test_few_rows(cuda, name):
    counts, N, K = FEW[name]
    M, G, I = sum(counts), len(counts), N // 32 * 16
    a, b, off = _ints((M, K), 1).to(cuda), _ints((G, N, K), 2).to(cuda), _offsets(counts)
    print(f"rows8 few {name}", flush=True)
    got = rows8.group_gemm_nt_rows8(rows8.quantize_rows(a), rows8.quantize_rows(b), off.to(cuda))
    group = torch.repeat_interleave(torch.arange(G), torch.tensor(counts)).to(cuda)
    want = torch.cat([torch.bmm(b[group[i:i + 50]].float(), a[i:i + 50].float().unsqueeze(2))[..., 0] for i in range(0, M, 50)])
    assert_exact(got, want.to(BF), name)
    # fc1 against the same call with every row in a group of its own copy's weights, on 128-row tiles
    w = rows8.quantize_rows(_randn((G, 2 * I, K), 3, std=0.06).to(cuda))
    q = rows8.quantize_rows(_randn((M, K), 4).to(cuda))
    act = rows8.gemm_fc1_swiglu_rows8(q, w, off.to(cuda))
    for g in (0, 2, G - 1):
        rows = slice(int(off[g]), int(off[g + 1]))
        many = torch.arange(rows.start, rows.stop, dtype=torch.int32, device=cuda).repeat(3000)
        one = rows8.Rows8(w.codes[g:g + 1].contiguous(), w.scales[g:g + 1].contiguous(), BF)
        ref = rows8.gemm_fc1_swiglu_rows8(q, one, torch.tensor([0, many.numel()], dtype=torch.int32, device=cuda), many)
        n = rows.stop - rows.start
        assert torch.equal(act.codes.view(torch.uint8)[rows], ref.codes.view(torch.uint8)[:n]), f"copy {g}"


def test_every_tiling_gives_the_same_bits(cuda):
    """4096 rows run on 256-row tiles, 1000 on 128-row ones, 10 on 32 x 64 ones (32 x 256 ones need many copies)."""
    N, K = 4096, 1024
    x, w = _randn((4096, K), 1).to(cuda), _randn((1, N, K), 2, std=0.03).to(cuda)
    qw = rows8.quantize_rows(w)
    nt, fc1 = [], []
    for rows in (4096, 1000, 10):
        q, off = rows8.quantize_rows(x[:rows]), torch.tensor([0, rows], dtype=torch.int32, device=cuda)
        nt.append(rows8.group_gemm_nt_rows8(q, qw, off))
        fc1.append(rows8.gemm_fc1_swiglu_rows8(q, qw, off).codes.view(torch.uint8))
    for rows, a, b in zip((1000, 10), nt[1:], fc1[1:]):
        assert_exact(a, nt[0][:rows], f"{rows} rows")
        assert torch.equal(b, fc1[0][:rows]), f"{rows} rows of fc1"


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("counts,I,H,T", [([1], 16, 16, 1), ([3, 0, 30, 7], 48, 144, 20), ([130, 90, 61], 144, 528, 100),
                                          ([300, 280], 208, 272, 290), ([40] * 3, 640, 64, 50)])
def test_fc1_swiglu_in_8_bits(cuda, counts, I, H, T, dtype):
    G, A = len(counts), sum(counts)
    print(f"rows8 fc1 {counts} I={I} H={H} {dtype}", flush=True)
    g = torch.Generator().manual_seed(A + I)
    x, w = _randn((T, H), 1, dtype), _randn((G, 2 * I, H), 2, dtype, 1.5 / math.sqrt(H))
    token = torch.randint(0, T, (A,), generator=g).to(torch.int32)
    row_w = (0.05 + torch.rand(A, generator=g)).to(dtype)
    off = _offsets(counts)
    qx, qw = rows8.quantize_rows(x.to(cuda)), rows8.quantize_rows(w.to(cuda))
    act = rows8.gemm_fc1_swiglu_rows8(qx, qw, off.to(cuda), token.to(cuda), row_w.to(cuda))
    assert act.shape == (A, I) and act.codes.dtype == torch.float8_e4m3fn
    vx = O.values(qx.codes.cpu(), qx.scales.cpu())[token.numpy()]
    vw = np.stack([O.values(qw.codes[k].cpu(), qw.scales[k].cpu()) for k in range(G)])
    gu, big = O.grouped_nt(vx, vw, off.numpy())
    gate, up = gu[:, :I], gu[:, I:]
    rw = row_w.double().numpy()[:, None]
    exact = gate / (1 + np.exp(-gate)) * up * rw
    slack = rw * (1.1 * big[:, :I] * np.abs(up) + np.abs(gate) * big[:, I:]) * 2.0**-11 + np.abs(exact) * 2.0**-17
    # the block's power of two: that of the exact values, or of values that differ by the slack
    low, high = np.abs(exact) - slack, np.abs(exact) + slack
    e_low, e_high = O.block_exponents(np.maximum(low, 0), "e4m3"), O.block_exponents(high, "e4m3")
    nb = e_low.shape[1]
    e = act.scales.cpu().permute(1, 0, 2).reshape(A, -1)[:, :nb].numpy().astype(np.int64) - 127
    assert ((e >= e_low) & (e <= e_high)).all(), "exponents"
    got = O.values(act.codes.cpu(), act.scales.cpu())
    unit = np.repeat(2.0**e, 32, axis=1)[:, :I]
    # e4m3: half a step is 2^-4 of the value, at least 2^-10 of the unit
    tol = slack + np.maximum((np.abs(exact) + slack) * 2.0**-4, unit * 2.0**-10)
    assert (np.abs(got - exact) <= tol * 1.0001).all(), f"codes: {(np.abs(got - exact) - tol).max()}"
    # the blocks that fc2's last K-tile takes along stand beside 2^0
    tail = act.scales.cpu().permute(1, 0, 2).reshape(A, -1)[:, nb: max(2, -(-I // 128)) * 4]
    assert (tail == 127).all()
    plain = rows8.gemm_fc1_swiglu_rows8(rows8.Rows8(qx.codes[token.long()].contiguous(), qx.scales[:, token.long()].contiguous(), dtype),
                                        qw, off.to(cuda), None, row_w.to(cuda))
    assert torch.equal(plain.codes.view(torch.uint8), act.codes.view(torch.uint8)), "rows in place"


@pytest.mark.parametrize("rows", [3, 100, 1500, 9000])
@pytest.mark.parametrize("I", [16, 48, 144, 512, 528])
def test_fc1_writes_every_scale(cuda, I, rows):
    """The bytes past the last column stand for 2^0, as `quantize_rows` leaves them."""
    G, H = 3, 64
    x = rows8.quantize_rows(_randn((rows, H), 1).to(cuda))
    w = rows8.quantize_rows(_randn((G, 2 * I, H), 2).to(cuda))
    junk = torch.full((1 << 24,), 3, dtype=torch.uint8, device=cuda)  # what the outputs' memory held before
    del junk
    act = rows8.gemm_fc1_swiglu_rows8(x, w, _offsets([rows - 2, 1, 1]).to(cuda))
    tail = act.scales.permute(1, 0, 2).reshape(rows, -1)[:, -(-I // 32):]
    assert (tail == 127).all()


def test_token_outside_reads_as_zeros(cuda):
    qx, qw = rows8.quantize_rows(_randn((4, 64), 1).to(cuda)), rows8.quantize_rows(_randn((1, 64, 64), 2).to(cuda))
    off = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    act = rows8.gemm_fc1_swiglu_rows8(qx, qw, off, torch.tensor([1, 4, -5], dtype=torch.int32, device=cuda))
    v = rows8.dequantize_rows(act)
    assert v[0].abs().max() > 0 and (v[1:] == 0).all()


def test_product_refusals(cuda):
    a, b = rows8.quantize_rows(_randn((8, 64), 1).to(cuda)), rows8.quantize_rows(_randn((2, 32, 64), 2).to(cuda))
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device=cuda)
    with pytest.raises(AssertionError, match="e4m3 for a product"):
        rows8.group_gemm_nt_rows8(rows8.quantize_rows(_randn((8, 64), 1).to(cuda), "int8"), b, off)
    with pytest.raises(AssertionError, match="stand for"):
        rows8.group_gemm_nt_rows8(rows8.quantize_rows(_randn((8, 64), 1, F16).to(cuda)), b, off)
    with pytest.raises(AssertionError, match="disagree on K"):
        rows8.group_gemm_nt_rows8(rows8.quantize_rows(_randn((8, 48), 1).to(cuda)), b, off)
    with pytest.raises(AssertionError, match="offsets"):
        rows8.group_gemm_nt_rows8(a, b, off[:2])
    with pytest.raises(ValueError, match="unsupported shape"):
        rows8.group_gemm_nt_rows8(rows8.quantize_rows(_randn((8, 40), 1).to(cuda)),
                                  rows8.quantize_rows(_randn((2, 32, 40), 2).to(cuda)), off)
    with pytest.raises(ValueError, match="unsupported shape"):
        rows8.group_gemm_nt_rows8(a, rows8.quantize_rows(_randn((2, 12, 64), 2).to(cuda)), off)
    empty = rows8.quantize_rows(torch.empty((0, 64), dtype=BF, device=cuda))
    assert rows8.group_gemm_nt_rows8(empty, b, torch.zeros(3, dtype=torch.int32, device=cuda)).shape == (0, 32)


# ---------------------------------------------------------------------------
# Streams, graphs, offsets past 32 bits
# ---------------------------------------------------------------------------


def _every_op(x, pos, d, w, offsets, fmt="e4m3"):
    """One call of each: x [R, N], pos [R, K], d [R, N / 2], w [G, n, N] in 8 bits."""
    q = rows8.quantize_rows(x, fmt)
    row_w = d[:, 0].contiguous()
    row_src = pos[:, 0].contiguous()
    dg, act, dw = rows8.swiglu_bwd_rows8(d, q, row_w, row_src, pos.numel())
    c = rows8.group_gemm_nt_rows8(q, w, offsets)
    a = rows8.gemm_fc1_swiglu_rows8(q, w, offsets)
    return [rows8.dequantize_rows(q, pos), dg, act, dw[row_src.long()], c, a.codes.view(torch.uint8), a.scales]


def _every_op_case(cuda, R, seed):
    N, K, G = 1056, 3, 4
    g = torch.Generator().manual_seed(seed)
    w = rows8.quantize_rows(_randn((G, 96, N), seed + 1).to(cuda))
    counts = np.random.default_rng(seed).multinomial(R, [1 / G] * G)
    return [_randn((R, N), seed + 2).to(cuda), torch.randperm(R * K, generator=g).to(torch.int32).view(R, K).to(cuda),
            _randn((R, N // 2), seed + 3).to(cuda), w, _offsets(counts).to(cuda)]


def test_every_op_on_two_streams_at_once(cuda):
    cases = [_every_op_case(cuda, R, R) for R in (37, 900)]
    want = [_every_op(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(_every_op(*cases[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for outs in got[k]:
            for j, (a, b) in enumerate(zip(outs, want[k])):
                assert_exact(a, b, f"case {k}, output {j}")


def test_every_op_in_a_graph(cuda):
    case = _every_op_case(cuda, 130, 7)
    _every_op(*case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _every_op(*case)
    for k in range(3):
        case[0].copy_(_randn(tuple(case[0].shape), 80 + k).to(cuda))
        graph.replay()
        eager = _every_op(*case)
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(outs, eager)):
            assert_exact(a, b, f"replay {k}, output {j}")


def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements: 500 rows over and over, each repeat the same as the first."""
    n, times, N = 500, 1100, 4112
    assert n * times * N > 2**31
    rows, d = _randn((n, N), 1).to(cuda), _randn((n, N // 2), 2).to(cuda)
    ref = rows8.quantize_rows(rows)
    print("past 32 bits: writing", flush=True)
    big = rows8.quantize_rows(rows.repeat(times, 1))
    assert torch.equal(big.codes.view(torch.uint8).view(times, n, N)[[0, -2, -1]],
                       ref.codes.view(torch.uint8).expand(3, n, N))
    assert torch.equal(big.scales.view(-1, times, n, 16)[:, -1], ref.scales)
    print("past 32 bits: reading back", flush=True)
    back = rows8.dequantize_rows(big)
    assert_exact(back[-n:], rows8.dequantize_rows(ref), "read back")
    del back
    print("past 32 bits: SwiGLU backward", flush=True)
    dg, act, _ = rows8.swiglu_bwd_rows8(d.repeat(times, 1), big)
    dg_ref, act_ref, _ = rows8.swiglu_bwd_rows8(d, ref)
    assert_exact(dg[-n:], dg_ref, "dG1")
    assert_exact(act[-n:], act_ref, "act_w")
    del dg, act
    for depth, cols in ((N, 64), (64, N)):  # long A, then a long output
        a = big if depth == N else rows8.quantize_rows(rows[:, :64].repeat(times, 1))
        small = ref if depth == N else rows8.quantize_rows(rows[:, :64].contiguous())
        b = rows8.quantize_rows(_randn((2, cols, depth), 3).to(cuda))
        half = n * times // 2
        print(f"past 32 bits: products {depth} deep, {cols} wide", flush=True)
        off, off_ref = _offsets([half, half]).to(cuda), _offsets([0, n]).to(cuda)
        assert_exact(rows8.group_gemm_nt_rows8(a, b, off)[-n:], rows8.group_gemm_nt_rows8(small, b, off_ref), "product")
        up = rows8.quantize_rows(_randn((2, 2 * cols, depth), 4).to(cuda))
        act, act_ref = rows8.gemm_fc1_swiglu_rows8(a, up, off), rows8.gemm_fc1_swiglu_rows8(small, up, off_ref)
        assert torch.equal(act.codes.view(torch.uint8)[-n:], act_ref.codes.view(torch.uint8))
        assert torch.equal(act.scales[:, -n:], act_ref.scales)
    T, K = 66000, 8
    print("past 32 bits: spreading", flush=True)
    pos = torch.randperm(T * K, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(T, K).to(cuda)
    few = rows8.quantize_rows(rows.repeat(T // n, 1))
    out = rows8.dequantize_rows(few, pos)
    plain = rows8.dequantize_rows(ref)
    at = torch.arange(0, T, 97, device=cuda)
    for k in range(K):
        assert_exact(out[pos[at, k].long()], plain[at % n], f"spread {k}")


# ---------------------------------------------------------------------------
# The serving layer
# ---------------------------------------------------------------------------


def _layer_oracle(hidden, w, phys, experts8, eps):
    """(out, tolerance) of the 8-bit layer in 64 bits, from the weights' 8-bit values.

    The kernel's activations, before they are rounded to 8 bits, lie within
    `slack` of the exact ones (products to 2^-11 of the largest of each 64,
    the sigmoid to 2^-17).  Rounding is monotonic, so each one's 8-bit value lies
    between those of act - slack and act + slack at the block's power of two:
    where these agree it is exact, where a border lies between them it may be
    either, off by at most their distance (a block whose power of two itself may
    differ: both powers are tried).  fc2 carries these distances on and adds its
    own 2^-11; its rows, 16-bit integers beside a power of two with the largest
    of 32 columns between 16383.5 and 32767, are off by at most half of it, 2^-15 of
    that largest.  The rows' sum is rounded once.
    """
    C = experts8.down.shape[0]
    T, K = phys.shape
    x, _ = O.quantize(hidden, "e4m3")
    H = hidden.shape[1]
    out, tol = np.zeros((T, H)), np.zeros((T, H))

    def rounded(v, e):
        unit = np.repeat(2.0 ** e.astype(np.float64), 32, axis=1)[:, : v.shape[1]]
        y = np.clip(v / unit, -448, 448)
        _, k = np.frexp(y)
        step = 2.0 ** np.maximum(k - 4, -9)
        return np.rint(y / step) * step * unit

    for c in range(C):
        at = np.argwhere(phys == c)
        if not len(at):
            continue
        up = O.values(experts8.gate_up.codes[c].cpu(), experts8.gate_up.scales[c].cpu())
        down = O.values(experts8.down.codes[c].cpu(), experts8.down.scales[c].cpu())
        I = down.shape[1]
        one = np.array([0, len(at)])
        gu, big = O.grouped_nt(x[at[:, 0]], up[None], one)
        g, u = gu[:, :I], gu[:, I:]
        wr = w.double().numpy()[at[:, 0], at[:, 1]][:, None]
        act = g / (1 + np.exp(-g)) * u * wr
        # |d silu / dg| <= 1.1
        slack = wr * (1.1 * big[:, :I] * np.abs(u) + np.abs(g) * big[:, I:]) * 2.0**-11 + np.abs(act) * 2.0**-17
        e = O.block_exponents(act, "e4m3")
        held = rounded(act, e)
        far = np.zeros_like(act)
        for e2 in {"low": O.block_exponents(np.maximum(np.abs(act) - slack, 0), "e4m3"),
                   "high": O.block_exponents(np.abs(act) + slack, "e4m3")}.values():
            for v in (act - slack, act + slack):
                far = np.maximum(far, np.abs(rounded(v, e2) - held))
        y, big2 = O.grouped_nt(held, down[None], one)
        off = far @ np.abs(down).T + big2 * 2.0**-11
        np.add.at(out, at[:, 0], y)
        most = np.pad(np.abs(y) + off, ((0, 0), (0, -H % 32))).reshape(len(at), -1, 32).max(-1)
        np.add.at(tol, at[:, 0], off + np.repeat(most, 32, axis=1)[:, :H] * 2.0**-15)
    return out, tol + (np.abs(out) + tol) * eps / 2


@pytest.mark.parametrize("T", [1, 5, 64, 700])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_layer_over_8_bit_weights(cuda, T, dtype):
    H, I, E, C, K, S = 272, 144, 12, 17, 3, 4
    g = torch.Generator().manual_seed(T)
    hidden = _randn((T, H), T, dtype)
    sel = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)])
    w = torch.softmax(torch.randn((T, K), generator=g), -1).to(dtype)
    src = torch.randint(0, S, (T,), generator=g)
    e, s = torch.arange(E), torch.arange(S).unsqueeze(1)
    mapping = torch.where((e < C - E) & (s % 2 == 1), E + e, e).contiguous()
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1, dtype, 0.1).to(cuda), _randn((C, H, I), 2, dtype, 0.1).to(cuda))
    print(f"layer rows8 T={T} {dtype}", flush=True)
    seen = []
    got = placemoe_amd.expert_layer_rows8(hidden.to(cuda), w.to(cuda), sel.to(cuda), q, mapping=mapping.to(cuda),
                                          sources=src.to(cuda), recorder=lambda c: seen.append(c.clone()))
    phys = moe_oracle.map_logical_to_physical(mapping.numpy(), src.numpy(), sel.numpy())
    exact, tol = _layer_oracle(hidden, w, np.asarray(phys), q, torch.finfo(dtype).eps)
    assert int(seen[0].sum()) == T * K
    off = np.abs(got.double().cpu().numpy() - exact)
    assert (off <= tol * 1.0001 + SUBNORMAL[dtype]).all(), (off - tol).max()
    # the tolerance itself stays small beside the outputs
    assert np.linalg.norm(tol) <= 0.1 * np.linalg.norm(exact), np.linalg.norm(tol) / np.linalg.norm(exact)
    assert_bf16_close(got, torch.from_numpy(exact), name="out")


def test_layer_refusals_and_edges(cuda):
    H, I, C = 64, 32, 4
    gate_up, down = _randn((C, 2 * I, H), 1).to(cuda), _randn((C, H, I), 2).to(cuda)
    q = rows8.Experts8.quantize(gate_up, down)
    x, w = _randn((5, H), 3).to(cuda), torch.ones((5, 1), dtype=BF, device=cuda)
    sel = torch.zeros((5, 1), dtype=torch.int64, device=cuda)
    assert placemoe_amd.expert_layer_rows8(x, w, sel, q).shape == (5, H)
    assert placemoe_amd.expert_layer_rows8(x[:0], w[:0], sel[:0], q).shape == (0, H)
    with pytest.raises(ValueError, match="no backward"):
        placemoe_amd.expert_layer_rows8(x.clone().requires_grad_(), w, sel, q)
    with torch.no_grad():
        placemoe_amd.expert_layer_rows8(x.clone().requires_grad_(), w, sel, q)
    with pytest.raises(AssertionError):
        placemoe_amd.expert_layer_rows8(x.to(F16), w.to(F16), sel, q)
    with pytest.raises(AssertionError):
        placemoe_amd.expert_layer_rows8(x, w, sel, (gate_up, down))
    with pytest.raises(AssertionError):
        placemoe_amd.expert_layer_rows8(x[:, :32].contiguous(), w, sel, q)
    with pytest.raises(AssertionError):
        rows8.Experts8.quantize(gate_up, down[:, :32].contiguous())
    bad = rows8.Experts8.quantize(_randn((C, 48, H), 1).to(cuda), _randn((C, H, 24), 2).to(cuda))
    with pytest.raises(ValueError, match="multiples of 16"):
        placemoe_amd.expert_layer_rows8(x, w, sel, bad)
    placemoe_amd.expert_layer_rows8(x, w, sel + 99, q)
    with pytest.raises(ValueError, match="expert id outside"):
        experts.check_pending_routes(block=True)


def test_layer_refuses_scales_on_the_host(cuda):
    """Each part of the weights is looked at: a host pointer never reaches a kernel."""
    C, H, I = 4, 64, 32
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1).to(cuda), _randn((C, H, I), 2).to(cuda))
    x, w = _randn((5, H), 3).to(cuda), torch.ones((5, 1), dtype=BF, device=cuda)
    sel = torch.zeros((5, 1), dtype=torch.int64, device=cuda)
    host = lambda r: rows8.Rows8(r.codes, r.scales.cpu(), r.dtype)  # noqa: E731
    for bad in (rows8.Experts8(host(q.gate_up), q.down), rows8.Experts8(q.gate_up, host(q.down))):
        with pytest.raises(AssertionError, match="GPU tensors"):
            placemoe_amd.expert_layer_rows8(x, w, sel, bad)


def test_layer_without_tokens_reports_its_counts(cuda):
    C, H, I = 4, 64, 32
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1).to(cuda), _randn((C, H, I), 2).to(cuda))
    seen = []
    placemoe_amd.expert_layer_rows8(_randn((0, H), 3).to(cuda), torch.ones((0, 2), dtype=BF, device=cuda),
                                    torch.zeros((0, 2), dtype=torch.int64, device=cuda), q, recorder=seen.append)
    assert len(seen) == 1 and seen[0].dtype == torch.int32 and seen[0].tolist() == [0] * C


def test_layer_keeps_what_is_not_finite_to_its_token(cuda):
    C, H, I, T = 3, 96, 64, 40
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1, BF, 0.1).to(cuda), _randn((C, H, I), 2, BF, 0.1).to(cuda))
    x, w = _randn((T, H), 3).to(cuda), torch.full((T, 2), 0.5, dtype=BF, device=cuda)
    sel = torch.stack([torch.arange(T) % C, (torch.arange(T) + 1) % C], 1).to(cuda)
    want = placemoe_amd.expert_layer_rows8(x, w, sel, q)
    bad = x.clone()
    bad[2, 7], bad[20, 50], w2 = math.nan, math.inf, w.clone()
    w2[31, 1] = math.nan
    got = placemoe_amd.expert_layer_rows8(bad, w2, sel, q)
    hit = torch.tensor([2, 20, 31], device=cuda)
    assert got[hit].isnan().all()
    rest = torch.ones(T, dtype=torch.bool, device=cuda)
    rest[hit] = False
    assert_exact(got[rest], want[rest], "the other tokens")


@pytest.mark.parametrize("K", [1, 2, 3, 4, 6, 8, 11])
@pytest.mark.parametrize("H", [16, 48, 2064])
def test_layer_sums_any_number_of_experts(cuda, H, K):
    T, C, I = 5, 12, 32
    hidden, g = _randn((T, H), H), torch.Generator().manual_seed(K)
    sel = torch.stack([torch.randperm(C, generator=g)[:K] for _ in range(T)])
    w = torch.softmax(torch.randn((T, K), generator=g), -1).to(BF)
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1, BF, 0.1).to(cuda), _randn((C, H, I), 2, BF, 0.1).to(cuda))
    got = placemoe_amd.expert_layer_rows8(hidden.to(cuda), w.to(cuda), sel.to(cuda), q)
    exact, tol = _layer_oracle(hidden, w, sel.numpy(), q, torch.finfo(BF).eps)
    off = np.abs(got.double().cpu().numpy() - exact)
    assert (off <= tol * 1.0001 + SUBNORMAL[BF]).all(), (off - tol).max()


def test_layer_with_one_expert_twice(cuda):
    """A token that names a copy twice has both of its rows, each with its weight."""
    T, C, H, I = 9, 3, 64, 48
    hidden = _randn((T, H), 1)
    sel = torch.arange(T).remainder(C).reshape(T, 1).repeat(1, 2)
    w = torch.softmax(_randn((T, 2), 2).float(), -1).to(BF)
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 3, BF, 0.1).to(cuda), _randn((C, H, I), 4, BF, 0.1).to(cuda))
    got = placemoe_amd.expert_layer_rows8(hidden.to(cuda), w.to(cuda), sel.to(cuda), q)
    exact, tol = _layer_oracle(hidden, w, sel.numpy(), q, torch.finfo(BF).eps)
    off = np.abs(got.double().cpu().numpy() - exact)
    assert (off <= tol * 1.0001 + SUBNORMAL[BF]).all(), (off - tol).max()


def test_two_layers_at_once(cuda):
    """Calls on two streams share nothing: each has its workspace."""
    C, H, I = 16, 512, 256
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1, BF, 0.1).to(cuda), _randn((C, H, I), 2, BF, 0.1).to(cuda))
    g = torch.Generator().manual_seed(5)
    calls = []
    for k in range(2):
        T = (700, 33)[k]
        sel = torch.stack([torch.randperm(C, generator=g)[:4] for _ in range(T)]).to(cuda)
        calls.append((_randn((T, H), 10 + k).to(cuda), torch.full((T, 4), 0.25, dtype=BF, device=cuda), sel, q))
    want = [placemoe_amd.expert_layer_rows8(*c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[k].append(placemoe_amd.expert_layer_rows8(*c))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert_exact(out, want[k], f"call {k}")


def test_layer_on_another_stream_and_in_a_graph(cuda):
    wl = make_workload("qwen3", device=cuda, tokens=24)
    q = rows8.Experts8.quantize(wl.fc1, wl.fc2)

    def step():
        return placemoe_amd.expert_layer_rows8(wl.hidden, wl.routing_weights, wl.selected, q, mapping=wl.mapping, sources=wl.sources)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert_exact(got, want, "side stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        wl.hidden.copy_(_randn(tuple(wl.hidden.shape), 50 + k).to(cuda))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert_exact(out, eager, f"replay {k}")


# ---------------------------------------------------------------------------
# Checkpointed training layer
# ---------------------------------------------------------------------------


def _grads(wl, cuda, split, **kw):
    leaf = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    x, w = leaf(wl.hidden), leaf(wl.routing_weights)
    if split:
        weights = dict(fc1_1_weight=leaf(wl.fc1[:, :wl.I]), fc1_2_weight=leaf(wl.fc1[:, wl.I:]))
        weights = {k: v.detach().contiguous().requires_grad_() for k, v in weights.items()}
    else:
        weights = dict(fc1_1_2_weight=leaf(wl.fc1))
    down = leaf(wl.fc2)
    out = experts.expert_layer(x, w, wl.selected, down, mapping=wl.mapping, sources=wl.sources, **weights, **kw)
    out.backward(_randn(tuple(out.shape), 77).to(cuda))
    fc1 = torch.cat([weights["fc1_1_weight"].grad, weights["fc1_2_weight"].grad], 1) if split else weights["fc1_1_2_weight"].grad
    return out.detach(), {"dx": x.grad, "dw": w.grad, "d_fc1": fc1, "d_fc2": down.grad}


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("name,tokens", [("toy", 300), ("dsv3", 200), ("qwen3", 40)])
def test_checkpointed_layer(cuda, name, tokens, weighted, split):
    """The output is the uncheckpointed one bit for bit.  The gradients are the
    formula's at the 8-bit hidden states and gate/up rows, to the bf16 bar (their products
    run on bf16 operands, rounded between the steps); those of int8, whose
    roundings are four times smaller, come near the uncheckpointed ones."""
    wl = make_workload(name, device=cuda, tokens=tokens, **({"num_slots": 4} if name == "dsv3" else {}))
    print(f"checkpointed {name} weighted={weighted} split={split}", flush=True)
    plain, ref = _grads(wl, cuda, split, weighted_input=weighted)
    for fmt in ("e4m3", "int8"):
        out, got = _grads(wl, cuda, split, weighted_input=weighted, activation_checkpoint=fmt)
        assert_exact(out, plain, f"{fmt} output")
        want = _checkpointed_oracle(wl, fmt, cuda)
        for k in got:
            assert_bf16_close(got[k], want[k], name=f"{fmt} {k}")
        for k in ("dx", "dw", "d_fc1", "d_fc2"):
            err = ((got[k].float() - ref[k].float()).norm() / ref[k].float().norm()).item()
            # a value is off by at most 2^-4 of itself (e4m3); three such factors meet in dx and dw
            assert err <= (3 * 2.0**-4 if fmt == "e4m3" else 0.04), (fmt, k, err)


def _checkpointed_oracle(wl, fmt, cuda):
    """The gradients in 64 bits, from what 8 bits hold of the hidden states and of the layer's own gate/up rows."""
    T, K, H, I, C = wl.T, wl.K, wl.H, wl.I, wl.C
    r = kernels.route(wl.selected, C, mapping=wl.mapping, sources=wl.sources)
    xp, row_src, _ = kernels.moe_scatter_src(wl.hidden, r.pos, wl.routing_weights)
    gu, _ = kernels.gemm_fc1_swiglu(xp, wl.fc1, wl.fc1.view(-1)[I * H:], 2 * I * H, r.offsets, C, I)
    back = lambda t: rows8.dequantize_rows(rows8.quantize_rows(t, fmt)).double()  # noqa: E731
    gu8, x8 = back(gu), back(wl.hidden)
    g, u = gu8[:, :I], gu8[:, I:]
    src = row_src.long()
    w = wl.routing_weights.double().reshape(-1)[src].unsqueeze(1)
    dy = _randn((T, H), 77).to(cuda).double()[src // K]
    sig = torch.sigmoid(g)
    s = g * sig
    off = r.offsets.tolist()
    d_act = torch.cat([dy[off[c]:off[c + 1]] @ wl.fc2[c].double() for c in range(C)])
    da = d_act * w
    dg1 = torch.cat([da * u * (sig + s * (1 - sig)), da * s], 1)
    act_w, xr = w * s * u, x8[src // K]
    rows = [slice(off[c], off[c + 1]) for c in range(C)]
    dw = torch.empty(T * K, dtype=torch.float64, device=cuda)
    dw[src] = (d_act * s * u).sum(1)
    dx = torch.zeros((T, H), dtype=torch.float64, device=cuda)
    dx.index_add_(0, src // K, torch.cat([dg1[q] @ wl.fc1[c].double() for c, q in enumerate(rows)]))
    return {"dx": dx, "dw": dw.view(T, K), "d_fc1": torch.stack([dg1[q].t() @ xr[q] for q in rows]),
            "d_fc2": torch.stack([dy[q].t() @ act_w[q] for q in rows])}


def test_checkpoint_keeps_less(cuda):
    wl = make_workload("qwen3", device=cuda, tokens=512)

    def kept(**kw):
        x = wl.hidden.clone().requires_grad_()
        total = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (total.append(t), t)[1], lambda t: t):
            experts.expert_layer(x, wl.routing_weights, wl.selected, wl.fc2, fc1_1_2_weight=wl.fc1, mapping=wl.mapping,
                                 sources=wl.sources, **kw)
        weights = {wl.fc1.data_ptr(), wl.fc2.data_ptr()}
        seen = {t.data_ptr(): t.numel() * t.element_size() for t in total if t.data_ptr() not in weights}
        seen.pop(wl.fc1.data_ptr() + wl.I * wl.H * 2, None)
        return sum(seen.values())

    A, H, I = wl.T * wl.K, wl.H, wl.I
    assert kept() >= A * (4 * H + 6 * I)
    assert kept(activation_checkpoint="e4m3") <= 1.1 * (wl.T * H + 2 * A * I) + 64 * A


def test_checkpoint_through_the_public_op(cuda):
    wl = make_workload("toy", device=cuda, tokens=64)
    fc1, fc2 = wl.fc1[:8].contiguous(), wl.fc2[:8].contiguous()

    def step(fmt):
        x, a, b = wl.hidden.clone().requires_grad_(), fc1.clone().requires_grad_(), fc2.clone().requires_grad_()
        prev = placemoe_amd.set_activation_checkpoint(fmt)
        try:
            out = placemoe_amd.hip_fused_moe_forward(8, wl.routing_weights, wl.selected, x, None, None, b, a)
        finally:
            placemoe_amd.set_activation_checkpoint(prev)
        out.sum().backward()
        return out.detach(), x.grad, a.grad, b.grad

    plain, kept = step(None), step("int8")
    assert_exact(kept[0], plain[0], "output")
    for k, (a, b) in enumerate(zip(kept[1:], plain[1:])):
        assert not torch.equal(a, b), "the checkpoint was not used"
        assert ((a.float() - b.float()).norm() / b.float().norm()).item() <= 0.04, k


def test_checkpointed_backward_in_a_graph(cuda):
    wl = make_workload("qwen3", device=cuda, tokens=32)
    dout = _randn((wl.T, wl.H), 5).to(cuda)
    x, x_eager = (wl.hidden.clone().requires_grad_() for _ in range(2))  # the captured graph has a leaf of its own

    def step(x):
        out = experts.expert_layer(x, wl.routing_weights, wl.selected, wl.fc2, fc1_1_2_weight=wl.fc1, mapping=wl.mapping,
                                   sources=wl.sources, activation_checkpoint="e4m3")
        return torch.autograd.grad(out, x, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x_eager)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step(x)
    for k in range(3):
        with torch.no_grad():
            x.copy_(_randn(tuple(x.shape), 60 + k).to(cuda))
            x_eager.copy_(x)
        graph.replay()
        eager = step(x_eager)
        torch.cuda.synchronize()
        assert_exact(grad, eager, f"replay {k}")


@pytest.mark.parametrize("weighted", [False, True])
def test_checkpointed_layer_without_tokens(cuda, weighted):
    wl = make_workload("toy", device=cuda, tokens=8)
    x = wl.hidden[:0].clone().requires_grad_()
    w = wl.routing_weights[:0].clone().requires_grad_()
    fc1, fc2 = wl.fc1.clone().requires_grad_(), wl.fc2.clone().requires_grad_()
    sources = wl.sources[:0] if wl.sources is not None else None
    out = experts.expert_layer(x, w, wl.selected[:0], fc2, fc1_1_2_weight=fc1, mapping=wl.mapping, sources=sources,
                               weighted_input=weighted, activation_checkpoint="e4m3")
    out.sum().backward()
    assert out.shape == x.shape and x.grad.shape == x.shape and w.grad.shape == w.shape
    assert not fc1.grad.any() and not fc2.grad.any()


@pytest.mark.parametrize("wanted", ["hidden", "weights", "fc1", "fc2"])
def test_checkpointed_layer_with_one_gradient_wanted(cuda, wanted):
    """Whatever is frozen, the one gradient asked for is the same."""
    wl = make_workload("toy", device=cuda, tokens=70)
    dout = _randn((wl.T, wl.H), 3).to(cuda)

    def grads(names):
        t = {"hidden": wl.hidden, "weights": wl.routing_weights, "fc1": wl.fc1, "fc2": wl.fc2}
        t = {k: v.clone().requires_grad_(k in names) for k, v in t.items()}
        out = experts.expert_layer(t["hidden"], t["weights"], wl.selected, t["fc2"], fc1_1_2_weight=t["fc1"],
                                   mapping=wl.mapping, sources=wl.sources, activation_checkpoint="e4m3")
        out.backward(dout)
        return {k: v.grad for k, v in t.items()}

    every, one = grads(("hidden", "weights", "fc1", "fc2")), grads((wanted,))
    assert_exact(one[wanted], every[wanted], wanted)
    assert all(g is None for k, g in one.items() if k != wanted)


def test_nothing_waits_for_the_gpu(cuda):
    """Every op, the serving layer and a checkpointed step under torch's synchronisation errors."""
    case = _every_op_case(cuda, 60, 3)
    wl = make_workload("toy", device=cuda, tokens=50)
    q = rows8.Experts8.quantize(wl.fc1, wl.fc2)
    x = wl.hidden.clone().requires_grad_()

    def step():
        outs = _every_op(*case)[:1]
        with torch.no_grad():
            outs.append(placemoe_amd.expert_layer_rows8(wl.hidden, wl.routing_weights, wl.selected, q, mapping=wl.mapping,
                                                        sources=wl.sources))
        out = experts.expert_layer(x, wl.routing_weights, wl.selected, wl.fc2, fc1_1_2_weight=wl.fc1, mapping=wl.mapping,
                                   sources=wl.sources, activation_checkpoint="int8")
        return outs + [out.detach(), torch.autograd.grad(out, x, torch.ones_like(out))[0]]

    want = step()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = step()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    for k, (a, b) in enumerate(zip(got, want)):
        assert_exact(a, b, f"output {k}")


def test_weights_through_the_host(cuda):
    """What a server writes down and loads again answers with the same bits."""
    C, H, I = 6, 96, 64
    q = rows8.Experts8.quantize(_randn((C, 2 * I, H), 1, BF, 0.1).to(cuda), _randn((C, H, I), 2, BF, 0.1).to(cuda))
    back = rows8.Experts8(q.gate_up.to("cpu").to(cuda), q.down.to("cpu").to(cuda))
    args = (_randn((7, H), 3).to(cuda), torch.ones((7, 1), dtype=BF, device=cuda), torch.arange(7, device=cuda).reshape(7, 1) % C)
    assert_exact(placemoe_amd.expert_layer_rows8(*args, back), placemoe_amd.expert_layer_rows8(*args, q), "out")


def test_checkpointed_backward_twice(cuda):
    """A retained graph's second backward reads the same checkpoint; the hidden states may have changed since."""
    wl = make_workload("toy", device=cuda, tokens=40)
    x, dout = wl.hidden.clone().requires_grad_(), _randn((wl.T, wl.H), 5).to(cuda)
    fc1 = wl.fc1.clone().requires_grad_()
    out = experts.expert_layer(x, wl.routing_weights, wl.selected, wl.fc2, fc1_1_2_weight=fc1, mapping=wl.mapping,
                               sources=wl.sources, activation_checkpoint="e4m3")
    first = torch.autograd.grad(out, (x, fc1), dout, retain_graph=True)
    with torch.no_grad():
        x.zero_()
    second = torch.autograd.grad(out, (x, fc1), dout)
    for a, b in zip(first, second):
        assert_exact(a, b, "gradient")


def test_a_tokens_output_does_not_depend_on_the_call(cuda):
    """Alone, in threes, and among 3000 others, on whatever tiles: the same bits."""
    C, H, I, T, K = 96, 1040, 528, 3000, 4
    g = torch.Generator().manual_seed(3)
    q = rows8.Experts8.quantize((torch.randn((C, 2 * I, H), device=cuda) * 0.05).to(BF), (torch.randn((C, H, I), device=cuda) * 0.05).to(BF))
    x, w = _randn((T, H), 4).to(cuda), torch.rand((T, K), generator=g).to(BF).to(cuda)
    sel = torch.stack([torch.randperm(C, generator=g)[:K] for _ in range(T)]).to(cuda)
    want = placemoe_amd.expert_layer_rows8(x, w, sel, q)
    for n, upto in ((1, 150), (3, 300), (40, 400), (500, T)):
        got = [placemoe_amd.expert_layer_rows8(x[t:t + n], w[t:t + n], sel[t:t + n], q) for t in range(0, upto, n)]
        assert_exact(torch.cat(got), want[:upto], f"calls of {n} tokens")
