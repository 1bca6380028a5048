"""Rows in 4 bits on the GPU against the 64-bit oracle.

Tolerances, from the arithmetic:

* writing and reading back are exact by definition (one rounding to the nearest
  value, powers of two): codes, exponents and values must be equal;
* a product of two 4-bit rows: every eight neighbouring products are multiples
  of a quarter of the blocks' powers of two, at most 144 quarters each, so that
  the matrix instruction's cut below 2^-13 of the largest takes nothing; their
  sums are added in fp32 (nine roundings per 64 columns, each half a step of
  2^-23 of what has been added up), and the result is rounded once;
* a product of 8-bit rows with 4-bit ones: the cut as well, less than 7 * 2^-13
  of the largest product of each eight;
* products of small integers, whose every sum is exact in fp32, must be equal
  after the one rounding.
"""

import math

import numpy as np
import pytest
import torch

import placemoe_amd
from oracle import moe_oracle
from oracle import rows4_oracle as O
from oracle import rows8_oracle as O8
from placemoe_amd import _capi, experts, kernels, rows4, rows8
from tests.helpers import assert_bf16_close, assert_exact
from tests.test_gpu_rows8 import FEW, LARGE, LAYOUTS, SUBNORMAL, WIDE, _layer_oracle, _near, _offsets, _randn, _same, _spiky
from tests.test_gpu_rows8_sums import _bound, _cancelling, _loud, _spread

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def _check_written(q, x, name):
    v, scales = O.quantize(x)
    assert torch.equal(q.scales.cpu(), scales), f"{name}: exponents"
    _same(O.values(q.codes.cpu(), q.scales.cpu(), q.columns), v, name)
    if q.columns % 2:
        assert (q.codes.cpu()[:, -1] < 16).all(), f"{name}: past the row's end"
    return v


def _levels(shape, seed, dtype=BF):
    """Values that 4 bits hold beside 2^0, among them 6 in every block, doubled (so that they are whole)."""
    g = torch.Generator().manual_seed(seed)
    x = LEVELS[torch.randint(0, 8, shape, generator=g)] * (2 * torch.randint(0, 2, shape, generator=g) - 1) * 2
    x[..., ::32] = 12
    return x.to(dtype)


def _ints8(shape, seed, dtype=BF):
    """Small integers, which e4m3 holds beside any power of two up to 2^3."""
    return torch.randint(-7, 8, shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _as8(q):
    """The same values in e4m3, which holds them all, beside the same powers of two."""
    *lead, R, n = q.codes.shape
    both = torch.stack((q.codes & 15, q.codes >> 4), -1).flatten(-2)[..., : q.columns].long()
    v = LEVELS.to(q.codes.device)[both & 7] * torch.where(both >= 8, -1.0, 1.0)
    return rows8.Rows8(v.to(torch.float8_e4m3fn).contiguous(), q.scales, q.dtype)


def _padded(layout):
    """A layout of the 8-bit tests with its depth a multiple of 32."""
    counts, N, K = layout
    return counts, N, -(-K // 32) * 32


def _write(x, bits):
    return rows8.quantize_rows(x) if bits == 8 else rows4.quantize_rows4(x)


def _rows(shape, seed, bits, dtype=BF):
    return (_ints8 if bits == 8 else _levels)(shape, seed, dtype)


# ---------------------------------------------------------------------------
# Writing and reading back
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("R,N", [(1, 1), (1, 2), (1, 8), (2, 7), (3, 31), (5, 33), (33, 512), (31, 513), (65, 1411), (4, 2048), (40, 100)])
def test_written_and_read_back_exactly(cuda, R, N, dtype):
    print(f"rows4 {R}x{N} {dtype}", flush=True)
    x = _spiky((R, N), R * 31 + N, dtype)
    q = rows4.quantize_rows4(x.to(cuda))
    assert q.shape == (R, N) and q.dtype == dtype and q.codes.shape == (R, (N + 1) // 2)
    v = _check_written(q, x, f"{R}x{N}")
    most = float(torch.finfo(dtype).max)
    _same(rows4.dequantize_rows4(q), np.clip(v, -most, most), "read back")


@pytest.mark.parametrize("dtype", [BF, F16])
def test_every_16_bit_value(cuda, dtype):
    """Each finite value of the type, alone in its block and beside another one eight times as large."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.isfinite()]
    rows = torch.zeros((x.numel(), 32), dtype=dtype)
    rows[:, 5] = x
    rows[:, 30] = x
    rows[1::2, 17] = (x[1::2].float() * 8).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    rows = rows.view(-1, 512)[: x.numel() // 16]
    q = rows4.quantize_rows4(rows.to(cuda))
    v = _check_written(q, rows, "every value")
    most = float(torch.finfo(dtype).max)
    _same(rows4.dequantize_rows4(q), np.clip(v, -most, most), "read back")


@pytest.mark.parametrize("dtype", [BF, F16])
def test_a_block_that_is_not_finite_is_nan(cuda, dtype):
    x = _randn((6, 99), 5, dtype)
    x[0, 3], x[1, 40], x[2, 98] = math.inf, -math.inf, math.nan
    x[3, 32:64] = math.inf
    x[4] = math.nan
    q = rows4.quantize_rows4(x.to(cuda))
    _check_written(q, x, "not finite")
    back = rows4.dequantize_rows4(q).cpu()
    bad = torch.nn.functional.pad(~x.isfinite(), (0, 29)).view(6, 4, 32).any(-1).repeat_interleave(32, 1)[:, :99]
    assert torch.equal(back.isnan(), bad)
    # zeros beside the exponent byte that stands for NaN are NaN too
    zeros = rows4.Rows4(torch.zeros_like(q.codes), q.scales, 99, dtype)
    assert torch.equal(rows4.dequantize_rows4(zeros).cpu().isnan(), bad)


def test_every_code_beside_every_power(cuda):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)[:, :256]  # 512 columns: every pair of codes
    scales = torch.arange(256, dtype=torch.uint8).view(1, 256, 1).repeat(1, 1, 16)
    want = O.values(codes, scales, 512)
    for dtype in (BF, F16):
        got = rows4.dequantize_rows4(rows4.Rows4(codes.to(cuda), scales.to(cuda), 512, dtype)).cpu()
        most = float(torch.finfo(dtype).max)
        _same(got, torch.from_numpy(np.clip(want, -most, most)).to(dtype).double().numpy(), str(dtype))


def test_strided_unaligned_and_grouped_rows(cuda):
    big = _randn((70, 1500), 6)
    dev = big.to(cuda)
    for part in (slice(0, 700), slice(1, 702), slice(3, 4), slice(9, 1410)):
        _check_written(rows4.quantize_rows4(dev[:, part]), big[:, part], f"columns {part}")
    _check_written(rows4.quantize_rows4(dev[::3, 5:600]), big[::3, 5:600], "every third row")
    one = rows4.quantize_rows4(dev.view(-1)[7: 7 + 2 * 515].view(2, 515))
    _check_written(one, big.view(-1)[7: 7 + 2 * 515].view(2, 515), "odd address")
    w = _randn((3, 37, 131), 7)
    q = rows4.quantize_rows4(w.to(cuda))
    assert q.shape == (3, 37, 131) and q.scales.shape == (3, 1, 37, 16)
    back = rows4.dequantize_rows4(q)
    assert back.shape == (3, 37, 131)
    for g in range(3):
        part = rows4.Rows4(q.codes[g], q.scales[g], 131, BF)
        _same(back[g], _check_written(part, w[g], f"group {g}"), f"group {g} read back")
    for bad in (dev.t(), dev[:, ::2], dev[0].expand(4, 1500), w.to(cuda).transpose(1, 2)):
        with pytest.raises(AssertionError):
            rows4.quantize_rows4(bad)
    with pytest.raises(AssertionError):
        rows4.quantize_rows4(dev.float())


def test_nothing_to_write(cuda):
    for shape in ((0, 64), (5, 0), (0, 0), (0, 4, 64), (2, 0, 64)):
        q = rows4.quantize_rows4(torch.empty(shape, dtype=BF, device=cuda))
        assert q.shape == shape and tuple(q.scales.shape) == rows8.scales_shape(shape)
        assert rows4.dequantize_rows4(q).shape == shape


def test_many_rows_are_written_like_few(cuda):
    """Eight rows to a wave against two."""
    x = _randn((4, 5003, 520), 8).to(cuda)
    q = rows4.quantize_rows4(x)
    back = rows4.dequantize_rows4(q)
    for g in range(4):
        for r in (0, 31, 2500, 4996):
            one = rows4.quantize_rows4(x[g, r:r + 7])
            assert torch.equal(q.codes[g, r:r + 7], one.codes) and torch.equal(q.scales[g, :, r:r + 7], one.scales)
            assert_exact(back[g, r:r + 7], rows4.dequantize_rows4(one))


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------


def _exact_product(a, b, off):
    return torch.cat([a[off[g]:off[g + 1]].double() @ b[g].double().t() for g in range(b.shape[0])])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("name", LAYOUTS)
def test_products_of_integers_are_exact(cuda, name, dtype, bits):
    counts, N, K = _padded(LAYOUTS[name])
    print(f"rows4 gemm {name} {bits} {dtype}", flush=True)
    M, G = sum(counts), len(counts)
    a, b = _rows((M, K), 1, bits, dtype).to(cuda), _levels((G, N, K), 2, dtype).to(cuda)
    off = _offsets(counts)
    # (an eighth: |sum| <= 12 * 1.5 * K stays within fp16)
    b = b / 8
    got = rows4.group_gemm_nt_rows4(_write(a, bits), rows4.quantize_rows4(b), off.to(cuda))
    # multiples of 1/4 below 2^16: fp32 holds every sum, and one rounding follows
    assert_exact(got, _exact_product(a, b, off).float().to(dtype), name)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("layouts,name", [(WIDE, n) for n in WIDE] + [(LARGE, n) for n in LARGE] + [(FEW, n) for n in FEW])
def test_wide_products_of_integers_are_exact(cuda, layouts, name, bits):
    counts, N, K = _padded(layouts[name])
    print(f"rows4 wide {name} {bits}", flush=True)
    M, G = sum(counts), len(counts)
    a, b = _rows((M, K), 1, bits).to(cuda), _levels((G, N, K), 2).to(cuda)
    off = _offsets(counts)
    got = rows4.group_gemm_nt_rows4(_write(a, bits), rows4.quantize_rows4(b), off.to(cuda))
    assert_exact(got, _exact_product(a, b, off).float().to(BF), name)


@pytest.mark.parametrize("kind", [_randn, _spread, _loud, _cancelling])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("counts,N,K", [([5, 0, 9], 40, 160), ([300, 170], 264, 544)])
def test_products_stay_within_their_bound(cuda, counts, N, K, dtype, bits, kind):
    M, G = sum(counts), len(counts)
    print(f"rows4 sums {kind.__name__} {bits} {counts} {N} {K} {dtype}", flush=True)
    a, b, off = kind((M, K), 1, dtype), _randn((G, N, K), 2, dtype, 0.1), _offsets(counts)
    qa, qb = _write(a.to(cuda), bits), rows4.quantize_rows4(b.to(cuda))
    got = rows4.group_gemm_nt_rows4(qa, qb, off.to(cuda))
    va = O8.values(qa.codes.cpu(), qa.scales.cpu()) if bits == 8 else O.values(qa.codes.cpu(), qa.scales.cpu(), K)
    for g in range(G):
        rows = slice(int(off[g]), int(off[g + 1]))
        if rows.stop > rows.start:
            vb = O.values(qb.codes[g].cpu(), qb.scales[g].cpu(), K)
            exact, tol = _bound(va[rows], vb)
            if bits == 4:  # nothing is cut
                tol = np.abs(va[rows]) @ np.abs(vb).T * (9 * math.ceil(K / 64)) * 2.0**-24
            _near(got[rows], exact, tol, dtype, f"group {g}")


@pytest.mark.parametrize("bits", [8, 4])
def test_a_block_that_is_nan_reaches_its_row_or_column_alone(cuda, bits):
    for rows in (3, 150, 1200):
        N, K = 136, 288
        a, b = _rows((rows, K), 1, bits).to(cuda), _levels((1, N, K), 2).to(cuda)
        qa, qb = _write(a, bits), rows4.quantize_rows4(b)
        want = rows4.group_gemm_nt_rows4(qa, qb, _offsets([rows]).to(cuda)).cpu()
        qb.scales[0, 0, 77, 8] = 255  # the last block of row 77 of b
        qb.codes[0, 77, 128:] = 0  # zeros beside NaN are NaN
        if bits == 4:
            qa.scales[0, rows // 2, 3] = 255
        else:
            qa.codes.view(torch.uint8)[rows // 2, 97] = 0x7f
        got = rows4.group_gemm_nt_rows4(qa, qb, _offsets([rows]).to(cuda)).cpu()
        nan = torch.zeros((rows, N), dtype=torch.bool)
        nan[:, 77] = True
        nan[rows // 2] = True
        assert torch.equal(got.isnan(), nan), f"{rows} rows"
        assert_exact(got[~nan], want[~nan], f"{rows} rows")


def test_a_block_that_is_nan_in_fc1(cuda):
    """Zeros beside the byte that stands for NaN: the gate or up value of its row of w, and the 32 activations that share its exponent."""
    for rows in (3, 150, 1200):
        I, H = 144, 288
        x, w = rows8.quantize_rows(_randn((rows, H), 1).to(cuda)), rows4.quantize_rows4(_randn((1, 2 * I, H), 2, std=0.1).to(cuda))
        want = rows8.dequantize_rows(rows4.gemm_fc1_swiglu_rows4(x, w, _offsets([rows]).to(cuda))).cpu()
        for at in (77, I + 77):
            w.scales[0, 0, at, 8] = 255
            w.codes[0, at, 128:] = 0
        got = rows8.dequantize_rows(rows4.gemm_fc1_swiglu_rows4(x, w, _offsets([rows]).to(cuda))).cpu()
        assert got[:, 77].isnan().all() and not got[:, :64].isnan().any() and not got[:, 96:].isnan().any()
        assert_exact(got[:, :64], want[:, :64]), assert_exact(got[:, 96:], want[:, 96:])


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_of_no_group_are_left_alone(cuda, bits):
    a, w = _rows((300, 64), 1, bits).to(cuda), _levels((2, 32, 64), 2).to(cuda)
    qa, qb = _write(a, bits), rows4.quantize_rows4(w)
    stream = torch.cuda.current_stream().cuda_stream
    for offsets in ([3, 20, 290], [0, 300, 300], [5, 5, 5], [-7, 20, 1 << 30], [40, 30, 20]):
        c = torch.full((300, 32), 7.5, dtype=BF, device=cuda)
        off = torch.tensor(offsets, dtype=torch.int32, device=cuda)
        _capi.call("pmx_rows4_group_gemm_nt", qa.codes.data_ptr(), qa.scales.data_ptr(), bits, qb.codes.data_ptr(),
                   qb.scales.data_ptr(), off.data_ptr(), 2, 300, 32, 64, c.data_ptr(), stream)
        lo, mid, hi = (min(max(o, 0), 300) for o in offsets)
        want = torch.full((300, 32), 7.5, dtype=BF)
        if lo <= mid <= hi:  # descending offsets: nothing is written
            want[lo:mid] = (a[lo:mid].double() @ w[0].double().t()).to(BF).cpu()
            want[mid:hi] = (a[mid:hi].double() @ w[1].double().t()).to(BF).cpu()
        assert_exact(c, want, str(offsets))


@pytest.mark.parametrize("bits", [8, 4])
def test_a_row_depends_on_itself_and_its_copy_alone(cuda, bits):
    """The same row in calls of one, a few, and many rows, in any slot, on every tiling: the same bits."""
    K, N = 1120, 248
    a, w = _randn((6400, K), 1).to(cuda), _randn((1, N, K), 2, std=0.05).to(cuda)
    ref = rows4.group_gemm_nt_rows4(_write(a.repeat(4, 1), bits), rows4.quantize_rows4(w),
                                    torch.tensor([0, 25600], dtype=torch.int32, device=cuda))[:6400]
    for rows, slots in ((1, 1), (16, 1), (20, 3), (130, 2), (300, 5), (400, 200), (2600, 1), (6400, 10)):
        counts = [0] * slots
        counts[slots // 2] = rows
        ww = torch.randn((slots, N, K), device=cuda).to(BF)
        ww[slots // 2] = w[0]
        got = rows4.group_gemm_nt_rows4(_write(a[:rows], bits), rows4.quantize_rows4(ww), _offsets(counts).to(cuda))
        assert_exact(got, ref[:rows], f"{rows} rows in slot {slots // 2}")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("counts,I,H,T", [([1], 16, 32, 1), ([3, 0, 30, 7], 48, 160, 20), ([130, 90, 61], 144, 544, 100),
                                          ([300, 280], 208, 288, 290), ([40] * 3, 640, 64, 50), ([2] * 100, 224, 288, 60)])
def test_fc1_swiglu(cuda, counts, I, H, T, dtype):
    G, A = len(counts), sum(counts)
    print(f"rows4 fc1 {counts[:4]} I={I} H={H} {dtype}", flush=True)
    g = torch.Generator().manual_seed(A + I)
    x, w = _randn((T, H), 1, dtype), _randn((G, 2 * I, H), 2, dtype, 1.5 / math.sqrt(H))
    token = torch.randint(0, T, (A,), generator=g).to(torch.int32)
    row_w = (0.05 + torch.rand(A, generator=g)).to(dtype)
    off = _offsets(counts)
    qx, qw = rows8.quantize_rows(x.to(cuda)), rows4.quantize_rows4(w.to(cuda))
    act = rows4.gemm_fc1_swiglu_rows4(qx, qw, off.to(cuda), token.to(cuda), row_w.to(cuda))
    assert act.shape == (A, I) and act.codes.dtype == torch.float8_e4m3fn
    vx = O8.values(qx.codes.cpu(), qx.scales.cpu())[token.numpy()]
    vw = np.stack([O.values(qw.codes[k].cpu(), qw.scales[k].cpu(), H) for k in range(G)])
    gu, _ = O8.grouped_nt(vx, vw, off.numpy())
    gate, up = gu[:, :I], gu[:, I:]
    rw = row_w.double().numpy()[:, None]
    exact = gate / (1 + np.exp(-gate)) * up * rw
    # sums in fp32: at most a rounding per product, each half a step of 2^-23 of what has been added up; |d silu| <= 1.1
    size = np.concatenate([np.abs(vx[off[k]:off[k + 1]]) @ np.abs(vw[k]).T for k in range(G)])
    slack = rw * (1.1 * size[:, :I] * np.abs(up) + np.abs(gate) * size[:, I:]) * H * 2.0**-24 + np.abs(exact) * 2.0**-17
    low, high = np.abs(exact) - slack, np.abs(exact) + slack
    e_low, e_high = O8.block_exponents(np.maximum(low, 0), "e4m3"), O8.block_exponents(high, "e4m3")
    nb = e_low.shape[1]
    bytes_ = act.scales.cpu().permute(1, 0, 2).reshape(A, -1)
    e = bytes_[:, :nb].numpy().astype(np.int64) - 127
    assert ((e >= e_low) & (e <= e_high)).all(), "exponents"
    got = O8.values(act.codes.cpu(), act.scales.cpu())
    unit = np.repeat(2.0**e, 32, axis=1)[:, :I]
    # e4m3: half a step is 2^-4 of the value, at least 2^-10 of the unit
    tol = slack + np.maximum((np.abs(exact) + slack) * 2.0**-4, unit * 2.0**-10)
    assert (np.abs(got - exact) <= tol * 1.0001).all(), f"codes: {(np.abs(got - exact) - tol).max()}"
    assert (bytes_[:, nb:] == 127).all(), "past the last column"
    plain = rows4.gemm_fc1_swiglu_rows4(rows8.Rows8(qx.codes[token.long()].contiguous(), qx.scales[:, token.long()].contiguous(), dtype),
                                        qw, off.to(cuda), None, row_w.to(cuda))
    assert torch.equal(plain.codes.view(torch.uint8), act.codes.view(torch.uint8)), "rows in place"


@pytest.mark.parametrize("name", WIDE)
def test_wide_fc1_equals_single_copies(cuda, name):
    """A copy's rows among those of many others, and alone on narrow tiles (tested against 64 bits): the same bits."""
    counts, N, K = _padded(WIDE[name])
    print(f"rows4 wide fc1 {name}", flush=True)
    A, G, I, T = sum(counts), len(counts), N // 32 * 16, 333
    x = rows8.quantize_rows(_randn((T, K), 3).to(cuda))
    w = rows4.quantize_rows4(_randn((G, 2 * I, K), 4, std=0.06).to(cuda))
    token = torch.randint(0, T, (A,), generator=torch.Generator().manual_seed(5)).to(torch.int32).to(cuda)
    row_w = torch.rand(A, generator=torch.Generator().manual_seed(6)).to(BF).to(cuda)
    off = _offsets(counts)
    act = rows4.gemm_fc1_swiglu_rows4(x, w, off.to(cuda), token, row_w)
    for g in (0, 1, 3, G // 2, G - 2, G - 1):
        rows = slice(int(off[g]), int(off[g + 1]))
        one = rows4.Rows4(w.codes[g:g + 1].contiguous(), w.scales[g:g + 1].contiguous(), K, BF)
        ref = rows4.gemm_fc1_swiglu_rows4(x, one, _offsets([rows.stop - rows.start]).to(cuda), token[rows].clone(), row_w[rows].clone())
        assert torch.equal(act.codes.view(torch.uint8)[rows], ref.codes.view(torch.uint8)), f"copy {g}"
        assert torch.equal(act.scales[:, rows], ref.scales), f"copy {g}"


# Sixteen kinds of rests past whole 256s, ten of each: calls whose short rests are launched apart
RESTS = ([0, 1, 127, 128, 129, 255, 256, 257, 383, 384, 385, 511, 512, 513, 641, 1100] * 10, 512, 2048)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_rests_apart_equal_single_copies(cuda, dtype):
    """Each copy alone runs on other tiles: the same bits; rows before the first group and behind the last stay."""
    counts, N, K = RESTS
    before, behind = 3, 5
    G, M, I = len(counts), before + sum(counts) + behind, N // 2
    off = (_offsets(counts) + before).to(torch.int32)
    x = rows8.quantize_rows(_randn((M, K), 11).to(cuda).to(dtype))
    w = rows4.quantize_rows4(_randn((G, N, K), 12, std=0.06).to(cuda).to(dtype))
    suffix = "_f16" if dtype == F16 else ""
    s, on = torch.cuda.current_stream().cuda_stream, off.to(cuda)
    lib = _capi.load()
    c = torch.full((M, N), -7.0, dtype=dtype, device=cuda)
    assert getattr(lib, "pmx_rows4_group_gemm_nt" + suffix)(
        x.codes.data_ptr(), x.scales.data_ptr(), 8, w.codes.data_ptr(), w.scales.data_ptr(), on.data_ptr(), G, M, N, K, c.data_ptr(),
        s) == _capi.PMX_OK
    act = torch.full((M, I), 0x55, dtype=torch.uint8, device=cuda)
    scales = torch.full((1, M, 16), 0x55, dtype=torch.uint8, device=cuda)
    assert getattr(lib, "pmx_rows4_gemm_fc1_swiglu" + suffix)(
        x.codes.data_ptr(), x.scales.data_ptr(), M, None, w.codes.data_ptr(), w.scales.data_ptr(), on.data_ptr(), G, M, K, I, None,
        act.data_ptr(), scales.data_ptr(), s) == _capi.PMX_OK
    for rows in (slice(0, before), slice(M - behind, M)):
        assert (c[rows] == -7).all() and (act[rows] == 0x55).all() and (scales[:, rows] == 0x55).all()
    for g, n in enumerate(counts):
        rows = slice(int(off[g]), int(off[g]) + n)
        one = rows4.Rows4(w.codes[g:g + 1].contiguous(), w.scales[g:g + 1].contiguous(), K, dtype)
        xg = rows8.Rows8(x.codes[rows].contiguous(), x.scales[:, rows].contiguous(), dtype)
        alone = _offsets([n]).to(cuda)
        assert_exact(c[rows], rows4.group_gemm_nt_rows4(xg, one, alone), f"copy {g}")
        ref = rows4.gemm_fc1_swiglu_rows4(xg, one, alone)
        assert torch.equal(act[rows], ref.codes.view(torch.uint8)) and torch.equal(scales[:, rows], ref.scales), f"copy {g}"


@pytest.mark.parametrize("rows", [3, 100, 1500, 9000])
@pytest.mark.parametrize("I", [16, 48, 144, 512, 528])
def test_fc1_writes_every_scale(cuda, I, rows):
    G, H = 3, 64
    x = rows8.quantize_rows(_randn((rows, H), 1).to(cuda))
    w = rows4.quantize_rows4(_randn((G, 2 * I, H), 2).to(cuda))
    junk = torch.full((1 << 24,), 3, dtype=torch.uint8, device=cuda)  # what the outputs' memory held before
    del junk
    act = rows4.gemm_fc1_swiglu_rows4(x, w, _offsets([rows - 2, 1, 1]).to(cuda))
    assert (act.scales.permute(1, 0, 2).reshape(rows, -1)[:, -(-I // 32):] == 127).all()


def test_token_outside_reads_as_zeros(cuda):
    qx, qw = rows8.quantize_rows(_randn((4, 64), 1).to(cuda)), rows4.quantize_rows4(_randn((1, 64, 64), 2).to(cuda))
    token = torch.tensor([0, -1, 4, 1 << 30, 3], dtype=torch.int32, device=cuda)
    act = rows8.dequantize_rows(rows4.gemm_fc1_swiglu_rows4(qx, qw, _offsets([5]).to(cuda), token))
    assert (act[1:4] == 0).all() and (act[0] != 0).any() and (act[4] != 0).any()


def test_product_refusals(cuda):
    a8, a4 = rows8.quantize_rows(_randn((8, 64), 1).to(cuda)), rows4.quantize_rows4(_randn((8, 64), 1).to(cuda))
    b, off = rows4.quantize_rows4(_randn((2, 32, 64), 2).to(cuda)), _offsets([4, 4]).to(cuda)
    half = rows4.quantize_rows4(_randn((2, 32, 64), 2, F16).to(cuda))
    odd = rows4.quantize_rows4(_randn((2, 32, 72), 2).to(cuda))
    swap = rows4.Rows4(b.codes, b.scales, 62, BF)  # 32 bytes hold 63 or 64
    for bad in (
        lambda: rows4.group_gemm_nt_rows4(rows8.quantize_rows(_randn((8, 64), 1).to(cuda), "int8"), b, off),
        lambda: rows4.group_gemm_nt_rows4(a4, half, off),
        lambda: rows4.group_gemm_nt_rows4(a8, half, off),
        lambda: rows4.group_gemm_nt_rows4(a4, b, off.long()),
        lambda: rows4.group_gemm_nt_rows4(a4, b, off[:2].contiguous()),
        lambda: rows4.group_gemm_nt_rows4(a4, odd, off),
        lambda: rows4.group_gemm_nt_rows4(a4, a4, off),
        lambda: rows4.group_gemm_nt_rows4(a4, swap, off),
        lambda: rows4.group_gemm_nt_rows4(a4, b.to("cpu"), off),
        lambda: rows4.group_gemm_nt_rows4(a4, b, off.cpu()),
        lambda: rows4.group_gemm_nt_rows4(a4, rows4.Rows4(b.codes, b.scales[:, :, :16].contiguous(), 64, BF), off),
        lambda: rows4.group_gemm_nt_rows4(a4, rows4.Rows4(b.codes.transpose(0, 1).contiguous().transpose(0, 1), b.scales, 64, BF), off),
        lambda: rows4.gemm_fc1_swiglu_rows4(a4, b, off),
        lambda: rows4.gemm_fc1_swiglu_rows4(a8, b, off, torch.zeros(8, dtype=torch.int64, device=cuda)),
        lambda: rows4.gemm_fc1_swiglu_rows4(a8, b, off, None, torch.ones(7, dtype=BF, device=cuda)),
        lambda: rows4.dequantize_rows4(a8),
        lambda: rows4.dequantize_rows4(swap),
    ):
        with pytest.raises(AssertionError):
            bad()
    a72 = rows8.quantize_rows(_randn((8, 72), 1).to(cuda))
    with pytest.raises(ValueError):  # 72 columns: not whole blocks
        rows4.group_gemm_nt_rows4(a72, odd, off)
    with pytest.raises(ValueError):  # 12 columns of C
        rows4.group_gemm_nt_rows4(a4, rows4.quantize_rows4(_randn((2, 12, 64), 2).to(cuda)), off)
    shifted = torch.zeros(2 * 32 * 32 + 8, dtype=torch.uint8, device=cuda)[8:].view(2, 32, 32)
    with pytest.raises(ValueError):  # alignment
        rows4.group_gemm_nt_rows4(a4, rows4.Rows4(shifted, b.scales, 64, BF), off)


def test_products_without_rows(cuda):
    b = rows4.quantize_rows4(_randn((2, 32, 64), 2).to(cuda))
    off = torch.zeros(3, dtype=torch.int32, device=cuda)
    for bits in (8, 4):
        a = _write(torch.empty((0, 64), dtype=BF, device=cuda), bits)
        assert rows4.group_gemm_nt_rows4(a, b, off).shape == (0, 32)
    assert rows4.gemm_fc1_swiglu_rows4(rows8.quantize_rows(torch.empty((0, 64), dtype=BF, device=cuda)), b, off).shape == (0, 16)


# ---------------------------------------------------------------------------
# Streams, graphs, long tensors
# ---------------------------------------------------------------------------


def _every_op(x, w, offsets):
    """One call of each: x [R, N], w [G, n, N] in 4 bits."""
    q8, q4 = rows8.quantize_rows(x), rows4.quantize_rows4(x)
    act = rows4.gemm_fc1_swiglu_rows4(q8, w, offsets)
    return [q4.codes, q4.scales, rows4.dequantize_rows4(q4), rows4.group_gemm_nt_rows4(q8, w, offsets),
            rows4.group_gemm_nt_rows4(q4, w, offsets), act.codes.view(torch.uint8), act.scales]


def _every_op_case(cuda, R, seed):
    N, G = 1056, 4
    counts = np.random.default_rng(seed).multinomial(R, [1 / G] * G)
    return [_randn((R, N), seed + 2).to(cuda), rows4.quantize_rows4(_randn((G, 96, N), seed + 1).to(cuda)), _offsets(counts).to(cuda)]


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
    """More than 2^32 codes: 500 rows over and over, each repeat the same as the first."""
    n, times, N = 500, 2100, 4128
    assert n * times * N > 2**32
    rows = _randn((n, N), 1).to(cuda)
    ref = rows4.quantize_rows4(rows)
    print("rows4 past 32 bits: writing", flush=True)
    big = rows4.quantize_rows4(rows.repeat(times, 1))
    assert torch.equal(big.codes.view(times, n, -1)[[0, -2, -1]], ref.codes.expand(3, -1, -1))
    assert torch.equal(big.scales.view(-1, times, n, 16)[:, -1], ref.scales)
    print("rows4 past 32 bits: reading back", flush=True)
    back = rows4.dequantize_rows4(big)
    assert_exact(back[-n:], rows4.dequantize_rows4(ref), "read back")
    del back
    half = n * times // 2
    off, off_ref = _offsets([half, half]).to(cuda), _offsets([0, n]).to(cuda)
    b = rows4.quantize_rows4(_randn((2, 64, N), 3).to(cuda))
    print("rows4 past 32 bits: products", flush=True)
    assert_exact(rows4.group_gemm_nt_rows4(big, b, off)[-n:], rows4.group_gemm_nt_rows4(ref, b, off_ref), "4 x 4")
    wide = rows4.quantize_rows4(_randn((2, N, 64), 3).to(cuda))
    few = rows[:, :64].contiguous()
    for bits in (8, 4):
        got = rows4.group_gemm_nt_rows4(_write(few.repeat(times, 1), bits), wide, off)
        assert_exact(got[-n:], rows4.group_gemm_nt_rows4(_write(few, bits), wide, off_ref), f"a long output, {bits} bits")
        del got


# ---------------------------------------------------------------------------
# The serving layer
# ---------------------------------------------------------------------------


def _layer_case(cuda, T, dtype, H=288, I=160, E=12, C=17, K=3, S=4):
    g = torch.Generator().manual_seed(T)
    hidden = _randn((T, H), T, dtype)
    sel = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]) if T else torch.zeros((0, K), dtype=torch.int64)
    w = torch.softmax(torch.randn((T, K), generator=g), -1).to(dtype)
    src = torch.randint(0, S, (T,), generator=g)
    e, s = torch.arange(E), torch.arange(S).unsqueeze(1)
    mapping = torch.where((e < C - E) & (s % 2 == 1), E + e, e).contiguous()
    q = rows4.Experts4.quantize(_randn((C, 2 * I, H), 1, dtype, 0.1).to(cuda), _randn((C, H, I), 2, dtype, 0.1).to(cuda))
    return hidden, sel, w, src, mapping, q


@pytest.mark.parametrize("T", [1, 5, 64, 700])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_layer_over_4_bit_weights(cuda, T, dtype):
    hidden, sel, w, src, mapping, q = _layer_case(cuda, T, dtype)
    print(f"layer rows4 T={T} {dtype}", flush=True)
    seen = []
    got = placemoe_amd.expert_layer_rows4(hidden.to(cuda), w.to(cuda), sel.to(cuda), q, mapping=mapping.to(cuda),
                                          sources=src.to(cuda), recorder=lambda c: seen.append(c.clone()))
    phys = moe_oracle.map_logical_to_physical(mapping.numpy(), src.numpy(), sel.numpy())
    same = rows8.Experts8(_as8(q.gate_up), _as8(q.down))
    exact, tol = _layer_oracle(hidden, w, np.asarray(phys), same, torch.finfo(dtype).eps)
    assert int(seen[0].sum()) == T * sel.shape[1]
    off = np.abs(got.double().cpu().numpy() - exact)
    assert (off <= tol * 1.0001 + SUBNORMAL[dtype]).all(), (off - tol).max()
    # the tolerance itself stays small beside the outputs
    assert np.linalg.norm(tol) <= 0.1 * np.linalg.norm(exact), np.linalg.norm(tol) / np.linalg.norm(exact)
    assert_bf16_close(got, torch.from_numpy(exact), name="out")


@pytest.mark.parametrize("T", [1, 96, 3000])
def test_layer_equals_its_steps(cuda, T):
    """The layer's rows are 24-bit floats, the steps' 16-bit: within the rounding of each row and of the sum."""
    hidden, sel, w, src, mapping, q = _layer_case(cuda, T, BF)
    hidden, sel, w, src, mapping = (t.to(cuda) for t in (hidden, sel, w, src, mapping))
    out = placemoe_amd.expert_layer_rows4(hidden, w, sel, q, mapping=mapping, sources=src)
    C = q.down.shape[0]
    r = kernels.route(sel, C, mapping=mapping, sources=src)
    x, token, row_w = rows8.quantize_rows_routed(hidden, r.pos, w)
    act = rows4.gemm_fc1_swiglu_rows4(x, q.gate_up, r.offsets, token, row_w)
    y = rows4.group_gemm_nt_rows4(act, q.down, r.offsets)
    per = y[r.pos.long()].double()
    tol = per.abs().sum(1) * (2.0**-8 + 2.0**-15) + per.sum(1).abs() * 2.0**-8 + 2.0**-120
    assert ((out.double() - per.sum(1)).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_a_tokens_output_does_not_depend_on_the_call(cuda, dtype):
    hidden, sel, w, src, mapping, q = _layer_case(cuda, 2500, dtype)
    hidden, sel, w, src, mapping = (t.to(cuda) for t in (hidden, sel, w, src, mapping))
    ref = placemoe_amd.expert_layer_rows4(hidden, w, sel, q, mapping=mapping, sources=src)
    for part in (slice(0, 1), slice(7, 8), slice(100, 164), slice(500, 1500)):
        got = placemoe_amd.expert_layer_rows4(hidden[part], w[part].contiguous(), sel[part], q, mapping=mapping, sources=src[part])
        assert_exact(got, ref[part], str(part))


def test_layer_refusals_and_edges(cuda):
    hidden, sel, w, src, mapping, q = _layer_case(cuda, 5, BF)
    hidden, sel, w, src, mapping = (t.to(cuda) for t in (hidden, sel, w, src, mapping))
    call = placemoe_amd.expert_layer_rows4
    with pytest.raises(ValueError, match="expert_layer_rows4 has no backward"):
        call(hidden.clone().requires_grad_(True), w, sel, q, mapping=mapping, sources=src)
    eight = rows8.Experts8(_as8(q.gate_up), _as8(q.down))
    for bad in (
        lambda: call(hidden, w, sel, eight, mapping=mapping, sources=src),
        lambda: placemoe_amd.expert_layer_rows8(hidden, w, sel, q, mapping=mapping, sources=src),
        lambda: call(hidden.half(), w, sel, q, mapping=mapping, sources=src),
        lambda: call(hidden[:, :256], w, sel, q, mapping=mapping, sources=src),
        lambda: call(hidden, w, sel, rows4.Experts4(q.gate_up, q.gate_up), mapping=mapping, sources=src),
        lambda: call(hidden, w, sel, rows4.Experts4(q.gate_up, q.down.to("cpu")), mapping=mapping, sources=src),
        lambda: call(hidden, w, sel, q, sources=src),
        lambda: rows4.Experts4.quantize(_randn((2, 64, 64), 1).to(cuda), _randn((2, 32, 64), 1).to(cuda)),
    ):
        with pytest.raises(AssertionError):
            bad()
    odd = rows4.Experts4.quantize(_randn((2, 96, 64), 1).to(cuda), _randn((2, 64, 48), 1).to(cuda))
    with pytest.raises(ValueError, match="multiples of 32"):
        call(_randn((3, 64), 1).to(cuda), w[:3].contiguous(), sel[:3] % 2, odd)
    empty = call(hidden[:0], w[:0], sel[:0], q, mapping=mapping)
    assert empty.shape == (0, 288)
    bad = sel.clone()
    bad[2, 1] = 12  # no such expert
    call(hidden, w, bad, q, mapping=mapping, sources=src)
    with pytest.raises(ValueError, match="expert id"):
        experts.check_pending_routes(block=True)
    with torch.no_grad():
        call(hidden.clone().requires_grad_(True), w, sel, q, mapping=mapping, sources=src)
    experts.check_pending_routes(block=True)


def test_layer_keeps_what_is_not_finite_to_its_token(cuda):
    hidden, sel, w, src, mapping, q = _layer_case(cuda, 40, BF)
    args = dict(mapping=mapping.to(cuda), sources=src.to(cuda))
    ref = placemoe_amd.expert_layer_rows4(hidden.to(cuda), w.to(cuda), sel.to(cuda), q, **args)
    hidden[11, 5] = math.nan
    hidden[30, 200] = math.inf
    got = placemoe_amd.expert_layer_rows4(hidden.to(cuda), w.to(cuda), sel.to(cuda), q, **args)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[11, 30]] = True
    assert got.cpu()[bad].isnan().all()
    assert_exact(got.cpu()[~bad], ref.cpu()[~bad], "the others")


def test_layers_at_once_and_in_a_graph(cuda):
    cases = []
    for T in (3, 400):
        hidden, sel, w, src, mapping, q = _layer_case(cuda, T, BF)
        cases.append(([hidden.to(cuda), w.to(cuda), sel.to(cuda), q], dict(mapping=mapping.to(cuda), sources=src.to(cuda))))
    call = placemoe_amd.expert_layer_rows4
    want = [call(*a, **k) for a, k in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, call(*cases[i][0], **cases[i][1])))
    torch.cuda.synchronize()
    for i, out in got:
        assert_exact(out, want[i], f"case {i}")
    graphs = []
    for a, k in cases:  # two captured layers, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*a, **k)
        graphs.append((graph, out))
    for turn in range(3):
        for (a, k), (graph, out) in zip(cases, graphs):
            a[0].copy_(_randn(tuple(a[0].shape), 50 + turn).to(cuda))
            graph.replay()
        eager = [call(*a, **k) for a, k in cases]
        torch.cuda.synchronize()
        for i, (_, out) in enumerate(graphs):
            assert_exact(out, eager[i], f"turn {turn}, case {i}")


def test_nothing_waits_for_the_gpu(cuda):
    hidden, sel, w, src, mapping, q = _layer_case(cuda, 64, BF)
    hidden, sel, w, src, mapping = (t.to(cuda) for t in (hidden, sel, w, src, mapping))
    case = _every_op_case(cuda, 100, 3)
    _every_op(*case)
    placemoe_amd.expert_layer_rows4(hidden, w, sel, q, mapping=mapping, sources=src)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        _every_op(*case)
        placemoe_amd.expert_layer_rows4(hidden, w, sel, q, mapping=mapping, sources=src)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
