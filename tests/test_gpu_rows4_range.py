"""Products with 4-bit weights at the ends of the exponents' range, against the 64-bit oracle.

Tolerances as in tests/test_gpu_rows4.py: sums in fp32 of products that the 4 x 4
instruction takes whole and the 8 x 4 one cuts (``_bound``), one rounding of the result.
"""

import math

import numpy as np
import pytest
import torch

from oracle import rows4_oracle as O
from oracle import rows8_oracle as O8
from placemoe_amd import rows4, rows8
from tests.test_gpu_rows4 import BF, _offsets, _randn, _write
from tests.test_gpu_rows8_sums import _bound

pytestmark = pytest.mark.gpu


def _scaled(shape, seed, exp):
    half = exp // 2  # (two factors: 2^-130 is no fp32 normal number)
    return (_randn(shape, seed, torch.float32) * 2.0**half * 2.0 ** (exp - half)).to(BF)


def _values(q, bits, K):
    return O8.values(q.codes.cpu(), q.scales.cpu()) if bits == 8 else O.values(q.codes.cpu(), q.scales.cpu(), K)


def _product_limits(va, vb, bits):
    exact, tol = _bound(va, vb)
    if bits == 4:
        tol = np.abs(va) @ np.abs(vb).T * (9 * math.ceil(va.shape[1] / 64)) * 2.0**-24
    return exact, tol + (np.abs(exact) + tol) * torch.finfo(BF).eps / 2


@pytest.mark.parametrize("rows", [3, 40, 700])
@pytest.mark.parametrize("x_exp,w_exp", [(-118, 110), (-126, 118), (-130, 121), (118, -110), (122, -116), (120, -130)])
def test_products_at_the_ends_of_the_range(cuda, x_exp, w_exp, rows):
    """Blocks beside 2^-127 and near 2^120, in products of ordinary size."""
    K, I = 288, 64
    x, w = _scaled((rows, K), 1, x_exp), _scaled((1, 2 * I, K), 2, w_exp)
    qw, off = rows4.quantize_rows4(w.to(cuda)), _offsets([rows]).to(cuda)
    vw = O.values(qw.codes[0].cpu(), qw.scales[0].cpu(), K)
    print(f"rows4 range {x_exp} {w_exp} {rows}", flush=True)
    for bits in (8, 4):
        qx = _write(x.to(cuda), bits)
        exact, limit = _product_limits(_values(qx, bits, K), vw, bits)
        got = rows4.group_gemm_nt_rows4(qx, qw, off).double().cpu().numpy()
        assert (np.abs(got - exact) <= limit * 1.0001).all(), bits
    # fc1: fp32 sums of K products, each exact; silu(gate) to 2^-17 and 1.1 of the gate's error; half a step of e4m3
    qx = rows8.quantize_rows(x.to(cuda))
    vx = _values(qx, 8, K)
    exact, size = vx @ vw.T, np.abs(vx) @ np.abs(vw).T * K * 2.0**-23
    gate, up = exact[:, :I], exact[:, I:]
    with np.errstate(over="ignore"):
        act = gate / (1 + np.exp(-gate)) * up
    slack = 1.1 * size[:, :I] * np.abs(up) + np.abs(gate) * size[:, I:] + np.abs(act) * 2.0**-16
    q = rows4.gemm_fc1_swiglu_rows4(qx, qw, off)
    unit = np.repeat(2.0 ** (q.scales.cpu().permute(1, 0, 2).reshape(rows, -1)[:, :I // 32].numpy().astype(np.float64) - 127), 32, axis=1)
    v = O8.values(q.codes.cpu(), q.scales.cpu())
    assert (np.abs(v - act) <= (slack + np.maximum((np.abs(act) + slack) * 2.0**-4, unit * 2.0**-10)) * 1.0001).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("a_byte,b_byte", [(0, 254), (254, 0), (1, 252), (127, 127), (60, 190), (0, 200)])
def test_every_pair_of_codes_beside_the_outermost_powers(cuda, bits, a_byte, b_byte):
    """Row i has code i in column 0, column j of C code j beside it: each product alone, exact in fp32."""
    K, codes = 32, 256 if bits == 8 else 16
    a = torch.zeros((codes, K if bits == 8 else K // 2), dtype=torch.uint8)
    a[:, 0] = torch.arange(codes)
    if bits == 8:
        a[torch.arange(256) % 128 == 127, 0] = 0  # e4m3's NaN
    b = torch.zeros((1, 16, K // 2), dtype=torch.uint8)
    b[0, :, 0] = torch.arange(16)
    a_s, b_s = (torch.full((*s, 16), 127, dtype=torch.uint8) for s in ((1, codes), (1, 1, 16)))
    a_s[..., 0], b_s[..., 0] = a_byte, b_byte
    qa = rows8.Rows8(a.view(torch.float8_e4m3fn).to(cuda), a_s.to(cuda), BF) if bits == 8 else rows4.Rows4(a.to(cuda), a_s.to(cuda), K, BF)
    qb = rows4.Rows4(b.to(cuda), b_s.to(cuda), K, BF)
    got = rows4.group_gemm_nt_rows4(qa, qb, torch.tensor([0, codes], dtype=torch.int32, device=cuda))
    va, vb = _values(qa, bits, K)[:, :1], O.values(qb.codes[0].cpu(), qb.scales[0].cpu(), K)[:, :1]
    want = torch.from_numpy(va @ vb.T)
    # products below 2^-126 may count as 0
    exact = want.float().to(BF).double()
    assert ((got.double().cpu() == exact) | ((want.abs() < 2.0**-126) & (got.double().cpu().abs() <= 2.0**-126))).all()


def test_weights_that_4_bits_round_past_the_range(cuda):
    """bf16's largest values are 2^128 in 4 bits: NT multiplies them as that, fc1, in bf16, as infinities; the
    other columns have what they have without."""
    K, I = 64, 64
    x, w = _randn((5, K), 1, BF, 2.0**-100), _randn((1, 2 * I, K), 2)
    loud = w.clone()
    loud[0, 40, 7] = torch.finfo(BF).max
    off = _offsets([5]).to(cuda)
    qw, ql = (rows4.quantize_rows4(t.to(cuda)) for t in (w, loud))
    vl = O.values(ql.codes[0].cpu(), ql.scales[0].cpu(), K)
    assert vl[40, 7] == 2.0**128
    others = torch.arange(2 * I, device=cuda) != 40
    for bits in (8, 4):
        qx = _write(x.to(cuda), bits)
        got = rows4.group_gemm_nt_rows4(qx, ql, off)
        assert torch.equal(got[:, others], rows4.group_gemm_nt_rows4(qx, qw, off)[:, others])
        exact, limit = _product_limits(_values(qx, bits, K), vl, bits)
        assert (np.abs(got.double().cpu().numpy() - exact) <= limit * 1.0001).all()
    act = rows8.dequantize_rows(rows4.gemm_fc1_swiglu_rows4(rows8.quantize_rows(x.to(cuda)), ql, off))
    plain = rows8.dequantize_rows(rows4.gemm_fc1_swiglu_rows4(rows8.quantize_rows(x.to(cuda)), qw, off))
    assert torch.equal(act[:, :32], plain[:, :32])  # the other block of 32 activations
    assert not act[:, 40].isfinite().any()
