"""Operands of another kind are refused by name before anything else is looked at."""

import pytest
import torch

import placemoe_amd
from placemoe_amd import rows4, rows8
from tests.test_rows4 import BF, _rows, _rows8


def test_operands_of_another_kind_are_refused():
    plain, i32 = torch.zeros((2, 32), dtype=BF), torch.zeros(3, dtype=torch.int32)
    a4, a8, w4, w8 = _rows((2, 32)), _rows8((2, 32)), _rows((2, 32, 32)), _rows8((2, 32, 32))
    layer = lambda w: placemoe_amd.expert_layer_rows4(plain, plain[:, :1], torch.zeros((2, 1), dtype=torch.int64), w)  # noqa: E731
    for name, call in (
        ("a", lambda: rows4.group_gemm_nt_rows4(plain, w4, i32)),
        ("b", lambda: rows4.group_gemm_nt_rows4(a8, w8, i32)),
        ("b", lambda: rows4.group_gemm_nt_rows4(a4, plain, i32)),
        ("x", lambda: rows4.gemm_fc1_swiglu_rows4(plain, w4, i32)),
        ("x", lambda: rows4.gemm_fc1_swiglu_rows4(a4, w4, i32)),
        ("w", lambda: rows4.gemm_fc1_swiglu_rows4(a8, plain, i32)),
        ("q", lambda: rows4.dequantize_rows4(plain)),
        ("weights", lambda: layer(plain)),
        ("weights", lambda: layer(rows8.Experts8(w8, w8))),
        ("gate_up", lambda: layer(rows4.Experts4(plain, w4))),
        ("down", lambda: layer(rows4.Experts4(w4, plain))),
        ("down", lambda: layer(rows4.Experts4(w4, w8))),
    ):
        with pytest.raises(AssertionError, match=f"^{name} must be (Rows8 or Rows4|Rows8|Rows4|Experts4), got"):
            call()
