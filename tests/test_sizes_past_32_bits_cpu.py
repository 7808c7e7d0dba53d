"""Sizes that a 32-bit number does not hold are refused, and not taken for what is left of them.  Tensors without memory stand in
for the large ones: nothing is launched."""
import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flydsl_b200.kernels.grouped_gemm import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad, grouped_linear
from flydsl_b200.kernels.lora import lora_add
from flydsl_b200.kernels.moe_routing import RoutedRows, moe_combine, moe_permute, route_rows, topk_gating

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
WRAPS = 2 ** 32 + 8                              # 8 in 32 bits


def empty(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda")


@contextlib.contextmanager
def refused():
    with FakeTensorMode(), pytest.raises(ValueError, match="must not exceed"):
        yield


@pytest.mark.parametrize("rows", [WRAPS, 2 ** 31 - 1024])
def test_rows(rows):
    for f in (grouped_gemm, grouped_linear):
        with refused():
            f(empty(rows, 8), empty(2, 8, 8), empty(3, dtype=I32))
    with refused():
        grouped_gemm(empty(rows, 8), empty(2, 8, 8), empty(3, dtype=I32), out=empty(rows, 8))
    with refused():
        grouped_gemm_dgrad(empty(rows, 8), empty(2, 8, 8), empty(3, dtype=I32))
    with refused():
        grouped_gemm_wgrad(empty(rows, 8), empty(rows, 8), empty(3, dtype=I32))
    with refused():
        lora_add(empty(rows, 8), empty(rows, 8), empty(2, 8, 8), empty(2, 8, 8), empty(rows, dtype=I32), empty(2, dtype=F32))
    with refused():
        topk_gating(empty(rows, 8), 1)
    with refused():
        route_rows(empty(rows, 1, dtype=I32), 8)
    with refused():
        route_rows(empty(2 ** 24, 1, dtype=I32), 8)
    plan = lambda: RoutedRows(empty(rows, dtype=I32), empty(2, dtype=I32), empty(9, dtype=I32), empty(8, 1, dtype=I32))  # noqa: E731
    with refused():
        moe_combine(empty(rows, 8), empty(8, 1, dtype=F32), plan())
    with refused():
        moe_permute(empty(rows, 8), plan())


def test_columns():
    k = WRAPS
    with refused():
        grouped_gemm(empty(4, k), empty(1, 8, k), empty(2, dtype=I32))
    with refused():
        grouped_gemm_wgrad(empty(4, 8), empty(4, k), empty(2, dtype=I32))
    with refused():
        lora_add(empty(4, 8), empty(4, k), empty(1, 8, k), empty(1, 8, 8), empty(4, dtype=I32), empty(1, dtype=F32))
    with refused():
        lora_add(empty(4, k), empty(4, 8), empty(1, 8, 8), empty(1, k, 8), empty(4, dtype=I32), empty(1, dtype=F32))
    plan = lambda: RoutedRows(empty(4, dtype=I32), empty(2, dtype=I32), empty(9, dtype=I32), empty(4, 1, dtype=I32))  # noqa: E731
    with refused():
        moe_combine(empty(4, 2 ** 30 + 8), empty(4, 1, dtype=F32), plan())
    with refused():
        moe_permute(empty(4, 2 ** 30 + 8, dtype=F32), plan())        # 2^32 + 32 bytes


def test_a_single_number_is_no_matrix():
    with FakeTensorMode(), pytest.raises(ValueError, match="x must have shape"):
        grouped_gemm(empty(), empty(2, 8, 8), empty(3, dtype=I32))
    with FakeTensorMode(), pytest.raises(ValueError, match="dy must have shape"):
        grouped_gemm_wgrad(empty(), empty(4, 8), empty(3, dtype=I32))


def test_c_entries(lib):
    most = 2 ** 31 - 1 - 1024
    assert lib.flymoe_grouped_gemm(None, None, None, None, most + 1, 2, 8, 16, 2, 0, 0, None) == -1
    assert b"2^31" in lib.flymoe_last_error()
    assert lib.flymoe_lora_add(None, None, None, None, None, None, None, None, 0, most + 1, 16, 16, 8, 1, 0, 2, None) == -1
    assert b"2^31" in lib.flymoe_last_error()
    assert lib.flymoe_combine_rows(64, 64, 64, 64, 64, 64, 4, 2, most + 1, 16, 2, None) == -1
    assert b"sizes" in lib.flymoe_last_error()
    assert lib.flymoe_grouped_gemm(None, None, None, None, most, 2, 8, 16, 2, 0, 0, None) == -1
    assert b"null" in lib.flymoe_last_error()
