"""Grouped products: what is refused, before anything is launched."""
import pytest
import torch

from flydsl_b200.kernels.grouped_gemm import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad

BF = torch.bfloat16


def args(rows=4, k=16, n=8, e=2, dtype=BF):
    return (torch.zeros((rows, k), dtype=dtype), torch.zeros((e, n, k), dtype=dtype), torch.zeros((rows, n), dtype=dtype),
            torch.zeros(e + 1, dtype=torch.int32))


def test_shapes_types_and_devices_are_checked():
    x, w, dy, off = args()
    with pytest.raises(ValueError, match="CUDA tensor"):
        grouped_gemm(x, w, off)
    with pytest.raises(ValueError, match="must have shape"):
        grouped_gemm(dy, w, off)
    with pytest.raises(ValueError, match="must have shape"):
        grouped_gemm_dgrad(x, w, off)
    with pytest.raises(ValueError, match="offsets must have shape"):
        grouped_gemm(x, w, off[:2])
    with pytest.raises(ValueError, match="x must have shape"):
        grouped_gemm_wgrad(dy, x[:3], off)
    with pytest.raises(ValueError, match="multiples of 8"):
        grouped_gemm(*(lambda a: (a[0], a[1], a[3]))(args(k=12)))
    with pytest.raises(ValueError, match="experts must be"):
        grouped_gemm_wgrad(dy, x, off[:1])
    with pytest.raises(ValueError, match="experts must be"):
        grouped_gemm(*(lambda a: (a[0], a[1], a[3]))(args(e=1025)))
    with pytest.raises(TypeError):
        grouped_gemm(x, w, [0, 2, 4])


def test_c_entries_refuse_bad_arguments(lib):
    for rows, experts, n, k, dtype, word in ((-1, 2, 8, 16, 2, b"rows"), (4, 0, 8, 16, 2, b"experts"),
                                             (4, 1025, 8, 16, 2, b"experts"), (4, 2, 12, 16, 2, b"multiples of 8"),
                                             (4, 2, 8, 0, 2, b"multiples of 8"), (4, 2, 8, 16, 0, b"dtype"),
                                             (4, 2, 8, 16, 2, b"null pointer")):
        assert lib.flymoe_grouped_gemm(None, None, None, None, rows, experts, n, k, dtype, 0, 0, None) == -1
        assert word in lib.flymoe_last_error()
        assert lib.flymoe_grouped_gemm_wgrad(None, None, None, None, rows, experts, n, k, dtype, None) == -1
        assert word in lib.flymoe_last_error()
    assert lib.flymoe_grouped_gemm(64, 72, 64, 64, 4, 2, 8, 16, 2, 0, 0, None) == -1
    assert b"aligned" in lib.flymoe_last_error()
