"""The differentiable router: what is refused, before anything is launched."""
import pytest
import torch

from flydsl_b200.kernels.moe_routing import RoutedRows, moe_combine, moe_permute, route_rows, topk_gating

I32 = torch.int32


def test_arguments_are_checked():
    with pytest.raises(ValueError, match="CUDA tensor"):
        topk_gating(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        route_rows(torch.zeros((4, 2), dtype=I32), 8)
    with pytest.raises(TypeError):
        topk_gating([[0.0]], 1)
    plan = RoutedRows(torch.zeros(8, dtype=I32), torch.zeros(2, dtype=I32), torch.zeros(9, dtype=I32),
                      torch.zeros((4, 2), dtype=I32))
    with pytest.raises(ValueError, match="CUDA tensor"):
        moe_permute(torch.zeros(4, 8), plan)
    with pytest.raises(ValueError, match="CUDA tensor"):
        moe_combine(torch.zeros(8, 8), torch.zeros(4, 2), plan)


def test_c_entries_refuse_bad_arguments(lib):
    err = lib.flymoe_last_error
    assert lib.flymoe_topk_gating_softmax_backward(None, 0, None, None, None, None, 4, 2048, 2, 1, None) == -1
    assert b"num_experts" in err()
    assert lib.flymoe_topk_gating_softmax_backward(None, 0, None, None, None, None, 4, 8, 9, 1, None) == -1
    assert b"topk" in err()
    assert lib.flymoe_topk_gating_softmax_backward(None, 0, None, None, None, None, 4, 8, 2, 1, None) == -1
    assert b"null" in err()
    assert lib.flymoe_topk_gating_softmax_backward(64, 3, 64, 64, 64, 64, 4, 8, 2, 1, None) == -1 and b"dtype" in err()
    assert lib.flymoe_route_tables(None, None, None, None, None, 4, 2, 0, 8, None) == -1 and b"experts" in err()
    assert lib.flymoe_route_tables(None, None, None, None, None, 4, 256, 8, 8, None) == -1 and b"sizes" in err()
    assert lib.flymoe_route_tables(None, None, None, None, None, 4, 2, 8, 8, None) == -1 and b"null" in err()
    assert lib.flymoe_permute_rows(64, 64, 64, 64, 64, 4, 2, 8, 24, None) == -1 and b"multiple of 16" in err()
    assert lib.flymoe_permute_rows(72, 64, 64, 64, 64, 4, 2, 8, 32, None) == -1 and b"aligned" in err()
    assert lib.flymoe_combine_rows(64, 64, 64, 64, 64, 64, 4, 2, 8, 12, 2, None) == -1 and b"dim" in err()
    assert lib.flymoe_combine_rows(64, 64, 64, 64, 64, 64, 4, 2, 8, 16, 3, None) == -1 and b"dtype" in err()
    assert lib.flymoe_combine_rows_backward(None, 64, 64, 64, 64, 64, 64, 64, 4, 2, 8, 16, 2, None) == -1 and b"null" in err()
    assert lib.flymoe_combine_rows_backward(64, 64, 64, 72, 64, 64, 64, 64, 4, 2, 8, 16, 2, None) == -1 and b"aligned" in err()
