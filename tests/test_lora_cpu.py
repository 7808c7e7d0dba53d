"""Adapters: what is refused, before anything is launched."""
import pytest
import torch

from flydsl_b200.kernels.lora import lora_add

BF = torch.bfloat16


def args(rows=4, k=16, n=24, rank=8, adapters=3):
    return dict(y=torch.zeros((rows, n), dtype=BF), x=torch.zeros((rows, k), dtype=BF),
                a=torch.zeros((adapters, rank, k), dtype=BF), b=torch.zeros((adapters, n, rank), dtype=BF),
                adapter_ids=torch.zeros(rows, dtype=torch.int32), scaling=torch.zeros(adapters))


@pytest.mark.parametrize("change,word", [
    ({}, "CUDA tensor"), ({"rank": 12}, "rank must be"), ({"rank": 136}, "rank must be"), ({"k": 12}, "multiples of 8"),
    ({"n": 4}, "multiples of 8"), ({"adapters": 0}, "adapters must be")])
def test_sizes(change, word):
    with pytest.raises(ValueError, match=word):
        lora_add(**args(**change))


@pytest.mark.parametrize("name", ["y", "a", "b", "adapter_ids", "scaling"])
def test_shapes(name):
    kw = args()
    kw[name] = torch.cat([kw[name], kw[name]])
    with pytest.raises(ValueError, match="must have shape"):
        lora_add(**kw)
    with pytest.raises(TypeError):
        lora_add(**{**args(), name: None})


def test_c_entries_refuse_bad_arguments(lib):
    err = lib.flymoe_last_error
    for rows, k, rank, adapters, splits, dtype, word in (
            (-1, 16, 8, 1, 1, 2, b"rows"), (4, 12, 8, 1, 1, 2, b"multiples of 8"), (4, 16, 4, 1, 1, 2, b"rank"),
            (4, 16, 136, 1, 1, 2, b"rank"), (4, 16, 8, 0, 1, 2, b"adapters"), (4, 16, 8, 1, 17, 2, b"splits"),
            (4, 16, 8, 1, 1, 0, b"dtype"), (4, 16, 8, 1, 1, 2, b"null")):
        assert lib.flymoe_lora_shrink(None, None, None, None, rows, k, rank, adapters, splits, 0, dtype, None) == -1
        assert word in err()
        assert lib.flymoe_lora_expand(None, None, None, None, None, None, rows, k, rank, adapters, splits, dtype, None) == -1
        assert word in err()
        assert lib.flymoe_lora_wgrad(64, 64, None, None, None, None, None, None, None, rows, k, 16, rank, adapters, splits,
                                     dtype, None) == -1
        assert word in err()
    assert lib.flymoe_lora_shrink(64, 72, 64, 64, 4, 16, 8, 1, 1, 0, 2, None) == -1 and b"aligned" in err()
    assert lib.flymoe_lora_wgrad(64, None, 64, 64, 64, 64, 64, 64, None, 4, 16, 16, 8, 1, 2, 2, None) == -1
    assert b"partial" in err()
    assert lib.flymoe_lora_transpose(None, None, 1, 0, 8, None) == -1
    assert 1 <= lib.flymoe_lora_shrink_splits(1, 7168) <= 16 and 1 <= lib.flymoe_lora_shrink_splits(8192, 64) <= 16
    assert lib.flymoe_lora_wgrad_splits(64, 4096, 4096, 16, 1) == 1
