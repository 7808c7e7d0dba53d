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
    for rows, k, rank, adapters, dtype, word in (
            (-1, 16, 8, 1, 2, b"rows"), (4, 12, 8, 1, 2, b"multiples of 8"), (4, 16, 4, 1, 2, b"rank"),
            (4, 16, 136, 1, 2, b"rank"), (4, 16, 8, 0, 2, b"adapters"), (4, 16, 8, 32768, 2, b"adapters"),
            (4, 16, 8, 1, 0, b"dtype"), (4, 16, 8, 1, 2, b"null")):
        assert lib.flymoe_lora_add(None, None, None, None, None, None, None, None, 0, rows, k, 16, rank, adapters, 0, dtype,
                                   None) == -1
        assert word in err()
        assert lib.flymoe_lora_backward(64, None, None, None, None, None, None, None, None, None, None, 0, rows, 16, k, rank,
                                        adapters, dtype, None) == -1
        assert word in err()
    assert lib.flymoe_lora_add(64, 64, 72, 64, 64, 64, 64, 64, 1 << 20, 4, 16, 16, 8, 1, 0, 2, None) == -1 and b"aligned" in err()
    assert lib.flymoe_lora_add(64, 64, 64, 64, 64, 64, 64, 64, 8, 4, 16, 16, 8, 1, 0, 2, None) == -4 and b"v_elems" in err()
    assert lib.flymoe_lora_backward(64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 8, 4, 16, 16, 8, 1, 2, None) == -4
    assert b"workspace" in err()
    assert lib.flymoe_lora_v_elems(0, 64, 8) == 0 and lib.flymoe_lora_v_elems(5, 64, 8) >= 40
    assert lib.flymoe_lora_backward_workspace_elems(5, 64, 64, 8, 2) >= 40
