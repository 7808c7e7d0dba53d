"""What autograd may hand to the operators: forward-mode tangents, gradients in any order and place."""
import pytest
import torch
from torch.autograd import forward_ad

from flydsl_b200.kernels.grouped_gemm import grouped_linear
from flydsl_b200.kernels.lora import lora_add
from flydsl_b200.kernels.moe_routing import moe_combine, moe_permute, route_rows, topk_gating

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def calls(rows=40):
    """name -> (function, differentiable inputs, the rest)"""
    g = torch.Generator(device="cuda").manual_seed(21)

    def r(*shape, dtype=BF):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    ids = torch.rand((rows, 8), generator=g, device="cuda").argsort(1)[:, :2].int()
    plan = route_rows(ids, 8)
    bounds = torch.tensor([0, rows // 4, rows // 4, rows - 3], dtype=torch.int32, device="cuda")
    adapter = torch.randint(-1, 4, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return {
        "grouped_linear": (grouped_linear, (r(rows, 72), r(3, 64, 72)), (bounds,)),
        "lora_add": (lambda y, x, a, b, s, i: lora_add(y, x, a, b, i, s),
                     (r(rows, 64), r(rows, 72), r(4, 16, 72), r(4, 64, 16), r(4, dtype=torch.float32)), (adapter,)),
        "topk_gating": (lambda z: topk_gating(z, 2)[0], (r(rows, 8, dtype=torch.float32),), ()),
        "moe_permute": (moe_permute, (r(rows, 64),), (plan,)),
        "moe_combine": (moe_combine, (r(rows * 2, 64), r(rows, 2, dtype=torch.float32)), (plan,)),
    }


NAMES = ["grouped_linear", "lora_add", "topk_gating", "moe_permute", "moe_combine"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_not_dropped(name):
    f, inputs, rest = calls()[name]
    plain = f(*inputs, *rest)
    for i, t in enumerate(inputs):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward mode"):
                    f(*inputs[:i], dual, *inputs[i + 1:], *rest)
            assert torch.equal(f(*inputs, *rest), plain)             # inputs without a tangent, beside one
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        y, x, a, b, s = calls()["lora_add"][1]
        lora_add(forward_ad.make_dual(y, y), x, a, b, calls()["lora_add"][2][0], s, out=torch.empty_like(y))


@pytest.mark.parametrize("rows", [40, 600])
@pytest.mark.parametrize("name", NAMES)
def test_gradients_of_any_strides_and_alignment(name, rows):
    f, inputs, rest = calls(rows)[name]
    leaves = [t.clone().requires_grad_(i < 4) for i, t in enumerate(inputs)]       # the adapters' scaling has no gradient
    out = f(*leaves, *rest)
    leaves = leaves[:4]
    dout = torch.randn(out.shape, generator=torch.Generator(device="cuda").manual_seed(22), device="cuda").to(out.dtype)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    shifted = torch.empty(out.numel() + 1, dtype=out.dtype, device="cuda")[1:].view(out.shape).copy_(dout)
    flipped = dout.t().contiguous().t()
    joined = torch.cat([dout, dout], 1)[:, : out.shape[1]]
    assert shifted.is_contiguous() and shifted.data_ptr() % 16 and not flipped.is_contiguous()
    for given in (shifted, flipped, joined):
        for a, b in zip(torch.autograd.grad(out, leaves, given, retain_graph=True), want):
            assert torch.equal(a, b)
    # as a loss makes them: behind a single number in one tensor, and one value for all of it
    both = torch.cat([torch.ones(1, dtype=out.dtype, device="cuda", requires_grad=True), out.reshape(-1)])
    pieces = torch.cat([torch.zeros(1, dtype=out.dtype, device="cuda"), dout.reshape(-1)])
    for a, b in zip(torch.autograd.grad(both, leaves, pieces, retain_graph=True), want):
        assert torch.equal(a, b)
    ones = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
    for a, b in zip(torch.autograd.grad(out.sum(), leaves), ones):
        assert torch.equal(a, b)
