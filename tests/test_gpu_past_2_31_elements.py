"""Tensors of more than 2^31 elements: rows behind that border against 64 bits, rows of the front against the same call on the
front alone."""
import pytest
import torch

from flydsl_b200.kernels.grouped_gemm import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad
from flydsl_b200.kernels.lora import lora_add
from flydsl_b200.kernels.moe_routing import RoutedRows, moe_combine, moe_permute

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()


def near(got, ref, mag, terms, what):
    """One rounding (half a step) after fp32 sums of `terms` terms, a step of the absolute products each; the adapters' middle
    factor keeps 16 bits (bf16) of its own."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + (1 + fi.eps) * (terms * 2.0 ** -23 + 2.0 ** -17) * mag
    assert bool(((got.double() - ref).abs() <= tol).all()), what


def fill(*shape, dtype=BF, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_adapters(dtype):
    rows, k, n, rank = 140000, 16, 16384, 16     # 2.29e9 outputs
    y, x = fill(rows, n, dtype=dtype), fill(rows, k, dtype=dtype, seed=1)
    a, b = fill(3, rank, k, dtype=dtype, seed=2) / 4, fill(3, n, rank, dtype=dtype, seed=3) / 4
    ids = (torch.arange(rows, device="cuda") // 50 % 4 - 1).int()
    scaling = torch.tensor([0.5, 1.0, 2.0], device="cuda")
    at = torch.cat([torch.arange(3), torch.arange(131000, 131300), torch.arange(rows - 300, rows)]).cuda()
    base = y[at].double()
    x.requires_grad_()
    out = lora_add(y, x, a, b, ids, scaling)
    (dx,) = torch.autograd.grad(out, x, y)       # y doubles as the gradient
    for l in range(3):
        s = at[ids[at] == l]
        here = ids[at] == l
        v, va = x.detach()[s].double() @ a[l].double().t(), x.detach()[s].double().abs() @ a[l].double().abs().t()
        sc = float(scaling[l])
        near(out.detach()[s], base[here] + sc * v @ b[l].double().t(), base[here].abs() + sc * va @ b[l].double().abs().t(), k + rank, "out")
        dv, dva = base[here] @ b[l].double(), base[here].abs() @ b[l].double().abs()
        near(dx[s], sc * dv @ a[l].double(), sc * dva @ a[l].double().abs(), n + rank, "dx")
    none = at[ids[at] < 0]
    assert torch.equal(out.detach()[none], y[none]) and not bool(dx[none].any())


def test_grouped_products():
    rows, k, n, experts = 300000, 64, 8192, 5    # 2.46e9 outputs
    x, w = fill(rows, k), fill(experts, n, k, seed=1)
    offsets = torch.tensor([0, 262000, 262000, 262333, 270001, rows - 7], dtype=torch.int32, device="cuda")
    y = grouped_gemm(x, w, offsets)
    assert not bool(y[-7:].any())
    for e, (i, j) in enumerate(((0, 3), (262000, 262000), (262000, 262333), (269900, 270001), (rows - 300, rows - 7))):
        xe, we = x[i:j].double(), w[e].double()
        near(y[i:j], xe @ we.t(), xe.abs() @ we.abs().t(), k, "y")
    dx = grouped_gemm_dgrad(y, w, offsets)
    dw = grouped_gemm_wgrad(y, x, offsets)
    for e, (i, j) in ((2, (262000, 262333)), (4, (rows - 300, rows - 7))):
        de, we = y[i:j].double(), w[e].double()
        near(dx[i:j], de @ we, de.abs() @ we.abs(), n, "dx")
    de, xe = y[262000:262333].double(), x[262000:262333].double()
    near(dw[2], de.t() @ xe, de.t().abs() @ xe.abs(), 333, "dw")
    assert not bool(dw[1].any())
    del x, w, y, dx, dw
    w = fill(40, 8192, 8192, seed=2)             # 2.68e9 weights
    x = fill(80, 8192, seed=3)
    offsets = (torch.arange(41, device="cuda") * 2).int()
    y = grouped_gemm(x, w, offsets)
    near(y[78:], x[78:].double() @ w[39].double().t(), x[78:].double().abs() @ w[39].double().abs().t(), 8192, "y")
    dw = grouped_gemm_wgrad(y, x, offsets, out=w)
    near(dw[39], y[78:].double().t() @ x[78:].double(), y[78:].double().t().abs() @ x[78:].double().abs(), 2, "dw")


def test_routed_rows():
    tokens, topk, dim = 70000, 4, 8192           # 2.29e9 elements in expert order
    pairs = tokens * topk
    order = torch.randperm(pairs, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    row_index = torch.empty_like(order)
    row_index[order] = torch.arange(pairs, device="cuda")
    plan = RoutedRows((order % topk << 24 | order // topk).int(), torch.tensor([pairs, 0], dtype=torch.int32, device="cuda"),
                      torch.zeros(2, dtype=torch.int32, device="cuda"), row_index.int().view(tokens, topk))
    x = fill(tokens, dim)
    rows = moe_permute(x, plan)
    at = torch.cat([torch.arange(5), torch.arange(262100, 262200), torch.arange(pairs - 100, pairs)]).cuda()
    assert torch.equal(rows[at], x[order[at] // topk])
    weights = torch.rand((tokens, topk), device="cuda", requires_grad=True)
    rows.requires_grad_()
    out = moe_combine(rows, weights, plan)
    some = torch.cat([torch.arange(200), torch.arange(tokens - 200, tokens)]).cuda()
    z, w = x[some].double(), weights.detach()[some].double()
    near(out.detach()[some], z * w.sum(1, keepdim=True), z.abs() * w.sum(1, keepdim=True), topk, "out")
    drows, dw = torch.autograd.grad(out, (rows, weights), x)
    ref = x[order[at] // topk].double() * weights.detach().reshape(-1)[order[at]][:, None].double()
    near(drows[at], ref, ref.abs(), 1, "drows")
    near(dw[some], z.square().sum(1, keepdim=True).expand(-1, topk), z.square().sum(1, keepdim=True).expand(-1, topk), dim, "dw")
