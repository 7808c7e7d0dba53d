"""The differentiable router (gate, plan, permute, combine) against plain 64-bit implementations, and a whole expert layer
with an adapter-free backward pass as it would be trained."""
import pytest
import torch

from flydsl_b200.kernels.grouped_gemm import grouped_linear
from flydsl_b200.kernels.moe_routing import RoutedRows, moe_combine, moe_permute, route_rows, topk_gating
from flydsl_b200.kernels.topk_gating_softmax_kernel import build_topk_gating_softmax_module

pytestmark = pytest.mark.gpu
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, ref, slack, what):
    """One rounding to the type (half a step, or half the smallest subnormal) plus `slack`, what the fp32 steps before may add."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps / 2 + (1 + fi.eps) * slack
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {int((~(err <= tol)).sum())} of {err.numel()} off, worst {float(err.max()):.3g}"


# ------------------------------------------------------------------------- gate
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,topk,dtype", [(1, 1, 1, F32), (5, 2, 2, BF), (33, 8, 2, HF), (130, 60, 6, F32),
                                                       (257, 256, 8, BF), (64, 1000, 32, F32), (3, 1024, 1, HF)])
def test_gate_gradient(tokens, experts, topk, dtype, renormalize):
    g = gen(experts + topk)
    logits = (torch.randn((tokens, experts), generator=g, device="cuda") * 2).to(dtype).requires_grad_()
    dw = torch.randn((tokens, topk), generator=g, device="cuda")
    weights, ids = topk_gating(logits, topk, renormalize=renormalize)
    launch = build_topk_gating_softmax_module(experts, topk, {F32: "f32", BF: "bf16", HF: "f16"}[dtype], renormalize)
    w0, i0, p0 = torch.empty_like(weights), torch.empty_like(ids), torch.empty_like(ids)
    launch(logits.detach(), w0, i0, p0, tokens)
    assert torch.equal(weights, w0) and torch.equal(ids, i0) and not ids.requires_grad
    (d,) = torch.autograd.grad(weights, logits, dw)
    z = logits.detach().double().requires_grad_()
    p = z.softmax(1).gather(1, ids.long())
    w = p / p.sum(1, keepdim=True) if renormalize else p
    (ref,) = torch.autograd.grad(w, z, dw.double())
    # fp32: exponentials and quotients good to a few steps, sums of up to `experts` terms; the terms of a gradient are
    # at most w_i (|g_i| + sum |w g|) on the picks and p_e sum |w g| elsewhere
    inner = (w.detach() * dw.double()).abs().sum(1, keepdim=True)
    mag = z.softmax(1).detach() * inner
    mag = mag.scatter_add(1, ids.long(), w.detach() * (dw.double().abs() + inner))
    close(d, ref, (experts + 64) * 2.0 ** -23 * mag, "dlogits")


def test_gate_masked_and_degenerate_logits():
    inf = float("inf")
    logits = torch.tensor([[1.0, -inf, 2.0, -inf], [0.0, 0.0, 0.0, 0.0], [3.0, -inf, -inf, -inf],
                           [torch.finfo(F32).min, 1.0, torch.finfo(F32).min, 1.0]], device="cuda", requires_grad=True)
    for renorm in (True, False):
        weights, ids = topk_gating(logits, 2, renormalize=renorm)
        assert ids.tolist()[1] == [0, 1] and ids.tolist()[3] == [1, 3]
        (d,) = torch.autograd.grad(weights, logits, torch.ones_like(weights))
        assert bool(torch.isfinite(d).all())
        assert d[0, 1].item() == 0 and d[0, 3].item() == 0 and not bool(d[2].any())
        if renorm:
            assert float(d.abs().max()) <= 4 * 2.0 ** -24            # the weights sum to one whatever the logits


def test_gate_without_tokens():
    logits = torch.empty((0, 8), device="cuda", requires_grad=True)
    weights, ids = topk_gating(logits, 2)
    assert weights.shape == (0, 2) and ids.shape == (0, 2)
    (d,) = torch.autograd.grad(weights, logits, torch.empty((0, 2), device="cuda"))
    assert d.shape == (0, 8)


# ------------------------------------------------------------------------- plan, permute, combine
def random_ids(tokens, topk, experts, seed, dropped=0.0):
    g = gen(seed)
    ids = torch.rand((tokens, experts), generator=g, device="cuda").argsort(1)[:, :topk].int()
    if dropped:
        ids[torch.rand((tokens, topk), generator=g, device="cuda") < dropped] = -1
    return ids


ROUTES = [(1, 1, 1, 8, 0.0), (1, 8, 8, 16, 0.0), (7, 2, 5, 136, 0.3), (300, 8, 64, 72, 0.0), (64, 2, 8, 4096, 0.1),
          (1500, 6, 256, 264, 0.0), (20, 3, 4, 24, 1.0)]


@pytest.mark.parametrize("tokens,topk,experts,dim,dropped", ROUTES)
def test_plan_tables(tokens, topk, experts, dim, dropped):
    ids = random_ids(tokens, topk, experts, 3, dropped)
    plan = route_rows(ids, experts)
    flat = ids.reshape(-1).long()
    kept = flat >= 0
    order = torch.where(kept, flat, experts).argsort(stable=True)[: int(kept.sum())]
    n = order.numel()
    assert plan.num_valid_ids[0].item() == n
    assert torch.equal(plan.sorted_ids[:n].long(), (order % topk) << 24 | order // topk)
    counts = torch.bincount(flat[kept], minlength=experts)
    assert torch.equal(plan.offsets[1:].long(), counts.cumsum(0)) and plan.offsets[0].item() == 0
    want = torch.full((tokens * topk,), -1, device="cuda", dtype=torch.int32)
    want[order] = torch.arange(n, device="cuda", dtype=torch.int32)
    assert torch.equal(plan.row_index.reshape(-1), want)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens,topk,experts,dim,dropped", ROUTES)
def test_permute_and_combine(tokens, topk, experts, dim, dropped, dtype):
    plan = route_rows(random_ids(tokens, topk, experts, 4, dropped), experts)
    g = gen(5)
    x = torch.randn((tokens, dim), generator=g, device="cuda").to(dtype).requires_grad_()
    at = plan.row_index.long()
    has = (at >= 0).double()
    xs = moe_permute(x, plan)
    want = torch.zeros((tokens * topk, dim), dtype=dtype, device="cuda")
    want[at[at >= 0]] = x.detach()[:, None].expand(-1, topk, -1)[at >= 0]
    assert torch.equal(xs, want)
    dxs = torch.randn(xs.shape, generator=g, device="cuda").to(dtype)
    (dx,) = torch.autograd.grad(xs, x, dxs)
    terms = dxs.double()[at.clamp(min=0)] * has[..., None]
    close(dx, terms.sum(1), topk * 2.0 ** -23 * terms.abs().sum(1), "dx")

    rows = torch.randn((tokens * topk, dim), generator=g, device="cuda").to(dtype).requires_grad_()
    weights = torch.rand((tokens, topk), generator=g, device="cuda").requires_grad_()
    dout = torch.randn((tokens, dim), generator=g, device="cuda").to(dtype)
    out = moe_combine(rows, weights, plan)
    z, w, do = rows.detach().double()[at.clamp(min=0)] * has[..., None], weights.detach().double(), dout.double()
    close(out, (z * w[..., None]).sum(1), topk * 2.0 ** -23 * (z * w[..., None]).abs().sum(1), "out")
    drows, dw = torch.autograd.grad(out, (rows, weights), dout)
    ref = torch.zeros((tokens * topk, dim), dtype=torch.float64, device="cuda")
    ref[at[at >= 0]] = (do[:, None] * w[..., None])[at >= 0]
    close(drows, ref, 2.0 ** -23 * ref.abs(), "drows")
    close(dw, (z * do[:, None]).sum(2), dim * 2.0 ** -23 * (z * do[:, None]).abs().sum(2), "dweights")
    # only one of the two gradients
    (only,) = torch.autograd.grad(moe_combine(rows.detach(), weights, plan), (weights,), dout)
    assert torch.equal(only, dw)
    (only,) = torch.autograd.grad(moe_combine(rows, weights.detach(), plan), (rows,), dout)
    assert torch.equal(only, drows)


def test_what_autograd_refuses():
    plan = route_rows(random_ids(40, 2, 8, 6), 8)
    rows = torch.ones((80, 64), dtype=BF, device="cuda", requires_grad=True)
    w = torch.ones((40, 2), device="cuda", requires_grad=True)
    x = torch.ones((40, 64), device="cuda", requires_grad=True)
    logits = torch.ones((40, 8), device="cuda", requires_grad=True)
    for out, leaf in ((moe_combine(rows, w, plan), w), (moe_permute(x, plan), x), (topk_gating(logits, 2)[0], logits)):
        (first,) = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()
    for out, leaf in ((moe_combine(rows, w, plan), w), (moe_permute(x, plan), x)):
        plan.row_index.add_(0)                   # written after the forward pass
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaf)
    with torch.no_grad():
        assert not moe_combine(rows, w, plan).requires_grad and not topk_gating(logits, 2)[0].requires_grad
    with torch.inference_mode():
        made = route_rows(random_ids(40, 2, 8, 6), 8)
        assert torch.equal(moe_combine(moe_permute(x, made), w, made), x * 2)


def test_tables_that_do_not_belong_together_lead_nowhere():
    plan = route_rows(random_ids(40, 2, 8, 6), 8)
    bad = plan.row_index.clone().reshape(-1)
    bad[0], bad[1], bad[2], bad[3] = 10 ** 6, -5, bad[4], 79
    bad = RoutedRows(plan.sorted_ids, plan.num_valid_ids, plan.offsets, bad.view(40, 2))
    rows = torch.ones((80, 64), dtype=BF, device="cuda", requires_grad=True)
    w = torch.ones((40, 2), device="cuda", requires_grad=True)
    out = moe_combine(rows, w, bad)
    named = plan.sorted_ids.long()
    pair = (named & 0xFFFFFF) * 2 + (named >> 24)
    ok = bad.row_index.reshape(-1)[pair] == torch.arange(80, device="cuda")
    counts = torch.zeros(80, device="cuda").index_add_(0, pair[ok], torch.ones(int(ok.sum()), device="cuda"))
    assert torch.equal(out[:, 0].float(), counts.view(40, 2).sum(1))
    drows, dw = torch.autograd.grad(out, (rows, w), torch.ones_like(out))
    assert torch.equal(drows[:, 0].float(), ok.float())
    assert torch.equal(dw.reshape(-1), counts * 64)


# ------------------------------------------------------------------------- together
def plain_layer(x, logits, w1, w2, topk, ids):
    """An expert layer in the type of its inputs, routed to the given ids."""
    p = logits.softmax(1).gather(1, ids)
    p = p / p.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(w1.shape[0]):
        t, s = (ids == e).nonzero(as_tuple=True)
        gate, up = (x[t] @ w1[e].t()).chunk(2, 1)
        z = (torch.nn.functional.silu(gate) * up) @ w2[e].t()
        out = out.index_add(0, t, z * p[t, s, None])
    return out


def layer(x, logits, w1, w2, topk):
    weights, ids = topk_gating(logits, topk)
    plan = route_rows(ids, w1.shape[0])
    gate, up = grouped_linear(moe_permute(x, plan), w1, plan.offsets).chunk(2, 1)
    z = grouped_linear(torch.nn.functional.silu(gate) * up, w2, plan.offsets)
    return moe_combine(z, weights, plan), ids


def layer_inputs(tokens, dim, inter, experts, seed, dtype=BF):
    g = gen(seed)
    x = torch.randn((tokens, dim), generator=g, device="cuda").to(dtype)
    logits = torch.randn((tokens, experts), generator=g, device="cuda")
    w1 = (torch.randn((experts, 2 * inter, dim), generator=g, device="cuda") * dim ** -0.5).to(dtype)
    w2 = (torch.randn((experts, dim, inter), generator=g, device="cuda") * inter ** -0.5).to(dtype)
    dout = torch.randn((tokens, dim), generator=g, device="cuda").to(dtype)
    return x, logits, w1, w2, dout


@pytest.mark.parametrize("tokens,dim,inter,experts,topk", [(1, 64, 64, 4, 2), (200, 256, 136, 8, 2), (333, 128, 72, 32, 6)])
def test_a_trained_expert_layer(tokens, dim, inter, experts, topk):
    x, logits, w1, w2, dout = layer_inputs(tokens, dim, inter, experts, 11)
    leaves = [t.clone().requires_grad_() for t in (x, logits, w1, w2)]
    out, ids = layer(*leaves, topk)
    got = torch.autograd.grad(out, leaves, dout)
    wide = [t.double().requires_grad_() for t in (x, logits, w1, w2)]
    ref = plain_layer(*wide, topk, ids.long())
    want = torch.autograd.grad(ref, wide, dout.double())
    # Five tensors of the chain are rounded to bf16 on the way (rows, activation and its two factors, output; as many on
    # the way back), each by at most 2^-8 of a value: the 2-norm of a result is off by less than 10 such roundings.
    for name, a, b in zip(("out", "dx", "dlogits", "dw1", "dw2"), (out.detach(), *got), (ref.detach(), *want)):
        off = float((a.double() - b).norm() / b.norm())
        assert off <= 10 * 2.0 ** -8, f"{name}: {off:.3g}"


def test_a_captured_training_step_beside_an_eager_one():
    x, logits, w1, w2, dout = layer_inputs(96, 128, 64, 8, 12)
    sets = [(x, logits), (x.flip(0).contiguous(), logits.roll(1, 1).contiguous())]
    static = [t.clone().requires_grad_() for t in (x, logits, w1, w2)]
    eager = []
    for xi, li in sets:
        leaves = [t.clone().requires_grad_() for t in (xi, li, w1, w2)]
        out, _ = layer(*leaves, 2)
        eager.append((out.detach(), *torch.autograd.grad(out, leaves, dout)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept, _ = layer(*static, 2)                                 # an eager graph of the same leaves that stays alive
        torch.autograd.grad(kept, static, dout, retain_graph=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer(*static, 2)
        res = (out.detach(), *torch.autograd.grad(out, static, dout))
    for i in (1, 0, 1):
        with torch.no_grad():
            static[0].copy_(sets[i][0])
            static[1].copy_(sets[i][1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, eager[i]):
            assert torch.equal(a, b)


def test_rows_that_do_not_fit_the_plan_are_refused():
    plan = route_rows(random_ids(40, 2, 8, 6, 0.3), 8)
    used = int(plan.num_valid_ids[0])
    rows, w = torch.ones((81, 64), dtype=BF, device="cuda"), torch.ones((40, 2), device="cuda")
    want = moe_combine(rows[:80], w, plan)
    for count in (0, 40, used, 79, 81):
        with pytest.raises(ValueError, match="rows"):
            moe_combine(rows[:count], w, plan)
    # a plan cut off behind the pairs that have rows, and one with room behind its last row
    cut = RoutedRows(plan.sorted_ids[:used], *plan[1:])
    long = RoutedRows(torch.cat([plan.sorted_ids, plan.sorted_ids[:6]]), *plan[1:])
    assert used < 80 and torch.equal(moe_combine(rows[:used], w, cut), want) and torch.equal(moe_combine(rows, w, long), want)
    with pytest.raises(ValueError, match="rows"):
        moe_combine(rows[: used - 1], w, cut)
